// The norms around a block, fused with its gate and the residual scale, and their gradients:
//
//   p = y * rsqrt(mean(y^2) + eps) * (1 + post_w)          (p = y without post_w)
//   r = round(res_scale * res + branch_scale * gate * p)   the residual stream, in its type
//   x = round(r * rsqrt(mean(r^2) + eps) * (1 + pre_w))    (only with pre_w) the next block's input
//
// The gate is one value per token, per channel or per element, or absent. p stays in fp32 between
// the norm and the residual; x is computed from the rounded r, which is what the next layer and
// the gradients read back. Backward, with s = rsqrt(mean(r^2) + eps), q = rsqrt(mean(y^2) + eps):
//
//   g   = d x (1 + pre_w);  du = s (g - r s mean(g r s)) + d r;   d pre_w = sum_t d x r s
//   d res = res_scale du;   d gate = branch_scale du p, summed over what the gate broadcasts
//   dp  = branch_scale gate du;                                     d post_w = sum_t dp y q
//   d y = q (h - y q mean(h y q)),  h = dp (1 + post_w)             (d y = dp without post_w)
//
// HBM-bound in both directions: every tensor is read and written once, 8 columns a thread held in
// registers across the reductions. A row takes a wave up to 512 columns, a workgroup of 256 threads
// up to 2048, of 512 up to 4096, of 1024 up to 8192. Sums are taken in a fixed order: in fp32 per
// thread over its columns, then in a butterfly in each wave and over the waves, where squares are summed
// in fp64; the weights' gradients in fp32 per workgroup over its rows, then over the workgroups.
#include <algorithm>
#include <initializer_list>

#include "common.h"
#include "elem.h"
#include "launch.h"

namespace {

constexpr int kMaxHidden = 8192;
enum { kGateNone = 0, kGateToken = 1, kGateChannel = 2, kGateFull = 3 };

// The value of lane i ^ M.
template <int M>
MOE_DEV double partner(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __float_as_uint(xor_partner<M>(__uint_as_float((uint32_t)b)));
  const uint32_t hi = __float_as_uint(xor_partner<M>(__uint_as_float((uint32_t)(b >> 32))));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

template <int M>
MOE_DEV float partner(float v) { return xor_partner<M>(v); }

// Sums of N values over the NT threads of a row (all threads get them). A is double for the sums of
// squares, at a cost that HBM's time mostly hides: what is left of their error are the 8 fp32 roundings of
// a thread's own columns, and a norm's factor is off by at most 5 half steps of fp32 (the root halves
// them, and it is rounded itself) whatever the row's width. A is float for the means that the gradients
// subtract. NT = 64: no barrier.
template <int NT, int N, class A>
MOE_DEV void row_sums(const float (&part)[N], A (&v)[N], A (*s_part)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = part[i];
    v[i] += partner<32>(v[i]);
    v[i] += partner<16>(v[i]);
    v[i] += partner<8>(v[i]);
    v[i] += partner<4>(v[i]);
    v[i] += partner<2>(v[i]);
    v[i] += partner<1>(v[i]);
  }
  if constexpr (NT > 64) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();  // the previous sums have been read
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) s_part[wave][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = A(0);
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) v[i] += s_part[w][i];
    }
  }
}

// 1 / sqrt(sum / H + eps): the hardware's approximation and a Newton step in 64 bits.
MOE_DEV float inv_rms(double sum, double inv_h, float eps) {
  const double m = sum * inv_h + (double)eps;
  const float v = (float)m;
  if (!(v >= 0x1p-100f && v < __builtin_inff())) return 1.0f / __builtin_sqrtf(v);
  const double r = (double)__builtin_amdgcn_rsqf(v);
  return (float)(r + 0.5 * r * (1.0 - m * r * r));
}

struct NormArgs {
  const void* y;
  const void* res;  // forward: the residual; backward: r
  const void* post;
  const void* gate;
  const void* pre;
  int gate_kind;
  int T, H;
  float res_scale, branch_scale, eps;
};

template <int DT, int NT, bool VEC>
MOE_DEV void load_gate(const NormArgs& a, int64_t t, int tid, float (&g)[8]) {
  using T = typename Elem<DT>::T;
  const T* p = static_cast<const T*>(a.gate);
  if (a.gate_kind == kGateFull) {
    Cols<DT, NT, VEC>::load(p + t * a.H, tid, a.H, g);
  } else if (a.gate_kind == kGateChannel) {
    Cols<DT, NT, VEC>::load(p, tid, a.H, g);
  } else {
    const float v = a.gate_kind == kGateToken ? Elem<DT>::get(p[t]) : 1.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = v;
  }
}

template <int NT>
constexpr int block_threads() { return NT < 256 ? 256 : NT; }

template <int DT, int NT, bool VEC>
__global__ __launch_bounds__(block_threads<NT>()) void block_norm_kernel(NormArgs a, void* res_out,
                                                                         void* x_out) {
  using T = typename Elem<DT>::T;
  using C = Cols<DT, NT, VEC>;
  __shared__ double s_part[NT / 64][1];
  const double inv_h = 1.0 / (double)a.H;
  const int tid = threadIdx.x % NT;
  const int rows = block_threads<NT>() / NT;
  const int sub = __builtin_amdgcn_readfirstlane((int)threadIdx.x / NT);
  for (int64_t t = (int64_t)blockIdx.x * rows + sub; t < a.T; t += (int64_t)gridDim.x * rows) {
    float p[8], r[8], g[8];
    C::load(static_cast<const T*>(a.y) + t * a.H, tid, a.H, p);
    C::load(static_cast<const T*>(a.res) + t * a.H, tid, a.H, r);
    load_gate<DT, NT, VEC>(a, t, tid, g);
    if (a.post) {
      float w[8];
      C::load(static_cast<const T*>(a.post), tid, a.H, w);
      float ss[1] = {0.0f};
#pragma unroll
      for (int e = 0; e < 8; ++e) ss[0] = __builtin_fmaf(p[e], p[e], ss[0]);
      double sum[1];
      row_sums<NT>(ss, sum, s_part);
      const float q = inv_rms(sum[0], inv_h, a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = (p[e] * q) * (1.0f + w[e]);
    }
    float ss[1] = {0.0f};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      r[e] = rounded<DT>(a.res_scale * r[e] + (a.branch_scale * g[e]) * p[e]);
      if (C::col(tid, e) < a.H) ss[0] = __builtin_fmaf(r[e], r[e], ss[0]);
    }
    C::store(static_cast<T*>(res_out) + t * a.H, tid, a.H, r);
    if (a.pre) {
      float w[8];
      C::load(static_cast<const T*>(a.pre), tid, a.H, w);
      double sum[1];
      row_sums<NT>(ss, sum, s_part);
      const float s = inv_rms(sum[0], inv_h, a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = (r[e] * s) * (1.0f + w[e]);
      C::store(static_cast<T*>(x_out) + t * a.H, tid, a.H, r);
    }
  }
}

struct NormGrads {
  const void* dr;  // nullable
  const void* dx;  // nullable (then pre is not looked at)
  void* dy;        // the outputs are nullable
  void* dres;
  void* dgate;     // token and full gates
  float* part;     // [3][partials][H]: d post_w, d gate per channel, d pre_w
  int partials;
  bool post, gate, pre;  // which of them are wanted
};

// The next row's loads are in flight while a row is worked on (two reductions with their barriers):
// 16384 x 2048 bf16 with both norms and a channel gate 140 -> 87 us, 4.6 TB/s.
template <int DT, int NT, bool VEC>
__global__ __launch_bounds__(block_threads<NT>()) void block_norm_backward_kernel(NormArgs a,
                                                                                  NormGrads d) {
  using T = typename Elem<DT>::T;
  using C = Cols<DT, NT, VEC>;
  using Raw = RawCols<DT, NT, VEC>;
  __shared__ double s3[NT / 64][3];
  __shared__ float s2[NT / 64][2];
  const double inv_h = 1.0 / (double)a.H;
  const int tid = threadIdx.x % NT, H = a.H;
  const int rows = block_threads<NT>() / NT;
  const int sub = __builtin_amdgcn_readfirstlane((int)threadIdx.x / NT);
  const int64_t stride = (int64_t)gridDim.x * rows;
  const bool post = a.post != nullptr, pre = d.dx != nullptr, dr = d.dr != nullptr;
  Raw wpost{}, wpre{}, gate{};
  // The weights' gradients over the workgroup's rows: in registers, or for 1024 threads, which have
  // 128 each, in LDS, a thread's own columns behind each other (spilled, with the next row in
  // flight too, 4096 x 8192 took 190 us instead of 120).
  constexpr bool kAhead = NT < 1024;
  __shared__ f32x4 s_sum[kAhead ? 1 : 6 * NT];
  float apost[8], agate[8], apre[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) apost[e] = agate[e] = apre[e] = 0.0f;
  auto at = [&](int which, float (&v)[8], bool put) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f32x4& m = s_sum[(2 * which + h) * NT + tid];
      if (put) {
        m = f32x4{v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
      } else {
        const f32x4 d = m;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * h + j] = d[j];
      }
    }
  };
  if constexpr (!kAhead) {
    at(0, apost, true);
    at(1, agate, true);
    at(2, apre, true);
  }
  if (post) wpost.load(static_cast<const T*>(a.post), tid, H);
  if (pre) wpre.load(static_cast<const T*>(a.pre), tid, H);
  if (a.gate_kind == kGateChannel) gate.load(static_cast<const T*>(a.gate), tid, H);
  struct Row {
    Raw y, r, dx, dr, gate;
    float token;
  };
  Row next{};
  auto load = [&](int64_t t) {
    const int64_t o = min(t, (int64_t)a.T - 1) * H;  // past the last row: read again, not used
    next.y.load(static_cast<const T*>(a.y) + o, tid, H);
    if (pre) {
      next.r.load(static_cast<const T*>(a.res) + o, tid, H);
      next.dx.load(static_cast<const T*>(d.dx) + o, tid, H);
    }
    if (dr) next.dr.load(static_cast<const T*>(d.dr) + o, tid, H);
    if (a.gate_kind == kGateFull) next.gate.load(static_cast<const T*>(a.gate) + o, tid, H);
    if (a.gate_kind == kGateToken) next.token = Elem<DT>::get(static_cast<const T*>(a.gate)[o / H]);
  };
  const int64_t first = (int64_t)blockIdx.x * rows + sub;
  if (kAhead && first < a.T) load(first);
  for (int64_t t = first; t < a.T; t += stride) {
    if (!kAhead) load(t);
    Row row = next;
    if (kAhead) load(t + stride);
    if (a.gate_kind == kGateChannel) row.gate = gate;
    float part[3] = {0.0f, 0.0f, 0.0f};  // y^2, r^2, d x (1 + pre_w) r
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = row.y.get(e, tid, H);
      part[0] = __builtin_fmaf(y, y, part[0]);
    }
    if (pre) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float r = row.r.get(e, tid, H);
        part[1] = __builtin_fmaf(r, r, part[1]);
        part[2] = __builtin_fmaf(row.dx.get(e, tid, H) * (1.0f + wpre.get(e, tid, H)), r, part[2]);
      }
    }
    double sum[3] = {0.0, 0.0, 0.0};
    if (post || pre) row_sums<NT>(part, sum, s3);
    float du[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) du[e] = dr ? row.dr.get(e, tid, H) : 0.0f;
    if (pre) {
      const float s = inv_rms(sum[1], inv_h, a.eps);
      const float m = (float)(sum[2] * inv_h) * s;  // mean(g r s)
      if constexpr (!kAhead) at(2, apre, false);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float rh = row.r.get(e, tid, H) * s, dx = row.dx.get(e, tid, H);
        du[e] += s * (dx * (1.0f + wpre.get(e, tid, H)) - rh * m);
        apre[e] = __builtin_fmaf(dx, rh, apre[e]);
      }
      if constexpr (!kAhead) at(2, apre, true);
    }
    if (d.dres) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = a.res_scale * du[e];
      C::store(static_cast<T*>(d.dres) + t * H, tid, H, o);
    }
    const float q = post ? inv_rms(sum[0], inv_h, a.eps) : 1.0f;
    const float one = a.gate_kind == kGateToken ? row.token : 1.0f;
    const bool wide = a.gate_kind >= kGateChannel;
    const bool full = a.gate_kind == kGateFull && d.dgate;
    float dg[8], dp[8];
    float some[2] = {0.0f, 0.0f};  // h y, d gate
    if constexpr (!kAhead) {
      at(0, apost, false);
      at(1, agate, false);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = row.y.get(e, tid, H), yh = y * q;
      const float w1 = post ? 1.0f + wpost.get(e, tid, H) : 1.0f;
      const float db = a.branch_scale * du[e];
      dg[e] = db * (yh * w1);
      dp[e] = db * (wide ? row.gate.get(e, tid, H) : one);
      apost[e] = __builtin_fmaf(dp[e], yh, apost[e]);
      agate[e] += dg[e];
      dp[e] *= w1;
      if (C::col(tid, e) < H) {  // 0 times a gate of infinity outside the row is no part of it
        some[0] = __builtin_fmaf(dp[e], y, some[0]);
        some[1] += dg[e];
      }
    }
    if constexpr (!kAhead) {
      at(0, apost, true);
      at(1, agate, true);
    }
    const bool token = a.gate_kind == kGateToken && d.dgate;
    float tot[2] = {0.0f, 0.0f};
    if (post || token) row_sums<NT>(some, tot, s2);
    if (token && tid == 0) static_cast<T*>(d.dgate)[t] = Elem<DT>::put(tot[1]);
    if (full) C::store(static_cast<T*>(d.dgate) + t * H, tid, H, dg);
    if (d.dy) {
      if (post) {
        const float m = (tot[0] * (float)inv_h) * q;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          dp[e] = q * (dp[e] - (row.y.get(e, tid, H) * q) * m);
      }
      C::store(static_cast<T*>(d.dy) + t * H, tid, H, dp);
    }
  }
  const int64_t me = first, all = (int64_t)d.partials * H;
  if constexpr (!kAhead) {
    at(0, apost, false);
    at(1, agate, false);
    at(2, apre, false);
  }
  Cols<kFp32, NT, VEC> f;
  if (d.post) f.store(d.part + me * H, tid, H, apost);
  if (d.gate) f.store(d.part + all + me * H, tid, H, agate);
  if (d.pre) f.store(d.part + 2 * all + me * H, tid, H, apre);
}

// The weights' gradients from the workgroups' sums: 32 columns a workgroup, 32 threads a column over
// strided partials, then those 32 in order.
constexpr int kSumCols = 32;
struct SumOut {
  void* out[3];
};
template <int DT>
__global__ __launch_bounds__(1024) void block_norm_sum_kernel(const float* part, int partials,
                                                              int H, SumOut o) {
  __shared__ float s_sum[32][kSumCols + 1];
  const int which = blockIdx.y;
  if (!o.out[which]) return;
  const int lane = threadIdx.x % kSumCols, slot = threadIdx.x / kSumCols;
  const int c = blockIdx.x * kSumCols + lane;
  const float* p = part + (int64_t)which * partials * H;
  float s = 0.0f;
  if (c < H) {
#pragma unroll 8
    for (int i = slot; i < partials; i += 32) s += p[(int64_t)i * H + c];
  }
  s_sum[slot][lane] = s;
  __syncthreads();
  if (slot == 0 && c < H) {
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v += s_sum[i][lane];
    static_cast<typename Elem<DT>::T*>(o.out[which])[c] = Elem<DT>::put(v);
  }
}

int threads_of(int H) { return H <= 512 ? 64 : H <= 2048 ? 256 : H <= 4096 ? 512 : 1024; }
int rows_of(int nt) { return nt < 256 ? 256 / nt : 1; }

// Workgroups of the backward pass: each keeps the weights' gradients of its rows in registers and
// writes them once.
int backward_groups(int T, int H) {
  const int nt = threads_of(H), rows = rows_of(nt);
  const int most = nt > 256 ? 512 : 768;
  return std::max(1, std::min((T - 1) / rows + 1, most));  // T + rows may pass 32 bits
}

#define MOE_NORM_NT(LAUNCH)                      \
  if (nt == 64) {                                \
    if (vec) LAUNCH(64, true); else LAUNCH(64, false);     \
  } else if (nt == 256) {                        \
    if (vec) LAUNCH(256, true); else LAUNCH(256, false);   \
  } else if (nt == 512) {                        \
    if (vec) LAUNCH(512, true); else LAUNCH(512, false);   \
  } else {                                       \
    if (vec) LAUNCH(1024, true); else LAUNCH(1024, false); \
  }

template <int DT>
hipError_t launch_forward(const NormArgs& a, void* res_out, void* x_out, bool vec, hipStream_t s) {
  const int nt = threads_of(a.H), rows = rows_of(nt);
  const dim3 grid((unsigned)std::min<int64_t>((a.T + (int64_t)rows - 1) / rows, 1 << 20));
#define MOE_NORM_FWD(NT, V)                                                                  \
  hipLaunchKernelGGL((block_norm_kernel<DT, NT, V>), grid, dim3(block_threads<NT>()), 0, s, a, \
                     res_out, x_out)
  MOE_NORM_NT(MOE_NORM_FWD)
#undef MOE_NORM_FWD
  return hipGetLastError();
}

template <int DT>
hipError_t launch_backward(const NormArgs& a, const NormGrads& d, void* dpost, void* dgate_channel,
                           void* dpre, bool vec, hipStream_t s) {
  const int nt = threads_of(a.H);
  const dim3 grid((unsigned)backward_groups(a.T, a.H));
#define MOE_NORM_BWD(NT, V)                                                                     \
  hipLaunchKernelGGL((block_norm_backward_kernel<DT, NT, V>), grid, dim3(block_threads<NT>()), 0, \
                     s, a, d)
  MOE_NORM_NT(MOE_NORM_BWD)
#undef MOE_NORM_BWD
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !(dpost || dgate_channel || dpre)) return e;
  hipLaunchKernelGGL(block_norm_sum_kernel<DT>, dim3((a.H + kSumCols - 1) / kSumCols, 3),
                     dim3(1024), 0, s, d.part, d.partials, a.H, SumOut{{dpost, dgate_channel, dpre}});
  return hipGetLastError();
}
#undef MOE_NORM_NT

int check_norm(const char* what, int32_t T, int32_t hidden, int32_t dtype, const void* gate,
               int32_t gate_kind, float eps) {
  if (dtype < kBf16 || dtype > kFp32)
    return op_fail(MOE_ERR_UNSUPPORTED, "%s: dtype=%d (0 bf16, 1 fp16, 2 fp32)", what, dtype);
  if (T < 0 || hidden < 1 || hidden > kMaxHidden)
    return op_fail(MOE_ERR_SHAPE, "%s: T=%d hidden=%d (hidden in [1, 8192])", what, T, hidden);
  if (gate_kind < kGateNone || gate_kind > kGateFull)
    return op_fail(MOE_ERR_UNSUPPORTED, "%s: gate_kind=%d", what, gate_kind);
  // A channel gate is read ahead of the rows; the other kinds hold nothing where there are no tokens.
  if ((gate != nullptr) != (gate_kind != kGateNone) && (T > 0 || gate_kind == kGateChannel))
    return op_fail(MOE_ERR_NULL, "%s: gate and gate_kind must be given together", what);
  if (!(eps >= 0.0f)) return op_fail(MOE_ERR_SHAPE, "%s: eps must be >= 0", what);
  return MOE_OK;
}

// A tensor's memory.
struct Span {
  const void* p;
  int64_t bytes;
};
int64_t row_bytes(int H, int dtype) { return H * dtype_bytes(dtype); }
int64_t gate_bytes(int kind, int T, int H, int dtype) {
  return (kind == kGateNone ? 0 : kind == kGateToken ? T : kind == kGateChannel ? H : (int64_t)T * H) *
         dtype_bytes(dtype);
}

bool vec_ok(int H, std::initializer_list<const void*> ps) {
  if (H % 8 != 0) return false;
  for (const void* p : ps)
    if (!aligned16(p)) return false;
  return true;
}

}  // namespace

extern "C" {

int moe_block_norm_v1(const void* y, const void* res, int32_t T, int32_t hidden, int32_t dtype,
                      const void* post_w, const void* gate, int32_t gate_kind, float res_scale,
                      float branch_scale, const void* pre_w, float eps, void* res_out, void* x_out,
                      void* stream) {
  const int rc = check_norm("block norm", T, hidden, dtype, gate, gate_kind, eps);
  if (rc) return rc;
  if (T == 0) return MOE_OK;
  if (!y || !res || !res_out || (pre_w && !x_out))
    return op_fail(MOE_ERR_NULL, "block norm: NULL pointer");
  const int64_t n = (int64_t)T * hidden * dtype_bytes(dtype);
  const Span outs[] = {{res_out, n}, {pre_w ? x_out : nullptr, n}};
  const Span ins[] = {{y, n}, {post_w, row_bytes(hidden, dtype)}, {pre_w, row_bytes(hidden, dtype)},
                      {gate, gate_bytes(gate_kind, T, hidden, dtype)}};
  bool shared = overlaps(outs[0].p, n, outs[1].p, n) || overlaps(outs[1].p, n, res, n) ||
                (res_out != res && overlaps(res_out, n, res, n));
  for (const Span& o : outs)
    for (const Span& i : ins) shared |= overlaps(o.p, o.bytes, i.p, i.bytes);
  if (shared)
    return op_fail(MOE_ERR_SHAPE,
                   "block norm: outputs must not overlap inputs or each other (res_out may be res)");
  const NormArgs a{y, res, post_w, gate, pre_w, gate_kind, T, hidden, res_scale, branch_scale, eps};
  const bool vec = vec_ok(hidden, {y, res, post_w, pre_w, res_out, x_out}) &&
                   (gate_kind < kGateChannel || aligned16(gate));
  const auto s = (hipStream_t)stream;
  MOE_OP_HIP(dtype == kBf16   ? launch_forward<kBf16>(a, res_out, x_out, vec, s)
             : dtype == kFp16 ? launch_forward<kFp16>(a, res_out, x_out, vec, s)
                              : launch_forward<kFp32>(a, res_out, x_out, vec, s),
             "block norm");
  return MOE_OK;
}

int64_t moe_block_norm_workspace_bytes_v1(int32_t T, int32_t hidden) {
  if (T < 0 || hidden < 1 || hidden > kMaxHidden) return -1;
  return (int64_t)3 * backward_groups(T, hidden) * rows_of(threads_of(hidden)) * hidden * 4;
}

int moe_block_norm_backward_v1(const void* y, const void* res_out, int32_t T, int32_t hidden,
                               int32_t dtype, const void* post_w, const void* gate,
                               int32_t gate_kind, float res_scale, float branch_scale,
                               const void* pre_w, float eps, const void* dres_out, const void* dx,
                               void* workspace, int64_t workspace_bytes, void* dy, void* dres,
                               void* dpost_w, void* dgate, void* dpre_w, void* stream) {
  const int rc = check_norm("block norm backward", T, hidden, dtype, gate, gate_kind, eps);
  if (rc) return rc;
  if ((T > 0 && (!y || (dx && !res_out))) || (dx && !pre_w) || (dpost_w && !post_w) ||
      (dgate && gate_kind == kGateNone) || (dpre_w && !dx))
    return op_fail(MOE_ERR_NULL, "block norm backward: NULL pointer");
  void* dchannel = gate_kind == kGateChannel ? dgate : nullptr;
  int64_t need = 0;
  if (dpost_w || dchannel || dpre_w) {
    need = moe_block_norm_workspace_bytes_v1(T, hidden);
    if (!workspace || workspace_bytes < need)
      return op_fail(MOE_ERR_WORKSPACE, "block norm backward: workspace of %lld bytes, needs %lld",
                     (long long)(workspace ? workspace_bytes : 0), (long long)need);
    if (!workspace_aligned(workspace))
      return op_fail(MOE_ERR_WORKSPACE, "block norm backward: workspace must be 256-byte aligned");
  } else if (T == 0) {
    return MOE_OK;
  }
  const int64_t n = (int64_t)T * hidden * dtype_bytes(dtype), nw = row_bytes(hidden, dtype);
  const int64_t ng = gate_bytes(gate_kind, T, hidden, dtype);
  const Span outs[] = {{dy, n}, {dres, n}, {dpost_w, nw}, {dgate, ng}, {dpre_w, nw}, {workspace, need}};
  const Span ins[] = {{y, n}, {res_out, n}, {post_w, nw}, {gate, ng}, {pre_w, nw}, {dres_out, n}, {dx, n}};
  for (const Span& o : outs) {
    for (const Span& i : ins)
      if (overlaps(o.p, o.bytes, i.p, i.bytes))
        return op_fail(MOE_ERR_SHAPE,
                       "block norm backward: gradients and workspace must not overlap inputs");
    for (const Span* i = outs; i != &o; ++i)
      if (overlaps(o.p, o.bytes, i->p, i->bytes))
        return op_fail(MOE_ERR_SHAPE,
                       "block norm backward: gradients and workspace must not overlap each other");
  }
  const NormArgs a{y, res_out, post_w, gate, pre_w, gate_kind, T, hidden,
                   res_scale, branch_scale, eps};
  const NormGrads d{dres_out, dx, dy, dres, gate_kind == kGateChannel ? nullptr : dgate,
                    static_cast<float*>(workspace),
                    backward_groups(T, hidden) * rows_of(threads_of(hidden)), dpost_w != nullptr,
                    dchannel != nullptr, dpre_w != nullptr};
  const bool vec = vec_ok(hidden, {y, res_out, post_w, pre_w, dres_out, dx, dy, dres, workspace}) &&
                   (gate_kind < kGateChannel || aligned16(gate)) &&
                   (gate_kind != kGateFull || aligned16(dgate));
  const auto s = (hipStream_t)stream;
  MOE_OP_HIP(dtype == kBf16   ? launch_backward<kBf16>(a, d, dpost_w, dchannel, dpre_w, vec, s)
             : dtype == kFp16 ? launch_backward<kFp16>(a, d, dpost_w, dchannel, dpre_w, vec, s)
                              : launch_backward<kFp32>(a, d, dpost_w, dchannel, dpre_w, vec, s),
             "block norm backward");
  return MOE_OK;
}

}  // extern "C"
