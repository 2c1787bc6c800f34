// Layer norm and its gradients:
//
//   h = (x - m) r,  m = mean(x),  r = 1 / sqrt(mean((x - m)^2) + eps)
//   y = round(h w + b)                                   (w = 1, b = 0 where they are absent)
//
//   g = dy w;  dx = r (g - mean(g) - h mean(g h));  dw = sum_t dy h;  db = sum_t dy
//
// HBM-bound in both directions: rows are read and written once, their columns held in registers 8 at a time
// across the reductions. Sums are taken in a fixed order. us on the GPU (a copy of 1 GiB runs at 5.2 TB/s):
//   forward   16384 x 2048 bf16 25 (5.4 TB/s), 8192 x 4096 fp16 25 (5.4), 2001 x 1000 fp32 5.2
//   backward  16384 x 2048 bf16 39 with all gradients (5.2 TB/s; 32 for dx alone), 2001 x 1000 fp32 14
// Up to 256 columns 2, 4 or 8 rows share a wave: 524288 x 128 bf16 54 (5.0 TB/s) and 79 (5.1).
//
// The mean is a sum in 64 bits and a division (a constant row's sum is exact, and so is then its mean): in 32
// bits a row whose mean is 2^12 times its spread would lose half of its digits. It is kept in two parts, and
// x - m taken as (x - m_hi) - m_lo, off by two half steps. The squares of that are summed 8 at a time in fp32
// (a tree: 4 roundings) and from there on in 64 bits, so r is off by 3 half steps whatever the row's width
// and mean.
//
// A row with var + eps outside [2^-80, 2^126], where squares may leave fp32's range, is taken again from memory
// with squares of 64 bits, and from there on in units of a power of two (1 / s) that brings it back:
//   h = (s x - s m) r,  r = 1 / sqrt(s^2 (var + eps)),  dx = s r (...)
// s x is not rounded but where it is 2^-100 of the row's spread, so such rows are as exact as the others (s = 1).
// They are read twice more, element by element (16384 x 2048 bf16 of them 97 us); the test for them is two
// comparisons a row.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "elem.h"
#include "launch.h"
#include "row_sums.h"

namespace {

struct LayerNormArgs {
  const void* x;
  const void* w;  // nullable
  const void* b;  // nullable
  int T, H;
  double eps;
};

// The rows of a thread, with NT threads a row in workgroups of BT: those of a wave that holds several run
// together, so the loop is over the first of them, and the last ones may lie behind the tensor. `mine`: this
// thread's, of the wave's.
template <int NT, int BT>
struct Rows {
  int mine;
  int64_t first, stride;
  MOE_DEV Rows() {
    constexpr int kWide = NT < 64 ? 64 : NT;
    mine = NT < 64 ? (int)(threadIdx.x & 63) / NT : 0;
    first = ((int64_t)blockIdx.x * (BT / kWide) + __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWide)) *
            (kWide / NT);
    stride = (int64_t)gridDim.x * (BT / NT);
  }
};

// var + eps of the rows that fp32's squares hold, and s for the others: 2^100 keeps a row below it in range (its
// columns are below 2^-7, since two of them are less than 2^-32 apart and differ) and 2^-80 any row above it, and
// s^2 (var + eps) lies between 2^-98 and 2^120. Without a spread, and with infinities or NaN, s = 1.
constexpr float kNearLow = 0x1p-80f, kNearHigh = 0x1p126f;
MOE_DEV bool near(float v) { return v >= kNearLow && v <= kNearHigh; }
MOE_DEV float row_scale(double var, double v) {
  if (!(var > 0.0 && v < __builtin_inf())) return 1.0f;
  return v < kNearLow ? 0x1p100f : v > kNearHigh ? 0x1p-80f : 1.0f;
}

// NT threads a row, NC chunks of 8 NT columns: a wave a row while it holds the row (2048 columns), with no
// barrier and 12 exchanges for up to 32 columns a lane; with 256 threads a row of 2048 these and the barriers
// were half of the kernel's instructions (16384 x 2048 bf16 31 us). A workgroup takes every so many rows and
// has the next one's loads in flight while it works on this one.
template <int DT, int NT, int NC, bool VEC>
__global__ __launch_bounds__(256) void layer_norm_kernel(LayerNormArgs a, void* y, f32x4* stats) {
  using T = typename Elem<DT>::T;
  using C = Cols<DT, NT, VEC>;
  using Raw = RawCols<DT, NT, VEC>;
  __shared__ double s_part[NT > 64 ? NT / 64 : 1][1];
  const double inv_h = 1.0 / (double)a.H;
  const int tid = threadIdx.x % NT, H = a.H;
  const Rows<NT, 256> rows;
  Raw next[NC], w[NC] = {}, b[NC] = {};
  auto load = [&](Raw (&v)[NC], const void* p, int64_t t) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
      v[c].load(static_cast<const T*>(p) + t * H + c * 8 * NT, tid, H - c * 8 * NT);
  };
  if (rows.first < a.T) load(next, a.x, min(rows.first + rows.mine, (int64_t)a.T - 1));
  if (a.w) load(w, a.w, 0);
  if (a.b) load(b, a.b, 0);
  for (int64_t lead = rows.first; lead < a.T; lead += rows.stride) {
    const int64_t t = lead + rows.mine;
    const bool in = NT >= 64 || t < a.T;
    float d[NC][8];
    double part[1] = {0.0}, sum[1];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int left = H - c * 8 * NT;
        d[c][e] = next[c].get(e, tid, left);
        part[0] += (double)d[c][e];
      }
    load(next, a.x, min(t + rows.stride, (int64_t)a.T - 1));  // past the last row: read again, not used
    row_sums<NT>(part, sum, s_part);
    const double mean = sum[0] / (double)H;
    float hi = (float)mean, lo = (float)(mean - (double)hi);
    part[0] = 0.0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        d[c][e] = C::col(tid, e) < H - c * 8 * NT ? (d[c][e] - hi) - lo : 0.0f;
      float q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = __builtin_fmaf(d[c][i], d[c][i], d[c][4 + i] * d[c][4 + i]);
      part[0] += (double)((q[0] + q[1]) + (q[2] + q[3]));
    }
    row_sums<NT>(part, sum, s_part);
    double v = sum[0] * inv_h + a.eps;
    float r = inv_sqrt_near(v), scale = 1.0f;
    // The whole wave, for the exchanges; a near row comes out as it went in. The row is read again, and `at` hides
    // that it is the same column, so that nothing is kept in registers for this.
    if (__builtin_expect(__ballot(!near((float)v)) != 0, 0)) {
      const T* const row = static_cast<const T*>(a.x) + min(t, (int64_t)a.T - 1) * H;
      int at = tid;
      asm volatile("" : "+v"(at));
      part[0] = 0.0;
#pragma unroll 1
      for (int c = at; c < H; c += NT) {
        const double u = (double)Elem<DT>::get(row[c]) - mean;
        part[0] = __builtin_fma(u, u, part[0]);
      }
      row_sums<NT>(part, sum, s_part);
      if (!near((float)v)) {
        v = sum[0] * inv_h + a.eps;
        scale = row_scale(sum[0], v);
        const double m = mean * (double)scale;
        hi = (float)m;
        lo = (float)(m - (double)hi);
        r = inv_sqrt(v * (double)scale * (double)scale);
      }
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = c * 8 * NT + C::col(at, e);
          d[c][e] = i < H ? __builtin_fmaf(Elem<DT>::get(row[i]), scale, -hi) - lo : 0.0f;
        }
    }
    if (stats && tid == 0 && in) stats[t] = f32x4{hi, lo, r, scale};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int left = H - c * 8 * NT;
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        o[e] = __builtin_fmaf(d[c][e] * r, a.w ? w[c].get(e, tid, left) : 1.0f,
                              a.b ? b[c].get(e, tid, left) : 0.0f);
      if (in) C::store(static_cast<T*>(y) + t * H + c * 8 * NT, tid, left, o);
    }
  }
}

struct LayerNormGrads {
  const void* dy;
  const f32x4* stats;
  void* dx;     // nullable
  float* part;  // [2][workgroups][H]: dw, db
  bool dw, db;  // which of them are wanted
};

template <int DT, int NT, bool VEC>
__global__ __launch_bounds__(block_threads<NT>()) void layer_norm_backward_kernel(LayerNormArgs a,
                                                                                  LayerNormGrads d) {
  using T = typename Elem<DT>::T;
  using C = Cols<DT, NT, VEC>;
  using Raw = RawCols<DT, NT, VEC>;
  __shared__ float s_part[NT > 64 ? NT / 64 : 1][2];
  const float inv_h = 1.0f / (float)a.H;
  const int tid = threadIdx.x % NT, H = a.H;
  const Rows<NT, block_threads<NT>()> rows;
  float w[8], dw[8], db[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    w[e] = 1.0f;
    dw[e] = db[e] = 0.0f;
  }
  if (a.w) C::load(static_cast<const T*>(a.w), tid, H, w);
  struct Row {
    Raw x, dy;
    f32x4 st;
  };
  Row next{};
  auto load = [&](int64_t t) {  // past the last row: read again, not used
    const int64_t u = min(t, (int64_t)a.T - 1);
    next.x.load(static_cast<const T*>(a.x) + u * H, tid, H);
    next.dy.load(static_cast<const T*>(d.dy) + u * H, tid, H);
    next.st = d.stats[u];
  };
  if (rows.first < a.T) load(rows.first + rows.mine);
  for (int64_t lead = rows.first; lead < a.T; lead += rows.stride) {
    const int64_t t = lead + rows.mine;
    const bool mine = NT >= 64 || t < a.T;
    const Row row = next;
    load(t + rows.stride);
    const float hi = row.st[0], lo = row.st[1], r = row.st[2], scale = row.st[3];
    auto take = [&](auto scaled) __attribute__((always_inline)) {
      float part[2] = {0.0f, 0.0f}, tot[2];
      float h[8], g[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = row.x.get(e, tid, H);
      if (scaled) {
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] *= scale;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = C::col(tid, e) < H;
        const float dy = mine ? row.dy.get(e, tid, H) : 0.0f;
        h[e] = in && mine ? ((h[e] - hi) - lo) * r : 0.0f;
        g[e] = dy * w[e];
        dw[e] = __builtin_fmaf(dy, h[e], dw[e]);
        db[e] += dy;
        part[0] += g[e];
        part[1] = __builtin_fmaf(g[e], h[e], part[1]);
      }
      if (d.dx) {
        row_sums<NT>(part, tot, s_part);
        const float mg = tot[0] * inv_h, mgh = tot[1] * inv_h;
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = r * ((g[e] - mg) - h[e] * mgh);
        if (scaled) {
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] *= scale;
        }
        if (mine) C::store(static_cast<T*>(d.dx) + t * H, tid, H, g);
      }
    };
    // s is 1 in nearly every wave. us without s / with its products always taken / in branches / in two bodies:
    // 300000 x 64 bf16 37.8 / 40.3 / 38.0 / 42, 100001 x 99 (element-wise) 24.7 / 25.7 / 28.7 / 24.2, 8192 x 4096
    // fp16 40.1 / 40.1 / 40.1 / 41.6.
    const bool scaled = __builtin_expect(__ballot(scale != 1.0f) != 0, 0);
    if constexpr (VEC || NT >= 64) {
      take(scaled);
    } else {
      if (scaled) take(std::true_type{});
      else take(std::false_type{});
    }
  }
  if constexpr (NT <= 64) {  // the workgroup's rows first
    constexpr int kRows = 256 / NT;
    const int sub = threadIdx.x / NT;
    __shared__ f32x4 s_all[kRows][4][NT];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float* v = (q < 2 ? dw : db) + 4 * (q & 1);
      s_all[sub][q][tid] = f32x4{v[0], v[1], v[2], v[3]};
    }
    __syncthreads();
    if (sub != 0) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f32x4 v = s_all[0][q][tid];
#pragma unroll
      for (int w = 1; w < kRows; ++w) v += s_all[w][q][tid];
#pragma unroll
      for (int j = 0; j < 4; ++j) (q < 2 ? dw : db)[4 * (q & 1) + j] = v[j];
    }
  }
  const int64_t me = blockIdx.x, all = (int64_t)gridDim.x * H;
  Cols<kFp32, NT, VEC> f;
  if (d.dw) f.store(d.part + me * H, tid, H, dw);
  if (d.db) f.store(d.part + all + me * H, tid, H, db);
}

// The weights' gradients from the workgroups' sums: 16 columns a workgroup, 64 threads a column over
// strided parts (12 loads each for the most workgroups, all in flight), a wave's four by a butterfly, then
// the 16 waves' in order.
constexpr int kSumCols = 16;
template <int DT>
__global__ __launch_bounds__(1024) void layer_norm_sum_kernel(const float* part, int parts, int H,
                                                              void* dw, void* db) {
  __shared__ float s_sum[16][kSumCols];
  void* const out = blockIdx.y ? db : dw;
  if (!out) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = threadIdx.x % kSumCols;
  const int c = blockIdx.x * kSumCols + col;
  const float* p = part + (int64_t)blockIdx.y * parts * H + min(c, H - 1);
  float s = 0.0f;
#pragma unroll 12
  for (int i = threadIdx.x / kSumCols; i < parts; i += 64) s += p[(int64_t)i * H];
  s += xor_partner<32>(s);
  s += xor_partner<16>(s);
  if (lane < kSumCols) s_sum[wave][lane] = s;
  __syncthreads();
  if (threadIdx.x < kSumCols && c < H) {
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += s_sum[i][threadIdx.x];
    static_cast<typename Elem<DT>::T*>(out)[c] = Elem<DT>::put(s);
  }
}

// Workgroups of the forward pass: 6 a CU (16384 x 2048 bf16 with 2, 4, 6, 8 and 16 of them 23.5, 23.1, 24.0,
// 24.0 and 26.1 us, 16384 x 512 10.7, 9.8, 9.3, 9.5 and 9.8, 8192 x 4096 fp16 28.6, 24.6, 24.1, 23.8, 24.8).
constexpr int kForwardGroups = 1536;

// Workgroups of the backward pass: each keeps the weights' gradients of its rows in registers and
// writes them once.
//
// Rows of up to 256 columns take 32, 16 or 8 threads, forward and backward (us a wave a row / with this):
// 65536 x 256 fp16 27 and 30 / 16 and 22, 524288 x 128 bf16 186 and 175 / 54 and 79, 300000 x 64 106 and 100 / 16
// and 38.
int narrow_threads_of(int H) { return H <= 64 ? 8 : H <= 128 ? 16 : H <= 256 ? 32 : threads_of(H); }
int backward_groups(int T, int H) {
  const int nt = narrow_threads_of(H), rows = rows_of(nt);
  const int most = nt > 256 ? 256 : 768;
  return std::max(1, std::min((T - 1) / rows + 1, most));  // T + rows may pass 32 bits
}

template <int DT>
hipError_t launch_forward(const LayerNormArgs& a, void* y, f32x4* stats, bool vec, hipStream_t s) {
#define MOE_LN_FWD(NT, NC)                                                                             \
  do {                                                                                                 \
    const int64_t groups = (a.T + int64_t(256 / NT) - 1) / (256 / NT);                                 \
    const dim3 grid((unsigned)std::min<int64_t>(groups, kForwardGroups));                              \
    if (vec)                                                                                           \
      hipLaunchKernelGGL((layer_norm_kernel<DT, NT, NC, true>), grid, dim3(256), 0, s, a, y, stats);   \
    else                                                                                               \
      hipLaunchKernelGGL((layer_norm_kernel<DT, NT, NC, false>), grid, dim3(256), 0, s, a, y, stats);  \
  } while (0)
  if (a.H <= 64) MOE_LN_FWD(8, 1);
  else if (a.H <= 128) MOE_LN_FWD(16, 1);
  else if (a.H <= 256) MOE_LN_FWD(32, 1);
  else if (a.H <= 512) MOE_LN_FWD(64, 1);
  else if (a.H <= 1024) MOE_LN_FWD(64, 2);
  else if (a.H <= 2048) MOE_LN_FWD(64, 4);
  else if (a.H <= 4096) MOE_LN_FWD(256, 2);
  else MOE_LN_FWD(256, 4);
#undef MOE_LN_FWD
  return hipGetLastError();
}

template <int DT>
hipError_t launch_backward(const LayerNormArgs& a, const LayerNormGrads& d, void* dw, void* db,
                           bool vec, hipStream_t s) {
  const int nt = narrow_threads_of(a.H);
  const dim3 grid((unsigned)backward_groups(a.T, a.H));
#define MOE_LN_BWD(NT, V)                                                                       \
  hipLaunchKernelGGL((layer_norm_backward_kernel<DT, NT, V>), grid, dim3(block_threads<NT>()), \
                     0, s, a, d)
  if (nt == 8) {
    if (vec) MOE_LN_BWD(8, true); else MOE_LN_BWD(8, false);
  } else if (nt == 16) {
    if (vec) MOE_LN_BWD(16, true); else MOE_LN_BWD(16, false);
  } else if (nt == 32) {
    if (vec) MOE_LN_BWD(32, true); else MOE_LN_BWD(32, false);
  } else {
    MOE_ROW_NT(MOE_LN_BWD)
  }
#undef MOE_LN_BWD
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !(dw || db)) return e;
  hipLaunchKernelGGL(layer_norm_sum_kernel<DT>, dim3((a.H + kSumCols - 1) / kSumCols, 2), dim3(1024),
                     0, s, d.part, (int)grid.x, a.H, dw, db);
  return hipGetLastError();
}

int check_layer_norm(const char* what, int32_t T, int32_t hidden, int32_t dtype) {
  if (dtype < kBf16 || dtype > kFp32)
    return op_fail(MOE_ERR_UNSUPPORTED, "%s: dtype=%d (0 bf16, 1 fp16, 2 fp32)", what, dtype);
  if (T < 0 || hidden < 1 || hidden > kMaxHidden)
    return op_fail(MOE_ERR_SHAPE, "%s: T=%d hidden=%d (hidden in [1, 8192])", what, T, hidden);
  return MOE_OK;
}

}  // namespace

extern "C" {

int moe_layer_norm_v1(const void* x, int32_t T, int32_t hidden, int32_t dtype, const void* weight,
                      const void* bias, float eps, void* y, float* stats, void* stream) {
  const int rc = check_layer_norm("layer norm", T, hidden, dtype);
  if (rc) return rc;
  if (!(eps >= 0.0f)) return op_fail(MOE_ERR_SHAPE, "layer norm: eps must be >= 0");
  if (T == 0) return MOE_OK;
  if (!x || !y) return op_fail(MOE_ERR_NULL, "layer norm: NULL pointer");
  if (!aligned16(stats))
    return op_fail(MOE_ERR_SHAPE, "layer norm: stats must start on a 16-byte boundary");
  const int64_t n = (int64_t)T * hidden * dtype_bytes(dtype), nw = hidden * dtype_bytes(dtype);
  const Span outs[] = {{y, n}, {stats, (int64_t)T * 16}}, ins[] = {{x, n}, {weight, nw}, {bias, nw}};
  bool shared = overlaps(y, n, stats, (int64_t)T * 16);
  for (const Span& o : outs)
    for (const Span& i : ins) shared |= overlaps(o.p, o.bytes, i.p, i.bytes);
  if (shared)
    return op_fail(MOE_ERR_SHAPE, "layer norm: outputs must not overlap inputs or each other");
  const LayerNormArgs a{x, weight, bias, T, hidden, (double)eps};
  const bool vec = vec_ok(hidden, {x, weight, bias, y});
  const auto s = (hipStream_t)stream;
  f32x4* st = reinterpret_cast<f32x4*>(stats);
  MOE_OP_HIP(dtype == kBf16   ? launch_forward<kBf16>(a, y, st, vec, s)
             : dtype == kFp16 ? launch_forward<kFp16>(a, y, st, vec, s)
                              : launch_forward<kFp32>(a, y, st, vec, s),
             "layer norm");
  return MOE_OK;
}

int64_t moe_layer_norm_workspace_bytes_v1(int32_t T, int32_t hidden) {
  if (T < 0 || hidden < 1 || hidden > kMaxHidden) return -1;
  return (int64_t)2 * backward_groups(T, hidden) * hidden * 4;
}

int moe_layer_norm_backward_v1(const void* x, int32_t T, int32_t hidden, int32_t dtype,
                               const void* weight, const float* stats, const void* dy,
                               void* workspace, int64_t workspace_bytes, void* dx, void* dweight,
                               void* dbias, void* stream) {
  const int rc = check_layer_norm("layer norm backward", T, hidden, dtype);
  if (rc) return rc;
  if (T > 0 && (!x || !stats || !dy))
    return op_fail(MOE_ERR_NULL, "layer norm backward: NULL pointer");
  if (!aligned16(stats))
    return op_fail(MOE_ERR_SHAPE, "layer norm backward: stats must start on a 16-byte boundary");
  int64_t need = 0;
  if (dweight || dbias) {
    need = moe_layer_norm_workspace_bytes_v1(T, hidden);
    if (!workspace || workspace_bytes < need)
      return op_fail(MOE_ERR_WORKSPACE, "layer norm backward: workspace of %lld bytes, needs %lld",
                     (long long)(workspace ? workspace_bytes : 0), (long long)need);
    if (!workspace_aligned(workspace))
      return op_fail(MOE_ERR_WORKSPACE, "layer norm backward: workspace must be 256-byte aligned");
  } else if (T == 0 || !dx) {
    return MOE_OK;
  }
  const int64_t n = (int64_t)T * hidden * dtype_bytes(dtype), nw = hidden * dtype_bytes(dtype);
  const Span outs[] = {{dx, n}, {dweight, nw}, {dbias, nw}, {workspace, need}};
  const Span ins[] = {{x, n}, {weight, nw}, {stats, (int64_t)T * 16}, {dy, n}};
  for (const Span& o : outs) {
    for (const Span& i : ins)
      if (overlaps(o.p, o.bytes, i.p, i.bytes))
        return op_fail(MOE_ERR_SHAPE,
                       "layer norm backward: gradients and workspace must not overlap inputs");
    for (const Span* i = outs; i != &o; ++i)
      if (overlaps(o.p, o.bytes, i->p, i->bytes))
        return op_fail(MOE_ERR_SHAPE,
                       "layer norm backward: gradients and workspace must not overlap each other");
  }
  const LayerNormArgs a{x, weight, nullptr, T, hidden, 0.0};
  const LayerNormGrads d{dy, reinterpret_cast<const f32x4*>(stats), dx,
                         static_cast<float*>(workspace), dweight != nullptr, dbias != nullptr};
  const bool vec = vec_ok(hidden, {x, weight, dy, dx, workspace});
  const auto s = (hipStream_t)stream;
  MOE_OP_HIP(dtype == kBf16   ? launch_backward<kBf16>(a, d, dweight, dbias, vec, s)
             : dtype == kFp16 ? launch_backward<kFp16>(a, d, dweight, dbias, vec, s)
                              : launch_backward<kFp32>(a, d, dweight, dbias, vec, s),
             "layer norm backward");
  return MOE_OK;
}

}  // extern "C"
