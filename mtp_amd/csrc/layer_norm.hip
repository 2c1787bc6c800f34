// Layer norm and its gradients:
//
//   h = (x - m) r,  m = mean(x),  r = 1 / sqrt(mean((x - m)^2) + eps)
//   y = round(h w + b)                                   (w = 1, b = 0 where they are absent)
//
//   g = dy w;  dx = r (g - mean(g) - h mean(g h));  dw = sum_t dy h;  db = sum_t dy
//
// HBM-bound in both directions: rows are read and written once, 8 columns a thread held in registers
// across the reduction. A row takes a wave up to 512 columns, a workgroup of 256 threads up to 2048, of
// 512 up to 4096, of 1024 up to 8192.
//
// One reduction gives both moments: with c the row's first value, d = x - c and both sums in 64 bits,
// the variance is mean(d^2) - mean(d)^2. (m - c)^2 is at most hidden times the variance, since c is one of
// the row's own values, so the difference loses at most log2(8192) of the 53 bits. Sums of raw x in 32 bits would lose all of a row whose mean is 2^12 times its
// spread. x - m is taken as (x - m_hi) - m_lo for the same reason.
#include <algorithm>

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

// What the backward pass needs of a row: the mean in two parts and r.
struct RowStats {
  float hi, lo, r;
};

template <int DT, int NT, bool VEC>
__global__ __launch_bounds__(block_threads<NT>()) void layer_norm_kernel(LayerNormArgs a, void* y,
                                                                         f32x4* stats) {
  using T = typename Elem<DT>::T;
  using C = Cols<DT, NT, VEC>;
  __shared__ double s_part[NT / 64][2];
  const double inv_h = 1.0 / (double)a.H;
  const int tid = threadIdx.x % NT;
  const int rows = block_threads<NT>() / NT;
  const int sub = __builtin_amdgcn_readfirstlane((int)threadIdx.x / NT);
  for (int64_t t = (int64_t)blockIdx.x * rows + sub; t < a.T; t += (int64_t)gridDim.x * rows) {
    const T* row = static_cast<const T*>(a.x) + t * a.H;
    float x[8], w[8], b[8];
    C::load(row, tid, a.H, x);
    const double c = (double)Elem<DT>::get(row[0]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = 1.0f;
      b[e] = 0.0f;
    }
    if (a.w) C::load(static_cast<const T*>(a.w), tid, a.H, w);
    if (a.b) C::load(static_cast<const T*>(a.b), tid, a.H, b);
    double part[2] = {0.0, 0.0}, sum[2];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double d = C::col(tid, e) < a.H ? (double)x[e] - c : 0.0;
      part[0] += d;
      part[1] = __builtin_fma(d, d, part[1]);
    }
    row_sums<NT>(part, sum, s_part);
    const double md = sum[0] * inv_h, mean = c + md;
    // a rounding could leave the variance of a nearly constant row below zero
    const double var = __builtin_fma(-md, md, sum[1] * inv_h);
    const RowStats st{(float)mean, (float)(mean - (double)(float)mean),
                      inv_sqrt((var < 0.0 ? 0.0 : var) + a.eps)};
    if (stats && tid == 0) stats[t] = f32x4{st.hi, st.lo, st.r, 0.0f};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = __builtin_fmaf(((x[e] - st.hi) - st.lo) * st.r, w[e], b[e]);
    C::store(static_cast<T*>(y) + t * a.H, tid, a.H, x);
  }
}

struct LayerNormGrads {
  const void* dy;
  const f32x4* stats;
  void* dx;     // nullable
  float* part;  // [2][partials][H]: dw, db
  int partials;
  bool dw, db;  // which of them are wanted
};

template <int DT, int NT, bool VEC>
__global__ __launch_bounds__(block_threads<NT>()) void layer_norm_backward_kernel(LayerNormArgs a,
                                                                                  LayerNormGrads d) {
  using T = typename Elem<DT>::T;
  using C = Cols<DT, NT, VEC>;
  using Raw = RawCols<DT, NT, VEC>;
  __shared__ float s_part[NT / 64][2];
  const float inv_h = 1.0f / (float)a.H;
  const int tid = threadIdx.x % NT, H = a.H;
  const int rows = block_threads<NT>() / NT;
  const int sub = __builtin_amdgcn_readfirstlane((int)threadIdx.x / NT);
  const int64_t stride = (int64_t)gridDim.x * rows, first = (int64_t)blockIdx.x * rows + sub;
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
  if (first < a.T) load(first);
  for (int64_t t = first; t < a.T; t += stride) {
    const Row row = next;
    load(t + stride);
    const float hi = row.st[0], lo = row.st[1], r = row.st[2];
    float part[2] = {0.0f, 0.0f}, tot[2];
    float h[8], g[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = C::col(tid, e) < H;
      const float dy = row.dy.get(e, tid, H);
      h[e] = in ? ((row.x.get(e, tid, H) - hi) - lo) * r : 0.0f;
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
      C::store(static_cast<T*>(d.dx) + t * H, tid, H, g);
    }
  }
  const int64_t all = (int64_t)d.partials * H;
  Cols<kFp32, NT, VEC> f;
  if (d.dw) f.store(d.part + first * H, tid, H, dw);
  if (d.db) f.store(d.part + all + first * H, tid, H, db);
}

// Workgroups of the backward pass: each keeps the weights' gradients of its rows in registers and
// writes them once.
int backward_groups(int T, int H) {
  const int nt = threads_of(H), rows = rows_of(nt);
  const int most = nt > 256 ? 512 : 768;
  return std::max(1, std::min((T - 1) / rows + 1, most));  // T + rows may pass 32 bits
}

template <int DT>
hipError_t launch_forward(const LayerNormArgs& a, void* y, f32x4* stats, bool vec, hipStream_t s) {
  const int nt = threads_of(a.H), rows = rows_of(nt);
  const dim3 grid((unsigned)std::min<int64_t>((a.T + (int64_t)rows - 1) / rows, 1 << 20));
#define MOE_LN_FWD(NT, V)                                                                      \
  hipLaunchKernelGGL((layer_norm_kernel<DT, NT, V>), grid, dim3(block_threads<NT>()), 0, s, a, \
                     y, stats)
  MOE_ROW_NT(MOE_LN_FWD)
#undef MOE_LN_FWD
  return hipGetLastError();
}

template <int DT>
hipError_t launch_backward(const LayerNormArgs& a, const LayerNormGrads& d, void* dw, void* db,
                           bool vec, hipStream_t s) {
  const int nt = threads_of(a.H);
  const dim3 grid((unsigned)backward_groups(a.T, a.H));
#define MOE_LN_BWD(NT, V)                                                                       \
  hipLaunchKernelGGL((layer_norm_backward_kernel<DT, NT, V>), grid, dim3(block_threads<NT>()), \
                     0, s, a, d)
  MOE_ROW_NT(MOE_LN_BWD)
#undef MOE_LN_BWD
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !(dw || db)) return e;
  hipLaunchKernelGGL(column_sum_kernel<DT>, dim3((a.H + kSumCols - 1) / kSumCols, 2), dim3(1024),
                     0, s, d.part, d.partials, a.H, SumOut{{dw, db, nullptr}});
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
  return (int64_t)2 * backward_groups(T, hidden) * rows_of(threads_of(hidden)) * hidden * 4;
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
                         static_cast<float*>(workspace),
                         backward_groups(T, hidden) * rows_of(threads_of(hidden)),
                         dweight != nullptr, dbias != nullptr};
  const bool vec = vec_ok(hidden, {x, weight, dy, dx, workspace});
  const auto s = (hipStream_t)stream;
  MOE_OP_HIP(dtype == kBf16   ? launch_backward<kBf16>(a, d, dweight, dbias, vec, s)
             : dtype == kFp16 ? launch_backward<kFp16>(a, d, dweight, dbias, vec, s)
                              : launch_backward<kFp32>(a, d, dweight, dbias, vec, s),
             "layer norm backward");
  return MOE_OK;
}

}  // extern "C"
