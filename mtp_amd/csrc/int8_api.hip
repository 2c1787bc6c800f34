// Entry points of the int8 products: argument checks, the experts' workspace and their launches.
#include <algorithm>

#include "elem.h"
#include "int8.h"

namespace {

constexpr int kMaxK = 65536;  // |sum| <= 128 * 128 * 65536 = 2^30: exact in 32 bits
constexpr int64_t kMaxBytes = int64_t(1) << 31;  // 32-bit buffer offsets

int64_t align256(int64_t v) { return (v + 255) & ~int64_t(255); }

template <typename T>
T* at(void* base, int64_t off) { return reinterpret_cast<T*>(static_cast<char*>(base) + off); }

int check_dtype(const char* what, int dtype) {
  if (dtype < kBf16 || dtype > kFp32)
    return op_fail(MOE_ERR_UNSUPPORTED, "%s: dtype=%d (0 bf16, 1 fp16, 2 fp32)", what, dtype);
  return MOE_OK;
}

int check_sizes(const char* what, int32_t T, int32_t K, int32_t N) {
  if (T < 0 || N < 1) return op_fail(MOE_ERR_SHAPE, "%s: T=%d N=%d", what, T, N);
  if (K < 16 || K % 16 != 0 || K > kMaxK)
    return op_fail(MOE_ERR_SHAPE, "%s: K=%d must be a multiple of 16 in [16, 65536]", what, K);
  if ((int64_t)T * K >= kMaxBytes || (int64_t)N * K >= kMaxBytes)
    return op_fail(MOE_ERR_SHAPE, "%s: T * K or N * K of T=%d N=%d K=%d exceeds 2 GiB", what, T, N,
                   K);
  return MOE_OK;
}

// Whether [p, p + n) holds a byte of a product's weights, scales or bias.
bool weights_overlap(const void* p, int64_t n, const int8_t* w, const float* w_scale,
                     const void* bias, int N, int K, int dtype) {
  return overlaps(p, n, w, (int64_t)N * K) || overlaps(p, n, w_scale, (int64_t)N * 4) ||
         overlaps(p, n, bias, (int64_t)N * dtype_bytes(dtype));
}

int matmul(const int8_t* q, const float* q_scale, int T, int K, const int8_t* w,
           const float* w_scale, int N, const void* bias, int dtype, void* out, hipStream_t s) {
  Int8Args a{};
  a.a = q;
  a.a_scale = q_scale;
  a.src_div = 1;
  a.a_bytes = (uint32_t)((int64_t)T * K);
  a.b0 = w;
  a.s0 = w_scale;
  a.M = T;
  a.N = N;
  a.K = K;
  a.out = out;
  a.bias = bias;
  const Int8Plan plan = int8_matrix_plan(T, N);
  a.m_tiles = (T + plan.bm - 1) / plan.bm;
  MOE_OP_HIP(launch_int8_product(a, plan, false, dtype, s), "int8 product");
  return MOE_OK;
}

struct ExpertsLayout {
  int64_t q, qs, offsets, row_slot, slot_row, tiles, scratch, h, hq, hs, y, total;
  Int8Plan plan;
  int tile_cap;
};

ExpertsLayout experts_layout(int T, int k, const moe_int8_set_v1& ex, int dtype) {
  ExpertsLayout L{};
  const int64_t S = (int64_t)T * k, es = dtype_bytes(dtype);
  L.plan = int8_experts_plan(S, ex.num_experts, ex.intermediate);
  L.tile_cap = (int)(S / L.plan.bm + std::min<int64_t>(S, ex.num_experts));
  int64_t o = 0;
  auto take = [&o](int64_t bytes) {
    const int64_t at = o;
    o += align256(bytes);
    return at;
  };
  L.q = take((int64_t)T * ex.hidden);
  L.qs = take((int64_t)T * 4);
  L.offsets = take((int64_t)(ex.num_experts + 1) * 4);
  L.row_slot = take(S * 4);
  L.slot_row = take(S * 4);
  L.tiles = take((int64_t)L.tile_cap * 16);
  L.scratch = take(dispatch_scratch_bytes(S, ex.num_experts));
  L.h = take(S * ex.intermediate * es);
  L.hq = take(S * ex.intermediate);
  L.hs = take(S * 4);
  L.y = take(S * ex.hidden * es);
  L.total = o;
  return L;
}

int check_experts(int32_t T, int32_t k, const moe_int8_set_v1* ex, int32_t dtype) {
  if (!ex) return op_fail(MOE_ERR_NULL, "int8 experts: experts is NULL");
  if (!ex->gate || !ex->up || !ex->down || !ex->gate_scale || !ex->up_scale || !ex->down_scale)
    return op_fail(MOE_ERR_NULL, "int8 experts: a weight or scale pointer is NULL");
  const int E = ex->num_experts, H = ex->hidden, I = ex->intermediate;
  int rc = check_dtype("int8 experts", dtype);
  if (rc) return rc;
  if (E < 1 || E > 512)
    return op_fail(MOE_ERR_SHAPE, "int8 experts: num_experts=%d outside [1, 512]", E);
  if (T < 0 || k < 1 || k > 64 || (int64_t)T * k > (1 << 22))
    return op_fail(MOE_ERR_SHAPE, "int8 experts: T=%d top_k=%d (top_k in [1, 64], at most 2^22 slots)",
                   T, k);
  rc = check_sizes("int8 experts (hidden)", T, H, I);
  if (!rc) rc = check_sizes("int8 experts (intermediate)", T * k, I, H);
  if (rc) return rc;
  if (!aligned16(ex->gate) || !aligned16(ex->up) || !aligned16(ex->down))
    return op_fail(MOE_ERR_SHAPE, "int8 experts: int8 weights must start on 16-byte boundaries");
  return MOE_OK;
}

}  // namespace

extern "C" {

int moe_quantize_tokens_v1(const void* x, int32_t T, int32_t K, int32_t dtype, int8_t* q,
                           float* scale, void* stream) {
  const int rc = check_dtype("quantize", dtype);
  if (rc) return rc;
  if (T < 0 || T >= (1 << 22) || K < 1 || K > kMaxK)  // a launch has fewer than 2^32 threads
    return op_fail(MOE_ERR_SHAPE, "quantize: T=%d K=%d (T < 2^22, K in [1, 65536])", T, K);
  if (T == 0) return MOE_OK;
  if (!x || !q || !scale) return op_fail(MOE_ERR_NULL, "quantize: NULL pointer");
  if (overlaps(q, (int64_t)T * K, x, (int64_t)T * K * dtype_bytes(dtype)) ||
      overlaps(scale, (int64_t)T * 4, x, (int64_t)T * K * dtype_bytes(dtype)) ||
      overlaps(scale, (int64_t)T * 4, q, (int64_t)T * K))
    return op_fail(MOE_ERR_SHAPE, "quantize: x and the outputs must not overlap");
  MOE_OP_HIP(launch_quantize(x, T, K, dtype, q, scale, (hipStream_t)stream), "quantize");
  return MOE_OK;
}

int moe_int8_matmul_v1(const int8_t* q, const float* q_scale, int32_t T, int32_t K,
                       const int8_t* w, const float* w_scale, int32_t N, const void* bias,
                       int32_t dtype, void* out, void* stream) {
  int rc = check_dtype("int8 matmul", dtype);
  if (!rc) rc = check_sizes("int8 matmul", T, K, N);
  if (rc) return rc;
  if (T == 0) return MOE_OK;
  if (!q || !q_scale || !w || !w_scale || !out)
    return op_fail(MOE_ERR_NULL, "int8 matmul: NULL pointer");
  if (!aligned16(q) || !aligned16(w))
    return op_fail(MOE_ERR_SHAPE, "int8 matmul: q and w must start on 16-byte boundaries");
  const int64_t no = (int64_t)T * N * dtype_bytes(dtype);
  if (overlaps(out, no, q, (int64_t)T * K) || overlaps(out, no, q_scale, (int64_t)T * 4) ||
      weights_overlap(out, no, w, w_scale, bias, N, K, dtype))
    return op_fail(MOE_ERR_SHAPE, "int8 matmul: out must not overlap the inputs");
  return matmul(q, q_scale, T, K, w, w_scale, N, bias, dtype, out, (hipStream_t)stream);
}

int64_t moe_int8_linear_workspace_bytes_v1(int32_t T, int32_t K) {
  if (T < 0 || K < 1) return -1;
  if (T == 0 || int8_fused_fits(T, K)) return 0;
  return align256((int64_t)T * K) + align256((int64_t)T * 4);
}

int moe_int8_linear_v1(const void* x, int32_t T, int32_t K, int32_t dtype, const int8_t* w,
                       const float* w_scale, int32_t N, const void* bias, void* workspace,
                       int64_t workspace_bytes, void* out, void* stream) {
  int rc = check_dtype("int8 linear", dtype);
  if (!rc) rc = check_sizes("int8 linear", T, K, N);
  if (rc) return rc;
  if (T >= (1 << 26))  // a wave a row to quantise, and a launch has fewer than 2^32 threads
    return op_fail(MOE_ERR_SHAPE, "int8 linear: T=%d (T < 2^26)", T);
  if (T == 0) return MOE_OK;
  if (!x || !w || !w_scale || !out) return op_fail(MOE_ERR_NULL, "int8 linear: NULL pointer");
  if (!aligned16(w))
    return op_fail(MOE_ERR_SHAPE, "int8 linear: w must start on a 16-byte boundary");
  const int64_t need = moe_int8_linear_workspace_bytes_v1(T, K);
  if (need > 0) {
    if (!workspace || workspace_bytes < need)
      return op_fail(MOE_ERR_WORKSPACE, "int8 linear: workspace of %lld bytes, needs %lld",
                     (long long)(workspace ? workspace_bytes : 0), (long long)need);
    if (!workspace_aligned(workspace))
      return op_fail(MOE_ERR_WORKSPACE, "int8 linear: workspace must be 256-byte aligned");
  }
  const int64_t es = dtype_bytes(dtype), nx = (int64_t)T * K * es, no = (int64_t)T * N * es;
  if (overlaps(out, no, workspace, need) || overlaps(x, nx, workspace, need) ||
      overlaps(out, no, x, nx) || weights_overlap(out, no, w, w_scale, bias, N, K, dtype) ||
      weights_overlap(workspace, need, w, w_scale, bias, N, K, dtype))
    return op_fail(MOE_ERR_SHAPE,
                   "int8 linear: out and the workspace must not overlap the inputs or each other");
  const auto s = (hipStream_t)stream;
  if (need == 0) {
    Int8Args a{};
    a.b0 = w;
    a.s0 = w_scale;
    a.M = T;
    a.N = N;
    a.K = K;
    a.out = out;
    a.bias = bias;
    MOE_OP_HIP(launch_int8_fused(a, x, dtype, s), "int8 linear");
    return MOE_OK;
  }
  int8_t* q = static_cast<int8_t*>(workspace);
  float* qs = at<float>(workspace, align256((int64_t)T * K));
  MOE_OP_HIP(launch_quantize(x, T, K, dtype, q, qs, s), "quantize");
  return matmul(q, qs, T, K, w, w_scale, N, bias, dtype, out, s);
}

int64_t moe_int8_experts_workspace_bytes_v1(int32_t T, int32_t top_k,
                                            const moe_int8_set_v1* experts, int32_t dtype) {
  if (check_experts(T, top_k, experts, dtype)) return -1;
  return experts_layout(T, top_k, *experts, dtype).total;
}

int moe_int8_experts_v1(const void* x, int32_t T, int32_t dtype, const int32_t* topk_ids,
                        const float* topk_weights, int32_t top_k, const moe_int8_set_v1* experts,
                        void* workspace, int64_t workspace_bytes, void* out, void* stream) {
  const int rc = check_experts(T, top_k, experts, dtype);
  if (rc) return rc;
  if (T == 0) return MOE_OK;
  if (!x || !topk_ids || !topk_weights || !out)
    return op_fail(MOE_ERR_NULL, "int8 experts: NULL pointer");
  const ExpertsLayout L = experts_layout(T, top_k, *experts, dtype);
  if (!workspace || workspace_bytes < L.total)
    return op_fail(MOE_ERR_WORKSPACE, "int8 experts: workspace of %lld bytes, needs %lld",
                   (long long)(workspace ? workspace_bytes : 0), (long long)L.total);
  if (!workspace_aligned(workspace))
    return op_fail(MOE_ERR_WORKSPACE, "int8 experts: workspace must be 256-byte aligned");
  const int E = experts->num_experts, H = experts->hidden, I = experts->intermediate;
  const int64_t S = (int64_t)T * top_k, nx = (int64_t)T * H * dtype_bytes(dtype);
  if (overlaps(x, nx, workspace, L.total) || overlaps(out, nx, workspace, L.total) ||
      overlaps(topk_ids, S * 4, workspace, L.total) ||
      overlaps(topk_weights, S * 4, workspace, L.total) || overlaps(out, nx, topk_weights, S * 4))
    return op_fail(MOE_ERR_SHAPE,
                   "int8 experts: x, out and the routing must not overlap the workspace, nor out "
                   "the weights");
  const int64_t nw = (int64_t)E * H * I;
  const struct {
    const void* p;
    int64_t bytes;
  } weights[] = {{experts->gate, nw}, {experts->gate_scale, (int64_t)E * I * 4},
                 {experts->up, nw}, {experts->up_scale, (int64_t)E * I * 4},
                 {experts->down, nw}, {experts->down_scale, (int64_t)E * H * 4}};
  for (const auto& w : weights)
    if (overlaps(w.p, w.bytes, workspace, L.total))
      return op_fail(MOE_ERR_SHAPE, "int8 experts: the workspace must not overlap the weights");
  const auto s = (hipStream_t)stream;
  int8_t* q = at<int8_t>(workspace, L.q);
  float* qs = at<float>(workspace, L.qs);
  int32_t* row_slot = at<int32_t>(workspace, L.row_slot);
  int32_t* slot_row = at<int32_t>(workspace, L.slot_row);
  i32x4* tiles = at<i32x4>(workspace, L.tiles);
  void* h = at<void>(workspace, L.h);
  int8_t* hq = at<int8_t>(workspace, L.hq);
  float* hs = at<float>(workspace, L.hs);
  void* y = at<void>(workspace, L.y);
  MOE_OP_HIP(launch_quantize_and_sort(x, T, H, dtype, q, qs, topk_ids, top_k, E,
                                      at<int32_t>(workspace, L.offsets), row_slot, slot_row,
                                      at<void>(workspace, L.scratch), tiles, L.plan.bm, L.tile_cap,
                                      s),
             "quantize and sort");
  Int8Args a{};
  a.a = q;
  a.a_scale = qs;
  a.row_src = row_slot;
  a.src_div = top_k;
  a.a_bytes = (uint32_t)((int64_t)T * H);
  a.b0 = experts->gate;
  a.b1 = experts->up;
  a.s0 = experts->gate_scale;
  a.s1 = experts->up_scale;
  a.tiles = tiles;
  a.m_tiles = L.tile_cap;
  a.M = (int)S;
  a.N = I;
  a.K = H;
  a.out = h;
  MOE_OP_HIP(launch_int8_product(a, L.plan, true, dtype, s), "gate and up");
  // dropped slots' rows of h are never written; what they hold is quantised and not read again
  MOE_OP_HIP(launch_quantize(h, (int)S, I, dtype, hq, hs, s), "quantize h");
  Int8Args b{};
  b.a = hq;
  b.a_scale = hs;
  b.src_div = 1;
  b.a_bytes = (uint32_t)(S * I);
  b.b0 = experts->down;
  b.s0 = experts->down_scale;
  b.tiles = tiles;
  b.m_tiles = L.tile_cap;
  b.M = (int)S;
  b.N = H;
  b.K = I;
  b.out = y;
  MOE_OP_HIP(launch_int8_product(b, L.plan, false, dtype, s), "down");
  MOE_OP_HIP(launch_combine(y, T, top_k, H, dtype, slot_row, topk_weights, out, s), "combine");
  return MOE_OK;
}

}  // extern "C"
