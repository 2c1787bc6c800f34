// A linear layer on int4 weights with a scale and a zero point per group of K (the GPTQ layout of the
// experts, one matrix):
//
//   y[t, n] = round(sum_g s[g, n] * (sum_{k in g} x[t, k] (q[k, n] - z[g, n])) (+ bias[n]))
//
// The weights are not rounded: a group's products are summed in fp32 on the integers q - z and scaled
// after that.
#include <algorithm>

#include "common.h"
#include "elem.h"
#include "launch.h"

namespace {

constexpr int kMaxK = 65536;
constexpr int64_t kMaxBytes = int64_t(1) << 31;  // 32-bit buffer offsets

struct Int4Args {
  const void* x;
  const uint32_t* qweight;  // [K / 8][N]
  const uint32_t* qzeros;   // [K / G][N / 8]
  const uint16_t* scales;   // fp16 [K / G][N]
  const void* bias;         // nullable
  void* out;
  int T, K, N, G;
};

constexpr int kRows = 8;

// A thread an output channel, kRows tokens.
template <int DT>
__global__ __launch_bounds__(256) void int4_linear_kernel(Int4Args a) {
  using T = typename Elem<DT>::T;
  const int blocks_n = (a.N + 255) / 256;
  const int n = blockIdx.x % blocks_n * 256 + threadIdx.x, t0 = blockIdx.x / blocks_n * kRows;
  if (n >= a.N) return;
  const int rows = min(kRows, a.T - t0);
  const T* x = static_cast<const T*>(a.x) + (int64_t)t0 * a.K;
  float acc[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) acc[r] = 0.0f;
  for (int g = 0; g < a.K / a.G; ++g) {
    const int z = (int)(a.qzeros[(int64_t)g * (a.N / 8) + n / 8] >> (4 * (n & 7))) & 15;
    const float s = f16_to_f32(a.scales[(int64_t)g * a.N + n]);
    float part[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) part[r] = 0.0f;
    for (int k = g * a.G; k < (g + 1) * a.G; k += 8) {
      const uint32_t q = a.qweight[(int64_t)(k / 8) * a.N + n];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float w = (float)((int)((q >> (4 * j)) & 15u) - z);
#pragma unroll
        for (int r = 0; r < kRows; ++r)
          part[r] = __builtin_fmaf(Elem<DT>::get(x[(int64_t)min(r, rows - 1) * a.K + k + j]), w, part[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) acc[r] = __builtin_fmaf(s, part[r], acc[r]);
  }
  const float b = a.bias ? Elem<DT>::get(static_cast<const T*>(a.bias)[n]) : 0.0f;
#pragma unroll
  for (int r = 0; r < kRows; ++r)
    if (r < rows) static_cast<T*>(a.out)[(int64_t)(t0 + r) * a.N + n] = Elem<DT>::put(acc[r] + b);
}

template <int DT>
hipError_t launch_int4(const Int4Args& a, hipStream_t s) {
  hipLaunchKernelGGL(int4_linear_kernel<DT>, dim3((a.N + 255) / 256 * ((a.T + kRows - 1) / kRows)),
                     dim3(256), 0, s, a);
  return hipGetLastError();
}

int check_int4(int32_t T, int32_t K, int32_t N, int32_t G, int32_t dtype) {
  if (dtype != kBf16 && dtype != kFp16)
    return op_fail(MOE_ERR_UNSUPPORTED, "int4 linear: dtype=%d (0 bf16, 1 fp16)", dtype);
  if (T < 0 || N < 8 || N % 8 != 0)
    return op_fail(MOE_ERR_SHAPE, "int4 linear: T=%d N=%d (N a multiple of 8)", T, N);
  if (G < 32 || G % 32 != 0 || K < G || K > kMaxK || K % G != 0)
    return op_fail(MOE_ERR_SHAPE,
                   "int4 linear: K=%d group_size=%d (the group a multiple of 32 that divides K, K at "
                   "most 65536)", K, G);
  if ((int64_t)T * K * 2 >= kMaxBytes || (int64_t)K / 8 * N * 4 >= kMaxBytes ||
      (int64_t)(K / G) * N * 2 >= kMaxBytes || (int64_t)T * N >= int64_t(1) << 33)
    return op_fail(MOE_ERR_SHAPE, "int4 linear: x, the weights or the scales of T=%d K=%d N=%d "
                   "exceed 2 GiB, or out 2^33 values", T, K, N);
  return MOE_OK;
}

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace

extern "C" {

int64_t moe_int4_linear_workspace_bytes_v1(int32_t T, int32_t K, int32_t N, int32_t group_size) {
  if (check_int4(T, K, N, group_size, kBf16)) return -1;
  return 0;
}

int moe_int4_linear_v1(const void* x, int32_t T, int32_t K, int32_t dtype,
                       const moe_gptq_proj_v1* weight, int32_t N, int32_t group_size,
                       const void* bias, void* workspace, int64_t workspace_bytes, void* out,
                       void* stream) {
  const int rc = check_int4(T, K, N, group_size, dtype);
  if (rc) return rc;
  if (!weight) return op_fail(MOE_ERR_NULL, "int4 linear: weight is NULL");
  if (T == 0) return MOE_OK;
  if (!x || !weight->qweight || !weight->qzeros || !weight->scales || !out)
    return op_fail(MOE_ERR_NULL, "int4 linear: NULL pointer");
  if (!aligned4(weight->qweight) || !aligned4(weight->qzeros))
    return op_fail(MOE_ERR_SHAPE, "int4 linear: qweight and qzeros must start on 4-byte boundaries");
  const int64_t need = 0;
  const int64_t nx = (int64_t)T * K * 2, no = (int64_t)T * N * 2, ng = K / group_size;
  const struct {
    const void* p;
    int64_t bytes;
  } ins[] = {{x, nx}, {weight->qweight, (int64_t)K / 8 * N * 4}, {weight->qzeros, ng * (N / 8) * 4},
             {weight->scales, ng * N * 2}, {bias, (int64_t)N * 2}};
  for (const auto& i : ins)
    if (overlaps(out, no, i.p, i.bytes) || overlaps(workspace, need, i.p, i.bytes))
      return op_fail(MOE_ERR_SHAPE, "int4 linear: out and the workspace must not overlap the inputs");
  if (overlaps(out, no, workspace, need))
    return op_fail(MOE_ERR_SHAPE, "int4 linear: out must not overlap the workspace");
  (void)workspace_bytes;
  const Int4Args a{x, reinterpret_cast<const uint32_t*>(weight->qweight),
                   reinterpret_cast<const uint32_t*>(weight->qzeros), weight->scales, bias, out, T,
                   K, N, group_size};
  const auto s = (hipStream_t)stream;
  MOE_OP_HIP(dtype == kBf16 ? launch_int4<kBf16>(a, s) : launch_int4<kFp16>(a, s), "int4 linear");
  return MOE_OK;
}

}  // extern "C"
