// Symmetric int8 quantisation of token rows: q = rint(127 x / a), scale = a / 127, a = max |x|.
//
// HBM-bound: one read of x, half (a quarter for fp32) of it written. The row stays in registers
// between the maximum, taken over magnitude bits, and the quotients.
#include "elem.h"
#include "int8.h"

namespace {

// NT threads a row, NC chunks of 8 NT columns.
template <int DT, int NT, int NC, bool VEC>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void quantize_kernel(
    const typename Elem<DT>::T* __restrict__ x, int T, int K, int8_t* __restrict__ q,
    float* __restrict__ scale) {
  using C = Cols<DT, NT, VEC>;
  __shared__ uint32_t s_max[NT / 64];
  const int tid = threadIdx.x % NT;
  constexpr int kRows = NT < 256 ? 256 / NT : 1;
  const int64_t t = (int64_t)blockIdx.x * kRows +
                    __builtin_amdgcn_readfirstlane((int)threadIdx.x / NT);
  if (t >= T) return;  // a whole wave (NT = 64, no barrier below), or never
  float v[NC][8];
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < NC; ++c) C::load(x + t * K + c * 8 * NT, tid, K - c * 8 * NT, v[c]);
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, magnitude(v[c][e]));
  top = bfly_umax(top);
  if constexpr (NT > 64) {
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) top = max(top, s_max[w]);
  }
  if (tid == 0) scale[t] = Quantizer::scale(top);
  const Quantizer quant(top);
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    int8_t* p = q + t * K + c * 8 * NT;
    const int left = K - c * 8 * NT;
    if constexpr (VEC) {
      const float (&x8)[8] = v[c];
      if (8 * tid < left)
        *reinterpret_cast<u32x2*>(p + 8 * tid) =
            u32x2{quant.four(x8[0], x8[1], x8[2], x8[3]), quant.four(x8[4], x8[5], x8[6], x8[7])};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (tid + NT * e < left) p[tid + NT * e] = quant.one(v[c][e]);
    }
  }
}

template <int DT>
hipError_t launch_quantize_t(const void* x, int T, int K, int8_t* q, float* scale, hipStream_t s) {
  const auto* xt = static_cast<const typename Elem<DT>::T*>(x);
  const bool vec = K % 8 == 0 && aligned16(x) && (reinterpret_cast<uintptr_t>(q) & 7u) == 0;
#define MOE_QUANT(NT, NC)                                                                       \
  do {                                                                                          \
    const dim3 grid((unsigned)(NT < 256 ? (T + 256 / NT - 1) / (256 / NT) : T));                \
    const dim3 block(NT < 256 ? 256 : NT);                                                      \
    if (vec)                                                                                    \
      hipLaunchKernelGGL((quantize_kernel<DT, NT, NC, true>), grid, block, 0, s, xt, T, K, q,   \
                         scale);                                                                \
    else                                                                                        \
      hipLaunchKernelGGL((quantize_kernel<DT, NT, NC, false>), grid, block, 0, s, xt, T, K, q,  \
                         scale);                                                                \
  } while (0)
  // a wave a row while it holds the row: no barrier between the loads and the quotients
  if (K <= 512) MOE_QUANT(64, 1);
  else if (K <= 1024) MOE_QUANT(64, 2);
  else if (K <= 2048) MOE_QUANT(64, 4);
  else if (K <= 4096) MOE_QUANT(256, 2);
  else if (K <= 8192) MOE_QUANT(256, 4);
  else MOE_QUANT(1024, 8);
#undef MOE_QUANT
  return hipGetLastError();
}

}  // namespace

hipError_t launch_quantize(const void* x, int T, int K, int dtype, int8_t* q, float* scale,
                           hipStream_t s) {
  if (T <= 0) return hipSuccess;
  if (dtype == kBf16) return launch_quantize_t<kBf16>(x, T, K, q, scale, s);
  if (dtype == kFp16) return launch_quantize_t<kFp16>(x, T, K, q, scale, s);
  return launch_quantize_t<kFp32>(x, T, K, q, scale, s);
}
