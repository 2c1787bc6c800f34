// Symmetric int8 quantisation of token rows: q = rint(127 x / a), scale = a / 127, a = max |x|.
//
// HBM-bound: one read of x, half (a quarter for fp32) of it written. The row stays in registers
// between the maximum, taken over magnitude bits, and the quotients.
#include "elem.h"
#include "int8.h"

namespace {

template <int DT, int NT, int NC, bool VEC>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void quantize_kernel(
    const typename Elem<DT>::T* __restrict__ x, int T, int K, int8_t* __restrict__ q,
    float* __restrict__ scale) {
  quantize_rows<DT, NT, NC, VEC>(blockIdx.x, x, T, K, q, scale);
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
