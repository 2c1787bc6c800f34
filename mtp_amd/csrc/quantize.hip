// Symmetric int8 quantisation of token rows: q = rint(127 x / a), scale = a / 127, a = max |x|.
//
// The quotient is taken in this order because 127 x is exact for bf16 and fp16 values (8 and 11 bits
// by 7 bits) and an IEEE division then rounds only once: a quotient that is a tie is represented, and
// one that is not lies further from the tie than the division's half step, so q equals the one of
// exact arithmetic (ties to even). Rows are scaled by a power of two before, where 127 x could
// overflow or the quotient's operands be subnormal. A row of zeros gives q = 0, scale = 0; a row with
// an infinity or NaN gives q = 0 and scale = a / 127 (inf or NaN), so that its products are NaN.
//
// HBM-bound: one read of x, half (a quarter for fp32) of it written. The row stays in registers
// between the maximum and the quotients; the maximum is taken over magnitude bits (NaN above
// infinity).
#include "elem.h"
#include "int8.h"

namespace {

MOE_DEV uint32_t bfly_umax(uint32_t v) {
  auto step = [](uint32_t a, float b) { return max(a, __float_as_uint(b)); };
  v = step(v, xor_partner<32>(__uint_as_float(v)));
  v = step(v, xor_partner<16>(__uint_as_float(v)));
  v = step(v, xor_partner<8>(__uint_as_float(v)));
  v = step(v, xor_partner<4>(__uint_as_float(v)));
  v = step(v, xor_partner<2>(__uint_as_float(v)));
  return step(v, xor_partner<1>(__uint_as_float(v)));
}

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
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[c][e]) & 0x7FFFFFFFu);
  top = bfly_umax(top);
  if constexpr (NT > 64) {
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) top = max(top, s_max[w]);
  }
  const float a = __uint_as_float(top);
  if (tid == 0) scale[t] = a / 127.0f;
  const bool usable = top != 0 && top < 0x7F800000u;
  const float m = a >= 0x1p64f ? 0x1p-64f : a < 0x1p-64f ? 0x1p64f : 1.0f;
  const float d = usable ? a * m : 1.0f, f = usable ? m : 0.0f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    int b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float n = usable ? v[c][e] * f * 127.0f : 0.0f;
      b[e] = (int)__builtin_rintf(n / d);
    }
    int8_t* p = q + t * K + c * 8 * NT;
    const int left = K - c * 8 * NT;
    if constexpr (VEC) {
      if (8 * tid < left) {
        u32x2 o;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          o[h] = (uint32_t)(b[4 * h] & 255) | (uint32_t)(b[4 * h + 1] & 255) << 8 |
                 (uint32_t)(b[4 * h + 2] & 255) << 16 | (uint32_t)(b[4 * h + 3] & 255) << 24;
        *reinterpret_cast<u32x2*>(p + 8 * tid) = o;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (tid + NT * e < left) p[tid + NT * e] = (int8_t)b[e];
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
  if (K <= 512) MOE_QUANT(64, 1);
  else if (K <= 2048) MOE_QUANT(256, 1);
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
