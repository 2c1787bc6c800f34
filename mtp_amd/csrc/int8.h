// The int8 products' kernels as the entry points see them.
#pragma once

#include "elem.h"

// a rows [rows][K] with a scale each; b [N][K] with a scale per channel, of one expert or of all
// of them, N * K bytes apart. Output row r of a tile comes from a's row row_src[r] / src_div (r
// without row_src).
struct Int8Args {
  const int8_t* a;
  const float* a_scale;
  const int32_t* row_src;
  int src_div;
  uint32_t a_bytes;
  const int8_t* b0;       // SiLU products: gate
  const int8_t* b1;       // SiLU products: up
  const float* s0;
  const float* s1;
  const i32x4* tiles;     // {expert, first row, rows, 0}; NULL: consecutive rows of one matrix
  int m_tiles;            // entries of the tile table, or the row blocks of one matrix
  int M, N, K;
  void* out;              // [M][N]
  const void* bias;       // [N] or NULL
};

// Symmetric quantisation of a row of values whose largest magnitude has the bits `top` (NaN above
// infinity): q = rint(127 x / a). 127 x is exact for bf16 and fp16 values (8 and 11 bits by 7) and a
// correctly rounded division then rounds only once: a quotient that is a tie is represented, and
// one that is not lies further from the tie than the division's half step, so q equals that of exact
// arithmetic (ties to even). Rows are scaled by a power of two first, where 127 x could overflow or
// the quotient's operands be subnormal. A row of zeros, and one that holds an infinity or NaN, gives 0.
// The quotient is that of an IEEE division: with y = 1 / d correctly rounded (once a row) and
// c = n y, c + (n - c d) y in fused operations is (Markstein). The compiler's division per value took
// two thirds of the kernel's time (8192 x 4096: 24 -> 16 us).
struct Quantizer {
  float f, d, y;
  uint32_t keep;
  MOE_DEV explicit Quantizer(uint32_t top) {
    const float a = __uint_as_float(top);
    const bool usable = top != 0 && top < 0x7F800000u;
    const float m = a >= 0x1p64f ? 0x1p-64f : a < 0x1p-64f ? 0x1p64f : 1.0f;
    f = usable ? 127.0f * m : 0.0f;
    d = usable ? a * m : 1.0f;
    y = 1.0f / d;
    keep = usable ? ~0u : 0u;
  }
  // q in the low byte: adding 1.5 * 2^23 rounds to an integer, half to even, in the low bits
  MOE_DEV uint32_t bits(float x) const {
    const float n = x * f, c = n * y;
    return __float_as_uint(__builtin_fmaf(__builtin_fmaf(-c, d, n), y, c) + 12582912.0f);
  }
  MOE_DEV uint32_t four(float x0, float x1, float x2, float x3) const {
    const uint32_t lo = __builtin_amdgcn_perm(bits(x1), bits(x0), 0x0C0C0400u);
    const uint32_t hi = __builtin_amdgcn_perm(bits(x3), bits(x2), 0x04000C0Cu);
    return (lo | hi) & keep;
  }
  MOE_DEV int8_t one(float x) const { return (int8_t)(bits(x) & keep); }
  // a / 127: inf or NaN for rows that hold one, so that their products are NaN
  MOE_DEV static float scale(uint32_t top) { return __uint_as_float(top) / 127.0f; }
};
MOE_DEV uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
MOE_DEV uint32_t bfly_umax(uint32_t v) {
  v = max(v, __float_as_uint(xor_partner<32>(__uint_as_float(v))));
  v = max(v, __float_as_uint(xor_partner<16>(__uint_as_float(v))));
  v = max(v, __float_as_uint(xor_partner<8>(__uint_as_float(v))));
  v = max(v, __float_as_uint(xor_partner<4>(__uint_as_float(v))));
  v = max(v, __float_as_uint(xor_partner<2>(__uint_as_float(v))));
  return max(v, __float_as_uint(xor_partner<1>(__uint_as_float(v))));
}

// The rows of one workgroup: NT threads a row, NC chunks of 8 NT columns.
template <int DT, int NT, int NC, bool VEC>
MOE_DEV void quantize_rows(int block, const typename Elem<DT>::T* __restrict__ x, int T, int K,
                           int8_t* __restrict__ q, float* __restrict__ scale) {
  using C = Cols<DT, NT, VEC>;
  __shared__ uint32_t s_max[NT / 64];
  const int tid = threadIdx.x % NT;
  constexpr int kRows = NT < 256 ? 256 / NT : 1;
  const int64_t t = (int64_t)block * kRows +
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

// Quantise rows of the dtype to int8 with a scale each.
hipError_t launch_quantize(const void* x, int T, int K, int dtype, int8_t* q, float* scale,
                           hipStream_t s);
// launch_quantize of x [T][K] and launch_dispatch's tables (no rows), which do not depend on each
// other, in one launch where a wave holds a row (K <= 2048), two or three otherwise.
hipError_t launch_quantize_and_sort(const void* x, int T, int K, int dtype, int8_t* q, float* scale,
                                    const int32_t* ids, int k, int E, int32_t* offsets,
                                    int32_t* row_slot, int32_t* slot_row, void* ws, i32x4* tiles,
                                    int bm, int tile_cap, hipStream_t s);
// The kernel of a product and its rows per tile (the bm of an expert table).
enum { kInt8Stream = 0, kInt8Ring = 1, kInt8Tile = 2 };
struct Int8Plan {
  int kind, bm;
  int bn = 0;  // channels a tile of the ring
};
Int8Plan int8_experts_plan(int64_t slots, int E, int I);
Int8Plan int8_matrix_plan(int64_t M, int64_t N);
hipError_t launch_int8_product(const Int8Args& a, Int8Plan plan, bool silu, int dtype,
                               hipStream_t s);
// The product of few rows of the dtype, quantised by the product's own workgroups (a's int8 rows and
// scales are not looked at): one launch, no workspace.
bool int8_fused_fits(int M, int K);
hipError_t launch_int8_fused(const Int8Args& a, const void* x, int dtype, hipStream_t s);
