// Sums over a row held 8 columns a thread, and over rows: what the norms share.
#pragma once

#include <algorithm>
#include <initializer_list>

#include "common.h"
#include "elem.h"

constexpr int kMaxHidden = 8192;

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

// Sums of N values over the NT threads of a row (all threads get them), in a fixed order. A is the type
// they are taken in, P that of a thread's own part. NT up to 64: no barrier.
template <int NT, int N, class P, class A>
MOE_DEV void row_sums(const P (&part)[N], A (&v)[N], A (*s_part)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = part[i];
    if constexpr (NT > 32) v[i] += partner<32>(v[i]);
    if constexpr (NT > 16) v[i] += partner<16>(v[i]);
    if constexpr (NT > 8) v[i] += partner<8>(v[i]);
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

// 1 / sqrt(m), rounded to fp32 at the end: the hardware's approximation and a Newton step in 64 bits.
// inv_sqrt_near: m within [2^-100, 2^127]. inv_sqrt: outside that of m rounded to fp32 (0 beyond its range).
MOE_DEV float inv_sqrt_near(double m) {
  const double r = (double)__builtin_amdgcn_rsqf((float)m);
  return (float)(r + 0.5 * r * (1.0 - m * r * r));
}
MOE_DEV float inv_sqrt(double m) {
  const float v = (float)m;
  if (!(v >= 0x1p-100f && v < __builtin_inff())) return 1.0f / __builtin_sqrtf(v);
  return inv_sqrt_near(m);
}

// Threads a row takes, and the workgroup of (at least 256) threads they lie in.
inline int threads_of(int H) { return H <= 512 ? 64 : H <= 2048 ? 256 : H <= 4096 ? 512 : 1024; }
inline int rows_of(int nt) { return nt < 256 ? 256 / nt : 1; }
template <int NT>
constexpr int block_threads() { return NT < 256 ? 256 : NT; }

#define MOE_ROW_NT(LAUNCH)                       \
  if (nt == 64) {                                \
    if (vec) LAUNCH(64, true); else LAUNCH(64, false);     \
  } else if (nt == 256) {                        \
    if (vec) LAUNCH(256, true); else LAUNCH(256, false);   \
  } else if (nt == 512) {                        \
    if (vec) LAUNCH(512, true); else LAUNCH(512, false);   \
  } else {                                       \
    if (vec) LAUNCH(1024, true); else LAUNCH(1024, false); \
  }

// A tensor's memory.
struct Span {
  const void* p;
  int64_t bytes;
};

// Whether rows of H columns can be taken 8 at a time (Cols<..., VEC = true>) in all of the tensors.
inline bool vec_ok(int H, std::initializer_list<const void*> ps) {
  if (H % 8 != 0) return false;
  for (const void* p : ps)
    if (!aligned16(p)) return false;
  return true;
}
