// Rows of bf16, fp16 or fp32 values as floats, 8 columns a thread: the I/O of the kernels that take
// all three types, and the error reports of their entry points.
#pragma once

#include <cstdarg>
#include <cstdio>

#include "common.h"
#include "launch.h"

// dtype codes of the C ABI (the ones of moe_dequant_v1's out_dtype).
enum { kBf16 = 0, kFp16 = 1, kFp32 = 2 };

template <int DT>
struct Elem {
  using T = uint16_t;
  MOE_DEV static float get(T v) { return DT == kBf16 ? bf16_to_f32(v) : f16_to_f32(v); }
  // round to nearest even, as the hardware conversions do (v_cvt_pk_bf16_f32, v_cvt_f16_f32)
  MOE_DEV static T put(float f) {
    if constexpr (DT == kBf16) return __builtin_bit_cast(uint16_t, (__bf16)f);
    return __builtin_bit_cast(uint16_t, (_Float16)f);
  }
};
template <>
struct Elem<kFp32> {
  using T = float;
  MOE_DEV static float get(float v) { return v; }
  MOE_DEV static float put(float f) { return f; }
};

// The 8 columns c .. c + 7 of a row (16-byte aligned).
template <int DT>
MOE_DEV void ld8(const typename Elem<DT>::T* p, float (&v)[8]) {
  if constexpr (DT == kFp32) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = a[j];
      v[4 + j] = b[j];
    }
  } else {
    const u32x4 d = ld128(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = Elem<DT>::get((uint16_t)(d[j] & 0xFFFFu));
      v[2 * j + 1] = Elem<DT>::get((uint16_t)(d[j] >> 16));
    }
  }
}
template <int DT>
MOE_DEV void st8(typename Elem<DT>::T* p, const float (&v)[8]) {
  if constexpr (DT == kFp32) {
    *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    u32x4 d;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      d[j] = (uint32_t)Elem<DT>::put(v[2 * j]) | ((uint32_t)Elem<DT>::put(v[2 * j + 1]) << 16);
    *reinterpret_cast<u32x4*>(p) = d;
  }
}

// The 8 columns of thread `tid` of NT in a row of H columns. VEC: columns 8 tid .. 8 tid + 7, all
// inside or all outside the row (H % 8 == 0, rows 16-byte aligned); otherwise columns tid + NT e
// (neighbouring threads on neighbouring elements), each checked. Columns outside read 0.
template <int DT, int NT, bool VEC>
struct Cols {
  using T = typename Elem<DT>::T;
  // Without branches: a thread outside the row reads columns inside it and drops them (in branches
  // every load was waited for before the next was issued). `row` may be a chunk of a row behind its
  // end (H <= 0): the row's last columns are read then, so the row itself holds at least 8 columns
  // (VEC) or one.
  MOE_DEV static void load(const T* row, int tid, int H, float (&v)[8]) {
    if constexpr (VEC) {
      ld8<DT>(row + min(8 * tid, H - 8), v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 8 * tid < H ? v[e] : 0.0f;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = Elem<DT>::get(row[min(tid + NT * e, H - 1)]);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = tid + NT * e < H ? v[e] : 0.0f;
    }
  }
  MOE_DEV static void store(T* row, int tid, int H, const float (&v)[8]) {
    if constexpr (VEC) {
      if (8 * tid < H) st8<DT>(row + 8 * tid, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (tid + NT * e < H) row[tid + NT * e] = Elem<DT>::put(v[e]);
    }
  }
  MOE_DEV static int col(int tid, int e) { return VEC ? 8 * tid + e : tid + NT * e; }
};

// The same columns as the registers they are loaded into, unpacked where they are used: half the
// registers of floats, for rows whose loads run ahead of their use.
template <int DT, int NT, bool VEC>
struct RawCols {
  using T = typename Elem<DT>::T;
  using C = Cols<DT, NT, VEC>;
  static constexpr int kWords = 2 * (int)sizeof(T);
  uint32_t w[kWords];
  MOE_DEV void load(const T* row, int tid, int H) {
    if constexpr (VEC) {
      const T* p = row + min(8 * tid, H - 8);
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const u32x4 d = ld128(reinterpret_cast<const u32x4*>(p) + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[4 * i + j] = d[j];
      }
    } else if constexpr (DT == kFp32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(row[min(tid + NT * e, H - 1)]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e += 2)
        w[e / 2] = (uint32_t)row[min(tid + NT * e, H - 1)] |
                   (uint32_t)row[min(tid + NT * (e + 1), H - 1)] << 16;
    }
  }
  // column e of the thread; 0 outside the row
  MOE_DEV float get(int e, int tid, int H) const {
    float v;
    if constexpr (DT == kFp32) v = __uint_as_float(w[e]);
    else v = Elem<DT>::get((T)(w[e / 2] >> (16 * (e & 1))));
    return C::col(tid, e) < H ? v : 0.0f;
  }
};

// The value as it reads back after being stored in the type: an fp32 result rounded to it (and not
// the last operation's exact result, as a fused multiply-add with an fp16 result would give).
template <int DT>
MOE_DEV float rounded(float f) {
  if constexpr (DT == kFp16) asm("" : "+v"(f));
  return Elem<DT>::get(Elem<DT>::put(f));
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline int64_t dtype_bytes(int dtype) { return dtype == kFp32 ? 4 : 2; }

// An entry point's failure: the message for moe_w4a16_last_error, the code to return. A HIP error
// is also cleared from the thread, so that it does not surface at the caller's next HIP call.
inline int op_fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(moe_error_buffer(), kErrorBufferBytes, fmt, ap);
  va_end(ap);
  return code;
}
inline int op_hip(hipError_t e, const char* where) {
  if (e == hipSuccess) return MOE_OK;
  (void)hipGetLastError();
  return op_fail(MOE_ERR_HIP + ((int)e % 100), "%s: HIP error %d (%s)", where, (int)e,
                 hipGetErrorString(e));
}
#define MOE_OP_HIP(expr, where)            \
  do {                                     \
    const int _rc = op_hip((expr), where); \
    if (_rc) return _rc;                   \
  } while (0)

// Whether [a, a + na) and [b, b + nb) share a byte (NULL shares none).
inline bool overlaps(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t p = (uintptr_t)a, q = (uintptr_t)b;
  return a && b && na > 0 && nb > 0 && p < q + (uintptr_t)nb && q < p + (uintptr_t)na;
}
