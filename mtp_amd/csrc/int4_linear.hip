// A linear layer on int4 weights with a scale and a zero point per group of K (the GPTQ layout of the
// experts, one matrix):
//
//   y[t, n] = round(sum_g s[g, n] * (sum_{k in g} x[t, k] (q[k, n] - z[g, n])) (+ bias[n]))
//
// The weights are not rounded: a group's products are summed in fp32 on the integers q - z and scaled
// after that. Of x up to 2^64 all sums stay in fp32's range: sums of x (16 + q) over K <= 2^16 below 2^85, and
// those of many rows, in units of a scale (2^-24 .. 2^16), below 2^124. Beyond it they may not, and infinities
// of both signs meet in a NaN. Four forms:
//   few rows   operands from memory to registers, the words made into MFMA operands there. Reading the
//              weights bounds it, and the launch where they are few: 1 row of 2048 x 4096 4.2 us, of 8192 x
//              16384 17 (4.1 TB/s), 16 rows of 4096 x 8192 8.8 (2.0 TB/s), of 8192 x 16384 21 (3.3 TB/s).
//   more rows  the same words, x shared through LDS: 128 rows of 4096 x 8192 18 us, 256 28 (605 TFLOP/s).
//              Vector operations and multiplications bound it.
//   many rows  integers unpacked once, then a tiled product from LDS: 4096 rows of 4096 x 8192 219 us, 12
//              of them the unpacking (1.33 PFLOP/s in the product). The matrix and vector pipes bound it.
//   unaligned  value by value, for tensors that start between two 16-byte boundaries.
// Times are of captured graphs, a call behind the other, each with weights of its own that come from HBM.
#include <algorithm>
#include <type_traits>

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
  int T, K, N, G, groups;
  void* workspace;
};

// ---------------------------------------------------------------- operands
// A packed word holds 8 consecutive k of one channel, which is what one lane contributes to a 16x16x32
// MFMA. The word becomes the operand in the types' own bits, in the order of k: a nibble lands in the
// mantissa of a constant OFF whose last place it then counts in, so a value is OFF + q, exact (bf16
// 16 + q: 0x4180 | q << 3; fp16 64 + q: 0x5400 | q << 4): two nibbles a register by a byte permute, a
// mask and an or, 10 VALU operations a word and 9. The offset and the zero point leave by the sum of x:
//   sum x (q - z) = sum x (OFF + q) - (OFF + z) sum x
// with OFF small, so that little is cancelled (a magnitude of up to 31 or 79 for q - z of up to 15).
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// Byte i of each word into a half of register i, masked, in the constant: one v_perm_b32 and one
// v_and_or_b32, which takes one scalar and no literal (left to itself the compiler used two literals in
// two operations).
MOE_DEV uint32_t constant_s(uint32_t c) {
  asm("" : "+s"(c));
  return c;
}
MOE_DEV uint32_t constant_v(uint32_t c) {
  asm("" : "+v"(c));
  return c;
}
MOE_DEV u32x4 spread(uint32_t even, uint32_t odd, uint32_t mask, uint32_t base) {
  u32x4 v;
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i)
    v[i] = (__builtin_amdgcn_perm(odd, even, 0x0C040C00u + 0x00010001u * i) & mask) | base;
  return v;
}

template <int DT>
struct Op;
template <>
struct Op<kBf16> {
  static constexpr uint32_t kOnes = 0x3F803F80u;
  // OFF + the nibble at bit `at`, as a float
  MOE_DEV static float zero_point(uint32_t z, int at) {
    return __uint_as_float(((at <= 19 ? z << (19 - at) : z >> (at - 19)) & 0x00780000u) | 0x41800000u);
  }
  MOE_DEV static u32x4 weights(uint32_t w) {
    return spread(w << 3, w >> 1, constant_s(0x00780078u), constant_v(0x41804180u));
  }
  MOE_DEV static f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
};
template <>
struct Op<kFp16> {
  static constexpr uint32_t kOnes = 0x3C003C00u;
  MOE_DEV static float zero_point(uint32_t z, int at) {
    return __uint_as_float(((at <= 17 ? z << (17 - at) : z >> (at - 17)) & 0x001E0000u) | 0x42800000u);
  }
  MOE_DEV static u32x4 weights(uint32_t w) {
    return spread(w << 4, w, constant_s(0x00F000F0u), constant_v(0x54005400u));
  }
  MOE_DEV static f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
};

// ---------------------------------------------------------------- few rows
// Workgroup: 16 MT tokens x 16 CT channels, K dealt to its KS waves in chunks of 32 SPG (a quantisation
// group or a part of one) in turn; the waves' sums meet in LDS. Weights and x go from memory to the
// registers that the MFMA reads, the next chunk's while this one is multiplied. The channels are the A
// operand's rows (lane l: channels CT (l & 15) .. + CT - 1, one load) and the tokens the B operand's
// columns, so a lane ends with channels 4 CT (l >> 4) .. + 4 CT - 1 of token l & 15. The sum of x comes
// from an MFMA with ones.
template <int MT, int CT, int SPG>
struct Chunk {
  u32x4 x[MT][SPG];
  uint32_t w[SPG][CT];
  uint32_t s[2 * CT];          // fp16 pairs of the lane's 4 CT results
  uint32_t z[(CT + 1) / 2];
};

template <int DT, int MT, int CT, int SPG, int KS>
__global__ __launch_bounds__(64 * KS) void int4_stream_kernel(Int4Args a, uint32_t row_tiles,
                                                             uint32_t row_magic,
                                                             uint32_t group_magic) {
  using T = typename Elem<DT>::T;
  using O = Op<DT>;
  __shared__ f32x4 red[KS][MT * CT][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // A channel tile's row tiles run behind each other on one XCD, which then holds its weights in L2.
  const uint32_t idx = blockIdx.x >> 3;
  const uint32_t ct = row_magic ? __umulhi(idx, row_magic) : idx;
  const int c0 = (int)(ct * 8 + (blockIdx.x & 7)) * 16 * CT, t0 = (int)(idx - ct * row_tiles) * 16 * MT;
  if (c0 >= a.N) return;
  const int lr = lane & 15, lq = lane >> 4;
  const __amdgpu_buffer_rsrc_t rx = buf_rsrc(a.x, (uint32_t)a.T * (uint32_t)a.K * 2u);
  const __amdgpu_buffer_rsrc_t rw = buf_rsrc(a.qweight, (uint32_t)(a.K / 8) * (uint32_t)a.N * 4u);
  const __amdgpu_buffer_rsrc_t rs = buf_rsrc(a.scales, (uint32_t)a.groups * (uint32_t)a.N * 2u);
  const __amdgpu_buffer_rsrc_t rz = buf_rsrc(a.qzeros, (uint32_t)a.groups * (uint32_t)(a.N / 8) * 4u);
  uint32_t xoff[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int t = t0 + 16 * m + lr;
    xoff[m] = t < a.T ? (uint32_t)t * (uint32_t)a.K * 2u + 16u * lq : kOutOfRange;
  }
  const int cw = c0 + CT * lr, cd = c0 + 4 * CT * lq;  // first channel loaded, first one of the result
  const uint32_t woff = cw < a.N ? ((uint32_t)lq * (uint32_t)a.N + (uint32_t)cw) * 4u : kOutOfRange;
  const uint32_t soff = cd < a.N ? (uint32_t)cd * 2u : kOutOfRange;
  const uint32_t zoff = cd < a.N ? (uint32_t)(cd / 8) * 4u : kOutOfRange;
  const int chunks = a.K / (32 * SPG);
  // a chunk past the last reads zeros without a memory access
  auto load = [&](Chunk<MT, CT, SPG>& c, int at) {
    const bool in = at < chunks;
    const uint32_t out = in ? 0u : kOutOfRange;
    const uint32_t k = in ? (uint32_t)at * 32u * SPG : 0u;
    const uint32_t g =
        !in ? 0u : group_magic ? __umulhi((uint32_t)at, group_magic) : (uint32_t)at;
#pragma unroll
    for (int s = 0; s < SPG; ++s) {
      const uint32_t row = (k / 8 + 4 * s) * (uint32_t)a.N * 4u;
      if constexpr (CT == 1) {
        c.w[s][0] = buf_ld32(rw, woff | out, row);
      } else if constexpr (CT == 2) {
        const u32x2 v = buf_ld64(rw, woff | out, row);
        c.w[s][0] = v[0];
        c.w[s][1] = v[1];
      } else {
        const u32x4 v = buf_ld128(rw, woff | out, row);
#pragma unroll
        for (int j = 0; j < CT; ++j) c.w[s][j] = v[j];
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int s = 0; s < SPG; ++s) c.x[m][s] = buf_ld128(rx, (xoff[m] + 64u * s) | out, k * 2u);
    const uint32_t srow = g * (uint32_t)a.N * 2u, zrow = g * (uint32_t)(a.N / 8) * 4u;
    if constexpr (CT == 1) {
      const u32x2 v = buf_ld64(rs, soff | out, srow);
      c.s[0] = v[0];
      c.s[1] = v[1];
    } else {
#pragma unroll
      for (int h = 0; h < CT / 2; ++h) {
        const u32x4 v = buf_ld128(rs, (soff + 16u * h) | out, srow);
#pragma unroll
        for (int i = 0; i < 4; ++i) c.s[4 * h + i] = v[i];
      }
    }
#pragma unroll
    for (int h = 0; h < (CT + 1) / 2; ++h) c.z[h] = buf_ld32(rz, (zoff + 4u * h) | out, zrow);
  };
  f32x4 acc[MT][CT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < CT; ++j) acc[m][j] = f32x4{0, 0, 0, 0};
  const u32x4 ones{O::kOnes, O::kOnes, O::kOnes, O::kOnes};
  auto multiply = [&](const Chunk<MT, CT, SPG>& c) {
    f32x4 part[MT][CT], sum[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      sum[m] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < CT; ++j) part[m][j] = f32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int s = 0; s < SPG; ++s) {
#pragma unroll
      for (int m = 0; m < MT; ++m) sum[m] = O::mfma(ones, c.x[m][s], sum[m]);
#pragma unroll
      for (int j = 0; j < CT; ++j) {
        const u32x4 w = O::weights(c.w[s][j]);
#pragma unroll
        for (int m = 0; m < MT; ++m) part[m][j] = O::mfma(w, c.x[m][s], part[m][j]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < CT; ++j) {
        const int v = CT * i + j;  // the lane's channel
        const float s = f16_to_f32(v & 1 ? c.s[v / 2] >> 16 : c.s[v / 2] & 0xFFFFu);
        const uint32_t z = CT == 1 ? c.z[0] >> (16 * (lq & 1)) : c.z[v / 8];
        const float zb = O::zero_point(z, 4 * (v & 7));
#pragma unroll
        for (int m = 0; m < MT; ++m)
          acc[m][j][i] = __builtin_fmaf(s, __builtin_fmaf(-zb, sum[m][0], part[m][j][i]), acc[m][j][i]);
      }
  };
  Chunk<MT, CT, SPG> ca, cb;
  load(ca, wave);
  for (int at = wave;; at += 2 * KS) {
    load(cb, at + KS);
    __builtin_amdgcn_sched_barrier(0);
    multiply(ca);
    if (at + KS >= chunks) break;
    load(ca, at + 2 * KS);
    __builtin_amdgcn_sched_barrier(0);
    multiply(cb);
    if (at + 2 * KS >= chunks) break;
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int u = 0; u < CT; ++u) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = acc[m][(4 * u + e) % CT][(4 * u + e) / CT];
      red[wave][m * CT + u][lane] = v;
    }
  __syncthreads();
  // a thread four channels: the waves' sums in their order
  for (int f = tid; f < MT * CT * 64; f += 64 * KS) {
    const int l = f & 63, u = (f >> 6) % CT, m = f / (64 * CT);
    f32x4 v = red[0][f >> 6][l];
#pragma unroll
    for (int w = 1; w < KS; ++w) v += red[w][f >> 6][l];
    const int t = t0 + 16 * m + (l & 15), n = c0 + 4 * CT * (l >> 4) + 4 * u;
    if (t >= a.T || n >= a.N) continue;
    T out[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (a.bias) v[e] += Elem<DT>::get(static_cast<const T*>(a.bias)[n + e]);
      out[e] = Elem<DT>::put(v[e]);
    }
    __builtin_memcpy(static_cast<T*>(a.out) + (int64_t)t * a.N + n, out, sizeof(out));
  }
}

// x / d is the upper half of x * magic(d) where x * d < 2^32; d == 1 would need 2^32 itself.
uint32_t magic(uint32_t d) { return (uint32_t)(((uint64_t(1) << 32) + d - 1) / d); }

template <int DT, int MT, int CT, int SPG, int KS>
hipError_t launch_stream(const Int4Args& a, hipStream_t s) {
  const int row_tiles = (a.T + 16 * MT - 1) / (16 * MT), tiles = (a.N + 16 * CT - 1) / (16 * CT);
  const int64_t blocks = (int64_t)((tiles + 7) / 8 * 8) * row_tiles;
  hipLaunchKernelGGL((int4_stream_kernel<DT, MT, CT, SPG, KS>), dim3((unsigned)blocks),
                     dim3(64 * KS), 0, s, a, (uint32_t)row_tiles, magic((uint32_t)row_tiles),
                     magic((uint32_t)(a.G / (32 * SPG))));
  return hipGetLastError();
}

// ---------------------------------------------------------------- more rows
// Workgroup: 64 tokens x 32 WN channels on WN x KS waves: K in KS shares, a share on WN waves in steps
// of 64, and the shares' sums added at the end. x reaches a share's waves through LDS, the words stay packed:
// every wave loads those of its own 32 channels, their scales and zero points. All of it goes through a ring
// of RING stages filled by loads that bypass the registers. The rest is as with few rows. EVERY: groups end at
// multiples of so many steps (1 or 2), where the sums of the group are scaled and added up.
//
// What bounds it is issuing vector operations (40 to make operands of a step's words, 80 to scale a group's
// sums) and multiplications (24, 8 of them for the sums of x; each takes 8 of its 16 cycles of the vector
// operations' issue): 1220 cycles a step for two waves a SIMD, which takes 1900 with the waits at the barrier.
// What is shared is x (few rows: 256 rows of 4096 x 8192 44 us, here 27), what is saved the unpacking and its
// launch (many rows: 39).
//
// LDS rows of x are 128 bytes, the 16-byte chunk c of row r at position c ^ (r & 7): the 8 rows that a phase
// of a 16-byte read spans lie in different banks.
constexpr int kGroupM = 4;
constexpr int kBK = 64;
// The kernels' bodies in pieces: called many times over, they would become functions.
#define MOE_INLINE __attribute__((always_inline))
// s_waitcnt immediate waiting for lgkmcnt <= 0 only.
constexpr int kWaitLgkm0 = 15 | (3 << 14) | (0x7 << 4);

template <int DT, int WN, int KS, int RING, int EVERY>
__global__ __launch_bounds__(64 * WN * KS) void int4_words_kernel(Int4Args a, uint32_t group_magic) {
  using T = typename Elem<DT>::T;
  using O = Op<DT>;
  constexpr int MT = 4, CT = 2, NT = 64 * WN, BK = kBK, BM = 16 * MT, CH = 16 * CT, BN = CH * WN;
  constexpr int LA = BM * 8 / NT, kLoads = LA + 3;
  // bytes: a wave's words, scales and zero points, a share's and all of a stage
  constexpr int kMine = 1024 + 256 + 256, kPart = BM * 128 + WN * kMine;
  constexpr int kSums = KS > 1 ? WN * MT * CT * 1024 : 0;
  constexpr int kStage = KS * kPart > kSums ? KS * kPart : kSums;
  static_assert(LA * NT == BM * 8, "whole loads");
  static_assert(RING >= 2 && RING <= 4 && KS <= RING + 1, "a stage an array, a share's sums a stage");
  // separate arrays: the compiler then knows which stage a load to LDS writes
  __shared__ __attribute__((aligned(16))) uint8_t lds0[kStage];
  __shared__ __attribute__((aligned(16))) uint8_t lds1[kStage];
  __shared__ __attribute__((aligned(16))) uint8_t lds2[RING > 2 ? kStage : 16];
  __shared__ __attribute__((aligned(16))) uint8_t lds3[RING > 3 ? kStage : 16];
  const int m_tiles = (a.T + BM - 1) / BM, blocks_n = (a.N + BN - 1) / BN;
  // each XCD takes a run of tiles, down kGroupM row blocks before the next channels
  const int idx = blockIdx.x >> 3, xcd = blockIdx.x & 7;
  const int total = m_tiles * blocks_n, per = (total + 7) / 8, id = xcd * per + idx;
  if (idx >= per || id >= total) return;
  const int group = id / (kGroupM * blocks_n), in = id - group * kGroupM * blocks_n;
  const int grows = min(kGroupM, m_tiles - group * kGroupM);
  const int t0 = (group * kGroupM + in % grows) * BM, n0 = in / grows * BN;
  const int ks = __builtin_amdgcn_readfirstlane((int)threadIdx.x / NT);  // the share of K
  const int tid = threadIdx.x % NT, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int steps = ((a.K + BK - 1) / BK + 2 * KS - 1) / (2 * KS) * 2;  // of a share
  const int k_first = ks * steps * BK, k_end = min(a.K, k_first + steps * BK);
  const int lr = lane & 15, lq = lane >> 4;
  const __amdgpu_buffer_rsrc_t rx = buf_rsrc(a.x, (uint32_t)a.T * (uint32_t)a.K * 2u);
  const __amdgpu_buffer_rsrc_t rw = buf_rsrc(a.qweight, (uint32_t)(a.K / 8) * (uint32_t)a.N * 4u);
  const __amdgpu_buffer_rsrc_t rs = buf_rsrc(a.scales, (uint32_t)a.groups * (uint32_t)a.N * 2u);
  const __amdgpu_buffer_rsrc_t rz = buf_rsrc(a.qzeros, (uint32_t)a.groups * (uint32_t)(a.N / 8) * 4u);
  // One offset a lane and a scalar one for each load. Rows behind the last token may hold anything (a
  // lane's results are of its own token), but are read inside the buffer: a load whose first row lies
  // behind reads another one's rows.
  const uint32_t xoff =
      (uint32_t)(tid / 8) * (uint32_t)a.K * 2u + (uint32_t)((tid & 7) ^ ((tid >> 3) & 7)) * 16u;
  uint32_t xrow[LA];
#pragma unroll
  for (int j = 0; j < LA; ++j) {
    const int t = t0 + j * (NT / 8);
    xrow[j] = t < a.T ? (uint32_t)t * (uint32_t)a.K * 2u : 0u;
  }
  const int nw = n0 + wave * CH;  // the wave's first channel
  const int nl = nw + lane % 8 * 4;  // of the words: 8 lanes a row of 32
  const uint32_t woff =
      nl < a.N ? ((uint32_t)(lane / 8) * (uint32_t)a.N + (uint32_t)nl) * 4u : kOutOfRange;
  const uint32_t soff = lane < CH / 2 && nw + 2 * lane < a.N ? (uint32_t)(nw + 2 * lane) * 2u : kOutOfRange;
  const uint32_t zoff = lane < CH / 8 && nw + 8 * lane < a.N ? (uint32_t)(nw / 8 + lane) * 4u : kOutOfRange;
  // A stage past the share reads zeros without a memory access, so that as many loads are in flight in
  // every step.
  // The scalar offsets stay inside the buffers: the bounds check takes them off the buffers' sizes.
  auto stage = [&](uint8_t* lds, int k0) MOE_INLINE {
    lds += ks * kPart;
    k0 += k_first;
    const uint32_t at = k0 < k_end ? (uint32_t)k0 : 0u, out = k0 < k_end ? 0u : kOutOfRange;
#pragma unroll
    for (int j = 0; j < LA; ++j)
      buf_ld128_lds(rx, lds + (j * NT + wave * 64) * 16, xoff | out, xrow[j] + at * 2u);
    uint8_t* const mine = lds + BM * 128 + wave * kMine;
    buf_ld128_lds(rw, mine, woff | out, at / 8 * (uint32_t)a.N * 4u);
    const uint32_t g = at / kBK * group_magic >> 21;
    buf_ld32_lds(rs, mine + 1024, soff | out, g * (uint32_t)a.N * 2u);
    buf_ld32_lds(rz, mine + 1024 + 256, zoff | out, g * (uint32_t)(a.N / 8) * 4u);
  };
  // The barrier without __syncthreads' release fence, which would wait for every load to LDS: this wave's
  // LDS accesses ahead of it are waited for, and the compiler keeps accesses on their sides.
  auto barrier = []() MOE_INLINE {
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  f32x4 acc[MT][CT], part[MT][CT], sum[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < CT; ++j) acc[m][j] = f32x4{0, 0, 0, 0};
  const u32x4 ones{O::kOnes, O::kOnes, O::kOnes, O::kOnes};
  const int sw0 = (lq ^ (lr & 7)) * 16, sw1 = ((4 + lq) ^ (lr & 7)) * 16;
  const int fa_at = ks * kPart + lr * 128;
  const int mine_at = ks * kPart + BM * 128 + wave * kMine;
  u32x4 fa[2][MT];
  uint32_t raw[2][CT];
  auto fetch = [&](const uint8_t* lds, int half) MOE_INLINE {
    const int sw = half ? sw1 : sw0;
#pragma unroll
    for (int m = 0; m < MT; ++m) fa[half][m] = ld128(lds + fa_at + m * 16 * 128 + sw);
    const uint8_t* p = lds + mine_at + ((4 * half + lq) * CH + CT * lr) * 4;
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
    raw[half][0] = v[0];
    raw[half][1] = v[1];
  };
  // fresh: a group starts (or a part of one)
  auto multiply = [&](int half, bool fresh) MOE_INLINE {
    const f32x4 zero{0, 0, 0, 0};
#pragma unroll
    for (int m = 0; m < MT; ++m) sum[m] = O::mfma(ones, fa[half][m], fresh ? zero : sum[m]);
#pragma unroll
    for (int j = 0; j < CT; ++j) {
      const u32x4 w = O::weights(raw[half][j]);
#pragma unroll
      for (int m = 0; m < MT; ++m) part[m][j] = O::mfma(w, fa[half][m], fresh ? zero : part[m][j]);
    }
  };
  u32x4 sc;
  uint32_t zp;
  auto fetch_unit = [&](const uint8_t* lds) MOE_INLINE {
    const uint8_t* p = lds + mine_at + 1024;
    sc = ld128(p + 8 * CT * lq);
    zp = *reinterpret_cast<const uint32_t*>(p + 256 + 2 * CT * lq);
  };
  auto finish = [&]() MOE_INLINE {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < CT; ++j) {
        const int v = CT * i + j;  // the lane's channel
        const float s = f16_to_f32(v & 1 ? sc[v / 2] >> 16 : sc[v / 2] & 0xFFFFu);
        const float zb = O::zero_point(zp, 4 * v);
#pragma unroll
        for (int m = 0; m < MT; ++m)
          acc[m][j][i] = __builtin_fmaf(s, __builtin_fmaf(-zb, sum[m][0], part[m][j][i]), acc[m][j][i]);
      }
  };
  auto step = [&](uint8_t* here, uint8_t* next, int k0, bool starts, bool ends) MOE_INLINE {
    fetch(here, 1);
    if (ends) fetch_unit(here);
    multiply(0, starts);
    // This wave's loads of the next stage have landed (those of the stages after it stay in flight); behind
    // the barrier everybody's have, and this stage, all of it in registers, is free.
    __builtin_amdgcn_s_waitcnt(waitcnt_vm((RING - 2) * kLoads));
    barrier();
    stage(here, k0 + RING * BK);
    fetch(next, 0);  // behind the last step: zeros that nothing multiplies
    multiply(1, false);
    if (ends) finish();
    __builtin_amdgcn_sched_barrier(0);
  };
  stage(lds0, 0);
  stage(lds1, BK);
  if constexpr (RING > 2) stage(lds2, 2 * BK);
  if constexpr (RING > 3) stage(lds3, 3 * BK);
  __builtin_amdgcn_s_waitcnt(waitcnt_vm((RING - 1) * kLoads));
  barrier();
  fetch(lds0, 0);
  using std::integral_constant;
  // Which stage a step works on and whether a group may start or end there is known in a run of kSteps. Whole
  // runs first, without branches between their steps: at a join the compiler would wait for all loads to LDS.
  constexpr int kSteps = EVERY == 2 && RING % 2 ? 2 * RING : RING;
  auto nth = [&](auto i_c, int k0) MOE_INLINE {
    constexpr int i = decltype(i_c)::value, at = i % RING, to = (i + 1) % RING;
    uint8_t* const here = at == 0 ? lds0 : at == 1 ? lds1 : at == 2 ? lds2 : lds3;
    uint8_t* const next = to == 0 ? lds0 : to == 1 ? lds1 : to == 2 ? lds2 : lds3;
    step(here, next, k0 + i * BK, i % EVERY == 0, i % EVERY == EVERY - 1);
  };
  int k0 = 0;
#pragma unroll 1
  for (; k0 + (kSteps - 1) * BK < steps * BK; k0 += kSteps * BK) {
    nth(integral_constant<int, 0>{}, k0);
    nth(integral_constant<int, 1>{}, k0);
    if constexpr (kSteps > 2) nth(integral_constant<int, 2>{}, k0);
    if constexpr (kSteps > 3) nth(integral_constant<int, 3>{}, k0);
    if constexpr (kSteps > 4) nth(integral_constant<int, 4>{}, k0);
    if constexpr (kSteps > 5) nth(integral_constant<int, 5>{}, k0);
  }
  if (k0 < steps * BK) nth(integral_constant<int, 0>{}, k0);
  if constexpr (kSteps > 2)
    if (k0 + BK < steps * BK) nth(integral_constant<int, 1>{}, k0);
  if constexpr (kSteps > 3)
    if (k0 + 2 * BK < steps * BK) nth(integral_constant<int, 2>{}, k0);
  if constexpr (kSteps > 4)
    if (k0 + 3 * BK < steps * BK) nth(integral_constant<int, 3>{}, k0);
  if constexpr (kSteps > 5)
    if (k0 + 4 * BK < steps * BK) nth(integral_constant<int, 4>{}, k0);
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));  // no load to LDS may meet the sums below
  if constexpr (KS > 1) {  // the shares' sums, in their order
    __syncthreads();  // the stages have been read
    if (ks > 0) {
      f32x4* const p = reinterpret_cast<f32x4*>(ks == 1 ? lds0 : ks == 2 ? lds1 : lds2);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < CT; ++j) p[((wave * MT + m) * CT + j) * 64 + lane] = acc[m][j];
    }
    __syncthreads();
    if (ks > 0) return;
#pragma unroll
    for (int q = 1; q < KS; ++q) {
      const f32x4* const p = reinterpret_cast<const f32x4*>(q == 1 ? lds0 : q == 2 ? lds1 : lds2);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < CT; ++j) acc[m][j] += p[((wave * MT + m) * CT + j) * 64 + lane];
    }
  }
  // A lane holds 4 CT neighbouring channels of a token for each m.
  const int n = nw + 4 * CT * lq;
  if (n >= a.N) return;
  u32x4 bits{0, 0, 0, 0};
  if (a.bias) __builtin_memcpy(&bits, static_cast<const T*>(a.bias) + n, 16);
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int t = t0 + m * 16 + lr;
    if (t >= a.T) continue;
    T v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[e] = Elem<DT>::put(acc[m][e % CT][e / CT] + Elem<DT>::get((T)(bits[e >> 1] >> (16 * (e & 1)))));
    __builtin_memcpy(__builtin_assume_aligned(static_cast<T*>(a.out) + (int64_t)t * a.N + n, 16), v, 16);
  }
}

template <int DT, int WN, int KS, int RING>
hipError_t launch_words(const Int4Args& a, hipStream_t s) {
  constexpr int BM = 64, BN = 32 * WN;
  const int64_t tiles = (int64_t)((a.T + BM - 1) / BM) * ((a.N + BN - 1) / BN);
  const dim3 grid((unsigned)((tiles + 7) / 8 * 8)), block(64 * WN * KS);
  // x / d is x * g >> 21 for x and d up to 1024
  const uint32_t d = (uint32_t)a.G / kBK, g = ((1u << 21) + d - 1) / d;
  if (a.G % (2 * kBK))
    hipLaunchKernelGGL((int4_words_kernel<DT, WN, KS, RING, 1>), grid, block, 0, s, a, g);
  else
    hipLaunchKernelGGL((int4_words_kernel<DT, WN, KS, RING, 2>), grid, block, 0, s, a, g);
  return hipGetLastError();
}

// ---------------------------------------------------------------- many rows
// Two launches. The first turns the words into the integers q - z as fp8 (e4m3 holds 4 significant bits:
// exact), a wave 64 channels x 64 k, stored as the tiles below take them: [K / 64][N][64], a row's 16-byte
// chunk c holding k 8 c .. + 7 and 32 + 8 c .. + 7, zeros past K; and for each 64 k (32 where groups may end
// there) the ratio of the scale before to the one from there on. The second is a product of x with them,
// turned into x's type (exact) on the way from LDS.
//
// The product keeps its sums in units of the present group's scale: where a group ends they are multiplied
// by s[g - 1] / s[g], which takes an operation a sum and no second set of sums. A scale of zero counts as
// one, with integers of zero.

MOE_DEV float scale_unit(uint32_t s) {
  const float f = f16_to_f32(s & 0xFFFFu);
  return f == 0.0f ? 1.0f : f;
}

// Four nibbles of a word, from bit `at` on, less the zero point.
MOE_DEV uint32_t integers(uint32_t w, int at, float z) {
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = (float)((w >> (at + 4 * i)) & 15u) - z;
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], v, true);
}

__global__ __launch_bounds__(256) void int4_unpack_kernel(Int4Args a, uint8_t* __restrict__ w,
                                                          float* __restrict__ ratio, int halves) {
  const int lane = threadIdx.x & 63, c = lane & 3;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int blocks_n = (a.N + 255) / 256;
  const int n = (blockIdx.x % blocks_n * 4 + wave) * 64 + (lane >> 2) * 4, stage = blockIdx.x / blocks_n;
  if (n >= a.N) return;
  uint32_t row[4][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int k = stage * kBK + 32 * h + 8 * c;
    const bool in = k < a.K;
    const int g = in ? k / a.G : 0;
    const u32x4 q = ld128(a.qweight + (int64_t)(in ? k / 8 : 0) * a.N + n);
    const uint32_t z = a.qzeros[(int64_t)g * (a.N / 8) + n / 8] >> (4 * (n & 7));
    const u32x2 s = *reinterpret_cast<const u32x2*>(a.scales + (int64_t)g * a.N + n);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t keep = in && (s[j >> 1] >> (16 * (j & 1)) & 0x7FFFu) != 0 ? ~0u : 0u;
      const float zf = (float)((z >> (4 * j)) & 15u);
      row[j][2 * h] = integers(q[j], 0, zf) & keep;
      row[j][2 * h + 1] = integers(q[j], 16, zf) & keep;
    }
    if (c == 0 && (h == 0 || halves)) {
      const int before = in ? max(k - 1, 0) / a.G : 0;
      const u32x2 p = *reinterpret_cast<const u32x2*>(a.scales + (int64_t)before * a.N + n);
      f32x4 r;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        r[j] = scale_unit(p[j >> 1] >> (16 * (j & 1))) / scale_unit(s[j >> 1] >> (16 * (j & 1)));
      *reinterpret_cast<f32x4*>(ratio + (int64_t)(halves ? 2 * stage + h : stage) * a.N + n) = r;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<u32x4*>(w + ((int64_t)stage * a.N + n + j) * kBK + 16 * c) =
        u32x4{row[j][0], row[j][1], row[j][2], row[j][3]};
}

// Workgroup: BM tokens x BN channels on WM x WN waves, K steps of 64 in a ring of RING stages in LDS, filled
// by loads that bypass the registers. One wait and barrier in the middle of a step orders the arrival of the
// next stage and the reuse of this one, whose second half is in registers by then: loads have RING - 1 steps
// to arrive (whole steps held in registers, or rings of 5 to 8 stages, gained nothing). LDS rows of x are 128
// bytes, the 16-byte chunk c of row r at position c ^ (r & 7); rows of integers 64 bytes, chunk c at
// c ^ (r / 2 & 3): the 8 rows that a phase of a 16-byte read spans lie in different banks. EVERY: groups end
// at multiples of so many half steps (1, 2 or 4).

// 8 integers in fp8 as an MFMA operand.
template <int DT>
MOE_DEV u32x4 operand(uint32_t lo, uint32_t hi) {
  if constexpr (DT == kBf16)
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true))};
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true))};
}

template <int BM, int BN, int WM, int WN, int RING, int DT, int EVERY>
__global__ __launch_bounds__(64 * WM * WN) void int4_tile_kernel(Int4Args a,
                                                                 const uint8_t* __restrict__ w,
                                                                 const float* __restrict__ ratio) {
  using T = typename Elem<DT>::T;
  using O = Op<DT>;
  constexpr int NT = 64 * WM * WN, BK = kBK;
  constexpr int MT = BM / WM / 16, NG = BN / WN / 16;
  constexpr int LA = BM * 8 / NT, LB = BN * 4 / NT, LR = EVERY == 1 ? 2 : 1;
  constexpr int kRowsAt = BM * 128, kRatioAt = kRowsAt + BN * 64, kStage = kRatioAt + LR * 1024;  // bytes
  static_assert(LA * NT == BM * 8 && LB * NT == BN * 4 && BN <= 256, "whole loads");
  static_assert(RING >= 2 && RING <= 4, "a stage an array");
  // separate arrays: the compiler then knows which stage a load to LDS writes
  __shared__ __attribute__((aligned(16))) uint8_t lds0[kStage];
  __shared__ __attribute__((aligned(16))) uint8_t lds1[kStage];
  __shared__ __attribute__((aligned(16))) uint8_t lds2[RING > 2 ? kStage : 16];
  __shared__ __attribute__((aligned(16))) uint8_t lds3[RING > 3 ? kStage : 16];
  const int m_tiles = (a.T + BM - 1) / BM, blocks_n = (a.N + BN - 1) / BN;
  // each XCD takes a run of tiles, down kGroupM row blocks before the next channels
  const int idx = blockIdx.x >> 3, xcd = blockIdx.x & 7;
  const int total = m_tiles * blocks_n, per = (total + 7) / 8, id = xcd * per + idx;
  if (idx >= per || id >= total) return;
  const int group = id / (kGroupM * blocks_n), in = id - group * kGroupM * blocks_n;
  const int grows = min(kGroupM, m_tiles - group * kGroupM);
  const int t0 = (group * kGroupM + in % grows) * BM, n0 = in / grows * BN;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN, lr = lane & 15, lq = lane >> 4;
  const __amdgpu_buffer_rsrc_t rx = buf_rsrc(a.x, (uint32_t)a.T * (uint32_t)a.K * 2u);
  const uint32_t kc = (uint32_t)((tid & 7) ^ ((tid >> 3) & 7)) * 16;  // the chunk's byte of x's row
  // One offset a lane and a scalar one for each load. Rows behind the last token or channel may hold
  // anything (a lane's results are of its own token and channels, which are then not stored), but are read
  // inside the buffers: a load whose first row lies behind reads another one's rows.
  const uint32_t xoff = (uint32_t)(tid / 8) * (uint32_t)a.K * 2u + kc;
  const uint32_t woff = (uint32_t)(tid / 4) * kBK + 16u * ((tid & 3) ^ ((tid >> 3) & 3));
  uint32_t xrow[LA], wrow[LB];
#pragma unroll
  for (int j = 0; j < LA; ++j) {
    const int t = t0 + j * (NT / 8);
    xrow[j] = t < a.T ? (uint32_t)t * (uint32_t)a.K * 2u : 0u;
  }
#pragma unroll
  for (int j = 0; j < LB; ++j) {
    const int n = n0 + j * (NT / 4);
    wrow[j] = n < a.N ? (uint32_t)n * kBK : 0u;
  }
  const uint32_t roff = 4 * lane < BN && n0 + 4 * lane < a.N ? (uint32_t)(n0 + 4 * lane) * 4u : kOutOfRange;
  // A stage past K reads zeros without a memory access, so that as many loads are in flight in every step.
  // The scalar offsets stay inside the buffers: the bounds check takes them off the buffers' sizes.
  auto stage = [&](uint8_t* lds, int k0) MOE_INLINE {
    const uint32_t out = 2 * k0 + (int)kc < 2 * a.K ? 0u : kOutOfRange;
    const uint32_t at = k0 < a.K ? (uint32_t)k0 : 0u, none = k0 < a.K ? 0u : kOutOfRange;
    const __amdgpu_buffer_rsrc_t rw = buf_rsrc(w + (int64_t)at * a.N, (uint32_t)a.N * (uint32_t)BK);
#pragma unroll
    for (int j = 0; j < LA; ++j)
      buf_ld128_lds(rx, lds + (j * NT + wave * 64) * 16, xoff | out, xrow[j] + at * 2u);
#pragma unroll
    for (int j = 0; j < LB; ++j)
      buf_ld128_lds(rw, lds + kRowsAt + (j * NT + wave * 64) * 16, woff | none, wrow[j]);
    // the ratios; every wave stores the same
    const __amdgpu_buffer_rsrc_t rr = buf_rsrc(ratio + (int64_t)(at / kBK) * LR * a.N, LR * (uint32_t)a.N * 4u);
#pragma unroll
    for (int h = 0; h < LR; ++h)
      buf_ld128_lds(rr, lds + kRatioAt + h * 1024, roff | none, (uint32_t)h * (uint32_t)a.N * 4u);
  };
  // The barrier without __syncthreads' release fence, which would wait for every load to LDS: this wave's
  // LDS accesses ahead of it are waited for, and the compiler keeps accesses on their sides.
  auto barrier = []() MOE_INLINE {
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  f32x4 acc[NG][MT];
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[g][m] = f32x4{0, 0, 0, 0};
  const int sw0 = (lq ^ (lr & 7)) * 16, sw1 = ((4 + lq) ^ (lr & 7)) * 16, sww = (lq ^ ((lr >> 1) & 3)) * 16;
  const int fa_at = (wm * 16 + lr) * 128, fb_at = kRowsAt + (wn * NG * 16 + lr) * 64 + sww;
  // A step is four phases of half the wave's rows and half of the step's K, pipelined through two register
  // sets: while one phase's rows are multiplied the next one's are read from LDS. A phase in which a group
  // starts multiplies its sums by the ratios first, in the MFMA's shadow.
  constexpr int PM = MT / 2;
  static_assert(MT % 2 == 0, "phases of half the rows");
  u32x4 fa[2][PM], raw[NG], fb[2][NG];
  f32x4 unit[NG];
  auto fetch_x = [&](const uint8_t* lds, int half, int part) MOE_INLINE {
    const int sw = half ? sw1 : sw0;
#pragma unroll
    for (int m = 0; m < PM; ++m) fa[part][m] = ld128(lds + fa_at + (part * PM + m) * WM * 16 * 128 + sw);
  };
  auto fetch_w = [&](const uint8_t* lds) MOE_INLINE {
#pragma unroll
    for (int g = 0; g < NG; ++g) raw[g] = ld128(lds + fb_at + g * 16 * 64);
  };
  auto fetch_unit = [&](const uint8_t* lds, int half) MOE_INLINE {
#pragma unroll
    for (int g = 0; g < NG; ++g)
      unit[g] = *reinterpret_cast<const f32x4*>(lds + kRatioAt + half * 1024 +
                                                ((wn * NG + g) * 16 + 4 * lq) * 4);
  };
  auto operands = [&](int half) MOE_INLINE {
#pragma unroll
    for (int g = 0; g < NG; ++g) fb[half][g] = operand<DT>(raw[g][2 * half], raw[g][2 * half + 1]);
  };
  // reads, loads: the LDS reads and the loads to LDS of the phase, spread over its multiplications
  auto multiply = [&](int half, int part, bool starts, auto reads_c, auto loads_c) MOE_INLINE {
    constexpr int kReads = decltype(reads_c)::value, kLoads = decltype(loads_c)::value, kOps = PM * NG;
#pragma unroll
    for (int m = 0; m < PM; ++m)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        f32x4& c = acc[g][part * PM + m];
        if (starts) c *= unit[g];
        c = O::mfma(fb[half][g], fa[part][m], c);
      }
    constexpr int kEach = kOps / (kReads + 1) > 0 ? kOps / (kReads + 1) : 1;
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      if (i < kLoads) __builtin_amdgcn_sched_group_barrier(0x010, (kLoads + kReads - 1) / kReads, 0);
      if (starts) __builtin_amdgcn_sched_group_barrier(0x002, 4 * kEach, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  using std::integral_constant;
  auto step = [&](uint8_t* here, uint8_t* next, int k0, bool starts) MOE_INLINE {
    if (EVERY == 1) fetch_unit(here, 0);
    operands(1);
    fetch_x(here, 0, 1);
    multiply(0, 0, starts, integral_constant<int, PM>{}, integral_constant<int, 0>{});
    fetch_x(here, 1, 0);
    multiply(0, 1, starts, integral_constant<int, PM>{}, integral_constant<int, 0>{});
    if (EVERY == 1) fetch_unit(here, 1);
    fetch_x(here, 1, 1);
    multiply(1, 0, EVERY == 1, integral_constant<int, PM>{}, integral_constant<int, 0>{});
    // This wave's loads of the next stage have landed (those of the stages after it stay in flight); behind
    // the barrier everybody's have, and this stage, all of it in registers, is free.
    __builtin_amdgcn_s_waitcnt(waitcnt_vm((RING - 2) * (LA + LB + LR)));
    barrier();
    stage(here, k0 + RING * BK);
    fetch_w(next);  // behind the last step: zeros that nothing multiplies
    fetch_x(next, 0, 0);
    // past K both operands are zeros
    multiply(1, 1, EVERY == 1, integral_constant<int, PM + NG>{}, integral_constant<int, LA + LB + LR>{});
    if (EVERY != 1) fetch_unit(next, 0);
    operands(0);
  };
  stage(lds0, 0);
  stage(lds1, BK);
  if constexpr (RING > 2) stage(lds2, 2 * BK);
  if constexpr (RING > 3) stage(lds3, 3 * BK);
  __builtin_amdgcn_s_waitcnt(waitcnt_vm((RING - 1) * (LA + LB + LR)));
  barrier();
  fetch_w(lds0);
  fetch_x(lds0, 0, 0);
  fetch_unit(lds0, 0);
  operands(0);
  // Which stage a step works on and whether a group may start there is known in a run of kSteps. Whole runs
  // first, without branches between their steps: at a join the compiler would wait for all loads to LDS.
  constexpr int kSteps = EVERY == 4 && RING % 2 ? 2 * RING : RING;
  auto nth = [&](auto i_c, int k0) MOE_INLINE {
    constexpr int i = decltype(i_c)::value, at = i % RING, to = (i + 1) % RING;
    uint8_t* const here = at == 0 ? lds0 : at == 1 ? lds1 : at == 2 ? lds2 : lds3;
    uint8_t* const next = to == 0 ? lds0 : to == 1 ? lds1 : to == 2 ? lds2 : lds3;
    step(here, next, k0 + i * BK, EVERY < 4 || i % 2 == 0);
  };
  int k0 = 0;
#pragma unroll 1
  for (; k0 + (kSteps - 1) * BK < a.K; k0 += kSteps * BK) {
    nth(integral_constant<int, 0>{}, k0);
    nth(integral_constant<int, 1>{}, k0);
    if constexpr (kSteps > 2) nth(integral_constant<int, 2>{}, k0);
    if constexpr (kSteps > 3) nth(integral_constant<int, 3>{}, k0);
    if constexpr (kSteps > 4) nth(integral_constant<int, 4>{}, k0);
    if constexpr (kSteps > 5) nth(integral_constant<int, 5>{}, k0);
  }
  if (k0 < a.K) nth(integral_constant<int, 0>{}, k0);
  if constexpr (kSteps > 2)
    if (k0 + BK < a.K) nth(integral_constant<int, 1>{}, k0);
  if constexpr (kSteps > 3)
    if (k0 + 2 * BK < a.K) nth(integral_constant<int, 2>{}, k0);
  if constexpr (kSteps > 4)
    if (k0 + 3 * BK < a.K) nth(integral_constant<int, 3>{}, k0);
  if constexpr (kSteps > 5)
    if (k0 + 4 * BK < a.K) nth(integral_constant<int, 4>{}, k0);
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));  // no load to LDS may meet the rows below
  // Epilogue: 16 rows at a time through the wave's share of LDS, whole lines stored.
  constexpr int CH = NG * 16, PITCH = CH + 8;
  static_assert(NT / 64 * 16 * PITCH * 2 <= kStage, "the rows fit a stage");
  const int n_wave = n0 + wn * CH, lk4 = 4 * lq;
  u32x2 last[NG], bits[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const int c = min(n_wave + g * 16 + lk4, a.N - 4);
    last[g] = *reinterpret_cast<const u32x2*>(a.scales + (int64_t)(a.groups - 1) * a.N + c);
    bits[g] = u32x2{0, 0};
  }
  if (a.bias) {
#pragma unroll
    for (int g = 0; g < NG; ++g)
      __builtin_memcpy(&bits[g], static_cast<const T*>(a.bias) + min(n_wave + g * 16 + lk4, a.N - 4), 8);
  }
  __syncthreads();  // the stages have been read
  T* mine = reinterpret_cast<T*>(lds0) + wave * 16 * PITCH;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r0 = t0 + (m * WM + wm) * 16;
    if (r0 >= a.T) continue;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      T v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = Elem<DT>::put(__builtin_fmaf(acc[g][m][i], scale_unit(last[g][i >> 1] >> (16 * (i & 1))),
                                            Elem<DT>::get((T)(bits[g][i >> 1] >> (16 * (i & 1))))));
      __builtin_memcpy(__builtin_assume_aligned(mine + lr * PITCH + g * 16 + lk4, 8), v, sizeof(v));
    }
    // the lanes of this wave have written what its lanes read (one wave's LDS accesses are in order)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    constexpr int kPerRow = CH / 8;  // lanes a row
#pragma unroll
    for (int q = 0; q < (16 * kPerRow + 63) / 64; ++q) {
      const int row = (q * 64 + lane) / kPerRow, c = (lane % kPerRow) * 8;
      if (row < 16 && r0 + row < a.T && n_wave + c < a.N)
        *reinterpret_cast<u32x4*>(static_cast<T*>(a.out) + (int64_t)(r0 + row) * a.N + n_wave + c) =
            *reinterpret_cast<const u32x4*>(mine + row * PITCH + c);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// HALVES: groups may end in the middle of a step.
template <int BM, int BN, int WM, int WN, int RING, int DT, bool HALVES>
hipError_t launch_tile(const Int4Args& a, hipStream_t s) {
  const int64_t tiles = (int64_t)((a.T + BM - 1) / BM) * ((a.N + BN - 1) / BN);
  const int stages = (a.K + kBK - 1) / kBK;
  uint8_t* w = static_cast<uint8_t*>(a.workspace);
  float* ratio = reinterpret_cast<float*>(w + (int64_t)stages * a.N * kBK);
  hipLaunchKernelGGL(int4_unpack_kernel, dim3((unsigned)stages * (unsigned)((a.N + 255) / 256)),
                     dim3(256), 0, s, a, w, ratio, (int)HALVES);
  const dim3 grid((unsigned)((tiles + 7) / 8 * 8)), block(64 * WM * WN);
  if constexpr (HALVES)
    hipLaunchKernelGGL((int4_tile_kernel<BM, BN, WM, WN, RING, DT, 1>), grid, block, 0, s, a, w, ratio);
  else if (a.G % (2 * kBK))
    hipLaunchKernelGGL((int4_tile_kernel<BM, BN, WM, WN, RING, DT, 2>), grid, block, 0, s, a, w, ratio);
  else
    hipLaunchKernelGGL((int4_tile_kernel<BM, BN, WM, WN, RING, DT, 4>), grid, block, 0, s, a, w, ratio);
  return hipGetLastError();
}

// ---------------------------------------------------------------- any alignment
// A thread an output channel, kRows tokens, value by value: for tensors that start between two 16-byte
// boundaries.
constexpr int kRows = 8;

template <int DT>
__global__ __launch_bounds__(256) void int4_values_kernel(Int4Args a) {
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

// Workgroups of the few-rows kernel.
int64_t stream_groups(int T, int N, int rows, int channels) {
  return (int64_t)((T + rows - 1) / rows) * ((N + channels - 1) / channels);
}

// The larger a tile the fewer bytes of x and weights a workgroup reads for a result, the smaller the more
// workgroups there are: the largest of these that its rows fill half of and that still gives most of the CUs
// one. us with 16 x 16, 16 x 32, 16 x 64, 32 x 64, 64 x 64: 1 row of 2048 x 4096 4.3 / 4.7 / 5.7, of 4096 x 8192
// 9.3 / 7.1 / 8.4; 16 rows of 8192 x 16384 41 / 26 / 19 / 23 / 31, 32 of it 74 / 45 / 32 / 25 / 34; 48 rows of
// 2048 x 4096 9.5 / 8.1 / 6.6 / 8.6 / 13; 64 rows of 2048 x 4096 12 / 8.1 / 6.7 / 8.6 / 14, of 4096 x 8192 38 / 24
// / 18 / 15 / 23; 96 of 2048 x 4096 17 / 11 / 11 / 8.6 / 14; 203 of 1056 x 2008 13 / 9.2 / 8.1 / 7.0 / 10; 256 of
// 4096 x 8192 146 / 88 / 66 / 54 / 47 (groups of 64 and 128 have the kernel for more rows there). 32 x 32 and 64
// x 32 are never the best.
constexpr int kEnough = 192;
template <int DT, int SPG>
hipError_t launch_few_rows(const Int4Args& a, hipStream_t s) {
  if constexpr (SPG == 1) {
    if (a.T > 32 && stream_groups(a.T, a.N, 64, 64) >= kEnough) return launch_stream<DT, 4, 4, SPG, 4>(a, s);
  }
  if (a.T > 16 && stream_groups(a.T, a.N, 32, 64) >= kEnough) return launch_stream<DT, 2, 4, SPG, 8>(a, s);
  if (stream_groups(a.T, a.N, 16, 64) >= kEnough) return launch_stream<DT, 1, 4, SPG, 8>(a, s);
  if (stream_groups(a.T, a.N, 16, 32) >= kEnough) return launch_stream<DT, 1, 2, SPG, 8>(a, s);
  return launch_stream<DT, 1, 1, SPG, 8>(a, s);
}

// Tiles of 64 tokens x 64 channels.
int64_t words_tiles(int T, int N) { return (int64_t)((T + 63) / 64) * ((N + 63) / 64); }

// Which form takes aligned tensors. us with few / more / many rows' kernels, groups of 128:
//   64 rows of 4096 x 8192 (128 tiles of 64 x 64) 15 / 18 / 39, 96 of 2048 x 4096 (128) 11 / 11 / 21, 192 of
//   2048 x 4096 (192) 16 / 11 / 22, 48 of 4096 x 16384 (256) 25 / 19 / 48, 128 of 4096 x 8192 (256) 23 / 18 /
//   39, 256 (512) 44 / 27 / 39, 512 (1024) 86 / 48 / 50, 640 (1280) 106 / 71 / 68, 1024 (2048) - / 93 / 75.
// A row tile of 64 is half empty for 32 rows, which few rows' kernels take in tiles of 32. Unpacking costs as
// much however few rows read the integers (12 us for 4096 x 8192) and a tile's products save about 28 of 92
// us for 1024 rows: they pay from some 400 rows on.
// Groups that are no multiple of 64 end inside a step, which doubles more rows' vector operations (256 rows of
// 4096 x 8192 with 32 a group 61 us). There few / many rows: 256 rows of 4096 x 8192 44 / 54, 512 80 / 64,
// 1000 of 1056 x 2048 15 / 19: the sides meet at about the same T sqrt(N K).
// (The tiles' 32-bit offsets hold 2^24 channels.)
bool many_rows(int T, int K, int N, int G) {
  if (T < 64 || N > (1 << 24)) return false;
  return G % kBK ? (double)T * T * N * K >= 4e12 : T >= 400 && words_tiles(T, N) > 1024;
}
bool more_rows(int T, int K, int N, int G) {
  return G % kBK == 0 && T > 32 && words_tiles(T, N) > 160 && !many_rows(T, K, N, G);
}

// 64 x 64 in four shares of K while that is a workgroup a CU, 64 x 128 in two then, and in one at two
// workgroups a CU: us 128 rows of 4096 x 8192 (256 tiles of 64 x 64) 18 / 27 / 33, 256 rows (512) 34 / 27 /
// 34, 384 rows (768) 49 / 51 / 46.
template <int DT>
hipError_t launch_more_rows(const Int4Args& a, hipStream_t s) {
  const int64_t tiles = words_tiles(a.T, a.N);
  if (tiles <= 256) return launch_words<DT, 2, 4, 3>(a, s);
  if (tiles <= 512) return launch_words<DT, 4, 2, 3>(a, s);
  return launch_words<DT, 4, 1, 4>(a, s);
}

// By the number of 128 x 128 tiles, us with 64 x 128 / 128 x 128 / 128 x 256 / 256 x 256: 128 tiles (256 rows
// of 4096 x 8192) 40 / 48 / 66 / 107, 192 (384 rows) 51 / 49 / 67 / 105, 256 (512 rows) 56 / 51 / 67 / 107, 384
// (768 rows) 76 / 79 / 69 / 108, 512 (1024 rows) 91 / 84 / 76 / 108, 768 (3000 of 2048 x 4096) 71 / 67 / 69 /
// 61, 2048 (4096 of 4096 x 8192) 302 / 290 / 250 / 217. Between 64 x 128 tiles of 4 waves and of 8 there is
// nothing to choose; 128 x 128 on 4 waves takes 55 us for the 512 rows. The small tiles are for groups that
// are no multiple of 64: the others get here with more than 256 tiles only.
template <int DT>
hipError_t launch_many_rows(const Int4Args& a, hipStream_t s) {
  const int64_t tiles = (int64_t)((a.T + 127) / 128) * ((a.N + 127) / 128);
  if (a.G % kBK) {
    if (tiles <= 160) return launch_tile<64, 128, 2, 2, 4, DT, true>(a, s);
    if (tiles <= 320) return launch_tile<128, 128, 2, 4, 4, DT, true>(a, s);
    if (tiles <= 640) return launch_tile<128, 256, 2, 4, 3, DT, true>(a, s);
    return launch_tile<256, 256, 2, 4, 2, DT, true>(a, s);
  }
  if (tiles <= 640) return launch_tile<128, 256, 2, 4, 3, DT, false>(a, s);
  return launch_tile<256, 256, 2, 4, 2, DT, false>(a, s);
}

template <int DT>
hipError_t launch_int4(const Int4Args& a, bool aligned, hipStream_t s) {
  if (!aligned) {
    const int64_t blocks = (int64_t)((a.N + 255) / 256) * ((a.T + kRows - 1) / kRows);
    hipLaunchKernelGGL(int4_values_kernel<DT>, dim3((unsigned)blocks), dim3(256), 0, s, a);
    return hipGetLastError();
  }
  if (many_rows(a.T, a.K, a.N, a.G)) return launch_many_rows<DT>(a, s);
  if (more_rows(a.T, a.K, a.N, a.G)) return launch_more_rows<DT>(a, s);
  if (a.G % 128 == 0) return launch_few_rows<DT, 4>(a, s);
  if (a.G % 64 == 0) return launch_few_rows<DT, 2>(a, s);
  return launch_few_rows<DT, 1>(a, s);
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
  // the integers, and two ratios for each 64 of them
  return many_rows(T, K, N, group_size) ? (int64_t)((K + 63) / 64) * N * (64 + 8) : 0;
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
  const int64_t need = moe_int4_linear_workspace_bytes_v1(T, K, N, group_size);
  if (need > 0) {
    if (!workspace || workspace_bytes < need)
      return op_fail(MOE_ERR_WORKSPACE, "int4 linear: workspace of %lld bytes, needs %lld",
                     (long long)(workspace ? workspace_bytes : 0), (long long)need);
    if (!workspace_aligned(workspace))
      return op_fail(MOE_ERR_WORKSPACE, "int4 linear: workspace must be 256-byte aligned");
  }
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
  const Int4Args a{x, reinterpret_cast<const uint32_t*>(weight->qweight),
                   reinterpret_cast<const uint32_t*>(weight->qzeros), weight->scales, bias, out, T,
                   K, N, group_size, K / group_size, workspace};
  const bool aligned = aligned16(x) && aligned16(weight->qweight) && aligned16(weight->scales) &&
                       aligned16(out);
  const auto s = (hipStream_t)stream;
  MOE_OP_HIP(dtype == kBf16 ? launch_int4<kBf16>(a, aligned, s) : launch_int4<kFp16>(a, aligned, s),
             "int4 linear");
  return MOE_OK;
}

}  // extern "C"
