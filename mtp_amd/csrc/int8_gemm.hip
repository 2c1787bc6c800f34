// int8 x int8 products on MFMA with a scale per token and per channel, dense or over the tiles of
// sorted expert rows, plain or as silu(gate) * up:
//
//   y[r, n] = round((float(sum_k a[r, k] b[n, k]) * a_scale[r]) * b_scale[n] (+ bias[n]))
//   h[r, n] = round(silu(g) * u),  g and u as y in fp32 with the gate's and the up projection's b
//
// The sums are exact 32-bit integers (K <= 65536: |sum| <= 2^14 K < 2^31), so any split over K gives
// the same bits.
//
// MFMA 16x16x64: the channels are the A operand's rows and the tokens the B operand's columns, so a
// lane ends with 4 consecutive channels of one token: one 8-byte store for 16-bit outputs. Lane l
// holds bytes [16 (l >> 4), 16 (l >> 4) + 16) of row l & 15 of both operands (the same k order on both
// sides), and channels 4 (l >> 4) .. + 3 of token l & 15 of the result.
#include <algorithm>
#include <type_traits>

#include "elem.h"
#include "int8.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int64_t kMaxBlocks = int64_t(1) << 23;  // a launch holds under 2^32 threads

struct Tile {
  int expert, row0, rows;
};

// The workgroup's tile (uniform), rows 0 when there is nothing to do.
MOE_DEV Tile tile_of(const Int8Args& a, int bm, int m) {
  if (a.tiles) {
    const i32x4 t = a.tiles[m];
    return Tile{__builtin_amdgcn_readfirstlane(t[0]), __builtin_amdgcn_readfirstlane(t[1]),
                __builtin_amdgcn_readfirstlane(t[2])};
  }
  return Tile{0, m * bm, min(bm, a.M - m * bm)};
}

MOE_DEV i32x4 mfma_i8(i32x4 a, i32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// a's row of output row r.
MOE_DEV int source_row(const Int8Args& a, int r) {
  return a.row_src ? (int)((uint32_t)a.row_src[r] / (uint32_t)a.src_div) : r;
}

// SiLU of the gate and up products. silu_f32's fast exponential and reciprocal are off by up to about
// |g| half steps of fp32: little next to a 16-bit h's own half step (2^-17 of the value at |g| = 80), but
// 60 of an fp32 h's, which takes the library's exponential and a division (5 in all).
template <int DT>
MOE_DEV float silu(float g) {
  if constexpr (DT == kFp32) return g / (1.0f + expf(-g));
  return silu_f32(g);
}

// Four channels n .. n + 3 of output row r.
template <int DT>
MOE_DEV void finish(const Int8Args& a, int64_t r, int n, float rs, i32x4 sum, bool vec) {
  using T = typename Elem<DT>::T;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int ni = n + i < a.N ? n + i : a.N - 1;
    v[i] = ((float)sum[i] * rs) * a.s0[ni];
    if (a.bias) v[i] += Elem<DT>::get(static_cast<const T*>(a.bias)[ni]);
  }
  T* p = static_cast<T*>(a.out) + r * a.N + n;
  if (vec && n + 3 < a.N) {
    if constexpr (DT == kFp32) {
      *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
      *reinterpret_cast<u32x2*>(p) =
          u32x2{(uint32_t)Elem<DT>::put(v[0]) | (uint32_t)Elem<DT>::put(v[1]) << 16,
                (uint32_t)Elem<DT>::put(v[2]) | (uint32_t)Elem<DT>::put(v[3]) << 16};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) p[i] = Elem<DT>::put(v[i]);
  }
}

// ---------------------------------------------------------------- up to 16 rows
// Workgroup: all rows x 16 channels, the K steps of 64 dealt to the four waves in turn, whose sums
// meet in LDS. Weights go from memory to the registers the MFMA reads, kKU steps ahead; a byte is used
// by one wave once. 16 channels a workgroup keep 256 CUs streaming from 4096 channels on (one row of
// 2048 x 4096: 3.9 us, with 32 channels 5.0).
// FUSED: the rows come as values of the dtype and every workgroup quantises them itself, into LDS,
// while its first weights arrive: one launch instead of two, but every workgroup reads and divides
// all of x. 2048 x 4096: 5.0 us for one row (two launches 3.9 + 2.1), 11.6 for eight (4.2 + 2.3).
constexpr int kKU = 8;  // steps a load
constexpr int kFusedRows = 4, kFusedBytes = 48 << 10;

template <int DT, bool FUSED>
__global__ __launch_bounds__(kThreads) void int8_stream_kernel(
    Int8Args a, const typename Elem<DT>::T* __restrict__ x, int vec, int x_vec) {
  extern __shared__ __attribute__((aligned(16))) int8_t s_q[];  // FUSED: [M][K + 16]
  __shared__ i32x4 s_acc[kWaves][64];
  __shared__ uint32_t s_top[kWaves][kFusedRows];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lk = (lane >> 4) * 16, lk4 = (lane >> 4) * 4;
  const int n0 = blockIdx.x * 16, pitch = a.K + 16;
  const __amdgpu_buffer_rsrc_t ra = buf_rsrc(a.a, a.a_bytes);
  const __amdgpu_buffer_rsrc_t rb = buf_rsrc(a.b0, (uint32_t)((int64_t)a.N * a.K));
  const uint32_t aoff = lr < a.M ? (uint32_t)lr * (uint32_t)a.K + lk : kOutOfRange;
  const uint32_t boff = n0 + lr < a.N ? (uint32_t)(n0 + lr) * (uint32_t)a.K + lk : kOutOfRange;
  // the wave's steps s0 .. s0 + kKU - 1 (64 bytes of K, kWaves apart); zeros past K
  auto load = [&](i32x4 (&fb)[kKU], int s0) {
#pragma unroll
    for (int u = 0; u < kKU; ++u) {
      const int k = ((s0 + u) * kWaves + wave) * 64;
      const uint32_t out = k + lk < a.K ? 0u : kOutOfRange;  // K % 16 == 0: a lane's 16 bytes
      fb[u] = __builtin_bit_cast(i32x4, buf_ld128(rb, (boff + (uint32_t)k) | out));
    }
  };
  i32x4 acc{0, 0, 0, 0};
  auto multiply = [&](const i32x4 (&fb)[kKU], int s0) {
    i32x4 fa[kKU];
#pragma unroll
    for (int u = 0; u < kKU; ++u) {
      const int k = ((s0 + u) * kWaves + wave) * 64;
      const bool in = k + lk < a.K;
      if constexpr (FUSED) {
        // a token past the rows or a step past K reads another place; its product is not used, or
        // meets weights of zero
        fa[u] = *reinterpret_cast<const i32x4*>(s_q + min(lr, a.M - 1) * pitch + (in ? k + lk : 0));
      } else {
        fa[u] = __builtin_bit_cast(i32x4,
                                   buf_ld128(ra, (aoff + (uint32_t)k) | (in ? 0u : kOutOfRange)));
      }
    }
#pragma unroll
    for (int u = 0; u < kKU; ++u) acc = mfma_i8(fb[u], fa[u], acc);
  };
  const int steps = (a.K + kWaves * 64 - 1) / (kWaves * 64);
  i32x4 f0[kKU], f1[kKU];
  load(f0, 0);
  uint32_t top[kFusedRows];
  if constexpr (FUSED) {
    __builtin_amdgcn_sched_barrier(0);
    auto load_x = [&](int r, int c, float (&v)[8]) {
      const typename Elem<DT>::T* p = x + (int64_t)r * a.K + c;
      if (x_vec) {
        ld8<DT>(p, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = Elem<DT>::get(p[e]);
      }
    };
#pragma unroll
    for (int r = 0; r < kFusedRows; ++r) {
      top[r] = 0;
      if (r < a.M) {
#pragma unroll 2
        for (int c = 8 * tid; c < a.K; c += 8 * kThreads) {
          float v[8];
          load_x(r, c, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) top[r] = max(top[r], magnitude(v[e]));
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kFusedRows; ++r) {
      if (r < a.M) {
        const uint32_t t = bfly_umax(top[r]);
        if (lane == 0) s_top[wave][r] = t;
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kFusedRows; ++r) {
      if (r >= a.M) break;
      top[r] = s_top[0][r];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) top[r] = max(top[r], s_top[w][r]);
      const Quantizer quant(top[r]);
#pragma unroll 2
      for (int c = 8 * tid; c < a.K; c += 8 * kThreads) {
        float v[8];
        load_x(r, c, v);
        *reinterpret_cast<u32x2*>(s_q + r * pitch + c) =
            u32x2{quant.four(v[0], v[1], v[2], v[3]), quant.four(v[4], v[5], v[6], v[7])};
      }
    }
    __syncthreads();
  }
  for (int s0 = 0;; s0 += 2 * kKU) {
    load(f1, s0 + kKU);
    multiply(f0, s0);
    if (s0 + kKU >= steps) break;
    load(f0, s0 + 2 * kKU);
    multiply(f1, s0 + kKU);
    if (s0 + 2 * kKU >= steps) break;
  }
  s_acc[wave][lane] = acc;
  __syncthreads();
  if (wave == 0) {
    const int n = n0 + lk4;
    i32x4 sum = s_acc[0][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) sum += s_acc[w][lane];
    if (lr < a.M && n < a.N) {
      float rs;
      if constexpr (FUSED) {
        uint32_t t = s_top[0][lr];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) t = max(t, s_top[w][lr]);
        rs = Quantizer::scale(t);
      } else {
        rs = a.a_scale[lr];
      }
      finish<DT>(a, lr, n, rs, sum, vec != 0);
    }
  }
}

template <int DT, bool FUSED>
hipError_t launch_few_rows(const Int8Args& a, const void* x, hipStream_t s) {
  constexpr int es = DT == kFp32 ? 4 : 2;
  const int vec =
      a.N % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & (uintptr_t)(4 * es - 1)) == 0;
  const int64_t blocks = (a.N + 15) / 16;
  if (blocks > kMaxBlocks) return hipErrorInvalidValue;
  hipLaunchKernelGGL((int8_stream_kernel<DT, FUSED>), dim3((unsigned)blocks), dim3(kThreads),
                     FUSED ? a.M * (a.K + 16) : 0, s, a,
                     static_cast<const typename Elem<DT>::T*>(x), vec, aligned16(x) ? 1 : 0);
  return hipGetLastError();
}

// ---------------------------------------------------------------- many rows a tile
// Workgroup: BM rows x BN GEMM channels on WM x WN waves, K steps of 128 bytes staged in LDS, two
// stages filled by loads that go straight to LDS (buffer_load ... lds). One wait and barrier in the
// middle of a step orders the arrival of the next stage and the reuse of this one, whose second half
// is in registers by then: the loads of step s + 2 have a whole step to arrive. LDS rows
// are 128 bytes of K; the 16-byte chunk c of row r sits at position c ^ (r & 7), so that the 8 rows
// that one phase of a 16-byte LDS read spans lie in different banks.
// SiLU: the tile's groups of 16 channels alternate between gate and up, so that a wave holds both
// sums of a channel in the same lane.
constexpr int kGroupM = 4;
// s_waitcnt immediate waiting for lgkmcnt <= 0 only.
constexpr int kWaitLgkm0 = 15 | (3 << 14) | (0x7 << 4);

template <int BM, int BN, int WM, int WN, int DT, bool SILU>
__global__ __launch_bounds__(64 * WM * WN) void int8_tile_kernel(Int8Args a, int vec) {
  using T = typename Elem<DT>::T;
  constexpr int NT = 64 * WM * WN;
  constexpr int BK = 128;
  constexpr int MT = BM / WM / 16, NG = BN / WN / 16;
  constexpr int LA = BM * 8 / NT, LB = BN * 8 / NT;  // 16-byte loads a thread and step
  static_assert(LA * NT == BM * 8 && LB * NT == BN * 8 && NT % 256 == 0, "whole loads");
  __shared__ __attribute__((aligned(16))) int8_t lds0[(BM + BN) * BK];
  __shared__ __attribute__((aligned(16))) int8_t lds1[(BM + BN) * BK];
  __shared__ __attribute__((aligned(16))) float s_row[BM], s_col[BN], s_bias[SILU ? 4 : BN];
  const int cols = SILU ? BN / 2 : BN;
  const int blocks_n = (a.N + cols - 1) / cols;
  // Workgroups go to the 8 XCDs in turn. Of one matrix each XCD takes a run of consecutive tiles,
  // down kGroupM row blocks before the next channels, so that the 32 tiles it works on at a time are
  // about 4 x 8 and share their operands in its L2. Of experts each XCD takes every eighth row block,
  // all its channels in a row.
  const int idx = blockIdx.x >> 3, xcd = blockIdx.x & 7;
  int tile_m, tile_n;
  if (a.tiles) {
    tile_m = idx / blocks_n * 8 + xcd;
    tile_n = idx % blocks_n;
    if (tile_m >= a.m_tiles) return;
  } else {
    const int total = a.m_tiles * blocks_n, per = (total + 7) / 8, id = xcd * per + idx;
    if (idx >= per || id >= total) return;
    const int group = id / (kGroupM * blocks_n), in = id - group * kGroupM * blocks_n;
    const int rows = min(kGroupM, a.m_tiles - group * kGroupM);
    tile_m = group * kGroupM + in % rows;
    tile_n = in / rows;
  }
  const Tile tl = tile_of(a, BM, tile_m);
  if (tl.rows <= 0) return;
  const int n0 = tile_n * cols;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int lr = lane & 15;
  const int64_t eb = (int64_t)tl.expert * a.N * a.K;
  const uint32_t b_bytes = (uint32_t)((int64_t)a.N * a.K);
  const __amdgpu_buffer_rsrc_t ra = buf_rsrc(a.a, a.a_bytes);
  // a wave's 8 rows of a load lie in one group of 16 channels, the same parity in every load
  const bool up = SILU && ((wave >> 1) & 1);
  const __amdgpu_buffer_rsrc_t rb = buf_rsrc((up ? a.b1 : a.b0) + eb, b_bytes);
  const uint32_t kc = (uint32_t)((tid & 7) ^ ((tid >> 3) & 7)) * 16;  // the chunk's byte of K
  uint32_t aoff[LA], boff[LB];
#pragma unroll
  for (int j = 0; j < LA; ++j) {
    const int r = (j * NT + tid) / 8;
    aoff[j] = r < tl.rows ? (uint32_t)source_row(a, tl.row0 + r) * (uint32_t)a.K + kc : kOutOfRange;
  }
#pragma unroll
  for (int j = 0; j < LB; ++j) {
    const int i = (j * NT + tid) / 8;
    const int n = n0 + (SILU ? (i >> 5) * 16 + (i & 15) : i);
    boff[j] = n < a.N ? (uint32_t)n * (uint32_t)a.K + kc : kOutOfRange;
  }
  auto stage = [&](int8_t* lds, int k0) {
    const uint32_t out = k0 + (int)kc < a.K ? 0u : kOutOfRange;  // zeros past K
#pragma unroll
    for (int j = 0; j < LA; ++j)
      buf_ld128_lds(ra, lds + (j * NT + wave * 64) * 16, aoff[j] | out, (uint32_t)k0);
#pragma unroll
    for (int j = 0; j < LB; ++j)
      buf_ld128_lds(rb, lds + BM * BK + (j * NT + wave * 64) * 16, boff[j] | out, (uint32_t)k0);
  };
  // the epilogue's scales, loaded now: a dependent chain of loads there would be waited for
  const int64_t sb = (int64_t)tl.expert * a.N;
#pragma unroll
  for (int r = tid; r < BM; r += NT)
    s_row[r] = r < tl.rows ? a.a_scale[source_row(a, tl.row0 + r)] : 0.0f;
#pragma unroll
  for (int i = tid; i < BN; i += NT) {
    const int n = min(n0 + (SILU ? (i >> 5) * 16 + (i & 15) : i), a.N - 1);
    s_col[i] = (SILU && (i & 16) ? a.s1 : a.s0)[sb + n];
    if (!SILU && a.bias) s_bias[i] = Elem<DT>::get(static_cast<const T*>(a.bias)[n]);
  }
  i32x4 acc[NG][MT];
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[g][m] = i32x4{0, 0, 0, 0};
  const int sw0 = (((lane >> 4) ^ (lr & 7)) * 16), sw1 = ((4 + (lane >> 4)) ^ (lr & 7)) * 16;
  const int fa_at = (wm * 16 + lr) * BK, fb_at = (BM + wn * NG * 16 + lr) * BK;
  // The product over K of the first L row groups of each wave (group m of wave wm holds the tile's
  // rows 16 (m WM + wm) .. + 15, so that a tile's rows spread over its waves).
  auto product = [&](auto live_c) {
    constexpr int L = decltype(live_c)::value;
    // A step's two halves of 64 bytes of K, pipelined through two register sets: while one half is
    // multiplied the next one's operands are read from LDS.
    i32x4 fa[2][L], fb[2][NG];
    auto fetch = [&](const int8_t* lds, int half) {
      const int sw = half ? sw1 : sw0;
#pragma unroll
      for (int g = 0; g < NG; ++g)
        fb[half][g] = *reinterpret_cast<const i32x4*>(lds + fb_at + g * 16 * BK + sw);
#pragma unroll
      for (int m = 0; m < L; ++m)
        fa[half][m] = *reinterpret_cast<const i32x4*>(lds + fa_at + m * WM * 16 * BK + sw);
    };
    auto multiply = [&](int half) {
#pragma unroll
      for (int m = 0; m < L; ++m)
#pragma unroll
        for (int g = 0; g < NG; ++g) acc[g][m] = mfma_i8(fb[half][g], fa[half][m], acc[g][m]);
      // one LDS read of the next half among every few multiplications of this one
      constexpr int kReads = L + NG, kEach = L * NG / kReads > 0 ? L * NG / kReads : 1;
#pragma unroll
      for (int i = 0; i < kReads; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, L * NG, 0);
      __builtin_amdgcn_sched_barrier(0);
    };
    auto step = [&](int8_t* here, int8_t* next, int k0) {
      fetch(here, 1);
      multiply(0);
      // The other half of this stage is in registers, so the stage is free; the next has landed.
      __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
      __syncthreads();
      if (k0 + 2 * BK < a.K) stage(here, k0 + 2 * BK);
      __builtin_amdgcn_sched_barrier(0);
      fetch(next, 0);  // behind the last step: LDS bytes that nothing multiplies
      multiply(1);
    };
    stage(lds0, 0);
    if (BK < a.K) stage(lds1, BK);
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    __syncthreads();
    fetch(lds0, 0);
    for (int k0 = 0; k0 < a.K; k0 += 2 * BK) {
      step(lds0, lds1, k0);
      if (k0 + BK < a.K) step(lds1, lds0, k0 + BK);
    }
  };
  // Tiles of few rows (an expert's last, or all it has) multiply only the groups that hold some.
  const int live = (tl.rows + 16 * WM - 1) / (16 * WM);
  if (MT >= 4 && live <= MT / 4)
    product(std::integral_constant<int, (MT >= 4 ? MT / 4 : 1)>{});
  else if (MT >= 2 && live <= MT / 2)
    product(std::integral_constant<int, (MT >= 2 ? MT / 2 : 1)>{});
  else
    product(std::integral_constant<int, MT>{});
  // Epilogue: 16 rows at a time through the wave's share of LDS, from which a lane stores 16
  // consecutive bytes (whole lines for 64 channels of 16 bits). Stored from the accumulators, with the
  // scales loaded again between the stores, it took 30 us a tile of 256 x 256 instead of 6.
  constexpr int kOut = SILU ? NG / 2 : NG;
  constexpr int CH = kOut * 16, PITCH = CH * (int)sizeof(T) + 16;  // channels a wave, bytes a row
  static_assert(NT / 64 * 16 * PITCH <= (BM + BN) * BK, "the rows fit a stage");
  const int n_wave = n0 + wn * CH, lk4 = (lane >> 4) * 4;
  f32x4 sc[NG], bias[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const int i = wn * NG * 16 + g * 16 + lk4;
    sc[g] = *reinterpret_cast<const f32x4*>(s_col + i);
    if (!SILU && a.bias) bias[g] = *reinterpret_cast<const f32x4*>(s_bias + i);
  }
  __syncthreads();  // the stages have been read
  int8_t* mine = lds0 + wave * 16 * PITCH;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r0w = (m * WM + wm) * 16;
    if (r0w >= tl.rows) continue;
    const float rs = s_row[r0w + lr];
#pragma unroll
    for (int g = 0; g < kOut; ++g) {
      T v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f = ((float)acc[SILU ? 2 * g : g][m][i] * rs) * sc[SILU ? 2 * g : g][i];
        if constexpr (SILU)
          f = silu<DT>(f) * (((float)acc[2 * g + 1][m][i] * rs) * sc[2 * g + 1][i]);
        else if (a.bias)
          f += bias[g][i];
        v[i] = Elem<DT>::put(f);
      }
      __builtin_memcpy(__builtin_assume_aligned(mine + lr * PITCH + (g * 16 + lk4) * sizeof(T), 8), v,
                       sizeof(v));
    }
    // the lanes of this wave have written what its lanes read (one wave's LDS accesses are in order)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (vec) {
      constexpr int kVec = 16 / (int)sizeof(T), kPerRow = CH / kVec;  // lanes a row
#pragma unroll
      for (int q = 0; q < (16 * kPerRow + 63) / 64; ++q) {
        const int row = (q * 64 + lane) / kPerRow, c = (lane % kPerRow) * kVec;
        if (row < 16 && r0w + row < tl.rows && n_wave + c < a.N)
          *reinterpret_cast<u32x4*>(static_cast<T*>(a.out) + (int64_t)(tl.row0 + r0w + row) * a.N +
                                    n_wave + c) =
              *reinterpret_cast<const u32x4*>(mine + row * PITCH + c * sizeof(T));
      }
    } else {
      for (int row = 0; row < 16 && r0w + row < tl.rows; ++row)
#pragma unroll
        for (int c = lane; c < CH; c += 64) {
          const T d = *reinterpret_cast<const T*>(mine + row * PITCH + c * sizeof(T));
          if (n_wave + c < a.N)
            static_cast<T*>(a.out)[(int64_t)(tl.row0 + r0w + row) * a.N + n_wave + c] = d;
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

template <int BM, int BN, int WM, int WN, int DT, bool SILU>
hipError_t launch_tile(const Int8Args& a, int vec, hipStream_t s) {
  const int cols = SILU ? BN / 2 : BN;
  const int64_t blocks_n = (a.N + cols - 1) / cols;
  const int64_t blocks =
      a.tiles ? (a.m_tiles + 7) / 8 * 8 * blocks_n : (a.m_tiles * blocks_n + 7) / 8 * 8;
  if (blocks > kMaxBlocks / 2) return hipErrorInvalidValue;
  hipLaunchKernelGGL((int8_tile_kernel<BM, BN, WM, WN, DT, SILU>), dim3((unsigned)blocks),
                     dim3(64 * WM * WN), 0, s, a, vec);
  return hipGetLastError();
}

// ---------------------------------------------------------------- few tiles
// One matrix whose tiles do not fill the chip: a workgroup has its CU to itself and streams its
// weights at what it keeps in flight. BM rows x BN channels on WM x WN waves, both operands through LDS
// as in the tile kernel, in a ring of four stages of 128 bytes of K, three of them in flight. The
// steps are made a multiple of four (steps past K load zeros without a memory access), so that the
// ring's places are fixed arrays and the loads in flight always as many. Weights are not loaded
// straight into the registers the MFMA reads: 16 lanes then touch 16 lines, which passes 36 GB/s a
// CU (measured, L2-resident); rows of 128 bytes pass 100 GB/s.
constexpr int kRing = 4;

template <int BM, int BN, int WM, int WN, int DT>
__global__ __launch_bounds__(kThreads) void int8_ring_kernel(Int8Args a, int vec) {
  static_assert(WM * WN == kWaves, "four waves");
  using T = typename Elem<DT>::T;
  constexpr int BK = 128;
  constexpr int MT = BM / WM / 16, NG = BN / WN / 16;
  constexpr int LA = BM * 8 / kThreads, LB = BN * 8 / kThreads;  // 16-byte loads a thread and step
  constexpr int PITCH = BN * (int)sizeof(T) + 16, kRows = 16 * WM;
  constexpr int kStage = (BM + BN) * BK;
  // separate arrays: the compiler then knows which stage a load to LDS writes
  __shared__ __attribute__((aligned(16))) int8_t lds0[kStage];
  __shared__ __attribute__((aligned(16))) int8_t lds1[kStage];
  __shared__ __attribute__((aligned(16))) int8_t lds2[kStage];
  __shared__ __attribute__((aligned(16))) int8_t lds3[kStage];
  __shared__ __attribute__((aligned(16))) int8_t lds_out[kRows * PITCH];
  __shared__ float s_scale[BM];  // the rows' scales
  const int blocks_n = (a.N + BN - 1) / BN;
  const Tile tl{0, (int)blockIdx.x / blocks_n * BM, min(BM, a.M - (int)blockIdx.x / blocks_n * BM)};
  const int n0 = (int)blockIdx.x % blocks_n * BN;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int lr = lane & 15, lk4 = (lane >> 4) * 4;
  const __amdgpu_buffer_rsrc_t ra = buf_rsrc(a.a, a.a_bytes);
  const __amdgpu_buffer_rsrc_t rb = buf_rsrc(a.b0, (uint32_t)((int64_t)a.N * a.K));
  const uint32_t kc = (uint32_t)((tid & 7) ^ ((tid >> 3) & 7)) * 16;  // the chunk's byte of K
  uint32_t aoff[LA], boff[LB];
#pragma unroll
  for (int j = 0; j < LA; ++j) {
    const int r = (j * kThreads + tid) / 8;
    aoff[j] = r < tl.rows ? (uint32_t)(tl.row0 + r) * (uint32_t)a.K + kc : kOutOfRange;
  }
#pragma unroll
  for (int j = 0; j < LB; ++j) {
    const int i = (j * kThreads + tid) / 8;
    boff[j] = n0 + i < a.N ? (uint32_t)(n0 + i) * (uint32_t)a.K + kc : kOutOfRange;
  }
  auto stage = [&](int8_t* lds, int k0) {
    const uint32_t out = k0 + (int)kc < a.K ? 0u : kOutOfRange;  // zeros past K
    // The bounds check takes the scalar offset off the buffer's size, so it stays inside it: a step
    // past K of a small matrix could lie behind its end.
    const uint32_t soff = k0 < a.K ? (uint32_t)k0 : 0u;
#pragma unroll
    for (int j = 0; j < LB; ++j)
      buf_ld128_lds(rb, lds + BM * BK + (j * kThreads + wave * 64) * 16, boff[j] | out, soff);
#pragma unroll
    for (int j = 0; j < LA; ++j)
      buf_ld128_lds(ra, lds + (j * kThreads + wave * 64) * 16, aoff[j] | out, soff);
    __builtin_amdgcn_sched_barrier(0);
  };
  if (tid < BM)
    s_scale[tid] = tid < tl.rows ? a.a_scale[tl.row0 + tid] : 0.0f;
  const int sw0 = (((lane >> 4) ^ (lr & 7)) * 16), sw1 = ((4 + (lane >> 4)) ^ (lr & 7)) * 16;
  const int fa_at = (wm * 16 + lr) * BK, fb_at = (BM + wn * NG * 16 + lr) * BK;
  // The barrier without __syncthreads' release fence, which would wait for every load to LDS: this
  // wave's LDS accesses ahead of it are waited for, and the compiler keeps accesses on their sides.
  auto barrier = [] {
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  i32x4 acc[NG][MT], fa[2][MT], fb[2][NG];
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[g][m] = i32x4{0, 0, 0, 0};
  auto fetch = [&](const int8_t* lds, int half) {
    const int sw = half ? sw1 : sw0;
#pragma unroll
    for (int g = 0; g < NG; ++g)
      fb[half][g] = *reinterpret_cast<const i32x4*>(lds + fb_at + g * 16 * BK + sw);
#pragma unroll
    for (int m = 0; m < MT; ++m)
      fa[half][m] = *reinterpret_cast<const i32x4*>(lds + fa_at + m * WM * 16 * BK + sw);
  };
  auto multiply = [&](int half) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int g = 0; g < NG; ++g) acc[g][m] = mfma_i8(fb[half][g], fa[half][m], acc[g][m]);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto step = [&](int8_t* here, int8_t* next, int k0) {
    fetch(here, 1);
    multiply(0);
    // This wave's loads of the next stage have landed (the two stages after it stay in flight);
    // behind the barrier everybody's have, and this stage, all of it in registers, is free.
    __builtin_amdgcn_s_waitcnt(waitcnt_vm((kRing - 2) * (LA + LB)));
    barrier();
    stage(here, k0 + kRing * BK);
    fetch(next, 0);  // behind the last step: zeros that nothing multiplies
    multiply(1);
  };
  // the channels' scales and biases, asked for now: in the epilogue each would be waited for
  const int n_wave = wn * NG * 16 + lk4;  // in the tile
  float sc[NG][4];
  T bias[NG][4] = {};
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int i = 0; i < 4; ++i) sc[g][i] = a.s0[min(n0 + n_wave + g * 16 + i, a.N - 1)];
  if (a.bias) {
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        bias[g][i] = static_cast<const T*>(a.bias)[min(n0 + n_wave + g * 16 + i, a.N - 1)];
  }
  stage(lds0, 0);
  stage(lds1, BK);
  stage(lds2, 2 * BK);
  stage(lds3, 3 * BK);
  __builtin_amdgcn_s_waitcnt(waitcnt_vm((kRing - 1) * (LA + LB)));
  barrier();
  fetch(lds0, 0);
#pragma unroll 1
  for (int k0 = 0; k0 < a.K; k0 += kRing * BK) {
    step(lds0, lds1, k0);
    step(lds1, lds2, k0 + BK);
    step(lds2, lds3, k0 + 2 * BK);
    step(lds3, lds0, k0 + 3 * BK);
  }
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));  // no load to LDS may outlive the workgroup
  // Results 16 WM rows at a time through LDS, from which a thread stores 16 consecutive bytes.
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (m * kRows >= tl.rows) break;  // the same for the whole workgroup
    if (m > 0) __syncthreads();       // the rows before these have been read
    const float rs = s_scale[(m * WM + wm) * 16 + lr];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      T v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f = ((float)acc[g][m][i] * rs) * sc[g][i];
        if (a.bias) f += Elem<DT>::get(bias[g][i]);
        v[i] = Elem<DT>::put(f);
      }
      __builtin_memcpy(__builtin_assume_aligned(
                           lds_out + (wm * 16 + lr) * PITCH + (n_wave + g * 16) * sizeof(T), 8),
                       v, sizeof(v));
    }
    __syncthreads();
    const int64_t first = (int64_t)tl.row0 + m * kRows;
    const int rows = min(kRows, tl.rows - m * kRows);
    if (vec) {
      constexpr int kVec = 16 / (int)sizeof(T), kPerRow = BN / kVec;  // threads a row
#pragma unroll
      for (int q = 0; q < (kRows * kPerRow + kThreads - 1) / kThreads; ++q) {
        const int i = q * kThreads + tid, row = i / kPerRow, c = i % kPerRow * kVec;
        if (row < rows && n0 + c < a.N)
          *reinterpret_cast<u32x4*>(static_cast<T*>(a.out) + (first + row) * a.N + n0 + c) =
              *reinterpret_cast<const u32x4*>(lds_out + row * PITCH + c * sizeof(T));
      }
    } else {
#pragma unroll 1
      for (int i = tid; i < rows * BN; i += kThreads) {
        const int row = i / BN, c = i % BN;
        if (n0 + c < a.N)
          static_cast<T*>(a.out)[(first + row) * a.N + n0 + c] =
              *reinterpret_cast<const T*>(lds_out + row * PITCH + c * sizeof(T));
      }
    }
  }
}

template <int BM, int BN, int WM, int WN, int DT>
hipError_t launch_ring(const Int8Args& a, int vec, hipStream_t s) {
  const int64_t blocks = (int64_t)((a.N + BN - 1) / BN) * a.m_tiles;
  if (blocks > kMaxBlocks) return hipErrorInvalidValue;
  hipLaunchKernelGGL((int8_ring_kernel<BM, BN, WM, WN, DT>), dim3((unsigned)blocks),
                     dim3(kThreads), 0, s, a, vec);
  return hipGetLastError();
}

template <int DT, bool SILU>
hipError_t launch_product(const Int8Args& a, Int8Plan plan, hipStream_t s) {
  const int wide = a.N % (DT == kFp32 ? 4 : 8) == 0 && aligned16(a.out);
  if (plan.kind == kInt8Tile) {
    if (plan.bm == 256) return launch_tile<256, 256, 2, 4, DT, SILU>(a, wide, s);
    if (plan.bm == 128) return launch_tile<128, 128, 2, 2, DT, SILU>(a, wide, s);
    if (plan.bm == 32) return launch_tile<32, 64, 2, 2, DT, SILU>(a, wide, s);
    return launch_tile<64, 128, 2, 2, DT, SILU>(a, wide, s);
  }
  if constexpr (!SILU) {
    if (plan.kind == kInt8Ring)
      return plan.bn == 32   ? launch_ring<32, 32, 2, 2, DT>(a, wide, s)
             : plan.bm == 32 ? launch_ring<32, 64, 2, 2, DT>(a, wide, s)
                             : launch_ring<64, 64, 2, 2, DT>(a, wide, s);
    return launch_few_rows<DT, false>(a, nullptr, s);
  }
  return hipErrorInvalidValue;
}

template <int DT>
hipError_t launch_product_t(const Int8Args& a, Int8Plan plan, bool silu, hipStream_t s) {
  return silu ? launch_product<DT, true>(a, plan, s) : launch_product<DT, false>(a, plan, s);
}

}  // namespace

// Rows a tile by the rows an expert has on average (hidden 2048, intermediate 512, 256 experts, top-8,
// us a layer with tiles of 64 / 128 / 256 rows): 512 tokens 173 / 180 / 196, 2048 tokens 238 / 234 /
// 251, 4096 tokens 339 / 310 / 319, 8192 tokens 552 / 484 / 453. Where few experts share the rows the
// larger tiles also have to be enough for the chip: 8192 rows over 8 experts of 2048 x 1024 106 / 101 /
// 82 (256 tiles of 256 rows), 4096 rows over 16 of them 93 / 80 / 67 (128 tiles), over 8 of 2048 x 512
// 57 / 47 / 59 (64 tiles), 4000 rows over 8 of 512 x 128 24 / 27 / 35. Where experts have a few rows each
// tiles of 32 x 64 keep twice the workgroups of 64 x 128 on a CU, all of them streaming weights (us on
// the GPU, 32 x 64 / 64 x 128): 1 token 20.5 / 22.6, 16 tokens 45.0 / 47.6, 256 tokens 149 / 153, 512 tokens
// (16 rows an expert) 182 / 174. So do they where tiles are few at up to 32 rows (64 tokens, top-2 of 8
// experts of 1024 x 512 18.4 / 20.8; 50 tokens, top-4 of 16 of 512 x 256 15.9 / 17.1).
Int8Plan int8_experts_plan(int64_t slots, int E, int I) {
  const int64_t rows = (slots + E - 1) / E;
  if (rows <= 8 || (rows <= 32 && (int64_t)E * ((I + 63) / 64) < 256)) return Int8Plan{kInt8Tile, 32};
  if (rows >= 192 && slots / 256 * ((I + 127) / 128) >= 96) return Int8Plan{kInt8Tile, 256};
  if (rows > 48 && slots / 128 * ((I + 63) / 64) >= 256) return Int8Plan{kInt8Tile, 128};
  return Int8Plan{kInt8Tile, 64};
}

// One matrix: the larger the tile the fewer bytes a product moves, the smaller the more workgroups
// there are. By the number of 64 x 128 tiles (us, 4096 x 8192 channels, ring / 64 / 128 / 256 rows):
// 256 tiles 17 / 22 / 25 / 43, 512 30 / 25 / 28 / 45, 1024 55 / 48 / 38 / 48, 2048 107 / 81 / 70 / 57.
// In the ring by the number of 64 x 64 tiles (us with tiles of 32 x 32 / 32 x 64 / 64 x 64): 64 of 4096 x
// 1024 6.2 / 7.7 / 9.9, 128 of 1040 x 2001 4.9 / 5.5 / 7.1, 128 of 2048 x 4096 5.2 / 5.6 / 6.8, 256 of 2048
// x 4096 8.2 / 6.7 / 7.1, 448 of it 12.7 / 11.5 / 8.9.
Int8Plan int8_matrix_plan(int64_t M, int64_t N) {
  if (M <= 16) return Int8Plan{kInt8Stream, 16};
  const int64_t tiles = (M + 63) / 64 * ((N + 127) / 128), small = (M + 63) / 64 * ((N + 63) / 64);
  if (tiles <= 256) return Int8Plan{kInt8Ring, small <= 256 ? 32 : 64, small <= 128 ? 32 : 64};
  return Int8Plan{kInt8Tile, tiles <= 768 ? 64 : tiles <= 1408 ? 128 : 256};
}

hipError_t launch_int8_product(const Int8Args& a, Int8Plan plan, bool silu, int dtype,
                               hipStream_t s) {
  if (a.m_tiles <= 0) return hipSuccess;
  if (dtype == kBf16) return launch_product_t<kBf16>(a, plan, silu, s);
  if (dtype == kFp16) return launch_product_t<kFp16>(a, plan, silu, s);
  return launch_product_t<kFp32>(a, plan, silu, s);
}

bool int8_fused_fits(int M, int K) {
  return M >= 1 && M <= kFusedRows && (int64_t)M * (K + 16) <= kFusedBytes;
}

hipError_t launch_int8_fused(const Int8Args& a, const void* x, int dtype, hipStream_t s) {
  if (dtype == kBf16) return launch_few_rows<kBf16, true>(a, x, s);
  if (dtype == kFp16) return launch_few_rows<kFp16, true>(a, x, s);
  return launch_few_rows<kFp32, true>(a, x, s);
}
