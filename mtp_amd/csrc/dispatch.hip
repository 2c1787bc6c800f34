// Token rows sorted by expert and back, with the routed weights applied, and the gradients.
//
// Slot f = t * k + i of token t has key(f) = ids[f] if 0 <= ids[f] < E, else E (dropped). Rows are
// ordered by (key, f): a stable sort, so dropped slots lie behind the last expert's rows.
//   dispatch   rows[r] = x[t(r)] for kept slots, zeros for dropped ones
//   combine    out[t]  = sum_i w[t, i] rows[row(t, i)] over the kept slots, in slot order, in fp32
//   gradients  d rows[row(f)] = w[f] d out[t] (zeros for dropped slots)
//              d w[f] = <d out[t], rows[row(f)]>, and dispatch's own is combine with weights of 1
// Every row belongs to exactly one slot, so every row has one writer: no atomics, and nothing is
// left unwritten. A dropped slot's row travels as its bitwise complement, so the sign says that
// it is dropped.
//
// All of it moves T (k + 1) rows and computes next to nothing: bound by HBM, at few tokens by the
// launches and the latency of ids -> rank -> copy.
#include <algorithm>

#include "access.h"
#include "common.h"
#include "elem.h"
#include "int8.h"
#include "launch.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxK = 64;
constexpr int kMaxE = 512;

MOE_DEV int key_of(int id, int E) { return (unsigned)id < (unsigned)E ? id : E; }

// Orders as (key, slot) does: keys up to 512, slots below 2^22.
MOE_DEV uint32_t pair_of(int key, int slot) { return ((uint32_t)key << 22) | (uint32_t)slot; }

struct SortOut {
  int32_t* offsets;   // [E + 1]
  int32_t* row_slot;  // [T * k]
  int32_t* slot_row;  // [T * k]
};

// ---------------------------------------------------------------- tables of the experts
// offsets and the GEMM tiles from the keys' counts in LDS (cnt [E], E <= kMaxE), by one workgroup
// of NT threads. tiles (nullable): {expert, first row, rows, 0} of each block of bm rows, behind
// them entries of no rows up to tile_cap.
template <int NT>
MOE_DEV void write_tables(const int* cnt, int E, int32_t* offsets, i32x4* tiles, int bm,
                          int tile_cap) {
  constexpr int kPer = (kMaxE + NT - 1) / NT;  // experts a thread
  __shared__ int s_wave[2][NT / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int rows = 0, blocks = 0;
  int c[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = tid * kPer + j;
    c[j] = e < E ? cnt[e] : 0;
    rows += c[j];
    if (tiles) blocks += (c[j] + bm - 1) / bm;
  }
  int r = rows, b = blocks;  // inclusive scans over the wave
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int pr = __shfl_up(r, d), pb = __shfl_up(b, d);
    if (lane >= d) {
      r += pr;
      b += pb;
    }
  }
  if (lane == 63) {
    s_wave[0][wave] = r;
    s_wave[1][wave] = b;
  }
  __syncthreads();
  int row = r - rows, blk = b - blocks, all = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wave) {
      row += s_wave[0][w];
      blk += s_wave[1][w];
    }
    all += s_wave[1][w];
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = tid * kPer + j;
    if (e <= E) offsets[e] = row;
    if (tiles && e < E)
      for (int o = 0; o < c[j]; o += bm, ++blk)
        if (blk < tile_cap) tiles[blk] = i32x4{e, row + o, min(bm, c[j] - o), 0};
    row += c[j];
  }
  if (tid * kPer + kPer == E && E == NT * kPer) offsets[E] = row;  // E fills the last thread
  if (tiles)
    for (int i = all + tid; i < tile_cap; i += NT) tiles[i] = i32x4{0, 0, 0, 0};
}

// ---------------------------------------------------------------- few slots: one launch
// Workgroup (t, y): every thread compares its share of all (key, slot) pairs with the token's k; the
// ballots' population counts are the rows. S ids per workgroup from L2 instead of two further
// launches. Workgroup (T, 0) counts the experts' slots for the tables.
template <typename U>
MOE_DEV void dispatch_small(int bx, int by, const int32_t* __restrict__ ids, int T, int k, int E,
                            const U* __restrict__ x, int64_t units, U* __restrict__ rows, SortOut o,
                            i32x4* tiles, int bm, int tile_cap) {
  __shared__ int s_cnt[kThreads / 64][kMaxK];
  __shared__ int s_row[kMaxK];
  __shared__ int s_hist[kMaxE + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int S = T * k;
  if (bx == T) {
    if (by != 0) return;
    for (int e = tid; e <= E; e += kThreads) s_hist[e] = 0;
    __syncthreads();
    for (int s = tid; s < S; s += kThreads) atomicAdd(&s_hist[key_of(ids[s], E)], 1);
    __syncthreads();
    write_tables<kThreads>(s_hist, E, o.offsets, tiles, bm, tile_cap);
    return;
  }
  const int t = bx;
  for (int i0 = 0; i0 < k; i0 += 8) {
    uint32_t mine[8];
    int cnt[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int f = t * k + i0 + j;
      mine[j] = i0 + j < k ? pair_of(key_of(ids[f], E), f) : 0u;
      cnt[j] = 0;
    }
#pragma unroll 2
    for (int s0 = wave * 64; s0 < S; s0 += kThreads) {
      const int s = s0 + lane;
      const uint32_t pair = s < S ? pair_of(key_of(ids[s], E), s) : ~0u;
#pragma unroll
      for (int j = 0; j < 8; ++j) cnt[j] += __popcll(__ballot(pair < mine[j]));
    }
    if (lane == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i0 + j < k) s_cnt[wave][i0 + j] = cnt[j];
    }
  }
  __syncthreads();
  if (tid < k) {
    const int f = t * k + tid;
    int r = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) r += s_cnt[w][tid];
    const int v = key_of(ids[f], E) < E ? r : ~r;
    s_row[tid] = v;
    if (by == 0) {
      o.slot_row[f] = v;
      o.row_slot[r] = f;
    }
  }
  if (!x) return;
  __syncthreads();
  const int64_t c = (int64_t)by * kThreads + tid;
  if (c >= units) return;
  const U v = x[(int64_t)t * units + c];
  for (int i = 0; i < k; ++i) {
    const int r = s_row[i];
    rows[(int64_t)(r < 0 ? ~r : r) * units + c] = r < 0 ? U{} : v;
  }
}

template <typename U>
__global__ __launch_bounds__(kThreads) void dispatch_small_kernel(
    const int32_t* __restrict__ ids, int T, int k, int E, const U* __restrict__ x, int64_t units,
    U* __restrict__ rows, SortOut o, i32x4* tiles, int bm, int tile_cap) {
  dispatch_small<U>(blockIdx.x, blockIdx.y, ids, T, k, E, x, units, rows, o, tiles, bm, tile_cap);
}

// ---------------------------------------------------------------- many slots: count, scan, copy
constexpr int kCountWaves = kThreads / 64;
constexpr int kPerLane = 4;
constexpr int kChunk = kThreads * kPerLane;  // slots a workgroup

// rank[s] = how many slots of the chunk ahead of s have its key; hist[chunk][e] = the keys' counts.
// A wave ranks 64 slots at a time: lanes of equal keys find each other by ballots over the key's
// bits, the first of them moves the wave's running count.
MOE_DEV void dispatch_count(int block, const int32_t* __restrict__ ids, int S, int E,
                            uint16_t* __restrict__ rank, int32_t* __restrict__ hist) {
  __shared__ int s_cnt[kCountWaves][kMaxE + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < kCountWaves * (kMaxE + 1); i += kThreads) (&s_cnt[0][0])[i] = 0;
  const int first = block * kChunk + wave * 64 * kPerLane;
  int key[kPerLane], local[kPerLane];
#pragma unroll
  for (int j = 0; j < kPerLane; ++j) {
    const int s = first + 64 * j + lane;
    key[j] = s < S ? key_of(ids[s], E) : -1;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPerLane; ++j) {
    const bool in = key[j] >= 0;
    uint64_t same = __ballot(in);
#pragma unroll
    for (int b = 0; b < 10; ++b) {  // keys below 1024
      const bool bit = (key[j] >> b) & 1;
      const uint64_t set = __ballot(bit);
      same &= bit ? set : ~set;
    }
    const int ahead = __popcll(same & ((1ull << lane) - 1));
    // One wave's LDS accesses complete in order; volatile keeps the compiler to that order.
    volatile int* cnt = s_cnt[wave];
    const int before = in ? cnt[key[j]] : 0;
    if (in && ahead == 0) cnt[key[j]] = before + __popcll(same);
    local[j] = before + ahead;
  }
  __syncthreads();
  for (int e = tid; e <= E; e += kThreads) {
    int run = 0;
#pragma unroll
    for (int w = 0; w < kCountWaves; ++w) {
      const int n = s_cnt[w][e];
      s_cnt[w][e] = run;
      run += n;
    }
    hist[(int64_t)block * (E + 1) + e] = run;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPerLane; ++j)
    if (key[j] >= 0)
      rank[first + 64 * j + lane] = (uint16_t)(s_cnt[wave][key[j]] + local[j]);
}

__global__ __launch_bounds__(kThreads) void dispatch_count_kernel(
    const int32_t* __restrict__ ids, int S, int E, uint16_t* __restrict__ rank,
    int32_t* __restrict__ hist) {
  dispatch_count(blockIdx.x, ids, S, E, rank, hist);
}

constexpr int kScanThreads = 1024;

// hist[c][e] becomes the slots of key e in the chunks ahead of c; the tables from the totals.
__global__ __launch_bounds__(kScanThreads) void dispatch_scan_kernel(
    int32_t* __restrict__ hist, int chunks, int E, int32_t* offsets, i32x4* tiles, int bm,
    int tile_cap) {
  __shared__ int s_hist[kMaxE + 1];
  const int e = threadIdx.x;
  if (e <= E) {
    int run = 0;
    for (int c0 = 0; c0 < chunks; c0 += 8) {
      int v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = c0 + j < chunks ? hist[(int64_t)(c0 + j) * (E + 1) + e] : 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (c0 + j < chunks) hist[(int64_t)(c0 + j) * (E + 1) + e] = run;
        run += v[j];
      }
    }
    s_hist[e] = run;
  }
  __syncthreads();
  write_tables<kScanThreads>(s_hist, E, offsets, tiles, bm, tile_cap);
}

// Rows from the ranks, and the copy: tpt threads a token (a power of two from 32 to 256).
template <typename U>
__global__ __launch_bounds__(kThreads) void dispatch_copy_kernel(
    const int32_t* __restrict__ ids, int T, int k, int E, const U* __restrict__ x, int64_t units,
    U* __restrict__ rows, SortOut o, const uint16_t* __restrict__ rank,
    const int32_t* __restrict__ hist, int tpt_log) {
  __shared__ int s_row[(kThreads / 32) * kMaxK];
  const int tid = threadIdx.x, tpt = 1 << tpt_log, per = kThreads >> tpt_log;
  const int64_t t0 = (int64_t)blockIdx.x * per;
  const int S = T * k;
  for (int i = tid; i < per * k; i += kThreads) {
    const int64_t f = t0 * k + i;
    if (f < S) {
      const int key = key_of(ids[f], E);
      const int r = o.offsets[key] + hist[(f / kChunk) * (E + 1) + key] + rank[f];
      const int v = key < E ? r : ~r;
      s_row[i] = v;
      if (blockIdx.y == 0) {
        o.slot_row[f] = v;
        o.row_slot[r] = (int)f;
      }
    }
  }
  if (!x) return;
  __syncthreads();
  const int64_t t = t0 + (tid >> tpt_log);
  const int64_t c = (int64_t)blockIdx.y * tpt + (tid & (tpt - 1));
  if (t >= T || c >= units) return;
  const U v = x[t * units + c];
  const int* mine = s_row + (tid >> tpt_log) * k;
  for (int i = 0; i < k; ++i) {
    const int r = mine[i];
    rows[(int64_t)(r < 0 ? ~r : r) * units + c] = r < 0 ? U{} : v;
  }
}

// The workspace of many slots: the chunks' counts and the slots' ranks in their chunks.
struct LargeSort {
  int chunks;
  int32_t* hist;
  uint16_t* rank;
  LargeSort(int S, int E, void* ws)
      : chunks((S + kChunk - 1) / kChunk),
        hist(static_cast<int32_t*>(ws)),
        rank(reinterpret_cast<uint16_t*>(hist + (int64_t)chunks * (E + 1))) {}
};

// The scan and the copy behind the chunks' counts.
template <typename U>
hipError_t launch_ranked(const LargeSort& w, const int32_t* ids, int T, int k, int E, const U* x,
                         int64_t units, U* rows, const SortOut& o, i32x4* tiles, int bm,
                         int tile_cap, hipStream_t s) {
  hipLaunchKernelGGL(dispatch_scan_kernel, dim3(1), dim3(kScanThreads), 0, s, w.hist, w.chunks, E,
                     o.offsets, tiles, bm, tile_cap);
  int tpt_log = 5;
  while (tpt_log < 8 && (int64_t(1) << tpt_log) < units) ++tpt_log;
  const int per = kThreads >> tpt_log;
  const unsigned gy = x ? (unsigned)((units + (1 << tpt_log) - 1) >> tpt_log) : 1u;
  hipLaunchKernelGGL(dispatch_copy_kernel<U>, dim3((T + per - 1) / per, gy), dim3(kThreads), 0, s,
                     ids, T, k, E, x, units, rows, o, w.rank, w.hist, tpt_log);
  return hipGetLastError();
}

// Slots up to which every workgroup ranks its token's slots itself.
constexpr int kSmallSlots = 4096;

template <typename U>
hipError_t launch_dispatch_units(const int32_t* ids, int T, int k, int E, const void* x,
                                 int64_t units, void* rows, const SortOut& o, void* ws,
                                 i32x4* tiles, int bm, int tile_cap, hipStream_t s) {
  const int S = T * k;
  const U* xu = static_cast<const U*>(x);
  U* ru = static_cast<U*>(rows);
  if (S <= kSmallSlots) {
    const unsigned gy = x ? (unsigned)((units + kThreads - 1) / kThreads) : 1u;
    hipLaunchKernelGGL(dispatch_small_kernel<U>, dim3(T + 1, gy), dim3(kThreads), 0, s, ids, T, k,
                       E, xu, units, ru, o, tiles, bm, tile_cap);
    return hipGetLastError();
  }
  const LargeSort w(S, E, ws);
  hipLaunchKernelGGL(dispatch_count_kernel, dim3(w.chunks), dim3(kThreads), 0, s, ids, S, E, w.rank,
                     w.hist);
  return launch_ranked<U>(w, ids, T, k, E, xu, units, ru, o, tiles, bm, tile_cap, s);
}

// ---------------------------------------------------------------- the experts' first launch
// Workgroups [0, qblocks) quantise four rows each, the others sort (SMALL: the whole sort, else the
// chunks' counts): neither waits for the other, and one launch less. 16 tokens of 2048 over 256
// experts 60.9 -> 55.9 us a call, 4096 tokens 312 -> 309 us. Only where a wave holds a row: a
// workgroup of 1024 threads a row has no use for the sort's 256.
template <int DT, int NC, bool VEC, bool SMALL>
__global__ __launch_bounds__(kThreads) void quantize_and_sort_kernel(
    const typename Elem<DT>::T* __restrict__ x, int T, int K, int8_t* __restrict__ q,
    float* __restrict__ scale, int qblocks, const int32_t* __restrict__ ids, int k, int E, SortOut o,
    uint16_t* __restrict__ rank, int32_t* __restrict__ hist, i32x4* tiles, int bm, int tile_cap) {
  if ((int)blockIdx.x < qblocks)
    quantize_rows<DT, 64, NC, VEC>(blockIdx.x, x, T, K, q, scale);
  else if constexpr (SMALL)
    dispatch_small<u32x4>(blockIdx.x - qblocks, 0, ids, T, k, E, nullptr, 0, nullptr, o, tiles, bm,
                          tile_cap);
  else
    dispatch_count(blockIdx.x - qblocks, ids, T * k, E, rank, hist);
}

template <int DT, int NC>
hipError_t launch_quantize_and_sort_t(const void* x, int T, int K, int8_t* q, float* scale,
                                      const int32_t* ids, int k, int E, const SortOut& o, void* ws,
                                      i32x4* tiles, int bm, int tile_cap, hipStream_t s) {
  const int S = T * k, qblocks = (T + 3) / 4;
  const bool vec = K % 8 == 0 && aligned16(x) && (reinterpret_cast<uintptr_t>(q) & 7u) == 0;
  const auto* xt = static_cast<const typename Elem<DT>::T*>(x);
  const bool small = S <= kSmallSlots;
  const LargeSort w(S, E, ws);
  const dim3 grid((unsigned)(qblocks + (small ? T + 1 : w.chunks)));
#define MOE_QUANT_SORT(V, SM)                                                                    \
  hipLaunchKernelGGL((quantize_and_sort_kernel<DT, NC, V, SM>), grid, dim3(kThreads), 0, s, xt, T, \
                     K, q, scale, qblocks, ids, k, E, o, w.rank, w.hist, tiles, bm, tile_cap)
  if (small) {
    if (vec) MOE_QUANT_SORT(true, true);
    else MOE_QUANT_SORT(false, true);
    return hipGetLastError();
  }
  if (vec) MOE_QUANT_SORT(true, false);
  else MOE_QUANT_SORT(false, false);
#undef MOE_QUANT_SORT
  return launch_ranked<u32x4>(w, ids, T, k, E, nullptr, 1, nullptr, o, tiles, bm, tile_cap, s);
}

// ---------------------------------------------------------------- combine
// NT threads a token (a wave, or the workgroup) and 8 NT of its columns. Slots are taken 8 at a time,
// all their loads in flight together; a dropped slot (and a slot_row entry outside the rows) reads
// row 0 and does not count, so that nothing a dropped row holds reaches the sum.
template <int DT, int NT, bool VEC, bool WEIGHTED>
__global__ __launch_bounds__(kThreads) void combine_kernel(
    const typename Elem<DT>::T* __restrict__ rows, int T, int k, int H,
    const int32_t* __restrict__ slot_row, const float* __restrict__ w,
    typename Elem<DT>::T* __restrict__ out) {
  using C = Cols<DT, NT, VEC>;
  const int tid = threadIdx.x % NT, c = blockIdx.y * 8 * NT;
  const int64_t t = (int64_t)blockIdx.x * (kThreads / NT) +
                    __builtin_amdgcn_readfirstlane((int)threadIdx.x / NT);
  if (t >= T) return;
  const int S = T * k;
  float s[8] = {};
  for (int i0 = 0; i0 < k; i0 += 8) {
    float wt[8], v[8][8];
    bool ok[8];
    int row[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool in = i0 + i < k;
      const int64_t f = t * k + (in ? i0 + i : 0);
      const int r = slot_row[f];
      ok[i] = in && (unsigned)r < (unsigned)S;
      row[i] = ok[i] ? r : 0;
      wt[i] = WEIGHTED ? w[f] : 1.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) C::load(rows + (int64_t)row[i] * H + c, tid, H - c, v[i]);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        s[j] = ok[i] ? __builtin_fmaf(wt[i], v[i][j], s[j]) : s[j];
  }
  C::store(out + t * H + c, tid, H - c, s);
}

// NT threads a token (a wave, or the workgroup). d rows from the token's d out, and the slots' dot
// products: per thread over its columns, a butterfly in each wave, the waves in order.
template <int DT, int NT, bool VEC>
__global__ __launch_bounds__(kThreads) void combine_backward_kernel(
    const typename Elem<DT>::T* __restrict__ dout, const typename Elem<DT>::T* __restrict__ rows,
    int T, int k, int H, const int32_t* __restrict__ slot_row, const float* __restrict__ w,
    typename Elem<DT>::T* __restrict__ drows, float* __restrict__ dw) {
  using C = Cols<DT, NT, VEC>;
  constexpr int kPer = kThreads / NT;  // tokens a workgroup
  __shared__ float s_part[kThreads / 64][8];
  const int tid = threadIdx.x % NT, lane = threadIdx.x & 63;
  const int64_t t =
      (int64_t)blockIdx.x * kPer + __builtin_amdgcn_readfirstlane((int)threadIdx.x / NT);
  if (t >= T) return;  // NT < kThreads: no barrier below; else the grid has T workgroups
  const int S = T * k;
  for (int i0 = 0; i0 < k; i0 += 8) {
    int row[8];
    float wt[8], part[8];
    bool own[8], kept[8];  // the slot names a row; and is not dropped
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool in = i0 + i < k;
      const int64_t f = t * k + (in ? i0 + i : 0);
      const int r = slot_row[f];
      kept[i] = in && r >= 0 && r < S;
      own[i] = in && (r < 0 ? ~r : r) < S;
      row[i] = own[i] ? (r < 0 ? ~r : r) : 0;
      wt[i] = w[f];
      part[i] = 0.0f;
    }
    for (int c = 0; c < H; c += 8 * NT) {
      float g[8];
      C::load(dout + t * H + c, tid, H - c, g);
      if (dw) {
        float y[8][8];
#pragma unroll
        for (int i = 0; i < 8; ++i) C::load(rows + (int64_t)row[i] * H + c, tid, H - c, y[i]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) part[i] = __builtin_fmaf(g[e], y[i][e], part[i]);
      }
      if (drows) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (!own[i]) continue;
          float d[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] = kept[i] ? wt[i] * g[e] : 0.0f;
          C::store(drows + (int64_t)row[i] * H + c, tid, H - c, d);
        }
      }
    }
    if (dw) {
      float mine = 0.0f;  // lane i's: slot i0 + i
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = bfly_sum(part[i]);
        if (lane == i) mine = kept[i] ? p : 0.0f;
      }
      if constexpr (NT > 64) {
        if (i0 > 0) __syncthreads();
        if (lane < 8) s_part[threadIdx.x >> 6][lane] = mine;
        __syncthreads();
        mine = 0.0f;
        if (tid < 8) {
#pragma unroll
          for (int q = 0; q < NT / 64; ++q) mine += s_part[q][tid];
        }
      }
      if (tid < 8 && i0 + tid < k) dw[t * k + i0 + tid] = mine;
    }
  }
}

template <int DT>
hipError_t launch_combine_t(const void* rows, int T, int k, int H, const int32_t* slot_row,
                            const float* w, void* out, hipStream_t s) {
  using E = typename Elem<DT>::T;
  const E* r = static_cast<const E*>(rows);
  E* o = static_cast<E*>(out);
  const bool vec = H % 8 == 0 && aligned16(rows) && aligned16(out);
#define MOE_COMBINE(NT, V, W)                                                                   \
  hipLaunchKernelGGL((combine_kernel<DT, NT, V, W>),                                            \
                     dim3((unsigned)((T + kThreads / NT - 1) / (kThreads / NT)),                \
                          (unsigned)((H + 8 * NT - 1) / (8 * NT))),                             \
                     dim3(kThreads), 0, s, r, T, k, H, slot_row, w, o)
#define MOE_COMBINE_W(NT, V)        \
  do {                              \
    if (w) MOE_COMBINE(NT, V, true); \
    else MOE_COMBINE(NT, V, false); \
  } while (0)
  if (H <= 1024) {
    if (vec) MOE_COMBINE_W(64, true);
    else MOE_COMBINE_W(64, false);
  } else {
    if (vec) MOE_COMBINE_W(256, true);
    else MOE_COMBINE_W(256, false);
  }
#undef MOE_COMBINE_W
#undef MOE_COMBINE
  return hipGetLastError();
}

template <int DT>
hipError_t launch_combine_backward_t(const void* dout, const void* rows, int T, int k, int H,
                                     const int32_t* slot_row, const float* w, void* drows,
                                     float* dw, hipStream_t s) {
  using E = typename Elem<DT>::T;
  const bool vec = H % 8 == 0 && aligned16(dout) && aligned16(rows) && aligned16(drows);
#define MOE_COMBINE_BWD(NT, V)                                                                   \
  hipLaunchKernelGGL((combine_backward_kernel<DT, NT, V>),                                       \
                     dim3((unsigned)((T + kThreads / NT - 1) / (kThreads / NT))), dim3(kThreads), 0, \
                     s, static_cast<const E*>(dout), static_cast<const E*>(rows), T, k, H,       \
                     slot_row, w, static_cast<E*>(drows), dw)
  if (H <= 1024) {
    if (vec) MOE_COMBINE_BWD(64, true);
    else MOE_COMBINE_BWD(64, false);
  } else {
    if (vec) MOE_COMBINE_BWD(256, true);
    else MOE_COMBINE_BWD(256, false);
  }
#undef MOE_COMBINE_BWD
  return hipGetLastError();
}

int check_slots(const char* what, int32_t T, int32_t top_k) {
  if (T < 0 || top_k < 1 || top_k > kMaxK)
    return op_fail(MOE_ERR_SHAPE, "%s: T=%d top_k=%d (T >= 0, top_k in [1, 64])", what, T, top_k);
  if ((int64_t)T * top_k > (1 << 22))
    return op_fail(MOE_ERR_SHAPE, "%s: %lld slots exceed 2^22", what, (long long)T * top_k);
  return MOE_OK;
}

int check_rows(const char* what, int32_t hidden, int32_t dtype) {
  if (dtype < kBf16 || dtype > kFp32)
    return op_fail(MOE_ERR_UNSUPPORTED, "%s: dtype=%d (0 bf16, 1 fp16, 2 fp32)", what, dtype);
  if (hidden < 1 || hidden > (1 << 16))
    return op_fail(MOE_ERR_SHAPE, "%s: hidden=%d outside [1, 65536]", what, hidden);
  return MOE_OK;
}

}  // namespace

int64_t dispatch_scratch_bytes(int64_t slots, int E) {
  if (slots <= kSmallSlots) return 0;
  const int64_t chunks = (slots + kChunk - 1) / kChunk;
  return chunks * (E + 1) * 4 + chunks * kChunk * 2;
}

hipError_t launch_dispatch(const int32_t* ids, int T, int k, int E, const void* x,
                           int64_t row_bytes, void* rows, int32_t* offsets, int32_t* row_slot,
                           int32_t* slot_row, void* ws, i32x4* tiles, int bm, int tile_cap,
                           hipStream_t s) {
  const SortOut o{offsets, row_slot, slot_row};
  const int width = copy_access_bytes(row_bytes, x, rows);
  if (width == 16)
    return launch_dispatch_units<u32x4>(ids, T, k, E, x, row_bytes / 16, rows, o, ws, tiles, bm,
                                        tile_cap, s);
  if (width == 4)
    return launch_dispatch_units<uint32_t>(ids, T, k, E, x, row_bytes / 4, rows, o, ws, tiles, bm,
                                           tile_cap, s);
  return launch_dispatch_units<uint16_t>(ids, T, k, E, x, row_bytes / 2, rows, o, ws, tiles, bm,
                                         tile_cap, s);
}

hipError_t launch_quantize_and_sort(const void* x, int T, int K, int dtype, int8_t* q, float* scale,
                                    const int32_t* ids, int k, int E, int32_t* offsets,
                                    int32_t* row_slot, int32_t* slot_row, void* ws, i32x4* tiles,
                                    int bm, int tile_cap, hipStream_t s) {
  const SortOut o{offsets, row_slot, slot_row};
  if (K > 2048) {
    const hipError_t e = launch_quantize(x, T, K, dtype, q, scale, s);
    if (e != hipSuccess) return e;
    return launch_dispatch(ids, T, k, E, nullptr, 16, nullptr, offsets, row_slot, slot_row, ws, tiles,
                           bm, tile_cap, s);
  }
#define MOE_QUANT_SORT_DT(DT)                                                                     \
  (K <= 512    ? launch_quantize_and_sort_t<DT, 1>(x, T, K, q, scale, ids, k, E, o, ws, tiles, bm, \
                                                   tile_cap, s)                                   \
   : K <= 1024 ? launch_quantize_and_sort_t<DT, 2>(x, T, K, q, scale, ids, k, E, o, ws, tiles, bm, \
                                                   tile_cap, s)                                   \
               : launch_quantize_and_sort_t<DT, 4>(x, T, K, q, scale, ids, k, E, o, ws, tiles, bm, \
                                                   tile_cap, s))
  if (dtype == kBf16) return MOE_QUANT_SORT_DT(kBf16);
  if (dtype == kFp16) return MOE_QUANT_SORT_DT(kFp16);
  return MOE_QUANT_SORT_DT(kFp32);
#undef MOE_QUANT_SORT_DT
}

hipError_t launch_combine(const void* rows, int T, int k, int H, int dtype,
                          const int32_t* slot_row, const float* w, void* out, hipStream_t s) {
  if (dtype == kBf16) return launch_combine_t<kBf16>(rows, T, k, H, slot_row, w, out, s);
  if (dtype == kFp16) return launch_combine_t<kFp16>(rows, T, k, H, slot_row, w, out, s);
  return launch_combine_t<kFp32>(rows, T, k, H, slot_row, w, out, s);
}

extern "C" {

int64_t moe_dispatch_workspace_bytes_v1(int32_t T, int32_t top_k, int32_t num_experts) {
  if (T < 0 || top_k < 1 || num_experts < 1) return -1;
  return dispatch_scratch_bytes((int64_t)T * top_k, num_experts);
}

int moe_dispatch_v1(const void* x, int32_t T, int32_t hidden, int32_t dtype,
                    const int32_t* topk_ids, int32_t top_k, int32_t num_experts, void* workspace,
                    int64_t workspace_bytes, void* rows, int32_t* offsets, int32_t* row_slot,
                    int32_t* slot_row, void* stream) {
  int rc = check_slots("dispatch", T, top_k);
  if (!rc) rc = check_rows("dispatch", hidden, dtype);
  if (rc) return rc;
  if (num_experts < 1 || num_experts > kMaxE)
    return op_fail(MOE_ERR_SHAPE, "dispatch: num_experts=%d outside [1, 512]", num_experts);
  if (!offsets || (T > 0 && (!x || !topk_ids || !rows || !row_slot || !slot_row)))
    return op_fail(MOE_ERR_NULL, "dispatch: NULL pointer");
  const int64_t need = dispatch_scratch_bytes((int64_t)T * top_k, num_experts);
  if (need > 0) {
    if (!workspace || workspace_bytes < need)
      return op_fail(MOE_ERR_WORKSPACE, "dispatch: workspace of %lld bytes, needs %lld",
                     (long long)(workspace ? workspace_bytes : 0), (long long)need);
    if (!workspace_aligned(workspace))
      return op_fail(MOE_ERR_WORKSPACE, "dispatch: workspace must be 256-byte aligned");
  }
  const int64_t row_bytes = (int64_t)hidden * dtype_bytes(dtype);
  const int64_t S = (int64_t)T * top_k, nr = S * row_bytes;
  const struct {
    const void* p;
    int64_t bytes;
  } outs[] = {{rows, nr}, {offsets, (num_experts + 1) * (int64_t)4}, {row_slot, S * 4},
              {slot_row, S * 4}, {workspace, need}};
  for (const auto& o : outs) {
    if (overlaps(o.p, o.bytes, x, T * row_bytes) || overlaps(o.p, o.bytes, topk_ids, S * 4))
      return op_fail(MOE_ERR_SHAPE, "dispatch: outputs and workspace must not overlap x or the ids");
    for (const auto* i = outs; i != &o; ++i)
      if (overlaps(o.p, o.bytes, i->p, i->bytes))
        return op_fail(MOE_ERR_SHAPE, "dispatch: outputs and workspace must not overlap each other");
  }
  MOE_OP_HIP(launch_dispatch(topk_ids, T, top_k, num_experts, T ? x : nullptr, row_bytes, rows,
                             offsets, row_slot, slot_row, workspace, nullptr, 1, 0,
                             (hipStream_t)stream),
             "dispatch");
  return MOE_OK;
}

int moe_combine_v1(const void* rows, int32_t T, int32_t top_k, int32_t hidden, int32_t dtype,
                   const int32_t* slot_row, const float* topk_weights, void* out, void* stream) {
  int rc = check_slots("combine", T, top_k);
  if (!rc) rc = check_rows("combine", hidden, dtype);
  if (rc) return rc;
  if (T == 0) return MOE_OK;
  if (!rows || !slot_row || !out) return op_fail(MOE_ERR_NULL, "combine: NULL pointer");
  const int64_t row_bytes = (int64_t)hidden * dtype_bytes(dtype);
  const int64_t S = (int64_t)T * top_k;
  if (overlaps(rows, S * row_bytes, out, T * row_bytes) ||
      overlaps(slot_row, S * 4, out, T * row_bytes) ||
      overlaps(topk_weights, S * 4, out, T * row_bytes))
    return op_fail(MOE_ERR_SHAPE, "combine: out must not overlap the inputs");
  MOE_OP_HIP(launch_combine(rows, T, top_k, hidden, dtype, slot_row, topk_weights, out,
                            (hipStream_t)stream),
             "combine");
  return MOE_OK;
}

int moe_combine_backward_v1(const void* dout, const void* rows, int32_t T, int32_t top_k,
                            int32_t hidden, int32_t dtype, const int32_t* slot_row,
                            const float* topk_weights, void* drows, float* dweights,
                            void* stream) {
  int rc = check_slots("combine backward", T, top_k);
  if (!rc) rc = check_rows("combine backward", hidden, dtype);
  if (rc) return rc;
  if (T == 0) return MOE_OK;
  if (!dout || !slot_row || !topk_weights || (!drows && !dweights) || (dweights && !rows))
    return op_fail(MOE_ERR_NULL, "combine backward: NULL pointer");
  const int64_t row_bytes = (int64_t)hidden * dtype_bytes(dtype), n = T * (int64_t)top_k;
  const struct {
    const void* p;
    int64_t bytes;
  } outs[] = {{drows, n * row_bytes}, {dweights, n * 4}};
  for (const auto& o : outs)
    if (overlaps(o.p, o.bytes, rows, n * row_bytes) || overlaps(o.p, o.bytes, dout, T * row_bytes) ||
        overlaps(o.p, o.bytes, slot_row, n * 4) || overlaps(o.p, o.bytes, topk_weights, n * 4))
      return op_fail(MOE_ERR_SHAPE, "combine backward: gradients must not overlap the inputs");
  if (overlaps(drows, n * row_bytes, dweights, n * 4))
    return op_fail(MOE_ERR_SHAPE, "combine backward: gradients must not overlap each other");
  const auto s = (hipStream_t)stream;
  const hipError_t e =
      dtype == kBf16   ? launch_combine_backward_t<kBf16>(dout, rows, T, top_k, hidden, slot_row,
                                                          topk_weights, drows, dweights, s)
      : dtype == kFp16 ? launch_combine_backward_t<kFp16>(dout, rows, T, top_k, hidden, slot_row,
                                                          topk_weights, drows, dweights, s)
                       : launch_combine_backward_t<kFp32>(dout, rows, T, top_k, hidden, slot_row,
                                                          topk_weights, drows, dweights, s);
  MOE_OP_HIP(e, "combine backward");
  return MOE_OK;
}

}  // extern "C"
