// Router logits to routed ids and weights, tokens per expert, the balance and the z loss, and the
// gradient of the logits:
//
//   p = softmax(l);  ids = the top_k largest logits, equal ones by the lower id;  w = p[ids] (/ their sum)
//   balance = E sum_e (c[e] / (n top_k)) (1/n) sum_t p[t, e]        c[e]: slots of expert e, not differentiated
//   z = (1/n) sum_t lse[t]^2,  lse = log sum exp l                  n: tokens that count
//
//   dl[j] = p[j] ((db E / n) (f[j] - <p, f>) + (2 dz / n) lse - q) + s[j],   f = c / (n top_k)
//     renormalised: q = 0, s[ids[i]] = w[i] (dw[i] - <w, dw>);  otherwise q = <w, dw>, s[ids[i]] = w[i] dw[i]
//
// p is taken as exp((l - max) - log sum exp(l - max)): of lse itself, rounded to fp32, it would be off by as
// much as lse's half step, |lse| 2^-24.
//
// A token counts if the mask keeps it and one of its logits is above -inf or a NaN; other tokens have ids
// -1, weights 0 and no gradient. Only logits above -inf are chosen; places without one have id -1.
//
// Not the bytes but vector instructions bound it: a wave a token, or for many tokens of at most 256 experts (512
// with 16 bits) four tokens a wave. Of the 1341 that four tokens of 256 16-bit logits take with top-8 the
// selection's rounds are 264 (33 a round: a subtraction and a maximum a key, and the row's maximum), the keys
// 240, exponentials and the sums of p 270, and what a wave does once, however many tokens it takes, 450
// (addresses, the butterflies and the workgroup's sums; with 8192 tokens that is once for every four). Of 1701
// for fp32 the rounds are 704. us on the GPU: 8 x 256 fp32 4.8, 8192 x 256 bf16 8.3 (0.5 TB/s) and 4.9 for the
// workgroups' sums, 16384 x 256 fp32 20 (0.9 TB/s) and 5.8; the gradient 12 there (2.8 TB/s).
//
// A wave keeps its sums of p in registers and its workgroup the counts in LDS (integer atomics: the order does
// not matter), so that a workgroup leaves one row of partial sums. Sums are taken in a fixed order: those of p in
// fp32 over a wave's tokens and a workgroup's waves, in 64 bits over the workgroups, those of lse^2 in 64 bits
// (fp32's would overflow for logits of 10^19 whose mean of squares it holds).
#include <algorithm>

#include "common.h"
#include "elem.h"
#include "launch.h"
#include "routing.h"
#include "row_sums.h"

namespace {

constexpr int kWaves = 16, kMaxExperts = 512, kMaxGroups = 512;

// The order of a token's logits in 32-bit keys, 0 for "not a candidate", and the selection of the largest
// top_k of a wave's keys (expert lane + 64 c in key[c]): lane r < top_k gets the r-th one's id and value,
// `mine` false where no logit above -inf was left.
//
// Logits of 16 bits leave room for the id: a key is (order, complement of the id), unique, its maximum names
// the expert, and a round is the maximum and one comparison a register (19 VALU operations at 256 experts).
template <int DT, int NC>
struct Select {
  static constexpr uint32_t kInf = DT == kBf16 ? 0x7F80u : 0x7C00u;
  static constexpr uint32_t kLowest = (~(kInf | 0x8000u) & 0xFFFFu) << 16 | 0xFFFFu;  // above any -inf
  MOE_DEV static uint32_t key(uint16_t v, int id) {
    uint32_t u = v;
    u = (u & 0x7FFFu) == 0 ? 0u : u;  // -0 -> +0
    uint32_t o = u & 0x8000u ? ~u & 0xFFFFu : u | 0x8000u;
    o = (u & 0x7FFFu) > kInf ? 0u : o;  // NaN below every number
    return o << 16 | (0xFFFFu - (uint32_t)id);
  }
  MOE_DEV static float value(uint32_t key) {
    const uint32_t o = key >> 16;
    return Elem<DT>::get((uint16_t)(o & 0x8000u ? o & 0x7FFFu : ~o));
  }
  MOE_DEV static void select(uint32_t (&key)[NC], int top_k, int lane, int& id, float& v, bool& mine) {
    uint32_t my = 0;
    for (int r = 0; r < top_k; ++r) {
      uint32_t m = key[0];
#pragma unroll
      for (int c = 1; c < NC; ++c) m = max(m, key[c]);
      m = wave_max_u32(m);
      if (m <= kLowest) break;
#pragma unroll
      for (int c = 0; c < NC; ++c) key[c] = key[c] == m ? 0u : key[c];
      my = lane == r ? m : my;
    }
    id = (int)(0xFFFFu - (my & 0xFFFFu));
    v = value(my);
    mine = my != 0;
  }
};
// Logits of 32 bits: the lanes that hold the maximum name their lowest id; where several do, the lowest of
// theirs is looked for register by register.
template <int NC>
struct Select<kFp32, NC> {
  static constexpr uint32_t kLowest = 0x007FFFFFu;  // topk_ord(-inf)
  MOE_DEV static uint32_t key(float v, int) { return topk_ord(v); }
  MOE_DEV static float value(uint32_t key) { return topk_ord_value(key); }
  MOE_DEV static void select(uint32_t (&key)[NC], int top_k, int lane, int& id, float& v, bool& mine) {
    uint32_t my = 0;
    id = 0;
    for (int r = 0; r < top_k; ++r) {
      uint32_t m = key[0];
#pragma unroll
      for (int c = 1; c < NC; ++c) m = max(m, key[c]);
      m = wave_max_u32(m);
      if (m <= kLowest) break;
      int held = -1;
#pragma unroll
      for (int c = NC - 1; c >= 0; --c) held = key[c] == m ? lane + 64 * c : held;
      const uint64_t holds = __ballot(held >= 0);
      int sel = __builtin_amdgcn_readlane(held, __builtin_ctzll(holds));
      if (holds & (holds - 1)) {
        sel = -1;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const uint64_t b = __ballot(key[c] == m);
          if (sel < 0 && b != 0) sel = 64 * c + __builtin_ctzll(b);
        }
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) key[c] = lane + 64 * c == sel ? 0u : key[c];
      if (lane == r) {
        id = sel;
        my = m;
      }
    }
    v = value(my);
    mine = my != 0;
  }
};

// Behind one another in the workspace: the workgroups' sums, and the sums kernel's own.
struct RouteWs {
  uint32_t* arrived;  // [1]
  double* parts;      // [kMaxExperts / kCols] of the balance
  double* z;          // [groups]
  int32_t* n;         // [groups]
  float* p;           // [groups][E]
  int32_t* c;         // [groups][E]
};

struct RouteArgs {
  const void* logits;
  const uint8_t* mask;  // nullable
  int T, E, k, renorm, groups;
  int32_t* ids;
  float* weights;
  int32_t* counts;
  float* balance;
  float* z;
  float* stats;  // nullable: [2 T + 1], each token's largest logit and log sum exp less it (+inf: does not
                 // count), then n
  RouteWs ws;
};

MOE_DEV float wave_sum(float v) { return bfly_sum(v); }
MOE_DEV double wave_sum(double v) {
  v += partner<32>(v);
  v += partner<16>(v);
  v += partner<8>(v);
  v += partner<4>(v);
  v += partner<2>(v);
  return v + partner<1>(v);
}

constexpr int kCols = 16;  // experts a workgroup of the sums: at most 32 workgroups

// The losses from their sums.
MOE_DEV void finish(const RouteArgs& a, double dot, double zsum, int n) {
  const double inv = n > 0 ? 1.0 / (double)n : 0.0;
  *a.balance = (float)((double)a.E * dot * inv * inv / (double)a.k);
  *a.z = (float)(zsum * inv);
  if (a.stats) a.stats[2 * (int64_t)a.T] = (float)n;
}

// A workgroup's sums: p of each wave and expert, slots of each expert.
template <int W, int NE>
struct BlockSums {
  float p[W][NE];
  int c[NE];
  double z[W];
  int n[W];
  double dot[W];
  MOE_DEV void clear(const RouteArgs& a) {
    for (int e = threadIdx.x; e < NE; e += blockDim.x) c[e] = 0;
    if (a.groups > 1 && blockIdx.x == 0 && threadIdx.x == 0) *a.ws.arrived = 0;
    __syncthreads();
  }
};

// Behind every wave's p: the workgroup's row of partial sums, or the results where it is the only one. z and n
// are the wave's.
template <int W, int NE>
MOE_DEV void block_sums(const RouteArgs& a, BlockSums<W, NE>& s, double zsum, int n) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
  if (lane == 0) {
    s.z[wave] = zsum;
    s.n[wave] = n;
  }
  __syncthreads();
  double z = 0.0;
  int live = 0;
  for (int w = 0; w < waves; ++w) {
    z += s.z[w];
    live += s.n[w];
  }
  if (a.groups > 1) {
    for (int e = tid; e < a.E; e += blockDim.x) {
      float p = 0.0f;
      for (int w = 0; w < waves; ++w) p += s.p[w][e];
      a.ws.p[(int64_t)blockIdx.x * a.E + e] = p;
      a.ws.c[(int64_t)blockIdx.x * a.E + e] = s.c[e];
    }
    if (tid == 0) {
      a.ws.z[blockIdx.x] = z;
      a.ws.n[blockIdx.x] = live;
    }
    return;
  }
  double dot = 0.0;
  for (int e = tid; e < a.E; e += blockDim.x) {
    float p = 0.0f;
    for (int w = 0; w < waves; ++w) p += s.p[w][e];
    a.counts[e] = s.c[e];
    dot += (double)s.c[e] * (double)p;
  }
  dot = wave_sum(dot);
  if (lane == 0) s.dot[wave] = dot;
  __syncthreads();
  if (tid == 0) {
    dot = 0.0;
    for (int w = 0; w < waves; ++w) dot += s.dot[w];
    finish(a, dot, z, live);
  }
}

// exp(x) for x <= 0, and a NaN for a NaN: 2^(x log2 e) with the product in two parts, off by about 2 half
// steps; a third of the library's operations. The hardware's 2^x gives zero below 2^-126. SMALL: it is taken 2^64
// higher there, down to fp32's smallest number. The weights take it so. Beside the 1 in a token's sum, and in
// the balance beside a token's first expert, such a term counts for less than 2^-100.
template <bool SMALL = false>
MOE_DEV float exp_neg(float x) {
  constexpr float kLog2e = 0x1.715476p+0f, kLog2eLow = 0x1.4ae0c0p-26f, kLn2 = 0x1.62e430p-1f;
  x = x < -110.0f ? -110.0f : x;
  const float hi = x * kLog2e;
  const float lo = __builtin_fmaf(x, kLog2eLow, __builtin_fmaf(x, kLog2e, -hi));
  const bool small = SMALL && hi < -126.0f;
  const float r = __builtin_amdgcn_exp2f(small ? hi + 64.0f : hi);
  const float e = __builtin_fmaf(r * lo, kLn2, r);
  return small ? e * 0x1p-64f : e;
}

// ---------------------------------------------------------------- 16 lanes a token
template <int M>
MOE_DEV uint32_t row_partner(uint32_t v) { return __float_as_uint(xor_partner<M>(__uint_as_float(v))); }
// Neighbour, pair, mirrored half and mirrored row: once they agree within what is mirrored, that is the other.
MOE_DEV uint32_t row_max(uint32_t v) {
  v = max(v, MOE_DPP(v, 0xB1, 0xF));
  v = max(v, MOE_DPP(v, 0x4E, 0xF));
  v = max(v, MOE_DPP(v, 0x141, 0xF));
  return max(v, MOE_DPP(v, 0x140, 0xF));
}
MOE_DEV float row_max(float v) {  // of a NaN and a number the number
  v = __builtin_fmaxf(v, xor_partner<8>(v));
  v = __builtin_fmaxf(v, xor_partner<4>(v));
  v = __builtin_fmaxf(v, xor_partner<2>(v));
  return __builtin_fmaxf(v, xor_partner<1>(v));
}
MOE_DEV float row_sum(float v) {
  v += xor_partner<8>(v);
  v += xor_partner<4>(v);
  v += xor_partner<2>(v);
  return v + xor_partner<1>(v);
}

// The order of a token's logits in PL keys a lane (expert 16 j + lane), 0 for "not a candidate", and the
// selection: lane r < top_k gets the r-th largest one's id and value, `mine` false where no logit above -inf
// was left. m: the row's largest key.
//
// Logits of 16 bits leave room for the id: (order, complement of the id), unique, 25 bits. Below a maximum m the
// next one is the largest of key - m, in which those not below it are the small ones.
template <int DT, int PL>
struct GroupSelect {
  static constexpr uint32_t kInf = DT == kBf16 ? 0x7F80u : 0x7C00u;
  static constexpr uint32_t kLowest = (~(kInf | 0x8000u) & 0xFFFFu) << 9 | 511u;  // -inf, of any id
  MOE_DEV static uint32_t key(uint16_t v, int id) {
    uint32_t u = v;
    u = (u & 0x7FFFu) == 0 ? 0u : u;  // -0 -> +0
    uint32_t o = u & 0x8000u ? ~u & 0xFFFFu : u | 0x8000u;
    o = (u & 0x7FFFu) > kInf ? 0u : o;  // NaN below every number
    return o << 9 | (511u - (uint32_t)id);
  }
  MOE_DEV static void select(uint32_t (&key)[PL], uint32_t m, int top_k, int l16, int& id, float& v, bool& mine) {
    uint32_t my = 0;
    for (int r = 0; r < top_k; ++r) {
      if (l16 == r) my = m;
      uint32_t d = 0;
#pragma unroll
      for (int j = 0; j < PL; ++j) d = max(d, key[j] - m);
      d = row_max(d);
      m = d >> 31 ? m + d : 0u;  // none left: 0 is below every key
    }
    mine = l16 < top_k && my > kLowest;
    id = (int)(511u - (my & 511u));
    const uint32_t o = my >> 9;
    v = Elem<DT>::get((uint16_t)(o & 0x8000u ? o & 0x7FFFu : ~o));
  }
};
// Logits of 32 bits: the lowest id among those that hold the maximum, which leave.
template <int PL>
struct GroupSelect<kFp32, PL> {
  static constexpr uint32_t kLowest = 0x007FFFFFu;  // topk_ord(-inf)
  MOE_DEV static uint32_t key(float v, int) { return topk_ord(v); }
  MOE_DEV static void select(uint32_t (&key)[PL], uint32_t m, int top_k, int l16, int& id, float& v, bool& mine) {
    uint32_t my = 0;
    id = 0;
    for (int r = 0; r < top_k; ++r) {
      uint32_t held = 0;  // 512 less the id
#pragma unroll
      for (int j = PL - 1; j >= 0; --j) held = key[j] == m ? 512u - 16u * j : held;
      held = row_max(held != 0 ? held - (uint32_t)l16 : 0u);
      if (l16 == r) {
        my = m;
        id = (int)(512u - held);
      }
      const uint32_t at = 512u - held - (uint32_t)l16;
      m = 0;
#pragma unroll
      for (int j = 0; j < PL; ++j) {
        key[j] = at == 16u * j ? 0u : key[j];
        m = max(m, key[j]);
      }
      m = row_max(m);
    }
    mine = l16 < top_k && my > kLowest;
    v = topk_ord_value(my);
  }
};

// Four tokens a wave: a round of the selection is a few operations for each of a lane's logits and one or two
// maxima over 16 lanes, for all four. us of the routing with a wave a token / with this: bf16 8192 x 256, top-8
// 17.4 / 13.4, 32768 x 64 25.7 / 13.6, 1501 x 60 (fp16, top-5) 9.4 / 8.7; fp32 32768 x 8, top-2 20.2 / 12.0, 32768 x
// 64 28.9 / 15.9, 32768 x 128 32.8 / 20.4, 16384 x 256 25.4 / 24.1, 32768 x 512, top-10 59.7 / 64.6. Of few tokens
// a wave's own are done sooner (256 x 256 fp32 11.2 / 15.4).
constexpr int kGroupWaves = 8, kGroupTokens = 4 * kGroupWaves, kGroupMaxTopK = 16, kGroupMinT = 1024;
constexpr int kGroupMaxFp32 = 256;
bool route_grouped(int T, int E, int k, int dtype) {
  return (dtype != kFp32 || E <= kGroupMaxFp32) && k <= kGroupMaxTopK && T >= kGroupMinT;
}

// PL logits a lane: expert 16 j + (lane & 15).
template <int DT, int PL>
__global__ __launch_bounds__(64 * kGroupWaves) void route_group_kernel(RouteArgs a) {
  using T = typename Elem<DT>::T;
  using S = GroupSelect<DT, PL>;
  __shared__ BlockSums<kGroupWaves, 16 * PL> s;
  const int lane = threadIdx.x & 63, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = blockDim.x >> 6;
  s.clear(a);
  float psum[PL];
  double zsum = 0.0;
  int n = 0;
#pragma unroll
  for (int j = 0; j < PL; ++j) psum[j] = 0.0f;
  const int64_t stride = (int64_t)gridDim.x * waves * 4;
  T next[PL];
  bool next_kept = false;
  auto load = [&](int64_t t) {  // past the last token: read again, not used
    const int64_t u = min(t, (int64_t)a.T - 1);
    const T* row = static_cast<const T*>(a.logits) + u * a.E;
#pragma unroll
    for (int j = 0; j < PL; ++j) next[j] = row[min(16 * j + l16, a.E - 1)];
    next_kept = !a.mask || a.mask[u] != 0;
  };
  int64_t t = ((int64_t)blockIdx.x * waves + wave) * 4 + (lane >> 4);
  if (t - (lane >> 4) < a.T) load(t);
  for (; t - (lane >> 4) < a.T; t += stride) {
    float x[PL];
    uint32_t key[PL], m = 0;
    float top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < PL; ++j) {
      const bool in = 16 * j + l16 < a.E;
      x[j] = in ? Elem<DT>::get(next[j]) : -__builtin_inff();
      key[j] = in ? S::key(next[j], 16 * j + l16) : 0u;
      top = __builtin_fmaxf(top, x[j]);
      m = max(m, key[j]);
    }
    const bool kept = next_kept && t < a.T;
    load(t + stride);
    top = row_max(top);
    const bool some = top > -__builtin_inff();
    if (!some) top = 0.0f;
    m = row_max(m);
    int id;
    float v;
    bool chosen;
    S::select(key, m, a.k, l16, id, v, chosen);
    float total = 0.0f;
#pragma unroll
    for (int j = 0; j < PL; ++j) {
      x[j] = exp_neg(x[j] - top);
      total += x[j];
    }
    total = row_sum(total);
    const bool live = kept && (some || total != total);
    chosen = chosen && live;
    const float mine = chosen ? exp_neg<true>(v - top) : 0.0f;
    float over = total;
    if (a.renorm) {
      // a NaN or +inf among the logits makes the weights NaN, also where it is not chosen
      over = row_sum(mine);
      if (!(total < __builtin_inff())) over = total;
    }
    if (t < a.T && l16 < a.k) {
      a.ids[t * a.k + l16] = chosen ? id : -1;
      a.weights[t * a.k + l16] = chosen ? mine / over : 0.0f;
    }
    if (chosen) atomicAdd(&s.c[id], 1);
    const float rest = logf(total), lse = top + rest;
    if (a.stats && l16 == 0 && t < a.T) {
      a.stats[2 * t] = top;
      a.stats[2 * t + 1] = live ? rest : __builtin_inff();
    }
    if (live) {
      const float inv = 1.0f / total;
#pragma unroll
      for (int j = 0; j < PL; ++j) psum[j] = __builtin_fmaf(x[j], inv, psum[j]);
      if (l16 == 0) {
        zsum = __builtin_fma((double)lse, (double)lse, zsum);
        ++n;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < PL; ++j) {
    psum[j] += xor_partner<16>(psum[j]);
    psum[j] += xor_partner<32>(psum[j]);
    if (lane < 16) s.p[wave][16 * j + l16] = psum[j];
  }
  zsum = wave_sum(zsum);
  n = (int)wave_sum((float)n);  // at most 2^22
  block_sums(a, s, zsum, n);
}

// ---------------------------------------------------------------- a wave a token
// NC registers of 64 experts each.
template <int DT, int NC>
__global__ __launch_bounds__(64 * kWaves) void route_kernel(RouteArgs a) {
  using T = typename Elem<DT>::T;
  __shared__ BlockSums<kWaves, 64 * NC> s;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int waves = blockDim.x >> 6;
  s.clear(a);
  float psum[NC];
  double zsum = 0.0;
  int n = 0;
#pragma unroll
  for (int c = 0; c < NC; ++c) psum[c] = 0.0f;
  using S = Select<DT, NC>;
  const int64_t stride = (int64_t)gridDim.x * waves;
  T next[NC];
  bool next_kept = false;
  auto load = [&](int64_t t) {  // past the last token: read again, not used
    const int64_t u = min(t, (int64_t)a.T - 1);
    const T* row = static_cast<const T*>(a.logits) + u * a.E;
#pragma unroll
    for (int c = 0; c < NC; ++c) next[c] = row[min(lane + 64 * c, a.E - 1)];
    next_kept = !a.mask || a.mask[u] != 0;
  };
  const int64_t first = (int64_t)blockIdx.x * waves + wave;
  if (first < a.T) load(first);
  for (int64_t t = first; t < a.T; t += stride) {
    float l[NC];
    uint32_t key[NC], peak = 0;
    bool nan = false;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const bool in = lane + 64 * c < a.E;
      key[c] = in ? S::key(next[c], lane + 64 * c) : 0u;
      l[c] = in ? Elem<DT>::get(next[c]) : -__builtin_inff();
      nan |= l[c] != l[c];
      peak = max(peak, key[c]);
    }
    const bool kept = next_kept;
    load(t + stride);
    peak = wave_max_u32(peak);
    const bool live = kept && (peak > S::kLowest || __ballot(nan) != 0);
    const float top = peak > S::kLowest ? S::value(peak) : 0.0f;
    float ex[NC], total = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      ex[c] = exp_neg(l[c] - top);
      total += ex[c];
    }
    total = wave_sum(total);
    int my_i;
    float my_v;
    bool chosen;
    S::select(key, live ? a.k : 0, lane, my_i, my_v, chosen);
    const float mine = chosen ? exp_neg<true>(my_v - top) : 0.0f;
    float over = total;
    if (a.renorm) {
      // a NaN or +inf among the logits makes the weights NaN, also where it is not chosen
      over = wave_sum(mine);
      if (!(total < __builtin_inff())) over = total;
    }
    if (lane < a.k) {
      a.ids[t * a.k + lane] = chosen ? my_i : -1;
      a.weights[t * a.k + lane] = chosen ? mine / over : 0.0f;
    }
    if (chosen) atomicAdd(&s.c[my_i], 1);
    const float rest = logf(total), lse = top + rest;
    if (a.stats && lane == 0) {
      a.stats[2 * t] = top;
      a.stats[2 * t + 1] = live ? rest : __builtin_inff();
    }
    if (live) {
      const float inv = 1.0f / total;
#pragma unroll
      for (int c = 0; c < NC; ++c) psum[c] = __builtin_fmaf(ex[c], inv, psum[c]);
      zsum = __builtin_fma((double)lse, (double)lse, zsum);
      ++n;
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) s.p[wave][lane + 64 * c] = psum[c];
  block_sums(a, s, zsum, n);
}

// The workgroups' sums: kCols experts a workgroup, 64 threads an expert. The last workgroup to arrive adds
// the workgroups' shares of the balance, in their order; z and the count each has summed ahead of that.
__global__ __launch_bounds__(1024) void route_sum_kernel(RouteArgs a) {
  __shared__ double s_p[16][kCols];
  __shared__ int s_c[16][kCols];
  __shared__ double s_z[16];
  __shared__ int s_n[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int col = tid % kCols, slot = tid / kCols;
  const int e = blockIdx.x * kCols + col, at = min(e, a.E - 1);
  double p = 0.0;
  int c = 0;
#pragma unroll 8
  for (int g = slot; g < a.groups; g += 1024 / kCols) {
    p += (double)a.ws.p[(int64_t)g * a.E + at];
    c += a.ws.c[(int64_t)g * a.E + at];
  }
  double z = tid < a.groups ? a.ws.z[tid] : 0.0;  // at most 512 workgroups
  int n = tid < a.groups ? a.ws.n[tid] : 0;
  // a wave's four slots of an expert: lanes col, col + 16, ...
  p += partner<32>(p);
  p += partner<16>(p);
  c += (int)row_partner<32>((uint32_t)c);
  c += (int)row_partner<16>((uint32_t)c);
  z = wave_sum(z);
  n = (int)wave_sum((double)n);
  if (lane < kCols) {
    s_p[wave][lane] = p;
    s_c[wave][lane] = c;
  }
  if (lane == 0) {
    s_z[wave] = z;
    s_n[wave] = n;
  }
  __syncthreads();
  if (wave != 0) return;
  double dot = 0.0;
  if (lane < kCols && e < a.E) {
    p = 0.0;
    c = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      p += s_p[i][lane];
      c += s_c[i][lane];
    }
    a.counts[e] = c;
    dot = (double)c * p;
  }
  z = lane < 16 ? s_z[lane] : 0.0;
  n = lane < 16 ? s_n[lane] : 0;
  dot = wave_sum(dot);
  z = wave_sum(z);
  n = (int)wave_sum((double)n);
  uint32_t before = 0;
  if (lane == 0) {
    __hip_atomic_store(a.ws.parts + blockIdx.x, dot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    before = __hip_atomic_fetch_add(a.ws.arrived, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
  }
  if ((uint32_t)__builtin_amdgcn_readfirstlane((int)before) != gridDim.x - 1) return;
  dot = lane < (int)gridDim.x ? __hip_atomic_load(a.ws.parts + lane, __ATOMIC_RELAXED,
                                                  __HIP_MEMORY_SCOPE_AGENT)
                              : 0.0;
  dot = wave_sum(dot);
  if (lane == 0) finish(a, dot, z, n);
}

struct RouteGradArgs {
  const void* logits;
  int T, E, k, renorm;
  const int32_t* ids;
  const float* weights;
  const int32_t* counts;
  const float* stats;     // [2 T + 1]
  const float* dweights;  // the three are nullable
  const float* dbalance;
  const float* dz;
  void* dlogits;
};

constexpr int kGradWaves = 4;

template <int DT, int NC>
__global__ __launch_bounds__(64 * kGradWaves) void route_backward_kernel(RouteGradArgs a) {
  using T = typename Elem<DT>::T;
  __shared__ float s_d[kGradWaves][64 * NC];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float n = a.stats[2 * (int64_t)a.T], inv_n = n > 0.0f ? 1.0f / n : 0.0f;
  const float cb = a.dbalance ? *a.dbalance * ((float)a.E * inv_n) : 0.0f;
  const float cz = a.dz ? 2.0f * *a.dz * inv_n : 0.0f;
  const float unit = inv_n / (float)a.k;
  float f[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    f[c] = lane + 64 * c < a.E ? (float)a.counts[min(lane + 64 * c, a.E - 1)] * unit : 0.0f;
    s_d[wave][lane + 64 * c] = 0.0f;
  }
  for (int64_t t = (int64_t)blockIdx.x * kGradWaves + wave; t < a.T;
       t += (int64_t)gridDim.x * kGradWaves) {
    const T* row = static_cast<const T*>(a.logits) + t * a.E;
    float p[NC], pf = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) p[c] = Elem<DT>::get(row[min(lane + 64 * c, a.E - 1)]);
    const float top = a.stats[2 * t], rest = a.stats[2 * t + 1], lse = top + rest;
    const bool live = rest != __builtin_inff();
    int id = lane < a.k ? a.ids[t * a.k + lane] : -1;
    id = id < a.E ? id : -1;
    float w = 0.0f, dw = 0.0f;
    if (a.dweights && id >= 0) {
      w = a.weights[t * a.k + lane];
      dw = a.dweights[t * a.k + lane];
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      p[c] = live && lane + 64 * c < a.E ? expf((p[c] - top) - rest) : 0.0f;
      pf = __builtin_fmaf(p[c], f[c], pf);
    }
    pf = wave_sum(pf);
    const float dot = a.dweights ? wave_sum(w * dw) : 0.0f;
    if (a.dweights && id >= 0) s_d[wave][id] = w * (a.renorm ? dw - dot : dw);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const float all = live ? cz * lse - (a.renorm ? 0.0f : dot) : 0.0f;
    T* out = static_cast<T*>(a.dlogits) + t * a.E;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float d = __builtin_fmaf(p[c], __builtin_fmaf(cb, f[c] - pf, all), s_d[wave][lane + 64 * c]);
      if (lane + 64 * c < a.E) out[lane + 64 * c] = Elem<DT>::put(live ? d : 0.0f);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (id >= 0) s_d[wave][id] = 0.0f;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

int64_t align256(int64_t v) { return (v + 255) & ~int64_t(255); }

// Workgroups; the workspace is sized for a wave a token, which has the more of them.
int route_groups(int T, int tokens) { return std::max(1, std::min((T - 1) / tokens + 1, kMaxGroups)); }

// The workspace's parts from `base`; its size in *bytes.
RouteWs route_ws(void* base, int T, int E, int64_t* bytes) {
  const int64_t g = route_groups(T, kWaves);
  int64_t o = 0;
  auto take = [&o](int64_t n) {
    const int64_t at = o;
    o += align256(n);
    return at;
  };
  const int64_t arrived = take(4), parts = take(kMaxExperts / kCols * 8), z = take(g * 8),
                n = take(g * 4), p = take(g * E * 4), c = take(g * E * 4);
  *bytes = g > 1 ? o : 0;
  char* b = static_cast<char*>(base);
  return RouteWs{reinterpret_cast<uint32_t*>(b + arrived), reinterpret_cast<double*>(b + parts),
                 reinterpret_cast<double*>(b + z), reinterpret_cast<int32_t*>(b + n),
                 reinterpret_cast<float*>(b + p), reinterpret_cast<int32_t*>(b + c)};
}

template <int DT, int NC>
hipError_t launch_route(const RouteArgs& a, hipStream_t s) {
  if constexpr (DT != kFp32 || 64 * NC <= kGroupMaxFp32) {
    if (route_grouped(a.T, a.E, a.k, DT))
      hipLaunchKernelGGL((route_group_kernel<DT, 4 * NC>), dim3(a.groups), dim3(64 * kGroupWaves), 0, s, a);
  }
  if (!route_grouped(a.T, a.E, a.k, DT)) {
    const int waves = std::max(1, std::min(a.T, kWaves));
    hipLaunchKernelGGL((route_kernel<DT, NC>), dim3(a.groups), dim3(64 * waves), 0, s, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.groups == 1) return e;
  hipLaunchKernelGGL(route_sum_kernel, dim3((a.E + kCols - 1) / kCols), dim3(1024), 0, s, a);
  return hipGetLastError();
}

template <int DT, int NC>
hipError_t launch_backward(const RouteGradArgs& a, hipStream_t s) {
  const int groups = std::min((a.T - 1) / kGradWaves + 1, 4096);
  hipLaunchKernelGGL((route_backward_kernel<DT, NC>), dim3(groups), dim3(64 * kGradWaves), 0, s, a);
  return hipGetLastError();
}

#define MOE_ROUTE_NC(E, CALL)                                                  \
  ((E) <= 64 ? CALL(1) : (E) <= 128 ? CALL(2) : (E) <= 256 ? CALL(4) : CALL(8))

template <int DT>
hipError_t launch_route_any(const RouteArgs& a, hipStream_t s) {
#define MOE_ROUTE_CALL(NC) launch_route<DT, NC>(a, s)
  return MOE_ROUTE_NC(a.E, MOE_ROUTE_CALL);
#undef MOE_ROUTE_CALL
}
template <int DT>
hipError_t launch_backward_any(const RouteGradArgs& a, hipStream_t s) {
#define MOE_ROUTE_CALL(NC) launch_backward<DT, NC>(a, s)
  return MOE_ROUTE_NC(a.E, MOE_ROUTE_CALL);
#undef MOE_ROUTE_CALL
}

int check_route(const char* what, int32_t T, int32_t E, int32_t dtype, int32_t k) {
  if (dtype < kBf16 || dtype > kFp32)
    return op_fail(MOE_ERR_UNSUPPORTED, "%s: dtype=%d (0 bf16, 1 fp16, 2 fp32)", what, dtype);
  if (E < 1 || E > kMaxExperts)
    return op_fail(MOE_ERR_SHAPE, "%s: num_experts=%d outside [1, %d]", what, E, kMaxExperts);
  if (T < 0 || k < 1 || k > 64 || k > E || (int64_t)T * k > (1 << 22))
    return op_fail(MOE_ERR_SHAPE,
                   "%s: T=%d top_k=%d (top_k in [1, 64] and at most the experts, at most 2^22 slots)",
                   what, T, k);
  return MOE_OK;
}

struct Mem {
  const void* p;
  int64_t bytes;
};
template <int NO, int NI>
bool any_overlap(const Mem (&outs)[NO], const Mem (&ins)[NI]) {
  for (const Mem& o : outs) {
    for (const Mem& i : ins)
      if (overlaps(o.p, o.bytes, i.p, i.bytes)) return true;
    for (const Mem* i = outs; i != &o; ++i)
      if (overlaps(o.p, o.bytes, i->p, i->bytes)) return true;
  }
  return false;
}

}  // namespace

extern "C" {

int64_t moe_route_workspace_bytes_v1(int32_t T, int32_t num_experts) {
  if (T < 0 || num_experts < 1 || num_experts > kMaxExperts) return -1;
  int64_t bytes;
  route_ws(nullptr, T, num_experts, &bytes);
  return bytes;
}

int moe_route_v1(const void* logits, int32_t T, int32_t num_experts, int32_t dtype, int32_t top_k,
                 const uint8_t* mask, int32_t renormalize, void* workspace,
                 int64_t workspace_bytes, int32_t* topk_ids, float* topk_weights, int32_t* counts,
                 float* balance, float* z, float* stats, void* stream) {
  const int rc = check_route("route", T, num_experts, dtype, top_k);
  if (rc) return rc;
  if ((T > 0 && (!logits || !topk_ids || !topk_weights)) || !counts || !balance || !z)
    return op_fail(MOE_ERR_NULL, "route: NULL pointer");
  int64_t need;
  const RouteWs ws = route_ws(workspace, T, num_experts, &need);
  if (need > 0) {
    if (!workspace || workspace_bytes < need)
      return op_fail(MOE_ERR_WORKSPACE, "route: workspace of %lld bytes, needs %lld",
                     (long long)(workspace ? workspace_bytes : 0), (long long)need);
    if (!workspace_aligned(workspace))
      return op_fail(MOE_ERR_WORKSPACE, "route: workspace must be 256-byte aligned");
  }
  const int64_t S = (int64_t)T * top_k;
  const Mem outs[] = {{workspace, need}, {topk_ids, S * 4}, {topk_weights, S * 4},
                      {counts, (int64_t)num_experts * 4}, {balance, 4}, {z, 4},
                      {stats, ((int64_t)2 * T + 1) * 4}};
  const Mem ins[] = {{logits, (int64_t)T * num_experts * dtype_bytes(dtype)}, {mask, T}};
  if (any_overlap(outs, ins))
    return op_fail(MOE_ERR_SHAPE,
                   "route: outputs and workspace must not overlap the inputs or each other");
  const RouteArgs a{logits, mask, T, num_experts, top_k, renormalize != 0,
                    route_groups(T, route_grouped(T, num_experts, top_k, dtype) ? kGroupTokens : kWaves), topk_ids,
                    topk_weights, counts, balance, z, stats, ws};
  const auto s = (hipStream_t)stream;
  MOE_OP_HIP(dtype == kBf16   ? launch_route_any<kBf16>(a, s)
             : dtype == kFp16 ? launch_route_any<kFp16>(a, s)
                              : launch_route_any<kFp32>(a, s),
             "route");
  return MOE_OK;
}

int moe_route_backward_v1(const void* logits, int32_t T, int32_t num_experts, int32_t dtype,
                          int32_t top_k, int32_t renormalize, const int32_t* topk_ids,
                          const float* topk_weights, const int32_t* counts, const float* stats,
                          const float* dweights, const float* dbalance, const float* dz,
                          void* dlogits, void* stream) {
  const int rc = check_route("route backward", T, num_experts, dtype, top_k);
  if (rc) return rc;
  if (T == 0) return MOE_OK;
  if (!logits || !topk_ids || !topk_weights || !counts || !stats || !dlogits)
    return op_fail(MOE_ERR_NULL, "route backward: NULL pointer");
  const int64_t S = (int64_t)T * top_k, nl = (int64_t)T * num_experts * dtype_bytes(dtype);
  const Mem outs[] = {{dlogits, nl}};
  const Mem ins[] = {{logits, nl}, {topk_ids, S * 4}, {topk_weights, S * 4},
                     {counts, (int64_t)num_experts * 4}, {stats, ((int64_t)2 * T + 1) * 4},
                     {dweights, S * 4}, {dbalance, 4}, {dz, 4}};
  if (any_overlap(outs, ins))
    return op_fail(MOE_ERR_SHAPE, "route backward: dlogits must not overlap the inputs");
  const RouteGradArgs a{logits, T, num_experts, top_k, renormalize != 0, topk_ids, topk_weights,
                        counts, stats, dweights, dbalance, dz, dlogits};
  const auto s = (hipStream_t)stream;
  MOE_OP_HIP(dtype == kBf16   ? launch_backward_any<kBf16>(a, s)
             : dtype == kFp16 ? launch_backward_any<kFp16>(a, s)
                              : launch_backward_any<kFp32>(a, s),
             "route backward");
  return MOE_OK;
}

}  // extern "C"
