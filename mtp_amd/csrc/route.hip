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
// A token counts if the mask keeps it and one of its logits is above -inf or a NaN; other tokens have ids
// -1, weights 0 and no gradient. Only logits above -inf are chosen; places without one have id -1.
//
// A wave takes a token, 64 experts a register; the selection's rounds (a wave maximum and a ballot each)
// bound it, not the bytes: they are a few VALU operations a byte read. A wave keeps its sums of p in
// registers and its workgroup the counts in LDS (integer atomics: the order does not matter), so that a
// workgroup leaves one row of partial sums. Sums are taken in a fixed order: fp32 over a wave's tokens
// and a workgroup's waves, 64 bits over the workgroups.
#include <algorithm>

#include "common.h"
#include "elem.h"
#include "launch.h"
#include "routing.h"

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
  float* z;           // [groups]
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
  float* lse;  // nullable: [T + 1], lse of each token (+inf: does not count), then n
  RouteWs ws;
};

MOE_DEV float wave_sum(float v) { return bfly_sum(v); }

constexpr int kCols = 16;  // experts a workgroup of the sums: at most 32 workgroups

// The losses from their sums.
MOE_DEV void finish(const RouteArgs& a, double dot, double zsum, int n) {
  const double inv = n > 0 ? 1.0 / (double)n : 0.0;
  *a.balance = (float)((double)a.E * dot * inv * inv / (double)a.k);
  *a.z = (float)(zsum * inv);
  if (a.lse) a.lse[a.T] = (float)n;
}

// NC registers of 64 experts each.
template <int DT, int NC>
__global__ __launch_bounds__(64 * kWaves) void route_kernel(RouteArgs a) {
  using T = typename Elem<DT>::T;
  __shared__ float s_p[kWaves][64 * NC];
  __shared__ int s_c[64 * NC];
  __shared__ float s_z[kWaves];
  __shared__ int s_n[kWaves];
  __shared__ double s_dot[kWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int waves = blockDim.x >> 6;
  for (int e = tid; e < 64 * NC; e += blockDim.x) s_c[e] = 0;
  if (a.groups > 1 && blockIdx.x == 0 && tid == 0) *a.ws.arrived = 0;
  __syncthreads();
  float psum[NC], zsum = 0.0f;
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
      ex[c] = expf(l[c] - top);
      total += ex[c];
    }
    total = wave_sum(total);
    int my_i;
    float my_v;
    bool chosen;
    S::select(key, live ? a.k : 0, lane, my_i, my_v, chosen);
    const float mine = chosen ? expf(my_v - top) : 0.0f;
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
    if (chosen) atomicAdd(&s_c[my_i], 1);
    const float lse = live ? top + logf(total) : 0.0f;
    if (a.lse && lane == 0) a.lse[t] = live ? lse : __builtin_inff();
    if (live) {
      const float inv = 1.0f / total;
#pragma unroll
      for (int c = 0; c < NC; ++c) psum[c] = __builtin_fmaf(ex[c], inv, psum[c]);
      zsum = __builtin_fmaf(lse, lse, zsum);
      ++n;
    }
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) s_p[wave][lane + 64 * c] = psum[c];
  if (lane == 0) {
    s_z[wave] = zsum;
    s_n[wave] = n;
  }
  __syncthreads();
  float z = 0.0f;
  int live = 0;
  for (int w = 0; w < waves; ++w) {
    z += s_z[w];
    live += s_n[w];
  }
  if (a.groups > 1) {
    for (int e = tid; e < a.E; e += blockDim.x) {
      float p = 0.0f;
      for (int w = 0; w < waves; ++w) p += s_p[w][e];
      a.ws.p[(int64_t)blockIdx.x * a.E + e] = p;
      a.ws.c[(int64_t)blockIdx.x * a.E + e] = s_c[e];
    }
    if (tid == 0) {
      a.ws.z[blockIdx.x] = z;
      a.ws.n[blockIdx.x] = live;
    }
    return;
  }
  // one workgroup: the sums are all here
  double dot = 0.0;
  for (int e = tid; e < a.E; e += blockDim.x) {
    float p = 0.0f;
    for (int w = 0; w < waves; ++w) p += s_p[w][e];
    a.counts[e] = s_c[e];
    dot += (double)s_c[e] * (double)p;
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) dot += __shfl_xor(dot, m);
  if (lane == 0) s_dot[wave] = dot;
  __syncthreads();
  if (tid == 0) {
    dot = 0.0;
    for (int w = 0; w < waves; ++w) dot += s_dot[w];
    finish(a, dot, (double)z, live);
  }
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
  double z = tid < a.groups ? (double)a.ws.z[tid] : 0.0;  // at most 512 workgroups
  int n = tid < a.groups ? a.ws.n[tid] : 0;
  // a wave's slots of an expert: lanes col, col + 16, ...
  for (int m = 32; m >= kCols; m >>= 1) {
    p += __shfl_xor(p, m);
    c += __shfl_xor(c, m);
  }
  for (int m = 32; m >= 1; m >>= 1) {
    z += __shfl_xor(z, m);
    n += __shfl_xor(n, m);
  }
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
  for (int m = 8; m >= 1; m >>= 1) {  // lanes 0 to 15 hold all of the three
    dot += __shfl_xor(dot, m);
    z += __shfl_xor(z, m);
    n += __shfl_xor(n, m);
  }
  uint32_t before = 0;
  if (lane == 0) {
    __hip_atomic_store(a.ws.parts + blockIdx.x, dot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    before = __hip_atomic_fetch_add(a.ws.arrived, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
  }
  if ((uint32_t)__builtin_amdgcn_readfirstlane((int)before) != gridDim.x - 1) return;
  dot = lane < (int)gridDim.x ? __hip_atomic_load(a.ws.parts + lane, __ATOMIC_RELAXED,
                                                  __HIP_MEMORY_SCOPE_AGENT)
                              : 0.0;
  for (int m = 32; m >= 1; m >>= 1) dot += __shfl_xor(dot, m);
  if (lane == 0) finish(a, dot, z, n);
}

struct RouteGradArgs {
  const void* logits;
  int T, E, k, renorm;
  const int32_t* ids;
  const float* weights;
  const int32_t* counts;
  const float* lse;       // [T + 1]
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
  const float n = a.lse[a.T], inv_n = n > 0.0f ? 1.0f / n : 0.0f;
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
    const float lse = a.lse[t];
    const bool live = lse != __builtin_inff();
    int id = lane < a.k ? a.ids[t * a.k + lane] : -1;
    id = id < a.E ? id : -1;
    float w = 0.0f, dw = 0.0f;
    if (a.dweights && id >= 0) {
      w = a.weights[t * a.k + lane];
      dw = a.dweights[t * a.k + lane];
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      p[c] = live && lane + 64 * c < a.E ? expf(p[c] - lse) : 0.0f;
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

int route_groups(int T) { return std::max(1, std::min((T - 1) / kWaves + 1, kMaxGroups)); }

// The workspace's parts from `base`; its size in *bytes.
RouteWs route_ws(void* base, int T, int E, int64_t* bytes) {
  const int64_t g = route_groups(T);
  int64_t o = 0;
  auto take = [&o](int64_t n) {
    const int64_t at = o;
    o += align256(n);
    return at;
  };
  const int64_t arrived = take(4), parts = take(kMaxExperts / kCols * 8), z = take(g * 4),
                n = take(g * 4), p = take(g * E * 4), c = take(g * E * 4);
  *bytes = g > 1 ? o : 0;
  char* b = static_cast<char*>(base);
  return RouteWs{reinterpret_cast<uint32_t*>(b + arrived), reinterpret_cast<double*>(b + parts),
                 reinterpret_cast<float*>(b + z), reinterpret_cast<int32_t*>(b + n),
                 reinterpret_cast<float*>(b + p), reinterpret_cast<int32_t*>(b + c)};
}

template <int DT, int NC>
hipError_t launch_route(const RouteArgs& a, hipStream_t s) {
  const int waves = std::max(1, std::min(a.T, kWaves));
  hipLaunchKernelGGL((route_kernel<DT, NC>), dim3(a.groups), dim3(64 * waves), 0, s, a);
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
                 float* balance, float* z, float* lse, void* stream) {
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
                      {lse, ((int64_t)T + 1) * 4}};
  const Mem ins[] = {{logits, (int64_t)T * num_experts * dtype_bytes(dtype)}, {mask, T}};
  if (any_overlap(outs, ins))
    return op_fail(MOE_ERR_SHAPE,
                   "route: outputs and workspace must not overlap the inputs or each other");
  const RouteArgs a{logits, mask, T, num_experts, top_k, renormalize != 0, route_groups(T), topk_ids,
                    topk_weights, counts, balance, z, lse, ws};
  const auto s = (hipStream_t)stream;
  MOE_OP_HIP(dtype == kBf16   ? launch_route_any<kBf16>(a, s)
             : dtype == kFp16 ? launch_route_any<kFp16>(a, s)
                              : launch_route_any<kFp32>(a, s),
             "route");
  return MOE_OK;
}

int moe_route_backward_v1(const void* logits, int32_t T, int32_t num_experts, int32_t dtype,
                          int32_t top_k, int32_t renormalize, const int32_t* topk_ids,
                          const float* topk_weights, const int32_t* counts, const float* lse,
                          const float* dweights, const float* dbalance, const float* dz,
                          void* dlogits, void* stream) {
  const int rc = check_route("route backward", T, num_experts, dtype, top_k);
  if (rc) return rc;
  if (T == 0) return MOE_OK;
  if (!logits || !topk_ids || !topk_weights || !counts || !lse || !dlogits)
    return op_fail(MOE_ERR_NULL, "route backward: NULL pointer");
  const int64_t S = (int64_t)T * top_k, nl = (int64_t)T * num_experts * dtype_bytes(dtype);
  const Mem outs[] = {{dlogits, nl}};
  const Mem ins[] = {{logits, nl}, {topk_ids, S * 4}, {topk_weights, S * 4},
                     {counts, (int64_t)num_experts * 4}, {lse, ((int64_t)T + 1) * 4},
                     {dweights, S * 4}, {dbalance, 4}, {dz, 4}};
  if (any_overlap(outs, ins))
    return op_fail(MOE_ERR_SHAPE, "route backward: dlogits must not overlap the inputs");
  const RouteGradArgs a{logits, T, num_experts, top_k, renormalize != 0, topk_ids, topk_weights,
                        counts, lse, dweights, dbalance, dz, dlogits};
  const auto s = (hipStream_t)stream;
  MOE_OP_HIP(dtype == kBf16   ? launch_backward_any<kBf16>(a, s)
             : dtype == kFp16 ? launch_backward_any<kFp16>(a, s)
                              : launch_backward_any<kFp32>(a, s),
             "route backward");
  return MOE_OK;
}

}  // extern "C"
