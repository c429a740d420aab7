// Group-limited routing of tokens to experts, forward and backward.
//
//   s_e = sigmoid(l_e) or softmax(l)_e over all E experts, c_e = s_e + bias_e (without a bias the experts' order is that of the
//   logits, which s follows); a group's score is the sum of its one or two best c; the top_groups best groups stay, of their
//   experts the K best are taken, and w_k = scale * s_k / (sum_j s_j + 1e-20) (or scale * s_k).
//   With g_k = scale * dw_k and D = sum_j s_j + 1e-20: ds_k = g_k / D - (sum_j g_j s_j) / D^2 (or g_k), and
//   dl_e = ds_e s_e (1 - s_e) at the experts taken, or s_e (ds_e - sum_j ds_j s_j) for every e of a softmax.
//
// A logit of -inf closes its expert: it is never taken, slots beyond the open experts get index -1 and score 0, and a group of
// closed experts comes behind all others.  NaN ranks as -inf; the first of equals is taken.
//
// What is selected must not depend on how an exponential was rounded, so the order is that of exact arithmetic as far as 64 bits
// tell.  A warp selects by 32-bit keys, and wherever two neighbours of that order are nearer to each other than the keys' error
// (a fraction of a percent of rows) it does the row again in 64 bits; equal logits under equal biases are equal, not near.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

#include "smoe_b200.h"

namespace smoe {

constexpr int kGrWarps = 8;
__host__ __device__ constexpr int gr_warps(int per) { return per > 8 ? kGrWarps / 2 : kGrWarps; }      // of a block, by their memory
constexpr float kGrEps = 1e-20f;
constexpr uint32_t kAll = 0xffffffffu;

struct GroupRoutingArgs {
  const void* logits;
  const float* bias;       // or null
  int64_t T;
  int E, K, groups, top_groups, group_score;
  int softmax, normalize;
  float scale;
  float* scores;
  int* idx;
  int group_size;
  int group_lanes;         // lanes that hold a group's experts, if they hold no others and are a power of two, else 0
};

__device__ __forceinline__ float gr_logit(const float* p, size_t i) { return p[i]; }
__device__ __forceinline__ float gr_logit(const __nv_bfloat16* p, size_t i) { return __bfloat162float(p[i]); }

// floats as unsigned numbers of the same order, -inf above 0: 0 is left for "closed"
__device__ __forceinline__ uint32_t gr_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float gr_unkey(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
// finite, NaN as the lowest; zeros of either sign are one value
__device__ __forceinline__ double gr_rank(double x) { return x != x ? -DBL_MAX : fmin(fmax(x, -DBL_MAX), DBL_MAX) + 0.0; }

template <typename V>
__device__ __forceinline__ void gr_top2(V x, V& a, V& b) {      // a >= b: the two best
  if (x > a) {
    b = a;
    a = x;
  } else if (x > b) {
    b = x;
  }
}

__device__ __forceinline__ uint32_t gr_max(uint32_t k) {
  uint32_t r;
  asm volatile("redux.sync.max.u32 %0, %1, 0xffffffff;" : "=r"(r) : "r"(k));
  return r;
}
__device__ __forceinline__ uint32_t gr_min(uint32_t k) {
  uint32_t r;
  asm volatile("redux.sync.min.u32 %0, %1, 0xffffffff;" : "=r"(r) : "r"(k));
  return r;
}
// doubles as unsigned numbers of the same order, 0 left for "closed"
__device__ __forceinline__ unsigned long long gr_key(double x) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(x);
  return b ^ ((unsigned long long)((long long)b >> 63) | 0x8000000000000000ull);
}

// A lane's experts are lane * PER + i: the first lane of several with the same key holds the lowest index.
// The whole selection of one row in 64 bits -> lane k's expert, -1 beyond the open ones.  mine: 32 * PER doubles of the warp's.
template <int PER, typename L>
__device__ __noinline__ int gr_select64(const GroupRoutingArgs& a, const L* row, double* mine) {
  const int lane = threadIdx.x & 31, E = a.E;
  double top = -INFINITY, sum = 0;
  if (a.softmax) {
    for (int e = lane; e < E; e += 32) top = fmax(top, (double)gr_logit(row, e));
    for (int d = 16; d > 0; d >>= 1) top = fmax(top, __shfl_xor_sync(kAll, top, d));
    for (int i = 0; i < PER; ++i) {
      const double x = lane * PER + i < E ? (double)gr_logit(row, lane * PER + i) : -INFINITY;
      if (x != -INFINITY) sum += exp(x - top);
    }
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kAll, sum, d);
  }
  unsigned long long key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane * PER + i;
    const double x = e < E ? (double)gr_logit(row, e) : -INFINITY;
    key[i] = 0;
    double c = -INFINITY;
    if (x != -INFINITY) {
      const double s = a.softmax ? exp(x - top) / sum : 1.0 / (1.0 + exp(-x));
      const double order = gr_rank(a.bias ? s + (double)a.bias[e] : x);      // without a bias the logits say it
      key[i] = gr_key(order);
      c = a.bias || a.group_score == 1 ? order : gr_rank(s);
    }
    if (a.groups > 1) mine[e] = c;
  }
  if (a.groups > 1) {
    const int n = E / a.groups;
    __syncwarp();
    double p = -INFINITY, q = -INFINITY;                       // of group `lane`
    if (lane < a.groups) {
      int j = lane % n;
      for (int i = 0; i < n; ++i) {
        gr_top2(mine[lane * n + j], p, q);
        if (++j == n) j = 0;
      }
    }
    __syncwarp();
    const double score = (a.group_score > 1 && q != -INFINITY ? p + q : p) + 0.0;
    const unsigned long long g_key = p != -INFINITY ? gr_key(score) : 0ull;
    int ahead = 0;
    for (int h = 0; h < a.groups; ++h) {
      const unsigned long long o = __shfl_sync(kAll, g_key, h);
      ahead += o > g_key || (o == g_key && h < lane);
    }
    const uint32_t kept = __ballot_sync(kAll, lane < a.groups && ahead < a.top_groups);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane * PER + i;
      if (e >= E || !((kept >> (e / n)) & 1)) key[i] = 0;
    }
  }
  int sel = -1;
  for (int k = 0; k < a.K; ++k) {
    unsigned long long best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
    const uint32_t hi = gr_max((uint32_t)(best >> 32));
    const bool first = (uint32_t)(best >> 32) == hi;
    const uint32_t lo = gr_max(first ? (uint32_t)best : 0u);
    if ((hi | lo) == 0) break;
    const int from = __ffs(__ballot_sync(kAll, first && (uint32_t)best == lo)) - 1;
    const int e = __shfl_sync(kAll, lane * PER + at, from);
    if (lane == k) sel = e;
    if (lane == from) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i == at) key[i] = 0;
    }
  }
  return sel;
}

// PER neighbouring logits from row + lane * PER on; a lane beyond E has -inf
template <int PER>
__device__ __forceinline__ void gr_load(const float* row, int E, int lane, bool wide, float (&x)[PER]) {
  constexpr int V = PER % 4 == 0 ? 4 : PER % 2 == 0 ? 2 : 1;
  if (wide && V > 1) {
#pragma unroll
    for (int i = 0; i < PER; i += V) {
      if (lane * PER + i < E) {
        if (V == 4) {
          const float4 v = *reinterpret_cast<const float4*>(row + lane * PER + i);
          x[i] = v.x; x[i + 1 < PER ? i + 1 : 0] = v.y; x[i + 2 < PER ? i + 2 : 0] = v.z; x[i + 3 < PER ? i + 3 : 0] = v.w;
        } else {
          const float2 v = *reinterpret_cast<const float2*>(row + lane * PER + i);
          x[i] = v.x; x[i + 1 < PER ? i + 1 : 0] = v.y;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane * PER + i < E) x[i] = row[lane * PER + i];
  }
}
template <int PER>
__device__ __forceinline__ void gr_load(const __nv_bfloat16* row, int E, int lane, bool wide, float (&x)[PER]) {
  constexpr int V = PER % 8 == 0 ? 8 : PER % 4 == 0 ? 4 : PER % 2 == 0 ? 2 : 1;
  if (wide && V > 1) {
#pragma unroll
    for (int i = 0; i < PER; i += V) {
      if (lane * PER + i < E) {
        uint32_t w[4];
        if (V == 8) {
          const uint4 v = *reinterpret_cast<const uint4*>(row + lane * PER + i);
          w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else if (V == 4) {
          const uint2 v = *reinterpret_cast<const uint2*>(row + lane * PER + i);
          w[0] = v.x; w[1] = v.y;
        } else {
          w[0] = *reinterpret_cast<const uint32_t*>(row + lane * PER + i);
        }
#pragma unroll
        for (int j = 0; j < V; ++j)
          x[i + j < PER ? i + j : 0] = __uint_as_float((j & 1) ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane * PER + i < E) x[i] = __bfloat162float(row[lane * PER + i]);
  }
}

// What a comparison of two keys may be off by.  A score is an exponential of 2 ulp, its argument's rounding and a quotient: less
// than 4e-7 of the largest score, and in a softmax the sum's rounding, up to 36 x 2^-24 over 1024 experts, which shifts the scores
// against the biases; of each of the two.  c adds a rounding of its own.
__device__ __forceinline__ float gr_near(float slack, float c) { return slack + 3e-7f * fabsf(c); }

__device__ __forceinline__ float gr_max(float x) {           // over the warp, a number before a NaN
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float gr_exp(float x) {           // 2 ulp and the rounding of x log2(e)
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}
__device__ __forceinline__ float gr_inverse(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A lane's open experts, best first: `head` is the key of the best one left, `next` its place, pop takes it away
template <int PER>
struct GrList {                                              // up to 8: sorted once, a step moves up
  uint32_t key[PER];
  int at[PER];
  __device__ __forceinline__ void fill(const uint32_t (&k)[PER]) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      key[i] = k[i];
      at[i] = i;
    }
#pragma unroll
    for (int round = 0; round < PER; ++round)                 // neighbours change places only if the later one is larger: the
#pragma unroll                                                // first of equals stays first
      for (int i = round & 1; i + 1 < PER; i += 2) {
        const bool swap = key[i + 1] > key[i];
        const int t = at[i];
        at[i] = swap ? at[i + 1] : at[i];
        at[i + 1] = swap ? t : at[i + 1];
        const uint32_t hi = max(key[i], key[i + 1]), lo = min(key[i], key[i + 1]);
        key[i] = hi;
        key[i + 1] = lo;
      }
  }
  __device__ __forceinline__ uint32_t head() const { return key[0]; }
  __device__ __forceinline__ int place() const { return at[0]; }
  __device__ __forceinline__ void pop(bool mine) {
#pragma unroll
    for (int i = 0; i + 1 < PER; ++i) {
      key[i] = mine ? key[i + 1] : key[i];
      at[i] = mine ? at[i + 1] : at[i];
    }
    key[PER - 1] = mine ? 0u : key[PER - 1];
  }
};
template <>
struct GrList<32> {                                          // a sort would cost more than finding the next best K times
  uint32_t key[32], best;
  int where;
  __device__ __forceinline__ void look() {
    best = 0;
    where = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (key[i] > best) {
        best = key[i];
        where = i;
      }
  }
  __device__ __forceinline__ void fill(const uint32_t (&k)[32]) {
#pragma unroll
    for (int i = 0; i < 32; ++i) key[i] = k[i];
    look();
  }
  __device__ __forceinline__ uint32_t head() const { return best; }
  __device__ __forceinline__ int place() const { return where; }
  __device__ __forceinline__ void pop(bool mine) {
    if (mine) {
#pragma unroll
      for (int i = 0; i < 32; ++i) key[i] = i == where ? 0u : key[i];
      look();
    }
  }
};

// A warp a row.  The keys are those of c, or without a bias of the logits: then the order of experts is exact.  K times the largest
// of the lanes' best keys (one reduction instruction) and its first lane.  Bound by the issue of instructions (73 % of the slots, the
// integer pipe 68 %), a small batch by their latency: 64 x 256 3.7 us, 16384 x 128 19, x 256 28, K = 8 of 4 groups in 8.
template <int PER, bool GROUPS, typename L>
__global__ void __launch_bounds__(32 * gr_warps(PER)) group_routing_kernel(const __grid_constant__ GroupRoutingArgs a) {
  extern __shared__ double s_rank[];                          // GROUPS: 32 * PER for each warp
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = a.E;
  const int64_t r = blockIdx.x * (int64_t)gr_warps(PER) + warp;
  if (r >= a.T) return;
  const L* row = (const L*)a.logits + r * E;
  const bool wide = E % PER == 0 && (reinterpret_cast<uintptr_t>(row) & (PER * sizeof(L) >= 16 ? 15 : PER * sizeof(L) - 1)) == 0;
  float x[PER], bias[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    x[i] = -INFINITY;
    bias[i] = 0.f;
  }
  gr_load(row, E, lane, wide, x);
  if (a.bias) gr_load(a.bias, E, lane, E % PER == 0 && (reinterpret_cast<uintptr_t>(a.bias) & (PER >= 4 ? 15 : 4 * PER - 1)) == 0, bias);
  const bool scores_rank = a.bias || (GROUPS && a.group_score > 1);      // else the logits tell
  float top = 0.f, sum = 1.f, slack = 1e-6f;
  if (a.softmax) {
    top = x[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) top = fmaxf(top, x[i]);
    top = gr_max(top);
    sum = 0.f;
    if (top != -INFINITY) {
#pragma unroll
      for (int i = 0; i < PER; ++i) sum += expf(x[i] - top);
    }
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kAll, sum, d);
    slack = 6e-6f / sum;
  }
  uint32_t key[PER];
  float c[PER];
  const float factor = a.softmax ? gr_inverse(sum) : 1.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    c[i] = x[i];
    if (scores_rank) c[i] = (a.softmax ? gr_exp(x[i] - top) * factor : gr_inverse(1.f + gr_exp(-x[i]))) + bias[i];
    const float o = (a.bias ? c[i] : x[i]) + 0.f;             // zeros of either sign are one value
    key[i] = x[i] == -INFINITY ? 0u : o == o ? gr_key(o) : 1u;
    // (as gr_rank: NaN and what a bias of -inf leaves are the lowest of numbers, only a closed expert is none)
    if (GROUPS) c[i] = x[i] == -INFINITY ? -INFINITY : fmaxf(c[i], -FLT_MAX);
  }
  bool sure = true;                                           // the order so far is beyond doubt
  if (GROUPS) {
    const int n = a.group_size;
    float p = -INFINITY, q = -INFINITY;                       // the two best of group `lane`
    if (a.group_lanes) {                                      // lanes of a group, a power of two; each lane in one group
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        q = fmaxf(q, fminf(p, c[i]));
        p = fmaxf(p, c[i]);
      }
      for (int d = 1; d < a.group_lanes; d <<= 1) {
        const float op = __shfl_xor_sync(kAll, p, d), oq = __shfl_xor_sync(kAll, q, d);
        q = fmaxf(fmaxf(q, oq), fminf(p, op));
        p = fmaxf(p, op);
      }
      p = __shfl_sync(kAll, p, lane * a.group_lanes & 31);
      q = __shfl_sync(kAll, q, lane * a.group_lanes & 31);
    } else {
      float* mine = reinterpret_cast<float*>(s_rank + warp * PER * 32);
#pragma unroll
      for (int i = 0; i < PER; ++i) mine[lane * PER + i] = c[i];
      __syncwarp();
      if (lane < a.groups) {
        int j = lane % n;                                     // lanes read different banks
        for (int i = 0; i < n; ++i) {
          gr_top2(mine[lane * n + j], p, q);
          if (++j == n) j = 0;
        }
      }
    }
    const float score = (a.group_score > 1 && q != -INFINITY ? p + q : p) + 0.f;
    const uint32_t g_key = lane < a.groups && p != -INFINITY ? gr_key(score) : 0u;
    int ahead = 0;
    for (int h = 0; h < a.groups; ++h) {
      const uint32_t o = __shfl_sync(kAll, g_key, h);
      ahead += o > g_key || (o == g_key && h < lane);
    }
    const bool in = lane < a.groups && ahead < a.top_groups;
    const uint32_t kept = __ballot_sync(kAll, in);
    // Each group's score may be off by what its terms were rounded by, and those may cancel: the least of those kept, less its own
    // error, against the largest left out, with its own.  (A closed one is kept only where no open one stays out.)  Logits are
    // exact, but the lowest of them is what stands for NaN.
    const bool two = a.group_score > 1 && q != -INFINITY;
    const float off = scores_rank ? gr_near(slack, 2.f * (fabsf(p) + (two ? fabsf(q) : 0.f))) : 0.f;
    const uint32_t least = gr_min(in ? gr_key(fmaxf(score - off, -INFINITY)) : kAll);         // fmaxf: no NaN of infinities
    // (a sum that overflows is one of two lowest numbers, and lies below every other)
    const uint32_t most = gr_max(in || g_key == 0 ? 0u : gr_key(score == -INFINITY ? -3.4e38f : score + off));
    if (most) {
      const float lo = gr_unkey(least);
      sure = lo > gr_unkey(most) || (!scores_rank && lo > -FLT_MAX);
    }
    if (a.group_lanes) {
      const bool stay = (kept >> (lane / a.group_lanes)) & 1;
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = stay ? key[i] : 0u;
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int e = lane * PER + i;
        if (e >= E || !((kept >> (e / n)) & 1)) key[i] = 0u;
      }
    }
  }
  int sel = -1;
  if (sure) {
    GrList<PER> list;
    list.fill(key);
    uint32_t took = 0, spare = 0;
    int other = -1;
    for (int k = 0; k < a.K; ++k) {
      const uint32_t m = gr_max(list.head());
      const int from = __ffs(__ballot_sync(kAll, list.head() == m)) - 1;
      const int e = __shfl_sync(kAll, lane * PER + list.place(), from);
      if (lane == k) {
        took = m;
        sel = m ? e : -1;
      }
      list.pop(lane == from);
    }
    if (a.bias) {
      // Each of those taken against the one before it, and the first that stays out against the last: a distance that the keys'
      // error could hide is no order, unless both are equal by input and their order that of their indices.  (Equals across
      // the border go the other way: how many there are, this does not know.)
      spare = gr_max(list.head());
      const uint32_t after = __shfl_down_sync(kAll, took, 1);
      other = __shfl_down_sync(kAll, sel, 1);
      const uint32_t low = lane == a.K - 1 ? spare : after;
      bool doubt = false;
      if (lane < a.K && took && low) {
        const float hi = gr_unkey(took), lo = gr_unkey(low);
        doubt = !(hi - lo > gr_near(slack, fabsf(hi) + fabsf(lo)));
        if (doubt && lane < a.K - 1) doubt = !(gr_logit(row, sel) == gr_logit(row, other) && a.bias[sel] == a.bias[other]);
      }
      sure = !__any_sync(kAll, doubt);
    }
  }
  __syncwarp();
  if (!sure) sel = gr_select64<PER, L>(a, row, s_rank + warp * PER * 32);

  float s = 0.f;
  if (sel >= 0) {
    const float v = gr_logit(row, sel);
    s = a.softmax ? expf(v - top) / sum : 1.f / (1.f + expf(-v));
  }
  float d = s;
  for (int i = 16; i > 0; i >>= 1) d += __shfl_xor_sync(kAll, d, i);
  if (lane < a.K) {
    a.scores[r * a.K + lane] = a.scale * (a.normalize ? s / (d + kGrEps) : s);
    a.idx[r * a.K + lane] = sel;
  }
}

__device__ __forceinline__ void gr_store(float* p, size_t i, float v) { p[i] = v; }
__device__ __forceinline__ void gr_store(__nv_bfloat16* p, size_t i, float v) { p[i] = __float2bfloat16_rn(v); }

// A warp a row, bound by the issue of instructions (73 % of the slots) where there are many rows, 4 MB written in 8.7 us for 16384 x 128
// in bf16, and by their latency where there are few.
template <typename L>
__global__ void __launch_bounds__(32 * kGrWarps)
group_routing_bwd_kernel(const L* __restrict__ logits, const int* __restrict__ idx, const float* __restrict__ dscores, int64_t T,
                         int E, int K, int softmax, int normalize, float scale, L* __restrict__ dlogits) {
  const int lane = threadIdx.x & 31;
  const int64_t r = blockIdx.x * (int64_t)kGrWarps + (threadIdx.x >> 5);
  if (r >= T) return;
  const L* row = logits + r * E;
  L* out = dlogits + r * E;
  float top = 0.f, inv = 1.f;
  if (softmax) {
    top = -INFINITY;
    for (int e = lane; e < E; e += 32) top = fmaxf(top, gr_logit(row, e));
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, d));
    float sum = 0.f;
    if (top != -INFINITY)
      for (int e = lane; e < E; e += 32) sum += expf(gr_logit(row, e) - top);
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kAll, sum, d);
    inv = 1.f / sum;
  }
  int sel = lane < K ? idx[r * K + lane] : -1;
  if (sel >= E) sel = -1;
  float s = 0.f, g = 0.f, slope = 0.f;                   // slope: s (1 - s) of a sigmoid
  if (sel >= 0) {
    const float x = gr_logit(row, sel);
    if (softmax) {
      s = expf(x - top) * inv;
    } else {
      s = 1.f / (1.f + expf(-x));
      const float t = expf(-fabsf(x));
      slope = t / ((1.f + t) * (1.f + t));
    }
    g = scale * dscores[r * K + lane];
  }
  float total = s, dot = g * s;
  for (int d = 16; d > 0; d >>= 1) {
    total += __shfl_xor_sync(kAll, total, d);
    dot += __shfl_xor_sync(kAll, dot, d);
  }
  float ds = g, all = dot;                               // all: sum_j ds_j s_j
  if (normalize) {
    // g_k / D - dot / D^2 = (sum_j s_j (g_k - g_j) + eps g_k) / D^2, and sum_j ds_j s_j = eps dot / D^2, with eps what the 1e-20 adds to
    // the f32 sum: where the g are alike (one expert a token) the left sides are differences of rounded equals
    const float sum = total;
    total += kGrEps;
    const float eps = total - sum;
    float diff = eps * g;
    for (int j = 0; j < K; ++j) diff = fmaf(__shfl_sync(kAll, s, j), g - __shfl_sync(kAll, g, j), diff);
    ds = diff / total / total;
    all = eps * dot / total / total;
  }
  for (int e = lane; e < E; e += 32)
    gr_store(out, e, softmax && top != -INFINITY ? -all * (expf(gr_logit(row, e) - top) * inv) : 0.f);
  __syncwarp();
  if (sel >= 0) gr_store(out, sel, softmax ? s * (ds - all) : ds * slope);
}

}  // namespace smoe

using namespace smoe;

extern "C" {

static int group_routing_sizes(int64_t T, int64_t E, int64_t K) {
  return T < 0 || E <= 0 || E > 1024 || K <= 0 || K > 32 || K > E ? SMOE_ERR_SHAPE : SMOE_OK;
}

int smoe_group_routing(const void* logits, int bf16, const float* bias, int64_t T, int64_t E, int64_t K, int64_t groups,
                       int64_t top_groups, int group_score, int softmax, int normalize, float scale, float* scores, int32_t* idx,
                       void* stream) {
  if (group_routing_sizes(T, E, K)) return SMOE_ERR_SHAPE;
  if (groups <= 0 || groups > 32 || E % groups || top_groups <= 0 || top_groups > groups || K > top_groups * (E / groups))
    return SMOE_ERR_SHAPE;
  if (group_score != 1 && group_score != 2) return SMOE_ERR_ARG;
  if (T == 0) return SMOE_OK;
  if (!logits || !scores || !idx) return SMOE_ERR_ARG;
  GroupRoutingArgs a{logits, bias, T, (int)E, (int)K, (int)groups, (int)top_groups, group_score, softmax, normalize, scale, scores,
                     idx, (int)(E / groups), 0};
  if (top_groups == groups) a.groups = a.top_groups = 1;       // every group stays
  const int per = E <= 32 ? 1 : E <= 64 ? 2 : E <= 128 ? 4 : E <= 256 ? 8 : 32;
  const int lanes = a.group_size / per;
  if (a.group_size % per == 0 && (lanes & (lanes - 1)) == 0) a.group_lanes = lanes;
#define SMOE_PER(G, L)                            \
  (per == 1   ? group_routing_kernel<1, G, L>     \
   : per == 2 ? group_routing_kernel<2, G, L>     \
   : per == 4 ? group_routing_kernel<4, G, L>     \
   : per == 8 ? group_routing_kernel<8, G, L>     \
              : group_routing_kernel<32, G, L>)
  auto kern = a.groups > 1 ? (bf16 ? SMOE_PER(true, __nv_bfloat16) : SMOE_PER(true, float))
                           : (bf16 ? SMOE_PER(false, __nv_bfloat16) : SMOE_PER(false, float));
#undef SMOE_PER
  const int warps = gr_warps(per);
  const size_t smem = a.groups > 1 ? sizeof(double) * warps * 32 * per : 0;
  kern<<<(unsigned)((T + warps - 1) / warps), 32 * warps, smem, (cudaStream_t)stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? SMOE_OK : SMOE_ERR_LAUNCH;
}

int smoe_group_routing_bwd(const void* logits, int bf16, const int32_t* idx, const float* dscores, int64_t T, int64_t E, int64_t K,
                           int softmax, int normalize, float scale, void* dlogits, void* stream) {
  if (group_routing_sizes(T, E, K)) return SMOE_ERR_SHAPE;
  if (T == 0) return SMOE_OK;
  if (!logits || !idx || !dscores || !dlogits) return SMOE_ERR_ARG;
  const unsigned grid = (unsigned)((T + kGrWarps - 1) / kGrWarps);
  if (bf16)
    group_routing_bwd_kernel<__nv_bfloat16><<<grid, 32 * kGrWarps, 0, (cudaStream_t)stream>>>(
        (const __nv_bfloat16*)logits, idx, dscores, T, (int)E, (int)K, softmax, normalize, scale, (__nv_bfloat16*)dlogits);
  else
    group_routing_bwd_kernel<float><<<grid, 32 * kGrWarps, 0, (cudaStream_t)stream>>>(
        (const float*)logits, idx, dscores, T, (int)E, (int)K, softmax, normalize, scale, (float*)dlogits);
  return cudaGetLastError() == cudaSuccess ? SMOE_OK : SMOE_ERR_LAUNCH;
}

}  // extern "C"
