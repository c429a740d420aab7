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
__device__ __forceinline__ float gr_rank(float x) { return x != x ? -FLT_MAX : fminf(fmaxf(x, -FLT_MAX), FLT_MAX) + 0.f; }
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

// A lane's experts are lane * PER + i: the first lane of several with the same key holds the lowest index.
// The whole selection of one row in 64 bits -> lane k's expert, -1 beyond the open ones
template <int PER, typename L>
__device__ __noinline__ int gr_select64(const GroupRoutingArgs& a, const L* row) {
  const int lane = threadIdx.x & 31, E = a.E, n = E / a.groups;
  double c[PER], x[PER];
  uint32_t open = 0;
  double top = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane * PER + i;
    x[i] = e < E ? (double)gr_logit(row, e) : -INFINITY;
    if (e < E && x[i] != -INFINITY) open |= 1u << i;
    top = fmax(top, x[i]);
  }
  double sum = 0;
  if (a.softmax) {
    for (int d = 16; d > 0; d >>= 1) top = fmax(top, __shfl_xor_sync(kAll, top, d));
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if ((open >> i) & 1) sum += exp(x[i] - top);
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kAll, sum, d);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    c[i] = -DBL_MAX;
    if ((open >> i) & 1) {
      const double s = a.softmax ? exp(x[i] - top) / sum : 1.0 / (1.0 + exp(-x[i]));
      c[i] = a.bias ? s + (double)a.bias[lane * PER + i] : (a.groups > 1 && a.group_score > 1 ? s : x[i]);
      c[i] = gr_rank(c[i]);
      x[i] = a.bias ? c[i] : gr_rank(x[i]);                    // what the experts are ordered by
    }
  }
  if (a.groups > 1) {
    double mine = -INFINITY;
    bool any = false;                                          // of group `lane`
    for (int g = 0; g < a.groups; ++g) {
      double p = -INFINITY, q = -INFINITY;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int e = lane * PER + i;
        if (((open >> i) & 1) && e / n == g) gr_top2(c[i], p, q);
      }
      for (int d = 16; d > 0; d >>= 1) {
        const double op = __shfl_xor_sync(kAll, p, d), oq = __shfl_xor_sync(kAll, q, d);
        gr_top2(op, p, q);
        gr_top2(oq, p, q);
      }
      if (lane == g) {
        any = p != -INFINITY;
        mine = a.group_score > 1 && q != -INFINITY ? p + q : p;
      }
    }
    int ahead = 0;
    for (int h = 0; h < a.groups; ++h) {
      const double o = __shfl_sync(kAll, mine, h);
      const bool oa = __shfl_sync(kAll, (int)any, h);
      ahead += (oa && !any) || (oa == any && (o > mine || (o == mine && h < lane)));
    }
    const uint32_t kept = __ballot_sync(kAll, lane < a.groups && ahead < a.top_groups);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane * PER + i;
      if (e >= E || !((kept >> (e / n)) & 1)) open &= ~(1u << i);
    }
  }
  int sel = -1;
  for (int k = 0; k < a.K; ++k) {
    double v = 0;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (((open >> i) & 1) && (at == 0x7fffffff || x[i] > v)) {
        v = x[i];
        at = lane * PER + i;
      }
    for (int d = 16; d > 0; d >>= 1) {
      const double ov = __shfl_xor_sync(kAll, v, d);
      const int oat = __shfl_xor_sync(kAll, at, d);
      if (oat != 0x7fffffff && (at == 0x7fffffff || ov > v || (ov == v && oat < at))) {
        v = ov;
        at = oat;
      }
    }
    if (at == 0x7fffffff) break;
    if (lane == k) sel = at;
    if (at / PER == lane) open &= ~(1u << (at % PER));
  }
  return sel;
}

template <int PER, typename L>
__global__ void __launch_bounds__(32 * kGrWarps) group_routing_kernel(const GroupRoutingArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t r = blockIdx.x * (int64_t)kGrWarps + (threadIdx.x >> 5);
  if (r >= a.T) return;
  const L* row = (const L*)a.logits + r * a.E;
  const int sel = gr_select64<PER, L>(a, row);

  float top = 0.f, sum = 1.f;
  if (a.softmax) {
    top = -INFINITY;
    for (int e = lane; e < a.E; e += 32) top = fmaxf(top, gr_logit(row, e));
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, d));
    sum = 0.f;
    if (top != -INFINITY)
      for (int e = lane; e < a.E; e += 32) sum += expf(gr_logit(row, e) - top);
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kAll, sum, d);
  }
  float s = 0.f;
  if (sel >= 0) {
    const float x = gr_logit(row, sel);
    s = a.softmax ? expf(x - top) / sum : 1.f / (1.f + expf(-x));
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
  float s = 0.f, g = 0.f;
  if (sel >= 0) {
    const float x = gr_logit(row, sel);
    s = softmax ? expf(x - top) * inv : 1.f / (1.f + expf(-x));
    g = scale * dscores[r * K + lane];
  }
  float total = s, dot = g * s;
  for (int d = 16; d > 0; d >>= 1) {
    total += __shfl_xor_sync(kAll, total, d);
    dot += __shfl_xor_sync(kAll, dot, d);
  }
  float ds = g;
  if (normalize) {
    total += kGrEps;
    ds = (g - dot / total) / total;
  }
  float all = ds * s;                                    // sum_j ds_j s_j
  for (int d = 16; d > 0; d >>= 1) all += __shfl_xor_sync(kAll, all, d);
  for (int e = lane; e < E; e += 32)
    gr_store(out, e, softmax && top != -INFINITY ? -all * (expf(gr_logit(row, e) - top) * inv) : 0.f);
  __syncwarp();
  if (sel >= 0) gr_store(out, sel, softmax ? s * (ds - all) : ds * s * (1.f - s));
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
                     idx};
  if (top_groups == groups) a.groups = a.top_groups = 1;       // every group stays
  const unsigned grid = (unsigned)((T + kGrWarps - 1) / kGrWarps);
#define SMOE_PER(L)                            \
  (E <= 32    ? group_routing_kernel<1, L>     \
   : E <= 64  ? group_routing_kernel<2, L>     \
   : E <= 128 ? group_routing_kernel<4, L>     \
   : E <= 256 ? group_routing_kernel<8, L>     \
              : group_routing_kernel<32, L>)
  auto kern = bf16 ? SMOE_PER(__nv_bfloat16) : SMOE_PER(float);
#undef SMOE_PER
  kern<<<grid, 32 * kGrWarps, 0, (cudaStream_t)stream>>>(a);
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
