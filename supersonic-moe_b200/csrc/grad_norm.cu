// The global norm of a list of gradients, and their clipping.
//
//   n = sqrt(sum over all tensors of the sum of g^2)      c = min(1, max_norm / (n + 1e-6))      out = c g
//
// One launch adds up squares, one more scales: the list travels in the launch's parameters, so that a captured graph keeps it and
// nothing is uploaded, and every block of the second launch adds the first one's partial sums up again instead of waiting for a
// kernel between the two.  Bound by HBM: f32 sums of eight values, f64 beyond, cost less than their loads.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "host.h"
#include "ptx.cuh"
#include "quant_groups.cuh"
#include "smoe_b200.h"

namespace smoe {

constexpr int kGradThreads = 256;
constexpr int kGradBlocks = 4;               // a block an SM takes at a time
constexpr int kGradStep = kGradThreads * 8;  // values of a block's step: eight a thread

// A list of tensors; `first` counts pieces of `chunk` values.  Small lists travel as small parameters.
template <int N>
struct GradList {
  const void* in[N];
  void* out[N];
  int64_t n[N];
  int first[N + 1];
  uint8_t in_f32[N], out_f32[N], vec[N];     // vec: they start on 16 bytes (the output where there is one)
  int count, chunk;
};

template <int N>
struct GradPiece {
  int i;
  int64_t from, to;                          // values of tensor i
  __device__ __forceinline__ GradPiece(const GradList<N>& l, int piece) {
    int lo = 0, hi = l.count - 1;            // the last one that begins at or before it, which is not empty
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (l.first[mid] <= piece) lo = mid; else hi = mid - 1;
    }
    i = lo;
    from = (int64_t)(piece - l.first[i]) * l.chunk;
    to = min(from + l.chunk, l.n[i]);
  }
};

__device__ __forceinline__ void grad_load8(const void* base, bool f32, int64_t at, float (&f)[8]) {
  if (f32) {
    const float4* p = reinterpret_cast<const float4*>((const float*)base + at);
    const float4 a = p[0], b = p[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    bf16x8_to_f32(*reinterpret_cast<const uint4*>((const uint16_t*)base + at), f);
  }
}
__device__ __forceinline__ float grad_load1(const void* base, bool f32, int64_t at) {
  return f32 ? ((const float*)base)[at] : __uint_as_float((uint32_t)((const uint16_t*)base)[at] << 16);
}
__device__ __forceinline__ void grad_store8(void* base, bool f32, int64_t at, const float (&f)[8]) {
  if (f32) {
    float4* p = reinterpret_cast<float4*>((float*)base + at);
    p[0] = make_float4(f[0], f[1], f[2], f[3]);
    p[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *reinterpret_cast<uint4*>((uint16_t*)base + at) =
        make_uint4(q_bf16x2(f[0], f[1]), q_bf16x2(f[2], f[3]), q_bf16x2(f[4], f[5]), q_bf16x2(f[6], f[7]));
  }
}
__device__ __forceinline__ void grad_store1(void* base, bool f32, int64_t at, float v) {
  if (f32) ((float*)base)[at] = v;
  else ((__nv_bfloat16*)base)[at] = __float2bfloat16_rn(v);
}

// Squares of eight values: in f32 where that neither overflows nor loses what it drops, else in f64
__device__ __forceinline__ double grad_squares8(const float (&f)[8]) {
  float a = 0.f, b = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    a = fmaf(f[i], f[i], a);
    b = fmaf(f[i + 1], f[i + 1], b);
  }
  const float s = a + b;
  if (s > 1e-25f && s < 1e30f) return s;     // (a square below 1e-38 is no more than 1e-13 of such a sum)
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) d = fma((double)f[i], (double)f[i], d);
  return d;
}

// every thread gets the sum, in one order; `shared` holds one value a warp
__device__ __forceinline__ double grad_block_sum(double s, double* shared) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int i = 0; i < kGradThreads / 32; ++i) s += shared[i];
  return s;
}

// partial[block]: sum of the squares of the pieces block, block + blocks, ...
template <int N>
__global__ void __launch_bounds__(kGradThreads, kGradBlocks)
grad_squares_kernel(const __grid_constant__ GradList<N> l, double* partial) {
  __shared__ double sums[kGradThreads / 32];
  next_kernel_may_start();                   // (which waits for this one's end)
  double s = 0.0;
  const int pieces = l.first[l.count];
  for (int piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
    const GradPiece<N> p(l, piece);
    const void* in = l.in[p.i];
    const bool f32 = l.in_f32[p.i];
    if (l.vec[p.i]) {
      int64_t at = p.from + threadIdx.x * 8;
      for (; at + 3 * kGradThreads * 8 + 8 <= p.to; at += 4 * kGradThreads * 8) {
        float f[4][8];
#pragma unroll
        for (int u = 0; u < 4; ++u) grad_load8(in, f32, at + u * kGradThreads * 8, f[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u) s += grad_squares8(f[u]);
      }
      for (; at + 8 <= p.to; at += kGradThreads * 8) {
        float f[8];
        grad_load8(in, f32, at, f);
        s += grad_squares8(f);
      }
      if (at < p.to)                         // fewer than eight are left, to one thread
        for (int64_t j = at; j < p.to; ++j) {
          const double v = grad_load1(in, f32, j);
          s = fma(v, v, s);
        }
    } else {
      for (int64_t j = p.from + threadIdx.x; j < p.to; j += kGradThreads) {
        const double v = grad_load1(in, f32, j);
        s = fma(v, v, s);
      }
    }
  }
  s = grad_block_sum(s, sums);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// (a kernel that begins while the one before ends: no pointer here promises memory that nobody writes meanwhile)
__device__ __forceinline__ double grad_total(const double* partial, int n, double* shared) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kGradThreads) s += partial[i];
  return grad_block_sum(s, shared);
}

__global__ void __launch_bounds__(kGradThreads) grad_norm_kernel(const double* partial, int n, float* norm) {
  __shared__ double sums[kGradThreads / 32];
  wait_for_kernel_before();
  const double s = grad_total(partial, n, sums);
  if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// Pieces from the last one on: what the first launch read last is what L2 still holds.
template <int N>
__global__ void __launch_bounds__(kGradThreads, kGradBlocks)
grad_scale_kernel(const __grid_constant__ GradList<N> l, const double* partial, int n_partial,
                  const float* given, double max_norm, float* norm) {
  __shared__ double sums[kGradThreads / 32];
  wait_for_kernel_before();
  const double total = given ? (double)*given : sqrt(grad_total(partial, n_partial, sums));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
  const double ratio = max_norm / (total + 1e-6);
  const float c = ratio < 1.0 || ratio != ratio ? (float)ratio : 1.f;
  const int pieces = l.first[l.count];
  for (int piece = pieces - 1 - blockIdx.x; piece >= 0; piece -= gridDim.x) {
    const GradPiece<N> p(l, piece);
    const void* in = l.in[p.i];
    void* out = l.out[p.i];
    if (in == out && c == 1.f) continue;     // they are there already
    const bool f32 = l.in_f32[p.i], o32 = l.out_f32[p.i];
    if (l.vec[p.i]) {
      int64_t at = p.from + threadIdx.x * 8;
      for (; at + kGradThreads * 8 + 8 <= p.to; at += 2 * kGradThreads * 8) {
        float f[2][8];
#pragma unroll
        for (int u = 0; u < 2; ++u) grad_load8(in, f32, at + u * kGradThreads * 8, f[u]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[u][i] *= c;
          grad_store8(out, o32, at + u * kGradThreads * 8, f[u]);
        }
      }
      for (; at + 8 <= p.to; at += kGradThreads * 8) {
        float f[8];
        grad_load8(in, f32, at, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= c;
        grad_store8(out, o32, at, f);
      }
      if (at < p.to)
        for (int64_t j = at; j < p.to; ++j) grad_store1(out, o32, j, grad_load1(in, f32, j) * c);
    } else {
      for (int64_t j = p.from + threadIdx.x; j < p.to; j += kGradThreads) grad_store1(out, o32, j, grad_load1(in, f32, j) * c);
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
constexpr int kGradSmall = 48, kGradLarge = 640;      // tensors of a launch

static int64_t grad_chunk(int64_t total) {
  // some eight pieces a block, so that the blocks end together, of one step to 32
  const int64_t want = total / ((int64_t)sm_count() * kGradBlocks * 8) / kGradStep + 1;
  return (want < 32 ? want : 32) * kGradStep;
}

// blocks of a launch over the tensors [from, to): as many as there are pieces, or find room together
static int grad_blocks(const smoe_gradient* list, int64_t from, int64_t to, int64_t chunk) {
  int64_t pieces = 0;
  for (int64_t i = from; i < to; ++i) pieces += (list[i].numel + chunk - 1) / chunk;
  const int64_t most = (int64_t)sm_count() * kGradBlocks;
  return (int)(pieces < most ? pieces : most);
}

template <int N>
static void grad_fill(GradList<N>& l, const smoe_gradient* list, int64_t from, int64_t to, int64_t chunk, bool outs) {
  l.count = (int)(to - from);
  l.chunk = (int)chunk;
  int64_t pieces = 0;
  for (int64_t i = from; i < to; ++i) {
    const smoe_gradient& g = list[i];
    const int j = (int)(i - from);
    l.in[j] = g.grad;
    l.out[j] = g.out;
    l.n[j] = g.numel;
    l.first[j] = (int)pieces;
    l.in_f32[j] = g.grad_f32 != 0;
    l.out_f32[j] = g.out_f32 != 0;
    l.vec[j] = (((uintptr_t)g.grad | (outs ? (uintptr_t)g.out : 0)) & 15) == 0;
    pieces += (g.numel + chunk - 1) / chunk;
  }
  l.first[l.count] = (int)pieces;
}

struct GradCall {
  const smoe_gradient* list;
  int64_t count, chunk;
  double* partial;
  const float* given;
  double max_norm;
  float* norm;
  cudaStream_t stream;
};

template <int N>
static cudaError_t grad_launch(const GradCall& c, int64_t from, int64_t to, int blocks, bool scale, int at) {
  GradList<N> l;
  grad_fill(l, c.list, from, to, c.chunk, scale);
  if (scale)
    return launch_early(grad_scale_kernel<N>, blocks, kGradThreads, 0, 0, c.stream, l, (const double*)c.partial, at, c.given, c.max_norm,
                        from == 0 ? c.norm : nullptr);
  grad_squares_kernel<N><<<blocks, kGradThreads, 0, c.stream>>>(l, c.partial + at);
  return cudaGetLastError();
}
// All launches of one kind; returns the partial sums there are, or -1.  `scale`: from the last tensors on, with `n` sums.
static int grad_launches(const GradCall& c, bool scale, int n) {
  int at = scale ? n : 0;
  const int64_t groups = (c.count + kGradLarge - 1) / kGradLarge;
  for (int64_t k = 0; k < groups; ++k) {
    const int64_t from = (scale ? groups - 1 - k : k) * kGradLarge, to = from + kGradLarge < c.count ? from + kGradLarge : c.count;
    int blocks = grad_blocks(c.list, from, to, c.chunk);
    if (blocks == 0) blocks = 1;             // (all of them empty)
    const cudaError_t rc = to - from <= kGradSmall ? grad_launch<kGradSmall>(c, from, to, blocks, scale, at)
                                                   : grad_launch<kGradLarge>(c, from, to, blocks, scale, at);
    if (rc != cudaSuccess) return -1;
    if (!scale) at += blocks;
  }
  return at;
}

static int grad_check(const smoe_gradient* list, int64_t count, int64_t* total, bool outs) {
  if (count < 0 || count > (int64_t)1 << 20 || (count > 0 && !list)) return SMOE_ERR_ARG;
  *total = 0;
  for (int64_t i = 0; i < count; ++i) {
    const smoe_gradient& g = list[i];
    if (g.numel < 0 || g.numel > (int64_t)1 << 40) return SMOE_ERR_SHAPE;
    if (g.numel > 0 && (!g.grad || (outs && !g.out))) return SMOE_ERR_ARG;
    if (((uintptr_t)g.grad & (g.grad_f32 ? 3 : 1)) || (outs && ((uintptr_t)g.out & (g.out_f32 ? 3 : 1)))) return SMOE_ERR_ALIGN;
    *total += g.numel;
  }
  return *total / (32 * kGradStep) < (int64_t)1 << 30 ? SMOE_OK : SMOE_ERR_SHAPE;
}

}  // namespace smoe

using namespace smoe;

extern "C" {

int64_t smoe_gradient_workspace(int64_t count) {
  if (count < 0 || count > (int64_t)1 << 20) return -1;
  const int64_t groups = (count + kGradLarge - 1) / kGradLarge;
  return (groups > 0 ? groups : 1) * sm_count() * kGradBlocks * 8;
}

int smoe_gradient_norm(const smoe_gradient* list, int64_t count, float* norm, void* workspace, void* stream) {
  int64_t total;
  const int rc = grad_check(list, count, &total, false);
  if (rc) return rc;
  if (!norm || !workspace) return SMOE_ERR_ARG;
  const GradCall c{list, count, grad_chunk(total), (double*)workspace, nullptr, 0.0, norm, (cudaStream_t)stream};
  const int n = grad_launches(c, false, 0);
  if (n < 0) return SMOE_ERR_LAUNCH;
  return launch_early(grad_norm_kernel, 1, kGradThreads, 0, 0, c.stream, (const double*)c.partial, n, norm) == cudaSuccess ? SMOE_OK
                                                                                                                   : SMOE_ERR_LAUNCH;
}

int smoe_gradient_clip(const smoe_gradient* list, int64_t count, double max_norm, const float* given_norm, float* norm, void* workspace,
                       void* stream) {
  int64_t total;
  const int rc = grad_check(list, count, &total, true);
  if (rc) return rc;
  if (!(max_norm >= 0) || (!given_norm && (!norm || !workspace))) return SMOE_ERR_ARG;
  const GradCall c{list, count, grad_chunk(total), (double*)workspace, given_norm, max_norm, norm, (cudaStream_t)stream};
  int n = 0;
  if (!given_norm) {
    n = grad_launches(c, false, 0);
    if (n < 0) return SMOE_ERR_LAUNCH;
  }
  if (count == 0 && norm && !given_norm) {
    grad_norm_kernel<<<1, kGradThreads, 0, c.stream>>>(c.partial, 0, norm);
    return cudaGetLastError() == cudaSuccess ? SMOE_OK : SMOE_ERR_LAUNCH;
  }
  return grad_launches(c, true, n) < 0 ? SMOE_ERR_LAUNCH : SMOE_OK;
}

}  // extern "C"
