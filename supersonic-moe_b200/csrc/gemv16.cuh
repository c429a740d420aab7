// The product of gemm16.cuh for a handful of rows (single tokens): weights straight from memory into registers.
//
//   y[r, n] = sum_k x[r, k] w[e(r)][n, k]
//
// A warp computes two weight rows times up to four routed rows of their expert: 16 bytes of either a lane, exact products of bf16 added up
// in f32, then over the lanes.  Every SM reads weights from the first clock on, without tensor maps, rings, TMEM and the exchange of
// sums between CTAs, which cost the tensor-core kernel for few rows some 6 us.  Bound by the read of the weights.
#pragma once
#include "gemm16.cuh"

namespace smoe {

constexpr int kGemvRows = 4;               // routed rows of a warp
// weight rows of a warp (with four: one row of 1024 x 1024 2.5 -> 2.8 us, 8 of 128 experts of 1536 x 2048 10.2 -> 10.8)
constexpr int kGemvCols = 2;
constexpr int kGemvMost = 16;              // rows of a call
constexpr int kGemvWarps = 8;
constexpr int kGemvBlocks = 4;             // of an SM at a time (three: one row of 4096 x 4096 8.2 -> 9.1 us, of 8192 x 8192 23.7 -> 26.1)
constexpr int kGemvAhead = 4;              // 16-byte pieces of a weight row on their way

struct Gemv16Params {
  int rows, N, K, E;
  int64_t ldx;
  const int *efo, *counts;
  const __nv_bfloat16 *x, *w;
  __nv_bfloat16* y;                        // [rows, N], rows that are not live become zero
};

// s += the products of eight bf16 pairs, each exact
__device__ __forceinline__ void gemv_dot8(float& s, const uint4& a, const uint4& b) {
  const uint32_t u[4] = {a.x, a.y, a.z, a.w}, v[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("{\n\t.reg .b16 a, b, c, d;\n\t"
        "mov.b32 {a, b}, %1;\n\tmov.b32 {c, d}, %2;\n\t"
        "fma.rn.f32.bf16 %0, a, c, %0;\n\tfma.rn.f32.bf16 %0, b, d, %0;\n\t}"
        : "+f"(s)
        : "r"(u[i]), "r"(v[i]));
}
// Weights pass once: not kept in L1.  (No read-only load: the kernel begins while the one before it, which may write them, ends.)
__device__ __forceinline__ uint4 gemv_load(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// C rows from x0 on times a warp's weight rows -> y
template <int C>
__device__ __forceinline__ void gemv_task(const Gemv16Params& p, const uint4* w, const __nv_bfloat16* x0, __nv_bfloat16* y0, int lane) {
  float s[kGemvCols][C];
#pragma unroll
  for (int j = 0; j < kGemvCols; ++j)
#pragma unroll
    for (int r = 0; r < C; ++r) s[j][r] = 0.f;
  const int pieces = p.K >> 3;
  for (int k0 = lane; k0 < pieces; k0 += 32 * kGemvAhead) {
    uint4 a[kGemvAhead][kGemvCols];
#pragma unroll
    for (int u = 0; u < kGemvAhead; ++u)
#pragma unroll
      for (int j = 0; j < kGemvCols; ++j)
        a[u][j] = k0 + 32 * u < pieces ? gemv_load(w + (int64_t)j * pieces + k0 + 32 * u) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < kGemvAhead; ++u) {
      if (k0 + 32 * u >= pieces) break;
#pragma unroll
      for (int r = 0; r < C; ++r) {
        const uint4 b = *reinterpret_cast<const uint4*>(x0 + r * p.ldx + (k0 + 32 * u) * 8);
#pragma unroll
        for (int j = 0; j < kGemvCols; ++j) gemv_dot8(s[j][r], a[u][j], b);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < C; ++r) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
#pragma unroll
      for (int j = 0; j < kGemvCols; ++j) s[j][r] += __shfl_xor_sync(0xffffffffu, s[j][r], d);
    }
    if (lane == r) *reinterpret_cast<uint32_t*>(y0 + (int64_t)r * p.N) = pack_bf16x2(s[0][r], s[1][r]);
  }
}

__global__ void __launch_bounds__(32 * kGemvWarps, kGemvBlocks) gemv16_kernel(const Gemv16Params p) {
  // Up to four rows of an expert each, and runs of rows that are nobody's, found by a thread an expert.  The units are put in one order,
  // since blocks divide them by their places; that of the runs says nothing.
  __shared__ int n_units, n_gaps, found_e[kGemvMost], found_row[kGemvMost], found_live[kGemvMost];
  __shared__ int unit_e[kGemvMost], unit_row[kGemvMost], unit_live[kGemvMost], gap_from[kGemvMost], gap_to[kGemvMost];
  static_assert(32 * kGemvWarps >= kMaxExperts2, "a thread an expert");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) n_units = n_gaps = 0;
  __syncthreads();
  wait_for_kernel_before();
  next_kernel_may_start();
  auto gap = [&](int from, int to) {
    if (from >= to) return;
    const int i = atomicAdd(&n_gaps, 1);
    if (i < kGemvMost) {
      gap_from[i] = from;
      gap_to[i] = to;
    }
  };
  for (int e = threadIdx.x; e < p.E; e += 32 * kGemvWarps) {
    const int start = p.efo ? min(max(p.efo[e], 0), p.rows) : 0, end = p.efo ? min(max(p.efo[e + 1], 0), p.rows) : p.rows;
    const int live = max(p.counts ? min(end, start + min(max(p.counts[e], 0), p.rows)) : end, start);
    for (int row = start; row < live; row += kGemvRows) {
      const int i = atomicAdd(&n_units, 1);
      if (i >= kGemvMost) break;                // (segments that overlap; those that ascend have no more rows than there are)
      found_e[i] = e;
      found_row[i] = row;
      found_live[i] = min(live - row, kGemvRows);
    }
    gap(live, end);
    if (e == 0) gap(0, start);
    if (e == p.E - 1) gap(end, p.rows);
  }
  __syncthreads();
  const int units = min(n_units, kGemvMost);
  if ((int)threadIdx.x < units) {
    const int e = found_e[threadIdx.x], row = found_row[threadIdx.x];
    int before = 0;
    for (int i = 0; i < units; ++i) before += found_e[i] < e || (found_e[i] == e && found_row[i] < row);
    unit_e[before] = e;
    unit_row[before] = row;
    unit_live[before] = found_live[threadIdx.x];
  }
  __syncthreads();
  const int w0 = (int)blockIdx.x * kGemvWarps + warp, n_warps = (int)gridDim.x * kGemvWarps;
  for (int i = 0; i < min(n_gaps, kGemvMost); ++i)
    for (int r = gap_from[i] + w0; r < gap_to[i]; r += n_warps)
      for (int col = lane * 8; col < p.N; col += 256) *reinterpret_cast<uint4*>(p.y + (int64_t)r * p.N + col) = make_uint4(0, 0, 0, 0);
  const int per = p.N / kGemvCols, total = units * per;
  for (int task = w0; task < total; task += n_warps) {
    const int unit = task / per, n = (task - unit * per) * kGemvCols;
    const int row = unit_row[unit];
    const uint4* w = reinterpret_cast<const uint4*>(p.w + ((int64_t)unit_e[unit] * p.N + n) * p.K);
    const __nv_bfloat16* x = p.x + row * p.ldx;
    __nv_bfloat16* y = p.y + (int64_t)row * p.N + n;
    switch (unit_live[unit]) {
      case 1: gemv_task<1>(p, w, x, y, lane); break;
      case 2: gemv_task<2>(p, w, x, y, lane); break;
      case 3: gemv_task<3>(p, w, x, y, lane); break;
      default: gemv_task<4>(p, w, x, y, lane);
    }
  }
}

}  // namespace smoe
