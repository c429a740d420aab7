// Quantizers for products with one f32 scale per block of 128: rows (1 x 128), columns (128 rows x 1), weights (128 x 128).
//
//   a = max(max |x| of the block, 2^-100),  scale = a / 448,  q = e4m3(x * (448 / a)),  each step rounded once in f32
//
// (the multiplier is the rounded quotient 448 / a, so that a block costs one division more and not one for each value).  NaN is
// no magnitude: it stays NaN in the payload and leaves its block's scale alone.  One read, one write: weights are bound by HBM, 8 x
// 4096 x 2048 34 us (5.9 TB/s), rows by the issue of instructions (72 % of the slots, the integer pipe as much; HBM 36 %), 8192 x
// 4096 22.7 us (4.5 TB/s).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "host.h"
#include "ptx.cuh"
#include "quant_groups.cuh"
#include "smoe_b200.h"
#include "smoe_internal.h"

namespace smoe {

__device__ __forceinline__ uint32_t q128_pack4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
// bytes from one payload row to the next: rows of the operands of a product start on 16 bytes
__host__ __device__ __forceinline__ int64_t q128_pitch(int64_t K) { return (K + 15) & ~(int64_t)15; }
__device__ __forceinline__ uint32_t q128_abs(uint32_t w) { return w & 0x7FFF7FFFu; }
// larger of two pairs of bf16, a number before a NaN
__device__ __forceinline__ uint32_t q128_max(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float q128_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float q128_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ float q128_max_of(uint32_t m) { return fmaxf(fmaxf(q128_lo(m), q128_hi(m)), kAmaxFloor); }
// eight bf16 times one number each -> eight e4m3
__device__ __forceinline__ uint2 q128_pack8(const uint4& v, float m) {
  return make_uint2(q128_pack4(q128_lo(v.x) * m, q128_hi(v.x) * m, q128_lo(v.y) * m, q128_hi(v.y) * m),
                    q128_pack4(q128_lo(v.z) * m, q128_hi(v.z) * m, q128_lo(v.w) * m, q128_hi(v.w) * m));
}

// To some 4e-7, and 8e-8 |g| more where g is negative (its exponential's argument is rounded).  What that may decide is decided by
// q128_gated_again.
__device__ __forceinline__ float q128_silu(float g) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * g));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return g * r;
}
// largest magnitude of eight bf16, in both halves
__device__ __forceinline__ uint32_t q128_max4(const uint4& v) {
  const uint32_t m = q128_max(q128_max(q128_abs(v.x), q128_abs(v.y)), q128_max(q128_abs(v.z), q128_abs(v.w)));
  return q128_max(m, __byte_perm(m, m, 0x1032));
}
// over sixteen lanes, for N blocks, two to a word
template <int N>
__device__ __forceinline__ void q128_max16(const uint32_t (&m)[N], uint32_t half, float (&amax)[N]) {
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    uint32_t two = j + 1 < N ? __byte_perm(m[j], m[j + 1 < N ? j + 1 : j], 0x5410) : m[j];
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) two = q128_max(two, __shfl_xor_sync(half, two, d));
    amax[j] = q128_lo(two);
    if (j + 1 < N) amax[j + 1 < N ? j + 1 : j] = q128_hi(two);
  }
}
// What N <= 8 blocks of sixteen lanes are multiplied by, from their maxima; returns, in lane 8 + j, block j's scale.  A division takes
// as many instructions as the rest of a block: each lane does one, of either kind, instead of all.
template <int N>
__device__ __forceinline__ float q128_quotients(const float (&amax)[N], int lane16, uint32_t half, float (&inv)[N]) {
  float a = amax[0];
#pragma unroll
  for (int j = 1; j < N; ++j) a = (lane16 & 7) == j ? amax[j] : a;
  a = fmaxf(a, kAmaxFloor);
  const bool scale = lane16 >= 8;
  const float r = (scale ? a : kE4m3Max) / (scale ? kE4m3Max : a);
#pragma unroll
  for (int j = 0; j < N; ++j) inv[j] = __shfl_sync(half, r, j, 16);
  return r;
}

// An activation's payload must not depend on how an exponential was rounded.  A value and its block's maximum are off by a unit or
// two of the last place of f32 (more than kQ128Near for g below -16 or so); where that leaves a value within kQ128Near of the border
// between two e4m3 values (three in 200,000), it and the maximum are made again in 64 bits.  Of 150 M values none is another than in
// 64 bits then, with 4 in place of 8 one, without it 226.  It takes 16384 x 768 from 13.4 to 16.5 us, 512 x 768 from 2.4 to 3.4: half
// for the look at every value, half for the last warp with such a block, whose code no cache holds.  (Borders below the least normal
// value, 2^-6 of a maximum of 448, are not looked for.)
constexpr uint32_t kQ128Near = 8;
__device__ __forceinline__ uint32_t q128_from_border(float v) {      // below 2 * kQ128Near << 12: near one
  return (__float_as_uint(v) << 12) + 0x80000000u + (kQ128Near << 12);
}
__device__ __noinline__ double q128_gated64(uint32_t w) {
  const double g = q128_lo(w);
  return g / (1.0 + exp(-g)) * q128_hi(w);
}
// A block of sixteen lanes: words, q: gate and up, and the payload, of a lane's eight values; which: those that may be the largest, and
// << 8 those near a border.  The payload of the others stands: none of them is near one.
__device__ __noinline__ void q128_gated_again(const uint32_t* words, uint8_t* q, float* scale, uint32_t which, uint32_t half) {
  uint32_t near = which >> 8;
  const uint32_t first = near & (0u - near);
  double mine = 0.0;
  float a = kAmaxFloor;
  for (uint32_t todo = (which & 0xFF) | first; __any_sync(half, todo); todo &= todo - 1) {      // lanes side by side: once, mostly
    const uint32_t bit = todo & (0u - todo);
    const double v = todo ? q128_gated64(words[__ffs(todo) - 1]) : 0.0;
    if (which & 0xFF & bit) a = fmaxf(a, (float)fabs(v));
    if (bit == first) mine = v;
  }
  for (int d = 8; d > 0; d >>= 1) a = fmaxf(a, __shfl_xor_sync(half, a, d));
  const float inv = kE4m3Max / a;
  if (scale) *scale = a / kE4m3Max;
  while (near) {
    const int at = __ffs(near) - 1;
    q[at] = (uint8_t)q128_pack4((float)(mine * inv), 0.f, 0.f, 0.f);
    near &= near - 1;
    if (near) mine = q128_gated64(words[__ffs(near) - 1]);
  }
}

// ---- rows -------------------------------------------------------------------------------------------------------------
// Sixteen lanes take a block of 128 values, eight each (with GLU: of gate and up, interleaved, 32 bytes a lane), and blocks
// that follow one another: all their loads are on their way before the first is looked at.  Which rows:
//   list == null, naept == null   row i -> row i, i < n
//   list                          row list[i] -> row list[i], i < min(n, *n_live)
//   naept                         row i -> rows s_rev[naept[i]] .. s_rev[naept[i+1] - 1], i < n: a token's places
struct Rows128Args {
  const void* x;
  int64_t n, out_rows;
  int K;                      // values of a row that leaves
  const int *list, *n_live;
  const int *naept, *s_rev;
  uint8_t* q;
  float* s;
};

template <bool GLU, int PER>
__global__ void __launch_bounds__(256, PER == 4 ? 4 : GLU ? 5 : 6) quant128_rows_kernel(const Rows128Args a) {
  wait_for_kernel_before();                               // (a launch of `chained`; the next one counts on it)
  next_kernel_may_start();
  const int kb = (a.K + 127) / 128;
  const int64_t n = a.list && a.n_live ? min((int64_t)*a.n_live, a.n) : a.n;
  const int lane16 = threadIdx.x & 15;
  const uint32_t half = 0xFFFFu << (threadIdx.x & 16);
  const uint64_t u0 = ((blockIdx.x * (uint64_t)blockDim.x + threadIdx.x) >> 4) * PER;
  // (a 32-bit quotient wherever it holds: the 64-bit one takes longer than a block's arithmetic)
  int64_t i = u0 >> 32 ? (int64_t)(u0 / kb) : (int64_t)((uint32_t)u0 / (uint32_t)kb);
  int b = (int)(u0 - (uint64_t)i * kb);
  uint4 v[PER][GLU ? 2 : 1];
  int64_t src[PER];
  int blk[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    src[j] = i < n ? (a.list ? (int64_t)a.list[i] : i) : -1;
    if (a.list && (src[j] < 0 || src[j] >= a.out_rows)) src[j] = -1;
    blk[j] = b;
    const int col = b * 128 + lane16 * 8;
    v[j][0] = make_uint4(0, 0, 0, 0);
    if (GLU) v[j][GLU ? 1 : 0] = make_uint4(0, 0, 0, 0);
    if (src[j] >= 0 && col < a.K) {                       // K % 8 == 0: a lane's eight values are there or not
      if (GLU) {
        const uint4* p = (const uint4*)((const uint16_t*)a.x + (src[j] * a.K + col) * 2);
        v[j][0] = __ldcs(p);
        v[j][GLU ? 1 : 0] = __ldcs(p + 1);
      } else {
        v[j][0] = __ldcs((const uint4*)((const uint16_t*)a.x + src[j] * a.K + col));
      }
    }
    if (++b == kb) {
      b = 0;
      ++i;
    }
  }
  float y[GLU ? PER : 1][8], amax[PER];
  if (GLU) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t* w = (const uint32_t*)v[j];
      amax[j] = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[GLU ? j : 0][e] = q128_silu(q128_lo(w[e])) * q128_hi(w[e]);
        amax[j] = fmaxf(amax[j], fabsf(y[GLU ? j : 0][e]));
      }
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) amax[j] = fmaxf(amax[j], __shfl_xor_sync(half, amax[j], d));
    }
  } else {
    uint32_t m[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) m[j] = q128_max4(v[j][0]);
    q128_max16<PER>(m, half, amax);
  }
  float inv[PER];
  const float scale = q128_quotients<PER>(amax, lane16, half, inv);
  const int64_t pitch = q128_pitch(a.K);
  uint2 gated[GLU ? PER : 1];
  uint32_t again = 0;                                     // GLU: values of each block to be made again, see q128_gated_again
  if (GLU) {
    uint32_t near = 0xFFFFFFFFu;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = y[GLU ? j : 0][e] * inv[j];
        near = min(near, q128_from_border(f[e]));
      }
      gated[GLU ? j : 0] = make_uint2(q128_pack4(f[0], f[1], f[2], f[3]), q128_pack4(f[4], f[5], f[6], f[7]));
    }
    if (__any_sync(0xffffffffu, near < 2 * kQ128Near << 12)) {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        uint32_t top = 0, by = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = y[GLU ? j : 0][e];
          top |= fabsf(x) >= amax[j] * (1.f - 1e-5f) ? 1u << e : 0u;
          by |= q128_from_border(x * inv[j]) < 2 * kQ128Near << 12 ? 1u << e : 0u;
        }
        if (__any_sync(half, by)) again |= (by << 8 | top) << (16 * j);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int col = blk[j] * 128 + lane16 * 8;
    const bool in = col < a.K, mine = lane16 == 8 + j;        // the lane that has this block's scale
    uint2 out;
    if (GLU) {
      out = gated[GLU ? j : 0];
    } else {
      out = q128_pack8(v[j][0], inv[j]);
    }
    if (src[j] < 0) continue;
    if (a.naept) {
      const int last = a.naept[src[j] + 1];
      for (int t = a.naept[src[j]]; t < last; ++t) {
        const int64_t dst = a.s_rev[t];
        if (dst < 0 || dst >= a.out_rows) continue;
        if (in) *(uint2*)(a.q + dst * pitch + col) = out;
        if (mine) a.s[dst * kb + blk[j]] = scale;
      }
    } else {
      if (in) *(uint2*)(a.q + src[j] * pitch + col) = out;
      if (mine) a.s[src[j] * kb + blk[j]] = scale;
    }
  }
  if (GLU && __any_sync(0xffffffffu, again)) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t which = again >> (16 * j) & 0xFFFF;
      if (!__any_sync(half, which)) continue;
      const int64_t at = blk[j] * 128 + lane16 * 8;            // (lanes beyond the columns ask for nothing)
      q128_gated_again((const uint32_t*)a.x + src[j] * a.K + at, a.q + src[j] * pitch + at,
                       lane16 == 8 + j ? a.s + src[j] * kb + blk[j] : nullptr, which, half);
    }
  }
}

// ---- tiles of 128 x 128 ----------------------------------------------------------------------------------------------------
// A block holds a tile in registers (eight rows of eight values a thread) and takes from it what is asked for: a scale a row, a
// scale a column, or one for all.  ROWS and COLS from one read is what a training step needs of an activation and of a
// gradient: the row form feeds the products over columns, the column form the weight gradient, whose sum runs over rows.
// The column form leaves transposed: a copy of the weight gradient's operands then starts on 16 bytes wherever a segment does, and the
// reduction is contiguous, which the MMAs read out of shared memory in 650 clocks a block (950 otherwise; the epilogue hides either).
// Bound by the issue of instructions (72 % of the slots, 3.8 TB/s of HBM): 16384 x 4096 to both forms 58 us, 41 at the copy rate.
//   efo, counts (column form): rows of a segment behind its live ones count as zero and leave zero; tiles without live rows stay
//   unwritten
struct Tile128Args {
  const void* x;
  int64_t rows;              // of a matrix
  int K, E;                  // columns; segments (or, WEIGHT, matrices)
  const int *efo, *counts;
  uint8_t *q, *qt;           // [rows, K]; [K, rows]
  float *s, *st;             // [rows, K/128] ([E, rows/128, K/128]); [rows/128, K]
};

template <bool ROWS, bool COLS, bool WEIGHT>
__global__ void __launch_bounds__(256) quant128_tile_kernel(const Tile128Args a) {
  __shared__ uint32_t s_max[8][64];                       // per warp: column maxima, two a word
  __shared__ __align__(16) float s_mul[128];
  __shared__ __align__(16) uint8_t s_t[COLS ? 128 * 128 : 16];      // the transposed tile, 16-byte pieces at places xor (column / 8) % 8
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kb = (a.K + 127) / 128;
  const int64_t mat = WEIGHT ? blockIdx.z : 0;
  const int64_t row0 = (int64_t)blockIdx.y * 128, my_row = row0 + warp * 16 + (lane >> 4) * 8;
  const int c0 = blockIdx.x * 128, col = c0 + (lane & 15) * 8;
  int64_t end = a.rows;                                   // live rows end here
  if (COLS && a.efo) {
    int lo = 0, hi = a.E;
    while (lo < hi) {                                     // the segment of this tile
      const int mid = (lo + hi) >> 1;
      if (a.efo[mid + 1] <= row0) lo = mid + 1; else hi = mid;
    }
    end = 0;
    if (lo < a.E && a.efo[lo] <= row0) {
      end = a.efo[lo + 1];
      if (a.counts) end = min(end, (int64_t)a.efo[lo] + a.counts[lo]);
      end = min(end, a.rows);
    }
    if (end <= row0 && !ROWS) return;
  }
  const uint16_t* x = (const uint16_t*)a.x + mat * a.rows * a.K;
  const bool in_col = col < a.K;
  uint4 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = make_uint4(0, 0, 0, 0);
    if (in_col && my_row + i < a.rows) v[i] = __ldcs((const uint4*)(x + (my_row + i) * a.K + col));
  }
  if (ROWS) {
    const uint32_t half = 0xFFFFu << (lane & 16);
    uint32_t m[8];
    float amax[8], inv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = q128_max4(v[i]);
    q128_max16<8>(m, half, amax);
    const float scale = q128_quotients<8>(amax, lane & 15, half, inv);
    if ((lane & 8) && my_row + (lane & 7) < a.rows) a.s[(my_row + (lane & 7)) * kb + blockIdx.x] = scale;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (in_col && my_row + i < a.rows) *(uint2*)(a.q + (my_row + i) * q128_pitch(a.K) + col) = q128_pack8(v[i], inv[i]);
  }
  if (COLS) {
    if (end <= row0) return;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (my_row + i >= end) v[i] = make_uint4(0, 0, 0, 0);
  }
  if (COLS || WEIGHT) {
    uint32_t m[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m[0] = q128_max(m[0], q128_abs(v[i].x));
      m[1] = q128_max(m[1], q128_abs(v[i].y));
      m[2] = q128_max(m[2], q128_abs(v[i].z));
      m[3] = q128_max(m[3], q128_abs(v[i].w));
    }
    if (WEIGHT) {
      uint32_t t = q128_max(q128_max(m[0], m[1]), q128_max(m[2], m[3]));
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) t = q128_max(t, __shfl_xor_sync(0xffffffffu, t, d));
      if (lane == 0) s_max[warp][0] = t;
      __syncthreads();
      t = s_max[0][0];
#pragma unroll
      for (int w = 1; w < 8; ++w) t = q128_max(t, s_max[w][0]);
      const float amax = q128_max_of(t), mul = kE4m3Max / amax;
      if (tid == 0) a.s[(mat * gridDim.y + blockIdx.y) * kb + blockIdx.x] = amax / kE4m3Max;
      uint8_t* q = a.q + mat * a.rows * q128_pitch(a.K);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (in_col && my_row + i < a.rows) *(uint2*)(q + (my_row + i) * q128_pitch(a.K) + col) = q128_pack8(v[i], mul);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) m[j] = q128_max(m[j], __shfl_xor_sync(0xffffffffu, m[j], 16));
      if (lane < 16) *(uint4*)&s_max[warp][lane * 4] = make_uint4(m[0], m[1], m[2], m[3]);
      __syncthreads();
      if (tid < 64) {
        uint32_t t = s_max[0][tid];
#pragma unroll
        for (int w = 1; w < 8; ++w) t = q128_max(t, s_max[w][tid]);
        const float lo = fmaxf(q128_lo(t), kAmaxFloor), hi = fmaxf(q128_hi(t), kAmaxFloor);
        s_mul[2 * tid] = kE4m3Max / lo;
        s_mul[2 * tid + 1] = kE4m3Max / hi;
        const int c = c0 + 2 * tid;
        if (c < a.K) *(float2*)(a.st + (int64_t)blockIdx.y * a.K + c) = make_float2(lo / kE4m3Max, hi / kE4m3Max);
      }
      __syncthreads();
      // eight rows of a column are eight consecutive bytes of the transposed tile
      const uint32_t* w = (const uint32_t*)v;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = (lane & 15) * 8 + j;
        const float f = s_mul[c];
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = ((j & 1) ? q128_hi(w[i * 4 + j / 2]) : q128_lo(w[i * 4 + j / 2])) * f;
        *(uint2*)(s_t + c * 128 + ((warp ^ (lane & 7)) << 4) + (lane >> 4) * 8) =
            make_uint2(q128_pack4(y[0], y[1], y[2], y[3]), q128_pack4(y[4], y[5], y[6], y[7]));
      }
      __syncthreads();
      const int64_t pitch = q128_pitch(a.rows);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = warp * 16 + i * 4 + (lane >> 3), piece = lane & 7;
        if (c0 + c < a.K && row0 + piece * 16 < a.rows)
          *(uint4*)(a.qt + (int64_t)(c0 + c) * pitch + row0 + piece * 16) =
              *(const uint4*)(s_t + c * 128 + ((piece ^ ((c >> 3) & 7)) << 4));
      }
    }
  }
}

static int quant128_check(const void* x, const void* q, const void* s, int64_t rows, int64_t K) {
  if (rows < 0 || K <= 0 || K % 8 || K >= (int64_t)1 << 30 || rows >= (int64_t)1 << 31) return SMOE_ERR_SHAPE;
  if (rows > 0 && (!x || !q || !s)) return SMOE_ERR_ARG;
  if (((uintptr_t)x & 15) || ((uintptr_t)q & 15) || ((uintptr_t)s & 3)) return SMOE_ERR_ALIGN;
  return SMOE_OK;
}

static int launch_rows(const Rows128Args& a, bool glu, bool chained, void* stream) {
  if (a.n == 0 || a.out_rows == 0) return SMOE_OK;
  const int64_t units = a.n * ((a.K + 127) / 128);
  // Several blocks each where that leaves every SM enough warps: four, or two where the activation's or a token's many rows need
  // the registers.  8192 x 4096 one block 28.0 us, two 24.2, four 22.7; gated 32768 x 768 40, 25.2, 26.5 (two with q128_gated_again
  // 28.9); eight places a token 18.6, 18.4, 19.9.
  const int most = glu || a.naept ? 2 : 4, per = units >= (int64_t)sm_count() * 64 * 4 ? most : 1;
  const int64_t grid = (units + 16 * per - 1) / (16 * per);
  if (grid >= (int64_t)1 << 31) return SMOE_ERR_SHAPE;
  auto kern = glu        ? (per == 2 ? quant128_rows_kernel<true, 2> : quant128_rows_kernel<true, 1>)
              : per == 4 ? quant128_rows_kernel<false, 4>
              : per == 2 ? quant128_rows_kernel<false, 2>
                         : quant128_rows_kernel<false, 1>;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(256);
  cfg.stream = (cudaStream_t)stream;
  cfg.attrs = &attr;
  cfg.numAttrs = chained ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kern, a) != cudaSuccess) return SMOE_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? SMOE_OK : SMOE_ERR_LAUNCH;
}

int quant128_rows(const void* x_bf16, int64_t rows, int64_t K, int swiglu, const int* list, const int* n_live, int64_t n_list, void* q,
                  float* scales, bool chained, void* stream) {
  const int rc = quant128_check(x_bf16, q, scales, rows, K);
  if (rc) return rc;
  if (list && (n_list < 0 || !n_live)) return SMOE_ERR_ARG;
  Rows128Args a{x_bf16, list ? n_list : rows, rows, (int)K, list, n_live, nullptr, nullptr, (uint8_t*)q, scales};
  return launch_rows(a, swiglu != 0, chained, stream);
}

int quant128_rows_scatter(const void* x_bf16, int64_t T, int64_t K, const int* naept, const int* s_rev, int64_t rows, void* q,
                          float* scales, bool chained, void* stream) {
  const int rc = quant128_check(x_bf16, q, scales, rows, K);
  if (rc) return rc;
  if (T < 0 || T >= (int64_t)1 << 31) return SMOE_ERR_SHAPE;
  if (T > 0 && rows > 0 && (!naept || !s_rev)) return SMOE_ERR_ARG;
  Rows128Args a{x_bf16, T, rows, (int)K, nullptr, nullptr, naept, s_rev, (uint8_t*)q, scales};
  return launch_rows(a, false, chained, stream);
}

}  // namespace smoe

using namespace smoe;

extern "C" {

int smoe_quant128_rows(const void* x_bf16, int64_t rows, int64_t K, int swiglu, const int32_t* list, const int32_t* n_live,
                       int64_t n_list, void* q, float* scales, void* stream) {
  return quant128_rows(x_bf16, rows, K, swiglu, list, n_live, n_list, q, scales, false, stream);
}

int smoe_quant128_rows_scatter(const void* x_bf16, int64_t T, int64_t K, const int32_t* naept, const int32_t* s_rev, int64_t rows,
                               void* q, float* scales, void* stream) {
  return quant128_rows_scatter(x_bf16, T, K, naept, s_rev, rows, q, scales, false, stream);
}

int smoe_quant128_dual(const void* x_bf16, int64_t rows, int64_t K, const int32_t* efo, const int32_t* counts, int64_t E, void* q,
                       float* scales, void* q_t, float* t_scales, void* stream) {
  int rc = quant128_check(x_bf16, q_t, t_scales, rows, K);
  if (!rc && q) rc = quant128_check(x_bf16, q, scales, rows, K);
  if (rc) return rc;
  if ((uintptr_t)t_scales & 7) return SMOE_ERR_ALIGN;
  if (E < 0 || (efo && E <= 0) || (counts && !efo)) return SMOE_ERR_ARG;
  if (rows == 0) return SMOE_OK;
  if (rows > (int64_t)65535 * 128) return SMOE_ERR_SHAPE;
  Tile128Args a{x_bf16, rows, (int)K, (int)E, efo, counts, (uint8_t*)q, (uint8_t*)q_t, scales, t_scales};
  const dim3 grid((unsigned)((K + 127) / 128), (unsigned)((rows + 127) / 128));
  if (q) quant128_tile_kernel<true, true, false><<<grid, 256, 0, (cudaStream_t)stream>>>(a);
  else quant128_tile_kernel<false, true, false><<<grid, 256, 0, (cudaStream_t)stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? SMOE_OK : SMOE_ERR_LAUNCH;
}

int smoe_quant128_weight(const void* w_bf16, int64_t E, int64_t N, int64_t K, void* q, float* scales, void* stream) {
  const int rc = quant128_check(w_bf16, q, scales, N, K);
  if (rc) return rc;
  if (E < 0 || E > 65535 || N > (int64_t)65535 * 128) return SMOE_ERR_SHAPE;
  if (E == 0 || N == 0) return SMOE_OK;
  Tile128Args a{w_bf16, N, (int)K, (int)E, nullptr, nullptr, (uint8_t*)q, nullptr, scales, nullptr};
  const dim3 grid((unsigned)((K + 127) / 128), (unsigned)((N + 127) / 128), (unsigned)E);
  quant128_tile_kernel<false, false, true><<<grid, 256, 0, (cudaStream_t)stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? SMOE_OK : SMOE_ERR_LAUNCH;
}

}  // extern "C"
