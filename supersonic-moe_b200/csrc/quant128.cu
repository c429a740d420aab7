// Quantizers for products with one f32 scale per block of 128: rows (1 x 128), columns (128 rows x 1), weights (128 x 128).
//
//   a = max(max |x| of the block, 2^-100),  scale = a / 448,  q = e4m3(x * (448 / a)),  each step rounded once in f32
//
// (the multiplier is the rounded quotient 448 / a, so that a block costs one division more and not one for each value).  NaN is
// no magnitude: it stays NaN in the payload and leaves its block's scale alone.  All three are bound by HBM: one read, one write.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "smoe_b200.h"

namespace smoe {

constexpr float kE4m3Max = 448.f;
constexpr float kAmaxFloor = 7.888609052210118e-31f;      // 2^-100: 448 / a stays finite, a / 448 normal

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

// ---- rows -------------------------------------------------------------------------------------------------------------
// Sixteen lanes take a block of 128 values, eight each (with GLU: of gate and up, interleaved, 32 bytes a lane).  Which rows:
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

template <bool GLU>
__global__ void __launch_bounds__(256) quant128_rows_kernel(const Rows128Args a) {
  const int kb = (a.K + 127) / 128;
  const int64_t units = (a.list && a.n_live ? min((int64_t)*a.n_live, a.n) : a.n) * kb;
  const int lane16 = threadIdx.x & 15;
  const uint32_t half = 0xFFFFu << (threadIdx.x & 16);
  for (int64_t u = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 4; u < units; u += ((int64_t)gridDim.x * blockDim.x) >> 4) {
    const int64_t i = u / kb;
    const int b = (int)(u - i * kb);
    const int64_t src = a.list ? a.list[i] : i;
    const int col = b * 128 + lane16 * 8;
    // K % 8 == 0: a lane's eight values are there or not
    const bool in = col < a.K && (!a.list || (src >= 0 && src < a.out_rows));
    uint2 out;
    float amax;
    if (GLU) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = 0.f;
      if (in) {
        const uint4* p = (const uint4*)((const uint16_t*)a.x + (src * a.K + col) * 2);
        const uint4 v[2] = {p[0], p[1]};
        const uint32_t* w = (const uint32_t*)v;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float g = q128_lo(w[j]), up = q128_hi(w[j]);
          y[j] = g / (1.f + expf(-g)) * up;
        }
      }
      amax = kAmaxFloor;
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(y[j]));
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(half, amax, d));
      const float m = kE4m3Max / amax;
      out = make_uint2(q128_pack4(y[0] * m, y[1] * m, y[2] * m, y[3] * m), q128_pack4(y[4] * m, y[5] * m, y[6] * m, y[7] * m));
    } else {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (in) v = *(const uint4*)((const uint16_t*)a.x + src * a.K + col);
      uint32_t m2 = q128_max(q128_max(q128_abs(v.x), q128_abs(v.y)), q128_max(q128_abs(v.z), q128_abs(v.w)));
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) m2 = q128_max(m2, __shfl_xor_sync(half, m2, d));
      amax = q128_max_of(m2);
      out = q128_pack8(v, kE4m3Max / amax);
    }
    const float scale = amax / kE4m3Max;
    if (a.naept) {
      const int last = a.naept[i + 1];
      for (int j = a.naept[i]; j < last; ++j) {
        const int64_t dst = a.s_rev[j];
        if (dst < 0 || dst >= a.out_rows) continue;
        if (in) *(uint2*)(a.q + dst * q128_pitch(a.K) + col) = out;
        if (lane16 == 0) a.s[dst * kb + b] = scale;
      }
    } else if (src >= 0 && src < a.out_rows) {
      if (in) *(uint2*)(a.q + src * q128_pitch(a.K) + col) = out;
      if (lane16 == 0) a.s[src * kb + b] = scale;
    }
  }
}

// ---- tiles of 128 x 128 ----------------------------------------------------------------------------------------------------
// A block holds a tile in registers (eight rows of eight values a thread) and takes from it what is asked for: a scale a row, a
// scale a column, or one for all.  ROWS and COLS from one read is what a training step needs of an activation and of a
// gradient: the row form feeds the products over columns, the column form the weight gradient, whose sum runs over rows.
// The column form leaves transposed: the tensor core reads 8-bit operands whose reduction is not contiguous at half the rate out of
// shared memory (the weight gradient's MMAs: 950 clocks a block against 650).
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
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t m2 = q128_max(q128_max(q128_abs(v[i].x), q128_abs(v[i].y)), q128_max(q128_abs(v[i].z), q128_abs(v[i].w)));
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) m2 = q128_max(m2, __shfl_xor_sync(half, m2, d));
      const float amax = q128_max_of(m2);
      if (my_row + i < a.rows) {
        if (in_col) *(uint2*)(a.q + (my_row + i) * q128_pitch(a.K) + col) = q128_pack8(v[i], kE4m3Max / amax);
        if ((lane & 15) == 0) a.s[(my_row + i) * kb + blockIdx.x] = amax / kE4m3Max;
      }
    }
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

static int launch_rows(const Rows128Args& a, bool glu, void* stream) {
  if (a.n == 0 || a.out_rows == 0) return SMOE_OK;
  const int64_t units = a.n * ((a.K + 127) / 128);
  int64_t grid = (units + 15) / 16;
  if (grid > 148 * 32) grid = 148 * 32;
  auto kern = glu ? quant128_rows_kernel<true> : quant128_rows_kernel<false>;
  kern<<<(unsigned)grid, 256, 0, (cudaStream_t)stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? SMOE_OK : SMOE_ERR_LAUNCH;
}

}  // namespace smoe

using namespace smoe;

extern "C" {

int smoe_quant128_rows(const void* x_bf16, int64_t rows, int64_t K, int swiglu, const int32_t* list, const int32_t* n_live,
                       int64_t n_list, void* q, float* scales, void* stream) {
  const int rc = quant128_check(x_bf16, q, scales, rows, K);
  if (rc) return rc;
  if (list && (n_list < 0 || !n_live)) return SMOE_ERR_ARG;
  Rows128Args a{x_bf16, list ? n_list : rows, rows, (int)K, list, n_live, nullptr, nullptr, (uint8_t*)q, scales};
  return launch_rows(a, swiglu != 0, stream);
}

int smoe_quant128_rows_scatter(const void* x_bf16, int64_t T, int64_t K, const int32_t* naept, const int32_t* s_rev, int64_t rows,
                               void* q, float* scales, void* stream) {
  const int rc = quant128_check(x_bf16, q, scales, rows, K);
  if (rc) return rc;
  if (T < 0 || T >= (int64_t)1 << 31) return SMOE_ERR_SHAPE;
  if (T > 0 && rows > 0 && (!naept || !s_rev)) return SMOE_ERR_ARG;
  Rows128Args a{x_bf16, T, rows, (int)K, nullptr, nullptr, naept, s_rev, (uint8_t*)q, scales};
  return launch_rows(a, false, stream);
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
