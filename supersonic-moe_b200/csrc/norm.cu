// Root-mean-square norm of rows in front of the experts, with the residual's addition before it and the 8-bit payload behind it.
//
//   h = x + residual (held in the residual's type)      r = 1 / sqrt(mean(h^2) + eps)      y = h r w
//   backward, g = dy w:  dh = r (g - h r^2 mean(g h)) + the gradient that comes in for h;   dw = sum over rows of dy h r
//
// A row is held in registers between its one read and its one write.  bf16 results and what is quantised from them are those of 64
// bits: the mean and r are f64 (8 conversions and 8 f64 additions a thread's 16 bytes, in the shadow of HBM), y is made in f32 and
// looked at: where it lies within kNormNear of the border between two bf16 values it is made again in f64 (one in 7000).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "host.h"
#include "quant_groups.cuh"
#include "smoe_b200.h"

namespace smoe {

constexpr int kNormMaxH = 16384;
constexpr int kNormMaxWarps = 16;

template <bool F32>
struct NormVec;                          // eight values of a row
template <>
struct NormVec<false> {
  uint4 v;
  __device__ __forceinline__ void load(const void* base, int64_t at) {
    v = *reinterpret_cast<const uint4*>((const uint16_t*)base + at);
  }
  __device__ __forceinline__ void load_some(const void* base, int64_t at, int n) {
    const uint16_t* p = (const uint16_t*)base + at;
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = i < n ? p[i] : 0u;
    v = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const { bf16x8_to_f32(v, f); }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    v = make_uint4(q_bf16x2(f[0], f[1]), q_bf16x2(f[2], f[3]), q_bf16x2(f[4], f[5]), q_bf16x2(f[6], f[7]));
  }
  __device__ __forceinline__ void clear() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void store(void* base, int64_t at) const { *reinterpret_cast<uint4*>((uint16_t*)base + at) = v; }
  __device__ __forceinline__ void store_some(void* base, int64_t at, int n) const {
    uint16_t* p = (uint16_t*)base + at;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
  }
};
template <>
struct NormVec<true> {
  float4 a, b;
  __device__ __forceinline__ void load(const void* base, int64_t at) {
    const float4* p = reinterpret_cast<const float4*>((const float*)base + at);
    a = p[0];
    b = p[1];
  }
  __device__ __forceinline__ void load_some(const void* base, int64_t at, int n) {
    const float* p = (const float*)base + at;
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? p[i] : 0.f;
    set(f);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    a = make_float4(f[0], f[1], f[2], f[3]);
    b = make_float4(f[4], f[5], f[6], f[7]);
  }
  __device__ __forceinline__ void clear() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void store(void* base, int64_t at) const {
    float4* p = reinterpret_cast<float4*>((float*)base + at);
    p[0] = a;
    p[1] = b;
  }
  __device__ __forceinline__ void store_some(void* base, int64_t at, int n) const {
    float f[8];
    get(f);
    float* p = (float*)base + at;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = f[i];
  }
};

// A thread's pieces of a row: piece c is eight columns from (c * threads + t) * 8 on, t the thread among the row's.  `vec`: rows and
// columns allow 16 bytes at a time (then H % 8 == 0 and a piece is there or not).
template <bool F32, int NC>
__device__ __forceinline__ void norm_load(NormVec<F32> (&v)[NC], const void* base, int64_t row_at, int t, int threads, int H, bool vec) {
  if (vec) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * threads + t) * 8;
      v[c].clear();
      if (col < H) v[c].load(base, row_at + col);
    }
  } else {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = (c * threads + t) * 8;
      v[c].load_some(base, row_at + col, H - col);
    }
  }
}
template <bool F32, int NC>
__device__ __forceinline__ void norm_store(const NormVec<F32> (&v)[NC], void* base, int64_t row_at, int t, int threads, int H,
                                           bool vec) {
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * threads + t) * 8;
    if (vec) {
      if (col < H) v[c].store(base, row_at + col);
    } else {
      v[c].store_some(base, row_at + col, H - col);
    }
  }
}
// the weight, of either type
template <int NC>
struct NormWeight {
  NormVec<true> v[NC];                   // bf16: the first half of a piece's registers
  __device__ __forceinline__ void load(const void* w, bool f32, int t, int threads, int H, bool vec) {
    if (f32) {
      norm_load<true, NC>(v, w, 0, t, threads, H, vec);
    } else {
      NormVec<false> b[NC];
      norm_load<false, NC>(b, w, 0, t, threads, H, vec);
#pragma unroll
      for (int c = 0; c < NC; ++c)
        v[c].a = make_float4(__uint_as_float(b[c].v.x), __uint_as_float(b[c].v.y), __uint_as_float(b[c].v.z),
                             __uint_as_float(b[c].v.w));
    }
  }
  __device__ __forceinline__ void get(int c, bool f32, float (&f)[8]) const {
    if (f32) v[c].get(f);
    else bf16x8_to_f32(make_uint4(__float_as_uint(v[c].a.x), __float_as_uint(v[c].a.y), __float_as_uint(v[c].a.z),
                                  __float_as_uint(v[c].a.w)), f);
  }
};

// over the warps of a row (one row a block if there are several), in one order
template <typename T>
__device__ __forceinline__ T norm_sum(T s, int warps, T* shared) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  if (warps == 1) return s;
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = s;
  __syncthreads();
  s = shared[0];
  for (int i = 1; i < warps; ++i) s += shared[i];
  return s;
}

// 1 / sqrt(v): the f32 approximation and one step of Newton's method, which leaves some 2^-44
__device__ __forceinline__ double norm_rsqrt(double v) {
  if (v > 1e-30 && v < 1e30) {
    const double r = rsqrtf((float)v);
    return r * (1.5 - 0.5 * v * r * r);
  }
  return 1.0 / sqrt(v);
}

// h r w in f32 is off by three roundings, each up to one unit of the last place
constexpr uint32_t kNormNear = 4;
// f32 that rounds to the bf16 nearest to d: a tie of f32 that is none of f64 is moved off
__device__ __forceinline__ float norm_for_bf16(double d) {
  float f = (float)d;
  if ((__float_as_uint(f) & 0xFFFFu) == 0x8000u) {
    const double away = fabs(d) - fabs((double)f);
    if (away > 0) f = __uint_as_float(__float_as_uint(f) + 1);
    if (away < 0) f = __uint_as_float(__float_as_uint(f) - 1);
  }
  return f;
}

struct NormArgs {
  const void *x, *res, *w;
  int64_t ldx, ldr, T;
  int H, warps, rows;                    // warps of a row, rows of a block
  int w_f32, vec_x, vec_r, vec_w, vec_y, vec_h;
  double eps, inv_H;
  void *y, *h;                           // null: not written
  double* rstd;
  uint8_t* q;
  void* s;
  int64_t pitch;                         // of the payload
};

enum NormQuant : int { NORM_PLAIN = 0, NORM_MX = 1, NORM_BLOCK128 = 2 };

// RES: 0 none, 1 of x's type, 2 f32 (beside bf16)
template <bool XF32, int RES, int QUANT, int NC>
__global__ void __launch_bounds__(32 * kNormMaxWarps) rms_norm_kernel(const NormArgs a) {
  constexpr bool HF32 = XF32 || RES == 2;
  __shared__ double sums[kNormMaxWarps];
  const int lane = threadIdx.x & 31;
  const int threads = a.warps * 32, t = a.warps == 1 ? lane : (int)threadIdx.x;
  const int64_t row = a.warps == 1 ? (int64_t)blockIdx.x * a.rows + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  if (row >= a.T) return;                               // a whole warp, and only where rows are of one warp
  NormVec<HF32> h[NC];
  if constexpr (RES == 0) {
    norm_load<HF32, NC>(h, a.x, row * a.ldx, t, threads, a.H, a.vec_x);
  } else {
    NormVec<XF32> x[NC];
    norm_load<XF32, NC>(x, a.x, row * a.ldx, t, threads, a.H, a.vec_x);
    norm_load<HF32, NC>(h, a.res, row * a.ldr, t, threads, a.H, a.vec_r);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float p[8], r[8];
      x[c].get(p);
      h[c].get(r);
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] += p[i];
      h[c].set(r);
    }
  }
  NormWeight<NC> w;
  w.load(a.w, a.w_f32, t, threads, a.H, a.vec_w);
  if constexpr (RES != 0) norm_store<HF32, NC>(h, a.h, row * a.H, t, threads, a.H, a.vec_h);
  double s0 = 0.0, s1 = 0.0;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float f[8];
    h[c].get(f);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const double p = f[i], q = f[i + 1];
      s0 = fma(p, p, s0);
      s1 = fma(q, q, s1);
    }
  }
  const double r64 = norm_rsqrt(norm_sum<double>(s0 + s1, a.warps, sums) * a.inv_H + a.eps);
  const float r = (float)r64;
  if (a.rstd && t == 0) a.rstd[row] = r64;
  const bool far = !(r64 > 1e-30 && r64 < 1e30);        // r in f32 would not have its full precision
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = (c * threads + t) * 8;
    float f[8], g[8], v[8];
    h[c].get(f);
    w.get(c, a.w_f32, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f[i] * r * g[i];
    if constexpr (XF32) {
      if (far) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)((double)f[i] * r64 * (double)g[i]);
      }
      NormVec<true> y;
      y.set(v);
      if (a.vec_y) {
        if (col < a.H) y.store(a.y, row * a.H + col);
      } else {
        y.store_some(a.y, row * a.H + col, a.H - col);
      }
    } else {
      uint32_t near = 0xFFFFFFFFu;                      // least distances above a border less kNormNear, of the even and the odd values
#pragma unroll
      for (int i = 0; i < 8; i += 2)
        near = __viaddmin_u16x2(__byte_perm(__float_as_uint(v[i]), __float_as_uint(v[i + 1]), 0x5410),
                                (0x8000u + kNormNear) * 0x10001u, near);
      if ((near & 0xFFFFu) <= 2 * kNormNear || (near >> 16) <= 2 * kNormNear || far) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = norm_for_bf16((double)f[i] * r64 * (double)g[i]);
      }
      NormVec<false> y;
      y.set(v);
      if (QUANT == NORM_PLAIN || a.y) {
        if (a.vec_y) {
          if (col < a.H) y.store(a.y, row * a.H + col);
        } else {
          y.store_some(a.y, row * a.H + col, a.H - col);
        }
      }
      if constexpr (QUANT == NORM_MX) {                 // four lanes a group
        uint32_t m = q_max_bf16x2(q_max_bf16x2(q_abs_bf16x2(y.v.x), q_abs_bf16x2(y.v.y)),
                                  q_max_bf16x2(q_abs_bf16x2(y.v.z), q_abs_bf16x2(y.v.w)));
        m = q_max_bf16x2(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = q_max_bf16x2(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const int e = q_e8m0_of(fmaxf(fmaxf(0.f, __uint_as_float(m << 16)), __uint_as_float(m & 0xFFFF0000u)));
        const float qs = q_scale_of(e);
        float b[8];
        y.get(b);
        if (col < a.H) {
          *reinterpret_cast<uint2*>(a.q + row * a.pitch + col) =
              make_uint2(q_pack4(b[0] * qs, b[1] * qs, b[2] * qs, b[3] * qs), q_pack4(b[4] * qs, b[5] * qs, b[6] * qs, b[7] * qs));
          if ((lane & 3) == 0) ((uint8_t*)a.s)[row * (a.H >> 5) + (col >> 5)] = (uint8_t)e;
        }
      }
      if constexpr (QUANT == NORM_BLOCK128) {           // sixteen
        uint32_t m = q_max_bf16x2(q_max_bf16x2(q_abs_bf16x2(y.v.x), q_abs_bf16x2(y.v.y)),
                                  q_max_bf16x2(q_abs_bf16x2(y.v.z), q_abs_bf16x2(y.v.w)));
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) m = q_max_bf16x2(m, __shfl_xor_sync(0xffffffffu, m, d));
        const float amax = fmaxf(fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u)), kAmaxFloor);
        // one division a lane, of either kind
        const float quotient = (lane & 1) ? kE4m3Max / amax : amax / kE4m3Max;
        const float qs = __shfl_sync(0xffffffffu, quotient, lane | 1);
        float b[8];
        y.get(b);
        if (col < a.H) {
          *reinterpret_cast<uint2*>(a.q + row * a.pitch + col) =
              make_uint2(q_pack4(b[0] * qs, b[1] * qs, b[2] * qs, b[3] * qs), q_pack4(b[4] * qs, b[5] * qs, b[6] * qs, b[7] * qs));
          if ((lane & 15) == 0) ((float*)a.s)[row * ((a.H + 127) >> 7) + (col >> 7)] = quotient;
        }
      }
    }
  }
}

// ---- backward -----------------------------------------------------------------------------------------------------------
struct NormBwdArgs {
  const void *dy, *h, *w, *dh;           // dh: null if none comes in
  const double* rstd;
  int64_t ldh, T;
  int H, warps, rows;
  int w_f32, vec_dy, vec_h, vec_w, vec_dh, vec_dx, vec_dres;
  void *dx, *dres;                       // null: not wanted
  float* part;                           // [blocks * flushes, H], null: no gradient of the weight
  int flushes;
};

// Rows that a block adds up in one f32 sum of a column; the sums of sums are f64
constexpr int kNormRun = 256;

// dx of x's type, dres of h's (where the two types differ; else dx serves both)
template <bool XF32, bool HF32, int NC>
__global__ void __launch_bounds__(32 * kNormMaxWarps) rms_norm_bwd_kernel(const NormBwdArgs a) {
  extern __shared__ float columns[];                    // [rows, H] where a block has several rows at a time
  __shared__ float sums[2][kNormMaxWarps];
  const int lane = threadIdx.x & 31;
  const int threads = a.warps * 32, t = a.warps == 1 ? lane : (int)threadIdx.x;
  const int group = a.warps == 1 ? threadIdx.x >> 5 : 0;
  const int64_t step = (int64_t)gridDim.x * a.rows;
  NormWeight<NC> w;
  w.load(a.w, a.w_f32, t, threads, a.H, a.vec_w);
  float dw[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[c][i] = 0.f;
  const float inv_H = 1.f / a.H;
  int turn = 0;
  int64_t row = (int64_t)blockIdx.x * a.rows + group;
  for (int flush = 0; flush < a.flushes; ++flush) {
    for (int n = 0; n < kNormRun && row < a.T; ++n, row += step) {
      NormVec<XF32> dy[NC];
      NormVec<HF32> h[NC], dh[NC];
      norm_load<XF32, NC>(dy, a.dy, row * a.H, t, threads, a.H, a.vec_dy);
      norm_load<HF32, NC>(h, a.h, row * a.ldh, t, threads, a.H, a.vec_h);
      if (a.dh) norm_load<HF32, NC>(dh, a.dh, row * a.H, t, threads, a.H, a.vec_dh);
      // r as a product of two f32, the first a power of two, so that rows of very large or very small values keep their precision
      const double r64 = a.rstd[row];
      const float pre = r64 < 1e-30 ? 0x1p-64f : r64 > 1e30 ? 0x1p64f : 1.f;
      const float r = (float)(r64 / pre);
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float fy[8], fh[8], fw[8];
        dy[c].get(fy);
        h[c].get(fh);
        w.get(c, a.w_f32, fw);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float hr = fh[i] * pre * r;
          s = fmaf(fy[i] * fw[i], hr, s);
          dw[c][i] = fmaf(fy[i], hr, dw[c][i]);
        }
      }
      s = norm_sum<float>(s, a.warps, sums[turn]) * inv_H;
      turn ^= 1;                                        // the next row's sums do not wait for this one's readers
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int col = (c * threads + t) * 8;
        float fy[8], fh[8], fw[8], d[8];
        dy[c].get(fy);
        h[c].get(fh);
        w.get(c, a.w_f32, fw);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = fmaf(-(fh[i] * pre * r), s, fy[i] * fw[i]) * r * pre;
        if (a.dh) {
          float e[8];
          dh[c].get(e);
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] += e[i];
        }
        if (a.dx) {
          NormVec<XF32> o;
          o.set(d);
          if (a.vec_dx) {
            if (col < a.H) o.store(a.dx, row * a.H + col);
          } else {
            o.store_some(a.dx, row * a.H + col, a.H - col);
          }
        }
        if constexpr (XF32 != HF32) {
          if (a.dres) {
            NormVec<HF32> o;
            o.set(d);
            if (a.vec_dres) {
              if (col < a.H) o.store(a.dres, row * a.H + col);
            } else {
              o.store_some(a.dres, row * a.H + col, a.H - col);
            }
          }
        }
      }
    }
    if (!a.part) continue;
    float* part = a.part + ((int64_t)blockIdx.x * a.flushes + flush) * a.H;
    if (a.rows > 1) {                                   // the block's rows first
      __syncthreads();
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int col = (c * threads + t) * 8 + i;
          if (col < a.H) columns[group * a.H + col] = dw[c][i];
        }
      __syncthreads();
      for (int col = threadIdx.x; col < a.H; col += blockDim.x) {
        float v = columns[col];
        for (int g = 1; g < a.rows; ++g) v += columns[g * a.H + col];
        part[col] = v;
      }
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int col = (c * threads + t) * 8 + i;
          if (col < a.H) part[col] = dw[c][i];
        }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) dw[c][i] = 0.f;
  }
}

// dw[col] (+)= the sum of its column, 32 columns a block
__global__ void __launch_bounds__(256) rms_norm_dw_kernel(const float* __restrict__ part, int64_t n, int H, void* dw, int f32,
                                                          int accumulate) {
  __shared__ double sums[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  double s = 0.0;
  if (col < H) {
#pragma unroll 8
    for (int64_t i = warp; i < n; i += 8) s += part[i * H + col];
  }
  sums[warp][lane] = s;
  __syncthreads();
  if (warp || col >= H) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += sums[i][lane];
  if (f32) {
    float* p = (float*)dw + col;
    *p = accumulate ? (float)(*p + s) : (float)s;
  } else {
    ((__nv_bfloat16*)dw)[col] = __float2bfloat16_rn(norm_for_bf16(s));
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
struct NormShape {
  int warps, rows, nc;
  explicit NormShape(int H) {
    nc = H > kNormMaxWarps * 512 ? 4 : 2;
    warps = 1;
    while (warps * 32 * 8 * nc < H) warps *= 2;
    rows = warps == 1 ? 8 : 1;
  }
  int threads() const { return 32 * warps * rows; }
};

static bool norm_vec(const void* p, bool f32, int64_t ld, int64_t H) {
  return ((uintptr_t)p & 15) == 0 && H % 8 == 0 && ld % (f32 ? 4 : 8) == 0;
}

template <bool XF32, int RES, int QUANT>
static cudaError_t norm_launch(const NormArgs& a, const NormShape& sh, cudaStream_t stream) {
  const unsigned blocks = (unsigned)((a.T + sh.rows - 1) / sh.rows);
  if (sh.nc == 2) rms_norm_kernel<XF32, RES, QUANT, 2><<<blocks, sh.threads(), 0, stream>>>(a);
  else rms_norm_kernel<XF32, RES, QUANT, 4><<<blocks, sh.threads(), 0, stream>>>(a);
  return cudaGetLastError();
}
template <int RES>
static cudaError_t norm_launch_bf16(const NormArgs& a, const NormShape& sh, int quant, cudaStream_t stream) {
  return quant == NORM_MX         ? norm_launch<false, RES, NORM_MX>(a, sh, stream)
         : quant == NORM_BLOCK128 ? norm_launch<false, RES, NORM_BLOCK128>(a, sh, stream)
                                  : norm_launch<false, RES, NORM_PLAIN>(a, sh, stream);
}

template <bool XF32, bool HF32, int NC>
static int norm_bwd_launch(const NormBwdArgs& a, const NormShape& sh, int blocks, cudaStream_t stream) {
  const size_t smem = sh.rows > 1 && a.part ? (size_t)sh.rows * a.H * 4 : 0;       // at most 8 x 512 x 4 bytes
  rms_norm_bwd_kernel<XF32, HF32, NC><<<blocks, sh.threads(), smem, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? SMOE_OK : SMOE_ERR_LAUNCH;
}

static int norm_bwd_blocks(int64_t T, const NormShape& sh) {
  const int64_t most = (int64_t)sm_count() * (1024 / sh.threads()), all = (T + sh.rows - 1) / sh.rows;
  return (int)(all < most ? all : most);
}
static int norm_flushes(int64_t T, const NormShape& sh, int blocks) {
  const int64_t turns = (T + (int64_t)blocks * sh.rows - 1) / ((int64_t)blocks * sh.rows);
  return (int)((turns + kNormRun - 1) / kNormRun);
}
static bool norm_sizes(int64_t T, int64_t H) { return T >= 0 && T < (int64_t)1 << 31 && H > 0 && H <= kNormMaxH; }

}  // namespace smoe

using namespace smoe;

extern "C" {

int smoe_rms_norm(const void* x, int x_f32, int64_t ldx, const void* residual, int residual_f32, int64_t ldr, const void* w, int w_f32,
                  int64_t T, int64_t H, double eps, void* y, void* h, double* rstd, int scale_kind, void* q, void* scales,
                  void* stream) {
  if (!norm_sizes(T, H) || ldx < H || (residual && ldr < H)) return SMOE_ERR_SHAPE;
  if (scale_kind < 0 || scale_kind > 2 || !(eps >= 0) || (x_f32 && (scale_kind || (residual && !residual_f32)))) return SMOE_ERR_ARG;
  if ((scale_kind == NORM_MX && H % 32) || (scale_kind == NORM_BLOCK128 && H % 8)) return SMOE_ERR_SHAPE;
  if (T == 0) return SMOE_OK;
  if (!x || !w || (residual && !h) || (scale_kind ? !q || !scales : !y)) return SMOE_ERR_ARG;
  if (scale_kind && (uintptr_t)q & 15) return SMOE_ERR_ALIGN;
  const NormShape sh((int)H);
  NormArgs a{};
  a.x = x; a.res = residual; a.w = w; a.ldx = ldx; a.ldr = ldr; a.T = T; a.H = (int)H;
  a.warps = sh.warps; a.rows = sh.rows; a.w_f32 = w_f32 != 0; a.eps = eps; a.inv_H = 1.0 / (double)H;
  const bool h_f32 = x_f32 || (residual && residual_f32);
  a.vec_x = norm_vec(x, x_f32, ldx, H);
  a.vec_r = norm_vec(residual, h_f32, ldr, H);
  a.vec_w = norm_vec(w, w_f32, H, H);
  a.vec_y = norm_vec(y, x_f32, H, H);
  a.vec_h = norm_vec(h, h_f32, H, H);
  a.y = y; a.h = h; a.rstd = rstd; a.q = (uint8_t*)q; a.s = scales; a.pitch = (H + 15) / 16 * 16;
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t rc;
  if (x_f32) rc = residual ? norm_launch<true, 1, NORM_PLAIN>(a, sh, st) : norm_launch<true, 0, NORM_PLAIN>(a, sh, st);
  else if (!residual) rc = norm_launch_bf16<0>(a, sh, scale_kind, st);
  else rc = residual_f32 ? norm_launch_bf16<2>(a, sh, scale_kind, st) : norm_launch_bf16<1>(a, sh, scale_kind, st);
  return rc == cudaSuccess ? SMOE_OK : SMOE_ERR_LAUNCH;
}

int64_t smoe_rms_norm_bwd_workspace(int64_t T, int64_t H) {
  if (!norm_sizes(T, H)) return -1;
  if (T == 0) return 0;
  const NormShape sh((int)H);
  const int blocks = norm_bwd_blocks(T, sh);
  return (int64_t)blocks * norm_flushes(T, sh, blocks) * H * 4;
}

int smoe_rms_norm_bwd(const void* dy, int x_f32, const void* h, int h_f32, int64_t ldh, const void* w, int w_f32, const double* rstd,
                      const void* dh, int64_t T, int64_t H, void* dx, void* dres, void* dw, int dw_f32, int dw_accumulate,
                      void* workspace, void* stream) {
  if (!norm_sizes(T, H) || ldh < H) return SMOE_ERR_SHAPE;
  if ((x_f32 && !h_f32) || (dw_accumulate && !dw_f32)) return SMOE_ERR_ARG;
  const cudaStream_t st = (cudaStream_t)stream;
  if (T == 0) {                                          // an empty sum
    if (!dw || dw_accumulate) return SMOE_OK;
    return cudaMemsetAsync(dw, 0, (size_t)H * (dw_f32 ? 4 : 2), st) == cudaSuccess ? SMOE_OK : SMOE_ERR_LAUNCH;
  }
  if (!dy || !h || !w || !rstd || (dw && !workspace)) return SMOE_ERR_ARG;
  const NormShape sh((int)H);
  const int blocks = norm_bwd_blocks(T, sh);
  NormBwdArgs a{};
  a.dy = dy; a.h = h; a.w = w; a.dh = dh; a.rstd = rstd; a.ldh = ldh; a.T = T; a.H = (int)H;
  a.warps = sh.warps; a.rows = sh.rows; a.w_f32 = w_f32 != 0;
  a.vec_dy = norm_vec(dy, x_f32, H, H);
  a.vec_h = norm_vec(h, h_f32, ldh, H);
  a.vec_w = norm_vec(w, w_f32, H, H);
  a.vec_dh = norm_vec(dh, h_f32, H, H);
  a.vec_dx = norm_vec(dx, x_f32, H, H);
  a.vec_dres = norm_vec(dres, h_f32, H, H);
  a.dx = dx; a.dres = dres;
  a.part = dw ? (float*)workspace : nullptr;
  a.flushes = norm_flushes(T, sh, blocks);
  int rc;
  if (x_f32) rc = sh.nc == 2 ? norm_bwd_launch<true, true, 2>(a, sh, blocks, st) : norm_bwd_launch<true, true, 4>(a, sh, blocks, st);
  else if (h_f32) rc = sh.nc == 2 ? norm_bwd_launch<false, true, 2>(a, sh, blocks, st) : norm_bwd_launch<false, true, 4>(a, sh, blocks, st);
  else rc = sh.nc == 2 ? norm_bwd_launch<false, false, 2>(a, sh, blocks, st) : norm_bwd_launch<false, false, 4>(a, sh, blocks, st);
  if (rc || !dw) return rc;
  rms_norm_dw_kernel<<<(unsigned)((H + 31) / 32), 256, 0, st>>>((const float*)workspace, (int64_t)blocks * a.flushes, (int)H, dw,
                                                               dw_f32 != 0, dw_accumulate != 0);
  return cudaGetLastError() == cudaSuccess ? SMOE_OK : SMOE_ERR_LAUNCH;
}

}  // extern "C"
