// Root-mean-square norm of rows in front of the experts, with the residual's addition before it and the 8-bit payload behind it.
//
//   h = x + residual (held in the residual's type)      r = 1 / sqrt(mean(h^2) + eps)      y = h r w
//   backward, g = dy w:  dh = r (g - h r^2 mean(g h)) + the gradient that comes in for h;   dw = sum over rows of dy h r
//
// A row is held in registers between its one read and its one write; a block stays and asks for its next row before it adds this one up.
// bf16 results and what is quantised from them are those of 64 bits: the mean and r are f64, y is made in f32 and looked at: where it
// lies within kNormNear of the border between two bf16 values it is made again in f64 (one in 7000), where one that is a tie but for the
// roundings of f64 counts as a tie.
//   What bounds it: HBM.  8192 x 4096 bf16 with residual, rows 43 us (6.2 TB/s), rows and payload 50 (6.1 TB/s); residual in f32 67 (6.0
//   TB/s), with payload 70 (6.2); 262144 x 128 47 (5.7 TB/s).  Without residual issue: 8192 x 4096 31 us (4.4 TB/s).  Backward, 16384 x 2048
//   bf16 49 us (5.5 TB/s), 8192 x 4096 with h in f32 94 (5.7): the column sums of dw take the registers that would keep more rows on their
//   way.  A single row takes 2.4 to 2.9 us.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "host.h"
#include "ptx.cuh"
#include "quant_groups.cuh"
#include "smoe_b200.h"

namespace smoe {

constexpr int kNormMaxH = 16384;
constexpr int kNormMaxWarps = 16;
constexpr double kNormLeastEps = 1e-90;    // the root's argument is brought into the range of f32: so far (a row that is not zero has 1e-94)

// ---- pairs of f32 in one instruction (round to nearest, as the scalar forms)
struct P2 {
  uint64_t v;
};
__device__ __forceinline__ P2 p2(float x, float y) {
  P2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 p2_get(P2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ P2 operator*(P2 a, P2 b) {
  P2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ P2 operator+(P2 a, P2 b) {
  P2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ P2 p2_fma(P2 a, P2 b, P2 c) {
  P2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

template <bool F32>
struct NormVec;                          // eight values of a row
template <>
struct NormVec<false> {
  uint32_t w[4];
  __device__ __forceinline__ void load(const void* base, int64_t at) {
    const uint4 v = *reinterpret_cast<const uint4*>((const uint16_t*)base + at);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
  // value i from at + i * step, the first n of them
  __device__ __forceinline__ void load_some(const void* base, int64_t at, int n, int step) {
    const uint16_t* p = (const uint16_t*)base + at;
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = i < n ? p[i * step] : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = u[2 * i] | u[2 * i + 1] << 16;
  }
  __device__ __forceinline__ P2 pair(int i) const { return p2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u)); }
  __device__ __forceinline__ void set(int i, P2 v) {
    const float2 f = p2_get(v);
    w[i] = q_bf16x2(f.x, f.y);
  }
  __device__ __forceinline__ void clear() { w[0] = w[1] = w[2] = w[3] = 0u; }
  // what follows from the values is made anew, here and not ahead of a loop
  __device__ __forceinline__ void anew() { asm volatile("" : "+r"(w[0]), "+r"(w[1]), "+r"(w[2]), "+r"(w[3])); }
  __device__ __forceinline__ void store(void* base, int64_t at) const {
    *reinterpret_cast<uint4*>((uint16_t*)base + at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void store_some(void* base, int64_t at, int n, int step) const {
    uint16_t* p = (uint16_t*)base + at;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i * step] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
  }
};
template <>
struct NormVec<true> {
  float f[8];
  __device__ __forceinline__ void load(const void* base, int64_t at) {
    const float4* p = reinterpret_cast<const float4*>((const float*)base + at);
    const float4 a = p[0], b = p[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  __device__ __forceinline__ void load_some(const void* base, int64_t at, int n, int step) {
    const float* p = (const float*)base + at;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? p[i * step] : 0.f;
  }
  __device__ __forceinline__ P2 pair(int i) const { return p2(f[2 * i], f[2 * i + 1]); }
  __device__ __forceinline__ void set(int i, P2 v) {
    const float2 x = p2_get(v);
    f[2 * i] = x.x;
    f[2 * i + 1] = x.y;
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.f;
  }
  __device__ __forceinline__ void anew() {
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("" : "+f"(f[i]));
  }
  __device__ __forceinline__ void store(void* base, int64_t at) const {
    float4* p = reinterpret_cast<float4*>((float*)base + at);
    p[0] = make_float4(f[0], f[1], f[2], f[3]);
    p[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
  __device__ __forceinline__ void store_some(void* base, int64_t at, int n, int step) const {
    float* p = (float*)base + at;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i * step] = f[i];
  }
};

// A row's columns among the `threads` threads of it, of which this one is t.  H a multiple of 8: piece c of a thread is eight columns
// from (c * threads + t) * 8 on, with VEC by 16 bytes of every tensor.  Else its values are `threads` columns apart, so that the loads
// of a warp lie side by side (eight neighbours a thread: T=1003, H=1001 in f32, forward and backward 30 us instead of 14).  Kernels of
// their own: what the loads one by one keep in registers over a row leaves too few for the others.
template <bool VEC>
struct NormRow {
  int t, threads, H;
  bool apart;
  __device__ __forceinline__ int col(int c) const { return !VEC && apart ? c * 8 * threads + t : (c * threads + t) * 8; }
  __device__ __forceinline__ int step() const { return !VEC && apart ? threads : 1; }
  __device__ __forceinline__ int left(int col) const {      // values of a piece that exist
    return apart ? (H - col + threads - 1) / threads : H - col;
  }
  template <bool F32, int NC>
  __device__ __forceinline__ void load(NormVec<F32> (&v)[NC], const void* base, int64_t row_at) const {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int at = col(c);
      if (VEC) {
        v[c].clear();
        if (at < H) v[c].load(base, row_at + at);
      } else {
        v[c].load_some(base, row_at + at, left(at), step());
      }
    }
  }
  template <bool F32>
  __device__ __forceinline__ void store(const NormVec<F32>& v, void* base, int64_t row_at, int c) const {
    const int at = col(c);
    if (VEC) {
      if (at < H) v.store(base, row_at + at);
    } else {
      v.store_some(base, row_at + at, left(at), step());
    }
  }
};

// over the threads of a row, in one order; `group` of the block's rows it is, each of several warps with sums and a barrier of its own
template <bool NARROW, typename T>
__device__ __forceinline__ T norm_sum(T s, int threads, int group, T* shared) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1)
    if (!NARROW || d < threads) s += __shfl_xor_sync(0xffffffffu, s, d);
  if (NARROW || threads == 32) return s;
  const int warps = threads >> 5;
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = s;
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(warps * 32) : "memory");
  shared += group * warps;
  s = shared[0] + shared[1];
  for (int i = 2; i < warps; i += 2) s += shared[i] + (i + 1 < warps ? shared[i + 1] : T(0));
  return s;
}

// 1 / sqrt(v) to the last place: with y the f32 approximation and e = 1 - v y^2, y (1 - e)^(-1/2) = y (1 + e / 2 + 3 e^2 / 8 + 5 e^3 / 16 ...), of
// which the third power, 2^-66, is left out; v is brought into the range of f32
__device__ __forceinline__ double norm_rsqrt(double v) {
  const double scale = v < 1e-30 ? 0x1p200 : v > 1e30 ? 0x1p-200 : 1.0, back = v < 1e-30 ? 0x1p100 : v > 1e30 ? 0x1p-100 : 1.0;
  v *= scale;
  const float r = rsqrtf((float)v);
  if (!(r > 0.f && r < __int_as_float(0x7f800000))) return r;      // of 0, infinity, NaN
  const double y = r, e = fma(-v * y, y, 1.0);
  return fma(y, e * fma(0.375, e, 0.5), y) * back;
}

// h r w in f32 is off by three roundings (r, two products), each up to one unit of the last place
constexpr uint32_t kNormNear = 4;
__device__ __forceinline__ uint32_t norm_min_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// f32 that rounds to the bf16 nearest to d: a tie of f32 that is none of f64 is moved off.  What is a tie but for `slack` of its size is one.
__device__ __forceinline__ float norm_for_bf16(double d, double slack) {
  float f = (float)d;
  if ((__float_as_uint(f) & 0xFFFFu) == 0x8000u) {
    const double away = fabs(d) - fabs((double)f), least = fabs(d) * slack;
    if (away > least) f = __uint_as_float(__float_as_uint(f) + 1);
    if (away < -least) f = __uint_as_float(__float_as_uint(f) - 1);
  }
  return f;
}
// Rounding of the mean (of its quotient, which is a product, and of eps's addition), r and h w r in f64: 2^-51 of a value that is a tie, as
// those of equal magnitudes whose weight lies between two bf16 are
constexpr double kNormTie = 0x1p-50;

struct NormArgs {
  const void *x, *res, *w;
  int64_t ldx, ldr, T;
  int H, lanes, rows;                    // threads of a row, rows of a block
  int w_f32, vec, apart;                 // vec: see NormRow
  double eps, inv_H;
  void *y, *h;                           // null: not written
  double* rstd;
  uint8_t* q;
  void* s;
  int64_t pitch;                         // of the payload
};

enum NormQuant : int { NORM_PLAIN = 0, NORM_MX = 1, NORM_BLOCK128 = 2 };

// Blocks an SM has at a time: two where h is f32, for the registers of the next row (us, two / three without it: 8192 x 4096 with residual
// in f32, rows and payload 69 / 71, 131072 x 128 39 / 45, 3001 x 1000, rows alone, 7.4 / 6.7, for which two take three turns instead of two).
constexpr int norm_blocks(bool h_f32, int pieces) { return pieces > 2 ? 1 : h_f32 ? 2 : 3; }

// RES: 0 none, 1 of x's type, 2 f32 (beside bf16).  A block stays and takes rows in turn, several at a time, each by threads of its own;
// a row's loads leave before the one ahead of it is added up.  NARROW: several rows a warp, of which those behind the last one have no
// columns.
template <bool XF32, int RES, int QUANT, int NC, bool WF32, bool VEC, bool NARROW>
__global__ void __launch_bounds__(NC == 2 ? 256 : 512, norm_blocks(XF32 || RES == 2, NC)) rms_norm_kernel(const NormArgs a) {
  constexpr bool HF32 = XF32 || RES == 2;
  // (x and residual both in f32 would need more registers: 8192 x 2048 53 us ahead and 44 so)
  constexpr bool AHEAD = VEC && (NC == 2 ? !(XF32 && RES) : !HF32);
  __shared__ double sums[2][kNormMaxWarps];
  const int lane = threadIdx.x & 31;
  const int group = threadIdx.x / a.lanes, in_warp = NARROW ? lane / a.lanes : 0;
  NormRow<VEC> at{(int)threadIdx.x - group * a.lanes, a.lanes, a.H, QUANT == NORM_PLAIN && a.apart};
  const int64_t stride = (int64_t)gridDim.x * a.rows;
  int64_t first = (int64_t)blockIdx.x * a.rows + group - in_warp;   // of the rows of this warp
  if (first >= a.T) return;
  NormVec<XF32> x[NC];
  NormVec<HF32> res[RES ? NC : 1];
  auto ask = [&](int64_t first) {
    if (first >= a.T) return;
    const int64_t of = first + in_warp;
    NormRow<VEC> in = at;
    in.H = !NARROW || of < a.T ? a.H : 0;
    in.load(x, a.x, of * a.ldx);
    if constexpr (RES != 0) in.load(res, a.res, of * a.ldr);
  };
  if (AHEAD) ask(first);
  NormVec<WF32> w[NC];
  at.load(w, a.w, 0);
  int turn = 0;
  for (; first < a.T; first += stride) {
    if (!AHEAD) ask(first);
    const int64_t row = first + in_warp;
    if (NARROW) at.H = row < a.T ? a.H : 0;
    NormVec<HF32> h[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if constexpr (RES == 0) {
        h[c] = x[c];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (!HF32) asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(h[c].w[i]) : "r"(x[c].w[i]), "r"(res[c].w[i]));
          else h[c].set(i, x[c].pair(i) + res[c].pair(i));
        }
      }
    }
    if (AHEAD) ask(first + stride);
    if constexpr (RES != 0) {
#pragma unroll
      for (int c = 0; c < NC; ++c) at.store(h[c], a.h, row * a.H, c);
    }
    double s0 = 0.0, s1 = 0.0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = p2_get(h[c].pair(i));
        const double p = f.x, q = f.y;
        s0 = fma(p, p, s0);
        s1 = fma(q, q, s1);
      }
    }
    const double r64 = norm_rsqrt(norm_sum<NARROW>(s0 + s1, a.lanes, group, sums[turn]) * a.inv_H + a.eps);
    turn ^= 1;                                            // the next row's sums do not wait for this one's readers
    const float r = (float)r64;
    if (a.rstd && at.t == 0 && (!NARROW || at.H)) a.rstd[row] = r64;
    const bool far = !(r64 > 1e-30 && r64 < 1e30);        // r in f32 would not have its full precision
    const P2 r2 = p2(r, r);
    NormVec<false> kept[NARROW && QUANT == NORM_BLOCK128 ? NC : 1];
    // y of columns from col on, whose group's largest magnitude is m
    auto quantise128 = [&](const NormVec<false>& y, uint32_t m, int col, bool first_of_group) {
      m &= 0x7FFF7FFFu;
      const float amax = fmaxf(fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u)), kAmaxFloor);
      // one division a lane, of either kind
      const float quotient = ((lane & 1) ? kE4m3Max : amax) / ((lane & 1) ? amax : kE4m3Max);
      const float qs = __shfl_sync(0xffffffffu, quotient, lane | 1);
      float2 b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = p2_get(y.pair(i) * p2(qs, qs));
      if (col < at.H) {
        *reinterpret_cast<uint2*>(a.q + row * a.pitch + col) =
            make_uint2(q_pack4(b[0].x, b[0].y, b[1].x, b[1].y), q_pack4(b[2].x, b[2].y, b[3].x, b[3].y));
        if (first_of_group) ((float*)a.s)[row * ((a.H + 127) >> 7) + (col >> 7)] = quotient;
      }
    };
    auto largest = [](const NormVec<false>& y) {
      return q_max_abs_bf16x2(q_max_abs_bf16x2(y.w[0], y.w[1]), q_max_abs_bf16x2(y.w[2], y.w[3]));
    };
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int col = at.col(c);
      P2 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = h[c].pair(i) * r2 * w[c].pair(i);
      if constexpr (XF32) {
        NormVec<true> y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y.set(i, v[i]);
        if (far) {
          NormVec<HF32> hc = h[c];
          NormVec<WF32> wc = w[c];
          hc.anew();
          wc.anew();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 f = p2_get(hc.pair(i >> 1)), g = p2_get(wc.pair(i >> 1));
            y.f[i] = (float)((double)(i & 1 ? f.y : f.x) * r64 * (double)(i & 1 ? g.y : g.x));
          }
        }
        at.store(y, a.y, row * a.H, c);
      } else {
        // least distances above a border less kNormNear, of the even and the odd values (a carry makes an odd one's one more)
        uint32_t near = 0xFFFFFFFFu;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = p2_get(v[i]);
          near = norm_min_u16x2(near, __byte_perm(__float_as_uint(f.x), __float_as_uint(f.y), 0x5410) + (0x8000u + kNormNear) * 0x10001u);
        }
        if ((near & 0xFFFFu) <= 2 * kNormNear || near < (2 * kNormNear + 2) << 16 || far) {
          // (anew: what is f64 of these values here would otherwise be kept from the sum of squares, and the weights' over all rows)
          NormVec<HF32> hc = h[c];
          NormVec<WF32> wc = w[c];
          hc.anew();
          wc.anew();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = p2_get(hc.pair(i)), g = p2_get(wc.pair(i));
            v[i] = p2(norm_for_bf16((double)f.x * (double)g.x * r64, kNormTie), norm_for_bf16((double)f.y * (double)g.y * r64, kNormTie));
          }
        }
        NormVec<false> y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y.set(i, v[i]);
        if (QUANT == NORM_PLAIN || a.y) at.store(y, a.y, row * a.H, c);
        if constexpr (QUANT == NORM_MX) {                 // four lanes a group
          uint32_t m = largest(y);
          m = q_max_abs_bf16x2(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = q_max_abs_bf16x2(m, __shfl_xor_sync(0xffffffffu, m, 2));
          m &= 0x7FFF7FFFu;
          const int e = q_e8m0_of(fmaxf(fmaxf(0.f, __uint_as_float(m << 16)), __uint_as_float(m & 0xFFFF0000u)));
          const uint32_t qs = (__float_as_uint(q_scale_of(e)) >> 16) * 0x10001u;      // a power of two is a bf16
          if (col < at.H) {
            *reinterpret_cast<uint2*>(a.q + row * a.pitch + col) =
                make_uint2(q_pack4_scaled(y.w[0], y.w[1], qs, qs), q_pack4_scaled(y.w[2], y.w[3], qs, qs));
            if ((lane & 3) == 0) ((uint8_t*)a.s)[row * (a.H >> 5) + (col >> 5)] = (uint8_t)e;
          }
        }
        if constexpr (QUANT == NORM_BLOCK128 && NARROW) kept[c] = y;
        if constexpr (QUANT == NORM_BLOCK128 && !NARROW) {      // sixteen
          uint32_t m = largest(y);
#pragma unroll
          for (int d = 1; d < 16; d <<= 1) m = q_max_abs_bf16x2(m, __shfl_xor_sync(0xffffffffu, m, d));
          quantise128(y, m, col, (lane & 15) == 0);
        }
      }
    }
    if constexpr (QUANT == NORM_BLOCK128 && NARROW) {     // sixteen lanes, or all of a row's two pieces
      const bool one = a.lanes < 16;
      uint32_t both = largest(kept[0]);
      if (one) both = q_max_abs_bf16x2(both, largest(kept[NC - 1]));
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint32_t m = c == 0 || one ? both : largest(kept[c]);
#pragma unroll
        for (int d = 1; d < 16; d <<= 1)
          if (d < a.lanes) m = q_max_abs_bf16x2(m, __shfl_xor_sync(0xffffffffu, m, d));
        quantise128(kept[c], m, at.col(c), at.t == 0 && (c == 0 || !one));
      }
    }
  }
}

// ---- backward -----------------------------------------------------------------------------------------------------------
struct NormBwdArgs {
  const void *dy, *h, *w, *dh;           // dh: null if none comes in
  const double* rstd;
  int64_t ldh, T;
  int H, lanes, rows;
  int w_f32, vec, apart;
  void *dx, *dres;                       // null: not wanted
  float* part;                           // [blocks * flushes, H], null: no gradient of the weight
  int flushes;
};

// Rows that a thread adds up in one f32 sum of a column; the sums of sums are f64
constexpr int kNormRun = 256;

// dx of x's type, dres of h's (where the two types differ; else dx serves both).  A block stays and takes rows in turn, several at a
// time, each by threads of its own, which keep their columns' part of dw in registers.  NARROW: as in
// the forward pass.
template <bool XF32, bool HF32, int NC, bool WF32, bool VEC, bool NARROW>
__global__ void __launch_bounds__(32 * kNormMaxWarps, 1) rms_norm_bwd_kernel(const NormBwdArgs a) {
  extern __shared__ float columns[];                    // [rows, or warps if they are fewer, H]
  next_kernel_may_start();                              // (the sums of the blocks' sums, which waits)
  __shared__ float sums[2][kNormMaxWarps];
  const int group = threadIdx.x / a.lanes, in_warp = NARROW ? (threadIdx.x & 31) / a.lanes : 0;
  const NormRow<VEC> at{(int)threadIdx.x - group * a.lanes, a.lanes, a.H, a.apart != 0};
  const int64_t stride = (int64_t)gridDim.x * a.rows;
  NormVec<WF32> w[NC];
  at.load(w, a.w, 0);
  P2 dw[NC][4];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) dw[c][i] = p2(0.f, 0.f);
  const float inv_H = 1.f / a.H;
  int turn = 0;
  int64_t first = (int64_t)blockIdx.x * a.rows + group - in_warp;   // of the rows of this warp
  // A row's loads leave before the one ahead of it is added up, which by then is held as h r and g.  (Rows in f32, or four pieces a thread:
  // neither, for want of registers; 8192 x 4096 with h in f32 109 us ahead and 94 so.)
  constexpr bool AHEAD = NC == 2 && !HF32;
  NormVec<XF32> dy[NC];
  NormVec<HF32> h[NC], dh[NC], next_dh[AHEAD ? NC : 1];
  double next_r = 1.0;
  auto ask = [&](int64_t first) {                       // (a row behind the last one adds zeros)
    if (first >= a.T) return;
    const int64_t of = first + in_warp;
    NormRow<VEC> in = at;
    in.H = !NARROW || of < a.T ? a.H : 0;
    in.load(dy, a.dy, of * a.H);
    in.load(h, a.h, of * a.ldh);
    if constexpr (AHEAD) {
      if (a.dh) in.load(next_dh, a.dh, of * a.H);
    } else {
      if (a.dh) in.load(dh, a.dh, of * a.H);
    }
    next_r = !NARROW || in.H ? a.rstd[of] : 0.0;
  };
  if (AHEAD) ask(first);
  for (int flush = 0; flush < a.flushes; ++flush) {
    for (int n = 0; n < kNormRun && first < a.T; ++n, first += stride) {
      if (!AHEAD) ask(first);
      const int64_t row = first + in_warp;
      NormRow<VEC> to = at;
      to.H = !NARROW || row < a.T ? a.H : 0;
      if (AHEAD) {                                      // (the weights unpacked anew: 16 registers less)
#pragma unroll
        for (int c = 0; c < NC; ++c) w[c].anew();
      }
      // r as a product of two f32, the first a power of two, so that rows of very large or very small values keep their precision
      const double r64 = next_r;
      const float pre = r64 < 1e-30 ? 0x1p-64f : r64 > 1e30 ? 0x1p64f : 1.f;
      const float r = (float)(r64 * (r64 < 1e-30 ? 0x1p64 : r64 > 1e30 ? 0x1p-64 : 1.0));
      const P2 pre2 = p2(pre, pre), r2 = p2(r, r);
      P2 s2 = p2(0.f, 0.f), hr[AHEAD ? NC : 1][4], g[AHEAD ? NC : 1][4];
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const P2 d = dy[c].pair(i), u = h[c].pair(i) * pre2 * r2, v = d * w[c].pair(i);
          s2 = p2_fma(v, u, s2);
          dw[c][i] = p2_fma(d, u, dw[c][i]);
          if constexpr (AHEAD) {
            hr[c][i] = u;
            g[c][i] = v;
          }
        }
      if constexpr (AHEAD) {
#pragma unroll
        for (int c = 0; c < NC; ++c) dh[c] = next_dh[c];
        ask(first + stride);
      }
      const float2 both = p2_get(s2);
      const float s = norm_sum<NARROW>(both.x + both.y, a.lanes, group, sums[turn]) * -inv_H;
      turn ^= 1;                                        // the next row's sums do not wait for this one's readers
      const P2 minus = p2(s, s);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        P2 d[4];
        if constexpr (!AHEAD) {
          dy[c].anew();
          h[c].anew();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (AHEAD) d[i] = p2_fma(hr[c][i], minus, g[c][i]);
          else d[i] = p2_fma(h[c].pair(i) * pre2 * r2, minus, dy[c].pair(i) * w[c].pair(i));
          d[i] = d[i] * r2 * pre2;
          if (a.dh) d[i] = d[i] + dh[c].pair(i);
        }
        if (a.dx) {
          NormVec<XF32> o;
#pragma unroll
          for (int i = 0; i < 4; ++i) o.set(i, d[i]);
          to.store(o, a.dx, row * a.H, c);
        }
        if constexpr (XF32 != HF32) {
          if (a.dres) {
            NormVec<HF32> o;
#pragma unroll
            for (int i = 0; i < 4; ++i) o.set(i, d[i]);
            to.store(o, a.dres, row * a.H, c);
          }
        }
      }
    }
    if (!a.part) continue;
    float* part = a.part + ((int64_t)blockIdx.x * a.flushes + flush) * a.H;
    const int sums_of = NARROW ? kNormMaxWarps : a.rows;
    float* mine = sums_of > 1 ? columns + (NARROW ? threadIdx.x >> 5 : group) * a.H : part;
    if (NARROW) {                                       // the warp's rows first
#pragma unroll
      for (int d = 16; d > 0; d >>= 1)
        if (d >= a.lanes) {
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) dw[c][i] = dw[c][i] + P2{__shfl_xor_sync(0xffffffffu, dw[c][i].v, d)};
        }
    }
    if (sums_of > 1) __syncthreads();                   // the flush before has been read
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int col = at.col(c) + i * at.step();
        const float2 v = p2_get(dw[c][i >> 1]);
        if (col < a.H && in_warp == 0) mine[col] = i & 1 ? v.y : v.x;
      }
    if (sums_of > 1) {                                  // the block's rows first
      __syncthreads();
      for (int col = threadIdx.x; col < a.H; col += blockDim.x) {
        float v = columns[col];
        for (int k = 1; k < sums_of; ++k) v += columns[k * a.H + col];
        part[col] = v;
      }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) dw[c][i] = p2(0.f, 0.f);
  }
}

// dw[col] (+)= the sum of its column, 32 columns a block
constexpr int kNormSumWarps = 32;
__global__ void __launch_bounds__(32 * kNormSumWarps) rms_norm_dw_kernel(const float* part, int64_t n, int H, void* dw,
                                                                         int f32, int accumulate) {
  __shared__ double sums[kNormSumWarps][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int col = blockIdx.x * 32 + lane;
  double s = 0.0;
  wait_for_kernel_before();
  if (col < H) {
#pragma unroll 8
    for (int64_t i = warp; i < n; i += kNormSumWarps) s += part[i * H + col];
  }
  sums[warp][lane] = s;
  __syncthreads();
  col = blockIdx.x * 32 + warp;                         // a warp a column
  s = sums[lane][warp];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  if (lane || col >= H) return;
  if (f32) {
    float* p = (float*)dw + col;
    if (accumulate) atomicAdd(p, (float)s);             // (once for each value: another stream's sums into it are not lost)
    else *p = (float)s;
  } else {
    ((__nv_bfloat16*)dw)[col] = __float2bfloat16_rn(norm_for_bf16(s, 0.0));
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
// Threads of a row of `nc` pieces a thread, at least `least`, and rows a block has at a time: as many warps as it fills, not a power of two
// (us, a power / so, bf16 with residual, rows and payload: 8192 x 2560 42.4 / 33.4, x 5120 74 / 66; backward 41 / 35, 80 / 73; 3968 x 5088
// without residual 34 / 28.6).  Narrow rows share a warp (us, one / several a
// warp, bf16: 262144 x 128 85 / 26, with mx payload too 113 / 36, with 128-blocks alone 128 / 38, backward 100 / 39; x 64 85 / 14, backward
// 96 / 22; 131072 x 256 45 / 27).
struct NormShape {
  int lanes, rows;
  NormShape(int H, int nc, int block_warps, int least) {
    lanes = least;
    while (lanes * 8 * nc < H) lanes *= 2;
    if (lanes > 32) {                                    // (seven warps of a row burden an SM's quarters unevenly: 4096 x 7168 42 us, eight 39)
      const int warps = (H + 256 * nc - 1) / (256 * nc);
      lanes = (warps == 7 ? 8 : warps) * 32;
    }
    rows = lanes < block_warps * 32 ? block_warps * 32 / lanes : 1;
  }
  int threads() const { return lanes * rows; }
};
static int norm_pieces(int H) { return H > 4096 ? 4 : 2; }
// (a group that is quantised together lies side by side in a warp)
static NormShape norm_forward_shape(int H, int quant) {
  return NormShape(H, norm_pieces(H), 8, quant == NORM_MX ? 4 : quant == NORM_BLOCK128 ? 2 : 1);
}
static int norm_bwd_pieces(int H) { return H > kNormMaxWarps * 512 ? 4 : 2; }
static NormShape norm_bwd_shape(int H) { return NormShape(H, norm_bwd_pieces(H), kNormMaxWarps, 1); }

// rows of it can be read by 16 bytes (null: there are none)
static bool norm_vec(const void* p, bool f32, int64_t ld, int64_t H) {
  if (!p) return H % 8 == 0;
  return ((uintptr_t)p & 15) == 0 && H % 8 == 0 && ld % (f32 ? 4 : 8) == 0;
}

template <bool XF32, int RES, int QUANT, int NC, bool NARROW>
static cudaError_t norm_launch_pieces(const NormArgs& a, const NormShape& sh, cudaStream_t stream) {
  const int64_t all = (a.T + sh.rows - 1) / sh.rows;
  const int64_t most = (int64_t)sm_count() * ((NC == 2 ? 256 * norm_blocks(XF32 || RES == 2, NC) : 512) / sh.threads());
  const unsigned blocks = (unsigned)(all < most ? all : most);
  if (a.vec) {
    if (a.w_f32) rms_norm_kernel<XF32, RES, QUANT, NC, true, true, NARROW><<<blocks, sh.threads(), 0, stream>>>(a);
    else rms_norm_kernel<XF32, RES, QUANT, NC, false, true, NARROW><<<blocks, sh.threads(), 0, stream>>>(a);
  } else {
    if (a.w_f32) rms_norm_kernel<XF32, RES, QUANT, NC, true, false, NARROW><<<blocks, sh.threads(), 0, stream>>>(a);
    else rms_norm_kernel<XF32, RES, QUANT, NC, false, false, NARROW><<<blocks, sh.threads(), 0, stream>>>(a);
  }
  return cudaGetLastError();
}
template <bool XF32, int RES, int QUANT>
static cudaError_t norm_launch(const NormArgs& a, const NormShape& sh, cudaStream_t stream) {
  if (sh.lanes < 32) return norm_launch_pieces<XF32, RES, QUANT, 2, true>(a, sh, stream);
  return norm_pieces(a.H) == 2 ? norm_launch_pieces<XF32, RES, QUANT, 2, false>(a, sh, stream)
                               : norm_launch_pieces<XF32, RES, QUANT, 4, false>(a, sh, stream);
}
template <int RES>
static cudaError_t norm_launch_bf16(const NormArgs& a, const NormShape& sh, int quant, cudaStream_t stream) {
  return quant == NORM_MX         ? norm_launch<false, RES, NORM_MX>(a, sh, stream)
         : quant == NORM_BLOCK128 ? norm_launch<false, RES, NORM_BLOCK128>(a, sh, stream)
                                  : norm_launch<false, RES, NORM_PLAIN>(a, sh, stream);
}

template <bool XF32, bool HF32, int NC, bool NARROW>
static int norm_bwd_launch(const NormBwdArgs& a, const NormShape& sh, int blocks, cudaStream_t stream) {
  const int sums = sh.rows < kNormMaxWarps ? sh.rows : kNormMaxWarps;
  const size_t smem = sums > 1 && a.part ? (size_t)sums * a.H * 4 : 0;              // at most 16 x 512 x 4 bytes
  if (a.vec) {
    if (a.w_f32) rms_norm_bwd_kernel<XF32, HF32, NC, true, true, NARROW><<<blocks, sh.threads(), smem, stream>>>(a);
    else rms_norm_bwd_kernel<XF32, HF32, NC, false, true, NARROW><<<blocks, sh.threads(), smem, stream>>>(a);
  } else {
    if (a.w_f32) rms_norm_bwd_kernel<XF32, HF32, NC, true, false, NARROW><<<blocks, sh.threads(), smem, stream>>>(a);
    else rms_norm_bwd_kernel<XF32, HF32, NC, false, false, NARROW><<<blocks, sh.threads(), smem, stream>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? SMOE_OK : SMOE_ERR_LAUNCH;
}
template <bool XF32, bool HF32>
static int norm_bwd_launch_any(const NormBwdArgs& a, const NormShape& sh, int blocks, cudaStream_t stream) {
  if (sh.lanes < 32) return norm_bwd_launch<XF32, HF32, 2, true>(a, sh, blocks, stream);
  return norm_bwd_pieces(a.H) == 2 ? norm_bwd_launch<XF32, HF32, 2, false>(a, sh, blocks, stream)
                                   : norm_bwd_launch<XF32, HF32, 4, false>(a, sh, blocks, stream);
}

static int norm_bwd_blocks(int64_t T, const NormShape& sh) {
  const int64_t most = sm_count(), all = (T + sh.rows - 1) / sh.rows;
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
  if (scale_kind < 0 || scale_kind > 2 || !(eps == 0 || eps >= kNormLeastEps) || (x_f32 && (scale_kind || (residual && !residual_f32)))) return SMOE_ERR_ARG;
  if ((scale_kind == NORM_MX && H % 32) || (scale_kind == NORM_BLOCK128 && H % 8)) return SMOE_ERR_SHAPE;
  if (T == 0) return SMOE_OK;
  if (!x || !w || (residual && !h) || (scale_kind ? !q || !scales : !y)) return SMOE_ERR_ARG;
  if (scale_kind && (uintptr_t)q & 15) return SMOE_ERR_ALIGN;
  const NormShape sh = norm_forward_shape((int)H, scale_kind);
  NormArgs a{};
  a.x = x; a.res = residual; a.w = w; a.ldx = ldx; a.ldr = ldr; a.T = T; a.H = (int)H;
  a.lanes = sh.lanes; a.rows = sh.rows; a.w_f32 = w_f32 != 0; a.apart = H % 8 != 0; a.eps = eps; a.inv_H = 1.0 / (double)H;
  const bool h_f32 = x_f32 || (residual && residual_f32);
  a.vec = norm_vec(x, x_f32, ldx, H) && norm_vec(residual, h_f32, ldr, H) && norm_vec(w, w_f32, H, H) && norm_vec(y, x_f32, H, H) &&
          norm_vec(h, h_f32, H, H);
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
  const NormShape sh = norm_bwd_shape((int)H);
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
  const NormShape sh = norm_bwd_shape((int)H);
  const int blocks = norm_bwd_blocks(T, sh);
  NormBwdArgs a{};
  a.dy = dy; a.h = h; a.w = w; a.dh = dh; a.rstd = rstd; a.ldh = ldh; a.T = T; a.H = (int)H;
  a.lanes = sh.lanes; a.rows = sh.rows; a.w_f32 = w_f32 != 0; a.apart = H % 8 != 0;
  a.vec = norm_vec(dy, x_f32, H, H) && norm_vec(h, h_f32, ldh, H) && norm_vec(w, w_f32, H, H) && norm_vec(dh, h_f32, H, H) &&
          norm_vec(dx, x_f32, H, H) && norm_vec(dres, h_f32, H, H);
  a.dx = dx; a.dres = dres;
  a.part = dw ? (float*)workspace : nullptr;
  a.flushes = norm_flushes(T, sh, blocks);
  int rc;
  if (x_f32) rc = norm_bwd_launch_any<true, true>(a, sh, blocks, st);
  else rc = h_f32 ? norm_bwd_launch_any<false, true>(a, sh, blocks, st) : norm_bwd_launch_any<false, false>(a, sh, blocks, st);
  if (rc || !dw) return rc;
  return launch_early(rms_norm_dw_kernel, (unsigned)((H + 31) / 32), 32 * kNormSumWarps, 0, 0, st, (const float*)workspace,
                      (int64_t)blocks * a.flushes, (int)H, dw, (int)(dw_f32 != 0), (int)(dw_accumulate != 0)) == cudaSuccess
             ? SMOE_OK
             : SMOE_ERR_LAUNCH;
}

}  // extern "C"
