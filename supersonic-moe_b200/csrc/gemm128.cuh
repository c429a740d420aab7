// Grouped products of e4m3 operands with one f32 scale per block of 128 (see quant128.cu), tcgen05 on CTA pairs.
//
//   ROWS128   c[r, n] = sum_kb as[r, kb] bs[e, n / 128, kb] (sum over the 128 k of kb of a[r, k] b[e][n, k])     rows by expert
//   WGRAD128  c[e][m, n] (+)= sum_tb as[tb, m] bs[tb, n] (sum over the 128 rows t of tb of a[t, m] b[t, n])      rows summed over
//
// f32 scales are not what the block-scaled MMA takes (powers of two, 32 wide), so the plain e4m3 MMA sums one block of 128 at a
// time into TMEM and the epilogue warps add it, scaled, to sums that stay in their registers: 128 f32 a thread, 256 x 256 outputs
// a CTA pair.  Two TMEM buffers of 256 columns: the MMAs of one block (512 clocks) run while the block before is read out (256
// clocks of TMEM reads, half as many of packed multiply-adds).
//   B [E, N, K] is read K-major, or with b_mn as [E, K, N] as it lies: the gradient of the rows needs no transposed weights.
//   Both operands of the weight gradient lie [rows, dim] and are read MN-major.
#pragma once
#include "gemm2.cuh"

namespace smoe {

enum Gemm128Mode : int { ROWS128 = 0, WGRAD128 = 1 };

struct Gemm128Params {
  int rows;                  // rows of the operand whose rows are cut into segments
  int M, N, K, E;            // M: rows of an expert's c (WGRAD128); N: columns of c; K: reduction length (ROWS128)
  const int *efo, *counts;   // [E+1] segments and [E] live rows; null: one segment of all rows, all rows of a segment live
  const float *a_s, *b_s;
  int64_t bs_e, bs_n;        // ROWS128: b's scales of expert e, column block j, reduction block kb: b_s[e*bs_e + j*bs_n + kb*bs_k]
  int bs_k, a_kb;            //          a's: a_s[row * a_kb + kb]
  int b_mn;
  void* c;                   // ROWS128: bf16 [rows, N]; WGRAD128: [E, M, N] f32 or bf16
  int out_bf16, accumulate;  // WGRAD128
  int zero_rest;             // ROWS128: rows that are not live are written as zero (else left as they are)
  int* status;
  volatile int* host_word;   // pinned mirror of *status, or null
};

// A wait ran out: the device word keeps the first code, and the host sees it without waiting for the GPU
__device__ __forceinline__ void fail128(int* status, volatile int* host_word, int code) {
  atomicCAS(status, 0, code);
  if (host_word) {
    *host_word = code;
    __threadfence_system();
  }
}

constexpr int kG128Segs = kMaxExperts2 + 1;        // the rows behind the last segment are one more

struct Gemm128Smem {
  static constexpr int A_BYTES = BM * BK, B_BYTES = 128 * BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES, STAGES = 6;
  static constexpr int EPI_WARPS = 8;
  static constexpr int STG_BYTES = 2048;                    // output staging of a warp
  static constexpr int SB_BYTES = 2 * 512;                  // WGRAD128: scales of a warp's 128 columns, two blocks
  static constexpr int AUX_BYTES = 512 + 4 * (kG128Segs + 1) * 4;
  static constexpr int TOTAL = 1024 + STAGES * STAGE_BYTES + EPI_WARPS * (STG_BYTES + SB_BYTES) + AUX_BYTES;
  // Two warpgroups of epilogue warps and one with the producer and the MMA issuer.  A thread of the former needs more than the 168
  // registers that three warps on each quarter of the SM leave: 2 x 224 + 56 = 3 x 168.
  static constexpr int THREADS = 32 * (EPI_WARPS + 4), EPI_REGS = 224, OTHER_REGS = 56;
  static constexpr uint32_t TX_BYTES = 2u * STAGE_BYTES;
  static_assert(TOTAL <= 227 * 1024, "shared memory budget");
  static_assert((2 * STAGES + 4) * 8 <= 496, "barrier storage");
};

// tcgen05.mma kind::f8f6f4: e4m3 x e4m3 -> f32
__host__ __device__ constexpr uint32_t make_idesc_f8(int M, int N, bool a_mn, bool b_mn) {
  return (1u << 4) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_f8_pair_lo(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %3};\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %4, p;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const void* tmap, uint32_t bar_cluster, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(tmap), "r"(bar_cluster), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* tmap, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(tmap), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// the values of a TMEM load are there from here on: nothing that reads them moves ahead of the wait
__device__ __forceinline__ void tmem_arrived(uint32_t (&r)[16]) {
  asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
               "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}

// Segments from efo / counts, any values taken as they fit: 0 <= start <= end <= rows, start <= live end <= end
struct Segs128 {
  int *start, *live, *tiles;       // [segs + 1] starts; [segs] ends of the live rows; [segs + 1] row tiles before
};
// one warp; segment `E` holds the rows behind the last one, none of them live
__device__ __forceinline__ void load_segs128(const Segs128& s, const int* efo, const int* counts, int E, int rows, int tile_rows,
                                             bool live_only, int lane) {
  for (int e = lane; e <= E; e += 32) s.start[e] = efo ? min(max(efo[e], 0), rows) : (e == 0 ? 0 : rows);
  if (lane == 0) s.start[E + 1] = rows;
  __syncwarp();
  int run = 0;
  for (int e0 = 0; e0 <= E; e0 += 32) {
    const int e = e0 + lane;
    int n = 0;
    if (e <= E) {
      const int a = s.start[e], end = s.start[e + 1];
      int live = e == E ? a : end;
      if (e < E && counts) live = min(end, a + min(max(counts[e], 0), rows));
      s.live[e] = max(live, a);
      n = max((live_only ? s.live[e] : end) - a, 0);
      n = (n + tile_rows - 1) / tile_rows;
    }
    int inc = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += y;
    }
    if (e <= E) s.tiles[e] = run + inc - n;
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) s.tiles[E + 1] = run;
}
__device__ __forceinline__ int seg_of_tile(const int* tiles, int segs, int t) {      // largest e with tiles[e] <= t, not empty
  int lo = 0, hi = segs;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (tiles[mid + 1] <= t) lo = mid + 1; else hi = mid;
  }
  return lo;
}

struct Tile128 {
  int e, m0, n0;             // m0: first row of this CTA's 128
  int t0, nkt;               // WGRAD128: first row of the reduction; blocks of 128
  int live, end;             // rows below live are computed, those up to end zero (WGRAD128: end = M)
};
template <int MODE>
__device__ __forceinline__ Tile128 tile128(int tile, int rank, const Gemm128Params& p, const Segs128& s) {
  Tile128 t;
  const int nt = (p.N + 255) / 256;
  if (MODE == WGRAD128) {
    const int mt = (p.M + 255) / 256, per = mt * nt;
    t.e = tile / per;
    const int r = tile - t.e * per;
    t.m0 = (r / nt) * 256 + rank * 128;
    t.n0 = (r % nt) * 256;
    t.t0 = s.start[t.e];
    t.nkt = (s.live[t.e] - t.t0 + 127) / 128;
    t.live = t.end = p.M;
  } else {
    const int pr = tile / nt;
    t.n0 = (tile - pr * nt) * 256;
    t.e = seg_of_tile(s.tiles, p.E + 1, pr);
    const int first = s.start[t.e] + (pr - s.tiles[t.e]) * 256;
    t.m0 = first + rank * 128;
    t.t0 = 0;
    t.live = s.live[t.e];
    t.end = p.zero_rest ? s.start[t.e + 1] : t.live;
    t.nkt = first < t.live ? (p.K + 127) / 128 : 0;
  }
  return t;
}

// 32 columns (bf16) or 16 (f32) of a warp's 32 rows through its staging tile: lanes hold rows, the stores take 64 bytes of a row
// each.  w: the lane's 16 words.  word0: column of the first word in 32-bit words from the row's start; words of a row.
template <typename F>
__device__ __forceinline__ void store_slab128(uint32_t stg, int lane, const uint32_t (&w)[16], F store) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    st_shared_v4(stg + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4), w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2), j = lane & 3;
    uint4 v;
    ld_shared_v4(stg + r * 64 + ((j ^ ((r >> 1) & 3)) << 4), v.x, v.y, v.z, v.w);
    store(r, j, v);
  }
  __syncwarp();
}

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Gemm128Smem::THREADS, 1)
gemm128_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const Gemm128Params p) {
  using S = Gemm128Smem;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi = smem + S::STAGES * S::STAGE_BYTES;
  uint8_t* aux = epi + S::EPI_WARPS * (S::STG_BYTES + S::SB_BYTES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(aux);            // full[S], empty[S], tfull[2], tempty[2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(aux + 496);
  volatile int* s_abort = reinterpret_cast<volatile int*>(aux + 500);
  Segs128 segs;
  segs.start = reinterpret_cast<int*>(aux + 512);
  segs.live = segs.start + kG128Segs + 1;
  segs.tiles = segs.live + kG128Segs + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair_id = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * S::STAGES;
  const uint32_t bar_tfull = bar_empty + 8 * S::STAGES, bar_tempty = bar_tfull + 16;

  constexpr int PRODUCER = S::EPI_WARPS, ISSUER = S::EPI_WARPS + 1;
  if (warp == 2) load_segs128(segs, p.efo, p.counts, p.E, p.rows, 256, false, lane);
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);                     // leader's: its producer arms it, both CTAs' copies credit it
      mbar_init(bar_empty + 8 * s, 1);                    // one commit arrival per use, in each CTA
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar_tfull + 8 * s, 1);                    // commit arrival, in each CTA
      mbar_init(bar_tempty + 8 * s, 2 * S::EPI_WARPS);    // leader's: the epilogue warps of both CTAs
    }
    *s_abort = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == ISSUER) {
    tmem_alloc2(smem_u32(tmem_slot), 512);
    tmem_relinquish2();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t smem_base = smem_u32(smem);
  const int nt = (p.N + 255) / 256;
  const int n_total = MODE == WGRAD128 ? p.E * ((p.M + 255) / 256) * nt : segs.tiles[p.E + 1] * nt;

  if (warp >= S::EPI_WARPS) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::OTHER_REGS));
  if (warp == PRODUCER) {
    // ------------------------------------------------------------ producer (both CTAs), one elected lane issues
    if (lane == 0) { prefetch_tmap(&tmap_a); prefetch_tmap(&tmap_b); }
    const uint32_t full0 = map_to_cta(bar_full, 0);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = pair_id; tile < n_total && ok; tile += n_pairs) {
      const Tile128 t = tile128<MODE>(tile, rank, p, segs);
      const int nkt = __shfl_sync(0xffffffffu, t.nkt, 0), m0 = __shfl_sync(0xffffffffu, t.m0, 0);
      const int n_row = __shfl_sync(0xffffffffu, t.n0, 0) + (int)rank * 128;
      const int e = MODE == WGRAD128 ? 0 : __shfl_sync(0xffffffffu, t.e, 0), t0 = __shfl_sync(0xffffffffu, t.t0, 0);
      for (int k = 0; k < nkt; ++k) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * stage, phase ^ 1));
        if (!ok) break;
        const uint32_t full = full0 + 8 * stage;
        const uint32_t a_dst = smem_base + stage * S::STAGE_BYTES, b_dst = a_dst + S::A_BYTES;
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(bar_full + 8 * stage, S::TX_BYTES);
          if (MODE == WGRAD128) {
            tma_load_2d_pair(a_dst, &tmap_a, full, m0, t0 + k * 128);
            tma_load_3d_pair(b_dst, &tmap_b, full, n_row, t0 + k * 128, 0);
          } else {
            tma_load_2d_pair(a_dst, &tmap_a, full, k * 128, m0);
            if (p.b_mn) tma_load_3d_pair(b_dst, &tmap_b, full, n_row, k * 128, e);
            else tma_load_3d_pair(b_dst, &tmap_b, full, k * 128, n_row, e);
          }
        }
        if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
      }
    }
    if (!ok && lane == 0) { *s_abort = 1; fail128(p.status, p.host_word, 401); }
  } else if (warp == ISSUER) {
    // ------------------------------------------------------------ MMA issuer (leader CTA only)
    if (rank == 0) {
      const bool a_mn = MODE == WGRAD128, b_mn = MODE == WGRAD128 || p.b_mn;
      const uint32_t idesc = make_idesc_f8(256, 256, a_mn, b_mn);
      // operand descriptors: see make_desc_kmajor_sw128 / make_desc_mnmajor_sw128; a step of 32 along the reduction is 32 bytes
      // (K-major) or 32 rows of 128 bytes
      const uint32_t desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);
      const uint32_t a_step = a_mn ? 256u : 2u, b_step = b_mn ? 256u : 2u;
      const uint32_t a_lo0 = ((smem_base & 0x3FFFF) >> 4) | ((a_mn ? (uint32_t)(S::A_BYTES >> 4) : 1u) << 16);
      const uint32_t b_lo0 = (((smem_base + S::A_BYTES) & 0x3FFFF) >> 4) | ((b_mn ? (uint32_t)(S::B_BYTES >> 4) : 1u) << 16);
      int stage = 0, as = 0;
      uint32_t phase = 0, aphase = 0;
      bool ok = true;
      for (int tile = pair_id; tile < n_total && ok; tile += n_pairs) {
        const int nkt = __shfl_sync(0xffffffffu, tile128<MODE>(tile, 0, p, segs).nkt, 0);
        for (int k = 0; k < nkt; ++k) {
          ok = __all_sync(0xffffffffu, mbar_wait(bar_tempty + 8 * as, aphase ^ 1));
          if (!ok) break;
          ok = __all_sync(0xffffffffu, mbar_wait(bar_full + 8 * stage, phase));
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_lo = a_lo0 + stage * (S::STAGE_BYTES >> 4), b_lo = b_lo0 + stage * (S::STAGE_BYTES >> 4);
          if (elect_one()) {
#pragma unroll
            for (int kb = 0; kb < BK / 32; ++kb)
              mma_f8_pair_lo(tmem_base + as * 256, a_lo + a_step * kb, b_lo + b_step * kb, desc_hi, idesc, kb != 0);
            tc_commit_pair(bar_empty + 8 * stage, 3);
            tc_commit_pair(bar_tfull + 8 * as, 3);
          }
          if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
          if (++as == 2) { as = 0; aphase ^= 1; }
        }
      }
      if (!ok && lane == 0) { *s_abort = 1; fail128(p.status, p.host_word, 402); }
    }
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::EPI_REGS));
    // ------------------------------------------------------------ epilogue: a warp owns 32 rows (its TMEM lanes) x 128 columns
    const int q = warp & 3, half = warp >> 2;
    const uint32_t tempty0 = map_to_cta(bar_tempty, 0);
    const uint32_t stg = smem_u32(epi) + warp * S::STG_BYTES;
    float* sb_buf = reinterpret_cast<float*>(epi + S::EPI_WARPS * S::STG_BYTES + warp * S::SB_BYTES);
    int as = 0;
    uint32_t aphase = 0;
    bool ok = true;
    for (int tile = pair_id; tile < n_total && ok; tile += n_pairs) {
      const Tile128 t = tile128<MODE>(tile, rank, p, segs);
      const int row = t.m0 + q * 32 + lane;               // of c (WGRAD128: of the expert's)
      const int col0 = t.n0 + half * 128;
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.f;
      // scales: one number a lane for its row, one for the 128 columns (ROWS128) or one a column (WGRAD128)
      const float* sa = p.a_s;
      const float* sb = p.b_s;
      int sa_k, sb_k;
      bool sb_in = true, row_in;
      if (MODE == WGRAD128) {
        row_in = row < p.M;
        sa += (int64_t)(t.t0 / 128) * p.M + (row_in ? row : 0);
        sb_in = col0 + lane * 4 < p.N;
        sb += (int64_t)(t.t0 / 128) * p.N + (sb_in ? col0 + lane * 4 : 0);
        sa_k = p.M;
        sb_k = p.N;
      } else {
        row_in = row < t.live;
        sa += (int64_t)(row_in ? row : 0) * p.a_kb;
        sb += t.e < p.E ? t.e * p.bs_e + (int64_t)min(col0 / 128, (p.N - 1) / 128) * p.bs_n : 0;
        sa_k = 1;
        sb_k = p.bs_k;
      }
      float sa_next = 0.f, sb_next = 0.f;
      float4 sb4_next = make_float4(0.f, 0.f, 0.f, 0.f);
      if (t.nkt > 0) {
        sa_next = *sa;
        if (MODE == WGRAD128) { if (sb_in) sb4_next = *reinterpret_cast<const float4*>(sb); }
        else sb_next = *sb;
      }
      for (int k = 0; k < t.nkt; ++k) {
        const float sa_now = sa_next, sb_now = sb_next;
        float* sbk = sb_buf + (k & 1) * 128;
        if (MODE == WGRAD128) {
          reinterpret_cast<float4*>(sbk)[lane] = sb4_next;
          __syncwarp();
        }
        if (k + 1 < t.nkt) {
          sa += sa_k;
          sb += sb_k;
          sa_next = *sa;
          if (MODE == WGRAD128) { if (sb_in) sb4_next = *reinterpret_cast<const float4*>(sb); }
          else sb_next = *sb;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * as, aphase));
        if (!ok) break;
        tc_fence_after();
        const uint32_t src = tmem_base + ((uint32_t)(q * 32) << 16) + as * 256 + half * 128;
        const float f = MODE == WGRAD128 ? sa_now : sa_now * sb_now;
        uint32_t r[2][16];
        tmem_ld16(src, r[0]);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          tmem_ld_wait();
          tmem_arrived(r[c & 1]);
          if (c < 7) {
            tmem_ld16(src + (c + 1) * 16, r[(c + 1) & 1]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(tempty0 + 8 * as);
          }
          const uint32_t(&v)[16] = r[c & 1];
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            if (MODE == WGRAD128) {
              const float4 s4 = *reinterpret_cast<const float4*>(sbk + c * 16 + i);
              const float x[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
              for (int j = 0; j < 4; ++j)
                acc[c * 16 + i + j] = fmaf(__uint_as_float(v[i + j]) * x[j], f, acc[c * 16 + i + j]);
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[c * 16 + i + j] = fmaf(__uint_as_float(v[i + j]), f, acc[c * 16 + i + j]);
            }
          }
        }
        if (++as == 2) { as = 0; aphase ^= 1; }
      }
      if (!ok) break;
      if (MODE == ROWS128 && t.m0 + q * 32 >= t.end) continue;      // nothing of this warp's rows is stored
      // ---- out
      if (MODE == ROWS128 || p.out_bf16) {
        uint16_t* c = reinterpret_cast<uint16_t*>(p.c) + (MODE == WGRAD128 ? (int64_t)t.e * p.M * p.N : 0);
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            w[i] = row_in ? pack_bf16x2(acc[cc * 32 + 2 * i], acc[cc * 32 + 2 * i + 1]) : 0u;
          }
          store_slab128(stg, lane, w, [&](int r, int j, const uint4& v) {
            const int gr = t.m0 + q * 32 + r, gc = col0 + cc * 32 + j * 8;
            if (gr < t.end && gc < p.N) *reinterpret_cast<uint4*>(c + (int64_t)gr * p.N + gc) = v;
          });
        }
      } else {
        float* c = reinterpret_cast<float*>(p.c) + (int64_t)t.e * p.M * p.N;
#pragma unroll
        for (int cc = 0; cc < 8; ++cc) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(acc[cc * 16 + i]);
          store_slab128(stg, lane, w, [&](int r, int j, const uint4& v) {
            const int gr = t.m0 + q * 32 + r, gc = col0 + cc * 16 + j * 4;
            if (gr < t.end && gc < p.N) {
              float4* dst = reinterpret_cast<float4*>(c + (int64_t)gr * p.N + gc);
              float4 o = make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
              if (p.accumulate) {
                const float4 b = *dst;
                o.x += b.x; o.y += b.y; o.z += b.z; o.w += b.w;
              }
              *dst = o;
            }
          });
        }
      }
    }
    if (!ok && lane == 0) { *s_abort = 1; fail128(p.status, p.host_word, 403); }
  }

  // common exit: everyone arrives here, also after a failed wait
  __syncthreads();
  if (*s_abort) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  tc_fence_before();
  cluster_sync_all();                         // the peer may still be signalling this CTA's barriers
  tc_fence_after();
  if (warp == ISSUER) tmem_dealloc2(tmem_base, 512);
}

}  // namespace smoe
