// Products of bf16 rows grouped by expert, tcgen05 on CTA pairs, 256 x 256 tiles.
//
//   ROWS16    c[r, n] = sum_k a[r, k] b[e][n, k]   (b_mn: b[e][k, n])     rows of expert e's segment
//   WGRAD16   c[e][m, n] (+)= sum over the rows r of e's segment of a[r, m] b[r, n]
//
// Segments begin and end at any row.  A tile of rows that reaches into the next segment computes rows that it does not store; a
// reduction over rows must not take any in: the last block of 64 gets as many MMAs of 16 rows as it needs, and the operands' rows behind
// the segment's last one, at most 15, are overwritten with zeros in shared memory by a warp of its own before they are read (us, all of
// the block / so, weight gradients of 128 experts of 1536 x 2048: 4 rows each 191 / 143, 65 244 / 192, 96 217 / 177; zeros alone 139).
//
// Operands by TMA in the 128-byte swizzle, 64 values of the reduction a stage: [128 rows][64] where the reduction lies along memory
// (K-major), two pieces of [64 of the reduction][64] where it lies across (MN-major), as weights do for the gradient of the rows and
// both operands for that of the weights; nothing is transposed in memory.  f32 sums stay in TMEM over the whole reduction, two
// buffers of 256 columns, so that a tile's results leave under the next one's MMAs.
#pragma once
#include "gemm128.cuh"

namespace smoe {

enum Gemm16Mode : int { ROWS16 = 0, WGRAD16 = 1 };

constexpr int kBK16 = 64;          // values of the reduction a stage: 128 bytes

struct Gemm16Params {
  int rows;                  // rows that are cut into segments
  int M, N, K, E;            // M: rows of an expert's c (WGRAD16); N: columns of c; K: reduction length (ROWS16)
  const int *efo, *counts;   // [E+1] segments and [E] live rows; null: one segment of all rows, all rows of a segment live
  int b_mn;
  void* c;                   // ROWS16: bf16 [rows, N], rows that are not live become zero; WGRAD16: [E, M, N] f32 or bf16
  int out_bf16, accumulate;  // WGRAD16
  int split;                 // WGRAD16: stretches that a segment's rows are cut into; stretch s goes to the s-th [E, M, N] of c
  int* status;
  volatile int* host_word;
};

constexpr int kPiece16 = 64 * 128;      // bytes of 64 x 64 values

// BN: columns of a tile, 256, or 128 where tiles are few or narrow
template <int COLS>
struct Gemm16Smem {
  static constexpr int BN = COLS;
  static constexpr int A_BYTES = BM * 128, B_BYTES = BN / 2 * 128, B_PIECES = BN / 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES, STAGES = BN == 256 ? 5 : 7;
  static constexpr int BUFS = 2;
  static constexpr int EPI_WARPS = 8, STG_BYTES = 4096;       // staging of a warp: 32 rows of 128 bytes
  static constexpr int BAR_BYTES = (4 * STAGES + 2 * BUFS) * 8;
  static constexpr int AUX_BYTES = 512 + 3 * (kG128Segs + 1) * 4;
  static constexpr int TOTAL = 1024 + STAGES * STAGE_BYTES + EPI_WARPS * STG_BYTES + AUX_BYTES;
  static constexpr int THREADS = 32 * (EPI_WARPS + 4);
  static_assert(TOTAL <= 227 * 1024, "shared memory budget");
  static_assert(BAR_BYTES <= 496, "barrier storage");
};

// tcgen05.mma kind::f16: bf16 x bf16 -> f32
__host__ __device__ constexpr uint32_t make_idesc_bf16(int M, int N, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_bf16_pair_lo(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc,
                                                 uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %3};\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %4, p;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// high word of every operand descriptor here: 8-row groups 1024 bytes apart, 128-byte swizzle (see make_desc_kmajor_sw128)
constexpr uint32_t kDescHi16 = (1024u >> 4) | (1u << 14) | (2u << 29);
// low word: start, and for an MN-major operand the distance between its pieces of 64
__device__ __forceinline__ uint32_t desc_lo16(uint32_t saddr, bool mn) {
  return ((saddr & 0x3FFFF) >> 4) | (mn ? (uint32_t)(kPiece16 >> 4) << 16 : 1u << 16);
}
// of an MMA's 16 values of the reduction: 32 bytes, or 16 rows of 128
__device__ __forceinline__ uint32_t desc_step16(bool mn) { return mn ? 128u : 2u; }

// the values of a TMEM load are there from here on: nothing that reads them moves ahead of the wait
template <int N>
__device__ __forceinline__ void tmem_values(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

// The L2 fetches what a sum is added to when the sum arrives, and the sums wait for that: the old values of a warp's next pieces are
// asked for kReduceAhead ahead, in tiles of few blocks, which this traffic bounds (us with / without, by rows an expert: 32 of 1536 x
// 2048, 128 rows 149 / 168; 8 of 2048 x 2048, 512 54 / 66; 128 of 1536 x 2048, 256 631 / 648, 1024 846 / 827).
constexpr int kAheadBlocks16 = 10;
__device__ __forceinline__ void tma_prefetch_l2_3d(const void* tmap, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(tmap), "r"(c0), "r"(c1), "r"(c2) : "memory");
}

struct Tile16 {
  int e, m0, n0;             // m0: first row of this CTA's 128
  int t0, nkt, tail;         // WGRAD16: first row of the reduction; blocks of 64; rows of the last one if it is not full
  int live;                  // rows below it are stored
  int out;                   // WGRAD16: which of c's [M, N]
};
template <int MODE, int BN>
__device__ __forceinline__ Tile16 tile16(int tile, int rank, const Gemm16Params& p, const Segs128& s) {
  Tile16 t;
  const int nt = (p.N + BN - 1) / BN;
  if (MODE == WGRAD16) {
    const int mt = (p.M + 255) / 256, per = mt * nt;
    t.out = tile / per;
    const int r = tile - t.out * per, part = t.out / p.E;
    t.e = t.out - part * p.E;
    t.m0 = (r / nt) * 256 + rank * 128;
    t.n0 = (r % nt) * BN;
    const int all = s.live[t.e] - s.start[t.e];
    const int stretch = ((all + p.split - 1) / p.split + kBK16 - 1) / kBK16 * kBK16;
    const int n = max(min(all - part * stretch, stretch), 0);
    t.t0 = s.start[t.e] + part * stretch;
    t.nkt = (n + kBK16 - 1) / kBK16;
    t.tail = n % kBK16;
    t.live = p.M;
  } else {
    const int pr = tile / nt;
    t.n0 = (tile - pr * nt) * BN;
    t.e = seg_of_tile_warp(s.tiles, p.E, pr);
    t.m0 = s.start[t.e] + (pr - s.tiles[t.e]) * 256 + rank * 128;
    t.t0 = t.tail = t.out = 0;
    t.nkt = (p.K + kBK16 - 1) / kBK16;
    t.live = s.live[t.e];
  }
  return t;
}

// Rows that belong to no segment, or lie behind a segment's live ones, become zero: warp w of n, N a multiple of 8.  The warps take the rows
// in turn over all gaps (each gap from warp 0 on: 128 experts of 1472 x 288, 10101 rows in 26496, 85 us instead of 49).
__device__ __forceinline__ void zero_gaps16(const Segs128& s, int E, __nv_bfloat16* c, int N, int w, int n, int lane) {
  int mine = w;                                         // rows of gaps until this warp's next one
  for (int e0 = -1; e0 <= E; e0 += 32) {
    const int e = e0 + lane;
    const int a = e < 0 ? 0 : e <= E ? s.live[e] : 0, end = e < 0 ? s.start[0] : e <= E ? s.start[e + 1] : 0;
    uint32_t some = __ballot_sync(0xffffffffu, a < end);
    while (some) {
      const int l = __ffs((int)some) - 1;
      some &= some - 1;
      const int from = __shfl_sync(0xffffffffu, a, l), to = __shfl_sync(0xffffffffu, end, l);
      int r = from + mine;
      for (; r < to; r += n)
        for (int col = lane * 8; col < N; col += 256) *reinterpret_cast<uint4*>(c + (int64_t)r * N + col) = make_uint4(0, 0, 0, 0);
      mine = r - to;
    }
  }
}

template <int MODE, int COLS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Gemm16Smem<COLS>::THREADS, 1)
gemm16_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
              const __grid_constant__ CUtensorMap tmap_c, const Gemm16Params p) {
  using S = Gemm16Smem<COLS>;
  constexpr int BN = S::BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi = smem + S::STAGES * S::STAGE_BYTES;
  uint8_t* aux = epi + S::EPI_WARPS * S::STG_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(aux);            // full[S], empty[S], tail[S], fixed[S], tfull[BUFS], tempty[BUFS]
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
  const uint32_t bar_tail = bar_empty + 8 * S::STAGES, bar_fixed = bar_tail + 8 * S::STAGES;
  const uint32_t bar_tfull = bar_fixed + 8 * S::STAGES, bar_tempty = bar_tfull + 8 * S::BUFS;

  constexpr int PRODUCER = S::EPI_WARPS, ISSUER = S::EPI_WARPS + 1, FIXER = S::EPI_WARPS + 2;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);                     // leader's: its producer arms it, both CTAs' copies credit it
      mbar_init(bar_empty + 8 * s, 1);                    // one commit arrival per use, in each CTA
      mbar_init(bar_tail + 8 * s, 1);                     // of this CTA alone: the copies of a block with rows to be overwritten
      mbar_init(bar_fixed + 8 * s, 2);                    // leader's: such a block is ready in both CTAs
    }
    for (int s = 0; s < S::BUFS; ++s) {
      mbar_init(bar_tfull + 8 * s, 1);                    // commit arrival, in each CTA
      mbar_init(bar_tempty + 8 * s, 2 * S::EPI_WARPS);    // leader's: the epilogue warps of both CTAs
    }
    *s_abort = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == ISSUER) {
    tmem_alloc2(smem_u32(tmem_slot), S::BUFS * BN);
    tmem_relinquish2();
  }
  wait_for_kernel_before();                   // so far nothing in memory has been touched
  next_kernel_may_start();
  if (warp == 2) load_segs128<false>(segs, p.efo, p.counts, p.E, p.rows, 256, true, 0, 0, lane);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t smem_base = smem_u32(smem);
  const int nt = (p.N + BN - 1) / BN;
  const int n_total = MODE == WGRAD16 ? p.split * p.E * ((p.M + 255) / 256) * nt : segs.tiles[p.E + 1] * nt;

  if (warp == PRODUCER) {
    // ------------------------------------------------------------ producer (both CTAs), one elected lane issues
    if (lane == 0) { prefetch_tmap(&tmap_a); prefetch_tmap(&tmap_b); prefetch_tmap(&tmap_c); }
    const uint32_t full0 = map_to_cta(bar_full, 0);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = pair_id; tile < n_total && ok; tile += n_pairs) {
      const Tile16 t = tile16<MODE, BN>(tile, rank, p, segs);
      const int nkt = __shfl_sync(0xffffffffu, t.nkt, 0), m0 = __shfl_sync(0xffffffffu, t.m0, 0);
      const int n_row = __shfl_sync(0xffffffffu, t.n0, 0) + (int)rank * (BN / 2);
      const int e = __shfl_sync(0xffffffffu, t.e, 0), t0 = __shfl_sync(0xffffffffu, t.t0, 0);
      const int tail = __shfl_sync(0xffffffffu, t.tail, 0);
      for (int k = 0; k < nkt; ++k) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * stage, phase ^ 1));
        if (!ok) break;
        const uint32_t full = full0 + 8 * stage;
        const uint32_t a_dst = smem_base + stage * S::STAGE_BYTES, b_dst = a_dst + S::A_BYTES;
        if (elect_one()) {
          if (MODE == WGRAD16 && (tail & 15) && k == nkt - 1) {      // to a barrier of this CTA, for its FIXER
            const uint32_t last = bar_tail + 8 * stage;
            mbar_expect_tx(last, S::STAGE_BYTES);
#pragma unroll
            for (int c = 0; c < 2; ++c) tma_load_2d(a_dst + c * kPiece16, &tmap_a, last, m0 + c * 64, t0 + k * kBK16);
#pragma unroll
            for (int c = 0; c < S::B_PIECES; ++c) tma_load_2d(b_dst + c * kPiece16, &tmap_b, last, n_row + c * 64, t0 + k * kBK16);
          } else {
            if (rank == 0) mbar_expect_tx(bar_full + 8 * stage, 2 * S::STAGE_BYTES);
            if (MODE == WGRAD16) {
#pragma unroll
              for (int c = 0; c < 2; ++c) tma_load_2d_pair(a_dst + c * kPiece16, &tmap_a, full, m0 + c * 64, t0 + k * kBK16);
#pragma unroll
              for (int c = 0; c < S::B_PIECES; ++c)
                tma_load_2d_pair(b_dst + c * kPiece16, &tmap_b, full, n_row + c * 64, t0 + k * kBK16);
            } else {
              tma_load_2d_pair(a_dst, &tmap_a, full, k * kBK16, m0);
              if (p.b_mn) {
#pragma unroll
                for (int c = 0; c < S::B_PIECES; ++c) tma_load_3d_pair(b_dst + c * kPiece16, &tmap_b, full, n_row + c * 64, k * kBK16, e);
              } else {
                tma_load_3d_pair(b_dst, &tmap_b, full, k * kBK16, n_row, e);
              }
            }
          }
        }
        if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
      }
    }
    if (!ok && lane == 0) { *s_abort = 1; fail128(p.status, p.host_word, 601); }
  } else if (warp == ISSUER) {
    // ------------------------------------------------------------ MMA issuer (leader CTA only)
    if (rank == 0) {
      const bool a_mn = MODE == WGRAD16, b_mn = MODE == WGRAD16 || p.b_mn;
      const uint32_t idesc = make_idesc_bf16(256, BN, a_mn, b_mn);
      const uint32_t a_step = desc_step16(a_mn), b_step = desc_step16(b_mn);
      const uint32_t a_lo0 = desc_lo16(smem_base, a_mn), b_lo0 = desc_lo16(smem_base + S::A_BYTES, b_mn);
      int stage = 0, as = 0;
      uint32_t fulls = 0, fixes = 0, aphase = 0;              // a stage's phase on either barrier it may be announced by: one bit each
      bool ok = true;
      for (int tile = pair_id; tile < n_total && ok; tile += n_pairs) {
        const Tile16 t = tile16<MODE, BN>(tile, 0, p, segs);
        const int nkt = __shfl_sync(0xffffffffu, t.nkt, 0), tail = __shfl_sync(0xffffffffu, t.tail, 0);
        if (nkt == 0) continue;
        ok = __all_sync(0xffffffffu, mbar_wait(bar_tempty + 8 * as, aphase ^ 1));
        if (!ok) break;
        for (int k = 0; k < nkt; ++k) {
          if (MODE == WGRAD16 && (tail & 15) && k == nkt - 1) {
            ok = __all_sync(0xffffffffu, mbar_wait_cluster(bar_fixed + 8 * stage, fixes >> stage & 1));
            fixes ^= 1u << stage;
          } else {
            ok = __all_sync(0xffffffffu, mbar_wait(bar_full + 8 * stage, fulls >> stage & 1));
            fulls ^= 1u << stage;
          }
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_lo = a_lo0 + stage * (S::STAGE_BYTES >> 4), b_lo = b_lo0 + stage * (S::STAGE_BYTES >> 4);
          const int steps = MODE == WGRAD16 && tail && k == nkt - 1 ? (tail + 15) / 16 : kBK16 / 16;
          if (elect_one()) {
#pragma unroll
            for (int kb = 0; kb < kBK16 / 16; ++kb)
              if (kb < steps)
                mma_bf16_pair_lo(tmem_base + as * BN, a_lo + a_step * kb, b_lo + b_step * kb, kDescHi16, idesc, (k | kb) != 0);
            tc_commit_pair(bar_empty + 8 * stage, 3);
            if (k == nkt - 1) tc_commit_pair(bar_tfull + 8 * as, 3);
          }
          if (++stage == S::STAGES) stage = 0;
        }
        if (++as == S::BUFS) { as = 0; aphase ^= 1; }
      }
      if (!ok && lane == 0) { *s_abort = 1; fail128(p.status, p.host_word, 602); }
    }
    __syncwarp();
  } else if (MODE == WGRAD16 && warp == FIXER) {
    // ------------------------------------------------------------ rows behind a segment's last one (both CTAs, each its own)
    const uint32_t fixed0 = map_to_cta(bar_fixed, 0);
    int stage = 0;
    uint32_t tails = 0;
    bool ok = true;
    for (int tile = pair_id; tile < n_total && ok; tile += n_pairs) {
      const Tile16 t = tile16<MODE, BN>(tile, rank, p, segs);
      stage = (stage + t.nkt) % S::STAGES;
      const int end = (t.tail + 15) & ~15;
      if (t.tail == end) continue;
      const int st = stage == 0 ? S::STAGES - 1 : stage - 1;
      ok = __all_sync(0xffffffffu, mbar_wait(bar_tail + 8 * st, tails >> st & 1));
      tails ^= 1u << st;
      if (!ok) break;
      const uint32_t at = smem_base + st * S::STAGE_BYTES;
#pragma unroll
      for (int c = 0; c < 2 + S::B_PIECES; ++c)               // the pieces of both operands, a row 128 bytes of each
        for (int b = t.tail * 128 + lane * 16; b < end * 128; b += 512) st_shared_v4(at + c * kPiece16 + b, 0u, 0u, 0u, 0u);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(fixed0 + 8 * st);
    }
    if (!ok && lane == 0) { *s_abort = 1; fail128(p.status, p.host_word, 604); }
  } else if (warp < S::EPI_WARPS) {
    // ------------------------------------------------------------ epilogue: a warp owns 32 rows (its TMEM lanes) x 128 columns
    const int q = warp & 3, half = warp >> 2;
    const uint32_t tempty0 = map_to_cta(bar_tempty, 0);
    const uint32_t stg = smem_u32(epi) + warp * S::STG_BYTES;
    int as = 0;
    uint32_t aphase = 0;
    bool ok = true;
    if (MODE == ROWS16)
      zero_gaps16(segs, p.E, (__nv_bfloat16*)p.c, p.N, (int)blockIdx.x * S::EPI_WARPS + warp, (int)gridDim.x * S::EPI_WARPS, lane);
    for (int tile = pair_id; tile < n_total; tile += n_pairs) {
      const Tile16 t = tile16<MODE, BN>(tile, rank, p, segs);
      const int row0 = t.m0 + q * 32, col0 = t.n0 + half * (BN / 2);
      if (t.nkt == 0 && p.accumulate) continue;               // an empty sum
      const bool stored = row0 < t.live && col0 < p.N;
      const bool ahead = MODE == WGRAD16 && p.accumulate && stored && t.nkt <= kAheadBlocks16 && lane == 0;
      auto prefetch_piece = [&](int i) {
        if (ahead && i < BN / 64 && col0 + i * 32 < p.N) tma_prefetch_l2_3d(&tmap_c, col0 + i * 32, row0, t.out);
      };
#pragma unroll
      for (int i = 0; i < kReduceAhead; ++i) prefetch_piece(i);
      if (t.nkt) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * as, aphase));
        if (!ok) break;
        tc_fence_after();
      }
      const uint32_t src = tmem_base + ((uint32_t)(q * 32) << 16) + as * BN + half * (BN / 2);
#pragma unroll
      for (int h = 0; h < BN / 128; ++h) {                    // 64 columns
        uint32_t r[2][32];
        if (t.nkt) {
          tmem_ld32(src + h * 64, r[0]);
          tmem_ld32(src + h * 64 + 32, r[1]);
          tmem_ld_wait();
          tmem_values(r[0]);
          tmem_values(r[1]);
          if (h == BN / 128 - 1) {                            // the buffer's values are in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(tempty0 + 8 * as);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[0][i] = r[1][i] = 0u;
        }
        const int col = col0 + h * 64;
        if (!stored || col >= p.N) continue;
        if (MODE == ROWS16 || p.out_bf16) {
          if (lane == 0) bulk_wait_group_read<0>();           // what was staged before has been read
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = pack_bf16x2(__uint_as_float(r[j >> 2][(j & 3) * 8 + 2 * i]), __uint_as_float(r[j >> 2][(j & 3) * 8 + 2 * i + 1]));
            st_shared_v4(stg + lane * 128 + ((j ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
          }
          if (MODE == WGRAD16 || row0 + 32 <= t.live) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(&tmap_c, stg, col, row0, MODE == WGRAD16 ? t.out : 0);      // (the map has three dimensions)
              bulk_commit_group();
            }
          } else {
            __syncwarp();
            store_slab128(stg, lane, reinterpret_cast<uint16_t*>(p.c), p.N, row0, t.live, col);
            __syncwarp();
          }
        } else {
#pragma unroll
          for (int u = 0; u < 2; ++u) {                       // 32 columns
            if (col + u * 32 >= p.N) break;
            prefetch_piece(2 * h + u + kReduceAhead);
            if (lane == 0) bulk_wait_group_read<0>();
            __syncwarp();
            stage_f32_32(stg, lane, r[u]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (p.accumulate) tma_reduce_add_3d(&tmap_c, stg, col + u * 32, row0, t.out);
              else tma_store_3d(&tmap_c, stg, col + u * 32, row0, t.out);
              bulk_commit_group();
            }
          }
        }
      }
      if (t.nkt && ++as == S::BUFS) { as = 0; aphase ^= 1; }
    }
    if (lane == 0) bulk_wait_group<0>();                      // all stores have left shared memory and are visible
    if (!ok && lane == 0) { *s_abort = 1; fail128(p.status, p.host_word, 603); }
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
  if (warp == ISSUER) tmem_dealloc2(tmem_base, S::BUFS * BN);
}

}  // namespace smoe
