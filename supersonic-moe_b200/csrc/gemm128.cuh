// Grouped products of e4m3 operands with one f32 scale per block of 128 (see quant128.cu), tcgen05 on CTA pairs.
//
//   ROWS128   c[r, n] = sum_kb as[r, kb] bs[e, n / 128, kb] (sum over the 128 k of kb of a[r, k] b[e][n, k])     rows by expert
//   WGRAD128  c[e][m, n] (+)= sum_tb as[tb, m] bs[tb, n] (sum over the 128 rows t of tb of a[m, t] b[n, t])      rows summed over
//
// f32 scales are not what the block-scaled MMA takes (powers of two, 32 wide), so the plain e4m3 MMA sums one block of 128 at a
// time into TMEM and the epilogue warps add it, scaled, to sums that stay in their registers: 128 f32 a thread, 256 x 256 outputs
// a CTA pair.  Two TMEM buffers of 256 columns: the MMAs of one block run while the block before is read out and added up.
//   What bounds it: by rows, shared memory, out of which the MMAs of a block (512 clocks of arithmetic) read their operands in some
//   640; a block takes 750, and a tile some 3400 clocks beside its blocks.  8192 x 4096 x 4096 123 us (2.2 PFLOP/s), 16384 x 4096 x
//   2048 over 8 experts 133, its dx 128.  The weight gradient: the epilogue's latencies, where a value has two scales of its own in
//   every block: two warps a scheduler, 0.7 of them eligible, no pipe more than half busy (issue 47 %, FMA 47, TMEM 47, MMA 34); the
//   same size 191 us (1.4 PFLOP/s), added to f32 221.
//   B [E, N, K] is read K-major, or with b_mn as [E, K, N] as it lies: the gradient of the rows needs no transposed weights.
//   Both operands of the weight gradient lie [dim, rows].
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
  int independent;           // of the kernel before in the stream: waited for at the end only
  int zero_rest;             // ROWS128: rows that are not live are written as zero (else left as they are; if it is below zero, the
                             // last tile of a segment is left out where it has no more live rows than - zero_rest)
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

constexpr int kG128N = 256;        // columns of a tile (128 with four buffers, weight gradient: 204 -> 259 us, more to do per block)

struct Gemm128Smem {
  static constexpr int BN = kG128N;
  static constexpr int A_BYTES = BM * BK, B_BYTES = BN / 2 * BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES, STAGES = 4;
  static constexpr int BUFS = 512 / BN;                     // TMEM buffers
  static constexpr int EPI_WARPS = 8;
  // Output staging of a warp: two tiles of 32 rows x 128 bytes, all of its bf16 columns, so that they pass through shared memory
  // with one fence.  (Four passes of 64 bytes and a fifth ring stage: 3200 clocks between the last block of a tile and the next
  // one's first, of which the MMAs have 1300 to do; 8192 x 4096 x 128 17.4 -> 15.4 us, x 8192 196 -> 200.)
  static constexpr int STG_TILE = 4096, STG_BYTES = 2 * STG_TILE;
  // WGRAD128: scales of this CTA's 128 rows and of the 256 columns in a block, in a ring of their own, filled by a warp of its own:
  // every block reads new lines of them, and a register's worth of look-ahead does not cover HBM (measured: 1650 clocks a block)
  static constexpr int SC_BYTES = (128 + BN) * 4, SC_SLOTS = 8;
  static constexpr int AUX_BYTES = 512 + 4 * (kG128Segs + 1) * 4;
  static constexpr int TOTAL = 1024 + STAGES * STAGE_BYTES + EPI_WARPS * STG_BYTES + SC_SLOTS * SC_BYTES + AUX_BYTES;
  // Two warpgroups of epilogue warps and one with the producer and the MMA issuer.  A thread of the former needs more than the 168
  // registers that three warps on each quarter of the SM leave: 2 x 224 + 56 = 3 x 168.
  static constexpr int THREADS = 32 * (EPI_WARPS + 4), EPI_REGS = 224, OTHER_REGS = 56;
  static constexpr uint32_t TX_BYTES = 2u * STAGE_BYTES;
  static_assert(TOTAL <= 227 * 1024, "shared memory budget");
  static_assert((2 * STAGES + 2 * BUFS + 2 * SC_SLOTS) * 8 <= 496, "barrier storage");
};

// tcgen05.mma kind::f8f6f4: e4m3 x e4m3 -> f32
__host__ __device__ constexpr uint32_t make_idesc_f8(int M, int N, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
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
// 16 lanes x 32 columns: thread t gets, of each 8 columns g, columns 2 (t % 4) and the next of lanes t / 4 (r[4g], r[4g+1]) and
// t / 4 + 8 (r[4g+2], r[4g+3]).
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ F2 f2_bits(uint32_t lo, uint32_t hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "r"(lo), "r"(hi));
  return r;
}

// Segments from efo / counts, any values taken as they fit: 0 <= start <= end <= rows, start <= live end <= end
struct Segs128 {
  int *start, *live, *tiles;       // [segs + 1] starts; [segs] ends of the live rows; [segs + 1] row tiles before
};
// one warp; segment `E` holds the rows behind the last one, none of them live
//   skip      what is left of a segment after its full tiles makes a tile only if it is more than `skip` rows
//   rest_of   (RESTS) if not 0, tiles are the rests alone, of segments cut into pieces of `rest_of` rows, that fit one tile
template <bool RESTS>
__device__ __forceinline__ void load_segs128(const Segs128& s, const int* efo, const int* counts, int E, int rows, int tile_rows,
                                             bool live_only, int skip, int rest_of, int lane) {
  for (int e = lane; e <= E; e += 32) s.start[e] = efo ? min(max(efo[e], 0), rows) : (e == 0 ? 0 : rows);
  if (lane == 0) s.start[E + 1] = rows;
  __syncwarp();
  int run = 0;
  for (int e0 = 0; e0 <= E; e0 += 32) {
    const int e = e0 + lane;
    int n = 0, rest0 = 0;
    if (e <= E) {
      const int a = s.start[e], end = s.start[e + 1];
      int live = e == E ? a : end;
      if (e < E && counts) live = min(end, a + min(max(counts[e], 0), rows));
      s.live[e] = max(live, a);
      n = max((live_only ? s.live[e] : end) - a, 0);
      if (RESTS && rest_of) {
        const int rest = n % rest_of;
        rest0 = a + n - rest;
        n = rest > 0 && rest <= tile_rows;
      } else {
        n = (n + tile_rows - 1 - skip) / tile_rows;
      }
    }
    if (RESTS) {
      __syncwarp();                                       // the starts have been read
      if (rest_of && e <= E) s.start[e] = rest0;
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

// the same by a whole warp: independent reads, where a search would wait for one after the other (each some 200 clocks beside the MMAs)
__device__ __forceinline__ int seg_of_tile_warp(const int* tiles, int segs, int t) {
  const int lane = threadIdx.x & 31;
  int n = 0;
  for (int e0 = 0; e0 < segs; e0 += 128) {
    int first[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) first[j] = tiles[min(e0 + 32 * j + lane, segs) + 1];
#pragma unroll
    for (int j = 0; j < 4; ++j) n += __popc(__ballot_sync(0xffffffffu, e0 + 32 * j + lane < segs && first[j] <= t));
  }
  return n;
}

struct Tile128 {
  int e, m0, n0;             // m0: first row of this CTA's 128
  int t0, nkt;               // WGRAD128: first row of the reduction (ROWS128: 0); blocks of 128
  int live, end;             // rows below live are computed, those up to end zero (WGRAD128: end = M)
};
template <int MODE>
__device__ __forceinline__ Tile128 tile128(int tile, int rank, const Gemm128Params& p, const Segs128& s) {
  Tile128 t;
  constexpr int BN = kG128N;
  const int nt = (p.N + BN - 1) / BN;
  if (MODE == WGRAD128) {
    const int mt = (p.M + 255) / 256, per = mt * nt;
    t.e = tile / per;
    const int r = tile - t.e * per;
    t.m0 = (r / nt) * 256 + rank * 128;
    t.n0 = (r % nt) * BN;
    t.t0 = s.start[t.e] & ~127;          // segments start there; a copy has to start on 16 bytes in any case
    t.nkt = (s.live[t.e] - s.start[t.e] + 127) / 128;
    t.live = t.end = p.M;
  } else {
    const int pr = tile / nt;
    t.n0 = (tile - pr * nt) * BN;
    t.e = seg_of_tile_warp(s.tiles, p.E, pr);               // (E: the rows behind the last)
    const int first = s.start[t.e] + (pr - s.tiles[t.e]) * 256;
    t.m0 = first + rank * 128;
    t.t0 = 0;
    t.live = s.live[t.e];
    t.end = p.zero_rest > 0 ? s.start[t.e + 1] : t.live;
    t.nkt = first < t.live ? (p.K + 127) / 128 : 0;
  }
  return t;
}

// A warp's staged 32 rows x 64 bf16 columns (16-byte pieces of a row at places xor row % 8, the 128-byte TMA swizzle), where not all
// rows are to be written: eight lanes a row
__device__ __forceinline__ void store_slab128(uint32_t stg, int lane, uint16_t* c, int N, int row0, int end, int col0) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = i * 4 + (lane >> 3), j = lane & 7, gr = row0 + r, gc = col0 + j * 8;
    uint4 v;
    ld_shared_v4(stg + r * 128 + ((j ^ (r & 7)) << 4), v.x, v.y, v.z, v.w);
    if (gr < end && gc < N) *reinterpret_cast<uint4*>(c + (int64_t)gr * N + gc) = v;
  }
}
__device__ __forceinline__ void tma_store_3d(const void* tmap, uint32_t src, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
               ::"l"(tmap), "r"(src), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void tma_reduce_add_3d(const void* tmap, uint32_t src, int c0, int c1, int c2) {
  asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];"
               ::"l"(tmap), "r"(src), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16x2(F2 a) {
  const float2 v = f2_get(a);
  return pack_bf16x2(v.x, v.y);
}
__device__ __forceinline__ void st_shared_b64(uint32_t addr, F2 v) {
  asm volatile("st.shared.b64 [%0], %1;" ::"r"(addr), "l"(v.v) : "memory");
}
__device__ __forceinline__ void st_shared_b32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Gemm128Smem::THREADS, 1)
gemm128_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
               const __grid_constant__ CUtensorMap tmap_c, const Gemm128Params p) {
  using S = Gemm128Smem;
  constexpr int BN = kG128N;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi = smem + S::STAGES * S::STAGE_BYTES;
  uint8_t* scales = epi + S::EPI_WARPS * S::STG_BYTES;
  uint8_t* aux = scales + S::SC_SLOTS * S::SC_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(aux);            // full[S], empty[S], tfull[BUFS], tempty[BUFS], scfull[], scempty[]
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
  const uint32_t bar_tfull = bar_empty + 8 * S::STAGES, bar_tempty = bar_tfull + 8 * S::BUFS;
  const uint32_t bar_scfull = bar_tempty + 8 * S::BUFS, bar_scempty = bar_scfull + 8 * S::SC_SLOTS;

  constexpr int PRODUCER = S::EPI_WARPS, ISSUER = S::EPI_WARPS + 1, SCALER = S::EPI_WARPS + 2;
  if (warp == 2)
    load_segs128<false>(segs, p.efo, p.counts, p.E, p.rows, 256, MODE == ROWS128 && p.zero_rest <= 0,
                        MODE == ROWS128 ? -min(p.zero_rest, 0) : 0, 0, lane);
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);                     // leader's: its producer arms it, both CTAs' copies credit it
      mbar_init(bar_empty + 8 * s, 1);                    // one commit arrival per use, in each CTA
    }
    for (int s = 0; s < S::BUFS; ++s) {
      mbar_init(bar_tfull + 8 * s, 1);                    // commit arrival, in each CTA
      mbar_init(bar_tempty + 8 * s, 2 * S::EPI_WARPS);    // leader's: the epilogue warps of both CTAs
    }
    for (int s = 0; s < S::SC_SLOTS; ++s) {
      mbar_init(bar_scfull + 8 * s, 1);                   // of this CTA alone
      mbar_init(bar_scempty + 8 * s, S::EPI_WARPS);
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
  // (so far offsets and counts alone have been read, which a caller that lets this kernel begin early vouches for)
  if (!p.independent) wait_for_kernel_before();
  next_kernel_may_start();                    // not earlier: an independent one counts on what this kernel has waited for
  const int nt = (p.N + BN - 1) / BN;
  const int n_total = MODE == WGRAD128 ? p.E * ((p.M + 255) / 256) * nt : segs.tiles[p.E + 1] * nt;

  if (warp >= S::EPI_WARPS) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::OTHER_REGS));
  if (warp == PRODUCER) {
    // ------------------------------------------------------------ producer (both CTAs), one elected lane issues
    if (lane == 0) { prefetch_tmap(&tmap_a); prefetch_tmap(&tmap_b); prefetch_tmap(&tmap_c); }
    const uint32_t full0 = map_to_cta(bar_full, 0);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = pair_id; tile < n_total && ok; tile += n_pairs) {
      const Tile128 t = tile128<MODE>(tile, rank, p, segs);
      const int nkt = __shfl_sync(0xffffffffu, t.nkt, 0), m0 = __shfl_sync(0xffffffffu, t.m0, 0);
      const int n_row = __shfl_sync(0xffffffffu, t.n0, 0) + (int)rank * (BN / 2);
      const int e = MODE == WGRAD128 ? 0 : __shfl_sync(0xffffffffu, t.e, 0), t0 = __shfl_sync(0xffffffffu, t.t0, 0);
      for (int k = 0; k < nkt; ++k) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar_empty + 8 * stage, phase ^ 1));
        if (!ok) break;
        const uint32_t full = full0 + 8 * stage;
        const uint32_t a_dst = smem_base + stage * S::STAGE_BYTES, b_dst = a_dst + S::A_BYTES;
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(bar_full + 8 * stage, S::TX_BYTES);
          tma_load_2d_pair(a_dst, &tmap_a, full, t0 + k * 128, m0);
          if (MODE == ROWS128 && p.b_mn) tma_load_3d_pair(b_dst, &tmap_b, full, n_row, k * 128, e);
          else tma_load_3d_pair(b_dst, &tmap_b, full, t0 + k * 128, n_row, e);
        }
        if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
      }
    }
    if (!ok && lane == 0) { *s_abort = 1; fail128(p.status, p.host_word, 401); }
  } else if (warp == ISSUER) {
    // ------------------------------------------------------------ MMA issuer (leader CTA only)
    if (rank == 0) {
      const bool b_mn = MODE == ROWS128 && p.b_mn;
      const uint32_t idesc = make_idesc_f8(256, BN, b_mn);
      // operand descriptors: see make_desc_kmajor_sw128 / make_desc_mnmajor_sw128; a step of 32 along the reduction is 32 bytes
      // (K-major) or 32 rows of 128 bytes
      const uint32_t desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);
      const uint32_t b_step = b_mn ? 256u : 2u;
      const uint32_t a_lo0 = ((smem_base & 0x3FFFF) >> 4) | (1u << 16);
      const uint32_t b_lo0 = (((smem_base + S::A_BYTES) & 0x3FFFF) >> 4) | ((b_mn ? (uint32_t)(S::B_BYTES >> 4) : 1u) << 16);
      int stage = 0, as = 0;
      uint32_t phase = 0, aphase = 0;
      bool ok = true;
      auto blocks_of = [&](int tile) { return tile < n_total ? __shfl_sync(0xffffffffu, tile128<MODE>(tile, 0, p, segs).nkt, 0) : 0; };
      int next_nkt = blocks_of(pair_id);
      for (int tile = pair_id; tile < n_total && ok; tile += n_pairs) {
        const int nkt = next_nkt;
        if (nkt == 0) next_nkt = blocks_of(tile + n_pairs);
        for (int k = 0; k < nkt; ++k) {
          // (the operands first: they are there long before the buffer is, and a look at a barrier takes some 200 clocks while the
          // MMAs read shared memory)
          ok = __all_sync(0xffffffffu, mbar_wait(bar_full + 8 * stage, phase));
          if (!ok) break;
          ok = __all_sync(0xffffffffu, mbar_wait(bar_tempty + 8 * as, aphase ^ 1));
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_lo = a_lo0 + stage * (S::STAGE_BYTES >> 4), b_lo = b_lo0 + stage * (S::STAGE_BYTES >> 4);
          if (elect_one()) {
#pragma unroll
            for (int kb = 0; kb < BK / 32; ++kb)
              mma_f8_pair_lo(tmem_base + as * BN, a_lo + 2 * kb, b_lo + b_step * kb, desc_hi, idesc, kb != 0);
            tc_commit_pair(bar_empty + 8 * stage, 3);
            tc_commit_pair(bar_tfull + 8 * as, 3);
          }
          if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
          if (++as == S::BUFS) { as = 0; aphase ^= 1; }
          if (k == 0) next_nkt = blocks_of(tile + n_pairs);       // (some 700 clocks, under this tile's MMAs)
        }
      }
      if (!ok && lane == 0) { *s_abort = 1; fail128(p.status, p.host_word, 402); }
    }
    __syncwarp();
  } else if (MODE == WGRAD128 && warp == SCALER) {
    // ------------------------------------------------------------ scales (both CTAs, each its own)
    if (lane == 0) {
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair_id; tile < n_total && ok; tile += n_pairs) {
        const Tile128 t = tile128<MODE>(tile, rank, p, segs);
        const uint32_t a_bytes = max(min(128, p.M - t.m0), 0) * 4, b_bytes = min(BN, p.N - t.n0) * 4;      // multiples of 32
        for (int k = 0; k < t.nkt; ++k) {
          ok = mbar_wait(bar_scempty + 8 * slot, phase ^ 1);
          if (!ok) break;
          const uint32_t full = bar_scfull + 8 * slot, dst = smem_u32(scales) + slot * S::SC_BYTES;
          const int64_t block = t.t0 / 128 + k;
          mbar_expect_tx(full, a_bytes + b_bytes);
          if (a_bytes) bulk_load(dst, p.a_s + block * p.M + t.m0, a_bytes, full);
          bulk_load(dst + 512, p.b_s + block * p.N + t.n0, b_bytes, full);
          if (++slot == S::SC_SLOTS) { slot = 0; phase ^= 1; }
        }
      }
      if (!ok) { *s_abort = 1; fail128(p.status, p.host_word, 404); }
    }
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::EPI_REGS));
    // ------------------------------------------------------------ epilogue: a warp owns 32 rows (its TMEM lanes) x 128 columns
    const int q = warp & 3, half = warp >> 2;
    const uint32_t tempty0 = map_to_cta(bar_tempty, 0);
    const uint32_t stg = smem_u32(epi) + warp * S::STG_BYTES;
    int as = 0, slot = 0;
    uint32_t aphase = 0, scphase = 0;
    bool ok = true;
    auto staging_free = [&] {                             // all that was staged before has been read
      if (lane == 0) bulk_wait_group_read<0>();
      __syncwarp();
    };
    // both staging tiles to columns col and col + cols on
    auto staged = [&](int col, int cols, int row, int e) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (col + u * cols >= p.N) break;
          if (MODE == WGRAD128 && p.accumulate) tma_reduce_add_3d(&tmap_c, stg + u * S::STG_TILE, col + u * cols, row, e);
          else tma_store_3d(&tmap_c, stg + u * S::STG_TILE, col + u * cols, row, e);
        }
        bulk_commit_group();
      }
    };
    auto release = [&] {                                  // the buffer's values are in registers
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(tempty0 + 8 * as);
    };
    Tile128 t{}, next{};
    const float *sa = nullptr, *sb = nullptr;             // ROWS128: scales of a lane's row, of the columns
    float sa_next = 0.f, sb_next = 0.f;
    // The next tile and its first scales are asked for while the last block of the one before it is on its way
    auto begin = [&](int tile) {
      next = tile128<MODE>(tile, rank, p, segs);
      if (MODE == ROWS128 && next.nkt > 0) {
        const int row = next.m0 + q * 32 + lane;
        sa = p.a_s + (int64_t)(row < next.live ? row : 0) * p.a_kb;
        sb = p.b_s + next.e * p.bs_e + (int64_t)min((next.n0 + half * (BN / 2)) / 128, (p.N - 1) / 128) * p.bs_n;
        sa_next = *sa;
        sb_next = *sb;
      }
    };
    if (pair_id < n_total) begin(pair_id);
    for (int tile = pair_id; tile < n_total; tile += n_pairs) {
      t = next;
      if (t.nkt == 0 && tile + n_pairs < n_total) begin(tile + n_pairs);
      float acc[MODE == ROWS128 ? BN / 2 : 1];               // [column]
      F2 acc2[MODE == WGRAD128 ? BN / 4 : 1];                 // [32 columns][16 rows][8 columns][row r4, row r4 + 8]: two columns
#pragma unroll
      for (int i = 0; i < (MODE == ROWS128 ? BN / 2 : 0); ++i) acc[i] = 0.f;
#pragma unroll
      for (int i = 0; i < (MODE == WGRAD128 ? BN / 4 : 0); ++i) acc2[i] = f2(0.f, 0.f);
      const int r4 = lane >> 2, c2 = (lane & 3) * 2;
      float fa[4];                                        // WGRAD128: scales of the rows r4 + 8 j; of two columns each
      F2 s2[2][4];
      bool have_scales = false, have_sums = false;
      for (int k = 0; k < t.nkt; ++k) {
        const uint32_t src = tmem_base + ((uint32_t)(q * 32) << 16) + as * BN + half * (BN / 2);
        if (MODE == ROWS128) {
          // A lane is a row, a register a column: one factor a thread and block, the row's scale times the weight's.
          const float f = sa_next * sb_next;
          if (k + 1 < t.nkt) {
            sa_next = *++sa;
            sb += p.bs_k;
            sb_next = *sb;
          } else if (tile + n_pairs < n_total) {
            begin(tile + n_pairs);
          }
          ok = __all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * as, aphase));
          if (!ok) break;
          tc_fence_after();
          // Half the columns, and the other half as each piece's registers come free: the buffer goes back to the MMAs when
          // half of the arithmetic is done (one piece ahead: when seven eighths are, and 783 clocks a block instead of 752).
          uint32_t r[4][16];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld16(src + c * 16, r[c]);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_arrived(r[c]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[c * 16 + i] = fmaf(__uint_as_float(r[c][i]), f, acc[c * 16 + i]);
            tmem_ld16(src + (c + 4) * 16, r[c]);
          }
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_arrived(r[c]);
          release();
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[64 + c * 16 + i] = fmaf(__uint_as_float(r[c][i]), f, acc[64 + c * 16 + i]);
        } else {
          // Both operands have a scale of their own in every block: two multiplications a value.  With a lane a row every lane
          // would read the scales of all 128 columns, 128 KB a block and SM out of shared memory; in the matrix layout a thread
          // has four rows and a quarter of the columns.  Two columns an instruction, which is half the issue (a load shape that
          // reads TMEM in half the time, 16x128b, pairs rows instead and needs more of it: 213 -> 227 us).
          // A look at a barrier or at shared memory takes some 200 clocks beside the MMAs, so that the next block's are asked for
          // under this one's arithmetic: whether its sums and its scales are there, and then its first scales.
          auto first_scales = [&] {
            const float* sak = reinterpret_cast<const float*>(scales + slot * S::SC_BYTES) + q * 32 + r4;
            const float* sbk = reinterpret_cast<const float*>(scales + slot * S::SC_BYTES + 512) + half * (BN / 2) + c2;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              fa[j] = sak[8 * j];
              s2[0][j].v = *reinterpret_cast<const uint64_t*>(sbk + j * 8);
            }
          };
          if (!have_scales) {
            ok = __all_sync(0xffffffffu, mbar_wait(bar_scfull + 8 * slot, scphase));
            if (!ok) break;
            first_scales();
          }
          if (!have_sums) {
            ok = __all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * as, aphase));
            if (!ok) break;
          }
          tc_fence_after();
          if (k + 1 == t.nkt && tile + n_pairs < n_total) begin(tile + n_pairs);
          const float* sbk = reinterpret_cast<const float*>(scales + slot * S::SC_BYTES + 512) + half * (BN / 2) + c2;
          const int next_slot = slot + 1 == S::SC_SLOTS ? 0 : slot + 1, next_as = as + 1 == S::BUFS ? 0 : as + 1;
          const uint32_t next_phase = scphase ^ (next_slot == 0 ? 1u : 0u), next_aphase = aphase ^ (next_as == 0 ? 1u : 0u);
          const bool more = k + 1 < t.nkt;
          bool seen = false, summed = false;
          F2 f[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) f[j] = f2(fa[j], fa[j]);
          uint32_t r[2][16];
          tmem_ld_16x32(src, r[0]);
#pragma unroll
          for (int c = 0; c < BN / 32; ++c) {             // 32 columns (c / 2) of 16 rows (c % 2), the next piece on its way
            tmem_ld_wait();
            tmem_arrived(r[c & 1]);
            if (c < BN / 32 - 1)
              tmem_ld_16x32(src + ((uint32_t)(((c + 1) & 1) * 16) << 16) + ((c + 1) >> 1) * 32, r[(c + 1) & 1]);
            else
              release();
            if ((c & 1) == 0 && c < BN / 32 - 2) {
#pragma unroll
              for (int g = 0; g < 4; ++g)
                s2[((c >> 1) + 1) & 1][g].v = *reinterpret_cast<const uint64_t*>(sbk + ((c >> 1) + 1) * 32 + g * 8);
            }
            if (c == BN / 32 - 2 && more) {
              seen = mbar_try_wait(bar_scfull + 8 * next_slot, next_phase);
              summed = mbar_try_wait(bar_tfull + 8 * next_as, next_aphase);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
              acc2[c * 8 + j] = f2_fma(f2_bits(r[c & 1][2 * j], r[c & 1][2 * j + 1]) * s2[(c >> 1) & 1][j >> 1],
                                       f[(c & 1) * 2 + (j & 1)], acc2[c * 8 + j]);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_scempty + 8 * slot);
          slot = next_slot;
          scphase = next_phase;
          have_scales = __all_sync(0xffffffffu, seen);
          have_sums = __all_sync(0xffffffffu, summed);
          if (have_scales) first_scales();
        }
        if (++as == S::BUFS) { as = 0; aphase ^= 1; }
      }
      if (!ok) break;
      // ---- out
      const int row0 = t.m0 + q * 32, col0 = t.n0 + half * (BN / 2);
      if (row0 >= t.end) continue;                        // nothing of this warp's rows is stored
      staging_free();
      if (MODE == ROWS128) {
        const bool row_in = row0 + lane < t.live;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = row_in ? pack_bf16x2(acc[8 * j + 2 * i], acc[8 * j + 2 * i + 1]) : 0u;
          st_shared_v4(stg + (j >> 3) * S::STG_TILE + lane * 128 + (((j & 7) ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
        }
        if (row0 + 32 <= t.end) {
          staged(col0, 64, row0, 0);
        } else {
          __syncwarp();
          store_slab128(stg, lane, reinterpret_cast<uint16_t*>(p.c), p.N, row0, t.end, col0);
          store_slab128(stg + S::STG_TILE, lane, reinterpret_cast<uint16_t*>(p.c), p.N, row0, t.end, col0 + 64);
          __syncwarp();
        }
      } else if (p.out_bf16) {
#pragma unroll
        for (int cc = 0; cc < BN / 64; ++cc) {            // 32 columns
#pragma unroll
          for (int j = 0; j < 4; ++j) {                   // rows r4 + 8 j
#pragma unroll
            for (int g = 0; g < 4; ++g)
              st_shared_b32(stg + (cc >> 1) * S::STG_TILE + (r4 + 8 * j) * 128 + ((((cc & 1) * 4 + g) ^ r4) << 4) + c2 * 2,
                            pack_bf16x2(acc2[cc * 16 + (j >> 1) * 8 + g * 2 + (j & 1)]));
          }
        }
        staged(col0, 64, row0, t.e);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {                     // 64 columns
          if (h) staging_free();
#pragma unroll
          for (int u = 0; u < 2; ++u) {                   // 32 columns
            const int cc = h * 2 + u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
              for (int g = 0; g < 4; ++g)
                st_shared_b64(stg + u * S::STG_TILE + (r4 + 8 * j) * 128 + (((g * 2 + (c2 >> 2)) ^ r4) << 4) + (c2 & 2) * 4,
                              acc2[cc * 16 + (j >> 1) * 8 + g * 2 + (j & 1)]);
            }
          }
          staged(col0 + h * 64, 32, row0, t.e);
        }
      }
    }
    if (lane == 0) bulk_wait_group<0>();                  // all stores have left shared memory and are visible
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
  if (p.independent) wait_for_kernel_before();
}

}  // namespace smoe
