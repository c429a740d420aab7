// The product of gemm16.cuh for few rows per expert (single tokens, decoding): the weights are the M operand.
//
// Such a call is bound by the read of the weights.  A CTA computes 128 weight rows x up to 64 routed rows, so that each SM streams
// weight tiles of its own; of the routed rows 16 or 64 are fetched and as many pieces of 16 multiplied as hold live ones.  The sum
// over the whole reduction lies transposed in TMEM (lane = weight row, column = routed row).
//
// Where the weight tiles are too few to occupy the SMs a cluster of 2, 4 or 8 CTAs shares one: each takes a stretch of the
// reduction, leaves its sums in its shared memory, and adds up a share of the columns from all of them, in rank order.
#pragma once
#include "gemm16.cuh"

namespace smoe {

struct Few16Params {
  int rows, N, K, E;
  const int *efo, *counts;
  int w_mn;                  // weights lie [E, K, N] (the gradient of the rows)
  __nv_bfloat16* c;          // [rows, N], rows that are not live become zero
  int split;                 // CTAs of a cluster
  int* status;
  volatile int* host_word;
};

struct Few16Smem {
  static constexpr int NT = 64;                               // routed rows of a tile
  static constexpr int A_BYTES = BM * 128, B_BYTES = NT * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES, STAGES = 7;
  static constexpr int EPI_WARPS = 4, EPI_SETS = 2;           // sets take turns by tile: one writes while the other waits for sums
  static constexpr int ACC = 4;                               // TMEM buffers, half of them each set's
  static constexpr int PART_BYTES = NT * BM * 4;              // sums of this CTA: [column][weight row]
  static constexpr int BAR_BYTES = (2 * STAGES + 2 * ACC + 2) * 8;
  static constexpr int AUX_BYTES = 256 + 3 * (kG128Segs + 1) * 4;
  static constexpr int TOTAL = 1024 + STAGES * STAGE_BYTES + PART_BYTES + AUX_BYTES;
  static constexpr int THREADS = 32 * (2 + EPI_WARPS * EPI_SETS);
  static_assert(TOTAL <= 227 * 1024, "shared memory budget");
  static_assert(BAR_BYTES <= 240, "barrier storage");
};

__device__ __forceinline__ void mma_bf16_lo(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %3};\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

struct FewTile16 {
  int e, w0, row0, live;     // live: 1 .. NT
};
// the row tiles of one weight tile are neighbours: L2 serves the weights
__device__ __forceinline__ FewTile16 few_tile16(int tile, int nw, int E, const Segs128& s) {
  FewTile16 t;
  t.e = seg_of_tile(s.tiles, E, tile / nw);
  const int n = s.tiles[t.e + 1] - s.tiles[t.e], r = tile - s.tiles[t.e] * nw;
  t.w0 = r / n * BM;
  t.row0 = s.start[t.e] + r % n * Few16Smem::NT;
  t.live = min(s.live[t.e] - t.row0, Few16Smem::NT);
  return t;
}

__global__ void __launch_bounds__(Few16Smem::THREADS, 1)
gemm16_few_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x16,
                  const __grid_constant__ CUtensorMap tmap_x64, const Few16Params p) {
  using S = Few16Smem;
  constexpr int NT = S::NT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* part = reinterpret_cast<float*>(smem + S::STAGES * S::STAGE_BYTES);
  uint8_t* aux = reinterpret_cast<uint8_t*>(part) + S::PART_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(aux);            // full[S], empty[S], tfull[ACC], tempty[ACC], pfull, pempty
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(aux + 240);
  volatile int* s_abort = reinterpret_cast<volatile int*>(aux + 244);
  Segs128 segs;
  segs.start = reinterpret_cast<int*>(aux + 256);
  segs.live = segs.start + kG128Segs + 1;
  segs.tiles = segs.live + kG128Segs + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split, rank = split > 1 ? (int)cluster_ctarank() : 0;
  const int group = blockIdx.x / split, n_groups = gridDim.x / split;
  const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * S::STAGES;
  const uint32_t bar_tfull = bar_empty + 8 * S::STAGES, bar_tempty = bar_tfull + 8 * S::ACC;
  const uint32_t bar_pfull = bar_tempty + 8 * S::ACC, bar_pempty = bar_pfull + 8;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int s = 0; s < S::ACC; ++s) {
      mbar_init(bar_tfull + 8 * s, 1);
      mbar_init(bar_tempty + 8 * s, S::EPI_WARPS);
    }
    mbar_init(bar_pfull, S::EPI_WARPS * split);
    mbar_init(bar_pempty, S::EPI_WARPS * split);
    *s_abort = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), S::ACC * NT);
    tmem_relinquish();
  }
  wait_for_kernel_before();                   // so far nothing in memory has been touched
  next_kernel_may_start();
  if (warp == 2) load_segs128<false>(segs, p.efo, p.counts, p.E, p.rows, NT, true, 0, 0, lane);
  tc_fence_before();
  __syncthreads();
  if (split > 1) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t smem_base = smem_u32(smem);
  const int nw = (p.N + BM - 1) / BM, nkt = (p.K + kBK16 - 1) / kBK16;
  const int n_total = segs.tiles[p.E] * nw;
  const int k0 = rank * nkt / split, k1 = (rank + 1) * nkt / split;        // split <= nkt: nobody is without
  // Each set of epilogue warps has buffers of its own, and meets every use of them in order.  CTAs that share a tile have few of
  // them and use one set.
  const int sets = split > 1 ? 1 : S::EPI_SETS, bufs = S::ACC / sets;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      prefetch_tmap(&tmap_w);
      prefetch_tmap(&tmap_x16);
      prefetch_tmap(&tmap_x64);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = group; tile < n_total && ok; tile += n_groups) {
        const FewTile16 t = few_tile16(tile, nw, p.E, segs);
        for (int k = k0; k < k1; ++k) {
          ok = mbar_wait(bar_empty + 8 * stage, phase ^ 1);
          if (!ok) break;
          const uint32_t full = bar_full + 8 * stage, at = smem_base + stage * S::STAGE_BYTES;
          mbar_expect_tx(full, S::A_BYTES + (t.live <= 16 ? 16 : NT) * 128);
          if (p.w_mn) {
            tma_load_3d(at, &tmap_w, full, t.w0, k * kBK16, t.e);
            tma_load_3d(at + kPiece16, &tmap_w, full, t.w0 + 64, k * kBK16, t.e);
          } else {
            tma_load_3d(at, &tmap_w, full, k * kBK16, t.w0, t.e);
          }
          tma_load_2d(at + S::A_BYTES, t.live <= 16 ? &tmap_x16 : &tmap_x64, full, k * kBK16, t.row0);
          if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) { *s_abort = 1; fail128(p.status, p.host_word, 701); }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      int stage = 0, turn = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t a_step = desc_step16(p.w_mn);
      for (int tile = group; tile < n_total && ok; tile += n_groups, ++turn) {
        const FewTile16 t = few_tile16(tile, nw, p.E, segs);
        const int use = turn / sets, as = turn % sets * bufs + use % bufs;
        const uint32_t idesc = make_idesc_bf16(BM, (t.live + 15) / 16 * 16, p.w_mn, false);
        ok = mbar_wait(bar_tempty + 8 * as, (use / bufs & 1) ^ 1);
        for (int k = k0; k < k1 && ok; ++k) {
          ok = mbar_wait(bar_full + 8 * stage, phase);
          if (!ok) break;
          tc_fence_after();
          const uint32_t at = smem_base + stage * S::STAGE_BYTES;
          const uint32_t a_lo = desc_lo16(at, p.w_mn), b_lo = desc_lo16(at + S::A_BYTES, false);
#pragma unroll
          for (int kb = 0; kb < kBK16 / 16; ++kb)
            mma_bf16_lo(tmem_base + as * NT, a_lo + a_step * kb, b_lo + 2 * kb, kDescHi16, idesc, k != k0 || kb != 0);
          tc_commit(bar_empty + 8 * stage);
          if (k == k1 - 1) tc_commit(bar_tfull + 8 * as);
          if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) { *s_abort = 1; fail128(p.status, p.host_word, 702); }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue: a warp owns 32 weight rows, its TMEM lanes
    const int q = warp & 3, set = (warp - 2) / S::EPI_WARPS;
    bool ok = true;
    int as = 0;                                               // of this set's
    uint32_t aphase = 0, pphase = 0;
    zero_gaps16(segs, p.E, p.c, p.N, (int)blockIdx.x * 8 + warp - 2, (int)gridDim.x * 8, lane);
    for (int tile = set < sets ? group + set * n_groups : n_total; tile < n_total && ok; tile += sets * n_groups) {
      const FewTile16 t = few_tile16(tile, nw, p.E, segs);
      const int w_row = t.w0 + q * 32 + lane;
      ok = __all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * (set * bufs + as), aphase));
      if (!ok) break;
      tc_fence_after();
      uint32_t r[NT / 16][16];
      const uint32_t src = tmem_base + ((uint32_t)(q * 32) << 16) + (set * bufs + as) * NT;
#pragma unroll
      for (int c = 0; c < NT / 16; ++c)
        if (c * 16 < t.live) tmem_ld16(src + c * 16, r[c]);
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < NT / 16; ++c) tmem_values(r[c]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_tempty + 8 * (set * bufs + as));
      if (++as == bufs) { as = 0; aphase ^= 1; }
      if (split == 1) {
        // (64 stores under a condition each took longer than three blocks: 3800 clocks for four rows)
        __nv_bfloat16* dst = p.c + (int64_t)t.row0 * p.N + w_row;
#pragma unroll
        for (int c = 0; c < NT / 16; ++c) {
          if (c * 16 >= t.live) break;
          const int n = w_row < p.N ? t.live - c * 16 : 0;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (i < n) *dst = __float2bfloat16_rn(__uint_as_float(r[c][i]));
            dst += p.N;
          }
        }
      } else {
        // everyone has read what this CTA left for the tile before
        ok = __all_sync(0xffffffffu, mbar_wait_cluster(bar_pempty, pphase ^ 1));
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < NT / 16; ++c) {
          if (c * 16 >= t.live) break;
#pragma unroll
          for (int i = 0; i < 16; ++i) part[(c * 16 + i) * BM + q * 32 + lane] = __uint_as_float(r[c][i]);
        }
        __syncwarp();
        if (lane < split) mbar_arrive_cluster(map_to_cta(bar_pfull, lane));
        ok = __all_sync(0xffffffffu, mbar_wait_cluster(bar_pfull, pphase));
        if (!ok) break;
        const uint32_t mine = smem_u32(part + q * 32 + lane);
        // a stretch of the rows each, eight of them on their way from a CTA at a time
        const int per = (t.live + split - 1) / split, last = min((rank + 1) * per, t.live);
        for (int i = rank * per; i < last; i += 8) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = 0.f;
#pragma unroll 4
          for (int s = 0; s < split; ++s) {
            const uint32_t from = map_to_cta(mine, s) + i * BM * 4;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += ld_cluster_f32(from + min(j, last - 1 - i) * BM * 4);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (i + j < last && w_row < p.N) p.c[(int64_t)(t.row0 + i + j) * p.N + w_row] = __float2bfloat16_rn(v[j]);
        }
        __syncwarp();
        if (lane < split) mbar_arrive_cluster(map_to_cta(bar_pempty, lane));
        pphase ^= 1;
      }
    }
    if (!ok && lane == 0) { *s_abort = 1; fail128(p.status, p.host_word, 703); }
  }

  // common exit: everyone arrives here, also after a failed wait
  __syncthreads();
  if (*s_abort) {                             // copies and MMAs in flight may still write this CTA's memory
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (split > 1) cluster_sync_all();          // the others may still read this CTA's sums
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, S::ACC * NT);
}

}  // namespace smoe
