// The product of gemm128.cuh for few rows per expert (single tokens, decoding): the weights are the M operand.
//
// Such a call is bound by the read of the weights (64 tokens x 8 over 128 experts of 2048 x 1536: 72 us, 5.6 TB/s; one row of 4096 x
// 4096 9 us).  A CTA computes 128 weight rows x up to 64 routed rows, so that each SM streams
// weight tiles of its own; of the routed rows 16 or 64 are fetched and as many pieces of 16 multiplied as hold live ones.  The sum
// of a block of 128 lies transposed in TMEM (lane = weight row, column = routed row) in one of eight buffers of 64 columns; the
// epilogue warps scale it - one number a column, which every lane reads from shared memory - and keep 64 f32 sums a thread.
//
// Where the weight tiles are too few to occupy the SMs a cluster of 2, 4 or 8 CTAs shares one: each takes a stretch of the
// reduction, leaves its sums in its shared memory, and adds up a share of the columns from all of them, in rank order.
//
// Where its caller allows it (see gemm128_few) the kernel starts before the one before it in the stream has ended: until
// wait_for_kernel_before it touches only offsets, counts and weights.
#pragma once
#include "gemm128.cuh"

namespace smoe {

struct Few128Params {
  int rows, N, K, E;
  const int *efo, *counts;
  const float *w_s, *x_s;    // [E, N/128, K/128], [rows, K/128]
  __nv_bfloat16* c;          // [rows, N], live rows only are written
  int split;                 // CTAs of a cluster
  int rest_of;               // see load_segs128
  int independent;           // of the kernel before in the stream: waited for at the end only
  int* status;
  volatile int* host_word;
};

constexpr int kFewBars = 640;        // bytes of barriers

struct Few128Smem {
  static constexpr int NT = 64;                               // routed rows of a tile
  static constexpr int A_BYTES = BM * BK, B_BYTES = NT * BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES, STAGES = 7;
  static constexpr int ACC = 8;                               // TMEM buffers
  static constexpr int EPI_WARPS = 4, EPI_SETS = 2;           // sets take turns by tile: one writes while the other reads sums
  static constexpr int PART_BYTES = NT * BM * 4;              // sums of this CTA: [column][weight row]
  static constexpr int SX_GROUP = 8;                          // blocks whose factors travel together
  static constexpr int SX_SLOTS = 4, SX_BYTES = SX_SLOTS * SX_GROUP * NT * 4;
  static constexpr int AUX_BYTES = kFewBars + 16 + 3 * (kG128Segs + 1) * 4;
  static constexpr int TOTAL = 1024 + STAGES * STAGE_BYTES + PART_BYTES + SX_BYTES + AUX_BYTES;
  static constexpr int SCALER = 2 + EPI_WARPS * EPI_SETS;                // warp
  static constexpr int THREADS = 32 * (SCALER + 1);
  static_assert(TOTAL <= 227 * 1024, "shared memory budget");
  static_assert((2 * STAGES + 2 * ACC + 2 + 2 * SX_SLOTS) * 8 <= kFewBars, "barrier storage");
};

struct FewTile128 {
  int e, w0, row0, live;     // live: 1 .. NT
};
// the row tiles of one weight tile are neighbours: L2 serves the weights
__device__ __forceinline__ FewTile128 few_tile128(int tile, int nw, int E, const Segs128& s) {
  FewTile128 t;
  t.e = seg_of_tile(s.tiles, E, tile / nw);
  const int n = s.tiles[t.e + 1] - s.tiles[t.e], r = tile - s.tiles[t.e] * nw;
  t.w0 = r / n * BM;
  t.row0 = s.start[t.e] + r % n * Few128Smem::NT;
  t.live = min(s.live[t.e] - t.row0, Few128Smem::NT);
  return t;
}

__global__ void __launch_bounds__(Few128Smem::THREADS, 1)
gemm128_few_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x16,
                   const __grid_constant__ CUtensorMap tmap_x64, const Few128Params p) {
  using S = Few128Smem;
  constexpr int NT = S::NT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* part = reinterpret_cast<float*>(smem + S::STAGES * S::STAGE_BYTES);
  uint8_t* sx_all = reinterpret_cast<uint8_t*>(part) + S::PART_BYTES;
  uint8_t* aux = sx_all + S::SX_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(aux);            // full[S], empty[S], tfull[ACC], tempty[ACC], pfull, pempty, sfull[], sempty[]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(aux + kFewBars);
  volatile int* s_abort = reinterpret_cast<volatile int*>(aux + kFewBars + 4);
  Segs128 segs;
  segs.start = reinterpret_cast<int*>(aux + kFewBars + 16);
  segs.live = segs.start + kG128Segs + 1;
  segs.tiles = segs.live + kG128Segs + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split, rank = split > 1 ? (int)cluster_ctarank() : 0;
  const int group = blockIdx.x / split, n_groups = gridDim.x / split;
  const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * S::STAGES;
  const uint32_t bar_tfull = bar_empty + 8 * S::STAGES, bar_tempty = bar_tfull + 8 * S::ACC;
  const uint32_t bar_pfull = bar_tempty + 8 * S::ACC, bar_pempty = bar_pfull + 8;
  const uint32_t bar_sfull = bar_pempty + 8, bar_sempty = bar_sfull + 8 * S::SX_SLOTS;

  if (warp == 2) load_segs128<true>(segs, p.efo, p.counts, p.E, p.rows, NT, true, 0, p.rest_of, lane);
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int s = 0; s < S::ACC; ++s) {
      mbar_init(bar_tfull + 8 * s, 1);
      mbar_init(bar_tempty + 8 * s, S::EPI_WARPS);
    }
    for (int s = 0; s < S::SX_SLOTS; ++s) {
      mbar_init(bar_sfull + 8 * s, 1);
      mbar_init(bar_sempty + 8 * s, S::EPI_WARPS);
    }
    mbar_init(bar_pfull, S::EPI_WARPS * split);
    mbar_init(bar_pempty, S::EPI_WARPS * split);
    *s_abort = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  if (split > 1) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t smem_base = smem_u32(smem);
  next_kernel_may_start();                    // (which waits for this one's end before it touches anything)
  const int nw = (p.N + BM - 1) / BM, nkt = (p.K + 127) / 128;
  const int n_total = segs.tiles[p.E] * nw;
  const int k0 = rank * nkt / split, k1 = (rank + 1) * nkt / split;        // split <= nkt: nobody is without
  // Each set of epilogue warps has buffers and slots of its own, and meets every use of them in order: a wait by parity cannot
  // tell a phase from the one after next.  CTAs that share a tile have few of them and use one set.
  const int sets = split > 1 ? 1 : S::EPI_SETS, bufs = S::ACC / sets, slots = S::SX_SLOTS / sets;
  const int blocks = k1 - k0, groups = (blocks + S::SX_GROUP - 1) / S::SX_GROUP;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      prefetch_tmap(&tmap_w);
      prefetch_tmap(&tmap_x16);
      prefetch_tmap(&tmap_x64);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      // 16 routed rows or all 64 (a copy takes this thread some 200 clocks to issue)
      auto weights = [&](const FewTile128& t, int k, int st) {
        mbar_expect_tx(bar_full + 8 * st, S::A_BYTES + (t.live <= 16 ? 16 : NT) * BK);
        tma_load_3d(smem_base + st * S::STAGE_BYTES, &tmap_w, bar_full + 8 * st, k * 128, t.w0, t.e);
      };
      // the weights of the first pass over the ring are asked for before the kernel that makes the routed rows has ended
      const int early = group < n_total ? min(S::STAGES, blocks) : 0;
      if (early) {
        const FewTile128 t = few_tile128(group, nw, p.E, segs);
        for (int i = 0; i < early; ++i) weights(t, k0 + i, i);
      }
      if (!p.independent) wait_for_kernel_before();
      for (int tile = group; tile < n_total && ok; tile += n_groups) {
        const FewTile128 t = few_tile128(tile, nw, p.E, segs);
        for (int k = k0; k < k1; ++k) {
          if (tile != group || k - k0 >= early) {
            ok = mbar_wait(bar_empty + 8 * stage, phase ^ 1);
            if (!ok) break;
            weights(t, k, stage);
          }
          tma_load_2d(smem_base + stage * S::STAGE_BYTES + S::A_BYTES, t.live <= 16 ? &tmap_x16 : &tmap_x64, bar_full + 8 * stage,
                      k * 128, t.row0);
          if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) { *s_abort = 1; fail128(p.status, p.host_word, 501); }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      int stage = 0, turn = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = group; tile < n_total && ok; tile += n_groups, ++turn) {
        const FewTile128 t = few_tile128(tile, nw, p.E, segs);
        const uint32_t use0 = (uint32_t)(turn / sets) * blocks;
        const uint32_t idesc = make_idesc_f8(BM, (t.live + 15) / 16 * 16, false);
        for (int k = k0; k < k1; ++k) {
          const uint32_t use = use0 + (k - k0), as = turn % sets * bufs + use % bufs, aphase = use / bufs & 1;
          ok = mbar_wait(bar_tempty + 8 * as, aphase ^ 1) && mbar_wait(bar_full + 8 * stage, phase);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_src = smem_base + stage * S::STAGE_BYTES;
          const uint64_t a_desc = make_desc_kmajor_sw128(a_src), b_desc = make_desc_kmajor_sw128(a_src + S::A_BYTES);
#pragma unroll
          for (int kb = 0; kb < BK / 32; ++kb) mma_f8(tmem_base + as * NT, a_desc + 2 * kb, b_desc + 2 * kb, idesc, kb != 0);
          tc_commit(bar_empty + 8 * stage);
          tc_commit(bar_tfull + 8 * as);
          if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) { *s_abort = 1; fail128(p.status, p.host_word, 502); }
    }
    __syncwarp();
  } else if (warp == S::SCALER) {
    // ------------------------------------------------------------ factors of the columns, the row's scale times the weight's
    // Rows of scales lie [rows, K/128]: a lane walks two of them, eight blocks at a time, and asks for the next eight, of whichever
    // tile, before it hands over these, so that nobody waits for HBM (one block ahead in the epilogue's registers: 4.6 TB/s).
    constexpr int G = S::SX_GROUP;
    float* sx = reinterpret_cast<float*>(sx_all);
    int tile = group, k = k0;
    uint32_t given = 0;                                       // groups handed over
    bool ok = true;
    const float *ws = nullptr, *xs0 = nullptr, *xs1 = nullptr;
    bool in0 = false, in1 = false;
    auto at_tile = [&] {
      if (tile >= n_total) return;
      const FewTile128 t = few_tile128(tile, nw, p.E, segs);
      ws = p.w_s + ((int64_t)t.e * nw + t.w0 / 128) * nkt;
      in0 = lane < t.live;
      in1 = lane + 32 < t.live;
      xs0 = p.x_s + (int64_t)(t.row0 + (in0 ? lane : 0)) * nkt;
      xs1 = p.x_s + (int64_t)(t.row0 + (in1 ? lane + 32 : 0)) * nkt;
    };
    auto ask = [&](float (&x0)[G], float (&x1)[G]) {          // and steps on
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const int kk = min(k + i, k1 - 1);
        const float w = ws[kk];
        x0[i] = in0 ? xs0[kk] * w : 0.f;
        x1[i] = in1 ? xs1[kk] * w : 0.f;
      }
      k += G;
      if (k >= k1) {
        k = k0;
        tile += n_groups;
        at_tile();
      }
    };
    auto give = [&](const float (&x0)[G], const float (&x1)[G]) {
      const uint32_t turn = given / groups, use = turn / sets * groups + given % groups;
      const uint32_t slot = turn % sets * slots + use % slots;
      ok = __all_sync(0xffffffffu, mbar_wait(bar_sempty + 8 * slot, (use / slots & 1) ^ 1));
      if (!ok) return;
      float* to = sx + slot * G * NT;
#pragma unroll
      for (int i = 0; i < G; ++i) {
        to[i * NT + lane] = x0[i];
        to[i * NT + 32 + lane] = x1[i];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_sfull + 8 * slot);
      ++given;
    };
    if (!p.independent) wait_for_kernel_before();             // every block, also one without tiles
    at_tile();
    float a0[G], a1[G], b0[G], b1[G];
    if (tile < n_total) {
      ask(a0, a1);
      while (ok) {
        const bool more = tile < n_total;
        if (more) ask(b0, b1);
        give(a0, a1);
        if (!more || !ok) break;
        const bool again = tile < n_total;
        if (again) ask(a0, a1);
        give(b0, b1);
        if (!again) break;
      }
    }
    if (!ok && lane == 0) { *s_abort = 1; fail128(p.status, p.host_word, 504); }
  } else {
    // ------------------------------------------------------------ epilogue: a warp owns 32 weight rows, its TMEM lanes
    const int q = warp & 3, set = (warp - 2) / S::EPI_WARPS;
    const float* sx = reinterpret_cast<const float*>(sx_all);
    bool ok = true;
    int as = 0, slot = 0;                                     // of this set's
    uint32_t aphase = 0, sphase = 0, pphase = 0;
    for (int tile = set < sets ? group + set * n_groups : n_total; tile < n_total && ok; tile += sets * n_groups) {
      const FewTile128 t = few_tile128(tile, nw, p.E, segs);
      const int w_row = t.w0 + q * 32 + lane;
      float acc[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) acc[i] = 0.f;
      for (int k = k0; k < k1; ++k) {
        const int in_group = (k - k0) % S::SX_GROUP;
        if (in_group == 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(bar_sfull + 8 * (set * slots + slot), sphase));
          if (!ok) break;
        }
        const float* sk = sx + ((set * slots + slot) * S::SX_GROUP + in_group) * NT;
        ok = __all_sync(0xffffffffu, mbar_wait(bar_tfull + 8 * (set * bufs + as), aphase));
        if (!ok) break;
        tc_fence_after();
        const uint32_t src = tmem_base + ((uint32_t)(q * 32) << 16) + (set * bufs + as) * NT;
#pragma unroll
        for (int c = 0; c < NT / 16; ++c) {
          if (c * 16 < t.live) {
            uint32_t r[16];
            tmem_ld16(src + c * 16, r);
            tmem_ld_wait();
            tmem_arrived(r);
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const float4 s4 = *reinterpret_cast<const float4*>(sk + c * 16 + i);
              acc[c * 16 + i] = fmaf(__uint_as_float(r[i]), s4.x, acc[c * 16 + i]);
              acc[c * 16 + i + 1] = fmaf(__uint_as_float(r[i + 1]), s4.y, acc[c * 16 + i + 1]);
              acc[c * 16 + i + 2] = fmaf(__uint_as_float(r[i + 2]), s4.z, acc[c * 16 + i + 2]);
              acc[c * 16 + i + 3] = fmaf(__uint_as_float(r[i + 3]), s4.w, acc[c * 16 + i + 3]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar_tempty + 8 * (set * bufs + as));
          if (in_group == S::SX_GROUP - 1 || k == k1 - 1) mbar_arrive(bar_sempty + 8 * (set * slots + slot));
        }
        if (in_group == S::SX_GROUP - 1 || k == k1 - 1) {
          if (++slot == slots) { slot = 0; sphase ^= 1; }
        }
        if (++as == bufs) { as = 0; aphase ^= 1; }
      }
      if (!ok) break;
      if (split == 1) {
        // (64 stores under a condition each took longer than three blocks: 3800 clocks for four rows)
        __nv_bfloat16* dst = p.c + (int64_t)t.row0 * p.N + w_row;
#pragma unroll
        for (int c = 0; c < NT; c += 16) {
          if (c >= t.live) break;
          const int n = w_row < p.N ? t.live - c : 0;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (i < n) *dst = __float2bfloat16_rn(acc[c + i]);
            dst += p.N;
          }
        }
      } else {
        // everyone has read what this CTA left for the tile before
        ok = __all_sync(0xffffffffu, mbar_wait_cluster(bar_pempty, pphase ^ 1));
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < NT; c += 16) {
          if (c >= t.live) break;
#pragma unroll
          for (int i = 0; i < 16; ++i) part[(c + i) * BM + q * 32 + lane] = acc[c + i];
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
          for (int r = 0; r < split; ++r) {
            const uint32_t from = map_to_cta(mine, r) + i * BM * 4;
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
    if (!ok && lane == 0) { *s_abort = 1; fail128(p.status, p.host_word, 503); }
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
  if (warp == 1) tmem_dealloc(tmem_base, 512);
  if (p.independent) wait_for_kernel_before();
}

}  // namespace smoe
