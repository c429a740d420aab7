// Host side of the products of bf16 rows grouped by expert.
#include "gemm16.cuh"
#include "gemm16_few.cuh"
#include "gemv16.cuh"
#include "host.h"
#include "smoe_b200.h"

namespace smoe {

// bf16 [depth, rows, cols], rows `pitch` values apart, box {64, box_rows, 1} in the 128-byte swizzle; what lies beyond an extent
// reads as zero
static int make_tmap16(CUtensorMap* m, const void* base, uint64_t depth, uint64_t rows, uint64_t cols, uint64_t pitch, uint32_t box_rows,
                       int dims) {
  if (!load_encode()) return SMOE_ERR_DRIVER;
  cuuint64_t extent[3] = {cols, rows, depth};
  cuuint64_t strides[2] = {pitch * 2, pitch * rows * 2};
  cuuint32_t box[3] = {64, box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = g_encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dims, const_cast<void*>(base), extent, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? SMOE_OK : SMOE_ERR_TMAP;
}

// The result [depth, rows, cols], box of 32 rows of 128 bytes
static int make_tmap16_out(CUtensorMap* m, void* base, bool bf16, uint64_t depth, uint64_t rows, uint64_t cols) {
  if (!load_encode()) return SMOE_ERR_DRIVER;
  const cuuint64_t es = bf16 ? 2 : 4;
  cuuint64_t extent[3] = {cols, rows, depth};
  cuuint64_t strides[2] = {cols * es, cols * rows * es};
  cuuint32_t box[3] = {(cuuint32_t)(128 / es), 32, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = g_encode(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, base, extent, strides,
                              box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? SMOE_OK : SMOE_ERR_TMAP;
}

static int64_t up16(int64_t n, int64_t m) { return (n + m - 1) / m; }
static bool size16(int64_t n) { return n > 0 && n % 8 == 0 && n < (int64_t)1 << 24; }
static bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }
// rows of n values, ld apart
static bool rows16(int64_t rows, int64_t n, int64_t ld) { return ld >= n && ld % 8 == 0 && ld < (int64_t)1 << 38; }

static int check16(int64_t rows, int64_t N, int64_t K, int64_t E, const int* efo, const int* counts, const int* status) {
  if (rows < 0 || rows >= (int64_t)1 << 30 || !size16(N) || !size16(K) || E <= 0 || E > kMaxExperts2) return SMOE_ERR_SHAPE;
  if (E * N * K >= (int64_t)1 << 40) return SMOE_ERR_SHAPE;
  if ((!efo && (E != 1 || counts)) || !status) return SMOE_ERR_ARG;
  return SMOE_OK;
}

template <int MODE, int COLS>
static int launch16(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const Gemm16Params& p, int64_t tiles,
                    cudaStream_t stream) {
  using S = Gemm16Smem<COLS>;
  static bool attr_set[kMaxDevices] = {};
  auto kern = gemm16_kernel<MODE, COLS>;
  if (!ensure_smem_attr(kern, S::TOTAL, attr_set)) return SMOE_ERR_LAUNCH;
  int64_t pairs = sm_count() / 2;
  if (tiles < pairs) pairs = tiles;
  return launch_early(kern, (unsigned)(2 * pairs), S::THREADS, S::TOTAL, 0, stream, ta, tb, tc, p) == cudaSuccess ? SMOE_OK
                                                                                                                 : SMOE_ERR_LAUNCH;
}
// Narrow tiles where the wide ones would leave half of the CTA pairs without any, or have no use for their width (us, wide / narrow: 512 x
// 4096 x 4096 24.6 / 18.1, 256 x 8192 x 2048 15.9 / 12.4, 8192 x 128 x 2048 15.3 / 12.1; of 64 tiles, 2048 x 2048 x 2048, 16.3 / 18.4)
static bool narrow16(int64_t tiles, int64_t cols) { return tiles <= sm_count() / 4 || cols <= 128; }

// Weights as the wide operand: where the rows of an expert make one tile of 64, or the tiles are few: one for each SM of a single
// projection, two of experts, whose 256-row tiles are then mostly empty (us, the other kernel / few):
//   1 expert    4096 x 4096  256 rows 17.4 / 15.8, 512 18.1 / 26.4;  1024 x 4096  1024 rows 16.8 / 15.3, 2048 18.0 / 26.1;
//               1000 x 720  2000 rows 7.7 / 9.1
//   8 experts   512 x 512  2048 rows 8.2 / 5.9, 4096 8.5 / 7.7, 8192 9.0 / 11.8;  1024 x 1024  1024 rows 11.3 / 8.1, 2048 9.2 / 10.9;
//               4096 x 2048  512 rows 31 / 26, 2048 35 / 50
//   128         1536 x 2048  4096 rows 177 / 128, 8192 170 / 133, 12288 168 / 170;  unevenly routed 166 / 142, 182 / 171, 189 / 206
// The gradient of the rows reads its weights across and takes up to a sixth longer with few.
//   Segments that are padded to multiples of 128, which counts and a table of a multiple of 128 rows stand for, have live rows that are not
// known here, and two tiles a block at most: one such block an expert and an eighth more, as the metadata allocates for up to 16 rows an
// expert (us, the other kernel / few, y; gradient of the rows, by live rows an expert of allocated ones):
//   128 of 1536 x 2048  16 of 144 177 / 139; 173 / 141   1 to 128 of 128 178 / 148; 174 / 150   90 on average 181 / 173; 175 / 181
//   128 of 2048 x 768   16 of 144 126 / 85; 117 / 81     1 to 128 of 128 124 / 95; 118 / 89     90 on average 104 / 103; 103 / 100
//   37 of 1024 x 1024    4 of 135 21.1 / 12.9; 19.3 / 12.4   1 to 128 of 128 21.5 / 21.8; 20.4 / 22.2   90 21.1 / 22.9; 19.6 / 23.1
//   8 of 4096 x 2048    16 of 144 32.8 / 26.7; 31.0 / 24.9   1 to 128 of 128 33.0 / 29.5; 31.0 / 34.9   90 32.6 / 34.2; 30.7 / 33.1
// Blocks that are all full pay: 0 to 20 %, 128 of 2048 x 768 a third on a GPU at lower clocks (115 / 150; at full clocks 89 / 98).
//   Of segments with gaps all rows may live, and those above 128 take a third tile (129 of 136 rows, 128 of 1536 x 2048: 170 / 219; 164 / 255).
static bool few_rows16(int64_t rows, int64_t N, int64_t E, bool padded) {
  if (rows <= (padded ? 9 * 128 * E / 8 : Few16Smem::NT * E)) return true;
  const int64_t busy = rows < E ? rows : E;
  return (rows + (Few16Smem::NT - 1) * busy) / Few16Smem::NT * up16(N, 128) <= (E == 1 ? 1 : 2) * sm_count();
}

static int few16(const void* x, int64_t ldx, const void* w, const int* efo, const int* counts, void* y, int64_t rows, int64_t N, int64_t K,
                 int64_t E, int w_mn, int* status, int* host_word, cudaStream_t stream) {
  CUtensorMap tw, tx16, tx64;
  int rc = w_mn ? make_tmap16(&tw, w, E, K, N, N, 64, 3) : make_tmap16(&tw, w, E, N, K, K, 128, 3);
  if (!rc) rc = make_tmap16(&tx16, x, 1, rows, K, ldx, 16, 2);
  if (!rc) rc = make_tmap16(&tx64, x, 1, rows, K, ldx, Few16Smem::NT, 2);
  if (rc) return rc;
  static bool attr_set[kMaxDevices] = {};
  if (!ensure_smem_attr(gemm16_few_kernel, Few16Smem::TOTAL, attr_set)) return SMOE_ERR_LAUNCH;
  const int sms = sm_count();
  const int64_t busy = rows < E ? rows : E;
  const int64_t tiles = (rows + (Few16Smem::NT - 1) * busy) / Few16Smem::NT * up16(N, 128);      // as many as there can be
  const int64_t kb = up16(K, kBK16);
  // Few tiles are shared by clusters, where the reduction is long enough for what the sums' exchange costs, some 1.7 us (us with 1 / 2 / 4
  // / 8 CTAs, one row: 4096 x 1024 6.4 / 7.3 / 7.3 / -, x 1792 8.4 / 8.5 / 8.1 / -, x 4096 15.6 / 13.1 / 11.0 / -; 1024 x 1280 6.6 / 6.7 /
  // 5.9 / 6.2, x 16384 47 / 28 / 17.7 / -; 8192 x 2560 11.2 / 11.8 / 16 / -, x 4096 16.5 / 15.6 / 19 / -; 64 rows: 4096 x 1536 8.4 / 10.4 /
  // 9.5 / -, 2048 x 2048 9.5 / 10.8 / 8.9 / -).  Eight find room together on half of the SMs only (2048 x 1536 7.0 with four, 13.2).
  int split = 1;
  if (tiles * 4 <= sms && kb >= (rows > 16 ? 32 : 20)) split = tiles * 16 <= sms && kb >= 64 ? 8 : 4;
  else if (tiles * 2 <= sms && kb >= 64) split = 2;
  Few16Params p{(int)rows, (int)N, (int)K, (int)E, efo, counts, w_mn, (__nv_bfloat16*)y, split, status, host_word};
  int64_t groups = sms / split;
  if (tiles < groups) groups = tiles;
  return launch_early(gemm16_few_kernel, (unsigned)(groups * split), Few16Smem::THREADS, Few16Smem::TOTAL, (unsigned)split, stream, tw, tx16,
                      tx64, p) == cudaSuccess
             ? SMOE_OK
             : SMOE_ERR_LAUNCH;
}

// Weight gradients of few tiles: a segment's rows are cut into stretches, so that every CTA pair has a tile; a stretch's sums pass through
// memory once, and a launch adds them up in their order.  Where that pays: it costs some 5 us, a block of 64 rows some 0.2 of a narrow
// tile and 0.3 of a wide one (us, 1 stretch with narrow tiles / 2 / 4 / 8 / 16, one expert: 512 x 512, 16384 rows 55 / 33 / 21 / 16 /
// 17; 64 x 512 54 / 31 / 19 / 14 / 12; 1024 x 1024 56 / 36 / 33 / 36 / 49, 2048 rows 11.4 / 11.5 / 12.5 / 16 / 25; 8 of 512 x 256, 16384
// rows 12.0 / 13.0 / 14.4 / 18 / 27).
static int wgrad_split16(int64_t N, int64_t K, int64_t rows, int64_t E) {
  const int64_t tiles = E * up16(N, 256) * up16(K, K <= 128 ? 128 : 256), pairs = sm_count() / 2, blocks = rows / E / kBK16;
  int64_t split = pairs / tiles;
  if (split > blocks / 8) split = blocks / 8;
  if (split > 16) split = 16;
  return split >= 2 && blocks * (2 * split - 3) > 50 * split ? (int)split : 1;
}

// out = (out +) the sum of `split` partial sums, each `fours` of four values
__global__ void __launch_bounds__(256) wgrad_sum_kernel(const float4* part, int split, int64_t fours, void* out, int bf16,
                                                        int accumulate) {
  wait_for_kernel_before();
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < fours; i += (int64_t)gridDim.x * blockDim.x) {
    float4 v = part[i];
#pragma unroll 4
    for (int s = 1; s < split; ++s) {
      const float4 u = part[s * fours + i];
      v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
    }
    if (bf16) {
      ((uint2*)out)[i] = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
    } else {
      float4* o = (float4*)out + i;
      if (accumulate) atomicAdd(o, v);                    // (once for each value: another stream's sums into it are not lost)
      else *o = v;
    }
  }
}

// A handful of rows without tensor cores: one an expert, or so few products that a warp's reading of x again for every two weight rows does
// not matter (us, tensor cores / without: one row of 4096 x 4096 10.9 / 8.2, of 8192 x 8192 26.0 / 23.7, of 1024 x 1024 5.8 / 2.7, of 1000 x
// 720 5.2 / 2.6; of 4096 x 4096 2 rows 11.0 / 10.6, 4 11.0 / 12.6, 8 11.1 / 21; 8 of 1024 x 1024 5.8 / 4.3; one for each of 8 experts of 4096
// x 2048 23.2 / 23.6, two each 23.4 / 31; of 128 experts of 1536 x 2048 8 rows 11.7 / 11.8, all of one expert 10.2 / 6.9, 16 23.3 / 18.9, of
// 2048 x 768 7.2 / 7.3 and 11.2 / 11.9).
static bool gemv_rows16(int64_t rows, int64_t N, int64_t K, int64_t E) {
  return rows <= kGemvMost && (rows <= E || rows * N * K <= (int64_t)12 << 20);
}

static int gemv16(const void* x, int64_t ldx, const void* w, const int* efo, const int* counts, void* y, int64_t rows, int64_t N, int64_t K,
                  int64_t E, cudaStream_t stream) {
  const Gemv16Params p{(int)rows, (int)N, (int)K, (int)E, ldx, efo, counts, (const __nv_bfloat16*)x, (const __nv_bfloat16*)w, (__nv_bfloat16*)y};
  const int64_t blocks = up16(rows * N, kGemvCols * kGemvWarps), most = (int64_t)sm_count() * kGemvBlocks;
  return launch_early(gemv16_kernel, (unsigned)(blocks < most ? blocks : most), 32 * kGemvWarps, 0, 0, stream, p) == cudaSuccess
             ? SMOE_OK
             : SMOE_ERR_LAUNCH;
}

}  // namespace smoe

using namespace smoe;

extern "C" {

int smoe_grouped_rows(const void* x_bf16, int64_t ldx, const void* w_bf16, int w_transposed, const int32_t* efo, const int32_t* counts,
                      void* y_bf16, int64_t rows, int64_t N, int64_t K, int64_t E, int32_t* status, int32_t* pinned_host_word,
                      void* stream) {
  int rc = check16(rows, N, K, E, efo, counts, status);
  if (rc) return rc;
  if (!rows16(rows, K, ldx)) return SMOE_ERR_SHAPE;
  if (rows == 0) return SMOE_OK;
  if (!x_bf16 || !w_bf16 || !y_bf16) return SMOE_ERR_ARG;
  if (!on16(x_bf16) || !on16(w_bf16) || !on16(y_bf16)) return SMOE_ERR_ALIGN;
  if (!w_transposed && gemv_rows16(rows, N, K, E))
    return gemv16(x_bf16, ldx, w_bf16, efo, counts, y_bf16, rows, N, K, E, (cudaStream_t)stream);
  if (few_rows16(rows, N, E, counts && rows % 128 == 0))
    return few16(x_bf16, ldx, w_bf16, efo, counts, y_bf16, rows, N, K, E, w_transposed != 0, status, pinned_host_word,
                 (cudaStream_t)stream);
  // every segment may end in a tile that is not full
  const int64_t row_tiles = efo ? (rows + 255 * (rows < E ? rows : E)) / 256 : up16(rows, 256);
  const bool narrow = narrow16(row_tiles * up16(N, 256), N);
  CUtensorMap ta, tb, tc;
  rc = make_tmap16(&ta, x_bf16, 1, rows, K, ldx, 128, 2);
  if (!rc) rc = w_transposed ? make_tmap16(&tb, w_bf16, E, K, N, N, 64, 3) : make_tmap16(&tb, w_bf16, E, N, K, K, narrow ? 64 : 128, 3);
  if (!rc) rc = make_tmap16_out(&tc, y_bf16, true, 1, rows, N);
  if (rc) return rc;
  Gemm16Params p{};
  p.rows = (int)rows; p.N = (int)N; p.K = (int)K; p.E = (int)E; p.split = 1;
  p.efo = efo; p.counts = counts; p.b_mn = w_transposed != 0; p.c = y_bf16;
  p.status = status; p.host_word = pinned_host_word;
  return narrow ? launch16<ROWS16, 128>(ta, tb, tc, p, row_tiles * up16(N, 128), (cudaStream_t)stream)
                : launch16<ROWS16, 256>(ta, tb, tc, p, row_tiles * up16(N, 256), (cudaStream_t)stream);
}

int64_t smoe_grouped_wgrad_workspace(int64_t N, int64_t K, int64_t rows, int64_t E) {
  if (!size16(N) || !size16(K) || rows < 0 || rows >= (int64_t)1 << 30 || E <= 0 || E > kMaxExperts2) return -1;
  const int split = wgrad_split16(N, K, rows, E);
  return split > 1 ? split * E * N * K * 4 : 0;
}

int smoe_grouped_wgrad(const void* dy_bf16, int64_t ldy, const void* x_bf16, int64_t ldx, const int32_t* efo, const int32_t* counts,
                       void* dw, int64_t N, int64_t K, int64_t rows, int64_t E, int out_bf16, int accumulate, void* workspace,
                       int32_t* status, int32_t* pinned_host_word, void* stream) {
  int rc = check16(rows, N, K, E, efo, counts, status);
  if (rc) return rc;
  if (!rows16(rows, N, ldy) || !rows16(rows, K, ldx)) return SMOE_ERR_SHAPE;
  if ((out_bf16 && accumulate) || !dw) return SMOE_ERR_ARG;
  if (!on16(dw)) return SMOE_ERR_ALIGN;
  if (rows == 0) {                                  // an empty sum
    if (accumulate) return SMOE_OK;
    return cudaMemsetAsync(dw, 0, (size_t)(E * N * K) * (out_bf16 ? 2 : 4), (cudaStream_t)stream) == cudaSuccess ? SMOE_OK
                                                                                                             : SMOE_ERR_LAUNCH;
  }
  if (!dy_bf16 || !x_bf16) return SMOE_ERR_ARG;
  if (!on16(dy_bf16) || !on16(x_bf16)) return SMOE_ERR_ALIGN;
  const int split = wgrad_split16(N, K, rows, E);
  if (split > 1 && !workspace) return SMOE_ERR_ARG;
  if (split > 1 && !on16(workspace)) return SMOE_ERR_ALIGN;
  CUtensorMap ta, tb, tc;
  rc = make_tmap16(&ta, dy_bf16, 1, rows, N, ldy, 64, 2);
  if (!rc) rc = make_tmap16(&tb, x_bf16, 1, rows, K, ldx, 64, 2);
  if (!rc) rc = make_tmap16_out(&tc, split > 1 ? workspace : dw, split == 1 && out_bf16, split * E, N, K);
  if (rc) return rc;
  Gemm16Params p{};
  p.rows = (int)rows; p.M = (int)N; p.N = (int)K; p.E = (int)E; p.split = split;
  p.efo = efo; p.counts = counts; p.c = split > 1 ? workspace : dw; p.out_bf16 = split == 1 && out_bf16;
  p.accumulate = split == 1 && accumulate;
  p.status = status; p.host_word = pinned_host_word;
  const cudaStream_t st = (cudaStream_t)stream;
  const int64_t row_tiles = split * E * up16(N, 256);
  rc = narrow16(row_tiles * up16(K, 256), K) ? launch16<WGRAD16, 128>(ta, tb, tc, p, row_tiles * up16(K, 128), st)
                                             : launch16<WGRAD16, 256>(ta, tb, tc, p, row_tiles * up16(K, 256), st);
  if (rc || split == 1) return rc;
  const int64_t fours = E * N * K / 4, blocks = up16(fours, 256), most = (int64_t)sm_count() * 8;
  return launch_early(wgrad_sum_kernel, (unsigned)(blocks < most ? blocks : most), 256, 0, 0, st, (const float4*)workspace, split, fours, dw,
                      (int)(out_bf16 != 0), (int)(accumulate != 0)) == cudaSuccess
             ? SMOE_OK
             : SMOE_ERR_LAUNCH;
}

}  // extern "C"
