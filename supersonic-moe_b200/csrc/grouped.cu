// Host side of the products of bf16 rows grouped by expert.
#include "gemm16.cuh"
#include "gemm16_few.cuh"
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

template <int MODE>
static int launch16(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const Gemm16Params& p, int64_t tiles,
                    cudaStream_t stream) {
  static bool attr_set[kMaxDevices] = {};
  auto kern = gemm16_kernel<MODE>;
  if (!ensure_smem_attr(kern, Gemm16Smem::TOTAL, attr_set)) return SMOE_ERR_LAUNCH;
  int64_t pairs = sm_count() / 2;
  if (tiles < pairs) pairs = tiles;
  return launch_early(kern, (unsigned)(2 * pairs), Gemm16Smem::THREADS, Gemm16Smem::TOTAL, 0, stream, ta, tb, tc, p) == cudaSuccess
             ? SMOE_OK
             : SMOE_ERR_LAUNCH;
}

static bool few_rows16(int64_t rows, int64_t E) { return rows <= Few16Smem::NT || rows <= 32 * E; }

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
  int split = 1;
  while (split < 8 && kb >= 12 && split * 6 <= kb && tiles * split * (split == 4 ? 4 : 2) <= sms) split *= 2;
  Few16Params p{(int)rows, (int)N, (int)K, (int)E, efo, counts, w_mn, (__nv_bfloat16*)y, split, status, host_word};
  int64_t groups = sms / split;
  if (tiles < groups) groups = tiles;
  return launch_early(gemm16_few_kernel, (unsigned)(groups * split), Few16Smem::THREADS, Few16Smem::TOTAL, (unsigned)split, stream, tw, tx16,
                      tx64, p) == cudaSuccess
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
  if (few_rows16(rows, E))
    return few16(x_bf16, ldx, w_bf16, efo, counts, y_bf16, rows, N, K, E, w_transposed != 0, status, pinned_host_word,
                 (cudaStream_t)stream);
  CUtensorMap ta, tb, tc;
  rc = make_tmap16(&ta, x_bf16, 1, rows, K, ldx, 128, 2);
  if (!rc) rc = w_transposed ? make_tmap16(&tb, w_bf16, E, K, N, N, 64, 3) : make_tmap16(&tb, w_bf16, E, N, K, K, 128, 3);
  if (!rc) rc = make_tmap16_out(&tc, y_bf16, true, 1, rows, N);
  if (rc) return rc;
  Gemm16Params p{};
  p.rows = (int)rows; p.N = (int)N; p.K = (int)K; p.E = (int)E;
  p.efo = efo; p.counts = counts; p.b_mn = w_transposed != 0; p.c = y_bf16;
  p.status = status; p.host_word = pinned_host_word;
  // every segment may end in a tile that is not full
  return launch16<ROWS16>(ta, tb, tc, p, (rows / 256 + E) * up16(N, 256), (cudaStream_t)stream);
}

int smoe_grouped_wgrad(const void* dy_bf16, int64_t ldy, const void* x_bf16, int64_t ldx, const int32_t* efo, const int32_t* counts,
                       void* dw, int64_t N, int64_t K, int64_t rows, int64_t E, int out_bf16, int accumulate, int32_t* status,
                       int32_t* pinned_host_word, void* stream) {
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
  CUtensorMap ta, tb, tc;
  rc = make_tmap16(&ta, dy_bf16, 1, rows, N, ldy, 64, 2);
  if (!rc) rc = make_tmap16(&tb, x_bf16, 1, rows, K, ldx, 64, 2);
  if (!rc) rc = make_tmap16_out(&tc, dw, out_bf16 != 0, E, N, K);
  if (rc) return rc;
  Gemm16Params p{};
  p.rows = (int)rows; p.M = (int)N; p.N = (int)K; p.E = (int)E;
  p.efo = efo; p.counts = counts; p.c = dw; p.out_bf16 = out_bf16 != 0; p.accumulate = accumulate != 0;
  p.status = status; p.host_word = pinned_host_word;
  return launch16<WGRAD16>(ta, tb, tc, p, E * up16(N, 256) * up16(K, 256), (cudaStream_t)stream);
}

}  // extern "C"
