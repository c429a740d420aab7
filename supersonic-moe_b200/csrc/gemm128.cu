// Host side of the products with a scale per block of 128.
#include "gemm128.cuh"
#include "gemm128_few.cuh"
#include "host.h"
#include "smoe_b200.h"
#include "smoe_internal.h"

namespace smoe {

// [depth, rows, cols] bytes, rows a multiple of 16 bytes apart, box {128, box_rows, 1} in the 128-byte swizzle; what lies beyond an
// extent reads as zero
static int make_tmap128(CUtensorMap* m, const void* base, uint64_t depth, uint64_t rows, uint64_t cols, uint32_t box_rows, int dims) {
  if (!load_encode()) return SMOE_ERR_DRIVER;
  if (reinterpret_cast<uintptr_t>(base) & 15) return SMOE_ERR_ALIGN;
  const cuuint64_t pitch = (cols + 15) & ~(uint64_t)15;
  cuuint64_t extent[3] = {cols, rows, depth};
  cuuint64_t strides[2] = {pitch, pitch * rows};
  cuuint32_t box[3] = {128, box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = g_encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, dims, const_cast<void*>(base), extent, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? SMOE_OK : SMOE_ERR_TMAP;
}

// The result [depth, rows, cols], box of 32 rows of 128 bytes
static int make_tmap128_out(CUtensorMap* m, void* base, bool bf16, uint64_t depth, uint64_t rows, uint64_t cols) {
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

template <int MODE>
static int launch128(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const Gemm128Params& p, int64_t tiles,
                     bool early, cudaStream_t stream) {
  static bool attr_set[kMaxDevices] = {};
  auto kern = gemm128_kernel<MODE>;
  if (!ensure_smem_attr(kern, Gemm128Smem::TOTAL, attr_set)) return SMOE_ERR_LAUNCH;
  int64_t pairs = sm_count() / 2;
  if (tiles < pairs) pairs = tiles;
  if (pairs <= 0) return SMOE_OK;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(2 * pairs));
  cfg.blockDim = dim3(Gemm128Smem::THREADS);
  cfg.dynamicSmemBytes = Gemm128Smem::TOTAL;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = early ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kern, ta, tb, tc, p) != cudaSuccess) return SMOE_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? SMOE_OK : SMOE_ERR_LAUNCH;
}

static bool size128(int64_t n) { return n > 0 && n % 8 == 0 && n < (int64_t)1 << 24; }

static int check128(const void* a, const float* a_s, const void* b, const float* b_s, const int* efo, const int* counts, const void* c,
                    int64_t rows, int64_t N, int64_t K, int64_t E, const int* status, bool bulk_scales) {
  if (rows < 0 || rows >= (int64_t)1 << 31 || !size128(N) || !size128(K) || E <= 0 || E > kMaxExperts2) return SMOE_ERR_SHAPE;
  if (!efo && (E != 1 || counts)) return SMOE_ERR_ARG;
  if (!status || (rows > 0 && (!a || !a_s || !b || !b_s || !c))) return SMOE_ERR_ARG;
  if (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15) return SMOE_ERR_ALIGN;
  // the weight gradient copies scales in bulk; the products by rows read them one by one, from wherever an expert's begin
  if (((uintptr_t)a_s | (uintptr_t)b_s) & (bulk_scales ? 15 : 3)) return SMOE_ERR_ALIGN;
  return SMOE_OK;
}

static int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m; }

int gemm128_rows(const void* a_fp8, const float* a_scales, const void* b_fp8, const float* b_scales, const int* efo, const int* counts,
                 void* c_bf16, int64_t rows, int64_t N, int64_t K, int64_t E, int b_mn, int zero_rest, bool without_rests, int* status,
                 int* pinned_host_word, bool early, void* stream) {
  int rc = check128(a_fp8, a_scales, b_fp8, b_scales, efo, counts, c_bf16, rows, N, K, E, status, false);
  if (rc || rows == 0) return rc;
  CUtensorMap ta, tb, tc;
  rc = make_tmap128(&ta, a_fp8, 1, rows, K, 128, 2);
  if (!rc) rc = make_tmap128_out(&tc, c_bf16, true, 1, rows, N);
  if (!rc) rc = b_mn ? make_tmap128(&tb, b_fp8, E, K, N, 128, 3) : make_tmap128(&tb, b_fp8, E, N, K, 128, 3);
  if (rc) return rc;
  Gemm128Params p{};
  p.rows = (int)rows; p.N = (int)N; p.K = (int)K; p.E = (int)E;
  p.efo = efo; p.counts = counts; p.a_s = a_scales; p.b_s = b_scales;
  const int64_t nb = up(N, 128), kb = up(K, 128);
  p.a_kb = (int)kb;
  p.bs_e = nb * kb;
  p.bs_n = b_mn ? 1 : kb;
  p.bs_k = b_mn ? (int)nb : 1;
  p.b_mn = b_mn != 0; p.c = c_bf16; p.zero_rest = without_rests ? -Few128Smem::NT : zero_rest != 0;
  p.status = status; p.host_word = pinned_host_word;
  // every segment may end in a tile that is not full, and so may the rows behind the last
  const int64_t tiles = efo ? (rows / 256 + E + 1) * up(N, 256) : up(rows, 256) * up(N, 256);
  return launch128<ROWS128>(ta, tb, tc, p, tiles, early, (cudaStream_t)stream);
}

int gemm128_wgrad(const void* a_fp8, const float* a_scales, const void* b_fp8, const float* b_scales, const int* efo, const int* counts,
                  void* c, int64_t M, int64_t N, int64_t rows, int64_t E, int out_bf16, int accumulate, int* status,
                  int* pinned_host_word, bool independent, void* stream) {
  int rc = check128(a_fp8, a_scales, b_fp8, b_scales, efo, counts, c, rows, N, M, E, status, true);
  if (rc) return rc;
  if (out_bf16 && accumulate) return SMOE_ERR_ARG;
  if (rows == 0) {                                  // an empty sum
    if (accumulate) return SMOE_OK;
    if (!c) return SMOE_ERR_ARG;
    return cudaMemsetAsync(c, 0, (size_t)(E * M * N) * (out_bf16 ? 2 : 4), (cudaStream_t)stream) == cudaSuccess ? SMOE_OK
                                                                                                             : SMOE_ERR_LAUNCH;
  }
  CUtensorMap ta, tb, tc;
  rc = make_tmap128(&ta, a_fp8, 1, M, rows, 128, 2);
  if (!rc) rc = make_tmap128_out(&tc, c, out_bf16, E, M, N);
  if (!rc) rc = make_tmap128(&tb, b_fp8, 1, N, rows, 128, 3);
  if (rc) return rc;
  Gemm128Params p{};
  p.rows = (int)rows; p.M = (int)M; p.N = (int)N; p.E = (int)E;
  p.efo = efo; p.counts = counts; p.a_s = a_scales; p.b_s = b_scales;
  p.c = c; p.out_bf16 = out_bf16 != 0; p.accumulate = accumulate != 0; p.status = status;
  p.host_word = pinned_host_word; p.independent = independent;
  return launch128<WGRAD128>(ta, tb, tc, p, E * up(M, 256) * up(N, 256), independent, (cudaStream_t)stream);
}

int gemm128_few(const void* a_fp8, const float* a_scales, const void* b_fp8, const float* b_scales, const int* efo, const int* counts,
                void* c_bf16, int64_t rows, int64_t N, int64_t K, int64_t E, int64_t live_rows, bool rests, int* status,
                int* pinned_host_word, bool early, bool independent, void* stream) {
  int rc = check128(a_fp8, a_scales, b_fp8, b_scales, efo, counts, c_bf16, rows, N, K, E, status, false);
  if (rc || rows == 0) return rc;
  if (live_rows <= 0 || live_rows > rows) live_rows = rows;
  CUtensorMap tw, tx16, tx64;
  rc = make_tmap128(&tw, b_fp8, E, N, K, 128, 3);
  if (!rc) rc = make_tmap128(&tx16, a_fp8, 1, rows, K, 16, 2);
  if (!rc) rc = make_tmap128(&tx64, a_fp8, 1, rows, K, Few128Smem::NT, 2);
  if (rc) return rc;
  static bool attr_set[kMaxDevices] = {};
  if (!ensure_smem_attr(gemm128_few_kernel, Few128Smem::TOTAL, attr_set)) return SMOE_ERR_LAUNCH;
  const int sms = sm_count();
  const int64_t nw = up(N, 128), busy = live_rows < E ? live_rows : E;
  const int64_t tiles = (rests ? busy : (live_rows + (Few128Smem::NT - 1) * busy) / Few128Smem::NT) * nw;      // as many as there can be
  // Few tiles are shared by clusters while each CTA keeps three blocks of a reduction of twelve or more (us at 16 rows with 1 / 2 / 4
  // CTAs: 4096 x 4096 15.0 / 12.3 / 11.2, 2048 x 1536 8.2 / 8.4 / 7.7, 8192 x 2048 10.6 / 10.6 / -; 1024 x 1024 7.0 / 7.8 / 7.4,
  // 2048 x 768 6.4 / 7.5 / 7.3).  Eight find room together on half of the SMs only, as they come from one part of the chip (with 8
  // instead of 4: 1024 x 16384 16.4 -> 13.7, 2048 x 8192, on 128 SMs, 12.5 -> 21.1).
  const int64_t kb = up(K, 128);
  int split = 1;
  while (split < 8 && kb >= 12 && split * 6 <= kb && tiles * split * (split == 4 ? 4 : 2) <= sms) split *= 2;
  Few128Params p{(int)rows, (int)N, (int)K, (int)E, efo, counts, b_scales, a_scales, (__nv_bfloat16*)c_bf16, split, rests ? 256 : 0,
                 independent, status, pinned_host_word};
  int64_t groups = sms / split;
  if (tiles < groups) groups = tiles;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(groups * split));
  cfg.blockDim = dim3(Few128Smem::THREADS);
  cfg.dynamicSmemBytes = Few128Smem::TOTAL;
  cfg.stream = (cudaStream_t)stream;
  cfg.attrs = attr;
  cfg.numAttrs = early || independent ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, gemm128_few_kernel, tw, tx16, tx64, p) != cudaSuccess) return SMOE_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? SMOE_OK : SMOE_ERR_LAUNCH;
}

}  // namespace smoe

using namespace smoe;

static bool on16(const void* p, const void* q) { return (((uintptr_t)p | (uintptr_t)q) & 15) == 0; }

extern "C" {

// (by themselves, the products ask the same of all their operands)
int smoe_gemm128_rows(const void* a_fp8, const float* a_scales, const void* b_fp8, const float* b_scales, const int32_t* efo,
                      const int32_t* counts, void* c_bf16, int64_t rows, int64_t N, int64_t K, int64_t E, int b_mn,
                      int zero_rest, int32_t* status, int32_t* pinned_host_word, void* stream) {
  if (!on16(a_scales, b_scales)) return SMOE_ERR_ALIGN;
  return gemm128_rows(a_fp8, a_scales, b_fp8, b_scales, efo, counts, c_bf16, rows, N, K, E, b_mn, zero_rest, false, status,
                      pinned_host_word, false, stream);
}

int smoe_gemm128_wgrad(const void* a_fp8, const float* a_scales, const void* b_fp8, const float* b_scales, const int32_t* efo,
                       const int32_t* counts, void* c, int64_t M, int64_t N, int64_t rows, int64_t E, int out_bf16, int accumulate,
                       int32_t* status, int32_t* pinned_host_word, void* stream) {
  return gemm128_wgrad(a_fp8, a_scales, b_fp8, b_scales, efo, counts, c, M, N, rows, E, out_bf16, accumulate, status, pinned_host_word,
                       false, stream);
}

int smoe_gemm128_few(const void* a_fp8, const float* a_scales, const void* b_fp8, const float* b_scales, const int32_t* efo,
                     const int32_t* counts, void* c_bf16, int64_t rows, int64_t N, int64_t K, int64_t E, int64_t live_rows,
                     int32_t* status, int32_t* pinned_host_word, void* stream) {
  if (!on16(a_scales, b_scales)) return SMOE_ERR_ALIGN;
  return gemm128_few(a_fp8, a_scales, b_fp8, b_scales, efo, counts, c_bf16, rows, N, K, E, live_rows, false, status, pinned_host_word,
                     false, false, stream);
}

}  // extern "C"
