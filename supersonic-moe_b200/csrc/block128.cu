// One call for what a caller would otherwise issue kernel by kernel: a projection with a scale per block of 128, its gradients,
// and routed SwiGLU experts.  The kernels of small problems end before a caller has issued them one by one.
#include <cuda_runtime.h>

#include "host.h"
#include "smoe_b200.h"
#include "smoe_internal.h"

namespace smoe {

// Parts of an arena, each on a 256-byte boundary; with a null base it only counts
struct Arena128 {
  uint8_t* base;
  int64_t used = 0;
  explicit Arena128(void* b) : base((uint8_t*)b) {}
  void* take(int64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += (bytes + 255) & ~(int64_t)255;
    return p;
  }
  float* floats(int64_t n) { return (float*)take(4 * n); }
  int32_t* ints(int64_t n) { return (int32_t*)take(4 * n); }
};
static int64_t pitch128(int64_t n) { return (n + 15) & ~(int64_t)15; }
static int64_t blocks128(int64_t n) { return (n + 127) / 128; }

struct Saved128 {             // of a forward pass: the weight's payload, if the call made it, and x by columns
  void *wq = nullptr, *xc = nullptr;
  float *ws = nullptr, *xcs = nullptr;
  int64_t bytes;
  Saved128(int64_t rows, int64_t N, int64_t K, int64_t E, int flags, void* base) {
    Arena128 m(base);
    if (flags & SMOE_B128_QUANT_W) {
      wq = m.take(E * N * pitch128(K));
      ws = m.floats(E * blocks128(N) * blocks128(K));
    }
    if (flags & SMOE_B128_DW) {
      xc = m.take(K * pitch128(rows));
      xcs = m.floats(blocks128(rows) * K);
    }
    bytes = m.used;
  }
};
struct Forward128 {           // x by rows
  void* xq;
  float* xs;
  int64_t bytes;
  Forward128(int64_t rows, int64_t K, void* base) {
    Arena128 m(base);
    xq = m.take(rows * pitch128(K));
    xs = m.floats(rows * blocks128(K));
    bytes = m.used;
  }
};
struct Backward128 {          // dy in the forms that the gradients asked for read
  void *dq = nullptr, *dc = nullptr;
  float *ds = nullptr, *dcs = nullptr;
  int64_t bytes;
  Backward128(int64_t rows, int64_t N, int flags, void* base) {
    Arena128 m(base);
    if (flags & SMOE_B128_DX) {
      dq = m.take(rows * pitch128(N));
      ds = m.floats(rows * blocks128(N));
    }
    if (flags & SMOE_B128_DW) {
      dc = m.take(N * pitch128(rows));
      dcs = m.floats(blocks128(rows) * N);
    }
    bytes = m.used;
  }
};

struct Experts128 {           // everything between the tokens and their sums
  int64_t rows, slots;
  int32_t *efo, *x_gather, *s_scatter, *s_rev, *naept, *src_idx, *counts;
  float* scores;
  void *ws, *xq, *z, *yq, *o;
  float *xs, *ys;
  int64_t bytes;
  Experts128(int64_t T, int64_t H, int64_t I, int64_t E, int64_t K, void* base) {
    Arena128 m(base);
    slots = T * K;
    rows = blocks128(slots) * 128 + E * 128;
    efo = m.ints(E + 1);
    x_gather = m.ints(rows);
    s_scatter = m.ints(rows);
    s_rev = m.ints(slots);
    naept = m.ints(T + 1);
    src_idx = m.ints(slots);
    counts = m.ints(E);
    scores = m.floats(rows);
    ws = m.take(smoe_topk_metadata_workspace(T, E));
    xq = m.take(rows * pitch128(H));
    xs = m.floats(rows * blocks128(H));
    z = m.take(rows * 2 * I * 2);
    yq = m.take(rows * pitch128(I));
    ys = m.floats(rows * blocks128(I));
    o = m.take(rows * H * 2);
    bytes = m.used;
  }
};

static bool sizes128(int64_t rows, int64_t N, int64_t K, int64_t E) {
  return rows >= 0 && rows < (int64_t)1 << 31 && N > 0 && N % 8 == 0 && N < (int64_t)1 << 24 && K > 0 && K % 8 == 0 &&
         K < (int64_t)1 << 24 && E > 0 && E <= 256;
}

// The weights are the wide operand of a product of so few rows that they make one tile
constexpr int64_t kFewRows = 64;
// One projection: also where tiles of 128 weight rows x 64 leave half of the SMs or more, which then share the tiles' reductions (us
// with / without, at 64, 128 and 256 rows: 4096 x 4096 13.5 / 19.5, 17.6 / 20.5, 21.3 / 20.5; 1024 x 4096 10 / 19, 12 / 19, 12.5 / 19;
// 2048 x 8192 16 / 33, 17 / 34, 24 / 34, at 384 35.0 / 34.0; 8192 x 2048 13.8 / 13.4, 14.2 / 14.2, 20.5 / 14.2; 16384 x 4096 at 16, 64
// and 128: 17 / 22, 22 / 22, 36 / 23).
static bool few_rows128(int64_t rows, int64_t N) {
  return rows <= kFewRows || (rows + kFewRows - 1) / kFewRows * blocks128(N) * 2 <= sm_count();
}
// Of routed experts: where an expert's rows, evenly routed, are 32 or fewer, or none can have more than one tile of them, reading the
// weights bounds the products, and all of them are of few rows.  Elsewhere tiles of 256 rows, and for the rest of an expert, if that
// is 64 rows or fewer, the product for few rows.  (us of a call, all of few rows / tiles and rests, 128 experts of 2048 x 768: 16
// rows an expert 133 / 142, 32 143 / 152, 64 208 / 194, 128 319 / 237; very unevenly routed, most rows at a few experts, 85 / 83,
// 115 / 103, 184 / 141; 8 of 4096 x 2048: 63 / 70, 67 / 73, 92 / 87, 134 / 89, unevenly 55 / 64, 71 / 86, 83 / 79.  4096 tokens x 8
// over the 128, tiles alone 329, with rests 333; unevenly 453 and 403.)
static bool few_experts128(int64_t T, int64_t E, int64_t K) { return T <= kFewRows || T * K <= 32 * E; }

#define SMOE_TRY(call)          \
  do {                          \
    const int rc_ = (call);     \
    if (rc_) return rc_;        \
  } while (0)

}  // namespace smoe

using namespace smoe;

extern "C" {

int64_t smoe_block128_bytes(int64_t rows, int64_t N, int64_t K, int64_t E, int flags, int which) {
  if (!sizes128(rows, N, K, E)) return -1;
  return which == 0   ? Saved128(rows, N, K, E, flags, nullptr).bytes
         : which == 1 ? Forward128(rows, K, nullptr).bytes
                      : Backward128(rows, N, flags, nullptr).bytes;
}

int smoe_block128_linear(const void* x_bf16, const void* w, const float* w_scales, const int32_t* efo, const int32_t* counts,
                         void* y_bf16, void* saved, void* scratch, int64_t rows, int64_t N, int64_t K, int64_t E, int flags,
                         int32_t* status, int32_t* pinned_host_word, void* stream) {
  if (!sizes128(rows, N, K, E)) return SMOE_ERR_SHAPE;
  const Saved128 sv(rows, N, K, E, flags, saved);
  const Forward128 f(rows, K, scratch);
  if ((sv.bytes && !saved) || (rows > 0 && !scratch)) return SMOE_ERR_ARG;
  if (flags & SMOE_B128_QUANT_W) {
    SMOE_TRY(smoe_quant128_weight(w, E, N, K, sv.wq, sv.ws, stream));
    w = sv.wq;
    w_scales = sv.ws;
  }
  if (flags & SMOE_B128_DW) SMOE_TRY(smoe_quant128_dual(x_bf16, rows, K, efo, counts, E, f.xq, f.xs, sv.xc, sv.xcs, stream));
  else SMOE_TRY(smoe_quant128_rows(x_bf16, rows, K, 0, nullptr, nullptr, 0, f.xq, f.xs, stream));
  // (segments and weights were complete when the quantiser ahead of the product began)
  if (!efo && few_rows128(rows, N))
    return gemm128_few(f.xq, f.xs, w, w_scales, efo, counts, y_bf16, rows, N, K, E, 0, false, status, pinned_host_word, true, false,
                       stream);
  return gemm128_rows(f.xq, f.xs, w, w_scales, efo, counts, y_bf16, rows, N, K, E, 0, 1, false, status, pinned_host_word, true, stream);
}

int smoe_block128_linear_bwd(const void* dy_bf16, const void* w_fp8, const float* w_scales, const int32_t* efo,
                             const int32_t* counts, const void* saved, void* scratch, void* dx_bf16, void* dw, int64_t rows,
                             int64_t N, int64_t K, int64_t E, int flags, int dw_f32_accumulate, int32_t* status,
                             int32_t* pinned_host_word, void* stream) {
  if (!sizes128(rows, N, K, E)) return SMOE_ERR_SHAPE;
  const Saved128 sv(rows, N, K, E, flags, const_cast<void*>(saved));
  const Backward128 b(rows, N, flags, scratch);
  if ((sv.bytes && !saved) || (rows > 0 && b.bytes && !scratch)) return SMOE_ERR_ARG;
  if (flags & SMOE_B128_QUANT_W) {
    w_fp8 = sv.wq;
    w_scales = sv.ws;
  }
  if (flags & SMOE_B128_DW) SMOE_TRY(smoe_quant128_dual(dy_bf16, rows, N, efo, counts, E, b.dq, b.ds, b.dc, b.dcs, stream));
  else if (flags & SMOE_B128_DX) SMOE_TRY(smoe_quant128_rows(dy_bf16, rows, N, 0, nullptr, nullptr, 0, b.dq, b.ds, stream));
  if (flags & SMOE_B128_DX)
    SMOE_TRY(gemm128_rows(b.dq, b.ds, w_fp8, w_scales, efo, counts, dx_bf16, rows, K, N, E, 1, 1, false, status, pinned_host_word, true,
                          stream));
  if (flags & SMOE_B128_DW)
    SMOE_TRY(gemm128_wgrad(b.dc, b.dcs, sv.xc, sv.xcs, efo, counts, dw, N, K, rows, E, !dw_f32_accumulate, dw_f32_accumulate, status,
                           pinned_host_word, (flags & SMOE_B128_DX) && rows > 0, stream));      // its operands were complete before dx began
  return SMOE_OK;
}

int64_t smoe_block128_experts_bytes(int64_t T, int64_t H, int64_t I, int64_t E, int64_t K) {
  if (T < 0 || K <= 0 || K > 16 || T * K >= (int64_t)1 << 30 || !sizes128(T, H, I, E)) return -1;
  return Experts128(T, H, I, E, K, nullptr).bytes;
}

int smoe_block128_experts(const void* x_bf16, const int32_t* idx, const float* scores, const void* w1_fp8, const float* w1_scales,
                          const void* w2_fp8, const float* w2_scales, void* out_bf16, void* scratch, int64_t T, int64_t H,
                          int64_t I, int64_t E, int64_t K, int32_t* status, int32_t* pinned_host_word, void* stream) {
  if (smoe_block128_experts_bytes(T, H, I, E, K) < 0) return SMOE_ERR_SHAPE;
  if (T == 0) return SMOE_OK;
  if (!x_bf16 || !idx || !scores || !out_bf16 || !scratch) return SMOE_ERR_ARG;
  const Experts128 s(T, H, I, E, K, scratch);
  // (a token's places in the order of its slots: one for each, also where two name one expert)
  SMOE_TRY(smoe_topk_metadata(idx, scores, T, K, E, 128, s.slots, s.rows, 1, 0, s.efo, s.x_gather, s.s_scatter, s.s_rev, s.naept,
                              s.scores, s.src_idx, s.counts, s.ws, stream));
  const bool few = few_experts128(T, E, K);
  auto product = [&](const void* a, const float* as, const void* w, const float* ws, void* c, int64_t N, int64_t Kr) {
    // (offsets and counts were complete when the quantiser ahead of the product began)
    if (few)
      return gemm128_few(a, as, w, ws, s.efo, s.counts, c, s.rows, N, Kr, E, s.slots, false, status, pinned_host_word, true, false, stream);
    const int rc = gemm128_rows(a, as, w, ws, s.efo, s.counts, c, s.rows, N, Kr, E, 0, 0, true, status, pinned_host_word, true, stream);
    // What is left of an expert after tiles of 256 rows, beside the last of those: its operands were complete when they began
    return rc ? rc
              : gemm128_few(a, as, w, ws, s.efo, s.counts, c, s.rows, N, Kr, E, s.slots, true, status, pinned_host_word, false, true,
                            stream);
  };
  SMOE_TRY(quant128_rows_scatter(x_bf16, T, H, s.naept, s.s_rev, s.rows, s.xq, s.xs, true, stream));
  SMOE_TRY(product(s.xq, s.xs, w1_fp8, w1_scales, s.z, 2 * I, H));
  SMOE_TRY(quant128_rows(s.z, s.rows, I, 1, s.s_rev, s.naept + T, s.slots, s.yq, s.ys, true, stream));
  SMOE_TRY(product(s.yq, s.ys, w2_fp8, w2_scales, s.o, H, I));
  return smoe_combine(s.o, s.s_rev, s.naept, s.scores, out_bf16, T, H, stream);
}

}  // extern "C"
