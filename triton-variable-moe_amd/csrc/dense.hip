// Entry points of the dense operators: fused linear and gated block, forward and
// backward (include/vmoe.h). Each checks its arguments on the host, chooses the
// kernels and queues them on one stream.

#include <algorithm>

#include "dense_launch.h"

namespace vmoe {
namespace dense {
namespace {

constexpr int64_t kMaxLd = 1 << 20;    // elements: 256 rows of a tile stay below 2 GiB
constexpr int64_t kMaxRows = 1 << 22;

int esize(int type) { return type == VMOE_DENSE_F32 ? 4 : 2; }
int64_t unit(int type) { return type == VMOE_DENSE_F32 ? 4 : 8; }  // values of 16 bytes
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// A matrix the kernels read or write: rows of `cols` values, ld apart.
int check_rows(int type, const void* p, int64_t cols, int64_t ld) {
  if (!p || ld < cols) return VMOE_ERR_INVALID_ARG;
  if (!aligned(p) || ld % unit(type) || ld > kMaxLd) return VMOE_ERR_UNSUPPORTED;
  return VMOE_OK;
}

int check_sizes(int type, int act, int64_t rows, int64_t a, int64_t b) {
  if (type != VMOE_DENSE_BF16 && type != VMOE_DENSE_F32) return VMOE_ERR_INVALID_ARG;
  if (act < VMOE_DENSE_NONE || act > VMOE_DENSE_GELU_TANH) return VMOE_ERR_INVALID_ARG;
  if (rows < 0 || a <= 0 || b <= 0) return VMOE_ERR_INVALID_ARG;
  if (rows > kMaxRows || a % unit(type) || b % unit(type)) return VMOE_ERR_UNSUPPORTED;
  return VMOE_OK;
}

#define VMOE_TRY(expr)                    \
  do {                                    \
    const int st_ = (expr);               \
    if (st_ != VMOE_OK) return st_;       \
  } while (0)

// How a product runs: its tiles and the slices its k is cut into.
struct Plan {
  Tiles tiles;
  int splits;
  int64_t kper;
  size_t part_bytes;  // of the slices' sums
};

Plan plan_of(int type, Epi epi, int64_t M, int64_t N, int64_t K) {
  Plan q;
  const int64_t n = epi == EPI_GATED ? 2 * N : N;  // columns staged
  const int64_t stage = 128 / esize(type);
  auto count = [&](int64_t t, int64_t tn) { return cdiv(M, t) * cdiv(n, tn); };
  q.tiles = type == VMOE_DENSE_BF16 && count(256, 256) >= 224 ? TILES_256
            : count(128, 128) >= 256                          ? TILES_128
                                                              : TILES_64;
  const int64_t tiles = std::max<int64_t>(1, q.tiles == TILES_256   ? count(256, 256)
                                             : q.tiles == TILES_128 ? count(128, 128)
                                             : epi == EPI_GATED     ? count(64, 128)
                                                                    : count(64, 64));
  q.splits = 1;
  const int64_t stages = cdiv(K, stage);
  if (tiles < 256 && q.tiles != TILES_256)
    q.splits = (int)std::max<int64_t>(1, std::min(512 / tiles, stages / 8));
  q.kper = cdiv(stages, q.splits) * stage;
  q.splits = (int)cdiv(K, q.kper);
  q.part_bytes = q.splits > 1 ? align256((size_t)q.splits * M * n * 4) : 0;
  return q;
}

// One product with its epilogue. part: Plan::part_bytes. sums (EPI_GATED_BWD):
// the rows of column sums written to p.part, 0 where the slices were joined.
int product(int type, Form form, Epi epi, GemmArgs p, float* part, int64_t* sums, hipStream_t s) {
  const Plan q = plan_of(type, epi, p.M, p.N, p.K);
  p.splits = q.splits;
  p.kper = q.kper;
  if (sums) *sums = 0;
  if (q.splits > 1) {
    GemmArgs g = p;
    g.N = g.ldp = epi == EPI_GATED ? 2 * p.N : p.N;
    g.part = part;
    VMOE_TRY(gemm_tiles(type, form, EPI_PARTIAL, g, q.tiles, s));
    p.part = part;
    p.ldp = g.ldp;
    return join_splits(type, epi, p, s);
  }
  if (sums) *sums = cdiv(p.M, q.tiles == TILES_64 ? 32 : q.tiles == TILES_128 ? 64 : 128);
  return gemm_tiles(type, form, epi, p, q.tiles, s);
}

GemmArgs args(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t M, int64_t N,
              int64_t K, void* c, int64_t ldc) {
  GemmArgs p = {};
  p.a = a;
  p.lda = lda;
  p.b = b;
  p.ldb = ldb;
  p.M = M;
  p.N = N;
  p.K = K;
  p.c = c;
  p.ldc = ldc;
  return p;
}

// x w of a weight [in, out], or of one stored [out, in].
Form forward_form(int transposed) { return transposed ? FORM_KK : FORM_KT; }
Form input_grad_form(int transposed) { return transposed ? FORM_KT : FORM_KK; }

// The weight gradient x^T g in the weight's own order: [in, out] or [out, in].
GemmArgs weight_grad_args(int transposed, const void* x, int64_t ldx, int64_t in, const void* g,
                          int64_t ldg, int64_t out, int64_t rows, void* gw, int64_t ldgw) {
  return transposed ? args(g, ldg, x, ldx, out, in, rows, gw, ldgw)
                    : args(x, ldx, g, ldg, in, out, rows, gw, ldgw);
}
size_t weight_grad_bytes(int type, int64_t in, int64_t out, int64_t rows, int transposed) {
  return transposed ? plan_of(type, EPI_LINEAR, out, in, rows).part_bytes
                    : plan_of(type, EPI_LINEAR, in, out, rows).part_bytes;
}

// Workspace: the slices' sums of one product at a time, then each buffer.
struct Bytes {
  size_t part, grads, sums, total;
};
Bytes linear_bytes(int type, int64_t rows, int64_t in, int64_t out, int act, int backward) {
  Bytes b = {};
  if (!backward) {
    b.part = plan_of(type, EPI_LINEAR, rows, out, in).part_bytes;
  } else {
    b.part = std::max({plan_of(type, EPI_LINEAR, rows, in, out).part_bytes,
                       weight_grad_bytes(type, in, out, rows, 0),
                       weight_grad_bytes(type, in, out, rows, 1)});
    if (act != VMOE_DENSE_NONE) b.grads = align256((size_t)rows * out * esize(type));
    b.sums = align256((size_t)sum_rows(rows) * out * 4);
  }
  b.total = b.part + b.grads + b.sums;
  return b;
}
Bytes gated_bytes(int type, int64_t rows, int64_t d, int64_t width, int backward) {
  Bytes b = {};
  if (!backward) {
    b.part = std::max(plan_of(type, EPI_GATED, rows, width, d).part_bytes,
                      plan_of(type, EPI_LINEAR, rows, d, width).part_bytes);
  } else {
    b.part = std::max({plan_of(type, EPI_GATED_BWD, rows, width, d).part_bytes,
                       plan_of(type, EPI_LINEAR, rows, d, 2 * width).part_bytes,
                       weight_grad_bytes(type, d, 2 * width, rows, 0),
                       weight_grad_bytes(type, d, 2 * width, rows, 1),
                       weight_grad_bytes(type, width, d, rows, 0),
                       weight_grad_bytes(type, width, d, rows, 1)});
    b.grads = align256((size_t)rows * 2 * width * esize(type));
    b.sums = align256((size_t)std::max(std::max(sum_rows(rows), cdiv(rows, 32)) * 2 * width,
                                       sum_rows(rows) * d) * 4);
  }
  b.total = b.part + b.grads + b.sums;
  return b;
}

int check_workspace(const void* p, size_t have, size_t need) {
  if (have < need) return VMOE_ERR_WORKSPACE;
  if (need && !p) return VMOE_ERR_INVALID_ARG;
  return need && !aligned(p) ? VMOE_ERR_UNSUPPORTED : VMOE_OK;
}

// A weight [in, out] (transposed: stored [out, in]).
int check_weight(int type, const void* w, int64_t ldw, int transposed, int64_t in, int64_t out) {
  return check_rows(type, w, transposed ? in : out, ldw);
}

}  // namespace
}  // namespace dense
}  // namespace vmoe

using namespace vmoe;
using namespace vmoe::dense;

extern "C" size_t vmoe_linear_workspace_bytes(int32_t type, int64_t rows, int64_t in, int64_t out,
                                              int32_t act, int32_t backward) {
  if (check_sizes(type, act, rows, in, out) != VMOE_OK) return 0;
  return linear_bytes(type, rows, in, out, act, backward).total;
}

extern "C" int vmoe_linear_forward(int32_t type, const void* x, int64_t ldx, int64_t rows,
                                   int64_t in, int64_t out, const void* w, int64_t ldw,
                                   int32_t w_transposed, const void* bias, int32_t bias_f32,
                                   int32_t act, const void* residual, int64_t ldr, void* y,
                                   int64_t ldy, float* z, void* workspace, size_t workspace_bytes,
                                   vmoe_stream_t stream) {
  VMOE_TRY(check_sizes(type, act, rows, in, out));
  if (rows == 0) return VMOE_OK;
  VMOE_TRY(check_rows(type, x, in, ldx));
  VMOE_TRY(check_weight(type, w, ldw, w_transposed, in, out));
  VMOE_TRY(check_rows(type, y, out, ldy));
  if (residual) VMOE_TRY(check_rows(type, residual, out, ldr));
  if (z && !aligned(z)) return VMOE_ERR_UNSUPPORTED;
  VMOE_TRY(check_workspace(workspace, workspace_bytes,
                           linear_bytes(type, rows, in, out, act, 0).total));
  GemmArgs p = args(x, ldx, w, ldw, rows, out, in, y, ldy);
  p.bias = bias;
  p.bias_f32 = bias_f32;
  p.act = act;
  p.res = residual;
  p.ldr = ldr;
  p.z = z;
  p.ldz = out;
  return product(type, forward_form(w_transposed), EPI_LINEAR, p, static_cast<float*>(workspace),
                 nullptr, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int vmoe_linear_backward(int32_t type, const void* gy, int64_t ldgy, const void* x,
                                    int64_t ldx, int64_t rows, int64_t in, int64_t out,
                                    const void* w, int64_t ldw, int32_t w_transposed,
                                    int32_t act, const float* z, void* gx, int64_t ldgx, void* gw,
                                    int64_t ldgw, void* gb, int32_t gb_f32, void* workspace,
                                    size_t workspace_bytes, vmoe_stream_t stream) {
  VMOE_TRY(check_sizes(type, act, rows, in, out));
  if (rows == 0) return VMOE_OK;
  VMOE_TRY(check_rows(type, gy, out, ldgy));
  if (gw) VMOE_TRY(check_rows(type, x, in, ldx));
  if (gx) VMOE_TRY(check_weight(type, w, ldw, w_transposed, in, out));
  if (gx) VMOE_TRY(check_rows(type, gx, in, ldgx));
  if (gw) VMOE_TRY(check_weight(type, gw, ldgw, w_transposed, in, out));
  if (act != VMOE_DENSE_NONE && !z) return VMOE_ERR_INVALID_ARG;
  if (z && !aligned(z)) return VMOE_ERR_UNSUPPORTED;
  const Bytes b = linear_bytes(type, rows, in, out, act, 1);
  VMOE_TRY(check_workspace(workspace, workspace_bytes, b.total));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  float* part = reinterpret_cast<float*>(ws);
  void* dz = ws + b.part;
  float* sums = reinterpret_cast<float*>(ws + b.part + b.grads);
  const bool has_act = act != VMOE_DENSE_NONE;
  if (has_act || gb) {
    VMOE_TRY(act_grad(type, gy, ldgy, has_act ? z : nullptr, out, act, dz, out,
                      gb ? sums : nullptr, rows, out, s));
    if (gb) VMOE_TRY(col_sum(sums, sum_rows(rows), out, out, gb, gb_f32, nullptr, 0, s));
  }
  const void* g = has_act ? dz : gy;
  const int64_t ldg = has_act ? out : ldgy;
  if (gx)
    VMOE_TRY(product(type, input_grad_form(w_transposed), EPI_LINEAR,
                     args(g, ldg, w, ldw, rows, in, out, gx, ldgx), part, nullptr, s));
  if (gw)
    VMOE_TRY(product(type, FORM_TT, EPI_LINEAR,
                     weight_grad_args(w_transposed, x, ldx, in, g, ldg, out, rows, gw, ldgw), part,
                     nullptr, s));
  return VMOE_OK;
}

extern "C" size_t vmoe_gated_workspace_bytes(int32_t type, int64_t rows, int64_t hidden,
                                             int64_t width, int32_t backward) {
  if (check_sizes(type, VMOE_DENSE_NONE, rows, hidden, width) != VMOE_OK) return 0;
  return gated_bytes(type, rows, hidden, width, backward).total;
}

namespace {
// (the up columns of a weight stored [2 width, hidden] are addressed from the
// gate's by a 32-bit offset)
int check_gated_weights(int type, const void* w1, int64_t ldw1, int t1, const void* w2,
                        int64_t ldw2, int t2, int64_t d, int64_t width) {
  VMOE_TRY(check_weight(type, w1, ldw1, t1, d, 2 * width));
  VMOE_TRY(check_weight(type, w2, ldw2, t2, width, d));
  if (t1 && (width + 256) * ldw1 * esize(type) >= (int64_t)1 << 31) return VMOE_ERR_UNSUPPORTED;
  return VMOE_OK;
}
}  // namespace

extern "C" int vmoe_gated_forward(int32_t type, const void* x, int64_t ldx, int64_t rows,
                                  int64_t hidden, int64_t width, const void* w1, int64_t ldw1,
                                  int32_t w1_transposed, const void* bias1, int32_t bias1_f32,
                                  int32_t act, const void* w2, int64_t ldw2,
                                  int32_t w2_transposed, const void* bias2, int32_t bias2_f32,
                                  const void* residual, int64_t ldr, void* h, float* z, void* y,
                                  int64_t ldy, void* workspace, size_t workspace_bytes,
                                  vmoe_stream_t stream) {
  VMOE_TRY(check_sizes(type, act, rows, hidden, width));
  if (rows == 0) return VMOE_OK;
  VMOE_TRY(check_rows(type, x, hidden, ldx));
  VMOE_TRY(check_gated_weights(type, w1, ldw1, w1_transposed, w2, ldw2, w2_transposed, hidden,
                               width));
  VMOE_TRY(check_rows(type, h, width, width));
  VMOE_TRY(check_rows(type, y, hidden, ldy));
  if (residual) VMOE_TRY(check_rows(type, residual, hidden, ldr));
  if (z && !aligned(z)) return VMOE_ERR_UNSUPPORTED;
  VMOE_TRY(check_workspace(workspace, workspace_bytes,
                           gated_bytes(type, rows, hidden, width, 0).total));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  float* part = static_cast<float*>(workspace);
  GemmArgs p = args(x, ldx, w1, ldw1, rows, width, hidden, h, width);
  p.bias = bias1;
  p.bias_f32 = bias1_f32;
  p.act = act;
  p.z = z;
  p.ldz = 2 * width;
  VMOE_TRY(product(type, forward_form(w1_transposed), EPI_GATED, p, part, nullptr, s));
  GemmArgs q = args(h, width, w2, ldw2, rows, hidden, width, y, ldy);
  q.bias = bias2;
  q.bias_f32 = bias2_f32;
  q.act = VMOE_DENSE_NONE;
  q.res = residual;
  q.ldr = ldr;
  return product(type, forward_form(w2_transposed), EPI_LINEAR, q, part, nullptr, s);
}

extern "C" int vmoe_gated_backward(int32_t type, const void* gy, int64_t ldgy, const void* x,
                                   int64_t ldx, int64_t rows, int64_t hidden, int64_t width,
                                   const void* w1, int64_t ldw1, int32_t w1_transposed,
                                   const void* w2, int64_t ldw2, int32_t w2_transposed,
                                   int32_t act, const void* h, const float* z, void* gx,
                                   int64_t ldgx, void* gw1, int64_t ldgw1, void* gb1,
                                   int32_t gb1_f32, void* gw2, int64_t ldgw2, void* gb2,
                                   int32_t gb2_f32, void* workspace, size_t workspace_bytes,
                                   vmoe_stream_t stream) {
  VMOE_TRY(check_sizes(type, act, rows, hidden, width));
  if (rows == 0) return VMOE_OK;
  VMOE_TRY(check_rows(type, gy, hidden, ldgy));
  VMOE_TRY(check_gated_weights(type, w1, ldw1, w1_transposed, w2, ldw2, w2_transposed, hidden,
                               width));
  const bool inner = gx || gw1 || gb1;  // what needs the gradient of [gate | up]
  if (inner && !z) return VMOE_ERR_INVALID_ARG;
  if (z && !aligned(z)) return VMOE_ERR_UNSUPPORTED;
  if (gw1) VMOE_TRY(check_rows(type, x, hidden, ldx));
  if (gw2) VMOE_TRY(check_rows(type, h, width, width));
  if (gx) VMOE_TRY(check_rows(type, gx, hidden, ldgx));
  if (gw1) VMOE_TRY(check_weight(type, gw1, ldgw1, w1_transposed, hidden, 2 * width));
  if (gw2) VMOE_TRY(check_weight(type, gw2, ldgw2, w2_transposed, width, hidden));
  const Bytes b = gated_bytes(type, rows, hidden, width, 1);
  VMOE_TRY(check_workspace(workspace, workspace_bytes, b.total));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  float* part = reinterpret_cast<float*>(ws);
  void* dz = ws + b.part;
  float* sums = reinterpret_cast<float*>(ws + b.part + b.grads);
  const int64_t w2x = 2 * width;
  if (inner) {
    GemmArgs p = args(gy, ldgy, w2, ldw2, rows, width, hidden, dz, w2x);
    p.act = act;
    p.z = const_cast<float*>(z);
    p.ldz = w2x;
    p.part = gb1 ? sums : nullptr;
    p.ldp = w2x;
    int64_t n = 0;
    VMOE_TRY(product(type, input_grad_form(w2_transposed), EPI_GATED_BWD, p, part, &n, s));
    if (gb1 && n == 0) {  // joined slices: sums of the rounded gradients
      VMOE_TRY(act_grad(type, dz, w2x, nullptr, 0, VMOE_DENSE_NONE, nullptr, 0, sums, rows, w2x, s));
      n = sum_rows(rows);
    }
    if (gb1) VMOE_TRY(col_sum(sums, n, w2x, w2x, gb1, gb1_f32, nullptr, 0, s));
  }
  if (gb2) {
    VMOE_TRY(act_grad(type, gy, ldgy, nullptr, 0, VMOE_DENSE_NONE, nullptr, 0, sums, rows, hidden,
                      s));
    VMOE_TRY(col_sum(sums, sum_rows(rows), hidden, hidden, gb2, gb2_f32, nullptr,
                     0, s));
  }
  if (gw2)
    VMOE_TRY(product(type, FORM_TT, EPI_LINEAR,
                     weight_grad_args(w2_transposed, h, width, width, gy, ldgy, hidden, rows, gw2,
                                      ldgw2), part, nullptr, s));
  if (gx)
    VMOE_TRY(product(type, input_grad_form(w1_transposed), EPI_LINEAR,
                     args(dz, w2x, w1, ldw1, rows, hidden, w2x, gx, ldgx), part, nullptr, s));
  if (gw1)
    VMOE_TRY(product(type, FORM_TT, EPI_LINEAR,
                     weight_grad_args(w1_transposed, x, ldx, hidden, dz, w2x, w2x, rows, gw1,
                                      ldgw1), part, nullptr, s));
  return VMOE_OK;
}
