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

// How a product runs.
struct Plan {
  Tiles tiles;
  int tiles_m, tiles_n, whole, splits;  // see GemmArgs
  int64_t kper;
  size_t part_bytes;  // of the slices' sums
};

// A kernel of tiles: its size, the workgroups a CU holds, the microseconds a stage of k
// takes each of them where a CU holds 1, 2, ..., and those that a round of workgroups
// takes besides (first loads, epilogue). Measured at 16 and 80 stages, where operands
// stay in the last-level cache bf16 tiles of 256 run 1360 TFLOP/s, of 128 1150, of 64
// 650, fp32 tiles of 128 142, of 64 125; bf16 stages of products that read from memory
// take 1.15 to 1.3 times as long, which is what stands here.
struct Kernel {
  Tiles tiles;
  int bm, bn, per_cu;
  float stage[3], round;
};
constexpr Kernel kBf16[] = {{TILES_256, 256, 256, 1, {1.85f}, 14.0f},
                            {TILES_128, 128, 128, 2, {0.87f, 1.15f}, 4.0f},
                            {TILES_64, 64, 64, 3, {0.45f, 0.55f, 0.70f}, 2.0f}};
constexpr Kernel kF32[] = {{TILES_128, 128, 128, 2, {2.03f, 3.8f}, 5.0f},
                           {TILES_64, 64, 64, 3, {0.68f, 1.14f, 1.62f}, 2.0f}};
constexpr int kCus = 256;
static_assert(kCus <= kFewWords, "a split product of few rows has fewer column blocks than CUs");

// Few rows: whether the kernel that streams the weight takes a product, and how. Up to
// 16 rows always (one row of 1024 x 4096: 5.0 us, on tiles 8.4); up to 64 for weights
// of at most 32 MB (61 rows of 1024 x 4096: 9.2 and 9.7; of 8192 x 8192: 41 and 36). k
// is split for a workgroup a CU, about 512 of k or more each (a round of the waves'
// loads): 4096 x 1024 14.5 -> 7.0; not at k <= 1024, where the joining costs more: k 512
// always (61 rows and 4096 columns 6.6 whole, 6.8 in two), k 1024 with 8192 columns (one
// row 5.6 and 7.1, 61 rows 9.5 and 11.5) or one row of 4096 (5.2 and 5.9). From 33 rows
// and up to 4096 columns two slices would be ahead there (61 rows 9.3 and 8.4).
bool plan_rows(int type, Form form, Epi epi, int64_t M, int64_t N, int64_t K, Plan& q) {
  if (form == FORM_TT || epi == EPI_GATED_BWD || M > kFewRows) return false;
  const int64_t n = epi == EPI_GATED ? 2 * N : N;
  const int64_t bytes = n * K * esize(type);
  if (M > 16 && bytes > (int64_t)32 << 20) return false;
  const int cols = type == VMOE_DENSE_BF16 && form == FORM_KT && bytes > (int64_t)12 << 20 ? 64 : 32;
  q.tiles = cols == 64 ? ROWS_64 : ROWS_32;
  q.tiles_m = 1;
  q.tiles_n = (int)cdiv(n, cols);
  const int64_t stage = 128 / esize(type);
  const int64_t most = K <= 1024 && cols == 32 ? 1 : cdiv(K, 512);
  const int64_t s = std::max<int64_t>(1, std::min<int64_t>(cdiv(kCus, q.tiles_n), most));
  q.kper = cdiv(cdiv(K, stage), s) * stage;
  q.splits = (int)cdiv(K, q.kper);  // (more than one: fewer than kFewWords column blocks)
  q.whole = 0;
  q.part_bytes = q.splits > 1 ? align256((size_t)q.splits * M * q.tiles_n * cols * 4) : 0;
  return true;
}

// Every kernel's time is estimated and the least taken. Tiles that do not fill the card
// a whole number of times leave it partly idle at the end: the remaining ones are split
// along k, where that is estimated to take less time with the joining (3 us and 0.22 us
// for each MB of sums, measured at 4 to 67 MB). Of 52 products drawn over the whole
// range those on tiles take 4 % longer than with the best of a sweep over tiles and
// splits, those of few rows 15 % less than on tiles.
Plan estimate(int type, Form form, Epi epi, int64_t M, int64_t N, int64_t K) {
  Plan best = {};
  if (plan_rows(type, form, epi, M, N, K, best)) return best;
  const int64_t n = epi == EPI_GATED ? 2 * N : N;  // columns staged
  const int64_t stage = 128 / esize(type), stages = cdiv(K, stage);
  float least = 0.0f;
  const bool bf16 = type == VMOE_DENSE_BF16;
  for (int i = 0; i < (bf16 ? 3 : 2); ++i) {
    const Kernel& k = bf16 ? kBf16[i] : kF32[i];
    const int bn = k.tiles == TILES_64 && epi == EPI_GATED ? 128 : k.bn;
    const float scale = bn == k.bn ? 1.0f : 1.8f;
    auto stage_us = [&](int residents) { return scale * k.stage[residents - 1]; };
    Plan q = {};
    q.tiles = k.tiles;
    q.tiles_m = (int)cdiv(M, k.bm);
    q.tiles_n = (int)cdiv(n, bn);
    const int64_t tiles = (int64_t)q.tiles_m * q.tiles_n;
    q.splits = 1;
    q.kper = stages * stage;
    // rounds of k.per_cu tiles a CU, then one of `last` and the rest
    const int each = (int)(tiles / kCus), last = each % k.per_cu;
    float time = (float)(each / k.per_cu) * ((float)stages * stage_us(k.per_cu) + k.round);
    if (tiles % (kCus * k.per_cu)) {
      float tail = (float)stages * stage_us(tiles % kCus ? last + 1 : last);
      q.whole = (int)tiles;
      // `beside` of the last round's tiles stay whole, the others' slices fill the free
      // places of each CU r / free times
      for (int beside = 0; beside <= last; beside += std::max(last, 1)) {
        const int rest = (int)(tiles - (int64_t)(each - last + beside) * kCus);
        if (!rest) continue;
        const int free = k.per_cu - beside;
        const float base = beside ? (float)stages * stage_us(beside) : 0.0f;
        int64_t before = 0;
        for (int r = 1; r <= 4 * free; ++r) {
          const int64_t slices = std::min<int64_t>(r * kCus / rest, stages / 4);
          if (slices < 2 || slices == before) continue;
          before = slices;
          const int64_t per = cdiv(stages, slices);
          const int units = rest * (int)cdiv(stages, per), u = (int)cdiv(units, kCus);
          const float mb = (float)units * (float)(k.bm * bn * 4) * 1e-6f;
          float t = 3.0f + mb * 0.22f;
          if (u <= free)
            t += base + (float)per * (stage_us(beside + u) - (beside ? stage_us(beside) : 0.0f));
          else  // every place taken to the end
            t += (float)(beside * stages + cdiv(u, free) * free * per) *
                 stage_us(k.per_cu) / (float)k.per_cu;
          if (t < tail) {
            tail = t;
            q.whole = (int)(tiles - rest);
            q.splits = (int)cdiv(stages, per);
            q.kper = per * stage;
          }
        }
      }
      time += tail + k.round;
    } else {
      q.whole = (int)tiles;
    }
    const int64_t split = tiles - q.whole;
    q.part_bytes = align256((size_t)split * q.splits * k.bm * bn * 4);
    if (!best.splits || time < least) {
      best = q;
      least = time;
    }
  }
  return best;
}

// The plan of a product; the last few are kept (an estimate takes 0.2 us, a backward call asks
// for up to twelve).
Plan plan_of(int type, Form form, Epi epi, int64_t M, int64_t N, int64_t K) {
  struct Kept {
    int64_t key[4];
    Plan plan;
  };
  constexpr int kKept = 64;
  static thread_local Kept kept[kKept] = {};  // (no product's key is zeros: M > 0)
  const int64_t key[4] = {M, N, K, type + 2 * form + 6 * epi};
  const uint64_t mix = (uint64_t)(M * 31 + N) * 31 + (uint64_t)(K * 31 + key[3]);
  Kept& e = kept[(mix * 0x9E3779B97F4A7C15ull) >> 58];
  if (!std::equal(key, key + 4, e.key)) {
    e.plan = estimate(type, form, epi, M, N, K);
    std::copy(key, key + 4, e.key);
  }
  return e.plan;
}

// Rows of column sums an EPI_GATED_BWD product leaves: one for each wave row (half a
// tile) that holds rows.
int64_t gated_sum_rows(const Plan& q, int64_t M) {
  return cdiv(M, q.tiles == TILES_256 ? 128 : q.tiles == TILES_128 ? 64 : 32);
}

// One product with its epilogue. part: Plan::part_bytes.
int product(int type, Form form, Epi epi, GemmArgs p, const Plan& q, float* part, hipStream_t s) {
  p.tiles_m = q.tiles_m;
  p.tiles_n = q.tiles_n;
  p.whole = q.whole;
  p.splits = q.splits;
  p.kper = q.kper;
  p.part = part;
  if (q.tiles == ROWS_32 || q.tiles == ROWS_64) {
    p.ldp = epi == EPI_GATED ? 2 * p.N : p.N;
    const int cols = q.tiles == ROWS_64 ? 64 : 32;
    if (q.splits == 1 || p.words) return gemm_few(type, form, epi, p, cols, s);
    GemmArgs g = p;
    g.N = p.ldp;
    VMOE_TRY(gemm_few(type, form, EPI_PARTIAL, g, cols, s));
    return join_rows(type, epi, p, s);
  }
  VMOE_TRY(gemm_tiles(type, form, epi, p, q.tiles, s));
  return q.splits > 1 ? join_tiles(type, epi, p, q.tiles, s) : VMOE_OK;
}
int product(int type, Form form, Epi epi, const GemmArgs& p, float* part, hipStream_t s) {
  return product(type, form, epi, p, plan_of(type, form, epi, p.M, p.N, p.K), part, s);
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
  return transposed ? plan_of(type, FORM_TT, EPI_LINEAR, out, in, rows).part_bytes
                    : plan_of(type, FORM_TT, EPI_LINEAR, in, out, rows).part_bytes;
}

// Workspace: the slices' sums of one product at a time, then each buffer. It does not
// depend on the weights' order: the larger of both.
struct Bytes {
  size_t part, grads, sums, total;
};
size_t either_order(int type, Epi epi, int64_t M, int64_t N, int64_t K) {
  return std::max(plan_of(type, FORM_KK, epi, M, N, K).part_bytes,
                  plan_of(type, FORM_KT, epi, M, N, K).part_bytes);
}
Bytes linear_bytes(int type, int64_t rows, int64_t in, int64_t out, int act, int backward) {
  Bytes b = {};
  if (!backward) {
    b.part = either_order(type, EPI_LINEAR, rows, out, in);
  } else {
    b.part = std::max({either_order(type, EPI_LINEAR, rows, in, out),
                       weight_grad_bytes(type, in, out, rows, 0),
                       weight_grad_bytes(type, in, out, rows, 1)});
    if (act != VMOE_DENSE_NONE) b.grads = align256((size_t)rows * out * esize(type));
    b.sums = align256((size_t)sum_rows(rows, out) * out * 4);
  }
  b.total = b.part + b.grads + b.sums;
  return b;
}
Bytes gated_bytes(int type, int64_t rows, int64_t d, int64_t width, int backward) {
  Bytes b = {};
  if (!backward) {
    b.part = std::max(either_order(type, EPI_GATED, rows, width, d),
                      either_order(type, EPI_LINEAR, rows, d, width));
  } else {
    const Plan q = plan_of(type, FORM_KK, EPI_GATED_BWD, rows, width, d);
    b.part = std::max({q.part_bytes, either_order(type, EPI_LINEAR, rows, d, 2 * width),
                       weight_grad_bytes(type, d, 2 * width, rows, 0),
                       weight_grad_bytes(type, d, 2 * width, rows, 1),
                       weight_grad_bytes(type, width, d, rows, 0),
                       weight_grad_bytes(type, width, d, rows, 1)});
    b.grads = align256((size_t)rows * 2 * width * esize(type));
    b.sums = align256((size_t)std::max(gated_sum_rows(q, rows) * 2 * width, sum_rows(rows, d) * d) * 4);
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

extern "C" int32_t vmoe_dense_arrival_words(void) { return kFewWords; }

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
                                   uint32_t* words, vmoe_stream_t stream) {
  VMOE_TRY(check_sizes(type, act, rows, in, out));
  if (rows == 0) return VMOE_OK;
  VMOE_TRY(check_rows(type, x, in, ldx));
  VMOE_TRY(check_weight(type, w, ldw, w_transposed, in, out));
  VMOE_TRY(check_rows(type, y, out, ldy));
  if (residual) VMOE_TRY(check_rows(type, residual, out, ldr));
  if (z && !aligned(z)) return VMOE_ERR_UNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(words) & 3) return VMOE_ERR_UNSUPPORTED;
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
  p.z_past = z_past(rows, out);
  p.words = words;
  return product(type, forward_form(w_transposed), EPI_LINEAR, p, static_cast<float*>(workspace),
                 reinterpret_cast<hipStream_t>(stream));
}

extern "C" int vmoe_linear_backward(int32_t type, const void* gy, int64_t ldgy, const void* x,
                                    int64_t ldx, int64_t rows, int64_t in, int64_t out,
                                    const void* w, int64_t ldw, int32_t w_transposed,
                                    int32_t act, const float* z, const void* y, int64_t ldy,
                                    void* gx, int64_t ldgx, void* gw, int64_t ldgw, void* gb,
                                    int32_t gb_f32, void* workspace, size_t workspace_bytes,
                                    vmoe_stream_t stream) {
  VMOE_TRY(check_sizes(type, act, rows, in, out));
  if (rows == 0) return VMOE_OK;
  VMOE_TRY(check_rows(type, gy, out, ldgy));
  if (gw) VMOE_TRY(check_rows(type, x, in, ldx));
  if (gx) VMOE_TRY(check_weight(type, w, ldw, w_transposed, in, out));
  if (gx) VMOE_TRY(check_rows(type, gx, in, ldgx));
  if (gw) VMOE_TRY(check_weight(type, gw, ldgw, w_transposed, in, out));
  const bool has_act = act != VMOE_DENSE_NONE;
  const bool from_y = has_act && !z;
  if (from_y && act != VMOE_DENSE_RELU) return VMOE_ERR_INVALID_ARG;
  if (from_y) VMOE_TRY(check_rows(type, y, out, ldy));
  if (z && !aligned(z)) return VMOE_ERR_UNSUPPORTED;
  const Bytes b = linear_bytes(type, rows, in, out, act, 1);
  VMOE_TRY(check_workspace(workspace, workspace_bytes, b.total));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  float* part = reinterpret_cast<float*>(ws);
  void* dz = ws + b.part;
  float* sums = reinterpret_cast<float*>(ws + b.part + b.grads);
  if (has_act || gb) {
    VMOE_TRY(act_grad(type, gy, ldgy, has_act ? z : nullptr, out, from_y ? y : nullptr, ldy, act,
                      dz, out, gb ? sums : nullptr, rows, out, s));
    if (gb) VMOE_TRY(col_sum(sums, sum_rows(rows, out), out, out, gb, gb_f32, nullptr, 0, s));
  }
  const void* g = has_act ? dz : gy;
  const int64_t ldg = has_act ? out : ldgy;
  if (gx)
    VMOE_TRY(product(type, input_grad_form(w_transposed), EPI_LINEAR,
                     args(g, ldg, w, ldw, rows, in, out, gx, ldgx), part, s));
  if (gw)
    VMOE_TRY(product(type, FORM_TT, EPI_LINEAR,
                     weight_grad_args(w_transposed, x, ldx, in, g, ldg, out, rows, gw, ldgw), part,
                     s));
  return VMOE_OK;
}

extern "C" size_t vmoe_gated_workspace_bytes(int32_t type, int64_t rows, int64_t hidden,
                                             int64_t width, int32_t backward) {
  if (check_sizes(type, VMOE_DENSE_NONE, rows, hidden, width) != VMOE_OK) return 0;
  return gated_bytes(type, rows, hidden, width, backward).total;
}

namespace {
// The weights that are read. (The up columns of a weight stored [2 width, hidden] are
// addressed from the gate's by a 32-bit offset.)
int check_gated_weights(int type, bool read1, const void* w1, int64_t ldw1, int t1, bool read2,
                        const void* w2, int64_t ldw2, int t2, int64_t d, int64_t width) {
  if (read1) VMOE_TRY(check_weight(type, w1, ldw1, t1, d, 2 * width));
  if (read2) VMOE_TRY(check_weight(type, w2, ldw2, t2, width, d));
  if (read1 && t1 && (width + 256) * ldw1 * esize(type) >= (int64_t)1 << 31) return VMOE_ERR_UNSUPPORTED;
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
                                  uint32_t* words, vmoe_stream_t stream) {
  VMOE_TRY(check_sizes(type, act, rows, hidden, width));
  if (rows == 0) return VMOE_OK;
  VMOE_TRY(check_rows(type, x, hidden, ldx));
  VMOE_TRY(check_gated_weights(type, true, w1, ldw1, w1_transposed, true, w2, ldw2, w2_transposed,
                               hidden, width));
  VMOE_TRY(check_rows(type, h, width, width));
  VMOE_TRY(check_rows(type, y, hidden, ldy));
  if (residual) VMOE_TRY(check_rows(type, residual, hidden, ldr));
  if (z && !aligned(z)) return VMOE_ERR_UNSUPPORTED;
  if (reinterpret_cast<uintptr_t>(words) & 3) return VMOE_ERR_UNSUPPORTED;
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
  p.z_past = z_past(rows, 2 * width);
  p.words = words;
  VMOE_TRY(product(type, forward_form(w1_transposed), EPI_GATED, p, part, s));
  GemmArgs q = args(h, width, w2, ldw2, rows, hidden, width, y, ldy);
  q.bias = bias2;
  q.bias_f32 = bias2_f32;
  q.act = VMOE_DENSE_NONE;
  q.res = residual;
  q.ldr = ldr;
  q.words = words;
  return product(type, forward_form(w2_transposed), EPI_LINEAR, q, part, s);
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
  const bool inner = gx || gw1 || gb1;  // what needs the gradient of [gate | up]
  VMOE_TRY(check_gated_weights(type, gx, w1, ldw1, w1_transposed, inner, w2, ldw2, w2_transposed,
                               hidden, width));
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
    p.z_past = z_past(rows, w2x);
    p.sums = gb1 ? sums : nullptr;
    const Form form = input_grad_form(w2_transposed);
    const Plan q = plan_of(type, form, EPI_GATED_BWD, rows, width, hidden);
    VMOE_TRY(product(type, form, EPI_GATED_BWD, p, q, part, s));
    if (gb1)
      VMOE_TRY(col_sum(sums, gated_sum_rows(q, rows), w2x, w2x, gb1, gb1_f32, nullptr, 0, s));
  }
  if (gb2) {
    VMOE_TRY(act_grad(type, gy, ldgy, nullptr, 0, nullptr, 0, VMOE_DENSE_NONE, nullptr, 0, sums, rows,
                      hidden, s));
    VMOE_TRY(col_sum(sums, sum_rows(rows, hidden), hidden, hidden, gb2, gb2_f32, nullptr,
                     0, s));
  }
  if (gw2)
    VMOE_TRY(product(type, FORM_TT, EPI_LINEAR,
                     weight_grad_args(w2_transposed, h, width, width, gy, ldgy, hidden, rows, gw2,
                                      ldgw2), part, s));
  if (gx)
    VMOE_TRY(product(type, input_grad_form(w1_transposed), EPI_LINEAR,
                     args(dz, w2x, w1, ldw1, rows, hidden, w2x, gx, ldgx), part, s));
  if (gw1)
    VMOE_TRY(product(type, FORM_TT, EPI_LINEAR,
                     weight_grad_args(w1_transposed, x, ldx, hidden, dz, w2x, w2x, rows, gw1,
                                      ldgw1), part, s));
  return VMOE_OK;
}
