// What the dense operators' entry points (dense.hip) call.
#pragma once

#include "dense.h"

namespace vmoe {
namespace dense {

enum Form { FORM_KK, FORM_KT, FORM_TT };  // A's, B's
enum Tiles { ROWS_32, ROWS_64, TILES_64, TILES_128, TILES_256 };  // ROWS: dense_few.hip

// Pre-activations of 64 MB or more are written and read past the caches: a pass reads
// them once, and the last-level cache (256 MB) keeps what the next launches read
// (a training pass of 8192 x 1024 x 4096, 128 MB: 353 -> 335 us; 6144 rows, 96 MB: 278 ->
// 266; gated 4096 x 1024 x 2816, 88 MB: 360 -> 339; 8192 rows, 176 MB: 647 -> 576. At 64 MB
// 187 and 188, below that it loses 0.5 to 3 %: 32 MB 111.8 -> 112.8, 16 MB 77 -> 80).
constexpr int64_t kPastCache = 64 << 20;
inline int z_past(int64_t rows, int64_t cols) { return rows * cols * 4 >= kPastCache; }

inline uint32_t workgroups(const GemmArgs& p) {
  return (uint32_t)(p.whole + (p.tiles_m * p.tiles_n - p.whole) * p.splits);
}

// dense_big.hip: TILES_256, bf16
int gemm_big(Form form, Epi epi, const GemmArgs& p, hipStream_t s);
// dense_few.hip: at most kFewRows rows, workgroups of `cols` columns (32, or for T-form
// weights in bf16 64)
constexpr int64_t kFewRows = 64;
constexpr int kFewWords = 256;  // arrival words: column blocks of a product that is split
int gemm_few(int type, Form form, Epi epi, const GemmArgs& p, int cols, hipStream_t s);
// dense_gemm.hip: the product on tiles; the epilogue of its split tiles; the epilogue
// of gemm_few's slices
int gemm_tiles(int type, Form form, Epi epi, const GemmArgs& p, Tiles tiles, hipStream_t s);
int join_tiles(int type, Epi epi, const GemmArgs& p, Tiles tiles, hipStream_t s);
int join_rows(int type, Epi epi, const GemmArgs& p, hipStream_t s);
int64_t sum_rows(int64_t M, int64_t N);  // rows of the sums that act_grad leaves
// (z, or for relu y; neither: dz is gy and not written)
int act_grad(int type, const void* gy, int64_t ldgy, const float* z, int64_t ldz, const void* y,
             int64_t ldy, int act, void* dz, int64_t lddz, float* part, int64_t M, int64_t N,
             hipStream_t s);
// column sums of part [rows, N]: columns below `split` into out0, the others into out1
int col_sum(const float* part, int64_t rows, int64_t N, int64_t split, void* out0, int out0_f32,
            void* out1, int out1_f32, hipStream_t s);

}  // namespace dense
}  // namespace vmoe
