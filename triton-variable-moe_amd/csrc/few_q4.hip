// Laying out matrices in 4 bits with group scales, and reading them back
// (layout: few_q4.h).
//
// Both move each byte once. A workgroup takes 128 rows x 64 columns, four blocks:
// it reads or writes the row-major side in runs of 64 columns (128 bytes a row
// in bf16) and the blocks in whole kilobytes, and LDS turns one order into the
// other. The nearest value is found by comparing |w| with the middles between
// values times the scale: a bf16 scale times a middle of at most three bits is
// exact in fp32, so no choice depends on a rounding, and a tie goes to the even
// place. Only the scale itself, max / 6, rounds.
#include <math.h>

#include "few_q4.h"

namespace vmoe {
namespace {

constexpr int kThreads = 256, kTileCols = 64;

struct Q4Args {
  const void* w;
  void* out;
  int64_t ld;
  const MatEntry* tab;
  void* codes;
  uint16_t* scales;
  int by_rows, fixed, tiles_n, tiles_k;
};

struct TilePos {
  int K, N, k0, n0, base;
  int64_t row0, col0;
  bool ok;
};

__device__ __forceinline__ TilePos tile_pos(const Q4Args& p) {
  const MatEntry m = p.tab[blockIdx.y];
  TilePos t;
  t.K = p.by_rows ? m.len : p.fixed;
  t.N = p.by_rows ? p.fixed : m.len;
  t.k0 = (int)(blockIdx.x / p.tiles_n) * kQ4Rows;
  t.n0 = (int)(blockIdx.x % p.tiles_n) * kTileCols;
  t.base = m.base;
  t.row0 = p.by_rows ? m.off : 0;
  t.col0 = p.by_rows ? 0 : m.off;
  t.ok = t.k0 < t.K && t.n0 < t.N;
  return t;
}

// The code of w for the scale s (finite, above 0).
__device__ __forceinline__ uint32_t code_of(float w, float s) {
  const float a = fabsf(w);
  const uint32_t c = (a > 0.25f * s) + (a >= 0.75f * s) + (a > 1.25f * s) + (a >= 1.75f * s) +
                     (a > 2.5f * s) + (a >= 3.5f * s) + (a > 5.0f * s);
  return c ? c | (w < 0.0f ? 8u : 0u) : 0u;
}

template <bool F32, int G>
__global__ __launch_bounds__(kThreads) void quantize_kernel(Q4Args p) {
  constexpr int S = kQ4Rows / G;  // groups of a tile's column
  const TilePos t = tile_pos(p);
  if (!t.ok) return;
  __shared__ float tile[kQ4Rows][kTileCols + 1];
  __shared__ float scale[S][kTileCols];
  const int c = threadIdx.x % kTileCols;
  for (int r = threadIdx.x / kTileCols; r < kQ4Rows; r += kThreads / kTileCols) {
    float v = 0.0f;
    if (t.k0 + r < t.K && t.n0 + c < t.N) {
      const int64_t at = (t.row0 + t.k0 + r) * p.ld + t.col0 + t.n0 + c;
      v = F32 ? static_cast<const float*>(p.w)[at]
              : bf16_to_f32(static_cast<const uint16_t*>(p.w)[at]);
    }
    tile[r][c] = v;
  }
  __syncthreads();
  const int kbs = (t.K + kQ4Rows - 1) / kQ4Rows, kb = t.k0 / kQ4Rows;
  for (int i = threadIdx.x; i < S * kTileCols; i += kThreads) {
    const int g = i / kTileCols, n = i % kTileCols;
    float top = 0.0f;
    bool finite = true;
    for (int r = 0; r < G; ++r) {
      const float a = fabsf(tile[g * G + r][n]);
      finite = finite && a <= 3.4028234e38f;
      top = fmaxf(top, a);
    }
    const uint32_t bits = finite ? f32_to_bf16(top / 6.0f) : 0x7FC0u;
    scale[g][n] = bf16_to_f32(bits);
    const int nb = (t.n0 + n) / kQ4Cols;
    if (nb * kQ4Cols < t.N) {
      const int64_t blk = t.base + (int64_t)nb * kbs + kb;
      p.scales[(blk * kQ4Cols + n % kQ4Cols) * S + g] = (uint16_t)bits;
    }
  }
  __syncthreads();
  // a thread writes the 16 bytes of one lane of a block
  const int b = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int nb = t.n0 / kQ4Cols + b, n = b * kQ4Cols + (lane & 15);
  if (nb * kQ4Cols >= t.N) return;
  uint32_t word[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = 32 * j + (lane >> 4) * 8;
    const float s = scale[r / G][n];
    uint32_t v = 0;
    if (s > 0.0f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v |= code_of(tile[r + i][n], s) << (4 * i);
    }
    word[j] = v;
  }
  const int64_t blk = t.base + (int64_t)nb * kbs + kb;
  reinterpret_cast<uint4*>(p.codes)[blk * kWave + lane] = {word[0], word[1], word[2], word[3]};
}

template <bool F32, int G>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(Q4Args p) {
  constexpr int S = kQ4Rows / G;
  const TilePos t = tile_pos(p);
  if (!t.ok) return;
  __shared__ float tile[kQ4Rows][kTileCols + 1];
  const int b = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int nb = t.n0 / kQ4Cols + b, n = b * kQ4Cols + (lane & 15);
  if (nb * kQ4Cols < t.N) {
    const int kbs = (t.K + kQ4Rows - 1) / kQ4Rows;
    const int64_t blk = t.base + (int64_t)nb * kbs + t.k0 / kQ4Rows;
    const uint4 word = reinterpret_cast<const uint4*>(p.codes)[blk * kWave + lane];
    const uint32_t words[4] = {word.x, word.y, word.z, word.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = 32 * j + (lane >> 4) * 8;
      const float s = bf16_to_f32(p.scales[(blk * kQ4Cols + (lane & 15)) * S + r / G]);
      const bf16x8_t v = q4_values(words[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) tile[r + i][n] = s * (float)v[i];
    }
  }
  __syncthreads();
  const int c = threadIdx.x % kTileCols;
  for (int r = threadIdx.x / kTileCols; r < kQ4Rows; r += kThreads / kTileCols) {
    if (t.k0 + r >= t.K || t.n0 + c >= t.N) continue;
    const int64_t at = (t.row0 + t.k0 + r) * p.ld + t.col0 + t.n0 + c;
    if (F32)
      static_cast<float*>(p.out)[at] = tile[r][c];
    else
      static_cast<uint16_t*>(p.out)[at] = (uint16_t)f32_to_bf16(tile[r][c]);
  }
}

int check(const void* w, int64_t ld, const int32_t* table, int32_t M, int32_t by_rows,
          int64_t fixed, int64_t max_len, int32_t group, const void* codes,
          const uint16_t* scales) {
  if (!w || !table || !codes || !scales || M <= 0 || fixed <= 0 || max_len <= 0 || by_rows < 0 ||
      by_rows > 1 || ld <= 0 || (by_rows && ld < fixed) || (!by_rows && ld < max_len))
    return VMOE_ERR_INVALID_ARG;
  if (group != 32 && group != 64 && group != 128) return VMOE_ERR_INVALID_ARG;
  if (M > 65535 || fixed > (1 << 28) || max_len > (1 << 28) ||
      reinterpret_cast<uintptr_t>(codes) % 16 || reinterpret_cast<uintptr_t>(table) % 16)
    return VMOE_ERR_UNSUPPORTED;
  return VMOE_OK;
}

bool grid_of(Q4Args& p, int M, int64_t max_len, dim3& grid) {
  const int64_t k = p.by_rows ? max_len : p.fixed, n = p.by_rows ? p.fixed : max_len;
  p.tiles_k = (int)((k + kQ4Rows - 1) / kQ4Rows);
  p.tiles_n = (int)((n + kTileCols - 1) / kTileCols);
  const int64_t tiles = (int64_t)p.tiles_k * p.tiles_n;
  grid = dim3((unsigned)tiles, M);
  return tiles <= (1 << 30);
}

}  // namespace
}  // namespace vmoe

using namespace vmoe;

#define VMOE_Q4_LAUNCH(K, F32, GROUP)                                                         \
  do {                                                                                        \
    if (GROUP == 32)                                                                          \
      VMOE_LAUNCH((K<F32, 32>), grid, dim3(kThreads), 0, stream, p);                          \
    else if (GROUP == 64)                                                                     \
      VMOE_LAUNCH((K<F32, 64>), grid, dim3(kThreads), 0, stream, p);                          \
    else                                                                                      \
      VMOE_LAUNCH((K<F32, 128>), grid, dim3(kThreads), 0, stream, p);                         \
  } while (0)

extern "C" int vmoe_q4_quantize(const void* w, int32_t w_is_f32, int64_t ldw, const int32_t* table,
                                int32_t num_matrices, int32_t by_rows, int64_t fixed,
                                int64_t max_len, int32_t group, void* codes, uint16_t* scales,
                                vmoe_stream_t stream) {
  const int st =
      check(w, ldw, table, num_matrices, by_rows, fixed, max_len, group, codes, scales);
  if (st != VMOE_OK) return st;
  Q4Args p = {w, nullptr, ldw, reinterpret_cast<const MatEntry*>(table), codes, scales, by_rows,
              (int)fixed};
  dim3 grid;
  if (!grid_of(p, num_matrices, max_len, grid)) return VMOE_ERR_UNSUPPORTED;
  if (w_is_f32)
    VMOE_Q4_LAUNCH(quantize_kernel, true, group);
  else
    VMOE_Q4_LAUNCH(quantize_kernel, false, group);
  VMOE_CHECK_LAUNCH();
  return VMOE_OK;
}

extern "C" int vmoe_q4_dequantize(const void* codes, const uint16_t* scales, const int32_t* table,
                                  int32_t num_matrices, int32_t by_rows, int64_t fixed,
                                  int64_t max_len, int32_t group, void* out, int32_t out_is_f32,
                                  int64_t ldo, vmoe_stream_t stream) {
  const int st =
      check(out, ldo, table, num_matrices, by_rows, fixed, max_len, group, codes, scales);
  if (st != VMOE_OK) return st;
  Q4Args p = {nullptr, out, ldo, reinterpret_cast<const MatEntry*>(table),
              const_cast<void*>(codes), const_cast<uint16_t*>(scales), by_rows, (int)fixed};
  dim3 grid;
  if (!grid_of(p, num_matrices, max_len, grid)) return VMOE_ERR_UNSUPPORTED;
  if (out_is_f32)
    VMOE_Q4_LAUNCH(dequantize_kernel, true, group);
  else
    VMOE_Q4_LAUNCH(dequantize_kernel, false, group);
  VMOE_CHECK_LAUNCH();
  return VMOE_OK;
}
