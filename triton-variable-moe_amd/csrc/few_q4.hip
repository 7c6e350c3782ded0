// Laying out matrices in 4 bits with group scales, and reading them back
// (layout: few_q4.h).
//
// Both move each byte once. A wave takes 128 rows x 64 columns, four blocks: lane
// l has four adjacent columns, 4 (l % 16).., of rows 8 (l / 16) + 0..7 of each 32,
// which is what the block order wants of a column in one lane, so the values stay
// in registers. Row-major accesses are runs of 64 columns (128 bytes in bf16). The
// maximum of a group is the maximum of four lanes. Bytes that are read or written
// once go past the caches, and the codes through LDS, so that a store is a whole
// kilobyte and not 64 pieces of it: 128 matrices 2048 x 576 in groups of 128, 302
// MB, are laid out in 91 us (4.2 TB/s; 128 us before these two) and read back in 98
// to 106 (3.6 to 3.9 TB/s); a copy moves 5.2 TB/s.
//
// The nearest value: |w| against the middles between values times the scale. Those
// products are exact in fp32 (a scale of 8 bits, a middle of 3), so no choice
// depends on a rounding, and a tie goes to the even place; only the scale itself,
// max / 6, rounds. For bf16 w the conversion instruction compares instead: it gets
// the quotient w / s, whose two-step reciprocal form is exact where w is a middle
// times s, and elsewhere w / s is at least 2^-12 of itself away from a middle.
#include "few_q4.h"

namespace vmoe {
namespace {

constexpr int kLaneCols = 4;  // adjacent columns of a lane
constexpr int kThreads = 256, kWaves = kThreads / kWave, kTileCols = 16 * kLaneCols;

struct Q4Args {
  const void* w;
  void* out;
  int64_t ld;
  const MatEntry* tab;
  void* codes;
  uint16_t* scales;
  int by_rows, fixed, tiles_n, tiles_k, units;
  int wide;  // four columns of w or out can be one access
};

struct TilePos {
  int K, N, k0, n0, base;
  int64_t row0, col0;
  bool ok;
};

// Wave -> tile, the columns fastest; an XCD (blockIdx % 8) takes a contiguous
// eighth, so that it uses every channel of its L2 whatever the row stride.
__device__ __forceinline__ TilePos tile_pos(const Q4Args& p) {
  TilePos t = {};
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int per = (p.units + 7) / 8, j = (blockIdx.x >> 3) * kWaves + wave;
  const int u = (blockIdx.x & 7) * per + j;
  if (j >= per || u >= p.units) return t;
  const int nt = u % p.tiles_n, mk = u / p.tiles_n;
  const MatEntry m = p.tab[mk / p.tiles_k];
  t.K = p.by_rows ? m.len : p.fixed;
  t.N = p.by_rows ? p.fixed : m.len;
  t.k0 = mk % p.tiles_k * kQ4Rows;
  t.n0 = nt * kTileCols;
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

// w / s for bf16 values, r = 1 / s to a unit in the last place.
__device__ __forceinline__ float quotient(float w, float s, float r) {
  const float q = w * r;
  return fmaf(fmaf(-q, s, w), r, q);
}

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// A lane's columns of a row.
template <bool F32>
struct RowPart {
  static constexpr int D = F32 ? kLaneCols : kLaneCols / 2;  // dwords
  typedef uint32_t vec __attribute__((ext_vector_type(D)));
  uint32_t v[D];
  __device__ __forceinline__ uint32_t bits(int c) const {  // as fp32
    if constexpr (F32) {
      return v[c];
    } else {
      return (c & 1) ? v[c / 2] & 0xFFFF0000u : v[c / 2] << 16;
    }
  }
  __device__ __forceinline__ void load(const void* w, int64_t at, bool wide) {
    if (wide) {
      const vec x = __builtin_nontemporal_load(
          reinterpret_cast<const vec*>(static_cast<const char*>(w) + at * (F32 ? 4 : 2)));
#pragma unroll
      for (int i = 0; i < D; ++i) v[i] = x[i];
    } else if constexpr (F32) {
#pragma unroll
      for (int c = 0; c < kLaneCols; ++c) v[c] = static_cast<const uint32_t*>(w)[at + c];
    } else {
      const uint16_t* q = static_cast<const uint16_t*>(w) + at;
#pragma unroll
      for (int c = 0; c < kLaneCols; c += 2) v[c / 2] = q[c] | (uint32_t)q[c + 1] << 16;
    }
  }
  __device__ __forceinline__ void store(void* out, int64_t at, bool wide) const {
    if (wide) {
      vec x;
#pragma unroll
      for (int i = 0; i < D; ++i) x[i] = v[i];
      __builtin_nontemporal_store(
          x, reinterpret_cast<vec*>(static_cast<char*>(out) + at * (F32 ? 4 : 2)));
    } else if constexpr (F32) {
#pragma unroll
      for (int c = 0; c < kLaneCols; ++c) static_cast<uint32_t*>(out)[at + c] = v[c];
    } else {
      uint16_t* q = static_cast<uint16_t*>(out) + at;
#pragma unroll
      for (int c = 0; c < kLaneCols; ++c) q[c] = (uint16_t)(v[c / 2] >> (c % 2 * 16));
    }
  }
};

template <bool F32, int G>
__global__ __launch_bounds__(kThreads) void quantize_kernel(Q4Args p) {
  constexpr int S = kQ4Rows / G;  // groups of a column
  constexpr int J = G / 32;       // 32-row quarters of a group
  __shared__ u32x4_t blocks[kWaves][kLaneCols][kWave];
  const TilePos t = tile_pos(p);
  if (!t.ok) return;  // (the whole wave)
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, g = lane >> 4;
  const int c0 = t.n0 + (lane & 15) * kLaneCols;
  const bool in = c0 < t.N;
  RowPart<F32> w[4][8];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = t.k0 + 32 * j + 8 * g + i;
      w[j][i] = {};
      if (in && r < t.K) w[j][i].load(p.w, (t.row0 + r) * p.ld + t.col0 + c0, p.wide);
    }
  const int kbs = (t.K + kQ4Rows - 1) / kQ4Rows;
  const int64_t blk = t.base + (int64_t)(c0 / kQ4Cols) * kbs + t.k0 / kQ4Rows;
#pragma unroll
  for (int c = 0; c < kLaneCols; ++c) {
    const int col = c0 % kQ4Cols + c;  // of the block
    u32x4_t word;
#pragma unroll
    for (int q = 0; q < S; ++q) {
      // magnitudes order as their bits, infinities and NaN above all numbers
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, w[q * J + j][i].bits(c) & 0x7FFFFFFFu);
      top = max(top, (uint32_t)__shfl_xor((int)top, 16, kWave));
      top = max(top, (uint32_t)__shfl_xor((int)top, 32, kWave));
      const uint32_t sb = top < 0x7F800000u ? f32_to_bf16(__uint_as_float(top) / 6.0f) : 0x7FC0u;
      const float s = bf16_to_f32(sb);
      // (a block's columns past the matrix get zeros)
      if (g == 0 && c0 / kQ4Cols * kQ4Cols < t.N)
        p.scales[(blk * kQ4Cols + col) * S + q] = (uint16_t)sb;
      // (the reciprocal of smaller scales would leave fp32's range)
      const bool fast = !F32 && s >= 0x1p-100f;
      const float r = fast ? __builtin_amdgcn_rcpf(s) : 0.0f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const RowPart<F32>* v = w[q * J + j];
        uint32_t codes = 0;
        if (fast) {
          auto two = [&](int i) {
            return f32x2_t{quotient(__uint_as_float(v[i].bits(c)), s, r),
                           quotient(__uint_as_float(v[i + 1].bits(c)), s, r)};
          };
          const f32x2_t q0 = two(0), q1 = two(2), q2 = two(4), q3 = two(6);
          codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, q0.x, q0.y, 1.0f, 0);
          codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, q1.x, q1.y, 1.0f, 1);
          codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, q2.x, q2.y, 1.0f, 2);
          codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, q3.x, q3.y, 1.0f, 3);
        } else if (s > 0.0f) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            codes |= code_of(__uint_as_float(v[i].bits(c)), s) << (4 * i);
        }
        word[q * J + j] = codes;
      }
    }
    blocks[wave][(lane & 15) * kLaneCols / kQ4Cols][g * 16 + col] = word;
  }
  // (each wave reads what it wrote)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int b = 0; b < kLaneCols; ++b) {
    const int nb = t.n0 / kQ4Cols + b;
    if (nb * kQ4Cols >= t.N) break;
    __builtin_nontemporal_store(
        blocks[wave][b][lane],
        reinterpret_cast<u32x4_t*>(p.codes) +
            (t.base + (int64_t)nb * kbs + t.k0 / kQ4Rows) * kWave + lane);
  }
}

template <bool F32, int G>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(Q4Args p) {
  constexpr int S = kQ4Rows / G;
  const TilePos t = tile_pos(p);
  if (!t.ok) return;
  const int lane = threadIdx.x % kWave, g = lane >> 4;
  const int c0 = t.n0 + (lane & 15) * kLaneCols;
  if (c0 >= t.N) return;
  const int kbs = (t.K + kQ4Rows - 1) / kQ4Rows;
  const int64_t blk = t.base + (int64_t)(c0 / kQ4Cols) * kbs + t.k0 / kQ4Rows;
  u32x4_t word[kLaneCols];
  float s[kLaneCols][S];
#pragma unroll
  for (int c = 0; c < kLaneCols; ++c) {
    const int64_t col = blk * kQ4Cols + c0 % kQ4Cols + c;
    word[c] = reinterpret_cast<const u32x4_t*>(p.codes)[blk * kWave + g * 16 + c0 % kQ4Cols + c];
#pragma unroll
    for (int q = 0; q < S; ++q) s[c][q] = bf16_to_f32(p.scales[col * S + q]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    bf16x8_t v[kLaneCols];
#pragma unroll
    for (int c = 0; c < kLaneCols; ++c) v[c] = q4_values(word[c][j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = t.k0 + 32 * j + 8 * g + i;
      if (r >= t.K) break;
      const int64_t at = (t.row0 + r) * p.ld + t.col0 + c0;
      float f[kLaneCols];
#pragma unroll
      for (int c = 0; c < kLaneCols; ++c) f[c] = s[c][32 * j / G] * (float)v[c][i];
      RowPart<F32> part;
      if constexpr (F32) {
#pragma unroll
        for (int c = 0; c < kLaneCols; ++c) part.v[c] = __float_as_uint(f[c]);
      } else {
#pragma unroll
        for (int c = 0; c < kLaneCols; c += 2) part.v[c / 2] = pack_bf16(f[c], f[c + 1]);
      }
      part.store(p.out, at, p.wide);
    }
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

bool grid_of(Q4Args& p, int M, int64_t max_len, bool f32, dim3& grid) {
  // (starts and lengths along the columns are multiples of 8)
  const uintptr_t base = reinterpret_cast<uintptr_t>(p.w ? p.w : p.out);
  p.wide = base % 16 == 0 && p.ld % 4 == 0;
  const int64_t k = p.by_rows ? max_len : p.fixed, n = p.by_rows ? p.fixed : max_len;
  p.tiles_k = (int)((k + kQ4Rows - 1) / kQ4Rows);
  p.tiles_n = (int)((n + kTileCols - 1) / kTileCols);
  const int64_t units = (int64_t)p.tiles_k * p.tiles_n * M;
  p.units = (int)units;
  grid = dim3((unsigned)(((units + 7) / 8 + kWaves - 1) / kWaves * 8));
  return units <= (1 << 30);
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
  if (!grid_of(p, num_matrices, max_len, w_is_f32, grid)) return VMOE_ERR_UNSUPPORTED;
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
  if (!grid_of(p, num_matrices, max_len, out_is_f32, grid)) return VMOE_ERR_UNSUPPORTED;
  if (out_is_f32)
    VMOE_Q4_LAUNCH(dequantize_kernel, true, group);
  else
    VMOE_Q4_LAUNCH(dequantize_kernel, false, group);
  VMOE_CHECK_LAUNCH();
  return VMOE_OK;
}
