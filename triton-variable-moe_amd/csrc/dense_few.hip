// Matrix products of the dense operators for few rows (a generation step, up to 64
// rows), where the time is that of reading the weight once.
//
// The weight goes from memory straight into the operands of 16-wide matrix
// instructions. A workgroup takes CB columns and all of k (or a slice of it): its
// waves take steps of k in turn, several steps' loads under way each, and meet in
// LDS, where the sums are added in the order of the waves and go through the
// epilogue. One step is 32 k (fp32: 16), a quarter of the wave (16 lanes) 8 (4) of
// them. T-form: a lane loads CB / 16 adjacent columns of each of its k-rows, and
// byte permutes turn 8 rows into the operands of those columns. K-form: a lane's 16
// bytes are an operand of one column. Rows of x come as operands too, 16 bytes a lane
// and tile of 16 rows; they are in cache after the first workgroup.
//
// Measured at one row, weights from memory, joined by a second launch, us (floor at
// 5.2 TB/s):
// 1024 x 4096 stored [out, in] 5.0 (1.6), [in, out] 6.1; 2048 x 2048 6.6 and 6.9 (1.6);
// 5632 x 2048 10.0 and 9.4 (4.4); gated 2048 x 5632 14.4 and 15.4 (8.9); 8192 x 8192
// 27.5 and 28.1 (25.8). A CU draws 20 to 60 GB/s, so that weights below some 40 MB are
// bound by starting, one or two chains of loads and the joining. 64 columns for T-form
// weights over 12 MB: whole 128-byte lines of a k-row (gated 2048 x 5632 16.7 -> 15.4,
// 8192 x 8192 36 -> 28); below, and for K-form, 32 give more workgroups. 16 waves a
// workgroup, or one step a batch, changed nothing above the noise.

#include "dense_launch.h"

namespace vmoe {
namespace dense {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// Loads whose offset is kOob give zeros.
__device__ __forceinline__ u32x4_t load16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}

// A step's operands: of the weight w[j] for each 16 columns, of x for each 16 rows.
template <typename E, bool T, int RT, int CB>
struct Step {
  static constexpr int kCols = CB / 16;                  // columns (K-form: loads) of a lane
  static constexpr int kK = 16 / E::kSize;               // k of a lane
  static constexpr int kWords = kCols * E::kSize / 4;    // T-form: words of a lane's k-row
  uint32_t raw[T ? kK * kWords : kCols * 4];
  u32x4_t x[RT];

  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rw, __amdgpu_buffer_rsrc_t rx,
                                       const uint32_t (&woff)[T ? 1 : kCols], uint32_t ldw_bytes,
                                       const uint32_t (&xoff)[RT], bool in) {
    if constexpr (T) {
#pragma unroll
      for (int i = 0; i < kK; ++i) {
        const uint32_t o = in && woff[0] != kOob ? woff[0] + i * ldw_bytes : kOob;
        if constexpr (kWords == 1) {
          raw[i] = __builtin_amdgcn_raw_buffer_load_b32(rw, o, 0, 0);
        } else if constexpr (kWords == 2) {
          const u32x2_t v =
              __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(rw, o, 0, 0));
          raw[2 * i] = v.x;
          raw[2 * i + 1] = v.y;
        } else {
          const u32x4_t v = load16(rw, o);
#pragma unroll
          for (int q = 0; q < 4; ++q) raw[4 * i + q] = v[q];
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        const u32x4_t v = load16(rw, in ? woff[j] : kOob);
#pragma unroll
        for (int q = 0; q < 4; ++q) raw[4 * j + q] = v[q];
      }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) x[t] = load16(rx, in ? xoff[t] : kOob);
  }

  // acc[t][j][r]: row 16 t + 4 (lane / 16) + r, the lane's column of set j.
  __device__ __forceinline__ void multiply(f32x4 (&acc)[RT][kCols]) const {
    if constexpr (E::kSize == 2) {
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        u32x4_t b;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (T) {
            // column j of k-rows 2 q and 2 q + 1
            const uint32_t lo = raw[2 * q * kWords + j / 2], hi = raw[(2 * q + 1) * kWords + j / 2];
            b[q] = __builtin_amdgcn_perm(hi, lo, j & 1 ? 0x07060302u : 0x05040100u);
          } else {
            b[q] = raw[4 * j + q];
          }
        }
#pragma unroll
        for (int t = 0; t < RT; ++t)
          acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8_t, x[t]), __builtin_bit_cast(bf16x8_t, b), acc[t][j], 0, 0,
              0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kK; ++i)
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          const float b = __uint_as_float(T ? raw[i * kWords + j] : raw[4 * j + i]);
#pragma unroll
          for (int t = 0; t < RT; ++t)
            acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x[t][i]), b,
                                                             acc[t][j], 0, 0, 0);
        }
    }
  }
};

// Sums of slices travel between XCDs, whose L2s are not coherent with one another:
// they are written and read with device-scope cache policy (sc1).
constexpr int kDevice = 16;

// D: steps of a wave's batch; the next batch's loads are under way during one. A slice
// of k (EPI_PARTIAL aside) leaves its sums in part [column block][slice][M][CB] and
// counts itself in the block's arrival word, by an increment that wraps to zero at the
// last one, which adds the slices in order. No workgroup waits for another. That takes
// 2 to 2.8 us at the end of the launch (stores to the device-coherent level, the word,
// loads from there), about what a second launch takes the device (2.8 and the gap before
// it), and saves the host one: 2048 x 2048, one row, 8.2 -> 6.0 us a call.
template <typename E, bool T, int EPI, int RT, int CB, int NW, int D>
__global__ __launch_bounds__(NW * 64) void few_rows_kernel(GemmArgs p) {
  typedef Step<E, T, RT, CB> S;
  constexpr int kCols = S::kCols, kK = S::kK, kStep = 4 * kK;
  constexpr bool GATED = EPI == EPI_GATED;
  constexpr int OUT = GATED ? CB / 2 : CB;
  __shared__ __align__(16) float sums[NW][RT * 16][CB];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  // Each XCD (workgroup b % 8) takes a run of column blocks: T-form rows of a run
  // are shared cache lines.
  const int64_t n0 = (int64_t)xcd_run(blockIdx.x, p.tiles_n) * OUT;
  const int slice = blockIdx.y;
  const int64_t k0 = slice * p.kper, k1 = min(p.K, k0 + p.kper);

  // byte offsets from the step's first k: of the lane's k-rows (K-form: k) and
  // columns, of its rows of x
  uint32_t woff[T ? 1 : kCols], xoff[RT];
  const uint32_t ldw_bytes = (uint32_t)(p.ldb * E::kSize);
  // staged column s: for EPI_GATED the first half gates, then the ups
  auto source = [&](int s) -> int64_t {
    const int o = GATED ? s % OUT : s;
    return n0 + o >= p.N ? -1 : n0 + o + (GATED && s >= OUT ? p.N : 0);
  };
  if constexpr (T) {
    const int64_t n = source(c * kCols);
    woff[0] = n < 0 ? kOob : (uint32_t)(g * kK) * ldw_bytes + (uint32_t)((n - n0) * E::kSize);
  } else {
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      const int64_t n = source(16 * j + c);
      woff[j] = n < 0 ? kOob : (uint32_t)(n - n0) * ldw_bytes + g * 16;
    }
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int m = 16 * t + c;
    xoff[t] = m < p.M ? (uint32_t)(m * p.lda * E::kSize) + g * 16 : kOob;
  }
  const uint64_t wb = reinterpret_cast<uint64_t>(p.b) + (uint64_t)(T ? n0 : n0 * p.ldb) * E::kSize;
  const uint64_t xb = reinterpret_cast<uint64_t>(p.a);
  const uint64_t kbytes = T ? (uint64_t)p.ldb * E::kSize : E::kSize;

  f32x4 acc[RT][kCols] = {};
  S st[2][D];
  auto load = [&](int64_t k, S& s) {
    s.load(make_rsrc(wb + k * kbytes), make_rsrc(xb + k * E::kSize), woff, ldw_bytes, xoff,
           k + g * kK < k1);
  };
  // a wave's batch is D adjacent steps (whole cache lines along k), then the next
  // waves', so that the workgroup goes through k together
  constexpr int64_t kBatch = (int64_t)NW * D * kStep;
  const int64_t kw = k0 + wave * (D * kStep);
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (kw + d * kStep < k1) load(kw + d * kStep, st[0][d]);
  for (int64_t k = kw; k < k1; k += 2 * kBatch) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t kh = k + h * kBatch;
#pragma unroll
      for (int d = 0; d < D; ++d)
        if (kh + kBatch + d * kStep < k1) load(kh + kBatch + d * kStep, st[h ^ 1][d]);
#pragma unroll
      for (int d = 0; d < D; ++d)
        if (kh + d * kStep < k1) st[h][d].multiply(acc);
    }
  }
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float* row = &sums[wave][16 * t + 4 * g + r][0];
#pragma unroll
      for (int j = 0; j < kCols; ++j) row[T ? c * kCols + j : 16 * j + c] = acc[t][j][r];
    }
  __syncthreads();
  if constexpr (EPI != EPI_PARTIAL)
    if (p.splits > 1) {
      __shared__ uint32_t arrived;
      const int64_t block = n0 / OUT, slice_bytes = p.M * CB * 4;
      const auto part = make_rsrc(reinterpret_cast<uint64_t>(p.part) +
                                  (uint64_t)(block * p.splits * slice_bytes));
      for (int id = threadIdx.x; id < (int)p.M * (CB / 4); id += NW * 64) {
        const int m = id / (CB / 4), col = (id % (CB / 4)) * 4;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int w = 0; w < NW; ++w) v += *reinterpret_cast<const f32x4*>(&sums[w][m][col]);
        __builtin_amdgcn_raw_buffer_store_b128(
            __builtin_bit_cast(u32x4_t, v), part,
            (uint32_t)(slice * slice_bytes) + (m * CB + col) * 4, 0, kDevice);
      }
      wait_vmcnt<0>();  // this wave's sums are at the device-coherent level
      __syncthreads();
      if (threadIdx.x == 0)
        arrived = __builtin_amdgcn_atomic_inc32(p.words + block, (uint32_t)(p.splits - 1),
                                                __ATOMIC_RELAXED, "agent");
      __syncthreads();
      if (arrived != (uint32_t)(p.splits - 1)) return;
      for (int id = threadIdx.x; id < (int)p.M * (OUT / 4); id += NW * 64) {
        const int m = id / (OUT / 4), col = (id % (OUT / 4)) * 4;
        const int64_t n = n0 + col;
        if (n >= p.N) continue;
        float v[4] = {}, u[4] = {}, none[4] = {};
#pragma unroll 4
        for (int q = 0; q < p.splits; ++q) {
          const uint32_t at = (uint32_t)(q * slice_bytes) + (m * CB + col) * 4;
          const f32x4 a = __builtin_bit_cast(
              f32x4, __builtin_amdgcn_raw_buffer_load_b128(part, at, 0, kDevice));
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] += a[i];
          if constexpr (GATED) {
            const f32x4 b = __builtin_bit_cast(
                f32x4, __builtin_amdgcn_raw_buffer_load_b128(part, at + OUT * 4, 0, kDevice));
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] += b[i];
          }
        }
        EpiCols<EPI, 4> cols;
        epi_cols<EPI, 4>(p, n, cols);
        epi_row<E, EPI, 4>(p, cols, m, n, v, u, GateUp(), none, none);
      }
      return;
    }
  constexpr int kGroups = OUT / 4;
  for (int id = threadIdx.x; id < RT * 16 * kGroups; id += NW * 64) {
    const int m = id / kGroups, col = (id % kGroups) * 4;
    const int64_t n = n0 + col;
    if (m >= p.M || n >= p.N) continue;
    float v[4] = {}, u[4] = {}, none[4] = {};
#pragma unroll 4
    for (int w = 0; w < NW; ++w) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(&sums[w][m][col]);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += a[i];
      if constexpr (GATED) {
        const f32x4 b = *reinterpret_cast<const f32x4*>(&sums[w][m][OUT + col]);
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] += b[i];
      }
    }
    if constexpr (EPI == EPI_PARTIAL) {
      store_c<F32, 4>(p.part + ((int64_t)slice * p.M + m) * p.ldp, n, v);
    } else {
      EpiCols<EPI, 4> cols;
      epi_cols<EPI, 4>(p, n, cols);
      epi_row<E, EPI, 4>(p, cols, m, n, v, u, GateUp(), none, none);
    }
  }
}

template <typename E, bool T, int EPI, int RT, int CB>
int launch(GemmArgs p, hipStream_t s) {
  constexpr int NW = 8, D = RT == 4 ? 1 : 2;
  constexpr int OUT = EPI == EPI_GATED ? CB / 2 : CB;
  p.tiles_n = (int)((p.N + OUT - 1) / OUT);
  VMOE_LAUNCH((few_rows_kernel<E, T, EPI, RT, CB, NW, D>),
              dim3((uint32_t)p.tiles_n, (uint32_t)p.splits), dim3(NW * 64), 0, s, p);
  VMOE_CHECK_LAUNCH();
  return VMOE_OK;
}

template <typename E, bool T, int EPI>
int by_rows(const GemmArgs& p, int cols, hipStream_t s) {
  if constexpr (T && E::kSize == 2)
    if (cols == 64)
      return p.M <= 16   ? launch<E, T, EPI, 1, 64>(p, s)
             : p.M <= 32 ? launch<E, T, EPI, 2, 64>(p, s)
                         : launch<E, T, EPI, 4, 64>(p, s);
  return p.M <= 16   ? launch<E, T, EPI, 1, 32>(p, s)
         : p.M <= 32 ? launch<E, T, EPI, 2, 32>(p, s)
                     : launch<E, T, EPI, 4, 32>(p, s);
}

template <typename E, bool T>
int by_epi(Epi epi, const GemmArgs& p, int cols, hipStream_t s) {
  switch (epi) {
    case EPI_LINEAR: return by_rows<E, T, EPI_LINEAR>(p, cols, s);
    case EPI_GATED: return by_rows<E, T, EPI_GATED>(p, cols, s);
    case EPI_PARTIAL: return by_rows<E, T, EPI_PARTIAL>(p, cols, s);
    default: return VMOE_ERR_INVALID_ARG;
  }
}

}  // namespace

int gemm_few(int type, Form form, Epi epi, const GemmArgs& p, int cols, hipStream_t s) {
  if (type == VMOE_DENSE_F32)
    return form == FORM_KK ? by_epi<F32, false>(epi, p, cols, s)
                           : by_epi<F32, true>(epi, p, cols, s);
  return form == FORM_KK ? by_epi<Bf16, false>(epi, p, cols, s)
                         : by_epi<Bf16, true>(epi, p, cols, s);
}

}  // namespace dense
}  // namespace vmoe
