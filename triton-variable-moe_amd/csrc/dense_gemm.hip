// Matrix products of the dense operators on 128 x 128 and 64 x 64 tiles (bf16 and
// fp32), and what goes with them: the joining of tiles split along k, gradients
// through the activation, column sums.
//
// Tiles: four waves, each a quarter of the tile in 32 x 32 blocks, both operands
// by DMA into a ring of LDS stages of 128 bytes of k: two for 128 x 128, three for
// 64 x 64, so that a CU holds two and three workgroups and one's epilogue runs beside
// another's products. bf16 128: 0.95 us a stage of two workgroups (1150 TFLOP/s; 4099 x
// 2048 with k 4096 and the weight from memory 74 us with its split tiles, 930);
// fp32 128: 3.8 us (142 of 157 TFLOP/s), 64: 1.6 of three (125). Smaller products are
// bound by the start of a launch (5 us), the epilogue and what is left of the last
// round of tiles.

#include "dense_launch.h"

namespace vmoe {
namespace dense {
namespace {

template <typename E, bool AT, bool BT, int EPI, int BM, int BN, int ST>
__global__ __launch_bounds__(256, 2) void gemm_kernel(GemmArgs p) {
  constexpr int WM = 2, WN = 2, NW = WM * WN;
  constexpr int FM = BM / 32 / WM, FN = BN / 32 / WN;
  constexpr int A_BYTES = BM * 128, STAGE = (BM + BN) * 128;
  constexpr int OUT = EPI == EPI_GATED ? BN / 2 : BN;  // output columns of the tile
  __shared__ __align__(1024) char lds_[ST * STAGE];
  lds_char* lds = (lds_char*)lds_;
  static_assert(NW * 32 * 32 * FN * 4 <= ST * STAGE, "epilogue scratch");
  const Tile t = tile_of(p, blockIdx.x, kGroup);
  const int64_t m0 = (int64_t)t.m * BM, n0 = (int64_t)t.n * OUT;
  int64_t k0, k1;
  tile_k(p, t, k0, k1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;

  Stager<E, AT, BM, NW> sa;
  Stager<E, BT, BN, NW> sb;
  const char* a = static_cast<const char*>(p.a) +
                  (AT ? k0 * p.lda + m0 : m0 * p.lda + k0) * E::kSize;
  const char* b = static_cast<const char*>(p.b) +
                  (BT ? k0 * p.ldb + n0 : n0 * p.ldb + k0) * E::kSize;
  sa.init(a, p.lda, wave, [&](int r) -> int64_t { return m0 + r < p.M ? r : -1; });
  sb.init(b, p.ldb, wave, [&](int r) -> int64_t {
    if (EPI != EPI_GATED) return n0 + r < p.N ? r : -1;
    // staged: for each wave column 32 gates, then the ups of the same outputs
    const int o = (r >> 6) * 32 + (r & 31);
    return n0 + o >= p.N ? -1 : ((r >> 5) & 1) ? p.N + o : o;
  });

  const int nk = (int)((k1 - k0 + kStageK<E> - 1) / kStageK<E>);
  constexpr int PER = Stager<E, AT, BM, NW>::kInsts + Stager<E, BT, BN, NW>::kInsts;
  const uint32_t la = lds_addr(lds) + wave * (Stager<E, AT, BM, NW>::kInsts * 1024);
  const uint32_t lb = lds_addr(lds) + A_BYTES + wave * (Stager<E, BT, BN, NW>::kInsts * 1024);
  auto issue = [&](int kt) {
    const int64_t left = k1 - k0 - (int64_t)kt * kStageK<E>;
    sa.issue(la + (kt % ST) * STAGE, left);
    sb.issue(lb + (kt % ST) * STAGE, left);
  };
  f32x16_t acc[FM][FN] = {};
#pragma unroll
  for (int s = 0; s < ST - 1; ++s)
    if (s < nk) issue(s);
  for (int kt = 0; kt < nk; ++kt) {
    if (kt + ST - 2 < nk) wait_vmcnt<(ST - 2) * PER>();
    else wait_vmcnt<0>();
    block_barrier();
    if (kt + ST - 1 < nk) issue(kt + ST - 1);
    const lds_char* st = lds + (kt % ST) * STAGE;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      typename E::Frag af[FM], bf[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) af[i] = frag<E, AT, BM>(st, (wm * FM + i) * 32, s);
#pragma unroll
      for (int j = 0; j < FN; ++j) bf[j] = frag<E, BT, BN>(st + A_BYTES, (wn * FN + j) * 32, s);
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mma(af[i], bf[j], acc[i][j]);
    }
  }
  if (t.slice >= 0) {
    write_part<FM, FN>(acc, tile_part<BM * BN>(p, t) + wave * (BM * BN / NW));
    return;
  }
  block_barrier();  // every wave has read the last stages
  write_tile<E, EPI, FM, FN>(p, acc, lds + wave * (32 * 32 * FN * 4), m0 + wm * 32 * FM,
                             n0 + wn * (EPI == EPI_GATED ? 32 : 32 * FN), (int64_t)t.m * WM + wm);
}

template <typename E, bool AT, bool BT, int EPI, int BM, int BN, int ST>
int launch_tile(const GemmArgs& p, hipStream_t s) {
  VMOE_LAUNCH((gemm_kernel<E, AT, BT, EPI, BM, BN, ST>), dim3(workgroups(p)), dim3(256), 0, s, p);
  VMOE_CHECK_LAUNCH();
  return VMOE_OK;
}

template <typename E, bool AT, bool BT, int EPI>
int launch_form(const GemmArgs& p, Tiles tiles, hipStream_t s) {
  if constexpr (EPI != EPI_GATED) {
    if (tiles == TILES_64) return launch_tile<E, AT, BT, EPI, 64, 64, 3>(p, s);
  } else {
    if (tiles == TILES_64) return launch_tile<E, AT, BT, EPI, 64, 128, 2>(p, s);
  }
  return launch_tile<E, AT, BT, EPI, 128, 128, 2>(p, s);
}

// ---------------------------------------------------------------------------
// Split tiles: the sums of their slices, in order, through the epilogue. Waves of the
// product in WM x WN, FM x FN blocks of 32 x 32 each. A workgroup takes one wave's
// row of FN blocks (EPI_GATED_BWD, for its column sums: all FM of them): they are read as they lie (see write_part; a wave of
// the workgroup one register group, the next row while this one is worked on), turned
// in LDS, and written as rows: 64 columns in one piece (EPI_GATED: 32), where lanes
// that kept their values would write 32 pieces of 4 columns (128 tiles of 256 x 256 in
// two slices with a residual: 31 -> 22 us, 4.5 TB/s; 256 of 128 x 128 in two 10).
template <typename E, int EPI, int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(256) void join_kernel(GemmArgs p, int gm) {
  constexpr bool GATED = EPI == EPI_GATED, BWD = EPI == EPI_GATED_BWD;
  constexpr int NW = WM * WN, VALUES = NW * FM * FN * 1024;
  constexpr int COLS = 32 * FN, OUT = GATED ? 32 : COLS;  // staged and output columns
  constexpr int PITCH = COLS + 4;                         // (banks: 16 bytes off a row)
  constexpr int LR = OUT / 4, RP = 256 / LR;              // threads of a row, rows at a time
  __shared__ __align__(16) float turn[2][32 * PITCH];
  const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
  constexpr int PER = BWD ? FM : 1;  // rows of blocks of a workgroup
  const int first = blockIdx.x % (FM / PER) * PER, unit = blockIdx.x / (FM / PER);
  const int wave = unit % NW, split = unit / NW;
  const Tile t = tile_at(p, p.whole + split, gm);
  const int wm = wave / WN, wn = wave % WN;
  const int64_t m0 = ((int64_t)t.m * WM + wm) * 32 * FM;
  const int64_t n0 = ((int64_t)t.n * WN + wn) * OUT;
  if (m0 + 32 * first >= p.M || n0 >= p.N) return;
  const int c = (threadIdx.x % LR) * 4;
  const int64_t n = n0 + c;
  const bool n_ok = n < p.N;
  const int64_t step = (int64_t)(p.tiles_m * p.tiles_n - p.whole) * VALUES;
  const float* part = p.part + (int64_t)split * VALUES + (wave * FM * FN * 4 + g) * 256 + lane * 4;
  EpiCols<EPI, 4> cols;
  epi_cols<EPI, 4>(p, n, cols);
  float sg[4] = {}, su[4] = {};
  f32x4_t sum[FN];
  auto read = [&](int i) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
      sum[j] = *reinterpret_cast<const f32x4_t*>(part + (i * FN + j) * 1024);
#pragma unroll 8
    for (int s = 1; s < p.splits; ++s)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        sum[j] += *reinterpret_cast<const f32x4_t*>(part + s * step + (i * FN + j) * 1024);
  };
  read(first);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = first + k;
    float* buf = turn[k & 1];
#pragma unroll
    for (int j = 0; j < FN; ++j)
      *reinterpret_cast<f32x4_t*>(buf + (lane & 31) * PITCH + 32 * j + 8 * g + 4 * (lane >> 5)) =
          sum[j];
    if (k + 1 < PER) read(i + 1);
    __syncthreads();
#pragma unroll
    for (int r = threadIdx.x / LR; r < 32; r += RP) {
      const int64_t m = m0 + 32 * i + r;
      if (m >= p.M || !n_ok) continue;
      float v[4], u[4] = {};
      const f32x4_t a = *reinterpret_cast<const f32x4_t*>(buf + r * PITCH + c);
      const f32x4_t b = *reinterpret_cast<const f32x4_t*>(buf + r * PITCH + (GATED ? 32 : 0) + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = a[e];
        u[e] = b[e];
      }
      GateUp z = {};
      if constexpr (BWD) z = load_z(p, m, n);
      epi_row<E, EPI, 4>(p, cols, m, n, v, u, z, sg, su);
    }
  }
  if constexpr (BWD) {
    if (p.sums) {
      // threads of the same columns, in order
      __shared__ __align__(16) float part_sums[2][RP][OUT];
      const int r = threadIdx.x / LR;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        part_sums[0][r][c + e] = sg[e];
        part_sums[1][r][c + e] = su[e];
      }
      __syncthreads();
      for (int id = threadIdx.x; id < 2 * OUT; id += 256) {
        const int q = id / OUT, col = id % OUT;
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < RP; ++i) total += part_sums[q][i][col];
        if (n0 + col < p.N)
          p.sums[((int64_t)t.m * WM + wm) * 2 * p.N + q * p.N + n0 + col] = total;
      }
    }
  }
}

// The same for the sums of dense_few.hip, [splits, M, ldp] (EPI_GATED: gates, then
// ups). 2.5 to 3.7 us, most of it the launch.
template <typename E, int EPI>
__global__ __launch_bounds__(128) void join_rows_kernel(GemmArgs p) {
  const int64_t groups = p.N / 4;
  const int64_t id = (int64_t)blockIdx.x * 128 + threadIdx.x;
  if (id >= p.M * groups) return;
  const int64_t m = id / groups, n = (id - m * groups) * 4;
  EpiCols<EPI, 4> cols;
  epi_cols<EPI, 4>(p, n, cols);
  float v[4] = {}, u[4] = {}, none[4] = {};
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float* row = p.part + ((int64_t)s * p.M + m) * p.ldp;
    float x[4];
    load_c<F32, 4>(row, n, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += x[i];
    if constexpr (EPI == EPI_GATED) {
      load_c<F32, 4>(row, p.N + n, x);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] += x[i];
    }
  }
  epi_row<E, EPI, 4>(p, cols, m, n, v, u, GateUp(), none, none);
}

// dz = gy * act'(z), rounded, and the column sums of what it stores before
// rounding: a workgroup takes `per` rows of 256 columns, part its row of them. Where
// the output y says what the slope is (relu: y > 0), z is not kept: 8192 x 4096 in bf16
// the forward pass writes 134 MB less (118 -> 98 us), and this one reads 67 MB of y in
// place of 134 of z (55 -> 37 us, 5.4 TB/s). The same for relu squared, 2 sqrt(y) of the rounded y,
// took the weight's gradient from 2.3e-3 to 2.5e-3 off float64: not done. Fewer rows a workgroup where rows are few: 2051 x 2048 in
// fp32 19 -> 10 us.
enum SlopeOf { SLOPE_NONE, SLOPE_Z, SLOPE_Y };
template <typename E, SlopeOf FROM>
__global__ __launch_bounds__(256) void act_grad_kernel(const void* gy, int64_t ldgy,
                                                       const void* z, int64_t ldz, int act,
                                                       void* dz, int64_t lddz, float* part,
                                                       int64_t M, int64_t N, int per, int past) {
  __shared__ float red[4][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n = (int64_t)blockIdx.x * 256 + lane * 4;
  const int64_t m0 = (int64_t)blockIdx.y * per;
  float sum[4] = {};
  if (n < N) {
    const int64_t m1 = min(M, m0 + per);
#pragma unroll 4
    for (int64_t m = m0 + wave; m < m1; m += 4) {
      float g[4];
      load_c<E, 4>(static_cast<const typename E::Store*>(gy) + m * ldgy, n, g);
      if constexpr (FROM == SLOPE_Z) {
        const f32x4_t x = load_z4(static_cast<const float*>(z) + m * ldz + n, past);
        act_switch(act, [&](auto A) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float slope;
            act1<decltype(A)::value, true>(x[i], slope);
            g[i] *= slope;
          }
        });
      } else if constexpr (FROM == SLOPE_Y) {
        float y[4];
        load_c<E, 4>(static_cast<const typename E::Store*>(z) + m * ldz, n, y);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          g[i] *= y[i] > 0.0f ? 1.0f : y[i];
      }
      if constexpr (FROM != SLOPE_NONE)
        store_c<E, 4>(static_cast<typename E::Store*>(dz) + m * lddz, n, g);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += g[i];
    }
  }
  if (!part) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) red[wave][lane * 4 + i] = sum[i];
  __syncthreads();
  const int c = threadIdx.x;
  const int64_t col = (int64_t)blockIdx.x * 256 + c;
  if (col < N)
    part[(int64_t)blockIdx.y * N + col] = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
}

// Column sums of part [rows, N], the first `split` columns into out0, the others
// into out1 (bf16 or fp32; null: not wanted): 16 columns a workgroup, 16 threads a
// column, 8 loads of each under way. 1024 rows of 4096: 6.6 us, 2.5 TB/s; 64 rows: 3 to
// 5 us, the launch and one round of loads.
__global__ __launch_bounds__(256) void col_sum_kernel(const float* part, int64_t rows, int64_t N,
                                                      int64_t split, void* out0, int out0_f32,
                                                      void* out1, int out1_f32) {
  __shared__ float red[16][17];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  const int64_t n = (int64_t)blockIdx.x * 16 + c;
  float s[8] = {};
  if (n < N) {
    int64_t m = r;
    for (; m + 112 < rows; m += 128)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += part[(m + 16 * i) * N + n];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (m + 16 * i < rows) s[i] += part[(m + 16 * i) * N + n];
  }
  red[r][c] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  if (r == 0 && n < N) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += red[i][c];
    void* out = n < split ? out0 : out1;
    const int f32 = n < split ? out0_f32 : out1_f32;
    const int64_t at = n < split ? n : n - split;
    if (out && f32) static_cast<float*>(out)[at] = t;
    else if (out) static_cast<uint16_t*>(out)[at] = (uint16_t)f32_to_bf16(t);
  }
}

}  // namespace

int gemm_tiles(int type, Form form, Epi epi, const GemmArgs& p, Tiles tiles, hipStream_t s) {
  if (tiles == TILES_256) return gemm_big(form, epi, p, s);
  auto go = [&](auto e, auto f) -> int {
    typedef decltype(e) E;
    constexpr int F = decltype(f)::value;
    constexpr bool AT = F == FORM_TT, BT = F != FORM_KK;
    if (epi == EPI_LINEAR) return launch_form<E, AT, BT, EPI_LINEAR>(p, tiles, s);
    if constexpr (!AT) {
      if (epi == EPI_GATED) return launch_form<E, AT, BT, EPI_GATED>(p, tiles, s);
      if (epi == EPI_GATED_BWD) return launch_form<E, AT, BT, EPI_GATED_BWD>(p, tiles, s);
    }
    return VMOE_ERR_INVALID_ARG;
  };
  auto by_form = [&](auto e) -> int {
    switch (form) {
      case FORM_KK: return go(e, std::integral_constant<int, FORM_KK>());
      case FORM_KT: return go(e, std::integral_constant<int, FORM_KT>());
      default: return go(e, std::integral_constant<int, FORM_TT>());
    }
  };
  return type == VMOE_DENSE_F32 ? by_form(F32()) : by_form(Bf16());
}

namespace {
template <typename E, int EPI, int WM, int WN, int FM, int FN>
int launch_join(const GemmArgs& p, int gm, hipStream_t s) {
  const int rest = p.tiles_m * p.tiles_n - p.whole;
  const int blocks = rest * WM * WN * (EPI == EPI_GATED_BWD ? 1 : FM);
  VMOE_LAUNCH((join_kernel<E, EPI, WM, WN, FM, FN>), dim3((uint32_t)blocks), dim3(256), 0, s, p,
              gm);
  VMOE_CHECK_LAUNCH();
  return VMOE_OK;
}
template <typename E, int EPI>
int join_epi(const GemmArgs& p, Tiles tiles, hipStream_t s) {
  if constexpr (E::kSize == 2)
    if (tiles == TILES_256) return launch_join<E, EPI, 2, 4, 4, 2>(p, kGroup256, s);
  if (tiles == TILES_128) return launch_join<E, EPI, 2, 2, 2, 2>(p, kGroup, s);
  return launch_join<E, EPI, 2, 2, 1, EPI == EPI_GATED ? 2 : 1>(p, kGroup, s);
}
}  // namespace

int join_tiles(int type, Epi epi, const GemmArgs& p, Tiles tiles, hipStream_t s) {
  auto go = [&](auto e) -> int {
    typedef decltype(e) E;
    if (epi == EPI_LINEAR) return join_epi<E, EPI_LINEAR>(p, tiles, s);
    if (epi == EPI_GATED) return join_epi<E, EPI_GATED>(p, tiles, s);
    return join_epi<E, EPI_GATED_BWD>(p, tiles, s);
  };
  return type == VMOE_DENSE_F32 ? go(F32()) : go(Bf16());
}

int join_rows(int type, Epi epi, const GemmArgs& p, hipStream_t s) {
  const dim3 grid((uint32_t)((p.M * (p.N / 4) + 127) / 128));
  auto go = [&](auto e) {
    typedef decltype(e) E;
    if (epi == EPI_LINEAR)
      VMOE_LAUNCH((join_rows_kernel<E, EPI_LINEAR>), grid, dim3(128), 0, s, p);
    else
      VMOE_LAUNCH((join_rows_kernel<E, EPI_GATED>), grid, dim3(128), 0, s, p);
  };
  if (type == VMOE_DENSE_F32) go(F32());
  else go(Bf16());
  VMOE_CHECK_LAUNCH();
  return VMOE_OK;
}

// Rows of a workgroup of act_grad: 64, fewer where that leaves the card short of
// workgroups.
static int act_grad_rows(int64_t M, int64_t N) {
  const int64_t cols = (N + 255) / 256;
  int per = 64;
  while (per > 16 && (M + per - 1) / per * cols < 2048) per /= 2;
  while ((M + per - 1) / per > 32768) per *= 2;  // (a grid's second dimension)
  return per;
}
int64_t sum_rows(int64_t M, int64_t N) {
  const int per = act_grad_rows(M, N);
  return (M + per - 1) / per;
}

int act_grad(int type, const void* gy, int64_t ldgy, const float* z, int64_t ldz, const void* y,
             int64_t ldy, int act, void* dz, int64_t lddz, float* part, int64_t M, int64_t N,
             hipStream_t s) {
  const dim3 grid((uint32_t)((N + 255) / 256), (uint32_t)sum_rows(M, N));
  const int per = act_grad_rows(M, N), past = z_past(M, N);
  auto go = [&](auto e) {
    typedef decltype(e) E;
    if (z)
      VMOE_LAUNCH((act_grad_kernel<E, SLOPE_Z>), grid, dim3(256), 0, s, gy, ldgy, z, ldz, act, dz,
                  lddz, part, M, N, per, past);
    else if (y)
      VMOE_LAUNCH((act_grad_kernel<E, SLOPE_Y>), grid, dim3(256), 0, s, gy, ldgy, y, ldy, act, dz,
                  lddz, part, M, N, per, past);
    else
      VMOE_LAUNCH((act_grad_kernel<E, SLOPE_NONE>), grid, dim3(256), 0, s, gy, ldgy, z, ldz, act,
                  dz, lddz, part, M, N, per, past);
  };
  if (type == VMOE_DENSE_F32) go(F32());
  else go(Bf16());
  VMOE_CHECK_LAUNCH();
  return VMOE_OK;
}

int col_sum(const float* part, int64_t rows, int64_t N, int64_t split, void* out0, int out0_f32,
            void* out1, int out1_f32, hipStream_t s) {
  VMOE_LAUNCH(col_sum_kernel, dim3((uint32_t)((N + 15) / 16)), dim3(256), 0, s, part, rows, N,
              split, out0, out0_f32, out1, out1_f32);
  VMOE_CHECK_LAUNCH();
  return VMOE_OK;
}

}  // namespace dense
}  // namespace vmoe
