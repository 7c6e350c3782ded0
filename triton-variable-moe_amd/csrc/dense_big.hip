// Matrix products of the dense operators on 256 x 256 tiles (bf16), for products
// that fill the card with them.
//
// Eight waves in a 2 (m) x 4 (n) grid, 128 x 64 of the tile each, two waves a SIMD:
// wave w and wave w + 4, of the upper and the lower half of the tile. A stage of k
// (64) is four half-tiles of 16 KB: rows of A and columns of B in two halves, so
// that a wave's 128 x 64 is four products of 64 x 32, one a phase:
//
//   phase 0: read A0, B0   multiply A0 B0
//   phase 1: read B1       multiply A0 B1   fetch A0, B0 of the stage after next
//   phase 2: read A1       multiply A1 B1   fetch B1
//   phase 3:               multiply A1 B0   fetch A1
//
// A half-tile is free once all waves have read it into registers, in the phase
// after, so that two buffers (128 KB) give each DMA more than a stage of time. The
// two waves of a SIMD run half a phase apart: barriers part a phase into reading
// and multiplying, and the lower waves pass one barrier more before they begin.
//
// Long k: the matrix units bound it, 1.6 us a stage (16384 x 2048 with k 16384: 830 us,
// 1320 TFLOP/s; weight gradients 1240 to 1270; a plain tile loop of the same size 900).
// k 2048: the epilogue, 7 to 50 us in which the CU multiplies nothing (gated, 16384 x
// 8192, fp32 gates and ups kept: 1130 us, 970 TFLOP/s; its gradient, which reads them
// again, 1 GB: 790 to 810 us, 690 TFLOP/s; its epilogue spills 7 of 256 registers, 32
// bytes a lane). First workgroups started 20 to 40 us apart, so that the CUs' epilogues
// do not meet, took 8 % off the gradient and nothing off the others: open, for that
// epilogue alone.

#include "dense_launch.h"

namespace vmoe {
namespace dense {
namespace {

constexpr int kHalf = 16384;
enum { A0 = 0, A1 = 1, B0 = 2, B1 = 3 };

template <bool AT, bool BT, int EPI>
__global__ __launch_bounds__(512, 2) void big_kernel(GemmArgs p) {
  typedef Bf16 E;
  constexpr int OUT = EPI == EPI_GATED ? 128 : 256;  // output columns of the tile
  __shared__ __align__(1024) char lds_[8 * kHalf];
  lds_char* lds = (lds_char*)lds_;
  const Tile t = tile_of(p, blockIdx.x, kGroup256);
  const int64_t m0 = (int64_t)t.m * 256, n0 = (int64_t)t.n * OUT;
  int64_t k0, k1;
  tile_k(p, t, k0, k1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 2, wn = wave & 3;

  Stager<E, AT, 128, 8> sa[2];
  Stager<E, BT, 128, 8> sb[2];
  const char* a = static_cast<const char*>(p.a) + (AT ? k0 * p.lda + m0 : m0 * p.lda + k0) * 2;
  const char* b = static_cast<const char*>(p.b) + (BT ? k0 * p.ldb + n0 : n0 * p.ldb + k0) * 2;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    // half h: of each wave's 128 rows the h-th 64, of its 64 columns the h-th 32
    sa[h].init(a, p.lda, wave, [&](int r) -> int64_t {
      const int m = (r >> 6) * 128 + h * 64 + (r & 63);
      return m0 + m < p.M ? m : -1;
    });
    sb[h].init(b, p.ldb, wave, [&](int r) -> int64_t {
      if (EPI != EPI_GATED) {
        const int n = (r >> 5) * 64 + h * 32 + (r & 31);
        return n0 + n < p.N ? n : -1;
      }
      return n0 + r >= p.N ? -1 : h ? p.N + r : r;  // gates, ups
    });
  }
  const int nk = (int)((k1 - k0 + 63) / 64);
  const uint32_t dst = lds_addr(lds) + wave * 2048;
  // half-tile H of stage kt (past the last: zeros, so that the counts of DMAs in
  // flight stay the same)
  auto fetch = [&](int kt, auto H) {
    constexpr int h = decltype(H)::value;
    const int64_t left = k1 - k0 - (int64_t)kt * 64;
    const uint32_t to = dst + (kt & 1) * (4 * kHalf) + h * kHalf;
    if constexpr (h < 2) sa[h].issue(to, left);
    else sb[h - 2].issue(to, left);
  };
  std::integral_constant<int, A0> a0;
  std::integral_constant<int, A1> a1;
  std::integral_constant<int, B0> b0;
  std::integral_constant<int, B1> b1;

  f32x16_t acc[4][2] = {};
  bf16x8_t af[2][4], bf[2][4];
  auto read_a = [&](const lds_char* st) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) af[i][s] = frag<E, AT, 128>(st, wm * 64 + i * 32, s);
  };
  auto read_b = [&](const lds_char* st, bf16x8_t (&f)[4]) {
#pragma unroll
    for (int s = 0; s < 4; ++s) f[s] = frag<E, BT, 128>(st, wn * 32, s);
  };
  // reads done, and what the next phase reads has come: all but the newest N DMAs
  auto turn = [&](auto N) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if constexpr (decltype(N)::value >= 0) wait_vmcnt<decltype(N)::value>();
    __builtin_amdgcn_sched_barrier(0);
    bare_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  auto multiply = [&](int h, int j) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) acc[2 * h + i][j] = mma(af[i][s], bf[j][s], acc[2 * h + i][j]);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
    bare_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  std::integral_constant<int, -1> none;
  std::integral_constant<int, 10> w10;
  std::integral_constant<int, 12> w12;

  fetch(0, a0); fetch(0, b0); fetch(0, b1); fetch(0, a1);
  fetch(1, a0); fetch(1, b0); fetch(1, b1); fetch(1, a1);
  wait_vmcnt<12>();
  bare_barrier();
  if (wm == 1) bare_barrier();
  __builtin_amdgcn_sched_barrier(0);
  for (int kt = 0; kt < nk; ++kt) {
    const lds_char* st = lds + (kt & 1) * (4 * kHalf);
    read_a(st + A0 * kHalf);
    read_b(st + B0 * kHalf, bf[0]);
    turn(w10);
    multiply(0, 0);
    read_b(st + B1 * kHalf, bf[1]);
    fetch(kt + 2, a0);
    fetch(kt + 2, b0);
    turn(w12);
    multiply(0, 1);
    read_a(st + A1 * kHalf);
    fetch(kt + 2, b1);
    turn(none);
    multiply(1, 1);
    fetch(kt + 2, a1);
    turn(w12);
    multiply(1, 0);
  }
  wait_vmcnt<0>();
  if (wm == 0) bare_barrier();
  bare_barrier();  // every wave has read the last stage, no DMA is in flight
  if (t.slice >= 0)
    write_part<4, 2>(acc, tile_part<65536>(p, t) + wave * 8192);
  else
    write_tile<E, EPI, 4, 2>(p, acc, lds + wave * 8192, m0 + wm * 128,
                             n0 + wn * (EPI == EPI_GATED ? 32 : 64), (int64_t)t.m * 2 + wm);
}

template <bool AT, bool BT, int EPI>
int launch(const GemmArgs& p, hipStream_t s) {
  VMOE_LAUNCH((big_kernel<AT, BT, EPI>), dim3(workgroups(p)), dim3(512), 0, s, p);
  VMOE_CHECK_LAUNCH();
  return VMOE_OK;
}

template <bool AT, bool BT>
int by_epi(Epi epi, const GemmArgs& p, hipStream_t s) {
  if (epi == EPI_LINEAR) return launch<AT, BT, EPI_LINEAR>(p, s);
  if constexpr (!AT) {
    if (epi == EPI_GATED) return launch<AT, BT, EPI_GATED>(p, s);
    return launch<AT, BT, EPI_GATED_BWD>(p, s);
  }
  return VMOE_ERR_INVALID_ARG;
}

}  // namespace

int gemm_big(Form form, Epi epi, const GemmArgs& p, hipStream_t s) {
  switch (form) {
    case FORM_KK: return by_epi<false, false>(epi, p, s);
    case FORM_KT: return by_epi<false, true>(epi, p, s);
    default: return by_epi<true, true>(epi, p, s);
  }
}

}  // namespace dense
}  // namespace vmoe
