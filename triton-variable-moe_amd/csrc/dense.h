// Shared parts of the dense operators (fused linear, gated block): arguments,
// activations, operand staging and epilogues of their matrix products.
//
//   linear:  y = act(x w + b) + r
//   gated:   z = x [wg | wu] + b1, h = act(zg) * zu, y = h w2 + b2 + r
//
// Every product is C(m, n) = sum_k A(m, k) B(k, n) with operands in one of two
// forms: "K-form", contiguous along k (rows of x, gradients, a weight stored
// [out, in]), and "T-form", contiguous along m or n (a weight stored [in, out];
// both operands of a weight gradient). Sums are fp32; an output is rounded once,
// after bias, activation and residual.
#pragma once

#include <type_traits>

#include "vmoe_common.h"

namespace vmoe {
namespace dense {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) bf16x4_t lds_bf16x4;
typedef __attribute__((address_space(3))) f32x4_t lds_f32x4;
typedef __attribute__((address_space(3))) float lds_float;

struct Bf16 {
  static constexpr int kSize = 2;
  typedef uint16_t Store;
  typedef bf16x8_t Frag;  // 16 bytes of a lane: 8 k
};
struct F32 {
  static constexpr int kSize = 4;
  typedef float Store;
  typedef f32x4_t Frag;  // 16 bytes of a lane: 4 k
};

// What a product's results go through (see epi_row).
enum Epi {
  EPI_LINEAR,    // act(acc + bias) + residual; acc + bias kept in z
  EPI_GATED,     // act(gate + bias) * (up + bias); gate and up kept in z
  EPI_GATED_BWD, // acc is dh: [dgate | dup] from z, with their column sums
  EPI_PARTIAL,   // the fp32 sums of one slice of k (dense_few.hip)
};

constexpr int kGroup256 = 8, kGroup = 16;  // row tiles of a group (see tile_of)

struct GemmArgs {
  const void* a;
  const void* b;
  int64_t lda, ldb;   // elements
  int64_t M, N, K;    // N: output columns (gated: the width)
  const void* bias;   // [N] ([2 N] gated), or null
  int32_t bias_f32;
  const void* res;    // residual [M, ldr], or null
  int64_t ldr;
  void* c;            // output [M, ldc]
  int64_t ldc;
  float* z;           // fp32 pre-activations [M, ldz] (written; EPI_GATED_BWD: read), or null
  int64_t ldz;
  int32_t z_past;     // z goes past the caches
  float* sums;        // EPI_GATED_BWD: column sums [row blocks, 2 N], or null
  int32_t act;
  int32_t tiles_m, tiles_n;
  // The first `whole` tiles are one workgroup's; each of the others is `splits`
  // workgroups', which take kper of k (a multiple of the kernel's stage) and leave
  // their sums in part.
  int32_t whole, splits;
  int64_t kper;
  float* part;        // dense_few.hip: [splits, M, ldp] (words: its own); tiles: see write_part
  int64_t ldp;
  uint32_t* words;    // dense_few.hip: arrival words, or null
};

__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.0f + expf(-x));
}

// The activation of z and, where SLOPE, its derivative. NaN stays NaN.
template <int ACT, bool SLOPE>
__device__ __forceinline__ float act1(float z, float& slope) {
  if constexpr (ACT == VMOE_DENSE_RELU) {
    if (SLOPE) slope = z > 0.0f ? 1.0f : z <= 0.0f ? 0.0f : z;
    return z < 0.0f ? 0.0f : z;
  } else if constexpr (ACT == VMOE_DENSE_RELU_SQUARED) {
    const float r = z < 0.0f ? 0.0f : z;
    if (SLOPE) slope = 2.0f * r;
    return r * r;
  } else if constexpr (ACT == VMOE_DENSE_SILU) {
    const float s = sigmoid(z);
    if (SLOPE) slope = s * (1.0f + z * (1.0f - s));
    return z * s;
  } else if constexpr (ACT == VMOE_DENSE_GELU) {
    const float phi = 0.5f * (1.0f + erff(z * 0.70710678118654752f));
    if (SLOPE) slope = phi + z * expf(-0.5f * z * z) * 0.39894228040143268f;
    return z * phi;
  } else if constexpr (ACT == VMOE_DENSE_GELU_TANH) {
    // (1 + tanh v) / 2 = sigmoid(2 v), v = sqrt(2 / pi) (z + 0.044715 z^3)
    const float s = sigmoid(1.5957691216057308f * (z + 0.044715f * z * z * z));
    if (SLOPE) {
      // (z^2 must not overflow: beyond 64 s (1 - s) is 0)
      const float c = fminf(fabsf(z), 64.0f);
      slope = s + z * (s * (1.0f - s)) * (1.5957691216057308f * (1.0f + 0.134145f * c * c));
    }
    return z * s;
  } else {
    if (SLOPE) slope = 1.0f;
    return z;
  }
}

// f(ACT constant) for the uniform runtime value act.
template <typename F>
__device__ __forceinline__ void act_switch(int act, F&& f) {
  switch (act) {
    case VMOE_DENSE_RELU: f(std::integral_constant<int, VMOE_DENSE_RELU>()); break;
    case VMOE_DENSE_RELU_SQUARED: f(std::integral_constant<int, VMOE_DENSE_RELU_SQUARED>()); break;
    case VMOE_DENSE_SILU: f(std::integral_constant<int, VMOE_DENSE_SILU>()); break;
    case VMOE_DENSE_GELU: f(std::integral_constant<int, VMOE_DENSE_GELU>()); break;
    case VMOE_DENSE_GELU_TANH: f(std::integral_constant<int, VMOE_DENSE_GELU_TANH>()); break;
    default: f(std::integral_constant<int, VMOE_DENSE_NONE>()); break;
  }
}

// C consecutive values of a row, 4 or 8 (8: bf16 alone). n is a multiple of C, rows
// are 16-byte aligned.
template <typename E, int C>
__device__ __forceinline__ void load_c(const void* row, int64_t n, float (&v)[C]) {
  if constexpr (E::kSize == 4) {
    static_assert(C == 4, "16 bytes");
    const f32x4_t w = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(row) + n);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = w[i];
  } else {
    typedef uint32_t words __attribute__((ext_vector_type(C / 2)));
    const words w = *reinterpret_cast<const words*>(static_cast<const uint16_t*>(row) + n);
#pragma unroll
    for (int i = 0; i < C / 2; ++i) {
      v[2 * i] = lo_f32(w[i]);
      v[2 * i + 1] = hi_f32(w[i]);
    }
  }
}

template <typename E, int C>
__device__ __forceinline__ void store_c(void* row, int64_t n, const float (&v)[C]) {
  if constexpr (E::kSize == 4) {
    static_assert(C == 4, "16 bytes");
    const f32x4_t w = {v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4_t*>(static_cast<float*>(row) + n) = w;
  } else {
    typedef uint32_t words __attribute__((ext_vector_type(C / 2)));
    words w;
#pragma unroll
    for (int i = 0; i < C / 2; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<words*>(static_cast<uint16_t*>(row) + n) = w;
  }
}

// 4 pre-activations kept for the backward pass; `past` (see kPastCache): past the caches.
__device__ __forceinline__ f32x4_t load_z4(const float* p, int past) {
  const f32x4_t* q = reinterpret_cast<const f32x4_t*>(p);
  if (!past) return *q;
  // (the two asm statements keep the compiler from merging the branches, which would
  // lose the hint)
  asm volatile("");
  const f32x4_t v = __builtin_nontemporal_load(q);
  asm volatile("");
  return v;
}
__device__ __forceinline__ void store_z4(float* p, int past, const float (&v)[4]) {
  const f32x4_t w = {v[0], v[1], v[2], v[3]};
  f32x4_t* q = reinterpret_cast<f32x4_t*>(p);
  if (past) {
    asm volatile("");
    __builtin_nontemporal_store(w, q);
    asm volatile("");
  } else {
    *q = w;
  }
}

// C values of the bias from column n on (its address may be any multiple of its
// type's size: a slice of a longer vector).
template <int C>
__device__ __forceinline__ void bias_c(const void* bias, int f32, int64_t n, float (&v)[C]) {
#pragma unroll
  for (int i = 0; i < C; ++i)
    v[i] = f32 ? static_cast<const float*>(bias)[n + i]
               : bf16_to_f32(static_cast<const uint16_t*>(bias)[n + i]);
}

// Columns of a row that a thread takes in an epilogue: 16 bytes of its widest
// buffer (the fp32 sums, pre-activations or outputs where there are any).
template <typename E, int EPI>
constexpr int kEpiCols = E::kSize == 2 && EPI == EPI_LINEAR ? 8 : 4;

// What is the same for every row of C columns: their bias.
template <int EPI, int C>
struct EpiCols {
  float b[C], b2[C];
};
template <int EPI, int C>
__device__ __forceinline__ void epi_cols(const GemmArgs& p, int64_t n, EpiCols<EPI, C>& q) {
  if constexpr (EPI == EPI_LINEAR || EPI == EPI_GATED) {
#pragma unroll
    for (int i = 0; i < C; ++i) q.b[i] = q.b2[i] = 0.0f;
    if (p.bias && n < p.N) {
      bias_c<C>(p.bias, p.bias_f32, n, q.b);
      if (EPI == EPI_GATED) bias_c<C>(p.bias, p.bias_f32, p.N + n, q.b2);
    }
  }
}

// EPI_GATED_BWD: the gates and ups of row m, columns n .. n + 3.
struct GateUp {
  f32x4_t g, u;
};
__device__ __forceinline__ GateUp load_z(const GemmArgs& p, int64_t m, int64_t n) {
  GateUp q;
  q.g = load_z4(p.z + m * p.ldz + n, p.z_past);
  q.u = load_z4(p.z + m * p.ldz + p.N + n, p.z_past);
  return q;
}

// Row m, columns n .. n + C - 1 (the caller has checked m < M and n < N): v are the
// sums, u the up half's for EPI_GATED. Pre-activations are stored too, if wanted (of 8
// columns by write_tile, 4 columns a lane). EPI_GATED_BWD adds what it stores, before
// rounding, to sg and su (this thread's columns of the bias gradient).
template <typename E, int EPI, int C>
__device__ __forceinline__ void epi_row(const GemmArgs& p, const EpiCols<EPI, C>& q, int64_t m,
                                        int64_t n, float (&v)[C], float (&u)[C],
                                        const GateUp& z, float (&sg)[C], float (&su)[C]) {
  typename E::Store* c = static_cast<typename E::Store*>(p.c) + m * p.ldc;
  float unused;
  if constexpr (EPI == EPI_LINEAR) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] += q.b[i];
    if constexpr (C == 4)
      if (p.z) store_z4(p.z + m * p.ldz + n, p.z_past, v);
    act_switch(p.act, [&](auto A) {
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] = act1<decltype(A)::value, false>(v[i], unused);
    });
    if (p.res) {
      float r[C];
      load_c<E, C>(static_cast<const typename E::Store*>(p.res) + m * p.ldr, n, r);
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] += r[i];
    }
    store_c<E, C>(c, n, v);
  } else if constexpr (EPI == EPI_GATED) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      v[i] += q.b[i];
      u[i] += q.b2[i];
    }
    if (p.z) {
      store_z4(p.z + m * p.ldz + n, p.z_past, v);
      store_z4(p.z + m * p.ldz + p.N + n, p.z_past, u);
    }
    act_switch(p.act, [&](auto A) {
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] = act1<decltype(A)::value, false>(v[i], unused) * u[i];
    });
    store_c<E, C>(c, n, v);
  } else if constexpr (EPI == EPI_GATED_BWD) {
    float g[C], up[C];
    act_switch(p.act, [&](auto A) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        float slope;
        const float a = act1<decltype(A)::value, true>(z.g[i], slope);
        g[i] = v[i] * z.u[i] * slope;
        up[i] = v[i] * a;
      }
    });
#pragma unroll
    for (int i = 0; i < C; ++i) {
      sg[i] += g[i];
      su[i] += up[i];
    }
    store_c<E, C>(c, n, g);
    store_c<E, C>(c + p.N, n, up);
  }
}

// ---------------------------------------------------------------------------
// Staging: operand tiles go from memory to LDS by DMA, 16 bytes a lane.

constexpr uint32_t kOob = 0x80000000u;  // an offset past every resource: reads zeros

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Barrier without the fences of __syncthreads(), which would wait for every DMA
// in flight: those are waited for with wait_vmcnt. The caller has no LDS read in flight.
__device__ __forceinline__ void bare_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// The same where there may be LDS reads: another wave's DMA may write after the barrier
// what they read, and the matrix instructions that use them may come later.
__device__ __forceinline__ void block_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  bare_barrier();
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(uint64_t a) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), 0,
                                           0x7FFFFFFF, 0x00020000);
}

// (inline asm, so that the compiler does not wait for the DMA before every LDS
// read; no register output, M0 declared clobbered. A load to LDS may read M0 one wait
// state after its write at the earliest: s_nop, as the compiler puts it)
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               ::"v"(voff), "s"(r), "s"(lds) : "memory", "m0");
}

__device__ __forceinline__ uint32_t lds_addr(const lds_char* p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)reinterpret_cast<uintptr_t>(p));
}

// A stage holds 128 bytes of k in K-form (64 bf16, 32 fp32), as many k-rows in
// T-form.
template <typename E>
constexpr int kStageK = 128 / E::kSize;

// The 16-byte chunk a staged chunk c of row r is kept at is c ^ swz(r). K-form
// rows are 8 chunks; the 16 rows that one phase of a ds_read_b128 covers share
// 256-byte bank lines two by two, so (r / 2) % 8 spreads them. T-form rows of R
// values: a transposing read of bf16 takes k-rows k .. k + 3 at two columns 16
// apart, and k + 8 ...; a 4-byte read of fp32 takes rows k and k + 4.
template <typename E, bool T, int R>
__device__ __forceinline__ int swz(int r) {
  if (!T) return (r >> 1) & 7;
  if (E::kSize == 4) return ((r >> 2) & 1) << 3;
  return R >= 128 ? ((r & 3) << 2) | (((r >> 3) & 1) << 1)
                  : (((r >> 1) & 1) << 2) | (((r >> 3) & 1) << 1);
}

// The lane's part of staging R rows (columns) of an operand with NW waves: one
// byte offset an instruction, constant while the base moves along k.
template <typename E, bool T, int R, int NW>
struct Stager {
  static constexpr int kInsts = R / 8 / NW;  // 1 KB each
  static constexpr int kRowBytes = T ? R * E::kSize : 128;
  static constexpr int kLanes = kRowBytes / 16, kRows = 64 / kLanes;  // of one instruction
  static_assert(kInsts * NW * 8 == R, "whole instructions");
  uint64_t base;
  uint64_t step;       // bytes from a stage to the next
  uint32_t off[kInsts];
  int k[kInsts];       // first k of the lane's chunk, within the stage

  // `first`: address of the tile's first row (column) at the first k. row_of(r):
  // the source row (column) of the staged one, relative to first, -1: none.
  template <typename F>
  __device__ __forceinline__ void init(const void* first, int64_t ld, int wave, F&& row_of) {
    const int lane = threadIdx.x & 63;
    base = reinterpret_cast<uint64_t>(first);
    step = T ? (uint64_t)ld * E::kSize * kStageK<E> : 128;
#pragma unroll
    for (int i = 0; i < kInsts; ++i) {
      const int r = (wave * kInsts + i) * kRows + lane / kLanes;
      const int c = (lane % kLanes) ^ swz<E, T, R>(r);
      int64_t o;
      if (T) {
        const int64_t n = row_of(c * (16 / E::kSize));
        k[i] = r;
        o = n < 0 ? -1 : ((int64_t)r * ld + n) * E::kSize;
      } else {
        const int64_t n = row_of(r);
        k[i] = c * (16 / E::kSize);
        o = n < 0 ? -1 : n * ld * E::kSize + c * 16;
      }
      off[i] = o < 0 ? kOob : (uint32_t)o;
    }
  }
  // Issues the stage at `base` (left: k from it to the end) and moves on.
  __device__ __forceinline__ void issue(uint32_t lds, int64_t left) {
    const auto rs = make_rsrc(base);
    if (left >= kStageK<E>) {
#pragma unroll
      for (int i = 0; i < kInsts; ++i) dma16(rs, off[i], lds + i * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < kInsts; ++i) dma16(rs, k[i] < left ? off[i] : kOob, lds + i * 1024);
    }
    base += step;
  }
};

// Fragment of rows (columns) x0 .. x0 + 31 of a staged operand for step s of 4:
// 16 k (bf16) or 8 k (fp32; the halves of a wave hold 4 each).
template <typename E, bool T, int R>
__device__ __forceinline__ typename E::Frag frag(const lds_char* st, int x0, int s) {
  const int lane = threadIdx.x & 63;
  if constexpr (!T) {
    const int r = x0 + (lane & 31), c = 2 * s + (lane >> 5);
    return *reinterpret_cast<const __attribute__((address_space(3))) typename E::Frag*>(
        st + r * 128 + ((c ^ swz<E, T, R>(r)) << 4));
  } else if constexpr (E::kSize == 2) {
    const int g = lane >> 4, l = lane & 15;
    const int x = x0 + 16 * (g & 1) + 4 * (l & 3);
    const int kr = 16 * s + 8 * (g >> 1) + (l >> 2);
    const lds_char* q = st + kr * (2 * R) + (((x >> 3) ^ swz<E, T, R>(kr)) << 4) + ((x & 7) << 1);
    // (k-row + 4 has the same swizzle for R >= 128; for 64 too: bits 0, 1 and 3 of it)
    const bf16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)q);
    const bf16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(q + 4 * (2 * R)));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    const int x = x0 + (lane & 31), kr = 8 * s + 4 * (lane >> 5);
    f32x4_t v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = *reinterpret_cast<const lds_float*>(
          st + (kr + i) * (4 * R) + (((x >> 2) ^ swz<E, T, R>(kr + i)) << 4) + ((x & 3) << 2));
    return v;
  }
}

// acc += A B for one step. The operands are swapped, so that a lane holds 4
// consecutive n of one m: acc[4 g + r] is m = lane & 31, n = 8 g + 4 (lane >> 5) + r.
__device__ __forceinline__ f32x16_t mma(bf16x8_t a, bf16x8_t b, f32x16_t acc) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(b, a, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mma(f32x4_t a, f32x4_t b, f32x16_t acc) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    acc = __builtin_amdgcn_mfma_f32_32x32x2f32(b[i], a[i], acc, 0, 0, 0);
  return acc;
}

// Writes the results of a wave: FM x FN blocks of 32 x 32 from (m0, n0) on, 32
// rows at a time through the wave's own 32 x 32 FN x 4 bytes of LDS, so that
// memory sees whole rows, 16 bytes a lane. EPI_GATED: block 0 holds gates, block 1
// the ups of the same 32 columns. sum_row: the row of p.sums that takes the wave's
// column sums.
template <typename E, int EPI, int FM, int FN>
__device__ __forceinline__ void write_tile(const GemmArgs& p, const f32x16_t (&acc)[FM][FN],
                                           lds_char* scr, int64_t m0, int64_t n0,
                                           int64_t sum_row) {
  constexpr int WN = 32 * FN, CH = WN / 4;        // staged columns, 16-byte chunks of a row
  constexpr bool GATED = EPI == EPI_GATED, BWD = EPI == EPI_GATED_BWD;
  static_assert(!GATED || FN == 2, "gate and up");
  constexpr int C = kEpiCols<E, EPI>;
  constexpr int OUT = GATED ? 32 : WN;            // output columns
  constexpr int LR = OUT / C, RP = 64 / LR;       // lanes of a row, rows of a pass
  constexpr int PASSES = 32 / RP;
  const int lane = threadIdx.x & 63;
  const int64_t n = n0 + (lane % LR) * C;
  const bool n_ok = n < p.N;
  EpiCols<EPI, C> cols;
  epi_cols<EPI, C>(p, n, cols);
  float sg[C], su[C];
#pragma unroll
  for (int i = 0; i < C; ++i) sg[i] = su[i] = 0.0f;
  auto at = [&](int r, int c) {
    return scr + r * (WN * 4) + ((c ^ (CH == 16 ? r & 15 : (r >> 1) & 7)) << 4);
  };
  // EPI_GATED_BWD: the gates and ups of a half of 32 rows are fetched while the half
  // before is written, the first while the last rows' sums are staged
  constexpr int HALF = BWD ? PASSES / 2 : 1;
  GateUp z[2][HALF] = {};
  auto fetch = [&](int i, int h) {
#pragma unroll
    for (int t = 0; t < HALF; ++t) {
      const int64_t m = m0 + 32 * i + (h * HALF + t) * RP + lane / LR;
      if (m < p.M && n_ok) z[h][t] = load_z(p, m, n);
    }
  };
  if constexpr (BWD) fetch(0, 0);
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    if (m0 + 32 * i >= p.M) break;
    asm volatile("" ::: "memory");  // (a wave's LDS accesses complete in order)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4_t v = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2],
                           acc[i][j][4 * g + 3]};
        *reinterpret_cast<lds_f32x4*>(at(lane & 31, 8 * j + 2 * g + (lane >> 5))) = v;
      }
    asm volatile("" ::: "memory");
    if constexpr (EPI == EPI_LINEAR && C == 8) {
      if (p.z) {  // the pre-activations first: 4 columns a lane
        const int64_t nz = n0 + (lane % CH) * 4;
        EpiCols<EPI, 4> qz;
        epi_cols<EPI, 4>(p, nz, qz);
#pragma unroll
        for (int t = 0; t < CH / 2; ++t) {
          const int r = t * (64 / CH) + lane / CH;
          const f32x4_t a = *reinterpret_cast<lds_f32x4*>(at(r, lane % CH));
          const float v[4] = {a[0] + qz.b[0], a[1] + qz.b[1], a[2] + qz.b[2], a[3] + qz.b[3]};
          const int64_t m = m0 + 32 * i + r;
          if (m < p.M && nz < p.N) store_z4(p.z + m * p.ldz + nz, p.z_past, v);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < PASSES; ++t) {
      if constexpr (BWD) {
        if (t == 0) fetch(i, 1);
        if (t == HALF && i + 1 < FM) fetch(i + 1, 0);
      }
      const int r = t * RP + lane / LR, c = (lane % LR) * (C / 4);
      float v[C], u[C];
#pragma unroll
      for (int q = 0; q < C / 4; ++q) {
        const f32x4_t a = *reinterpret_cast<lds_f32x4*>(at(r, c + q));
        f32x4_t b = a;
        if (GATED) b = *reinterpret_cast<lds_f32x4*>(at(r, c + q + 8));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[4 * q + e] = a[e];
          u[4 * q + e] = b[e];
        }
      }
      const int64_t m = m0 + 32 * i + r;
      if (m < p.M && n_ok)
        epi_row<E, EPI, C>(p, cols, m, n, v, u, z[t / HALF & 1][t % HALF], sg, su);
    }
  }
  if constexpr (BWD) {
    if (p.sums && n0 < p.N && m0 < p.M) {
      // lanes of the same columns, in a fixed order
#pragma unroll
      for (int o = LR; o < 64; o *= 2)
#pragma unroll
        for (int i = 0; i < C; ++i) {
          sg[i] += __shfl_xor(sg[i], o, 64);
          su[i] += __shfl_xor(su[i], o, 64);
        }
      if (lane < LR && n_ok) {
        store_c<F32, C>(p.sums + sum_row * 2 * p.N, n, sg);
        store_c<F32, C>(p.sums + sum_row * 2 * p.N + p.N, n, su);
      }
    }
  }
}

// A wave's sums of a slice, in the order its registers hold them, so that every
// store is a kilobyte in one piece: 4 values of each lane for block (i, j) and
// register group g at ((i FN + j) 4 + g) 64 + lane (see mma for their rows and
// columns). dst: the wave's part.
template <int FM, int FN>
__device__ __forceinline__ void write_part(const f32x16_t (&acc)[FM][FN], float* dst) {
  f32x4_t* out = reinterpret_cast<f32x4_t*>(dst) + (threadIdx.x & 63);
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4_t v = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2],
                           acc[i][j][4 * g + 3]};
        out[((i * FN + j) * 4 + g) * 64] = v;
      }
}

// Place t of n in which XCD b % 8 takes a contiguous run (workgroup b is the b / 8 th
// of its XCD).
__device__ __forceinline__ int xcd_run(int b, int n) {
  const int x = b & 7;
  return x * (n >> 3) + min(x, n & 7) + (b >> 3);
}

// The tile of workgroup b, and its slice of k (-1: all of it). Tiles go through
// groups of GM row tiles column by column, so that the tiles an XCD works on at a
// time share operand rows and columns in its L2.
struct Tile {
  int m, n, slice;
  int split;  // index among the split tiles
};
__device__ __forceinline__ Tile tile_at(const GemmArgs& p, int t, int GM) {
  Tile o = {};
  const int gsize = GM * p.tiles_n;
  const int g = t / gsize, first = g * GM;
  const int rows = min(GM, p.tiles_m - first);
  t -= g * gsize;
  o.m = first + t % rows;
  o.n = t / rows;
  return o;
}
__device__ __forceinline__ Tile tile_of(const GemmArgs& p, int b, int GM) {
  if (b < p.whole) {
    Tile o = tile_at(p, xcd_run(b, p.whole), GM);
    o.slice = -1;
    return o;
  }
  const int rest = p.tiles_m * p.tiles_n - p.whole;
  const int t = xcd_run(b - p.whole, rest * p.splits);
  const int slice = t / rest, split = t - slice * rest;
  Tile o = tile_at(p, p.whole + split, GM);
  o.slice = slice;
  o.split = split;
  return o;
}
// k of the tile's workgroup: [first, last)
__device__ __forceinline__ void tile_k(const GemmArgs& p, const Tile& t, int64_t& k0, int64_t& k1) {
  k0 = t.slice < 0 ? 0 : t.slice * p.kper;
  k1 = t.slice < 0 ? p.K : min(p.K, k0 + p.kper);
}
// Where the sums of its slice go (VALUES: of a tile).
template <int VALUES>
__device__ __forceinline__ float* tile_part(const GemmArgs& p, const Tile& t) {
  const int rest = p.tiles_m * p.tiles_n - p.whole;
  return p.part + ((int64_t)t.slice * rest + t.split) * VALUES;
}

}  // namespace dense
}  // namespace vmoe
