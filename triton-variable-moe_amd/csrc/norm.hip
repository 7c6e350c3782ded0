// Layer norm, forward and backward:
//   y = (x - mean) rstd w + b, rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   xh = (x - mean) rstd, gn = gy w
//   gx = rstd (gn - mean(gn) - xh mean(gn xh)), gw = sum_rows gy xh, gb = sum_rows gy
//
// Memory bound: a row is read once and kept in registers (fp32) for the mean, the
// centred sum of squares and the result; statistics, gradients and sums are fp32.
// A row belongs to 64 threads (one wave, no barrier) or, where it is long, to 256
// or 1024; workgroups go on to further rows with the weights, and in the backward
// pass their gradients' sums, in registers. The forward pass fetches a row while the
// one before is worked on (32768 x 2048 in bf16: 64 -> 48 us with 256 threads a row
// instead of 64, 5.6 TB/s); the backward pass, with two streams of rows, gained
// nothing by that (77 to 83 us, 4.9 to 5.2 TB/s). Those sums are joined in a fixed
// order: within a workgroup, then by a launch of their own.

#include "dense_launch.h"

namespace vmoe {
namespace {

using dense::Bf16;
using dense::F32;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// VEC values of a row as they lie in memory: 16 bytes, or one value (VEC = 1).
template <typename E, int VEC>
struct Raw {
  static constexpr bool kWide = VEC > 1;
  static_assert(!kWide || VEC * E::kSize == 16, "16 bytes");
  std::conditional_t<kWide, u32x4, typename E::Store> q;
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    q = *reinterpret_cast<const decltype(q)*>(static_cast<const typename E::Store*>(p) + i);
  }
  __device__ __forceinline__ void get(float* v) const {
    if constexpr (!kWide) {
      if constexpr (E::kSize == 4) v[0] = q;
      else v[0] = bf16_to_f32(q);
    } else if constexpr (E::kSize == 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(q[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[2 * e] = lo_f32(q[e]);
        v[2 * e + 1] = hi_f32(q[e]);
      }
    }
  }
};

// VEC values at p[i] (rows' values come as Raw): a weight, of either type.
template <typename E, int VEC>
__device__ __forceinline__ void load_vec(const void* p, int64_t i, float* v) {
  if constexpr (VEC * E::kSize == 32) {
    load_vec<E, VEC / 2>(p, i, v);
    load_vec<E, VEC / 2>(p, i + VEC / 2, v + VEC / 2);
  } else if constexpr (VEC * E::kSize == 8) {
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
    v[0] = lo_f32(w.x);
    v[1] = hi_f32(w.x);
    v[2] = lo_f32(w.y);
    v[3] = hi_f32(w.y);
  } else {
    Raw<E, VEC> q;
    q.load(p, i);
    q.get(v);
  }
}

template <typename E, int VEC>
__device__ __forceinline__ void store_vec(void* p, int64_t i, const float* v) {
  if constexpr (VEC == 1) {
    if constexpr (E::kSize == 4) static_cast<float*>(p)[i] = v[0];
    else static_cast<uint16_t*>(p)[i] = (uint16_t)f32_to_bf16(v[0]);
  } else if constexpr (E::kSize == 4) {
#pragma unroll
    for (int j = 0; j < VEC / 4; ++j) {
      const f32x4 w = {v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]};
      *reinterpret_cast<f32x4*>(static_cast<float*>(p) + i + 4 * j) = w;
    }
  } else if constexpr (VEC == 8) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pack_bf16(v[2 * e], v[2 * e + 1]);
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + i) = w;
  } else {
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) =
        make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
  }
}

template <int VEC>
__device__ __forceinline__ void load_weight(const void* p, int f32, int64_t i, float* v) {
  if (f32) load_vec<F32, VEC>(p, i, v);
  else load_vec<Bf16, VEC>(p, i, v);
}

// Sums over the TPR threads of a row, the same value in each of them. red: one
// row of TPR / 64 values a quantity, used in turn (`flip`) by successive calls,
// so that one barrier a call is enough.
template <int TPR, int Q>
__device__ __forceinline__ void row_sums(float (&v)[Q], float (*red)[Q][16], int& flip) {
#pragma unroll
  for (int q = 0; q < Q; ++q) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v[q] += __shfl_xor(v[q], o, 64);
  }
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (lane == 0)
#pragma unroll
      for (int q = 0; q < Q; ++q) red[flip][q][wave] = v[q];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) s += red[flip][q][w];
      v[q] = s;
    }
    flip ^= 1;
  }
}

struct NormArgs {
  const void* x;
  int64_t ldx;
  const void* w;
  const void* b;
  int32_t w_f32, b_f32;
  float eps;
  int64_t rows, d;
  void* y;        // backward: gx
  int64_t ldy;
  float* stats;   // [rows, 2]: mean, rstd (forward: may be null)
  const void* gy;
  int64_t ldgy;
  float* part;    // backward: [workgroups, 2, d], or null
};

template <int TPR>
constexpr int kNormThreads = TPR < 256 ? 256 : TPR;

template <typename E, int TPR, int VEC, int NCH>
__global__ __launch_bounds__(kNormThreads<TPR>) void norm_fwd_kernel(NormArgs p) {
  constexpr int ROWS = kNormThreads<TPR> / TPR;
  __shared__ float red[2][1][16];
  const int t = threadIdx.x % TPR;
  int flip = 0;
  float w[NCH][VEC], b[NCH][VEC];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int64_t i = ((int64_t)c * TPR + t) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[c][e] = 1.0f;
      b[c][e] = 0.0f;
    }
    if (i < p.d) {
      if (p.w) load_weight<VEC>(p.w, p.w_f32, i, w[c]);
      if (p.b) load_weight<VEC>(p.b, p.b_f32, i, b[c]);
    }
  }
  const float inv = 1.0f / (float)p.d;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  Raw<E, VEC> next[NCH];
  auto fetch = [&](int64_t row) {
    const typename E::Store* at = static_cast<const typename E::Store*>(p.x) + row * p.ldx;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int64_t i = ((int64_t)c * TPR + t) * VEC;
      if (i < p.d) next[c].load(at, i);
    }
  };
  if (r < p.rows) fetch(r);
  for (; r < p.rows; r += step) {
    float x[NCH][VEC];
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int64_t i = ((int64_t)c * TPR + t) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[c][e] = 0.0f;
      if (i < p.d) next[c].get(x[c]);
    }
    if (r + step < p.rows) fetch(r + step);
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[0] += x[c][e];
    row_sums<TPR, 1>(s, red, flip);
    const float mean = s[0] * inv;
    s[0] = 0.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const bool in = ((int64_t)c * TPR + t) * VEC < p.d;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        x[c][e] -= mean;
        s[0] += in ? x[c][e] * x[c][e] : 0.0f;
      }
    }
    row_sums<TPR, 1>(s, red, flip);
    const float rstd = 1.0f / sqrtf(s[0] * inv + p.eps);
    if (p.stats && t == 0)
      *reinterpret_cast<float2*>(p.stats + 2 * r) = make_float2(mean, rstd);
    typename E::Store* out = static_cast<typename E::Store*>(p.y) + r * p.ldy;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int64_t i = ((int64_t)c * TPR + t) * VEC;
      float y[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) y[e] = x[c][e] * rstd * w[c][e] + b[c][e];
      if (i < p.d) store_vec<E, VEC>(out, i, y);
    }
  }
}

// WG: gw and gb are wanted (part).
template <typename E, int TPR, int VEC, int NCH, bool WG>
__global__ __launch_bounds__(kNormThreads<TPR>) void norm_bwd_kernel(NormArgs p) {
  constexpr int ROWS = kNormThreads<TPR> / TPR;
  __shared__ float red[2][2][16];
  const int t = threadIdx.x % TPR;
  int flip = 0;
  float w[NCH][VEC], gw[NCH][VEC], gb[NCH][VEC];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int64_t i = ((int64_t)c * TPR + t) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[c][e] = 1.0f;
      gw[c][e] = gb[c][e] = 0.0f;
    }
    if (i < p.d && p.w) load_weight<VEC>(p.w, p.w_f32, i, w[c]);
  }
  const float inv = 1.0f / (float)p.d;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  for (; r < p.rows; r += step) {
    const typename E::Store* row = static_cast<const typename E::Store*>(p.x) + r * p.ldx;
    const typename E::Store* grow = static_cast<const typename E::Store*>(p.gy) + r * p.ldgy;
    const float2 st = *reinterpret_cast<const float2*>(p.stats + 2 * r);
    float x[NCH][VEC], g[NCH][VEC];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int64_t i = ((int64_t)c * TPR + t) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        x[c][e] = st.x;
        g[c][e] = 0.0f;
      }
      if (i < p.d) {
        load_vec<E, VEC>(row, i, x[c]);
        load_vec<E, VEC>(grow, i, g[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        x[c][e] = (x[c][e] - st.x) * st.y;
        if (WG) {
          gw[c][e] += g[c][e] * x[c][e];
          gb[c][e] += g[c][e];
        }
        g[c][e] *= w[c][e];
        s[0] += g[c][e];
        s[1] += g[c][e] * x[c][e];
      }
    if (p.y) {
      row_sums<TPR, 2>(s, red, flip);
      const float m0 = s[0] * inv, m1 = s[1] * inv;
      typename E::Store* out = static_cast<typename E::Store*>(p.y) + r * p.ldy;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int64_t i = ((int64_t)c * TPR + t) * VEC;
        float y[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) y[e] = st.y * (g[c][e] - m0 - x[c][e] * m1);
        if (i < p.d) store_vec<E, VEC>(out, i, y);
      }
    }
  }
  if constexpr (WG) {
    float* dst = p.part + (int64_t)blockIdx.x * 2 * p.d;
    if constexpr (ROWS == 1) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int64_t i = ((int64_t)c * TPR + t) * VEC;
        if (i < p.d) {
          store_vec<F32, VEC>(dst, i, gw[c]);
          store_vec<F32, VEC>(dst + p.d, i, gb[c]);
        }
      }
    } else {
      // the waves of a workgroup, in order
      constexpr int D = NCH * VEC * TPR;
      __shared__ float sum[2][D];
      for (int k = 0; k < ROWS; ++k) {
        if ((int)(threadIdx.x / TPR) == k) {
#pragma unroll
          for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const int i = (c * VEC + e) * TPR + t;
              sum[0][i] = k ? sum[0][i] + gw[c][e] : gw[c][e];
              sum[1][i] = k ? sum[1][i] + gb[c][e] : gb[c][e];
            }
        }
        __syncthreads();
      }
      for (int i = threadIdx.x; i < D; i += kNormThreads<TPR>) {
        const int ce = i / TPR, c = ce / VEC, e = ce % VEC;
        const int64_t col = ((int64_t)c * TPR + i % TPR) * VEC + e;
        if (col < p.d) {
          dst[col] = sum[0][i];
          dst[p.d + col] = sum[1][i];
        }
      }
    }
  }
}

constexpr int64_t kMaxNorm = 16384;  // 1024 threads of 16 values
constexpr int64_t kNormGroups = 1024;  // workgroups of a backward pass: rows of its sums

// Threads of a row by its length: up to 16 values a thread.
inline int norm_threads(int64_t d) { return d <= 1024 ? 64 : d <= 4096 ? 256 : 1024; }

inline int64_t norm_groups(int64_t rows, int tpr) {
  const int64_t per = tpr < 256 ? 256 / tpr : 1;
  const int64_t most = tpr == 1024 ? 256 : kNormGroups;
  const int64_t g = (rows + per - 1) / per;
  return g < most ? g : most;
}

// f(TPR, VEC, NCH) for rows of d values; vec: the widest load that rows and
// weights allow, in values (1, or 16 bytes).
template <typename E, typename F>
int norm_pick(int64_t d, bool vec, F&& f) {
  constexpr int V = 16 / E::kSize;
  const int tpr = norm_threads(d);
  auto width = [&](auto T) -> int {
    constexpr int TPR = decltype(T)::value;
    auto chunks = [&](auto VEC_) -> int {
      constexpr int VEC = decltype(VEC_)::value;
      typedef std::integral_constant<int, TPR> I;
      if (d <= TPR * 8) return f(I(), VEC_, std::integral_constant<int, 8 / VEC>());
      if (d <= TPR * 16) return f(I(), VEC_, std::integral_constant<int, 16 / VEC>());
      return VMOE_ERR_UNSUPPORTED;
    };
    if (vec) return chunks(std::integral_constant<int, V>());
    return chunks(std::integral_constant<int, 1>());
  };
  if (tpr == 64) return width(std::integral_constant<int, 64>());
  if (tpr == 256) return width(std::integral_constant<int, 256>());
  return width(std::integral_constant<int, 1024>());
}

int check_norm(int type, int64_t rows, int64_t d) {
  if (type != VMOE_DENSE_BF16 && type != VMOE_DENSE_F32) return VMOE_ERR_INVALID_ARG;
  if (rows < 0 || d <= 0) return VMOE_ERR_INVALID_ARG;
  if (d > kMaxNorm) return VMOE_ERR_UNSUPPORTED;
  return VMOE_OK;
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace vmoe

using namespace vmoe;

extern "C" int64_t vmoe_layer_norm_max(void) { return kMaxNorm; }

extern "C" int vmoe_layer_norm(int32_t type, const void* x, int64_t ldx, int64_t rows, int64_t d,
                               const void* w, int32_t w_f32, const void* b, int32_t b_f32,
                               float eps, void* y, int64_t ldy, float* stats,
                               vmoe_stream_t stream) {
  if (int st = check_norm(type, rows, d)) return st;
  if (rows == 0) return VMOE_OK;
  if (!x || !y || ldx < 0 || (ldx < d && ldx != 0 && rows > 1) || ldy < d)
    return VMOE_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(stats) & 7) return VMOE_ERR_UNSUPPORTED;
  NormArgs p = {};
  p.x = x; p.ldx = ldx; p.rows = rows; p.d = d;
  p.w = w; p.w_f32 = w_f32; p.b = b; p.b_f32 = b_f32;
  p.eps = eps;
  p.y = y; p.ldy = ldy; p.stats = stats;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  auto go = [&](auto e) -> int {
    typedef decltype(e) E;
    constexpr int V = 16 / E::kSize;
    const bool vec = d % V == 0 && ldx % V == 0 && ldy % V == 0 && al16(x) && al16(y) &&
                     al16(w) && al16(b);
    return norm_pick<E>(d, vec, [&](auto T, auto VEC, auto N) -> int {
      constexpr int TPR = decltype(T)::value;
      const int64_t per = TPR < 256 ? 256 / TPR : 1;
      const int64_t need = (rows + per - 1) / per;
      const uint32_t grid = (uint32_t)(need < 2048 ? need : 2048);
      VMOE_LAUNCH((norm_fwd_kernel<E, TPR, decltype(VEC)::value, decltype(N)::value>), dim3(grid),
                  dim3(kNormThreads<TPR>), 0, s, p);
      VMOE_CHECK_LAUNCH();
      return VMOE_OK;
    });
  };
  return type == VMOE_DENSE_F32 ? go(F32()) : go(Bf16());
}

extern "C" size_t vmoe_layer_norm_workspace_bytes(int64_t rows, int64_t d) {
  if (rows <= 0 || d <= 0 || d > kMaxNorm) return 0;
  return (size_t)norm_groups(rows, norm_threads(d)) * 2 * d * 4;
}

extern "C" int vmoe_layer_norm_backward(int32_t type, const void* gy, int64_t ldgy, const void* x,
                                        int64_t ldx, int64_t rows, int64_t d, const void* w,
                                        int32_t w_f32, const float* stats, void* gx, int64_t ldgx,
                                        void* gw, int32_t gw_f32, void* gb, int32_t gb_f32,
                                        void* workspace, size_t workspace_bytes,
                                        vmoe_stream_t stream) {
  if (int st = check_norm(type, rows, d)) return st;
  if (rows == 0) return VMOE_OK;
  if (!x || !gy || !stats || ldx < 0 || (ldx < d && ldx != 0 && rows > 1) || ldgy < 0 ||
      (ldgy < d && ldgy != 0 && rows > 1) || (gx && ldgx < d))
    return VMOE_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(stats) & 7) return VMOE_ERR_UNSUPPORTED;
  const bool wg = gw || gb;
  if (wg) {
    if (!workspace) return VMOE_ERR_INVALID_ARG;
    if (workspace_bytes < vmoe_layer_norm_workspace_bytes(rows, d)) return VMOE_ERR_WORKSPACE;
    if (!al16(workspace)) return VMOE_ERR_UNSUPPORTED;
  }
  if (!gx && !wg) return VMOE_OK;
  NormArgs p = {};
  p.x = x; p.ldx = ldx; p.rows = rows; p.d = d;
  p.w = w; p.w_f32 = w_f32;
  p.y = gx; p.ldy = ldgx;
  p.stats = const_cast<float*>(stats);
  p.gy = gy; p.ldgy = ldgy;
  p.part = static_cast<float*>(workspace);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t groups = norm_groups(rows, norm_threads(d));
  auto go = [&](auto e) -> int {
    typedef decltype(e) E;
    constexpr int V = 16 / E::kSize;
    const bool vec = d % V == 0 && ldx % V == 0 && ldgy % V == 0 && (!gx || ldgx % V == 0) &&
                     al16(x) && al16(gy) && al16(gx) && al16(w);
    return norm_pick<E>(d, vec, [&](auto T, auto VEC, auto N) -> int {
      constexpr int TPR = decltype(T)::value, VE = decltype(VEC)::value, NC = decltype(N)::value;
      if (wg)
        VMOE_LAUNCH((norm_bwd_kernel<E, TPR, VE, NC, true>), dim3((uint32_t)groups),
                    dim3(kNormThreads<TPR>), 0, s, p);
      else
        VMOE_LAUNCH((norm_bwd_kernel<E, TPR, VE, NC, false>), dim3((uint32_t)groups),
                    dim3(kNormThreads<TPR>), 0, s, p);
      VMOE_CHECK_LAUNCH();
      return VMOE_OK;
    });
  };
  if (int st = type == VMOE_DENSE_F32 ? go(F32()) : go(Bf16())) return st;
  if (wg) return dense::col_sum(p.part, groups, 2 * d, d, gw, gw_f32, gb, gb_f32, s);
  return VMOE_OK;
}
