// Layer norm, forward and backward:
//   y = (x - mean) rstd w + b, rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   xh = (x - mean) rstd, gn = gy w
//   gx = rstd (gn - mean(gn) - xh mean(gn xh)), gw = sum_rows gy xh, gb = sum_rows gy
//
// Memory bound: a row is read once and kept in registers (fp32) for the mean, the
// centred sum of squares and the result; statistics, gradients and sums are fp32. The
// mean's own error (a share of |x|, not of the spread) is the mean of the centred values
// and is taken out of them: a row of 65537.3 gives 0, where without that 768 values gave
// 0.98 (32768 x 2048 in bf16 52.6 -> 53 us with its values out of the caches; 8192 x 8192,
// with 1024 threads a row, 55.5 -> 60). The backward pass reads the mean as one float, off by half a unit of its last place.
// A row belongs to 8, 16 or 64 threads (within a wave, no barrier) or, where it is
// long, to 256 or 1024; workgroups go on to further rows with the weights, and in the backward
// pass their gradients' sums, in registers. The forward pass fetches a row while the
// one before is worked on (32768 x 2048 in bf16: 64 -> 48 us with 256 threads a row
// instead of 64; 49 now, 5.5 TB/s); the backward pass, with two streams of rows, gained
// nothing by that (77 to 83 us, 4.9 to 5.2 TB/s). Those sums are joined in a fixed
// order: within a workgroup, then by a launch of their own. Rows of any length are read
// 16 bytes at a time (see Span): 16384 x 4095 in bf16, both passes, 489 us value by
// value, 240 so, 157 for 4096. Short rows by 8 or 16 threads instead of 64: 300000 x 47
// forward 62 -> 18 us, 300000 x 128 62 -> 29 (5.2 TB/s). Unaligned rows of more than 8192
// values spill in the backward pass (bf16 20 bytes a lane, fp32 52).

#include "dense_launch.h"

namespace vmoe {
namespace {

using dense::Bf16;
using dense::F32;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename E>
constexpr int kVec = 16 / E::kSize;  // values of a chunk

// A chunk of a row: 16 bytes from value i of p on. AL: rows are of whole chunks and
// aligned to them; else chunks have the alignment of a value (rows shorter than a chunk:
// d values, one by one).
template <typename E, bool AL>
struct Chunk {
  static constexpr int V = kVec<E>;
  typedef typename E::Store Store;
  u32x4 q;

  __device__ __forceinline__ void load(const void* p, int64_t i, int64_t d) {
    const Store* at = static_cast<const Store*>(p) + i;
    if constexpr (AL) {
      q = *reinterpret_cast<const u32x4*>(at);
    } else if (d >= V) {
      __builtin_memcpy(&q, at, 16);
    } else {
      Store v[V] = {};
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < d) v[e] = at[e];
      __builtin_memcpy(&q, v, 16);
    }
  }
  __device__ __forceinline__ void get(float (&v)[V]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (V == 4) {
        v[e] = __uint_as_float(q[e]);
      } else {
        v[2 * e] = lo_f32(q[e]);
        v[2 * e + 1] = hi_f32(q[e]);
      }
    }
  }
  static __device__ __forceinline__ void store(void* p, int64_t i, int64_t d,
                                               const float (&v)[V]) {
    Store* at = static_cast<Store*>(p) + i;
    u32x4 q;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (V == 4) q[e] = __float_as_uint(v[e]);
      else q[e] = pack_bf16(v[2 * e], v[2 * e + 1]);
    }
    if constexpr (AL) {
      *reinterpret_cast<u32x4*>(at) = q;
    } else if (d >= V) {
      __builtin_memcpy(at, &q, 16);
    } else {
      Store w[V];
      __builtin_memcpy(w, &q, 16);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < d) at[e] = w[e];
    }
  }
};

// What chunk c of thread t covers. A row's last chunk ends at its end: where the row is
// not of whole chunks it begins among the values of the chunk before, which it reads and
// writes too (the same bits), but which count there (lo) in sums.
struct Span {
  int64_t i;   // first value
  int lo, hi;  // those of its values that count
  bool on;     // any
  __device__ __forceinline__ bool counts(int e) const { return e >= lo && e < hi; }
};
template <typename E, int TPR, bool AL>
__device__ __forceinline__ Span span_of(int64_t d, int c, int t) {
  constexpr int V = kVec<E>;
  const int64_t first = ((int64_t)c * TPR + t) * V;
  if (AL) return {first, 0, first < d ? V : 0, first < d};
  const int64_t i = max((int64_t)0, min(first, d - V));
  return {i, (int)min((int64_t)V, first - i), first < d ? (int)min((int64_t)V, d - i) : 0, first < d};
}

// V values of a weight from value i on, of either type.
template <int V, bool AL>
__device__ __forceinline__ void load_weight(const void* p, int f32, int64_t i, int64_t d,
                                            float (&v)[V]) {
  if constexpr (AL) {
    if (f32) {
#pragma unroll
      for (int h = 0; h < V / 4; ++h) {
        const f32x4 w = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * h + e] = w[e];
      }
    } else {
      typedef uint32_t words __attribute__((ext_vector_type(V / 2)));
      const words w = *reinterpret_cast<const words*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        v[2 * e] = lo_f32(w[e]);
        v[2 * e + 1] = hi_f32(w[e]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < d)
        v[e] = f32 ? static_cast<const float*>(p)[i + e]
                   : bf16_to_f32(static_cast<const uint16_t*>(p)[i + e]);
  }
}

// Sums over the TPR threads of a row, the same value in each of them. red: one
// row of TPR / 64 values a quantity, used in turn (`flip`) by successive calls,
// so that one barrier a call is enough. Of two quantities each half of a wave sums one
// (8192 x 8192 forward 64.6 -> 59.7 us).
template <int TPR, int Q>
__device__ __forceinline__ void row_sums(float (&v)[Q], float (*red)[Q][16], int& flip) {
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float s = v[0];
    if constexpr (Q == 2) {
      const float other = lane < 32 ? v[1] : v[0];
      s = (lane < 32 ? v[0] : v[1]) + __shfl_xor(other, 32, 64);
    } else {
      s += __shfl_xor(s, 32, 64);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((lane & (Q == 2 ? 31 : 63)) == 0) red[flip][Q == 2 ? lane >> 5 : 0][wave] = s;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      s = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; w += 4) {
        const f32x4 r = *reinterpret_cast<const f32x4*>(red[flip][q] + w);
#pragma unroll
        for (int i = 0; i < 4; ++i) s += r[i];
      }
      v[q] = s;
    }
    flip ^= 1;
  } else {
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
      for (int o = TPR / 2; o > 0; o >>= 1) v[q] += __shfl_xor(v[q], o, 64);
  }
}

// a b, rounded: not joined with an addition of it to one rounding of both.
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
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

template <typename E, int TPR, int NCH, bool AL>
__global__ __launch_bounds__(kNormThreads<TPR>) void norm_fwd_kernel(NormArgs p) {
  constexpr int ROWS = kNormThreads<TPR> / TPR, V = kVec<E>;
  __shared__ __align__(16) float red[2][1][16];
  __shared__ __align__(16) float sums[2][2][16];
  const int t = threadIdx.x % TPR;
  int flip = 0;
  float w[NCH][V], b[NCH][V];
  Span span[NCH];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    span[c] = span_of<E, TPR, AL>(p.d, c, t);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      w[c][e] = 1.0f;
      b[c][e] = 0.0f;
    }
    if (span[c].on) {
      if (p.w) load_weight<V, AL>(p.w, p.w_f32, span[c].i, p.d, w[c]);
      if (p.b) load_weight<V, AL>(p.b, p.b_f32, span[c].i, p.d, b[c]);
    }
  }
  const float inv = 1.0f / (float)p.d;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  Chunk<E, AL> next[NCH];
  auto fetch = [&](int64_t row) {
    const typename E::Store* at = static_cast<const typename E::Store*>(p.x) + row * p.ldx;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
      if (span[c].on) next[c].load(at, span[c].i, p.d);
  };
  if (r < p.rows) fetch(r);
  for (; r < p.rows; r += step) {
    float x[NCH][V];
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
#pragma unroll
      for (int e = 0; e < V; ++e) x[c][e] = 0.0f;
      if (span[c].on) next[c].get(x[c]);
    }
    if (r + step < p.rows) fetch(r + step);
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) s[0] += AL || span[c].counts(e) ? x[c][e] : 0.0f;
    row_sums<TPR, 1>(s, red, flip);
    const float mean = product(s[0], inv);  // (`off` below is that of this value)
    float q[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        x[c][e] -= mean;
        const float v = (AL ? span[c].on : span[c].counts(e)) ? x[c][e] : 0.0f;
        q[0] += v;
        q[1] += v * v;
      }
    row_sums<TPR, 2>(q, sums, flip);
    const float off = product(q[0], inv);  // what the mean was off by
    float var = q[1] * inv - off * off;
    var = var < 0.0f ? 0.0f : var;  // (NaN stays)
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) x[c][e] -= off;
    const float rstd = 1.0f / sqrtf(var + p.eps);
    if (p.stats && t == 0)
      *reinterpret_cast<float2*>(p.stats + 2 * r) = make_float2(mean + off, rstd);
    typename E::Store* out = static_cast<typename E::Store*>(p.y) + r * p.ldy;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      float y[V];
#pragma unroll
      for (int e = 0; e < V; ++e) y[e] = x[c][e] * rstd * w[c][e] + b[c][e];
      if (span[c].on) Chunk<E, AL>::store(out, span[c].i, p.d, y);
    }
  }
}

// WG: gw and gb are wanted (part).
template <typename E, int TPR, int NCH, bool AL, bool WG>
__global__ __launch_bounds__(kNormThreads<TPR>) void norm_bwd_kernel(NormArgs p) {
  constexpr int ROWS = kNormThreads<TPR> / TPR, V = kVec<E>;
  __shared__ __align__(16) float red[2][2][16];
  const int t = threadIdx.x % TPR;
  int flip = 0;
  float w[NCH][V], gw[NCH][V], gb[NCH][V];
  Span span[NCH];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    span[c] = span_of<E, TPR, AL>(p.d, c, t);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      w[c][e] = 1.0f;
      gw[c][e] = gb[c][e] = 0.0f;
    }
    if (span[c].on && p.w) load_weight<V, AL>(p.w, p.w_f32, span[c].i, p.d, w[c]);
  }
  const float inv = 1.0f / (float)p.d;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  for (int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR; r < p.rows; r += step) {
    const typename E::Store* row = static_cast<const typename E::Store*>(p.x) + r * p.ldx;
    const typename E::Store* grow = static_cast<const typename E::Store*>(p.gy) + r * p.ldgy;
    const float2 st = *reinterpret_cast<const float2*>(p.stats + 2 * r);
    float x[NCH][V], g[NCH][V];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        x[c][e] = st.x;
        g[c][e] = 0.0f;
      }
      if (span[c].on) {
        Chunk<E, AL> qx, qg;
        qx.load(row, span[c].i, p.d);
        qg.load(grow, span[c].i, p.d);
        qx.get(x[c]);
        qg.get(g[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        x[c][e] = (x[c][e] - st.x) * st.y;
        if (WG) {
          gw[c][e] += g[c][e] * x[c][e];
          gb[c][e] += g[c][e];
        }
        g[c][e] *= w[c][e];
        const float n = AL || span[c].counts(e) ? g[c][e] : 0.0f;
        s[0] += n;
        s[1] += n * x[c][e];
      }
    if (p.y) {
      row_sums<TPR, 2>(s, red, flip);
      const float m0 = s[0] * inv, m1 = s[1] * inv;
      typename E::Store* out = static_cast<typename E::Store*>(p.y) + r * p.ldy;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        float y[V];
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = st.y * (g[c][e] - m0 - x[c][e] * m1);
        if (span[c].on) Chunk<E, AL>::store(out, span[c].i, p.d, y);
      }
    }
  }
  if constexpr (WG) {
    float* dst = p.part + (int64_t)blockIdx.x * 2 * p.d;
    if constexpr (ROWS == 1) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int64_t i = span[c].i;
        if constexpr (AL) {
          if (span[c].on)
#pragma unroll
            for (int e = 0; e < V; e += 4) {
              *reinterpret_cast<f32x4*>(dst + i + e) =
                  f32x4{gw[c][e], gw[c][e + 1], gw[c][e + 2], gw[c][e + 3]};
              *reinterpret_cast<f32x4*>(dst + p.d + i + e) =
                  f32x4{gb[c][e], gb[c][e + 1], gb[c][e + 2], gb[c][e + 3]};
            }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (span[c].counts(e)) {
              dst[i + e] = gw[c][e];
              dst[p.d + i + e] = gb[c][e];
            }
        }
      }
    } else {
      // the rows of a workgroup, in order
      constexpr int D = NCH * V * TPR;
      __shared__ float sum[2][D];
      for (int k = 0; k < ROWS; ++k) {
        if ((int)(threadIdx.x / TPR) == k) {
#pragma unroll
          for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const int i = (c * V + e) * TPR + t;
              sum[0][i] = k ? sum[0][i] + gw[c][e] : gw[c][e];
              sum[1][i] = k ? sum[1][i] + gb[c][e] : gb[c][e];
            }
        }
        __syncthreads();
      }
      for (int i = threadIdx.x; i < D; i += kNormThreads<TPR>) {
        const int ce = i / TPR, c = ce / V, e = ce % V;
        const Span q = span_of<E, TPR, AL>(p.d, c, i % TPR);
        if (q.counts(e)) {
          dst[q.i + e] = sum[0][i];
          dst[p.d + q.i + e] = sum[1][i];
        }
      }
    }
  }
}

constexpr int64_t kMaxNorm = 16384;  // 1024 threads of 16 values
constexpr int64_t kNormGroups = 1024;  // workgroups of a backward pass: rows of its sums

// Threads of a row by its length: up to 16 values a thread (8 threads: 8).
inline int norm_threads(int64_t d) {
  return d <= 64 ? 8 : d <= 256 ? 16 : d <= 1024 ? 64 : d <= 4096 ? 256 : 1024;
}

inline int64_t norm_groups(int64_t rows, int tpr) {
  const int64_t per = tpr < 256 ? 256 / tpr : 1;
  const int64_t most = tpr == 1024 ? 256 : kNormGroups;
  const int64_t g = (rows + per - 1) / per;
  return g < most ? g : most;
}

// f(TPR, NCH, AL) for rows of d values; al: whether rows and weights are of whole
// aligned chunks.
template <typename E, typename F>
int norm_pick(int64_t d, bool al, F&& f) {
  constexpr int V = kVec<E>;
  auto width = [&](auto T) -> int {
    constexpr int TPR = decltype(T)::value;
    auto chunks = [&](auto N) -> int {
      return al ? f(T, N, std::true_type()) : f(T, N, std::false_type());
    };
    if (d <= TPR * 8) return chunks(std::integral_constant<int, 8 / V>());
    if constexpr (TPR > 8)
      if (d <= TPR * 16) return chunks(std::integral_constant<int, 16 / V>());
    return VMOE_ERR_UNSUPPORTED;
  };
  switch (norm_threads(d)) {
    case 8: return width(std::integral_constant<int, 8>());
    case 16: return width(std::integral_constant<int, 16>());
    case 64: return width(std::integral_constant<int, 64>());
    case 256: return width(std::integral_constant<int, 256>());
    default: return width(std::integral_constant<int, 1024>());
  }
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
    return norm_pick<E>(d, vec, [&](auto T, auto N, auto AL) -> int {
      constexpr int TPR = decltype(T)::value;
      const int64_t per = TPR < 256 ? 256 / TPR : 1;
      const int64_t need = (rows + per - 1) / per;
      const uint32_t grid = (uint32_t)(need < 2048 ? need : 2048);
      VMOE_LAUNCH((norm_fwd_kernel<E, TPR, decltype(N)::value, decltype(AL)::value>), dim3(grid),
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
    return norm_pick<E>(d, vec, [&](auto T, auto N, auto AL) -> int {
      constexpr int TPR = decltype(T)::value, NC = decltype(N)::value;
      constexpr bool A = decltype(AL)::value;
      if (wg)
        VMOE_LAUNCH((norm_bwd_kernel<E, TPR, NC, A, true>), dim3((uint32_t)groups),
                    dim3(kNormThreads<TPR>), 0, s, p);
      else
        VMOE_LAUNCH((norm_bwd_kernel<E, TPR, NC, A, false>), dim3((uint32_t)groups),
                    dim3(kNormThreads<TPR>), 0, s, p);
      VMOE_CHECK_LAUNCH();
      return VMOE_OK;
    });
  };
  if (int st = type == VMOE_DENSE_F32 ? go(F32()) : go(Bf16())) return st;
  if (wg) return dense::col_sum(p.part, groups, 2 * d, d, gw, gw_f32, gb, gb_f32, s);
  return VMOE_OK;
}
