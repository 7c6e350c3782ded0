// The expert layer for a few tokens (a generation step): router logits, choice
// of experts, up and down projection and weighted sum, for bf16, fp32 and 4-bit
// weights, and the products of rows with 4-bit matrices.
//
// With T tokens of k experts each, an expert gets T k / E rows: far fewer than
// a matrix instruction's 16 or, at best, a few times that. Every weight of a
// chosen expert is then used a handful of times, so what bounds the layer is
// reading those weights once, and with one or two tokens the chain of dependent
// launches. The kernels are built for that:
//
// - No token is moved and no row is padded: a workgroup takes one expert and a
//   tile of its columns, finds the rows that chose the expert, and gathers them
//   as the 16-row operand of the matrix instructions.
// - Weights go from memory to registers straight into operand form. A lane's
//   operand is 8 consecutive rows of one column; the lane loads 8 rows of CPL
//   adjacent columns and forms CPL operands by byte permutes, no LDS between. The
//   sum over k may run in any order as long as both operands agree, so lane group
//   g takes rows 8 g..8 g + 7 of each 32. 4-bit matrices are stored in operand
//   order (few_q4.h). An expert's weights are read once while its rows fit a pass
//   (32 rows with two row tiles, else 16), and again for each further pass; where a
//   workgroup takes a pair or a token, once for each of them that chose the expert.
// - The waves of a workgroup split K; their partial sums meet in LDS in a fixed
//   order, so results do not change from run to run.
// - The router's choice needs no sort: expert e is chosen by a token if fewer
//   than k experts precede it (larger logit, or an equal one of lower index), and
//   that count is its place.
//
// What was measured and left: forming the logits in the up projection of one token
// (every workgroup reads all router weights: as long as the launch it saves),
// fetching the up projection's weights during the router's launch (the launch grows
// by what the next one saves), and more steps of a wave in flight where workgroups
// share a CU (fewer of them fit: 10 to 30 % slower on large layers).
//
// Sums, logits, routing weights and the activation are fp32. The activations h
// enter the second product as two bf16 halves, h = hi + lo to 2^-16: the matrix
// instructions are far from their limit, and one bf16 rounding of h would add as
// much error as the output's own.
#include <algorithm>

#include "few_q4.h"

namespace vmoe {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / kWave;
constexpr int kTileCols = 64;  // of an up projection's workgroup
constexpr int kMaxTokens = 256, kMaxRows = 4096, kMaxExperts = 2048, kMaxTopK = 64;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct Ids {
  const void* p;  // nullptr: row r takes matrix 0
  int is64;
};

__device__ __forceinline__ int load_id(const Ids& s, int i, int E) {
  if (!s.p) return 0;
  if (s.is64) {
    const int64_t v = static_cast<const int64_t*>(s.p)[i];
    return v >= 0 && v < E ? (int)v : -1;
  }
  const int32_t v = static_cast<const int32_t*>(s.p)[i];
  return v >= 0 && v < E ? v : -1;
}

// Total order of the logits as unsigned integers: NaN above everything, as
// torch.topk orders it; -0 and 0 equal.
__device__ __forceinline__ uint32_t sort_key(float f) {
  if (f != f) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(f == 0.0f ? 0.0f : f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float sigmoid_f32(float x) { return 1.0f / (1.0f + expf(-x)); }

// *(base + off bytes): a base that is one for the wave and a 32-bit offset of the
// lane, so that an address costs no vector registers.
template <class V>
__device__ __forceinline__ V at(const void* base, uint32_t off) {
  return *reinterpret_cast<const V*>(static_cast<const char*>(base) + off);
}

// ---------------------------------------------------------------------------
// Weight formats. A step is KS rows of K; a wave's tile is NC = 16 C columns.
// load() brings one lane's part of a step, mma() multiplies it with 16 rows.
// ---------------------------------------------------------------------------

// bf16, row-major. CPL columns a lane: 8 or 4 bytes of each row.
template <int CPL>
struct WBf16 {
  static constexpr int KS = 32, C = CPL, NC = 16 * CPL;
  using V = typename std::conditional<CPL == 4, u32x2, uint32_t>::type;
  using Row = uint16_t;
  struct A {
    bf16x8_t v;
  };
  V r[8];

  __device__ __forceinline__ static int col(int c, int lane) { return (lane & 15) * CPL + c; }

  // A lane's offset in bytes from the step's first row and the matrix's first
  // column. Columns past N read the last ones (not stored).
  __device__ __forceinline__ static uint32_t lane_offset(const Stack& w, int n0, int N, int lane) {
    const int n = min(n0 + (lane & 15) * CPL, N - CPL);
    return ((uint32_t)(lane >> 4) * 8 * (uint32_t)w.ld + n) * 2;
  }

  // Every lane loads, so that the number of loads in flight is known where their
  // results are awaited: rows past K are those of the first lanes, and finish()
  // takes them as zeros.
  __device__ __forceinline__ void load(const Stack& w, const MatEntry& m, bool by_rows, int k0,
                                       int K, int, int, uint32_t off, int lane) {
    const uint16_t* p = static_cast<const uint16_t*>(w.w) +
                        ((by_rows ? (int64_t)m.off : 0) + k0) * w.ld + (by_rows ? 0 : m.off);
    const uint32_t down = (lane >> 4) * 8;
    if (k0 + (int)down >= K) off -= down * (uint32_t)w.ld * 2;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = at<V>(p + j * w.ld, off);
  }
  __device__ __forceinline__ void finish(int k0, int K, int lane) {
    if (k0 + KS <= K) return;
    const bool in = k0 + (lane >> 4) * 8 < K;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = in ? r[j] : V{};
  }

  __device__ __forceinline__ static void load_a(A& a, const Row* base, uint32_t off, int k0, int K,
                                                int lane) {
    const uint32_t right = (lane >> 4) * 8;
    a.v = at<bf16x8_t>(base + k0, k0 + (int)right < K ? off : off - right * 2);
  }
  __device__ __forceinline__ static void finish_a(A& a, int k0, int K, int lane) {
    if (k0 + KS > K) a.v = k0 + (lane >> 4) * 8 < K ? a.v : bf16x8_t{};
  }

  // Operand of column c: the c-th value of each of the 8 rows.
  __device__ __forceinline__ bf16x8_t operand(int c) const {
    const uint32_t* q = reinterpret_cast<const uint32_t*>(r);
    constexpr int D = CPL / 2;  // dwords of a row
    const uint32_t sel = (c & 1) ? 0x07060302u : 0x05040100u;
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = __builtin_amdgcn_perm(q[(2 * i + 1) * D + c / 2], q[2 * i * D + c / 2], sel);
    return __builtin_bit_cast(bf16x8_t, v);
  }

  template <int MT, int PL>
  __device__ __forceinline__ void mma(const A (&a)[MT][PL], int tiles,
                                      f32x4_t (&acc)[MT][C]) const {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const bf16x8_t b = operand(c);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m > 0 && m >= tiles) break;
#pragma unroll
        for (int q = 0; q < PL; ++q)
          acc[m][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[m][q].v, b, acc[m][c], 0, 0, 0);
      }
    }
  }
};

// fp32, row-major: CPL (four or two) columns a lane and 16 rows a step, lane group
// g taking rows 4 g..4 g + 3.
template <int CPL>
struct WF32 {
  static constexpr int KS = 16, C = CPL, NC = 16 * CPL;
  using V = typename std::conditional<CPL == 4, f32x4_t, f32x2_t>::type;
  using Row = float;
  struct A {
    f32x4_t v;
  };
  V r[4];

  __device__ __forceinline__ static int col(int c, int lane) { return (lane & 15) * CPL + c; }

  __device__ __forceinline__ static uint32_t lane_offset(const Stack& w, int n0, int N, int lane) {
    const int n = min(n0 + (lane & 15) * CPL, N - CPL);
    return ((uint32_t)(lane >> 4) * 4 * (uint32_t)w.ld + n) * 4;
  }

  __device__ __forceinline__ void load(const Stack& w, const MatEntry& m, bool by_rows, int k0,
                                       int K, int, int, uint32_t off, int lane) {
    const float* p = static_cast<const float*>(w.w) +
                     ((by_rows ? (int64_t)m.off : 0) + k0) * w.ld + (by_rows ? 0 : m.off);
    const uint32_t down = (lane >> 4) * 4;
    if (k0 + (int)down >= K) off -= down * (uint32_t)w.ld * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = at<V>(p + j * w.ld, off);
  }
  __device__ __forceinline__ void finish(int k0, int K, int lane) {
    if (k0 + KS <= K) return;
    const bool in = k0 + (lane >> 4) * 4 < K;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = in ? r[j] : V{};
  }

  __device__ __forceinline__ static void load_a(A& a, const Row* base, uint32_t off, int k0, int K,
                                                int lane) {
    const uint32_t right = (lane >> 4) * 4;
    a.v = at<f32x4_t>(base + k0, k0 + (int)right < K ? off : off - right * 4);
  }
  __device__ __forceinline__ static void finish_a(A& a, int k0, int K, int lane) {
    if (k0 + KS > K) a.v = k0 + (lane >> 4) * 4 < K ? a.v : f32x4_t{};
  }

  template <int MT, int PL>
  __device__ __forceinline__ void mma(const A (&a)[MT][PL], int tiles,
                                      f32x4_t (&acc)[MT][C]) const {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m > 0 && m >= tiles) break;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < C; ++c)
          acc[m][c] =
              __builtin_amdgcn_mfma_f32_16x16x4f32(a[m][0].v[j], r[j][c], acc[m][c], 0, 0, 0);
    }
  }
};

// 4-bit, in operand order (few_q4.h): 16 bytes a lane are its column's values of
// 128 rows, four operands. GJ: operands that share a scale (group = 32 GJ). The
// values are exact in bf16; a group's fp32 sum is scaled once.
template <int CB, int GJ>
struct WQ4 {
  static constexpr int KS = kQ4Rows, C = CB, NC = 16 * CB, S = 4 / GJ;
  using Row = uint16_t;
  struct A {
    bf16x8_t v[4];
  };
  u32x4 r[CB];
  using Scales = typename std::conditional<
      S == 4, u32x2, typename std::conditional<S == 2, uint32_t, uint16_t>::type>::type;
  Scales s[CB];

  __device__ __forceinline__ static int col(int c, int lane) { return c * 16 + (lane & 15); }

  __device__ __forceinline__ static uint32_t lane_offset(const Stack&, int, int, int lane) {
    return lane * 16;
  }

  __device__ __forceinline__ void load(const Stack& w, const MatEntry& m, bool, int k0, int K,
                                       int n0, int N, uint32_t off, int lane) {
    const int kb = k0 / KS, kbs = (K + KS - 1) / KS;
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      // (blocks past the last column read that one; not stored)
      const int nb = min(n0 / 16 + c, (N - 1) / 16);
      const int64_t blk = m.base + (int64_t)nb * kbs + kb;
      r[c] = at<u32x4>(static_cast<const char*>(w.w) + blk * kQ4BlockBytes, off);
      s[c] = at<Scales>(w.scales + blk * 16 * S, (lane & 15) * S * 2);
    }
  }

  // Scale of group g: the g-th 16 bits, as fp32.
  __device__ __forceinline__ float scale(int c, int g) const {
    if constexpr (S == 4) {
      return (g & 1) ? hi_f32(s[c][g / 2]) : lo_f32(s[c][g / 2]);
    } else if constexpr (S == 2) {
      return g ? hi_f32(s[c]) : lo_f32(s[c]);
    } else {
      return bf16_to_f32(s[c]);
    }
  }

  __device__ __forceinline__ void finish(int, int, int) {}  // (blocks are whole)

  __device__ __forceinline__ static void load_a(A& a, const Row* base, uint32_t off, int k0, int K,
                                                int lane) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t right = (lane >> 4) * 8;
      a.v[j] = at<bf16x8_t>(base + k0, k0 + 32 * j + (int)right < K ? off + 64 * j
                                                                   : off - right * 2);
    }
  }
  __device__ __forceinline__ static void finish_a(A& a, int k0, int K, int lane) {
    if (k0 + KS <= K) return;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      a.v[j] = k0 + 32 * j + (lane >> 4) * 8 < K ? a.v[j] : bf16x8_t{};
  }

  template <int MT, int PL>
  __device__ __forceinline__ void mma(const A (&a)[MT][PL], int tiles,
                                      f32x4_t (&acc)[MT][C]) const {
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
      for (int g = 0; g < S; ++g) {
        bf16x8_t b[GJ];
#pragma unroll
        for (int j = 0; j < GJ; ++j) b[j] = q4_values(r[c][g * GJ + j]);
        const float f = scale(c, g);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if (m > 0 && m >= tiles) break;
          f32x4_t part = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < GJ; ++j)
#pragma unroll
            for (int q = 0; q < PL; ++q)
              part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[m][q].v[g * GJ + j], b[j], part, 0,
                                                             0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][c][i] = fmaf(f, part[i], acc[m][c][i]);
        }
      }
  }
};

// ---------------------------------------------------------------------------
// One expert's rows times its matrix
// ---------------------------------------------------------------------------

enum Mode { kUp, kDown, kPlain };

struct FewArgs {
  Stack w;
  const MatEntry* tab;
  const void* a;  // rows of x (kUp, kPlain) or h (kDown)
  int64_t lda, lo;  // row stride; distance of the second half (kDown)
  int T, k, E;
  const float* logits;  // kUp: [T, ldl], or nullptr: ids
  int ldl;
  Ids ids;
  int32_t* sel;  // kUp with logits: chosen experts and their sigmoids, [T, k]
  float* prob;
  const MatEntry* tab2;  // slots: the down projections' entries, and where the
  MatEntry* entry;       // assignments' go, [T, k]
  int fixed;  // kUp, kPlain: K of every matrix; kDown: N
  int cols;   // columns of the widest matrix
  int tiles;  // its column tiles
  const int32_t* tile_of;  // kUp: the expert of each kTileCols columns
  int num_tiles;
  bool slots;  // a workgroup takes an assignment
  int wk;     // waves that split K; kWaves / wk split the tile's columns
  void* out;  // h, y (fp32) or the products
  int64_t ldo;
};

// How many experts of a token come before expert e, whose logit is `mine`:
// eight lanes share the row (padded to kLogitPad with -inf), each gets the count.
// HAVE: the row's first values are in registers already.
constexpr int kLogitPad = 32;
template <bool HAVE = false>
__device__ __forceinline__ int place_of(const float* l, int ldl, int e, float mine, int part,
                                        const f32x4_t* have = nullptr) {
  const uint32_t key = sort_key(mine);
  int before = 0;
  auto count = [&](const f32x4_t& v, int f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t other = sort_key(v[i]);
      before += other > key || (other == key && f + i < e);
    }
  };
  constexpr int N = HAVE ? 4 : 0;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i * kLogitPad < ldl) count(have[i], part * 4 + i * kLogitPad);
#pragma unroll 4
  for (int f = part * 4 + N * kLogitPad; f < ldl; f += kLogitPad)
    count(*reinterpret_cast<const f32x4_t*>(l + f), f);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) before += __shfl_xor(before, o, kWave);
  return before;
}

// The assignments t k + s that take expert e, into LDS, and their number, in two
// steps: a thread's first loads, then the rest. Loads return in the order of their
// issue, so what is issued between the two comes after them. The rows' order does
// not matter: each is on its own.
struct RowProbe {
  static constexpr int N = 4;
  float mine;    // logits: of expert e and of others, for the thread's first token
  f32x4_t v[N];
  int id;        // ids: the thread's first one
};
__device__ __forceinline__ RowProbe probe_rows(const FewArgs& p, int e) {
  RowProbe r;
  if (p.logits) {
    const float* l = p.logits + (int64_t)min((int)threadIdx.x / 8, p.T - 1) * p.ldl;
    r.mine = l[e];
#pragma unroll
    for (int i = 0; i < RowProbe::N; ++i)
      r.v[i] = *reinterpret_cast<const f32x4_t*>(
          l + min((int)(threadIdx.x & 7) * 4 + i * kLogitPad, p.ldl - 4));
  } else {
    r.id = load_id(p.ids, min((int)threadIdx.x, p.T * p.k - 1), p.E);
  }
  return r;
}
__device__ __forceinline__ int find_rows(const FewArgs& p, int e, const RowProbe& first,
                                         bool writer, uint16_t* rows, int* count) {
  if (threadIdx.x == 0) *count = 0;
  lds_barrier();
  if (p.logits) {
    const int part = threadIdx.x & 7;
    auto take = [&](int t, float mine, int before) {
      if (before >= p.k || part != 0) return;
      const int a = t * p.k + before;
      rows[atomicAdd(count, 1)] = (uint16_t)a;
      if (writer) {
        p.sel[a] = e;
        p.prob[a] = sigmoid_f32(mine);
      }
    };
    int t = threadIdx.x / 8;
    const float* l = p.logits + (int64_t)min(t, p.T - 1) * p.ldl;
    const int before = place_of<true>(l, p.ldl, e, first.mine, part, first.v);
    if (t < p.T) take(t, first.mine, before);
    for (t += kThreads / 8; t < p.T; t += kThreads / 8) {
      l = p.logits + (int64_t)t * p.ldl;
      const float mine = l[e];
      take(t, mine, place_of(l, p.ldl, e, mine, part));
    }
  } else {
    const int want = e < p.E ? e : -1;
    for (int a = threadIdx.x; a < p.T * p.k; a += kThreads)
      if ((a < kThreads ? first.id : load_id(p.ids, a, p.E)) == want)
        rows[atomicAdd(count, 1)] = (uint16_t)a;
  }
  lds_barrier();
  return *count;
}

constexpr int kSlotExperts = 256;  // at most, where a workgroup takes one assignment
// The expert of assignment a, or -1.
__device__ __forceinline__ int find_expert(const FewArgs& p, int a, bool writer, float* lg,
                                           int* found) {
  if (!p.logits) {
    const int e = __builtin_amdgcn_readfirstlane(load_id(p.ids, a, p.E));
    if (writer && threadIdx.x == 0) {
      MatEntry m = load_entry(p.tab2 + max(e, 0));
      if (e < 0) m.len = 0;
      store_entry(p.entry + a, m);
    }
    return e;
  }
  const int lane8 = threadIdx.x & 7, t = a / p.k, s = a % p.k;
  if ((int)threadIdx.x < p.ldl) lg[threadIdx.x] = p.logits[(int64_t)t * p.ldl + threadIdx.x];
  lds_barrier();
  for (int e = threadIdx.x / 8; e < p.E; e += kThreads / 8) {
    const float mine = lg[e];
    const int before = place_of(lg, p.ldl, e, mine, lane8);
    if (before == s && lane8 == 0) {
      *found = e;
      if (writer) {
        p.sel[a] = e;
        p.prob[a] = sigmoid_f32(mine);
        store_entry(p.entry + a, load_entry(p.tab2 + e));
      }
    }
  }
  lds_barrier();
  return __builtin_amdgcn_readfirstlane(*found);
}

// Workgroup -> unit. An XCD (blockIdx % 8) has an L2 of its own, whose 16 channels
// take 256 bytes each in turn, and the rows of a weight matrix are a multiple of
// 4 KB apart: an XCD that reads every eighth 256 bytes of a row uses an eighth of
// its L2 (up projection of 128 experts 2048 x 576: 87 us so, 60 us with a
// contiguous run of columns).
//   kRuns: an XCD takes a contiguous eighth of the units.
//   kDeal: the owners (experts) are dealt over the XCDs, all tiles of one to the
//   same; owners of unequal length spread evenly.
//   kPairs: pairs of units are dealt; for calls too small to fill the card, where
//   two narrow tiles share a line.
// The grid is a multiple of 16.
enum Order { kRuns, kDeal, kPairs };
__device__ __forceinline__ int unit_of_block(Order order, int units, int tiles) {
  const int xcd = blockIdx.x & 7, j = blockIdx.x >> 3;
  if (order == kRuns) {
    const int per = (units + 7) / 8, u = xcd * per + j;
    return j < per && u < units ? u : -1;
  }
  const int u = order == kDeal ? (j / tiles * 8 + xcd) * tiles + j % tiles
                               : (j >> 1) * 16 + xcd * 2 + (j & 1);
  return u < units ? u : -1;
}

// Waves a SIMD holds at least: the long K of a down projection's many small tiles is
// covered by other workgroups (128 experts 576 x 2048: 65 us with two on a CU, 58
// with three).
template <class W, int MODE, int MT, int DEPTH>
constexpr int kMinWaves =
    MODE == kDown && MT == 1 && DEPTH == 1 && sizeof(typename W::Row) == 2 && W::KS == 32 ? 6 : 1;

// Bound by reading weights: 32 tokens through 128 experts of 2048 x 576 (262 MB a
// product) 58 us up and 57 down, 4.5 TB/s where a copy moves 5.2; 64 tokens through 64
// of 1024 x 256 (33 MB) 12.1 and 11.6 (10.7 and 10.3 where they lie in the last-level
// cache), of which 2.2 are the launch, 1 the tables, 2 the joining of the waves; in 4 bits
// (8.9 MB) 7.3 and 7.9.
// SLOT: a unit is an assignment and a tile (one row), else an expert and a tile. MT:
// 16-row tiles in one pass over the weights; NS: matrices of an expert (gate and
// up); DEPTH: steps of a wave in flight.
template <class W, int MODE, int MT, int NS, bool SLOT, int DEPTH, bool EARLY>
__global__ __launch_bounds__(kThreads, (kMinWaves<W, MODE, MT, DEPTH>)) void few_kernel(FewArgs p) {
  constexpr int PL = (MODE == kDown && sizeof(typename W::Row) == 2) ? 2 : 1;
  constexpr int NC = W::NC;
  constexpr int kPerLane = 16 / sizeof(typename W::Row);  // values of a 16-byte load
  __shared__ float red[NS * 16 * kWaves * NC];            // [NS][wk][16][width]
  __shared__ uint16_t rows[SLOT ? 8 : kMaxRows];
  __shared__ int count;
  // kPlain with ids: one matrix more, for the rows that name none (their products are 0)
  const int owners = SLOT ? p.T * p.k : p.E + (MODE == kPlain && p.ids.p ? 1 : 0);
  int owner, tile;
  if constexpr (MODE == kUp && !SLOT) {
    const int parts = kTileCols / (kWaves / p.wk * NC);  // a workgroup may take a part
    const int unit = unit_of_block(kRuns, p.num_tiles * parts, 1);
    if (unit < 0) return;
    owner = p.tile_of[unit / parts];
    tile = unit - p.tab[owner * NS].first_tile * parts;
  } else {
    const int unit = unit_of_block(SLOT ? kPairs : MODE == kDown ? kDeal : kRuns,
                                   owners * p.tiles, p.tiles);
    if (unit < 0) return;
    owner = unit / p.tiles, tile = unit % p.tiles;
  }
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wn_count = kWaves / p.wk;
  const int wk = wave / wn_count, wn = wave % wn_count;
  const int width = wn_count * NC;  // columns of the workgroup, a power of two
  const int shift = __builtin_ctz(width);
  const int nt = tile * width;  // the tile's first column
  const int n0 = nt + wn * NC;

  int e = owner, m = 1;
  if constexpr (SLOT) {
    // (red is free until the products are joined)
    static_assert(NS * 16 * kWaves * NC >= kSlotExperts, "room for the logits");
    e = find_expert(p, owner, tile == 0, red, &count);
    if (e < 0) return;
    if (threadIdx.x == 0) rows[0] = (uint16_t)owner;
    lds_barrier();  // (also: the logits in red have been read)
  }
  MatEntry mats[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) mats[s] = load_entry(p.tab + min(e, p.E - 1) * NS + s);
  if (MODE == kPlain && e == p.E) mats[0].len = 0;
  const int K = MODE == kDown ? mats[0].len : p.fixed;
  const int N = MODE == kDown ? p.fixed : min(mats[0].len, p.cols);
  if (MODE != kPlain && nt >= N) return;

  const uint32_t boff = W::lane_offset(p.w, n0, N, lane);
  const int stride = p.wk * W::KS, first = wk * W::KS;
  W b[DEPTH][NS];
  auto load_b = [&](int d, int k0) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
      b[d][s].load(p.w, mats[s], MODE == kDown, k0, K, n0, N, boff, lane);
  };
  if constexpr (!SLOT) {
    const RowProbe probe = probe_rows(p, min(e, p.E - 1));
    if (MODE == kPlain && nt + width > N) {
      // zeros in the columns of wider matrices than this one
      m = find_rows(p, e, probe, false, rows, &count);
      const int z0 = max(nt, N), zw = min(nt + width, p.cols) - z0;
      for (int x = threadIdx.x; x < m * zw; x += kThreads)
        static_cast<uint16_t*>(p.out)[rows[x / zw] * p.ldo + z0 + x % zw] = 0;
      if (nt >= N) return;
      lds_barrier();
    }
    // EARLY: where most experts have rows, the first weights are on their way before
    // it is known which rows (a wave without steps loads some all the same)
    if constexpr (EARLY) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) load_b(d, first + d * stride < K ? first + d * stride : 0);
    }
    m = find_rows(p, e, probe, tile == 0, rows, &count);
    if (m == 0) return;
  }
  const typename W::Row* abase = static_cast<const typename W::Row*>(p.a);

  for (int m0 = 0; m0 < m; m0 += 16 * MT) {
    const int tiles = min(MT, (m - m0 + 15) / 16);
    uint32_t aoff[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      // rows past the last repeat it; their results are not stored
      const int r = rows[min(m0 + 16 * i + (lane & 15), m - 1)];
      const uint32_t src = MODE == kDown ? r : r / p.k;
      aoff[i] = (src * (uint32_t)p.lda + (lane >> 4) * kPerLane) * sizeof(typename W::Row);
    }
    f32x4_t acc[NS][MT][W::C];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int c = 0; c < W::C; ++c) acc[s][i][c] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

    typename W::A a[DEPTH][MT][PL];
    auto load_a = [&](int d, int k0) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if (i > 0 && i >= tiles) break;
        W::load_a(a[d][i][0], abase, aoff[i], k0, K, lane);
        if constexpr (PL == 2) W::load_a(a[d][i][1], abase + p.lo, aoff[i], k0, K, lane);
      }
    };
    bool have = EARLY && m0 == 0;
    for (int k0 = first; k0 < K; k0 += DEPTH * stride) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        if (k0 + d * stride >= K) break;
        if (!have) load_b(d, k0 + d * stride);
        load_a(d, k0 + d * stride);
      }
      have = false;
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        const int kd = k0 + d * stride;
        if (kd >= K) break;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int q = 0; q < PL; ++q) W::finish_a(a[d][i][q], kd, K, lane);
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          b[d][s].finish(kd, K, lane);
          b[d][s].mma(a[d], tiles, acc[s]);
        }
      }
    }

    // join the waves' parts, one 16-row tile at a time
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if (i > 0 && i >= tiles) break;
      const int left = min(16, m - m0 - 16 * i);
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int c = 0; c < W::C; ++c)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            red[((s * p.wk + wk) * 16 + (lane >> 4) * 4 + q) * width + wn * NC +
                W::col(c, lane)] = acc[s][i][c][q];
      lds_barrier();
      for (int x = threadIdx.x; x < left * width; x += kThreads) {
        const int r = x >> shift, n = nt + (x & (width - 1));
        if (n >= N) continue;
        float z[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          z[s] = 0.0f;
          for (int v = 0; v < p.wk; ++v) z[s] += red[(s * p.wk + v) * 16 * width + x];
        }
        const int64_t at = (int64_t)rows[m0 + 16 * i + r] * p.ldo + n;
        if constexpr (MODE == kUp) {
          float h;
          if constexpr (NS == 2) {
            h = z[0] * sigmoid_f32(z[0]) * z[1];
          } else {
            h = z[0] > 0.0f || z[0] != z[0] ? z[0] * z[0] : 0.0f;
          }
          if constexpr (sizeof(typename W::Row) == 2) {
            // a finite h past bf16's largest value keeps that as its first half
            uint32_t hi = f32_to_bf16(h);
            const bool finite = (__float_as_uint(h) & 0x7F800000u) != 0x7F800000u;
            if (finite && (hi & 0x7FFFu) == 0x7F80u) --hi;
            const uint32_t lo = finite ? f32_to_bf16(h - bf16_to_f32(hi)) : 0u;
            static_cast<uint16_t*>(p.out)[at] = (uint16_t)hi;
            static_cast<uint16_t*>(p.out)[at + p.lo] = (uint16_t)lo;
          } else {
            static_cast<float*>(p.out)[at] = h;
          }
        } else if constexpr (MODE == kDown) {
          static_cast<float*>(p.out)[at] = z[0];
        } else {
          static_cast<uint16_t*>(p.out)[at] = (uint16_t)f32_to_bf16(z[0]);
        }
      }
      lds_barrier();
    }
  }
}

// ---------------------------------------------------------------------------
// Weights of a token's slots: the layer's sigmoids (normalised over the slots if
// asked) or the caller's.
// ---------------------------------------------------------------------------

struct SumArgs {
  int T, k, E, d;
  Ids ids;
  const void* weights;
  int wbf16, normalize;
  void* out;
  int64_t ldo;
  int out_f32;
  int32_t* sel_out;  // nullptr, or where the layer's choice goes
  float* wts_out;
};

// A slot a lane: its expert (-1: none) and its weight as stored.
struct SlotWeight {
  int id;
  float raw;
};
__device__ __forceinline__ SlotWeight load_slot(const SumArgs& p, int t) {
  static_assert(kMaxTopK == kWave, "a slot per lane");
  const int s = threadIdx.x & (kWave - 1), a = t * p.k + min(s, p.k - 1);
  SlotWeight v = {load_id(p.ids, a, p.E),
                  p.wbf16 ? bf16_to_f32(static_cast<const uint16_t*>(p.weights)[a])
                          : static_cast<const float*>(p.weights)[a]};
  if (s >= p.k) v = {-1, 0.0f};
  return v;
}
__device__ __forceinline__ float slot_weight(const SumArgs& p, int t, const SlotWeight& v,
                                             bool writer) {
  const int s = threadIdx.x & (kWave - 1);
  float w = v.raw;
  if (p.normalize) {
    float sum = w;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
    w = w / (sum + 1e-20f);
  }
  if (writer && s < p.k) {
    if (p.sel_out) p.sel_out[t * p.k + s] = v.id;
    if (p.wts_out) p.wts_out[t * p.k + s] = w;
  }
  return w;
}

// ---------------------------------------------------------------------------
// out[t] = sum_s weight[t, s] y[t k + s] over the slots that name an expert, in the
// slots' order. Latency: 2 to 5 us.
// ---------------------------------------------------------------------------

constexpr int kCombineThreads = 128;

__global__ __launch_bounds__(kCombineThreads) void few_combine_kernel(SumArgs p, const float* y0) {
  const int t = blockIdx.y;
  const SlotWeight sw = load_slot(p, t);  // (in every wave: no barrier)
  const int n = (blockIdx.x * kCombineThreads + threadIdx.x) * 4;
  const float* y = y0 + (int64_t)t * p.k * p.d + min(n, p.d - 4);
  f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
  float weight = 0.0f;
  constexpr int S = 8;  // rows on their way together, before it is known which count
  for (int s0 = 0; s0 < p.k; s0 += S) {
    f32x4_t v[S];
#pragma unroll
    for (int s = 0; s < S; ++s)
      v[s] = *reinterpret_cast<const f32x4_t*>(y + (int64_t)min(s0 + s, p.k - 1) * p.d);
    if (s0 == 0) weight = slot_weight(p, t, sw, blockIdx.x == 0 && threadIdx.x < kWave);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      // (a slot's row is written only where it names an expert)
      const int lane = min(s0 + s, kWave - 1);
      if (s0 + s >= p.k || __builtin_amdgcn_readlane(sw.id, lane) < 0) continue;
      const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(weight), lane));
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(f, v[s][i], acc[i]);
    }
  }
  if (n >= p.d) return;
  if (p.out_f32) {
    *reinterpret_cast<f32x4_t*>(static_cast<float*>(p.out) + t * p.ldo + n) = acc;
  } else {
    u32x2 v = {pack_bf16(acc[0], acc[1]), pack_bf16(acc[2], acc[3])};
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p.out) + t * p.ldo + n) = v;
  }
}

// ---------------------------------------------------------------------------
// Down projection and sum of one token: the experts of its slots one after the
// other as a single long K, so that no partial result leaves the workgroup. For
// calls with so few tokens that reading an expert's weights once for each costs less
// than another launch. BY_ID: `entry` is the experts' table, not the slots' entries.
// One token, eight experts of 256 x 1024 (4.2 MB) 6.5 us: 32 workgroups, each of which
// draws 128 KB at the 75 GB/s that one CU's loads in flight give.
// ---------------------------------------------------------------------------

constexpr int kTokenWaves = 16;

template <class W, int DEPTH, bool BY_ID>
__global__ __launch_bounds__(kTokenWaves* kWave) void few_token_kernel(SumArgs p, Stack w,
                                                                      const MatEntry* entry,
                                                                      const void* h, int64_t ldh,
                                                                      int64_t lo, int tiles) {
  using Row = typename W::Row;
  constexpr int PL = sizeof(Row) == 2 ? 2 : 1;
  __shared__ float red[kTokenWaves][W::NC];
  const int unit = unit_of_block(kPairs, p.T * tiles, tiles);
  if (unit < 0) return;
  const int t = unit / tiles, tile = unit % tiles;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  // A slot a lane, in every wave: no barrier before the weights are on their way.
  // An entry of length 0 is a slot without an expert.
  const SlotWeight sw = load_slot(p, t);
  MatEntry mine = load_entry(BY_ID ? entry + max(sw.id, 0) : entry + t * p.k + min(lane, p.k - 1));
  if (BY_ID && sw.id < 0) mine.len = 0;
  const int n0 = tile * W::NC;
  const uint32_t boff = W::lane_offset(w, n0, p.d, lane);
  const uint32_t aoff = (lane >> 4) * 16;

  // The wave's next step: slot s, step j of its expert's n.
  int s = -1, j = wave, n = 0;
  MatEntry mat = {};
  auto settle = [&]() {
    while (s < p.k && j >= n) {
      j -= n;
      ++s;
      n = 0;
      if (s < p.k) {
        mat.off = __builtin_amdgcn_readlane(mine.off, s);
        mat.len = __builtin_amdgcn_readlane(mine.len, s);
        mat.base = __builtin_amdgcn_readlane(mine.base, s);
        n = (mat.len + W::KS - 1) / W::KS;
      }
    }
  };
  settle();
  float weight = 0.0f;
  bool weighed = false;
  float total[W::C];
#pragma unroll
  for (int c = 0; c < W::C; ++c) total[c] = 0.0f;
  while (s < p.k) {
    W b[DEPTH];
    typename W::A a[DEPTH][1][PL];
    int slot[DEPTH], at_k[DEPTH], len[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      slot[d] = s;
      if (s >= p.k) continue;
      const int k0 = j * W::KS;
      at_k[d] = k0;
      len[d] = mat.len;
      b[d].load(w, mat, true, k0, mat.len, n0, p.d, boff, lane);
      const Row* row = static_cast<const Row*>(h) + (int64_t)(t * p.k + s) * ldh;
      W::load_a(a[d][0][0], row, aoff, k0, mat.len, lane);
      if constexpr (PL == 2) W::load_a(a[d][0][1], row + lo, aoff, k0, mat.len, lane);
      j += kTokenWaves;
      settle();
    }
    if (!weighed) {
      weighed = true;
      weight = slot_weight(p, t, sw, wave == 0 && tile == 0);
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (slot[d] >= p.k) continue;
      f32x4_t acc[1][W::C];
#pragma unroll
      for (int c = 0; c < W::C; ++c) acc[0][c] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      b[d].finish(at_k[d], len[d], lane);
#pragma unroll
      for (int q = 0; q < PL; ++q) W::finish_a(a[d][0][q], at_k[d], len[d], lane);
      b[d].mma(a[d], 1, acc);
      const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(weight), slot[d]));
#pragma unroll
      for (int c = 0; c < W::C; ++c) total[c] = fmaf(f, acc[0][c][0], total[c]);
    }
  }
  // (a wave without steps may still be the one that writes the choice)
  if (!weighed) slot_weight(p, t, sw, wave == 0 && tile == 0);
  // every row of the tile is the token's; the first lanes hold row 0
  if (lane < 16) {
#pragma unroll
    for (int c = 0; c < W::C; ++c) red[wave][W::col(c, lane)] = total[c];
  }
  lds_barrier();
  const int x = threadIdx.x;
  if (x < W::NC && n0 + x < p.d) {
    float z = 0.0f;
#pragma unroll
    for (int v = 0; v < kTokenWaves; ++v) z += red[v][x];
    const int64_t at = t * p.ldo + n0 + x;
    if (p.out_f32)
      static_cast<float*>(p.out)[at] = z;
    else
      static_cast<uint16_t*>(p.out)[at] = (uint16_t)f32_to_bf16(z);
  }
}

// ---------------------------------------------------------------------------
// Router logits: 16 tokens x 16 experts a workgroup, its waves split the hidden
// axis. fp32 sums of exact products, not rounded. Latency: 3.3 us for one token and 64
// experts, 4.4 for 64 tokens, 6 for 32 tokens and 128 experts of 2048.
// ---------------------------------------------------------------------------

template <bool F32>
__global__ __launch_bounds__(kThreads) void few_logits_kernel(const void* x, int64_t ldx, int T,
                                                              const void* wr, int64_t ldwr, int E,
                                                              int d, float* logits, int ldl) {
  __shared__ float red[kWaves][16][16];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int t0 = blockIdx.y * 16, e0 = blockIdx.x * 16;
  const int64_t ra = (int64_t)min(t0 + (lane & 15), T - 1) * ldx;
  const int64_t rb = (int64_t)min(e0 + (lane & 15), E - 1) * ldwr;
  constexpr int KS = F32 ? 16 : 32, PER = F32 ? 4 : 8;
  f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
  // A wave's columns are adjacent: the rows are a power of two apart in memory, and it
  // is the columns that spread the waves' reads over the L2's channels. The loads of
  // U steps go out together.
  constexpr int U = 4;
  using V = typename std::conditional<F32, f32x4_t, bf16x8_t>::type;
  using Row = typename std::conditional<F32, float, uint16_t>::type;
  const int per = (d + kWaves * KS - 1) / (kWaves * KS) * KS, end = min(d, wave * per + per);
  for (int k0 = wave * per; k0 < end; k0 += U * KS) {
    V a[U], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * KS + (lane >> 4) * PER, kc = k < end ? k : 0;
      a[u] = *reinterpret_cast<const V*>(static_cast<const Row*>(x) + ra + kc);
      b[u] = *reinterpret_cast<const V*>(static_cast<const Row*>(wr) + rb + kc);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = k0 + u * KS + (lane >> 4) * PER < end;
      a[u] = in ? a[u] : V{};
      b[u] = in ? b[u] : V{};
      if constexpr (F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[u][j], b[u][j], acc, 0, 0, 0);
      } else {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[u], b[u], acc, 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) red[wave][(lane >> 4) * 4 + q][lane & 15] = acc[q];
  __syncthreads();
  if (threadIdx.x < 256) {
    const int t = t0 + threadIdx.x / 16, e = e0 + threadIdx.x % 16;
    float s = 0.0f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) s += red[v][threadIdx.x / 16][threadIdx.x % 16];
    if (t < T) logits[(int64_t)t * ldl + e] = e < E ? s : -INFINITY;
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

int div_up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

template <class W, int MODE, int MT, int NS, bool SLOT, int DEPTH, bool EARLY>
int launch_early(FewArgs p, hipStream_t stream) {
  const int width = kWaves / p.wk * W::NC;
  p.tiles = div_up(p.cols, width);
  const int64_t owners = SLOT ? p.T * p.k : p.E + (MODE == kPlain && p.ids.p ? 1 : 0);
  // (dealt owners: eight at a time)
  int64_t units = (MODE == kDown ? div_up(owners, 8) * 8 : owners) * (int64_t)p.tiles;
  if (MODE == kUp && !SLOT) {
    if (kTileCols % width) return VMOE_ERR_UNSUPPORTED;
    units = (int64_t)p.num_tiles * (kTileCols / width);
  }
  if (units > (1 << 30)) return VMOE_ERR_UNSUPPORTED;
  VMOE_LAUNCH((few_kernel<W, MODE, MT, NS, SLOT, DEPTH, EARLY>), dim3(div_up(units, 16) * 16),
              dim3(kThreads), 0, stream, p);
  VMOE_CHECK_LAUNCH();
  return VMOE_OK;
}

template <class W, int MODE, int MT, int NS, bool SLOT, int DEPTH>
int launch_tiles(const FewArgs& p, hipStream_t stream) {
  // Early weights where most experts have rows. They cost registers, in 4 bits so many
  // that fewer workgroups share a CU; where those come in several rounds, they cover
  // for one another without (128 experts 2048 x 512, 128 rows: 24 us with, 16 without).
  if constexpr (MT == 2 && W::KS != kQ4Rows) {
    // (taken only from 8.5 pairs an expert on)
    return launch_early<W, MODE, MT, NS, SLOT, DEPTH, true>(p, stream);
  } else {
    if constexpr (!SLOT) {
      const int64_t units = MODE == kUp
                                ? (int64_t)p.num_tiles * kTileCols / (kWaves / p.wk * W::NC)
                                : (int64_t)p.E * div_up(p.cols, kWaves / p.wk * W::NC);
      if ((int64_t)p.T * p.k >= p.E && (W::KS != kQ4Rows || units <= 512))
        return launch_early<W, MODE, MT, NS, SLOT, DEPTH, true>(p, stream);
    }
    return launch_early<W, MODE, MT, NS, SLOT, DEPTH, false>(p, stream);
  }
}

template <class W, int MODE, int NS, int DEPTH = 1>
int launch(const FewArgs& p, hipStream_t stream) {
  // Row tiles in one pass over the weights: the mean number of rows, doubled (64 experts
  // 1024 x 256, 16 rows each: 15.6 us with one, 13.1 with two). Not for experts in 4
  // bits, where two leave one workgroup to a CU (128 experts 2048 x 576, 16 rows each:
  // 126 us both products with one, 171 with two).
  if constexpr (W::KS != kQ4Rows || MODE == kPlain) {
    const int64_t rows = p.ids.p || p.logits ? 2 * (int64_t)p.T * p.k / p.E : p.T;
    if (rows > 16) return launch_tiles<W, MODE, 2, NS, false, 1>(p, stream);
  }
  return launch_tiles<W, MODE, 1, NS, false, DEPTH>(p, stream);
}

// Waves that split K, `steps` steps long for the longest matrix.
int split_waves(int64_t steps) {
  int wk = 1;
  while (wk < kWaves && wk < steps) wk *= 2;
  return wk;
}

// Whether a token's down projections run in one workgroup: while the call's pairs
// read at most 2^24 weights of one matrix (2^23 in fp32; measured over 1 to 48 tokens
// of seven layers: up to 20 % faster than the experts' products and their sum at half
// of that, even at it, 5-8 % slower half above it, in 4 bits 20 %), or are a quarter of
// the experts and hardly share one (2 tokens of 8 through 128 experts 2048 x 576: 32 us
// so and 41 by experts, 4 bits 25 and 36; at a third of the experts either is faster).
bool small_call(const vmoe_few_weights& w, int64_t pairs) {
  const double width = (double)w.num_tiles1 * kTileCols / w.num_experts;  // in the mean
  return pairs * 4 <= w.num_experts ||
         pairs * width * w.hidden <= (w.format == VMOE_FEW_F32 ? 1 << 23 : 1 << 24);
}

// Whether, in such a call, the pairs share few experts: an up projection's workgroup
// then takes a pair.
bool few_pairs(int64_t pairs, int64_t E) { return pairs * 2 <= E && E <= kSlotExperts; }

template <int CB, int MODE, int NS>
int launch_q4(const FewArgs& p, int group, hipStream_t stream) {
  switch (group) {
    case 32: return launch<WQ4<CB, 1>, MODE, NS>(p, stream);
    case 64: return launch<WQ4<CB, 2>, MODE, NS>(p, stream);
    default: return launch<WQ4<CB, 4>, MODE, NS>(p, stream);
  }
}

template <int NS>
int launch_slots(const FewArgs& p, int format, int group, hipStream_t stream) {
  // Columns a workgroup: 64 where the call has enough tiles of 64, else 32, in 4 bits 16.
  // Up projections of 8 experts a token: experts 2048 x 576 in bf16, 4 tokens: 26 us
  // with 32 columns and 24 with 64 (4 experts of 1024 x 512, 8 tokens: 13 and 12).
  // 4 bits, experts of 2048 x 1024 / 512 / 256, 1, 2 and 4 tokens: 9.4, 16 and 24 us with
  // 16, 7.7, 8.8 and 12 with 64, but at 64 tiles 6.6 and 7.0. Gated 4-bit experts take
  // 32 of each matrix (2048 x 576, 4 tokens: 22 us with 16, 15 with 32, 16 with 64),
  // fp32 always 32 (the same call: 39 us, 45 with 64).
  // Around the lines, the up launch alone, 128 experts, 8 a token, narrow / wide:
  // 4 bits 2048 x 256 at 64, 96 and 128 tiles 4.8 / 5.6, 5.6 / 5.7 and 5.8 / 5.8,
  // 2048 x 512 at 192 and 256 7.0 / 6.3 and 9.4 / 6.8 (gated 5.7 / 6.3, 7.7 / 6.7,
  // 8.1 / 7.2; 10.7 / 9.8, 12.4 / 11.1): level between 96 and 128. bf16 2048 x 256 at
  // 96 and 128 11.9 / 13.5 and 12.6 / 13.6, 2048 x 512 at 192 and 256 18.1 / 14.2 and
  // 18.8 / 15.0: from about 160 tiles on wide ones win already.
  const int64_t units = (int64_t)p.T * p.k * div_up(p.cols, 64);  // tiles of 64 columns
  if (format == VMOE_FEW_BF16)
    return units >= 256 ? launch_tiles<WBf16<4>, kUp, 1, NS, true, 4 / NS>(p, stream)
                        : launch_tiles<WBf16<2>, kUp, 1, NS, true, 4>(p, stream);
  if (format == VMOE_FEW_F32) return launch_tiles<WF32<2>, kUp, 1, NS, true, 4>(p, stream);
#define SLOTS_Q4(GJ)                                                                  \
  return units >= 128 ? launch_tiles<WQ4<4 / NS, GJ>, kUp, 1, NS, true, 1>(p, stream) \
                      : launch_tiles<WQ4<1, GJ>, kUp, 1, NS, true, 2>(p, stream)
  switch (group) {
    case 32: SLOTS_Q4(1);
    case 64: SLOTS_Q4(2);
    default: SLOTS_Q4(4);
  }
#undef SLOTS_Q4
}

// max_k: rows of the longest matrix.
template <int MODE, int NS>
int launch_format(FewArgs p, int format, int group, int64_t max_k, hipStream_t stream) {
  // the columns of an up projection's tile are fixed (kTileCols)
  const int steps = div_up(max_k, format == VMOE_FEW_Q4 ? kQ4Rows : format ? 16 : 32);
  p.wk = kWaves;
  if (MODE == kDown) p.wk = split_waves(steps);
  if constexpr (MODE == kUp) {
    if (p.slots) return launch_slots<NS>(p, format, group, stream);
    // A workgroup takes kTileCols columns, or half of them where the tiles are fewer
    // than CUs.
    if (format == VMOE_FEW_Q4) {
      if (steps > 4 && p.num_tiles < 256) return launch_q4<2, MODE, NS>(p, group, stream);
      if constexpr (NS == 1)
        if (steps > 4) return launch_q4<4, MODE, NS>(p, group, stream);
      p.wk = 4;
      return launch_q4<2, MODE, NS>(p, group, stream);
    }
    if (p.num_tiles < 256)
      return format == VMOE_FEW_F32 ? launch<WF32<2>, MODE, NS>(p, stream)
                                    : launch<WBf16<2>, MODE, NS>(p, stream);
  } else if (format == VMOE_FEW_Q4) {
    // Four blocks a wave reuse its rows' operands twice as often as two (64 experts
    // 256 x 1024, 512 rows: 9.0 us with two, 7.9 with four; 128 experts 512 x 2048, 128
    // rows: 26 and 18), where enough workgroups are left.
    if ((int64_t)p.E * div_up(p.cols, kWaves / p.wk * 64) >= 256)
      return launch_q4<4, MODE, NS>(p, group, stream);
    return launch_q4<2, MODE, NS>(p, group, stream);
  }
  if (format == VMOE_FEW_F32) return launch<WF32<4>, MODE, NS>(p, stream);
  if constexpr (MODE == kDown)
    if (steps <= 8) {
      p.wk = split_waves(div_up(steps, 2));
      return launch<WBf16<4>, MODE, NS, 2>(p, stream);
    }
  return launch<WBf16<4>, MODE, NS>(p, stream);
}

template <class W, int DEPTH, bool BY_ID>
int launch_token(const SumArgs& p, const Stack& w, const MatEntry* entry, const void* h,
                 int64_t ldh, int64_t lo, hipStream_t stream) {
  const int tiles = div_up(p.d, W::NC);
  const int64_t units = (int64_t)p.T * tiles;
  if (units > (1 << 30)) return VMOE_ERR_UNSUPPORTED;
  VMOE_LAUNCH((few_token_kernel<W, DEPTH, BY_ID>), dim3(div_up(units, 16) * 16),
              dim3(kTokenWaves * kWave), 0, stream, p, w, entry, h, ldh, lo, tiles);
  VMOE_CHECK_LAUNCH();
  return VMOE_OK;
}

template <bool BY_ID>
int launch_tokens(const SumArgs& p, const vmoe_few_weights& w, const MatEntry* entry,
                  const void* h, int64_t ldh, int64_t lo, hipStream_t stream) {
  const Stack s = {w.w2, w.scales2, w.ldw2};
  if (w.format == VMOE_FEW_BF16)
    return launch_token<WBf16<2>, 4, BY_ID>(p, s, entry, h, ldh, lo, stream);
  if (w.format == VMOE_FEW_F32)
    return launch_token<WF32<2>, 4, BY_ID>(p, s, entry, h, ldh, lo, stream);
  switch (w.group) {
    case 32: return launch_token<WQ4<1, 1>, 2, BY_ID>(p, s, entry, h, ldh, lo, stream);
    case 64: return launch_token<WQ4<1, 2>, 2, BY_ID>(p, s, entry, h, ldh, lo, stream);
    default: return launch_token<WQ4<1, 4>, 2, BY_ID>(p, s, entry, h, ldh, lo, stream);
  }
}

struct FewLayout {
  int64_t logits, prob, sel, entry, h, y, bytes, ldh, ldl;
};

bool few_layout(int64_t T, int64_t E, int64_t k, int64_t d, int64_t w, int format, FewLayout& L) {
  if (T < 0 || E <= 0 || k <= 0 || d <= 0 || w <= 0 || format < 0 || format > VMOE_FEW_Q4)
    return false;
  const int64_t A = T * k;
  int64_t off = 0;
  auto slot = [&](int64_t bytes) {
    const int64_t o = off;
    off += (bytes + 255) / 256 * 256;
    return o;
  };
  L.ldh = (w + 7) / 8 * 8;
  L.ldl = (E + kLogitPad - 1) / kLogitPad * kLogitPad;
  L.logits = slot(4 * T * L.ldl);
  L.prob = slot(4 * A);
  L.sel = slot(4 * A);
  L.entry = slot(sizeof(MatEntry) * A);
  L.h = slot(4 * A * L.ldh);  // fp32, or two bf16 halves
  L.y = slot(4 * A * d);
  L.bytes = std::max<int64_t>(off, 256);
  return true;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check_sizes(int64_t T, int64_t E, int64_t k) {
  if (T < 0 || E <= 0 || k <= 0) return VMOE_ERR_INVALID_ARG;
  if (T > kMaxTokens || T * k > kMaxRows || E > kMaxExperts || k > kMaxTopK)
    return VMOE_ERR_UNSUPPORTED;
  return VMOE_OK;
}

int check_weights(const vmoe_few_weights* w) {
  if (!w || w->num_experts <= 0 || w->hidden <= 0 || w->max_width <= 0 || w->format < 0 ||
      w->format > VMOE_FEW_Q4)
    return VMOE_ERR_INVALID_ARG;
  if (w->act != VMOE_ACT_RELU_SQUARED && w->act != VMOE_ACT_SWIGLU) return VMOE_ERR_INVALID_ARG;
  if (!w->w1 || !w->w2 || !w->table1 || !w->table2 || !w->tiles1 || w->num_tiles1 <= 0)
    return VMOE_ERR_INVALID_ARG;
  const int64_t per = w->format == VMOE_FEW_F32 ? 4 : 8;
  if (w->hidden % per || w->max_width % per || w->hidden > (1 << 24) || w->max_width > (1 << 24))
    return VMOE_ERR_UNSUPPORTED;
  if (!aligned16(w->w1) || !aligned16(w->w2) || !aligned16(w->table1) || !aligned16(w->table2))
    return VMOE_ERR_UNSUPPORTED;
  if (w->format == VMOE_FEW_Q4) {
    if (!w->scales1 || !w->scales2) return VMOE_ERR_INVALID_ARG;
    if (w->group != 32 && w->group != 64 && w->group != 128) return VMOE_ERR_INVALID_ARG;
    if (!aligned16(w->scales1) || !aligned16(w->scales2)) return VMOE_ERR_UNSUPPORTED;
  } else {
    if (w->ldw1 <= 0 || w->ldw2 < w->hidden) return VMOE_ERR_INVALID_ARG;
    // (a lane's offset, up to 25 rows, has 32 bits)
    if (w->ldw1 % per || w->ldw2 % per || w->ldw1 > (1 << 24) || w->ldw2 > (1 << 24))
      return VMOE_ERR_UNSUPPORTED;
  }
  return VMOE_OK;
}

// (rows are addressed by 32-bit offsets)
bool spans(int64_t rows, int64_t ld, int64_t size) { return rows * ld * size >= (1ll << 32); }

int check_rows(int64_t T, const void* x, int64_t ldx, int64_t cols, const void* out, int64_t ldo,
               int64_t ocols, int64_t per) {
  if (!x || !out || ldx < cols || ldo < ocols) return VMOE_ERR_INVALID_ARG;
  if (ldx > (1ll << 31) || spans(T, ldx, 16 / per)) return VMOE_ERR_UNSUPPORTED;
  if (ldx % per || ldo % per || !aligned16(x) || !aligned16(out)) return VMOE_ERR_UNSUPPORTED;
  return VMOE_OK;
}

// Up, down and sum; the choice of experts is the logits' or the caller's ids'.
int few_experts(const vmoe_few_weights& w, const void* x, int64_t ldx, const float* logits,
                int32_t* sel, float* prob, const SumArgs& c,
                const FewLayout& L, char* ws, hipStream_t stream) {
  FewArgs p = {};
  p.w = {w.w1, w.scales1, w.ldw1};
  p.tab = reinterpret_cast<const MatEntry*>(w.table1);
  p.a = x;
  p.lda = ldx;
  p.T = c.T;
  p.k = c.k;
  p.E = c.E;
  p.logits = logits;
  p.ldl = (int)L.ldl;
  p.ids = c.ids;
  p.tab2 = reinterpret_cast<const MatEntry*>(w.table2);
  p.entry = reinterpret_cast<MatEntry*>(ws + L.entry);
  p.sel = sel;
  p.prob = prob;
  p.fixed = (int)w.hidden;
  p.cols = (int)w.max_width;
  p.tile_of = w.tiles1;
  p.num_tiles = w.num_tiles1;
  p.out = ws + L.h;
  p.ldo = w.format == VMOE_FEW_F32 ? L.ldh : 2 * L.ldh;
  p.lo = L.ldh;
  const bool small = small_call(w, (int64_t)c.T * c.k);
  p.slots = small && few_pairs((int64_t)c.T * c.k, c.E);
  int st = w.act == VMOE_ACT_SWIGLU
               ? launch_format<kUp, 2>(p, w.format, w.group, w.hidden, stream)
               : launch_format<kUp, 1>(p, w.format, w.group, w.hidden, stream);
  if (st != VMOE_OK) return st;

  const void* h = ws + L.h;
  if (p.slots) return launch_tokens<false>(c, w, p.entry, h, p.ldo, p.lo, stream);
  if (small) return launch_tokens<true>(c, w, p.tab2, h, p.ldo, p.lo, stream);
  p.w = {w.w2, w.scales2, w.ldw2};
  p.tab = p.tab2;
  p.a = h;
  p.lda = p.ldo;
  p.logits = nullptr;
  p.cols = p.fixed = (int)w.hidden;
  float* y = reinterpret_cast<float*>(ws + L.y);
  p.out = y;
  p.ldo = w.hidden;
  st = launch_format<kDown, 1>(p, w.format, w.group, w.max_width, stream);
  if (st != VMOE_OK) return st;
  VMOE_LAUNCH(few_combine_kernel, dim3(div_up(w.hidden, 4 * kCombineThreads), c.T),
              dim3(kCombineThreads), 0, stream, c, y);
  VMOE_CHECK_LAUNCH();
  return VMOE_OK;
}

}  // namespace
}  // namespace vmoe

using namespace vmoe;

extern "C" int vmoe_few_max_tokens(void) { return kMaxTokens; }

extern "C" size_t vmoe_few_workspace_bytes(int64_t T, int32_t E, int32_t k, int64_t hidden,
                                           int64_t max_width, int32_t format) {
  FewLayout L;
  return few_layout(T, E, k, hidden, max_width, format, L) ? (size_t)L.bytes : 0;
}

extern "C" int vmoe_few_layer(const vmoe_few_weights* w, const void* x, int64_t ldx,
                              int64_t num_tokens, const void* router_weight, int64_t ldwr,
                              int32_t top_k, int32_t normalize, void* out, int64_t ldo,
                              int32_t* selected, float* weights, void* workspace,
                              size_t workspace_bytes, vmoe_stream_t stream) {
  int st = check_weights(w);
  if (st != VMOE_OK) return st;
  st = check_sizes(num_tokens, w->num_experts, top_k);
  if (st != VMOE_OK) return st;
  if (top_k > w->num_experts) return VMOE_ERR_INVALID_ARG;
  if (num_tokens == 0) return VMOE_OK;
  const bool f32 = w->format == VMOE_FEW_F32;
  st = check_rows(num_tokens, x, ldx, w->hidden, out, ldo, w->hidden, f32 ? 4 : 8);
  if (st != VMOE_OK) return st;
  if (!router_weight || ldwr < w->hidden || !workspace) return VMOE_ERR_INVALID_ARG;
  if (ldwr % (f32 ? 4 : 8) || !aligned16(router_weight) || !aligned16(workspace))
    return VMOE_ERR_UNSUPPORTED;
  FewLayout L;
  if (!few_layout(num_tokens, w->num_experts, top_k, w->hidden, w->max_width, w->format, L))
    return VMOE_ERR_INVALID_ARG;
  if (workspace_bytes < (size_t)L.bytes) return VMOE_ERR_WORKSPACE;
  if (spans(num_tokens * top_k, L.ldh, 4)) return VMOE_ERR_UNSUPPORTED;
  char* ws = static_cast<char*>(workspace);
  float* logits = reinterpret_cast<float*>(ws + L.logits);
  const int T = (int)num_tokens, E = w->num_experts;
  int32_t* sel = reinterpret_cast<int32_t*>(ws + L.sel);
  float* prob = reinterpret_cast<float*>(ws + L.prob);
  const SumArgs c = {T, top_k, E, (int)w->hidden, {sel, 0}, prob, 0, normalize != 0, out, ldo, f32,
                     selected, weights};
  const dim3 grid(div_up(L.ldl, 16), div_up(T, 16));
  if (f32)
    VMOE_LAUNCH((few_logits_kernel<true>), grid, dim3(kThreads), 0, stream, x, ldx, T,
                router_weight, ldwr, E, (int)w->hidden, logits, (int)L.ldl);
  else
    VMOE_LAUNCH((few_logits_kernel<false>), grid, dim3(kThreads), 0, stream, x, ldx, T,
                router_weight, ldwr, E, (int)w->hidden, logits, (int)L.ldl);
  VMOE_CHECK_LAUNCH();
  return few_experts(*w, x, ldx, logits, sel, prob, c, L, ws, stream);
}

extern "C" int vmoe_few_experts(const vmoe_few_weights* w, const void* x, int64_t ldx,
                                int64_t num_tokens, const void* ids, int32_t ids_are_i64,
                                const void* weights, int32_t weights_are_bf16, int32_t top_k,
                                void* out, int64_t ldo, void* workspace, size_t workspace_bytes,
                                vmoe_stream_t stream) {
  int st = check_weights(w);
  if (st != VMOE_OK) return st;
  st = check_sizes(num_tokens, w->num_experts, top_k);
  if (st != VMOE_OK) return st;
  if (num_tokens == 0) return VMOE_OK;
  st = check_rows(num_tokens, x, ldx, w->hidden, out, ldo, w->hidden,
                  w->format == VMOE_FEW_F32 ? 4 : 8);
  if (st != VMOE_OK) return st;
  if (!ids || !weights || !workspace) return VMOE_ERR_INVALID_ARG;
  if (!aligned16(workspace)) return VMOE_ERR_UNSUPPORTED;
  FewLayout L;
  if (!few_layout(num_tokens, w->num_experts, top_k, w->hidden, w->max_width, w->format, L))
    return VMOE_ERR_INVALID_ARG;
  if (workspace_bytes < (size_t)L.bytes) return VMOE_ERR_WORKSPACE;
  if (spans(num_tokens * top_k, L.ldh, 4)) return VMOE_ERR_UNSUPPORTED;
  char* ws = static_cast<char*>(workspace);
  const SumArgs c = {(int)num_tokens, top_k, w->num_experts, (int)w->hidden, {ids, ids_are_i64},
                     weights, weights_are_bf16, 0, out, ldo, w->format == VMOE_FEW_F32, nullptr,
                     nullptr};
  return few_experts(*w, x, ldx, nullptr, nullptr, nullptr, c, L, ws, stream);
}

extern "C" int vmoe_q4_matvec(const void* x, int64_t ldx, int64_t num_rows, const void* ids,
                              int32_t ids_are_i64, int32_t per_row, const void* codes,
                              const uint16_t* scales, const int32_t* table, int32_t num_matrices,
                              int64_t k_rows, int64_t max_cols, int32_t group, void* y,
                              int64_t ldy, vmoe_stream_t stream) {
  int st = check_sizes(num_rows, num_matrices, per_row);
  if (st != VMOE_OK) return st;
  if (k_rows <= 0 || max_cols <= 0 || !codes || !scales || !table) return VMOE_ERR_INVALID_ARG;
  if (group != 32 && group != 64 && group != 128) return VMOE_ERR_INVALID_ARG;
  if (!ids && (num_matrices != 1 || per_row != 1)) return VMOE_ERR_INVALID_ARG;
  if (num_rows == 0) return VMOE_OK;
  if (k_rows % 8 || max_cols % 8 || k_rows > (1 << 24) || max_cols > (1 << 24) ||
      !aligned16(codes) || !aligned16(scales) || !aligned16(table))
    return VMOE_ERR_UNSUPPORTED;
  st = check_rows(num_rows, x, ldx, k_rows, y, ldy, max_cols, 8);
  if (st != VMOE_OK) return st;
  FewArgs p = {};
  p.w = {codes, scales, 0};
  p.tab = reinterpret_cast<const MatEntry*>(table);
  p.a = x;
  p.lda = ldx;
  p.T = (int)num_rows;
  p.k = per_row;
  p.E = num_matrices;
  p.ids = {ids, ids_are_i64};
  p.fixed = (int)k_rows;
  p.cols = (int)max_cols;
  p.out = y;
  p.ldo = ldy;
  p.wk = split_waves(div_up(k_rows, kQ4Rows));
  return launch_q4<2, kPlain, 1>(p, group, stream);
}
