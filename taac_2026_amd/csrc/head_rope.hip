// RMSNorm of every head of the queries and keys and the rotation by their positions, one pass over both; and its backward.
//
// Of a head's row x of d features, with u = x rsqrt(mean(x^2) + eps):   y = R(p) (w * u),   where R(p) turns the pairs (a, b) of the first
// `rotary` features by the table's (c, s) of position p, (a c - b s, a s + b c), and leaves the others. Pairs are neighbours (interleaved) or
// features rotary / 2 apart. Backward, with g the gradient of y and h = R(p)^T g:
//   dx = rstd (w h - u mean(w h u)),   dw = sum over all rows of h u;   without the norm dx = h.
//
// Bound by HBM: a row is read once and written once (backward: two reads and a write) and there are some ten operations to a feature. A lane holds
// four pairs of a row, i.e. two runs of four features: with the pairs half a head apart they are the two runs that belong together, so that the
// rotation never leaves the lane, and the sum of squares crosses d / 8 lanes. A wavefront's rows are heads of the same token, next to each other in memory and
// with one row of the table between them, or of a few tokens where a token has fewer heads. A lane keeps its head and walks the tokens: what a row costs besides
// its features is a few additions. All arithmetic is fp32, rounded once at the end.
//
// Measured: 1024 x 512 tokens of 16 heads of 32 features in bf16, 1.07 GB, 211 to 215 us, 5.0 TB/s, where torch's copy of as much takes 200 (with a product and two divisions to a
// row, an eighth more instructions, the same). 8 x 8192 tokens of 20 heads of 128: forward 146 us (4.6 TB/s), backward 200 (5.0), its partial rows 5.
#include "norm_rows.h"

namespace taac {
namespace {

constexpr int kMaxHeadWidth = 512;  // 64 lanes of 8 features
constexpr int kMaxHeads = 1 << 14;   // a wavefront each, at most, in the second dimension of a grid

constexpr int kForwardBlocks = 4096;  // 16 wavefronts to a SIMD; twice or four times as many, or half, are within what runs differ by

struct RopeParams {
  const void* x[2];       // queries, keys
  const void* g[2];       // backward: the gradients of the outputs
  void* y[2];             // outputs, or the gradients of x
  const void* w[2];       // [d] each, or null: no norm
  float* partial;         // backward: [workgroups][2][d]
  int64_t xs[2][3], gs[2][3], ys[2][3];  // element strides of (batch, head, token)
  const float* table;     // [places][rotary / 2][2]; null without places or rotation
  const void* positions;  // null: the position is the token's number
  int64_t ps[2];          // of (sample, token), words of 32 bits
  int64_t places;
  int32_t H[2], B, T, d, rotary;
  int32_t pos_int64, add_token;
  float eps, inv_d;
};

// How a lane reaches its features.
//   kSingles  one by one: the pairs s, s + L, ..
//   kRuns     two runs of four
//   kWide     eight neighbours of 16 bits in one access. Where pairs lie half a head apart two lanes, half of the turned ones apart, exchange four features for four.
// Eight bytes to a lane leave each access half of every line: 1024 x 512 tokens of 16 heads of 32 features take 233 us in runs, 209 wide.
enum { kSingles, kRuns, kWide };

// The four pairs of lane s of a row.
template <int L, int VEC, bool INTER>
struct Lane {
  int at[VEC != kSingles ? 2 : 8];  // features; -1: there is none
  int pair[4];          // of the table, -1: not turned
  int apart;            // kWide: lanes between the two that exchange
  bool gives_low;       // and which of its features this one gives
  // the lane whose runs this one has after an exchange
  __device__ __forceinline__ int run_lane(int s) const { return INTER || pair[0] < 0 ? s : pair[0] / 4; }
  __device__ __forceinline__ Lane(int s, int d, int rotary) {
    const int half = rotary / 2;
    if constexpr (VEC == kWide) {
      const bool turned = 8 * s < rotary, there = 8 * s < d;
      apart = rotary / 16;
      gives_low = turned && s >= apart;
      at[0] = there ? 8 * s : -1;
      at[1] = !INTER && turned ? 1 : 0;  // exchanges
      // the first of the two has the first four of its pairs, the second the last four
      const int first = INTER ? 4 * s : gives_low ? 8 * (s - apart) + 4 : 8 * s;
#pragma unroll
      for (int e = 0; e < 4; ++e) pair[e] = turned ? first + e : -1;
    } else if constexpr (VEC == kRuns) {
      const bool turned = 8 * s < rotary, there = 8 * s < d;
      at[0] = !there ? -1 : (turned && !INTER ? 4 * s : 8 * s);
      at[1] = !there ? -1 : (turned && !INTER ? half + 4 * s : 8 * s + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) pair[e] = turned ? 4 * s + e : -1;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int u = s + e * L;
        const bool turned = u < half;
        const int a = turned && !INTER ? u : 2 * u, b = turned && !INTER ? u + half : 2 * u + 1;
        at[2 * e] = a < d ? a : -1;
        at[2 * e + 1] = b < d ? b : -1;
        pair[e] = turned ? u : -1;
      }
    }
  }
};

template <typename T>
struct Run;  // four neighbouring features
template <>
struct Run<float> {
  typedef f32x4 type;
};
template <>
struct Run<bf16_t> {
  typedef bf16x4 type;
};
template <>
struct Run<f16_t> {
  typedef f16x4 type;
};

// Between the lanes s and s + apart, which hold features 8 s .. and half + 8 s ..: the one's last four for the other's first four, or back. Every lane of the
// wavefront that is on its way takes part; those that are not turned keep theirs.
template <int L, int VEC, bool INTER, typename V>
__device__ __forceinline__ void exchange(const Lane<L, VEC, INTER>& lane, V& first, V& second) {
  const u32x2 mine = __builtin_bit_cast(u32x2, lane.gives_low ? first : second);
  u32x2 other;
  if (L == 4 && lane.apart == 2) {  // heads of 32 features: within a quad
    other[0] = __builtin_amdgcn_mov_dpp(mine[0], 0x4e, 0xf, 0xf, false), other[1] = __builtin_amdgcn_mov_dpp(mine[1], 0x4e, 0xf, 0xf, false);
  } else {
    other[0] = __shfl_xor(mine[0], lane.apart, kWave), other[1] = __shfl_xor(mine[1], lane.apart, kWave);
  }
  if (lane.at[1] == 0) return;
  if (lane.gives_low) first = __builtin_bit_cast(V, other);
  else second = __builtin_bit_cast(V, other);
}

// A lane's features of a row as they arrive, converted when they are needed: the next row's are on their way meanwhile.
template <typename T, int L, int VEC, bool INTER>
struct Raw {
  typename Run<T>::type run[2];
  T one[8];
  __device__ __forceinline__ void load(const T* row, const Lane<L, VEC, INTER>& lane) {
    if constexpr (VEC == kWide) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (lane.at[0] >= 0) v = *reinterpret_cast<const u32x4*>(row + lane.at[0]);
      run[0] = __builtin_bit_cast(typename Run<T>::type, (u32x2{v[0], v[1]})), run[1] = __builtin_bit_cast(typename Run<T>::type, (u32x2{v[2], v[3]}));
    } else if constexpr (VEC == kRuns) {
      run[0] = typename Run<T>::type{}, run[1] = typename Run<T>::type{};
      if (lane.at[0] >= 0) {
        run[0] = *reinterpret_cast<const typename Run<T>::type*>(row + lane.at[0]);
        run[1] = *reinterpret_cast<const typename Run<T>::type*>(row + lane.at[1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) one[i] = lane.at[i] >= 0 ? row[lane.at[i]] : static_cast<T>(0.f);
    }
  }
  // v[2 e], v[2 e + 1]: pair e
  __device__ __forceinline__ void get(const Lane<L, VEC, INTER>& lane, float (&v)[8]) const {
    if constexpr (VEC != kSingles) {
      typename Run<T>::type first = run[0], second = run[1];
      if constexpr (VEC == kWide && !INTER) exchange(lane, first, second);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[INTER ? e : 2 * e] = static_cast<float>(first[e]);
        v[INTER ? 4 + e : 2 * e + 1] = static_cast<float>(second[e]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(one[i]);
    }
  }
};
template <typename T, int L, int VEC, bool INTER>
__device__ __forceinline__ void store_row(T* row, const Lane<L, VEC, INTER>& lane, const float (&v)[8]) {
  if constexpr (VEC != kSingles) {
    typename Run<T>::type a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] = static_cast<T>(v[INTER ? e : 2 * e]);
      b[e] = static_cast<T>(v[INTER ? 4 + e : 2 * e + 1]);
    }
    if constexpr (VEC == kWide) {
      if constexpr (!INTER) exchange(lane, a, b);
      const u32x2 x = __builtin_bit_cast(u32x2, a), y = __builtin_bit_cast(u32x2, b);
      if (lane.at[0] >= 0) *reinterpret_cast<u32x4*>(row + lane.at[0]) = u32x4{x[0], x[1], y[0], y[1]};
      return;
    }
    if (lane.at[0] >= 0) {
      *reinterpret_cast<typename Run<T>::type*>(row + lane.at[0]) = a;
      *reinterpret_cast<typename Run<T>::type*>(row + lane.at[1]) = b;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane.at[i] >= 0) row[lane.at[i]] = static_cast<T>(v[i]);
  }
}

// The tokens that a lane's row slot walks: heads of a token side by side in a wavefront, tokens a constant distance apart. Addresses move by a constant too, another one
// where the walk passes a sample's last token: a row costs no product and no division.
struct Walk {
  int which, h, t, step_t, left;  // left: tokens that are still to come, this one among them
  int64_t b, step_b;
  // slots: rows of a wavefront, of blockIdx.y's part of a token's heads where they need several wavefronts
  __device__ __forceinline__ Walk(const RopeParams& p, int slots, int slot) {
    const int heads = p.H[0] + p.H[1], side = heads < slots ? heads : slots;  // heads of a token in a wavefront
    const int at_once = slots / side;                                         // tokens of a wavefront
    const int head = static_cast<int>(blockIdx.y) * slots + slot % side, of = slot / side;
    which = head >= p.H[0];
    h = head - (which ? p.H[0] : 0);
    const int64_t wave = static_cast<int64_t>(blockIdx.x) * (kBlock / kWave) + threadIdx.x / kWave, token = wave * at_once + of;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (kBlock / kWave) * at_once, tokens = static_cast<int64_t>(p.B) * p.T;
    if (tokens < 0x7fffffff && step < 0x7fffffff) {  // the same for all: a fifth of the instructions
      const uint32_t T = p.T;
      b = static_cast<uint32_t>(token) / T, step_b = static_cast<uint32_t>(step) / T;
      left = token < tokens ? static_cast<int>((static_cast<uint32_t>(tokens - token) + static_cast<uint32_t>(step) - 1) / static_cast<uint32_t>(step)) : 0;
    } else {
      b = token / p.T, step_b = step / p.T;
      left = token < tokens ? static_cast<int>((tokens - token + step - 1) / step) : 0;
    }
    if (of >= at_once || head >= heads) left = 0;
    t = static_cast<int>(token - b * p.T), step_t = static_cast<int>(step - step_b * p.T);
  }
  // to the next token; whether that is behind the end of a sample more than step_b behind
  __device__ __forceinline__ bool next(const RopeParams& p) {
    --left;
    const uint32_t T = p.T, to = static_cast<uint32_t>(t) + static_cast<uint32_t>(step_t);  // below 2^32
    const bool wraps = to >= T;
    t = static_cast<int>(wraps ? to - T : to);
    return wraps;
  }
};
// The address of a walk's token in an array with strides of (sample, token), in elements of E.
template <typename E>
struct Cursor {
  E* p;
  int64_t plain, wrapped;  // elements to the next token
  __device__ __forceinline__ Cursor(E* base, const Walk& at, int T, int64_t sample, int64_t token) {
    p = base + at.b * sample + at.t * token;
    plain = at.step_b * sample + at.step_t * token;
    wrapped = plain + sample - T * token;
  }
  __device__ __forceinline__ void next(bool wraps) { p += wraps ? wrapped : plain; }
};
#define TAAC_ROWS(E, base, st) \
  Cursor<E>(static_cast<E*>(at.which ? base[1] : base[0]) + at.h * (at.which ? st[1][1] : st[0][1]), at, p.T, at.which ? st[1][0] : st[0][0], at.which ? st[1][2] : st[0][2])

// (c, s) of the lane's pairs; a position outside the table makes them NaN.
struct Angles {
  float c[4], s[4];
  bool inside;
  // without a branch, which would await what was asked for before it
  template <int L, int VEC, bool INTER>
  __device__ __forceinline__ void load(const RopeParams& p, const Walk& at, const Cursor<const int32_t>& place, const Lane<L, VEC, INTER>& lane) {
    if (p.rotary == 0) return;
    int64_t position = at.t;
    if (p.positions != nullptr) {
      position = p.pos_int64 ? *reinterpret_cast<const int64_t*>(place.p) : *place.p;
      if (p.add_token) position += at.t;
    }
    inside = position >= 0 && position < p.places;
    if (p.places == 0) return;
    const float* row = p.table + static_cast<uint64_t>(inside ? static_cast<uint32_t>(position) : 0u) * static_cast<uint32_t>(p.rotary);
    if constexpr (VEC != kSingles) {
      row += 2 * max(lane.pair[0], 0);
      const f32x4 lo = reinterpret_cast<const f32x4*>(row)[0], hi = reinterpret_cast<const f32x4*>(row)[1];
      c[0] = lo[0], s[0] = lo[1], c[1] = lo[2], s[1] = lo[3], c[2] = hi[0], s[2] = hi[1], c[3] = hi[2], s[3] = hi[3];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c[e] = row[2 * max(lane.pair[e], 0)];
        s[e] = row[2 * max(lane.pair[e], 0) + 1];
      }
    }
  }
  template <bool BACK, int L, int VEC, bool INTER>
  __device__ __forceinline__ void turn(const RopeParams& p, const Lane<L, VEC, INTER>& lane, float (&v)[8]) {
    if (p.rotary == 0 || (VEC != kSingles && lane.pair[0] < 0)) return;  // of runs all pairs are turned or none
    if (!inside) {
#pragma unroll
      for (int e = 0; e < 4; ++e) c[e] = s[e] = __builtin_nanf("");
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (VEC == kSingles && lane.pair[e] < 0) continue;
      const float a = v[2 * e], b = v[2 * e + 1];
      v[2 * e] = BACK ? fmaf(a, c[e], b * s[e]) : fmaf(a, c[e], -(b * s[e]));
      v[2 * e + 1] = BACK ? fmaf(b, c[e], -(a * s[e])) : fmaf(b, c[e], a * s[e]);
    }
  }
};

template <typename T, int L, int VEC, bool INTER>
__global__ __launch_bounds__(kBlock) void head_norm_rope_kernel(const RopeParams p) {
  const Lane<L, VEC, INTER> lane(threadIdx.x % L, p.d, p.rotary);
  const bool norm = p.w[0] != nullptr;
  Walk at(p, kWave / L, threadIdx.x % kWave / L);
  float w[8];
  Raw<T, L, VEC, INTER> next;
  if (norm) {
    next.load(static_cast<const T*>(at.which ? p.w[1] : p.w[0]), lane);
    next.get(lane, w);
  }
  if (at.left == 0) return;
  Cursor<const T> x = TAAC_ROWS(const T, p.x, p.xs);
  Cursor<T> y = TAAC_ROWS(T, p.y, p.ys);
  Cursor<const int32_t> place(static_cast<const int32_t*>(p.positions), at, p.T, p.ps[0], p.ps[1]);
  Angles angles;
  next.load(x.p, lane);
  angles.load(p, at, place, lane);
  while (true) {
    float v[8];
    next.get(lane, v);
    Angles now = angles;
    const bool wraps = at.next(p);
    if (at.left > 0) {
      x.next(wraps), place.next(wraps);
      next.load(x.p, lane);
      angles.load(p, at, place, lane);
    }
    if (norm) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(v[i], v[i], sum);
      const float rstd = rsqrtf(fmaf(group_sum<L>(sum), p.inv_d, p.eps));
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= rstd * w[i];
    }
    now.template turn<false>(p, lane, v);
    store_row<T, L, VEC, INTER>(y.p, lane, v);
    if (at.left == 0) return;
    y.next(wraps);
  }
}

template <typename T, int L, int VEC, bool INTER>
__global__ __launch_bounds__(kBlock) void head_norm_rope_bwd_kernel(const RopeParams p) {
  __shared__ float red[kBlock / kWave][2][kMaxHeadWidth];
  const Lane<L, VEC, INTER> lane(threadIdx.x % L, p.d, p.rotary);
  const bool norm = p.w[0] != nullptr;
  Walk at(p, kWave / L, threadIdx.x % kWave / L);
  float w[8], dw[2][8];
  Raw<T, L, VEC, INTER> next, next_g;
  if (norm) {
    next.load(static_cast<const T*>(at.which ? p.w[1] : p.w[0]), lane);
    next.get(lane, w);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[0][i] = dw[1][i] = 0.f;
  if (at.left > 0) {
    Cursor<const T> dy = TAAC_ROWS(const T, p.g, p.gs), x = TAAC_ROWS(const T, p.x, p.xs);
    Cursor<T> dx = TAAC_ROWS(T, p.y, p.ys);
    Cursor<const int32_t> place(static_cast<const int32_t*>(p.positions), at, p.T, p.ps[0], p.ps[1]);
    Angles angles;
    next_g.load(dy.p, lane);
    if (norm) next.load(x.p, lane);
    angles.load(p, at, place, lane);
    while (true) {
      float g[8], u[8];
      next_g.get(lane, g);
      if (norm) next.get(lane, u);
      Angles now = angles;
      const bool wraps = at.next(p);
      if (at.left > 0) {
        dy.next(wraps), x.next(wraps), place.next(wraps);
        next_g.load(dy.p, lane);
        if (norm) next.load(x.p, lane);
        angles.load(p, at, place, lane);
      }
      now.template turn<true>(p, lane, g);
      if (norm) {
        float sum = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sum = fmaf(u[i], u[i], sum);
          dot = fmaf(g[i] * w[i], u[i], dot);
        }
        const float rstd = rsqrtf(fmaf(group_sum<L>(sum), p.inv_d, p.eps));
        const float mean = group_sum<L>(dot) * rstd * p.inv_d;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          u[i] *= rstd;
          dw[0][i] = fmaf(g[i], u[i], dw[0][i]);
          g[i] = rstd * (g[i] * w[i] - u[i] * mean);
        }
      }
      store_row<T, L, VEC, INTER>(dx.p, lane, g);
      if (at.left == 0) break;
      dx.next(wraps);
    }
  }
  if (!norm) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[1][i] = at.which ? dw[0][i] : 0.f, dw[0][i] = at.which ? 0.f : dw[0][i];
  // the lanes that hold the same features, then the wavefronts, in a fixed order
#pragma unroll
  for (int off = L; off < kWave; off *= 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dw[0][i] += __shfl_xor(dw[0][i], off, kWave);
      dw[1][i] += __shfl_xor(dw[1][i], off, kWave);
    }
  }
  const int wave = threadIdx.x / kWave;
  if (threadIdx.x % kWave < L) {
    // as singles or runs: the lanes of wide accesses hold the runs of lanes that exchanged
    const Lane<L, VEC == kWide ? kRuns : VEC, INTER> plain(VEC == kWide ? lane.run_lane(threadIdx.x % L) : threadIdx.x % L, p.d, p.rotary);
    store_row<float, L, VEC == kWide ? kRuns : VEC, INTER>(red[wave][0], plain, dw[0]);
    store_row<float, L, VEC == kWide ? kRuns : VEC, INTER>(red[wave][1], plain, dw[1]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.d; i += kBlock) {
    const int which = i >= p.d, c = i - which * p.d;
    float total = 0.f;
#pragma unroll
    for (int v = 0; v < kBlock / kWave; ++v) total += red[v][which][c];
    p.partial[((static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * 2 + which) * p.d + c] = total;
  }
}

int lanes_of(int32_t d) {
  int lanes = 4;
  while (lanes * 8 < d) lanes *= 2;
  return lanes;
}
// Workgroups over the tokens, and over the heads where a token's need several wavefronts. A backward pass with weights has kBwdMaxBlocks at most, a partial row of both
// gradients each.
struct Grid {
  int64_t x;
  int32_t y;
};
Grid grid_of(int64_t tokens, int32_t heads, int32_t d, bool back) {
  const int slots = kWave / lanes_of(d), side = heads < slots ? heads : slots, at_once = slots / side * (kBlock / kWave);
  Grid grid{(tokens + at_once - 1) / at_once, (heads + slots - 1) / slots};
  // chunks of heads that are more than that (wide heads in great number) stay: a workgroup each
  const int64_t all = back ? kBwdMaxBlocks : kForwardBlocks, most = all > grid.y ? all / grid.y : 1;
  if (grid.x > most) grid.x = most;
  return grid;
}

template <typename T, int VEC, bool INTER>
void launch_rope(const RopeParams& p, bool back, hipStream_t s) {
  const int lanes = lanes_of(p.d);
  const Grid blocks = grid_of(static_cast<int64_t>(p.B) * p.T, p.H[0] + p.H[1], p.d, back);
  const dim3 grid(static_cast<uint32_t>(blocks.x), static_cast<uint32_t>(blocks.y));
#define TAAC_ROPE(L)                                                                                              \
  if (lanes == L) {                                                                                               \
    if (back) hipLaunchKernelGGL((head_norm_rope_bwd_kernel<T, L, VEC, INTER>), grid, dim3(kBlock), 0, s, p);     \
    else hipLaunchKernelGGL((head_norm_rope_kernel<T, L, VEC, INTER>), grid, dim3(kBlock), 0, s, p);              \
  }
  TAAC_ROPE(4) TAAC_ROPE(8) TAAC_ROPE(16) TAAC_ROPE(32) TAAC_ROPE(64)
#undef TAAC_ROPE
}

template <typename T>
void dispatch_rope(const RopeParams& p, bool interleaved, bool back, hipStream_t s) {
  // What strides, addresses and widths allow: eight bytes to a run (16 of fp32), sixteen to a lane where lanes that exchange are a power of two apart.
  constexpr int WIDE = sizeof(T) == 2 ? 8 : 4;
  int run = p.d % 8 == 0 && p.rotary % 8 == 0 ? WIDE : 1;
  auto allow = [&](const void* ptr, const int64_t (&st)[3]) {
    for (int64_t s : {static_cast<int64_t>(reinterpret_cast<uintptr_t>(ptr) / sizeof(T)), st[0], st[1], st[2]})
      while (s % run != 0) run /= 2;
  };
  const int64_t none[3] = {0, 0, 0};
  for (int i = 0; i < 2; ++i) {
    allow(p.x[i], p.xs[i]), allow(p.y[i], p.ys[i]), allow(p.w[i], none);
    if (back) allow(p.g[i], p.gs[i]);
  }
  if (!aligned16(p.table)) run = 1;
  const bool exchanges = interleaved || (p.rotary % 16 == 0 && (p.rotary / 16 & (p.rotary / 16 - 1)) == 0);
  if constexpr (WIDE == 8) {
    if (run == 8 && exchanges) return interleaved ? launch_rope<T, kWide, true>(p, back, s) : launch_rope<T, kWide, false>(p, back, s);
  }
  if (run >= 4) interleaved ? launch_rope<T, kRuns, true>(p, back, s) : launch_rope<T, kRuns, false>(p, back, s);
  else interleaved ? launch_rope<T, kSingles, true>(p, back, s) : launch_rope<T, kSingles, false>(p, back, s);
}

int take_rope(const char* name, RopeParams& p, const void* q, const void* k, void* q_out, void* k_out, int32_t B, int32_t H, int32_t key_heads, int32_t T,
              int32_t d, int32_t rotary, const int64_t* qs, const int64_t* ks, const int64_t* qos, const int64_t* kos, const void* qw, const void* kw,
              float eps, const float* table, int64_t places, const void* positions, int pos_int64, const int64_t* ps, int add_token, int dtype, bool* empty) {
  if (B < 0 || T < 0 || H <= 0 || key_heads <= 0 || d <= 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: batch and tokens must be >= 0, heads and width > 0", name);
  if (d > kMaxHeadWidth) return set_error(TAAC_ERR_UNSUPPORTED, "%s: a head has at most %d features (got %d)", name, kMaxHeadWidth, d);
  if (H > kMaxHeads || key_heads > kMaxHeads) return set_error(TAAC_ERR_UNSUPPORTED, "%s: at most %d heads", name, kMaxHeads);
  if (rotary < 0 || rotary > d || rotary % 2 != 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: the rotated features must be an even number, at most the head's (got %d of %d)", name, rotary, d);
  // a table of no places may have no address
  if (places < 0 || (table != nullptr && rotary == 0) || (table == nullptr && rotary > 0 && places > 0)) return set_error(TAAC_ERR_INVALID_VALUE, "%s: a table comes with rotated features, its size not negative", name);
  if (places > 0x7fffffff) return set_error(TAAC_ERR_UNSUPPORTED, "%s: a table has at most 2^31 - 1 positions", name);
  if ((qw == nullptr) != (kw == nullptr)) return set_error(TAAC_ERR_INVALID_VALUE, "%s: both norm weights or neither", name);
  if (dtype != TAAC_F32 && dtype != TAAC_BF16 && dtype != TAAC_F16) return set_error(TAAC_ERR_INVALID_VALUE, "%s: unknown dtype %d", name, dtype);
  if (!(eps >= 0.f)) return set_error(TAAC_ERR_INVALID_VALUE, "%s: eps must not be negative", name);
  const int64_t* from[4] = {qs, ks, qos, kos};
  int64_t* to[4] = {p.xs[0], p.xs[1], p.ys[0], p.ys[1]};
  for (int i = 0; i < 4; ++i) {
    if (from[i] == nullptr) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null strides", name);
    for (int j = 0; j < 3; ++j) to[i][j] = from[i][j];
  }
  if (positions != nullptr) {
    if (ps == nullptr) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null strides of the positions", name);
    const int64_t words = pos_int64 ? 2 : 1;  // of 32 bits
    p.ps[0] = ps[0] * words, p.ps[1] = ps[1] * words;
  }
  *empty = B == 0 || T == 0;
  if (*empty) return TAAC_OK;
  if (!q || !k || !q_out || !k_out) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null tensor pointer", name);
  if (table != nullptr && reinterpret_cast<uintptr_t>(table) % 4 != 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: misaligned table", name);
  p.x[0] = q, p.x[1] = k, p.y[0] = q_out, p.y[1] = k_out, p.w[0] = qw, p.w[1] = kw;
  p.table = table, p.places = places, p.positions = positions, p.pos_int64 = pos_int64 != 0, p.add_token = add_token != 0;
  p.H[0] = H, p.H[1] = key_heads, p.B = B, p.T = T, p.d = d, p.rotary = rotary, p.eps = eps, p.inv_d = 1.f / static_cast<float>(d);
  return TAAC_OK;
}

void dispatch_dtype(const RopeParams& p, bool interleaved, bool back, int dtype, hipStream_t s) {
  if (dtype == TAAC_F32) dispatch_rope<float>(p, interleaved, back, s);
  if (dtype == TAAC_BF16) dispatch_rope<bf16_t>(p, interleaved, back, s);
  if (dtype == TAAC_F16) dispatch_rope<f16_t>(p, interleaved, back, s);
}

// dw = the workgroups' partial rows added in a fixed order: sixteen columns to a workgroup, 64 slices of the rows.
template <typename T>
__global__ __launch_bounds__(1024) void head_weights_kernel(const float* __restrict__ partial, int blocks, int d, T* __restrict__ dqw, T* __restrict__ dkw) {
  __shared__ float red[64][16];
  const int column = threadIdx.x % 16, slice = threadIdx.x / 16, c = blockIdx.x * 16 + column;
  float sum = 0.f;
  if (c < 2 * d) {
#pragma unroll 4
    for (int i = slice; i < blocks; i += 64) sum += partial[static_cast<int64_t>(i) * 2 * d + c];
  }
  red[slice][column] = sum;
  __syncthreads();
  if (slice >= 4) return;  // one wavefront
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += red[slice + 4 * i][column];
  sum += __shfl_xor(sum, 16, kWave);
  sum += __shfl_xor(sum, 32, kWave);
  if (slice > 0 || c >= 2 * d) return;
  if (c < d) dqw[c] = static_cast<T>(sum);
  else dkw[c - d] = static_cast<T>(sum);
}

template <typename T>
void reduce_weights(const RopeParams& p, int blocks, void* dqw, void* dkw, hipStream_t s) {
  hipLaunchKernelGGL(head_weights_kernel<T>, dim3((2 * p.d + 15) / 16), dim3(1024), 0, s, p.partial, blocks, p.d, static_cast<T*>(dqw), static_cast<T*>(dkw));
}

}  // namespace
}  // namespace taac

extern "C" int taac_head_norm_rope_fwd(const void* q, const void* k, void* q_out, void* k_out, int32_t B, int32_t H, int32_t key_heads, int32_t T, int32_t d,
                                       int32_t rotary, const int64_t q_strides[3], const int64_t k_strides[3], const int64_t qo_strides[3],
                                       const int64_t ko_strides[3], const void* q_weight, const void* k_weight, float eps, const float* table,
                                       int64_t places, const void* positions, int positions_int64, const int64_t position_strides[2], int add_token,
                                       int interleaved, int dtype, void* stream) {
  using namespace taac;
  RopeParams p{};
  bool empty = false;
  const char* name = "taac_head_norm_rope_fwd";
  if (int rc = take_rope(name, p, q, k, q_out, k_out, B, H, key_heads, T, d, rotary, q_strides, k_strides, qo_strides, ko_strides, q_weight, k_weight, eps,
                         table, places, positions, positions_int64, position_strides, add_token, dtype, &empty))
    return rc;
  if (empty) return TAAC_OK;
  dispatch_dtype(p, interleaved != 0, false, dtype, as_stream(stream));
  return check_launch(name);
}

extern "C" int64_t taac_head_norm_rope_bwd_workspace_floats(int32_t B, int32_t H, int32_t key_heads, int32_t T, int32_t d) {
  using namespace taac;
  if (B < 0 || T < 0 || H <= 0 || key_heads <= 0 || d <= 0 || d > kMaxHeadWidth || H > kMaxHeads || key_heads > kMaxHeads) return -1;
  const Grid grid = grid_of(static_cast<int64_t>(B) * T, H + key_heads, d, true);
  return grid.x * grid.y * 2 * d;
}

extern "C" int taac_head_norm_rope_bwd(const void* q, const void* k, const void* grad_qo, const void* grad_ko, void* grad_q, void* grad_k, void* grad_qw,
                                       void* grad_kw, float* workspace, int64_t workspace_floats, int32_t B, int32_t H, int32_t key_heads, int32_t T,
                                       int32_t d, int32_t rotary, const int64_t q_strides[3], const int64_t k_strides[3], const int64_t gqo_strides[3],
                                       const int64_t gko_strides[3], const int64_t gq_strides[3], const int64_t gk_strides[3], const void* q_weight,
                                       const void* k_weight, float eps, const float* table, int64_t places, const void* positions, int positions_int64,
                                       const int64_t position_strides[2], int add_token, int interleaved, int dtype, void* stream) {
  using namespace taac;
  RopeParams p{};
  bool empty = false;
  const char* name = "taac_head_norm_rope_bwd";
  if (int rc = take_rope(name, p, q, k, grad_q, grad_k, B, H, key_heads, T, d, rotary, q_strides, k_strides, gq_strides, gk_strides, q_weight, k_weight, eps,
                         table, places, positions, positions_int64, position_strides, add_token, dtype, &empty))
    return rc;
  if (gqo_strides == nullptr || gko_strides == nullptr) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null strides", name);
  for (int j = 0; j < 3; ++j) p.gs[0][j] = gqo_strides[j], p.gs[1][j] = gko_strides[j];
  const bool norm = q_weight != nullptr;
  if (norm && (!grad_qw || !grad_kw)) return set_error(TAAC_ERR_INVALID_VALUE, "%s: the weights have gradients", name);
  if (!empty && (!grad_qo || !grad_ko)) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null tensor pointer", name);
  const int64_t need = taac_head_norm_rope_bwd_workspace_floats(B, H, key_heads, T, d);
  if (norm && need > 0 && (workspace == nullptr || workspace_floats < need || reinterpret_cast<uintptr_t>(workspace) % 4 != 0))
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: workspace must hold %lld floats", name, (long long)need);
  if (empty && !norm) return TAAC_OK;
  p.g[0] = grad_qo, p.g[1] = grad_ko, p.partial = workspace, p.d = d;
  hipStream_t s = as_stream(stream);
  if (!empty) dispatch_dtype(p, interleaved != 0, true, dtype, s);
  if (norm) {  // zeros where there are no rows
    const int blocks = static_cast<int>(need / (2 * d));
    if (dtype == TAAC_F32) reduce_weights<float>(p, blocks, grad_qw, grad_kw, s);
    if (dtype == TAAC_BF16) reduce_weights<bf16_t>(p, blocks, grad_qw, grad_kw, s);
    if (dtype == TAAC_F16) reduce_weights<f16_t>(p, blocks, grad_qw, grad_kw, s);
  }
  return check_launch(name);
}
