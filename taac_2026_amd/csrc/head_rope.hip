// RMSNorm of every head of the queries and keys and the rotation by their positions, one pass over both; and its backward.
//
// Of a head's row x of d features, with u = x rsqrt(mean(x^2) + eps):   y = R(p) (w * u),   where R(p) turns the pairs (a, b) of the first
// `rotary` features by the table's (c, s) of position p, (a c - b s, a s + b c), and leaves the others. Pairs are neighbours (interleaved) or
// features rotary / 2 apart. Backward, with g the gradient of y and h = R(p)^T g:
//   dx = rstd (w h - u mean(w h u)),   dw = sum over all rows of h u;   without the norm dx = h.
//
// Bound by HBM: a row is read once and written once (backward: two reads and a write) and there are some ten operations to a feature. A lane holds
// four pairs of a row, i.e. two runs of four features: with the pairs half a head apart they are the two runs that belong together, so that the
// rotation never leaves the lane, and the sum of squares crosses d / 8 lanes. The rows of a token's heads lie next to each other in lanes, and share
// their row of the table through the caches. All arithmetic is fp32, rounded once at the end.
#include "norm_rows.h"

namespace taac {
namespace {

constexpr int kMaxHeadWidth = 512;  // 64 lanes of 8 features

struct RopeParams {
  const void* x[2];       // queries, keys
  const void* g[2];       // backward: the gradients of the outputs
  void* y[2];             // outputs, or the gradients of x
  const void* w[2];       // [d] each, or null: no norm
  float* partial;         // backward: [workgroups][2][d]
  int64_t xs[2][3], gs[2][3], ys[2][3];  // element strides of (batch, head, token)
  const float* table;     // [places][rotary / 2][2] or null
  const void* positions;  // null: the position is the token's number
  int64_t ps[2];
  int64_t places, rows;   // rows of queries and keys together
  int32_t H[2], T, d, rotary;
  int32_t pos_int64, add_token;
  float eps;
};

// The four pairs of lane s of a row. In vectors: two runs of four features at `at[0]` and `at[1]`; else the pairs s, s + L, ..
template <int L, bool VEC, bool INTER>
struct Lane {
  int at[VEC ? 2 : 8];  // features; -1: there is none
  int pair[4];          // of the table, -1: not turned
  __device__ __forceinline__ Lane(int s, int d, int rotary) {
    const int half = rotary / 2;
    if constexpr (VEC) {
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

// v[2 e], v[2 e + 1]: pair e.
template <typename T, int L, bool VEC, bool INTER>
__device__ __forceinline__ void load_row(const T* row, const Lane<L, VEC, INTER>& lane, float (&v)[8]) {
  if constexpr (VEC) {
    typename Run<T>::type a = {}, b = {};
    if (lane.at[0] >= 0) {
      a = *reinterpret_cast<const typename Run<T>::type*>(row + lane.at[0]);
      b = *reinterpret_cast<const typename Run<T>::type*>(row + lane.at[1]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[INTER ? e : 2 * e] = static_cast<float>(a[e]);
      v[INTER ? 4 + e : 2 * e + 1] = static_cast<float>(b[e]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = lane.at[i] >= 0 ? static_cast<float>(row[lane.at[i]]) : 0.f;
  }
}
template <typename T, int L, bool VEC, bool INTER>
__device__ __forceinline__ void store_row(T* row, const Lane<L, VEC, INTER>& lane, const float (&v)[8]) {
  if constexpr (VEC) {
    typename Run<T>::type a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] = static_cast<T>(v[INTER ? e : 2 * e]);
      b[e] = static_cast<T>(v[INTER ? 4 + e : 2 * e + 1]);
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

// Where a row is: which of queries and keys, and its sample, token and head.
struct Place {
  int which, h, t;
  int64_t b;
  __device__ __forceinline__ Place(const RopeParams& p, int64_t row) {
    const uint32_t heads = p.H[0] + p.H[1];
    int64_t token;
    uint32_t head;
    if (p.rows < (int64_t{1} << 32)) {  // the same branch for all: 32-bit divisions are a third of the instructions
      token = static_cast<uint32_t>(row) / heads;
      head = static_cast<uint32_t>(row) - static_cast<uint32_t>(token) * heads;
      b = static_cast<uint32_t>(token) / static_cast<uint32_t>(p.T);
    } else {
      token = row / heads;
      head = static_cast<uint32_t>(row - token * heads);
      b = token / p.T;
    }
    t = static_cast<int>(token - b * p.T);
    which = head >= static_cast<uint32_t>(p.H[0]);
    h = static_cast<int>(head) - (which ? p.H[0] : 0);
  }
  __device__ __forceinline__ int64_t offset(const int64_t (&s)[2][3]) const {
    const int64_t *q = s[0], *k = s[1];
    return b * (which ? k[0] : q[0]) + h * (which ? k[1] : q[1]) + t * (which ? k[2] : q[2]);
  }
};

// (c, s) of the lane's pairs; a position outside the table makes them NaN.
template <int L, bool VEC, bool INTER>
__device__ __forceinline__ void load_angles(const RopeParams& p, const Place& at, const Lane<L, VEC, INTER>& lane, float (&c)[4], float (&s)[4]) {
  if (p.table == nullptr) return;
  int64_t position = at.t;
  if (p.positions != nullptr) {
    const int64_t i = at.b * p.ps[0] + at.t * p.ps[1];
    position = p.pos_int64 ? static_cast<const int64_t*>(p.positions)[i] : static_cast<const int32_t*>(p.positions)[i];
    if (p.add_token) position += at.t;
  }
  const bool inside = position >= 0 && position < p.places;
  const float* row = p.table + (inside ? position : 0) * p.rotary;
  if constexpr (VEC) {
    f32x4 lo = {}, hi = {};
    if (lane.pair[0] >= 0) {
      lo = *reinterpret_cast<const f32x4*>(row + 2 * lane.pair[0]);
      hi = *reinterpret_cast<const f32x4*>(row + 2 * lane.pair[0] + 4);
    }
    c[0] = lo[0], s[0] = lo[1], c[1] = lo[2], s[1] = lo[3], c[2] = hi[0], s[2] = hi[1], c[3] = hi[2], s[3] = hi[3];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      c[e] = lane.pair[e] >= 0 ? row[2 * lane.pair[e]] : 0.f;
      s[e] = lane.pair[e] >= 0 ? row[2 * lane.pair[e] + 1] : 0.f;
    }
  }
  if (!inside) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = s[e] = __builtin_nanf("");
  }
}

// sign 1: by the angles, -1: back.
template <int L, bool VEC, bool INTER>
__device__ __forceinline__ void turn(const RopeParams& p, const Lane<L, VEC, INTER>& lane, const float (&c)[4], const float (&s)[4], float sign, float (&v)[8]) {
  if (p.table == nullptr) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float a = v[2 * e], b = v[2 * e + 1], sn = sign * s[e];
    if (lane.pair[e] >= 0) {
      v[2 * e] = fmaf(a, c[e], -(b * sn));
      v[2 * e + 1] = fmaf(a, sn, b * c[e]);
    }
  }
}

template <typename T, int L, bool VEC, bool INTER>
__global__ __launch_bounds__(kBlock) void head_norm_rope_kernel(const RopeParams p) {
  constexpr int ROWS = kBlock / L;
  const Lane<L, VEC, INTER> lane(threadIdx.x % L, p.d, p.rotary);
  const bool norm = p.w[0] != nullptr;
  float w[2][8];
  if (norm) {
    load_row<T, L, VEC, INTER>(static_cast<const T*>(p.w[0]), lane, w[0]);
    load_row<T, L, VEC, INTER>(static_cast<const T*>(p.w[1]), lane, w[1]);
  }
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / L; row < p.rows; row += static_cast<int64_t>(gridDim.x) * ROWS) {
    const Place at(p, row);
    float v[8], c[4], s[4];
    load_row<T, L, VEC, INTER>(static_cast<const T*>(at.which ? p.x[1] : p.x[0]) + at.offset(p.xs), lane, v);
    load_angles(p, at, lane, c, s);
    if (norm) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(v[i], v[i], sum);
      const float rstd = 1.f / sqrtf(group_sum<L>(sum) / p.d + p.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= rstd * (at.which ? w[1][i] : w[0][i]);
    }
    turn(p, lane, c, s, 1.f, v);
    store_row<T, L, VEC, INTER>(static_cast<T*>(at.which ? p.y[1] : p.y[0]) + at.offset(p.ys), lane, v);
  }
}

template <typename T, int L, bool VEC, bool INTER>
__global__ __launch_bounds__(kBlock) void head_norm_rope_bwd_kernel(const RopeParams p) {
  constexpr int ROWS = kBlock / L;
  __shared__ float red[kBlock / kWave][2][kMaxHeadWidth];
  const Lane<L, VEC, INTER> lane(threadIdx.x % L, p.d, p.rotary);
  const bool norm = p.w[0] != nullptr;
  float w[2][8], dw[2][8];
  if (norm) {
    load_row<T, L, VEC, INTER>(static_cast<const T*>(p.w[0]), lane, w[0]);
    load_row<T, L, VEC, INTER>(static_cast<const T*>(p.w[1]), lane, w[1]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[0][i] = dw[1][i] = 0.f;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / L; row < p.rows; row += static_cast<int64_t>(gridDim.x) * ROWS) {
    const Place at(p, row);
    float g[8], c[4], s[4];
    load_row<T, L, VEC, INTER>(static_cast<const T*>(at.which ? p.g[1] : p.g[0]) + at.offset(p.gs), lane, g);
    load_angles(p, at, lane, c, s);
    if (norm) {
      float x[8];
      load_row<T, L, VEC, INTER>(static_cast<const T*>(at.which ? p.x[1] : p.x[0]) + at.offset(p.xs), lane, x);
      turn(p, lane, c, s, -1.f, g);
      float sum = 0.f, dot = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum = fmaf(x[i], x[i], sum);
        dot = fmaf(g[i] * (at.which ? w[1][i] : w[0][i]), x[i], dot);
      }
      const float rstd = 1.f / sqrtf(group_sum<L>(sum) / p.d + p.eps);
      const float mean = group_sum<L>(dot) * rstd / p.d;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = x[i] * rstd, part = g[i] * u;
        dw[0][i] += at.which ? 0.f : part;
        dw[1][i] += at.which ? part : 0.f;
        g[i] = rstd * (g[i] * (at.which ? w[1][i] : w[0][i]) - u * mean);
      }
    } else {
      turn(p, lane, c, s, -1.f, g);
    }
    store_row<T, L, VEC, INTER>(static_cast<T*>(at.which ? p.y[1] : p.y[0]) + at.offset(p.ys), lane, g);
  }
  if (!norm) return;
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
    store_row<float, L, VEC, INTER>(red[wave][0], lane, dw[0]);
    store_row<float, L, VEC, INTER>(red[wave][1], lane, dw[1]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.d; i += kBlock) {
    const int which = i >= p.d, c = i - which * p.d;
    float total = 0.f;
#pragma unroll
    for (int v = 0; v < kBlock / kWave; ++v) total += red[v][which][c];
    p.partial[(static_cast<int64_t>(blockIdx.x) * 2 + which) * p.d + c] = total;
  }
}

// Workgroups of a backward pass with weights: one partial row of both gradients each.
int64_t bwd_blocks(int64_t rows, int lanes) {
  const int64_t blocks = (rows + kBlock / lanes - 1) / (kBlock / lanes);
  return blocks < kBwdMaxBlocks ? blocks : kBwdMaxBlocks;
}
int lanes_of(int32_t d) {
  int lanes = 4;
  while (lanes * 8 < d) lanes *= 2;
  return lanes;
}

template <typename T, bool VEC, bool INTER>
void launch_rope(const RopeParams& p, bool back, hipStream_t s) {
  const int lanes = lanes_of(p.d);
  const int64_t blocks = (p.rows + kBlock / lanes - 1) / (kBlock / lanes);
  const dim3 grid(static_cast<uint32_t>(back ? bwd_blocks(p.rows, lanes) : (blocks < (1 << 20) ? blocks : 1 << 20)));
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
  // Runs of four features: 8 bytes, 16 of fp32, aligned.
  bool vec = p.d % 8 == 0 && p.rotary % 8 == 0;
  auto aligned = [&](const void* ptr) { vec &= reinterpret_cast<uintptr_t>(ptr) % (4 * sizeof(T)) == 0; };
  auto strided = [&](const int64_t (&st)[3]) { vec &= st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0; };
  for (int i = 0; i < 2; ++i) {
    aligned(p.x[i]), aligned(p.y[i]), aligned(p.w[i]), strided(p.xs[i]), strided(p.ys[i]);
    if (back) aligned(p.g[i]), strided(p.gs[i]);
  }
  vec &= aligned16(p.table);
  if (vec) interleaved ? launch_rope<T, true, true>(p, back, s) : launch_rope<T, true, false>(p, back, s);
  else interleaved ? launch_rope<T, false, true>(p, back, s) : launch_rope<T, false, false>(p, back, s);
}

int take_rope(const char* name, RopeParams& p, const void* q, const void* k, void* q_out, void* k_out, int32_t B, int32_t H, int32_t key_heads, int32_t T,
              int32_t d, int32_t rotary, const int64_t* qs, const int64_t* ks, const int64_t* qos, const int64_t* kos, const void* qw, const void* kw,
              float eps, const float* table, int64_t places, const void* positions, int pos_int64, const int64_t* ps, int add_token, int dtype, bool* empty) {
  if (B < 0 || T < 0 || H <= 0 || key_heads <= 0 || d <= 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: batch and tokens must be >= 0, heads and width > 0", name);
  if (d > kMaxHeadWidth) return set_error(TAAC_ERR_UNSUPPORTED, "%s: a head has at most %d features (got %d)", name, kMaxHeadWidth, d);
  if (H > 1 << 20 || key_heads > 1 << 20) return set_error(TAAC_ERR_UNSUPPORTED, "%s: at most 2^20 heads", name);
  if (rotary < 0 || rotary > d || rotary % 2 != 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: the rotated features must be an even number, at most the head's (got %d of %d)", name, rotary, d);
  if ((rotary > 0) != (table != nullptr) || places < 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: a table comes with rotated features, its size not negative", name);
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
    p.ps[0] = ps[0], p.ps[1] = ps[1];
  }
  *empty = B == 0 || T == 0;
  if (*empty) return TAAC_OK;
  if (!q || !k || !q_out || !k_out) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null tensor pointer", name);
  if (table != nullptr && reinterpret_cast<uintptr_t>(table) % 4 != 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: misaligned table", name);
  p.x[0] = q, p.x[1] = k, p.y[0] = q_out, p.y[1] = k_out, p.w[0] = qw, p.w[1] = kw;
  p.table = table, p.places = places, p.positions = positions, p.pos_int64 = pos_int64 != 0, p.add_token = add_token != 0;
  p.rows = static_cast<int64_t>(B) * T * (static_cast<int64_t>(H) + key_heads);
  p.H[0] = H, p.H[1] = key_heads, p.T = T, p.d = d, p.rotary = rotary, p.eps = eps;
  return TAAC_OK;
}

void dispatch_dtype(const RopeParams& p, bool interleaved, bool back, int dtype, hipStream_t s) {
  if (dtype == TAAC_F32) dispatch_rope<float>(p, interleaved, back, s);
  if (dtype == TAAC_BF16) dispatch_rope<bf16_t>(p, interleaved, back, s);
  if (dtype == TAAC_F16) dispatch_rope<f16_t>(p, interleaved, back, s);
}

template <typename T>
void reduce_weights(const RopeParams& p, int blocks, void* dqw, void* dkw, hipStream_t s) {
  hipLaunchKernelGGL(norm_bwd_reduce_kernel<T>, dim3((p.d + 15) / 16), dim3(kBlock), 0, s, p.partial, blocks, p.d, 2, static_cast<T*>(dqw), static_cast<T*>(dkw));
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
  if (B < 0 || T < 0 || H <= 0 || key_heads <= 0 || d <= 0 || d > kMaxHeadWidth) return -1;
  return bwd_blocks(static_cast<int64_t>(B) * T * (static_cast<int64_t>(H) + key_heads), lanes_of(d)) * 2 * d;
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
