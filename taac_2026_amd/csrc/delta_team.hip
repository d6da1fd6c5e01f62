// Gated delta rule, chunked form, for few heads and long histories (the mathematics, operand order and precision: delta.h).
//
// With few (sample, head) pairs the time is the chain of chunks, not the work: what does not depend on the state is made for all
// chunks at once (one wavefront each) and left in memory, and a chunk's step of the state is spread over four wavefronts to make it
// short. A workgroup has 16 value columns; wavefront w owns tokens 16 w .. 16 w + 15 of every chunk and a quarter of the key rows
// of the state. A step is three stages with a barrier behind each,
//   X (own tokens) from the state | N (own tokens) from X | the state (own rows) from N; the output beside them,
// whose results meet in LDS as operand fragments. Everything a chunk reads from memory is requested one chunk ahead.
#include "delta.h"

namespace taac {
namespace {

template <int DK, bool COLS>
__global__ __launch_bounds__(kWave) void delta_blocks_kernel(const DeltaParams p) {
  __shared__ __attribute__((aligned(16))) float rows[kRowFloats];
  __shared__ __attribute__((aligned(16))) float temp[kTempFloats];
  __shared__ __attribute__((aligned(16))) float scratch[kScratchFloats];
  const int chunk = static_cast<int>(blockIdx.x % p.chunks);
  const int64_t unit = blockIdx.x / p.chunks;
  const int h = static_cast<int>(unit % p.H);
  const int b = static_cast<int>(unit / p.H);
  int len = p.T;
  if (p.lengths != nullptr) len = p.lengths[b] < p.T ? p.lengths[b] : p.T;
  const int64_t token0 = static_cast<int64_t>(chunk) * kChunk;
  const int64_t left = len - token0;
  if (left <= 0) return;
  uint8_t* block = p.blocks + (unit * p.chunks + chunk) * kBlockBytes;
  chunk_block<DK, COLS>(p, b, h, token0, left < kChunk ? static_cast<int>(left) : kChunk, block, rows, temp, scratch);
  float* out = reinterpret_cast<float*>(block + kBlockRows);
  for (int i = threadIdx.x; i < kRowFloats; i += kWave) out[i] = rows[i];
}

// Half fragments: the four values of one 16-row result, as the first or second half of a fragment of 32 rows in LDS.
__device__ __forceinline__ void put_half(uint8_t* frags, int tile, int lane, const f32x4& v, int low_at) {
  const u32x2 hi = round4(v);
  uint8_t* at = frags + (tile / 2) * kFrag + lane * 16 + (tile % 2) * 8;
  *reinterpret_cast<u32x2*>(at) = hi;
  *reinterpret_cast<u32x2*>(at + low_at) = rest4(v, hi);
}
__device__ __forceinline__ bf16x8 get_frag(const uint8_t* frags, int f, int lane) {
  return *reinterpret_cast<const bf16x8*>(frags + f * kFrag + lane * 16);
}

template <int DK>
struct TeamLds {  // fragments hi, then lo, of each
  static constexpr int KB = DK / 32;
  static constexpr int kState = 0;                      // KB fragments
  static constexpr int kX = kState + 2 * KB * kFrag;    // 2
  static constexpr int kN = kX + 4 * kFrag;
  static constexpr int kW = kN + 4 * kFrag;
  static constexpr int kTileK = kW + 4 * kFrag;
  static constexpr int kForward = kTileK + Tile<DK>::BYTES;
  static constexpr int kTileQ = kForward;               // backward only
  static constexpr int kBackward = kTileQ + Tile<DK>::BYTES;
};

// What wavefront w needs of a chunk. Several of them take turns, so that nothing is copied.
constexpr int kTeamRow = 20;  // elements of a token's 16 columns in LDS

template <int KB>
struct TeamChunk {
  bf16x8 kf[KB], qf[KB];
  bf16x8 mh[2], ml[2], pf[2];
  f32x4 grown, keep;
  float grown_row, total;
  u32x2 x;  // four columns of a token of V (backward: of dO), on their way into LDS
};

template <int DK, bool COLS>
struct Team {
  static constexpr int KB = DK / 32, KA = DK / 16, OWN = KA >= 4 ? KA / 4 : 1;  // OWN: state tiles of a wavefront
  typedef TeamChunk<KB> Chunk;
  const DeltaParams& p;
  int wave, lane, l16, grp, col0, h, b, len, chunks;
  int64_t unit;
  bool col_ok, owner;
  // The chunk that is requested next: uniform pointers that move by whole chunks, and byte offsets of this lane that stay (token strides are
  // below 2^24 elements), so that a request costs no arithmetic.
  const uint8_t *k_at, *q_at, *x_at, *block_at;
  int64_t k_step, q_step, x_step;
  int32_t k_ld, q_ld, x_ld, k_less, q_less, x_less;  // bytes from row to row, and what a row is short of that
  int at, n_at;
  Buffer block;
  uint32_t k_off[KB], q_off[KB], x_off, frag_off[2], row_off;

  __device__ __forceinline__ Team(const DeltaParams& params) : p(params) {
    const int tid = threadIdx.x;
    wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    lane = tid % kWave, l16 = lane % 16, grp = lane / 16;
    const int col_groups = (p.dv + 15) / 16;
    const uint32_t block = xcd_remap(blockIdx.x, gridDim.x);  // the columns of a head, which read the same rows, on one die's L2
    unit = block / col_groups;
    col0 = static_cast<int>(block % col_groups) * 16;
    col_ok = col0 + l16 < p.dv;
    h = static_cast<int>(unit % p.H);
    b = static_cast<int>(unit / p.H);
    len = p.T;
    if (p.lengths != nullptr) {
      len = p.lengths[b];
      len = len < 0 ? 0 : (len > p.T ? p.T : len);
    }
    chunks = (len + kChunk - 1) / kChunk;
    const int64_t hk = h / p.group;
    const int64_t* xs = COLS ? p.dos : p.vs;
    at = COLS ? chunks - 1 : 0;
    const int64_t first = static_cast<int64_t>(at) * kChunk;
    k_at = reinterpret_cast<const uint8_t*>(p.k + b * p.ks[0] + hk * p.ks[1] + first * p.ks[2]);
    q_at = reinterpret_cast<const uint8_t*>(p.q + b * p.qs[0] + hk * p.qs[1] + first * p.qs[2]);
    x_at = reinterpret_cast<const uint8_t*>((COLS ? p.grad_o : p.v) + b * xs[0] + h * xs[1] + col0 + first * xs[2]);
    block_at = p.blocks + (unit * p.chunks + at) * kBlockBytes;
    constexpr int64_t kMove = (COLS ? -kChunk : kChunk) * 2;
    k_step = kMove * p.ks[2], q_step = kMove * p.qs[2], x_step = kMove * xs[2];
    k_ld = static_cast<int32_t>(p.ks[2]) * 2, q_ld = static_cast<int32_t>(p.qs[2]) * 2, x_ld = static_cast<int32_t>(xs[2]) * 2;
    k_less = k_ld - p.dk * 2, q_less = q_ld - p.dk * 2, x_less = x_ld - (p.dv - col0) * 2;
    owner = wave * OWN < KA;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const uint32_t feature = static_cast<uint32_t>(32 * kb + 8 * grp);
      k_off[kb] = feature < static_cast<uint32_t>(p.dk) ? (16 * wave + l16) * k_ld + feature * 2 : kNowhere;
      q_off[kb] = feature < static_cast<uint32_t>(p.dk) ? (16 * wave + l16) * q_ld + feature * 2 : kNowhere;
    }
    x_off = col0 + lane % 4 * 4 < p.dv ? (16 * wave + lane / 4) * x_ld + lane % 4 * 8 : kNowhere;
#pragma unroll
    for (int tk = 0; tk < 2; ++tk)
      frag_off[tk] = (COLS ? tk >= wave / 2 : tk <= wave / 2) ? (COLS ? frag_cols(wave, tk) : frag_rows(wave, tk)) * kFrag + lane * 16 : kNowhere;
    row_off = static_cast<uint32_t>(16 * wave + 4 * grp) * 4;
  }
  __device__ __forceinline__ int tokens_of(int chunk) const {
    const int left = len - chunk * kChunk;
    return left < kChunk ? left : kChunk;
  }

  // The first n rows at a base; none where n is not positive.
  static __device__ __forceinline__ Buffer rows_at(const uint8_t* base, int n, int32_t ld, int32_t less) {
    const int32_t bytes = n * ld - less;
    return buffer_of(base, bytes > 0 ? bytes : 0);
  }

  // The requests for a chunk (behind the last one: zeros), in three parts that the stages of the chunk before it issue beside their work:
  // in one run they would wait for each other in front of it. No branch around them, so that what was requested before can be awaited
  // without awaiting these.
  __device__ __forceinline__ void fetch_keys(Chunk& c) {
    n_at = !COLS || at >= 0 ? tokens_of(at) : 0;
    block = buffer_of(block_at, n_at > 0 ? kBlockBytes : 0);
    const Buffer k = rows_at(k_at, n_at, k_ld, k_less), x = rows_at(x_at, n_at, x_ld, x_less);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) c.kf[kb] = read8(k, k_off[kb]);
    c.x = read4(x, x_off);
    c.grown = read_floats(block, row_off, kBlockRows + kRowGrown * 4);
    c.keep = read_floats(block, row_off, kBlockRows + kRowKeep * 4);
    if (!COLS) c.grown_row = read_float(block, l16 * 4 + wave * 64, kBlockRows + kRowGrown * 4);
    c.total = read_float(block, 0, kBlockRows + kRowTotal * 4);
  }
  __device__ __forceinline__ void fetch_queries(Chunk& c) const {
    const Buffer q = rows_at(q_at, n_at, q_ld, q_less);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) c.qf[kb] = read8(q, q_off[kb]);
  }
  // the last part, then on to the next chunk
  __device__ __forceinline__ void fetch_block(Chunk& c) {
#pragma unroll
    for (int tk = 0; tk < 2; ++tk) {
      c.mh[tk] = read8(block, frag_off[tk], kBlockM);
      c.ml[tk] = read8(block, frag_off[tk], kBlockLow);
      c.pf[tk] = read8(block, frag_off[tk], kBlockP);
    }
    at += COLS ? -1 : 1;
    k_at += k_step, q_at += q_step, x_at += x_step;
    block_at += COLS ? -kBlockBytes : kBlockBytes;
  }

  // The 16 columns of V (dO) in LDS, token by token: written behind a chunk's last use of them, read by columns.
  __device__ __forceinline__ void place(const Chunk& c, bf16_t* tile_x) const {
    *reinterpret_cast<u32x2*>(tile_x + (16 * wave + lane / 4) * kTeamRow + lane % 4 * 4) = c.x;
  }
  __device__ __forceinline__ bf16x4 values(const bf16_t* tile_x, int token0) const {  // tokens token0 + 4 grp .. of column l16
    return Tile<DK>::read_tr(tile_x + (token0 + 4 * grp + l16 / 4) * kTeamRow + l16 % 4 * 4);
  }

  // The own rows of the state, bf16, at dst [dv][dk]
  __device__ __forceinline__ void store_state(bf16_t* dst, const f32x4 (&s)[OWN]) const {
    if (!owner || !col_ok) return;
    const uint32_t off = static_cast<uint32_t>((col0 + l16) * p.dk + 8 * grp) * 2;
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int a = wave * OWN + i;
      if (p.dk == DK || state_row(a, 4 * grp) < p.dk) put_offset(dst + 32 * (a / 2) + 4 * (a % 2), off, round4(s[i]));
    }
  }
};

template <int DK, bool TRAIN>
__global__ __launch_bounds__(4 * kWave) void delta_team_kernel(const DeltaParams p) {
  typedef Team<DK, false> M;
  typedef TeamLds<DK> L;
  typedef Tile<DK> TK;
  constexpr int KB = M::KB, OWN = M::OWN;
  __shared__ __attribute__((aligned(64))) uint8_t smem[L::kForward];
  __shared__ __attribute__((aligned(16))) bf16_t turned[TRAIN ? 4 : 1][320], tile_x[kChunk * kTeamRow];
  bf16_t* tile_k = reinterpret_cast<bf16_t*>(smem + L::kTileK);
  uint8_t *s_frags = smem + L::kState, *x_frags = smem + L::kX, *n_frags = smem + L::kN, *w_frags = smem + L::kW;
  M m(p);
  const int wave = m.wave, lane = m.lane, l16 = m.l16, grp = m.grp, col0 = m.col0;
  bf16_t* o0 = p.o + m.b * p.os[0] + m.h * p.os[1] + col0;
  const uint32_t o_off = static_cast<uint32_t>((16 * wave + l16) * p.os[2] + 4 * grp) * 2;
  const uint32_t n_off = static_cast<uint32_t>((16 * wave + l16) * p.dv + col0 + 4 * grp) * 2;
  const bool quad_ok = col0 + 4 * grp < p.dv;
  bf16_t* turn = turned[TRAIN ? wave : 0];

  f32x4 s[OWN];
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    s[i] = zero4();
    const int a = wave * OWN + i;
    if (p.state_in != nullptr && m.col_ok && m.owner) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = state_row(a, 4 * grp + r);
        if (row < p.dk) s[i][r] = p.state_in[(m.unit * p.dk + row) * p.dv + col0 + l16];
      }
    }
    if (m.owner) put_half(s_frags, a, lane, s[i], KB * kFrag);
  }

  bf16_t* o_at = o0;
  bf16_t* state_at = TRAIN ? p.chunk_states + m.unit * p.chunks * static_cast<int64_t>(p.dk) * p.dv : nullptr;
  bf16_t* miss_at = TRAIN ? p.misses + m.unit * p.T * p.dv : nullptr;
  auto step = [&](int chunk, typename M::Chunk& cur, typename M::Chunk& next) __attribute__((always_inline)) {
    const int n_tok = m.tokens_of(chunk);
    m.fetch_keys(next);
    if (TRAIN) {
      m.store_state(state_at, s);
      state_at += p.dk * p.dv;
    }
    // X of the own tokens; K's rows on their way into LDS
    bf16x8 sh[KB], sl[KB];
    f32x4 y = zero4(), y2 = zero4();
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      sh[kb] = get_frag(s_frags, kb, lane);
      sl[kb] = get_frag(s_frags + KB * kFrag, kb, lane);
      y = mfma16(cur.kf[kb], sh[kb], y);
      y2 = mfma16(cur.kf[kb], sl[kb], y2);
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      *reinterpret_cast<bf16x8*>(tile_k + (16 * wave + l16) * TK::STRIDE + kb * 32 + grp * 8) = cur.kf[kb];
    f32x4 x;
    const bf16x4 v = m.values(tile_x, 16 * wave);
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = fmaf(-cur.grown[r], y[r] + y2[r], static_cast<float>(v[r]));
    put_half(x_frags, wave, lane, x, 2 * kFrag);
    __syncthreads();
    m.fetch_queries(next);

    // N of the own tokens
    f32x4 x2 = zero4(), x3 = zero4();
#pragma unroll
    for (int tk = 0; tk < 2; ++tk)
      if (tk <= wave / 2) {
        const bf16x8 xh = get_frag(x_frags, tk, lane), xl = get_frag(x_frags + 2 * kFrag, tk, lane);
        x = mfma16(cur.mh[tk], xh, x);
        x2 = mfma16(cur.mh[tk], xl, x2);
        x3 = mfma16(cur.ml[tk], xh, x3);
      }
    f32x4 out = zero4(), out2 = zero4();  // the state's part of the output: lane = token, four columns each
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      out = mfma16(sh[kb], cur.qf[kb], out);
      out2 = mfma16(sl[kb], cur.qf[kb], out2);
    }
    f32x4 w;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[r] += x2[r] + x3[r];
      w[r] = x[r] * cur.keep[r];
    }
    put_half(w_frags, wave, lane, w, 2 * kFrag);
    put_half(n_frags, wave, lane, x, 2 * kFrag);
    if (TRAIN) {
      const u32x2 rounded = turn16(turn, x, l16, grp);
      if (16 * wave + l16 < n_tok && quad_ok) put_offset(miss_at, n_off, rounded);
      miss_at += kChunk * p.dv;
    }
    const float grown = cur.grown_row * p.scale;
#pragma unroll
    for (int r = 0; r < 4; ++r) out[r] = (out[r] + out2[r]) * grown;
    __syncthreads();
    m.fetch_block(next);

    // the own rows of the state
    if (m.owner) {
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const int a = wave * OWN + i;
        f32x4 s2 = zero4();
#pragma unroll
        for (int r = 0; r < 4; ++r) s[i][r] *= cur.total;
#pragma unroll
        for (int tk = 0; tk < 2; ++tk) {
          const bf16x8 kt = TK::keys_frag(tile_k, tk, a, l16, grp);
          s[i] = mfma16(kt, get_frag(w_frags, tk, lane), s[i]);
          s2 = mfma16(kt, get_frag(w_frags + 2 * kFrag, tk, lane), s2);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) s[i][r] += s2[r];
        put_half(s_frags, a, lane, s[i], KB * kFrag);
      }
    }
    // the output of the own tokens
    out2 = zero4();
#pragma unroll
    for (int tk = 0; tk < 2; ++tk)
      if (tk <= wave / 2) {
        out = mfma16(get_frag(n_frags, tk, lane), cur.pf[tk], out);
        out2 = mfma16(get_frag(n_frags + 2 * kFrag, tk, lane), cur.pf[tk], out2);
      }
    if (16 * wave + l16 < n_tok && quad_ok) {
#pragma unroll
      for (int r = 0; r < 4; ++r) out[r] += out2[r];
      put_offset(o_at, o_off, round4(out));
    }
    o_at += kChunk * p.os[2];
    m.place(next, tile_x);
    __syncthreads();
  };
  typename M::Chunk even, odd;
  if (m.chunks > 0) {
    m.fetch_keys(even);
    m.fetch_queries(even);
    m.fetch_block(even);
    m.place(even, tile_x);
  }
  __syncthreads();
  // Pairs, then the odd one: a way past the second half back to the first would have to await the requests of the wrong one.
  int chunk = 0;
  for (; chunk + 1 < m.chunks; chunk += 2) {
    step(chunk, even, odd);
    step(chunk + 1, odd, even);
  }
  if (chunk < m.chunks) step(chunk, even, odd);

  if (p.state_out != nullptr && m.col_ok && m.owner) {
#pragma unroll
    for (int i = 0; i < OWN; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = state_row(wave * OWN + i, 4 * grp + r);
        if (row < p.dk) p.state_out[(m.unit * p.dk + row) * p.dv + col0 + l16] = s[i][r];
      }
  }
  const bf16x4 none = {};
  for (int64_t i = threadIdx.x; i < static_cast<int64_t>(p.T - m.len) * 4; i += 4 * kWave) {
    const int at = static_cast<int>(i % 4) * 4;
    if (col0 + at < p.dv) *reinterpret_cast<bf16x4*>(o0 + (m.len + i / 4) * p.os[2] + at) = none;
  }
}

// The gradient of the state, chunks last to first (the formulas: delta_bwd.hip). Stages: beta dU (own tokens) | dX (own tokens) | dS (own
// rows). dO is read as fragments by every wavefront.
template <int DK>
__global__ __launch_bounds__(4 * kWave) void delta_team_back_kernel(const DeltaParams p) {
  typedef Team<DK, true> M;
  typedef TeamLds<DK> L;
  typedef Tile<DK> TK;
  constexpr int KB = M::KB, OWN = M::OWN;
  __shared__ __attribute__((aligned(64))) uint8_t smem[L::kBackward];
  __shared__ __attribute__((aligned(16))) bf16_t turned[4][320], tile_x[kChunk * kTeamRow];
  bf16_t* tile_k = reinterpret_cast<bf16_t*>(smem + L::kTileK);
  bf16_t* tile_q = reinterpret_cast<bf16_t*>(smem + L::kTileQ);
  uint8_t *s_frags = smem + L::kState, *z_frags = smem + L::kX, *x_frags = smem + L::kN, *o_frags = smem + L::kW;
  M m(p);
  const int wave = m.wave, lane = m.lane, l16 = m.l16, grp = m.grp, col0 = m.col0;
  bf16_t* v0 = p.grad_v + m.b * p.dvs[0] + m.h * p.dvs[1] + col0;
  const uint32_t v_off = static_cast<uint32_t>((16 * wave + l16) * p.dvs[2] + 4 * grp) * 2;
  const bool quad_ok = col0 + 4 * grp < p.dv;

  f32x4 s[OWN];
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    s[i] = zero4();
    if (m.owner) put_half(s_frags, wave * OWN + i, lane, s[i], KB * kFrag);
  }

  bf16_t* v_at = v0 + (m.chunks - 1) * kChunk * p.dvs[2];
  bf16_t* state_at = p.grad_states + (m.unit * p.chunks + m.chunks - 1) * static_cast<int64_t>(p.dk) * p.dv;
  auto step = [&](int chunk, typename M::Chunk& cur, typename M::Chunk& next) __attribute__((always_inline)) {
    const int n_tok = m.tokens_of(chunk);
    m.fetch_keys(next);
    m.store_state(state_at, s);
    state_at -= p.dk * p.dv;
    // beta dU of the own tokens
    f32x4 z = zero4(), z2 = zero4(), z3 = zero4();
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      z = mfma16(cur.kf[kb], get_frag(s_frags, kb, lane), z);
      z2 = mfma16(cur.kf[kb], get_frag(s_frags + KB * kFrag, kb, lane), z2);
    }
#pragma unroll
    for (int tk = 0; tk < 2; ++tk)
      if (tk >= wave / 2) {
        z3 = mfma16(cur.pf[tk], TK::join(m.values(tile_x, 32 * tk), m.values(tile_x, 32 * tk + 16)), z3);
      }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int at = (16 * wave + l16) * TK::STRIDE + kb * 32 + grp * 8;
      *reinterpret_cast<bf16x8*>(tile_k + at) = cur.kf[kb];
      *reinterpret_cast<bf16x8*>(tile_q + at) = cur.qf[kb];
    }
    f32x4 w;
    const bf16x4 own = m.values(tile_x, 16 * wave);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      z[r] = fmaf(cur.keep[r], z[r] + z2[r], z3[r]);
      w[r] = p.scale * cur.grown[r] * static_cast<float>(own[r]);
    }
    put_half(z_frags, wave, lane, z, 2 * kFrag);
    put_half(o_frags, wave, lane, w, 2 * kFrag);
    __syncthreads();
    m.fetch_queries(next);

    // dX of the own tokens
    z2 = z3 = zero4();
#pragma unroll
    for (int tk = 0; tk < 2; ++tk)
      if (tk >= wave / 2) {
        const bf16x8 zh = get_frag(z_frags, tk, lane), zl = get_frag(z_frags + 2 * kFrag, tk, lane);
        z = mfma16(cur.mh[tk], zh, z);
        z2 = mfma16(cur.mh[tk], zl, z2);
        z3 = mfma16(cur.ml[tk], zh, z3);
      }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      z[r] += z2[r] + z3[r];
      w[r] = -cur.grown[r] * z[r];
    }
    put_half(x_frags, wave, lane, w, 2 * kFrag);
    const u32x2 rounded = turn16(turned[wave], z, l16, grp);
    if (16 * wave + l16 < n_tok && quad_ok) put_offset(v_at, v_off, rounded);
    v_at -= kChunk * p.dvs[2];
    __syncthreads();
    m.fetch_block(next);

    // dS of the own rows
    if (m.owner) {
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const int a = wave * OWN + i;
        f32x4 s2 = zero4(), s3 = zero4(), s4 = zero4();
#pragma unroll
        for (int r = 0; r < 4; ++r) s[i][r] *= cur.total;
#pragma unroll
        for (int tk = 0; tk < 2; ++tk) {
          const bf16x8 kt = TK::keys_frag(tile_k, tk, a, l16, grp), qt = TK::keys_frag(tile_q, tk, a, l16, grp);
          s[i] = mfma16(kt, get_frag(x_frags, tk, lane), s[i]);
          s2 = mfma16(kt, get_frag(x_frags + 2 * kFrag, tk, lane), s2);
          s3 = mfma16(qt, get_frag(o_frags, tk, lane), s3);
          s4 = mfma16(qt, get_frag(o_frags + 2 * kFrag, tk, lane), s4);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) s[i][r] += (s2[r] + s4[r]) + s3[r];
        put_half(s_frags, a, lane, s[i], KB * kFrag);
      }
    }
    m.place(next, tile_x);
    __syncthreads();
  };
  typename M::Chunk even, odd;
  if (m.chunks > 0) {
    m.fetch_keys(even);
    m.fetch_queries(even);
    m.fetch_block(even);
    m.place(even, tile_x);
  }
  __syncthreads();
  int chunk = m.chunks - 1;  // pairs, then the odd one, as above
  for (; chunk > 0; chunk -= 2) {
    step(chunk, even, odd);
    step(chunk - 1, odd, even);
  }
  if (chunk == 0) step(0, even, odd);
  const bf16_t none = static_cast<bf16_t>(0.f);
  for (int64_t i = threadIdx.x; i < static_cast<int64_t>(p.T - m.len) * 16; i += 4 * kWave) {
    const int at = static_cast<int>(i % 16);
    if (col0 + at < p.dv) v0[(m.len + i / 16) * p.dvs[2] + at] = none;
  }
}

template <int DK, bool COLS>
int launch_team(const char* name, const DeltaParams& p, hipStream_t s) {
  const int64_t heads = static_cast<int64_t>(p.B) * p.H, teams = heads * ((p.dv + 15) / 16);
  if (heads * p.chunks > 0x7fffffffLL || teams > 0x7fffffffLL) return set_error(TAAC_ERR_UNSUPPORTED, "%s: too many workgroups", name);
  if (p.chunks > 0) hipLaunchKernelGGL((delta_blocks_kernel<DK, COLS>), dim3(static_cast<uint32_t>(heads * p.chunks)), dim3(kWave), 0, s, p);
  const dim3 grid(static_cast<uint32_t>(teams)), threads(4 * kWave);
  if constexpr (COLS) hipLaunchKernelGGL((delta_team_back_kernel<DK>), grid, threads, 0, s, p);
  else if (p.chunk_states != nullptr) hipLaunchKernelGGL((delta_team_kernel<DK, true>), grid, threads, 0, s, p);
  else hipLaunchKernelGGL((delta_team_kernel<DK, false>), grid, threads, 0, s, p);
  return check_launch(name);
}

}  // namespace

int delta_team_fwd(const char* name, const DeltaParams& p, hipStream_t s) {
  if (p.dk <= 32) return launch_team<32, false>(name, p, s);
  if (p.dk <= 64) return launch_team<64, false>(name, p, s);
  return launch_team<128, false>(name, p, s);
}
int delta_team_back(const char* name, const DeltaParams& p, hipStream_t s) {
  if (p.dk <= 32) return launch_team<32, true>(name, p, s);
  if (p.dk <= 64) return launch_team<64, true>(name, p, s);
  return launch_team<128, true>(name, p, s);
}

int64_t delta_team_bytes(int64_t heads, int32_t T, int32_t dk, int32_t dv) {
  // Two, three or six teams to a CU: beyond that the chain of chunks no longer counts, and a wavefront that walks its head alone, without the
  // blocks in memory, is faster. 2048 tokens, forward, this form against the other, by heads times groups of 16 columns: 32 wide 119 : 163 us
  // at 512, 192 : 171 at 768; 64 wide 152 : 194 at 768, 218 : 198 at 1024; 128 wide 340 : 418 at 1536, 445 : 428 at 2048; forward and backward
  // together the same order (402 : 473, 617 : 561; 532 : 572, 729 : 619; 1348 : 1403, 1793 : 1593).
  const int64_t teams = heads * ((dv + 15) / 16);
  if (teams > (dk <= 32 ? 512 : dk <= 64 ? 768 : 1536)) return 0;
  return heads * ((T + kChunk - 1) / kChunk) * kBlockBytes;
}

}  // namespace taac

extern "C" int64_t taac_delta_rule_workspace_bytes(int32_t B, int32_t H, int32_t T, int32_t dk, int32_t dv) {
  if (B < 0 || H <= 0 || T < 0 || dk <= 0 || dv <= 0) return -1;
  return taac::delta_team_bytes(static_cast<int64_t>(B) * H, T, dk, dv);
}
