// Gated delta rule, chunked form, for few or wide heads and long histories (the mathematics, operand order and precision: delta.h).
//
// With few (sample, head) pairs the time is the chain of chunks, not the work: what does not depend on the state is made for all
// chunks at once (one wavefront each) and left in memory, and a chunk's step of the state is spread over four wavefronts to make it
// short. A workgroup has 16 (or 32) value columns; wavefront w owns tokens 16 w .. 16 w + 15 of every chunk and a quarter of the key
// rows of the state. A step is three stages with a barrier behind each,
//   X (own tokens) from the state | N (own tokens) from X | the state (own rows) from N; the output beside them,
// whose results meet in LDS as operand fragments. Everything a chunk reads from memory is requested one chunk ahead, a third beside
// each stage.
//
// 2 samples x 16 heads x 8192 tokens, 128 wide: 41 us for the blocks (170 MB, 4.1 TB/s) and 239 us for 128 steps of 1.9 us (masked reads in one
// run at a step's start took 1.6 times as long). A step is a chain of eighteen dependent matrix instructions and three exchanges through LDS, among
// 370 instructions that every wavefront issues: bound by that chain, the matrix units are busy for a fifth of it, and a wavefront waits for 39 %.
#include "delta.h"

namespace taac {
namespace {

// Place of a fragment in a block. By rows (forward): row tile ti, token block tk <= ti / 2. By columns (backward): column tile tj, token
// block tk >= tj / 2.
__host__ __device__ constexpr int frag_rows(int ti, int tk) { return ti < 2 ? ti : 2 + (ti - 2) * 2 + tk; }
__host__ __device__ constexpr int frag_cols(int tj, int tk) { return tj < 2 ? tj * 2 + tk : 2 + tj; }

// One wavefront makes the block of one chunk (n valid tokens; rows beyond count as k = q = 0, g = 0, beta = 0): -M and P in parts, and the
// factors of its tokens. COLS: transposed fragments, for the backward. rows, temp, scratch: LDS.
//
// The 64 x 64 inverse: the four diagonal blocks of 16 by substitution, a column per lane, all four at once; the blocks below them by
// products, M_21 = T_22 A_21 T_11 with T = I - M, first pairs of 16, then of 32.
template <int DK, bool COLS>
__device__ __forceinline__ void chunk_block(const DeltaParams& p, int b, int h, int64_t token0, int n, uint8_t* block, float* rows,
                                            float* temp, float* scratch) {
  constexpr int KB = DK / 32;
  const int lane = threadIdx.x % kWave, l16 = lane % 16, grp = lane / 16;

  // everything is requested before any of it is waited for
  const int64_t hk = h / p.group;
  const Buffer k_rows = rows_buffer(p.k + b * p.ks[0] + hk * p.ks[1] + token0 * p.ks[2], p.ks[2], n, p.dk);
  const Buffer q_rows = rows_buffer(p.q + b * p.qs[0] + hk * p.qs[1] + token0 * p.qs[2], p.qs[2], n, p.dk);
  GateBits gates;
  gates.request(p, b, h, token0, n, lane);
  bf16x8 kf[4][KB], qf[4][KB];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      kf[t][kb] = read8(k_rows, 32 * kb + 8 * grp < p.dk ? (16 * t + l16) * static_cast<uint32_t>(p.ks[2]) * 2 + 64 * kb + 16 * grp : kNowhere);
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      qf[t][kb] = read8(q_rows, 32 * kb + 8 * grp < p.dk ? (16 * t + l16) * static_cast<uint32_t>(p.qs[2]) * 2 + 64 * kb + 16 * grp : kNowhere);
  chunk_rows(p, gates, n, rows, temp);
  wave_sync();

  f32x4 a_rows[10];  // A by rows, tile (ti, tj) at ti (ti + 1) / 2 + tj
  u32x2 pf[6][2], pl[6][2];
#pragma unroll
  for (int i = 0; i < 6; ++i) pf[i][0] = pf[i][1] = pl[i][0] = pl[i][1] = u32x2{0u, 0u};
#pragma unroll
  for (int ti = 0; ti < 4; ++ti) {
    const int row = 16 * ti + l16;
    const float hi_i = temp[kTempHi + row], lo_i = temp[kTempLow + row], in_i = temp[kTempIn + row];
#pragma unroll
    for (int tj = 0; tj <= ti; ++tj) {
      f32x4 kk = zero4(), qk = zero4();
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        kk = mfma16(kf[tj][kb], kf[ti][kb], kk);
        qk = COLS ? mfma16(qf[ti][kb], kf[tj][kb], qk) : mfma16(kf[tj][kb], qf[ti][kb], qk);
      }
      f32x4 a, s;
      if (ti > tj) {
        const float between = tiles_between(rows, ti, tj);
        const float a_i = in_i * between, s_i = a_i * p.scale;
        const f32x4 out_j = *reinterpret_cast<const f32x4*>(temp + kTempOutBeta + 16 * tj + 4 * grp);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          a[r] = a_i * out_j[r] * kk[r];
          if (!COLS) s[r] = s_i * out_j[r] * qk[r];
        }
        if (COLS) {
          const float s_j = temp[kTempOutBeta + 16 * tj + l16] * between * p.scale;
          const f32x4 in_r = *reinterpret_cast<const f32x4*>(temp + kTempIn + 16 * ti + 4 * grp);
#pragma unroll
          for (int r = 0; r < 4; ++r) s[r] = s_j * in_r[r] * qk[r];
        }
      } else {
        const f32x4 hi_j = *reinterpret_cast<const f32x4*>(temp + kTempHi + 16 * tj + 4 * grp);
        const f32x4 lo_j = *reinterpret_cast<const f32x4*>(temp + kTempLow + 16 * tj + 4 * grp);
        const f32x4 beta_j = *reinterpret_cast<const f32x4*>(temp + kTempBeta + 16 * tj + 4 * grp);
        const float beta_i = temp[kTempBeta + row];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int m = 4 * grp + r;
          const float diff = (hi_i - hi_j[r]) + (lo_i - lo_j[r]);  // of tokens l16 and m of the tile
          const float gam = __builtin_amdgcn_exp2f(diff) * beta_j[r];
          a[r] = l16 > m ? gam * kk[r] : 0.f;
          if (COLS) s[r] = m >= l16 ? p.scale * __builtin_amdgcn_exp2f(-diff) * beta_i * qk[r] : 0.f;
          else s[r] = l16 >= m ? p.scale * gam * qk[r] : 0.f;
        }
      }
      a_rows[ti * (ti + 1) / 2 + tj] = a;
      const int f = COLS ? frag_cols(tj, ti / 2) : frag_rows(ti, tj / 2);
      const int half = COLS ? ti % 2 : tj % 2;
      pf[f][half] = round4(s);
      pl[f][half] = rest4(s, pf[f][half]);
    }
  }

  // diagonal blocks
#pragma unroll
  for (int t = 0; t < 4; ++t) *reinterpret_cast<f32x4*>(scratch + t * kScratchBlock + l16 * kScratchRow + 4 * grp) = a_rows[t * (t + 1) / 2 + t];
  wave_sync();
  solve_diagonal(scratch, lane);
  f32x4 m_rows[4], m_cols[4], t_rows[4], t_cols[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    m_rows[t] = *reinterpret_cast<const f32x4*>(scratch + t * kScratchBlock + l16 * kScratchRow + 4 * grp);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      m_cols[t][r] = scratch[t * kScratchBlock + (4 * grp + r) * kScratchRow + l16];
      const float one = l16 == 4 * grp + r ? 1.f : 0.f;
      t_rows[t][r] = one - m_rows[t][r];
      t_cols[t][r] = one - m_cols[t][r];
    }
  }
  wave_sync();

  const f32x4 z10 = mul_cols(a_rows[1], t_cols[0], zero4());
  const f32x4 z32 = mul_cols(a_rows[8], t_cols[2], zero4());
  const f32x4 m10c = mul_cols(t_rows[1], z10, zero4());
  const f32x4 m32r = mul_rows(t_rows[3], z32, zero4());
  f32x4 m10n, m32n;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    m10n[r] = -m10c[r];
    m32n[r] = -m32r[r];
  }
  const f32x4 z20 = mul_cols(a_rows[4], m10n, mul_cols(a_rows[3], t_cols[0], zero4()));
  const f32x4 z21 = mul_cols(a_rows[4], t_cols[1], zero4());
  const f32x4 z30 = mul_cols(a_rows[7], m10n, mul_cols(a_rows[6], t_cols[0], zero4()));
  const f32x4 z31 = mul_cols(a_rows[7], t_cols[1], zero4());

  auto put = [&](int f, const f32x4& first, const f32x4& second) {
    f32x4 a, c;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      a[r] = -first[r];
      c[r] = -second[r];
    }
    bf16x8 hi8, mid8, lo8;
    if (COLS) split(a, c, hi8, mid8);
    else split3(a, c, hi8, mid8, lo8);
    *reinterpret_cast<bf16x8*>(block + kBlockM + f * kFrag + lane * 16) = hi8;
    *reinterpret_cast<bf16x8*>(block + kBlockMid + f * kFrag + lane * 16) = mid8;
    if (!COLS) *reinterpret_cast<bf16x8*>(block + kBlockLow + f * kFrag + lane * 16) = lo8;
    *reinterpret_cast<u32x4*>(block + kBlockP + f * kFrag + lane * 16) = u32x4{pf[f][0][0], pf[f][0][1], pf[f][1][0], pf[f][1][1]};
    if (COLS || low_scores(DK))
      *reinterpret_cast<u32x4*>(block + (COLS ? kBlockLow : kBlockPLow) + f * kFrag + lane * 16) = u32x4{pl[f][0][0], pl[f][0][1], pl[f][1][0], pl[f][1][1]};
  };
  if (!COLS) {
    const f32x4 m10r = mul_rows(t_rows[1], z10, zero4());
    put(frag_rows(0, 0), m_rows[0], zero4());
    put(frag_rows(1, 0), m10r, m_rows[1]);
    put(frag_rows(2, 0), mul_rows(t_rows[2], z20, zero4()), mul_rows(t_rows[2], z21, zero4()));
    put(frag_rows(2, 1), m_rows[2], zero4());
    put(frag_rows(3, 0), mul_rows(m32n, z20, mul_rows(t_rows[3], z30, zero4())), mul_rows(m32n, z21, mul_rows(t_rows[3], z31, zero4())));
    put(frag_rows(3, 1), m32r, m_rows[3]);
  } else {
    const f32x4 m32c = mul_cols(t_rows[3], z32, zero4());
    put(frag_cols(0, 0), m_cols[0], m10c);
    put(frag_cols(0, 1), mul_cols(t_rows[2], z20, zero4()), mul_cols(m32n, z20, mul_cols(t_rows[3], z30, zero4())));
    put(frag_cols(1, 0), zero4(), m_cols[1]);
    put(frag_cols(1, 1), mul_cols(t_rows[2], z21, zero4()), mul_cols(m32n, z21, mul_cols(t_rows[3], z31, zero4())));
    put(frag_cols(2, 1), m_cols[2], m32c);
    put(frag_cols(3, 1), zero4(), m_cols[3]);
  }
}

template <int DK, bool COLS>
__global__ __launch_bounds__(kWave) void delta_blocks_kernel(const DeltaParams p) {
  __shared__ __attribute__((aligned(16))) float rows[kRowFloats];
  __shared__ __attribute__((aligned(16))) float temp[kTempFloats];
  __shared__ __attribute__((aligned(16))) float scratch[kScratchFloats];
  const uint32_t chunks = p.chunks, heads = p.H, unit = blockIdx.x / chunks;
  const int chunk = static_cast<int>(blockIdx.x % chunks), h = static_cast<int>(unit % heads), b = static_cast<int>(unit / heads);
  int len = p.T;
  if (p.lengths != nullptr) len = p.lengths[b] < p.T ? p.lengths[b] : p.T;
  const int64_t token0 = static_cast<int64_t>(chunk) * kChunk;
  const int64_t left = len - token0;
  if (left <= 0) return;
  uint8_t* block = p.blocks + static_cast<int64_t>(blockIdx.x) * block_bytes(DK);
  chunk_block<DK, COLS>(p, b, h, token0, left < kChunk ? static_cast<int>(left) : kChunk, block, rows, temp, scratch);
  float* out = reinterpret_cast<float*>(block + kBlockRows);
  for (int i = threadIdx.x; i < kRowFloats; i += kWave) out[i] = rows[i];
}

// Half fragments: the four values of one 16-row result, as the first or second half of a fragment of 32 rows in LDS. In two parts, or in
// three.
__device__ __forceinline__ void put_half(uint8_t* frags, int tile, int lane, const f32x4& v, int low_at) {
  const u32x2 hi = round4(v);
  uint8_t* at = frags + (tile / 2) * kFrag + lane * 16 + (tile % 2) * 8;
  *reinterpret_cast<u32x2*>(at) = hi;
  *reinterpret_cast<u32x2*>(at + low_at) = rest4(v, hi);
}
__device__ __forceinline__ void put_half3(uint8_t* frags, int tile, int lane, const f32x4& v, int low_at) {
  const u32x2 hi = round4(v);
  const f32x4 left = left4(v, hi);
  const u32x2 mid = round4(left);
  uint8_t* at = frags + (tile / 2) * kFrag + lane * 16 + (tile % 2) * 8;
  *reinterpret_cast<u32x2*>(at) = hi;
  *reinterpret_cast<u32x2*>(at + low_at) = mid;
  *reinterpret_cast<u32x2*>(at + 2 * low_at) = rest4(left, mid);
}
__device__ __forceinline__ bf16x8 get_frag(const uint8_t* frags, int f, int lane) {
  return *reinterpret_cast<const bf16x8*>(frags + f * kFrag + lane * 16);
}

// NT: column tiles of 16 of a team.
template <int DK, int NT>
struct TeamLds {  // of every column tile: fragments of the first part, then of the second, and (not of N) of the third
  static constexpr int KB = DK / 32;
  static constexpr int kStateTile = 3 * KB * kFrag, kRowTile = 4 * kFrag, kRowTile3 = 6 * kFrag;
  static constexpr int kState = 0;
  static constexpr int kX = kState + NT * kStateTile;
  static constexpr int kN = kX + NT * kRowTile3;
  static constexpr int kW = kN + NT * kRowTile;
  static constexpr int kTileX = kW + NT * kRowTile3;
  static constexpr int kXRow = 16 * NT + 4;             // elements of a token's columns
  static constexpr int kTileK = (kTileX + kChunk * kXRow * 2 + 63) / 64 * 64;
  static constexpr int kForward = kTileK + Tile<DK>::BYTES;
  static constexpr int kTileQ = kForward;               // backward only
  static constexpr int kDX = kTileQ + Tile<DK>::BYTES;  // dX, high parts only
  static constexpr int kBackward = kDX + NT * 2 * kFrag;
};

// What wavefront w needs of a chunk. Several of them take turns, so that nothing is copied.
template <int KB, int NT>
struct TeamChunk {
  bf16x8 kf[KB], qf[KB];
  bf16x8 mh[2], mm[2], ml[2], pf[2], pl[2];
  f32x4 grown, keep;
  float grown_row, total;
  u32x2 x[NT];  // 4 NT columns of a token of V (backward: of dO), on their way into LDS
};

template <int DK, int NT, bool COLS>
struct Team {
  static constexpr int KB = DK / 32, KA = DK / 16, OWN = KA >= 4 ? KA / 4 : 1;  // OWN: state tiles of a wavefront
  static constexpr int kBlockBytes = block_bytes(DK);
  typedef TeamChunk<KB, NT> Chunk;
  typedef TeamLds<DK, NT> L;
  const DeltaParams& p;
  int wave, lane, l16, grp, col0, h, b, len, chunks;
  int64_t unit;
  bool owner;
  // The chunk that is requested next: uniform pointers that move by whole chunks, and byte offsets of this lane that stay (token strides are
  // below 2^24 elements), so that a request costs no arithmetic.
  const uint8_t *k_at, *q_at, *x_at, *block_at;
  int64_t k_step, q_step, x_step;
  int32_t k_ld, q_ld, x_ld, k_less, q_less, x_less;  // bytes from row to row, and what a row is short of that
  int at, n_at;
  Buffer block;
  uint32_t k_off[KB], q_off[KB], x_off[NT], frag_off[2], row_off;

  __device__ __forceinline__ Team(const DeltaParams& params) : p(params) {
    const int tid = threadIdx.x;
    wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    lane = tid % kWave, l16 = lane % 16, grp = lane / 16;
    const uint32_t col_groups = (p.dv + 16 * NT - 1) / (16 * NT);
    const uint32_t block = xcd_remap(blockIdx.x, gridDim.x);  // the columns of a head, which read the same rows, on one die's L2
    const uint32_t head = block / col_groups;
    unit = head;
    col0 = static_cast<int>(block % col_groups) * 16 * NT;
    h = static_cast<int>(head % static_cast<uint32_t>(p.H));
    b = static_cast<int>(head / static_cast<uint32_t>(p.H));
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
#pragma unroll
    for (int n = 0; n < NT; ++n)
      x_off[n] = col0 + 16 * n + lane % 4 * 4 < p.dv ? (16 * wave + lane / 4) * x_ld + 32 * n + lane % 4 * 8 : kNowhere;
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
#pragma unroll
    for (int n = 0; n < NT; ++n) c.x[n] = read4(x, x_off[n]);
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
      c.mm[tk] = read8(block, frag_off[tk], kBlockMid);
      if (!COLS) c.ml[tk] = read8(block, frag_off[tk], kBlockLow);
      c.pf[tk] = read8(block, frag_off[tk], kBlockP);
      if (COLS || low_scores(DK)) c.pl[tk] = read8(block, frag_off[tk], COLS ? kBlockLow : kBlockPLow);
    }
    at += COLS ? -1 : 1;
    k_at += k_step, q_at += q_step, x_at += x_step;
    block_at += COLS ? -kBlockBytes : kBlockBytes;
  }

  // The columns of V (dO) in LDS, token by token: written behind a chunk's last use of them, read by columns.
  __device__ __forceinline__ void place(const Chunk& c, bf16_t* tile_x) const {
#pragma unroll
    for (int n = 0; n < NT; ++n) *reinterpret_cast<u32x2*>(tile_x + (16 * wave + lane / 4) * L::kXRow + 16 * n + lane % 4 * 4) = c.x[n];
  }
  __device__ __forceinline__ bf16x4 values(const bf16_t* tile_x, int token0, int n) const {  // tokens token0 + 4 grp .. of column 16 n + l16
    return Tile<DK>::read_tr(tile_x + (token0 + 4 * grp + l16 / 4) * L::kXRow + 16 * n + l16 % 4 * 4);
  }
  __device__ __forceinline__ bool col_ok(int n) const { return col0 + 16 * n + l16 < p.dv; }

  // Writes without branches, as the reads. The own rows of the state, bf16, at dst [dv][dk]:
  __device__ __forceinline__ void state_offsets(uint32_t (&off)[OWN][NT]) const {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const int row = state_row(wave * OWN + i, 4 * grp);
        off[i][n] = owner && col_ok(n) && row < p.dk ? static_cast<uint32_t>((col0 + 16 * n + l16) * p.dk + row) * 2 : kNowhere;
      }
  }
  __device__ __forceinline__ void store_state(bf16_t* dst, const uint32_t (&off)[OWN][NT], const f32x4 (&s)[OWN][NT]) const {
    const Buffer to = buffer_of(dst, static_cast<uint32_t>(p.dk * p.dv) * 2);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < OWN; ++i) write4(to, off[i][n], round4(s[i][n]));
  }
  // four columns of the own token in rows ld elements apart
  __device__ __forceinline__ void quad_offsets(int64_t ld, uint32_t (&off)[NT]) const {
#pragma unroll
    for (int n = 0; n < NT; ++n)
      off[n] = col0 + 16 * n + 4 * grp < p.dv ? static_cast<uint32_t>((16 * wave + l16) * ld + 16 * n + 4 * grp) * 2 : kNowhere;
  }
};

template <int DK, int NT, bool TRAIN>
__global__ __launch_bounds__(4 * kWave) void delta_team_kernel(const DeltaParams p) {
  typedef Team<DK, NT, false> M;
  typedef TeamLds<DK, NT> L;
  typedef Tile<DK> TK;
  constexpr int KB = M::KB, OWN = M::OWN;
  extern __shared__ __attribute__((aligned(64))) uint8_t smem[];
  bf16_t *tile_k = reinterpret_cast<bf16_t*>(smem + L::kTileK), *tile_x = reinterpret_cast<bf16_t*>(smem + L::kTileX);
  uint8_t *s_frags = smem + L::kState, *x_frags = smem + L::kX, *n_frags = smem + L::kN, *w_frags = smem + L::kW;
  M m(p);
  const int wave = m.wave, lane = m.lane, l16 = m.l16, grp = m.grp, col0 = m.col0;
  bf16_t* o0 = p.o + m.b * p.os[0] + m.h * p.os[1] + col0;
  uint32_t o_off[NT], n_off[NT], s_off[OWN][NT];
  m.quad_offsets(p.os[2], o_off);
  m.quad_offsets(p.dv, n_off);
  m.state_offsets(s_off);
  // Lane (column c, tokens 4 q ..) of a half fragment holds four tokens: read_tr over the lanes c = 4 grp + l16 / 4, q = l16 % 4.
  const uint32_t turned_at = (wave / 2) * kFrag + (l16 % 4 * 16 + 4 * grp + l16 / 4) * 16 + wave % 2 * 8;

  f32x4 s[OWN][NT];
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    const int a = wave * OWN + i;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      s[i][n] = zero4();
      if (p.state_in != nullptr && m.col_ok(n) && m.owner) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = state_row(a, 4 * grp + r);
          if (row < p.dk) s[i][n][r] = p.state_in[(m.unit * p.dk + row) * p.dv + col0 + 16 * n + l16];
        }
      }
      if (m.owner) put_half3(s_frags + n * L::kStateTile, a, lane, s[i][n], KB * kFrag);
    }
  }

  bf16_t* o_at = o0;
  bf16_t* state_at = TRAIN ? p.chunk_states + m.unit * p.chunks * static_cast<int64_t>(p.dk) * p.dv : nullptr;
  bf16_t* miss_at = TRAIN ? p.misses + m.unit * p.T * p.dv + col0 : nullptr;
  const int64_t low_at = TRAIN ? p.misses_low - p.misses : 0;
  auto step = [&](int chunk, typename M::Chunk& cur, typename M::Chunk& next) __attribute__((always_inline)) {
    const int n_tok = m.tokens_of(chunk);
    m.fetch_keys(next);
    if (TRAIN) {
      m.store_state(state_at, s_off, s);
      state_at += p.dk * p.dv;
    }
    // X of the own tokens; K's rows on their way into LDS
    f32x4 x[NT], out[NT];  // out, the state's part of the output: lane = token, four columns each
    bf16x8 sh[NT][NT > 1 ? 1 : KB], sl[NT][NT > 1 ? 1 : KB];  // of one column tile the state's fragments stay for the output
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4 y = zero4(), y2 = zero4();
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const uint8_t* state = s_frags + n * L::kStateTile;
        const bf16x8 hi = get_frag(state, kb, lane), mid = get_frag(state + KB * kFrag, kb, lane);
        y = mfma16(cur.kf[kb], hi, y);
        y2 = mfma16(cur.kf[kb], mid, y2);
        y2 = mfma16(cur.kf[kb], get_frag(state + 2 * KB * kFrag, kb, lane), y2);
        if (NT == 1) sh[n][NT > 1 ? 0 : kb] = hi, sl[n][NT > 1 ? 0 : kb] = mid;
      }
      const bf16x4 v = m.values(tile_x, 16 * wave, n);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[n][r] = fmaf(-cur.grown[r], y[r] + y2[r], static_cast<float>(v[r]));
      put_half3(x_frags + n * L::kRowTile3, wave, lane, x[n], 2 * kFrag);
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      *reinterpret_cast<bf16x8*>(tile_k + (16 * wave + l16) * TK::STRIDE + kb * 32 + grp * 8) = cur.kf[kb];
    __syncthreads();
    m.fetch_queries(next);

    // N of the own tokens
    const float grown = cur.grown_row * p.scale;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint8_t* from = x_frags + n * L::kRowTile3;
      f32x4 x2 = zero4(), x3 = zero4();  // products of parts whose sizes are 2^-8 and 2^-16 of the first ones'
#pragma unroll
      for (int tk = 0; tk < 2; ++tk)
        if (tk <= wave / 2) {
          const bf16x8 xh = get_frag(from, tk, lane), xm = get_frag(from + 2 * kFrag, tk, lane), xl = get_frag(from + 4 * kFrag, tk, lane);
          x[n] = mfma16(cur.mh[tk], xh, x[n]);
          x2 = mfma16(cur.mh[tk], xm, x2);
          x3 = mfma16(cur.mh[tk], xl, x3);
          x2 = mfma16(cur.mm[tk], xh, x2);
          x3 = mfma16(cur.mm[tk], xm, x3);
          x3 = mfma16(cur.ml[tk], xh, x3);
        }
      f32x4 out2 = zero4();
      out[n] = zero4();
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const uint8_t* state = s_frags + n * L::kStateTile;
        out[n] = mfma16(NT == 1 ? sh[n][NT > 1 ? 0 : kb] : get_frag(state, kb, lane), cur.qf[kb], out[n]);
        out2 = mfma16(NT == 1 ? sl[n][NT > 1 ? 0 : kb] : get_frag(state + KB * kFrag, kb, lane), cur.qf[kb], out2);
      }
      f32x4 w;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[n][r] += x2[r] + x3[r];
        w[r] = x[n][r] * cur.keep[r];
      }
      put_half3(w_frags + n * L::kRowTile3, wave, lane, w, 2 * kFrag);
      put_half(n_frags + n * L::kRowTile, wave, lane, x[n], 2 * kFrag);
#pragma unroll
      for (int r = 0; r < 4; ++r) out[n][r] = (out[n][r] + out2[r]) * grown;
    }
    __syncthreads();
    m.fetch_block(next);

    // the own rows of the state
    if (m.owner) {
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const int a = wave * OWN + i;
        bf16x8 kt[2];
#pragma unroll
        for (int tk = 0; tk < 2; ++tk) kt[tk] = TK::keys_frag(tile_k, tk, a, l16, grp);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint8_t* from = w_frags + n * L::kRowTile3;
          f32x4 s2 = zero4();
#pragma unroll
          for (int r = 0; r < 4; ++r) s[i][n][r] *= cur.total;
#pragma unroll
          for (int tk = 0; tk < 2; ++tk) {
            s[i][n] = mfma16(kt[tk], get_frag(from, tk, lane), s[i][n]);
            s2 = mfma16(kt[tk], get_frag(from + 2 * kFrag, tk, lane), s2);
            s2 = mfma16(kt[tk], get_frag(from + 4 * kFrag, tk, lane), s2);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) s[i][n][r] += s2[r];
          put_half3(s_frags + n * L::kStateTile, a, lane, s[i][n], KB * kFrag);
        }
      }
    }
    // the output of the own tokens
    const Buffer to = rows_buffer(o_at, p.os[2], n_tok, p.dv - col0);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint8_t* from = n_frags + n * L::kRowTile;
      f32x4 out2 = zero4();
#pragma unroll
      for (int tk = 0; tk < 2; ++tk)
        if (tk <= wave / 2) {
          const bf16x8 nh = get_frag(from, tk, lane);
          out[n] = mfma16(nh, cur.pf[tk], out[n]);
          out2 = mfma16(get_frag(from + 2 * kFrag, tk, lane), cur.pf[tk], out2);
          if (low_scores(DK)) out2 = mfma16(nh, cur.pl[tk], out2);
        }
#pragma unroll
      for (int r = 0; r < 4; ++r) out[n][r] += out2[r];
      write4(to, o_off[n], round4(out[n]));
    }
    if (TRAIN) {  // both parts of N of the own tokens, by rows
      const Buffer misses = rows_buffer(miss_at, p.dv, n_tok, p.dv - col0), low = rows_buffer(miss_at + low_at, p.dv, n_tok, p.dv - col0);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint8_t* from = n_frags + n * L::kRowTile + turned_at;
        write4(misses, n_off[n], __builtin_bit_cast(u32x2, TK::read_tr(reinterpret_cast<const bf16_t*>(from))));
        write4(low, n_off[n], __builtin_bit_cast(u32x2, TK::read_tr(reinterpret_cast<const bf16_t*>(from + 2 * kFrag))));
      }
      miss_at += kChunk * p.dv;
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

  if (p.state_out != nullptr && m.owner) {
#pragma unroll
    for (int i = 0; i < OWN; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = state_row(wave * OWN + i, 4 * grp + r);
          if (row < p.dk && m.col_ok(n)) p.state_out[(m.unit * p.dk + row) * p.dv + col0 + 16 * n + l16] = s[i][n][r];
        }
  }
  const bf16x4 none = {};
  for (int64_t i = threadIdx.x; i < static_cast<int64_t>(p.T - m.len) * 4 * NT; i += 4 * kWave) {
    const int at = static_cast<int>(i % (4 * NT)) * 4;
    if (col0 + at < p.dv) *reinterpret_cast<bf16x4*>(o0 + (m.len + i / (4 * NT)) * p.os[2] + at) = none;
  }
}

// The gradient of the state, chunks last to first (the formulas: delta.h). Stages: beta dU (own tokens) | dX (own tokens) | dS (own
// rows). dO is read as fragments by every wavefront.
template <int DK, int NT>
__global__ __launch_bounds__(4 * kWave) void delta_team_back_kernel(const DeltaParams p) {
  typedef Team<DK, NT, true> M;
  typedef TeamLds<DK, NT> L;
  typedef Tile<DK> TK;
  constexpr int KB = M::KB, OWN = M::OWN;
  extern __shared__ __attribute__((aligned(64))) uint8_t smem[];
  bf16_t *tile_k = reinterpret_cast<bf16_t*>(smem + L::kTileK), *tile_q = reinterpret_cast<bf16_t*>(smem + L::kTileQ),
         *tile_x = reinterpret_cast<bf16_t*>(smem + L::kTileX);
  uint8_t *s_frags = smem + L::kState, *z_frags = smem + L::kX, *x_frags = smem + L::kN, *o_frags = smem + L::kW;
  M m(p);
  const int wave = m.wave, lane = m.lane, l16 = m.l16, grp = m.grp, col0 = m.col0;
  uint8_t* dx_frags = smem + L::kDX;
  const uint32_t turned_at = (wave / 2) * kFrag + (l16 % 4 * 16 + 4 * grp + l16 / 4) * 16 + wave % 2 * 8;  // as in the forward
  bf16_t* v0 = p.grad_v + m.b * p.dvs[0] + m.h * p.dvs[1] + col0;
  uint32_t v_off[NT], s_off[OWN][NT];
  m.quad_offsets(p.dvs[2], v_off);
  m.state_offsets(s_off);

  f32x4 s[OWN][NT];
#pragma unroll
  for (int i = 0; i < OWN; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      s[i][n] = zero4();
      if (m.owner) put_half(s_frags + n * L::kStateTile, wave * OWN + i, lane, s[i][n], KB * kFrag);
    }

  bf16_t* v_at = v0 + (m.chunks - 1) * kChunk * p.dvs[2];
  bf16_t* state_at = p.grad_states + (m.unit * p.chunks + m.chunks - 1) * static_cast<int64_t>(p.dk) * p.dv;
  auto step = [&](int chunk, typename M::Chunk& cur, typename M::Chunk& next) __attribute__((always_inline)) {
    const int n_tok = m.tokens_of(chunk);
    m.fetch_keys(next);
    m.store_state(state_at, s_off, s);
    state_at -= p.dk * p.dv;
    // beta dU of the own tokens
    f32x4 z[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4 z2 = zero4(), z3 = zero4();
      z[n] = zero4();
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        z[n] = mfma16(cur.kf[kb], get_frag(s_frags + n * L::kStateTile, kb, lane), z[n]);
        z2 = mfma16(cur.kf[kb], get_frag(s_frags + n * L::kStateTile + KB * kFrag, kb, lane), z2);
      }
#pragma unroll
      for (int tk = 0; tk < 2; ++tk)
        if (tk >= wave / 2) {
          const bf16x8 of = TK::join(m.values(tile_x, 32 * tk, n), m.values(tile_x, 32 * tk + 16, n));
          z3 = mfma16(cur.pf[tk], of, z3);
          z3 = mfma16(cur.pl[tk], of, z3);
        }
      f32x4 w;
      const bf16x4 own = m.values(tile_x, 16 * wave, n);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        z[n][r] = fmaf(cur.keep[r], z[n][r] + z2[r], z3[r]);
        w[r] = p.scale * cur.grown[r] * static_cast<float>(own[r]);
      }
      put_half(z_frags + n * L::kRowTile, wave, lane, z[n], 2 * kFrag);
      put_half(o_frags + n * L::kRowTile, wave, lane, w, 2 * kFrag);
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int at = (16 * wave + l16) * TK::STRIDE + kb * 32 + grp * 8;
      *reinterpret_cast<bf16x8*>(tile_k + at) = cur.kf[kb];
      *reinterpret_cast<bf16x8*>(tile_q + at) = cur.qf[kb];
    }
    __syncthreads();
    m.fetch_queries(next);

    // dX of the own tokens
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint8_t* from = z_frags + n * L::kRowTile;
      f32x4 z2 = zero4(), z3 = zero4(), w;
#pragma unroll
      for (int tk = 0; tk < 2; ++tk)
        if (tk >= wave / 2) {
          const bf16x8 zh = get_frag(from, tk, lane), zl = get_frag(from + 2 * kFrag, tk, lane);
          z[n] = mfma16(cur.mh[tk], zh, z[n]);
          z2 = mfma16(cur.mh[tk], zl, z2);
          z3 = mfma16(cur.mm[tk], zh, z3);
        }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        z[n][r] += z2[r] + z3[r];
        w[r] = -cur.grown[r] * z[n][r];
      }
      put_half(x_frags + n * L::kRowTile, wave, lane, w, 2 * kFrag);
      *reinterpret_cast<u32x2*>(dx_frags + n * 2 * kFrag + (wave / 2) * kFrag + lane * 16 + wave % 2 * 8) = round4(z[n]);
    }
    __syncthreads();
    m.fetch_block(next);

    // dS of the own rows
    if (m.owner) {
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const int a = wave * OWN + i;
        bf16x8 kt[2], qt[2];
#pragma unroll
        for (int tk = 0; tk < 2; ++tk) kt[tk] = TK::keys_frag(tile_k, tk, a, l16, grp), qt[tk] = TK::keys_frag(tile_q, tk, a, l16, grp);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint8_t *from_x = x_frags + n * L::kRowTile, *from_o = o_frags + n * L::kRowTile;
          f32x4 s2 = zero4(), s3 = zero4(), s4 = zero4();
#pragma unroll
          for (int r = 0; r < 4; ++r) s[i][n][r] *= cur.total;
#pragma unroll
          for (int tk = 0; tk < 2; ++tk) {
            s[i][n] = mfma16(kt[tk], get_frag(from_x, tk, lane), s[i][n]);
            s2 = mfma16(kt[tk], get_frag(from_x + 2 * kFrag, tk, lane), s2);
            s3 = mfma16(qt[tk], get_frag(from_o, tk, lane), s3);
            s4 = mfma16(qt[tk], get_frag(from_o + 2 * kFrag, tk, lane), s4);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) s[i][n][r] += (s2[r] + s4[r]) + s3[r];
          put_half(s_frags + n * L::kStateTile, a, lane, s[i][n], KB * kFrag);
        }
      }
    }
    const Buffer to = rows_buffer(v_at, p.dvs[2], n_tok, p.dv - col0);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bf16x4 rounded = TK::read_tr(reinterpret_cast<const bf16_t*>(dx_frags + n * 2 * kFrag + turned_at));
      write4(to, v_off[n], __builtin_bit_cast(u32x2, rounded));
    }
    v_at -= kChunk * p.dvs[2];
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
  const bf16x4 none = {};
  for (int64_t i = threadIdx.x; i < static_cast<int64_t>(p.T - m.len) * 4 * NT; i += 4 * kWave) {
    const int at = static_cast<int>(i % (4 * NT)) * 4;
    if (col0 + at < p.dv) *reinterpret_cast<bf16x4*>(v0 + (m.len + i / (4 * NT)) * p.dvs[2] + at) = none;
  }
}

template <typename K>
int launch_columns(const char* name, K* kernel, const DeltaParams& p, int64_t teams, int lds, hipStream_t s) {
  if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
    return set_error(TAAC_ERR_LAUNCH, "%s: cannot reserve %d bytes of LDS", name, lds);
  hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(teams)), dim3(4 * kWave), lds, s, p);
  return check_launch(name);
}

template <int DK, int NT, bool COLS>
int launch_team(const char* name, const DeltaParams& p, hipStream_t s) {
  typedef TeamLds<DK, NT> L;
  const int64_t heads = static_cast<int64_t>(p.B) * p.H, teams = heads * ((p.dv + 16 * NT - 1) / (16 * NT));
  if (heads * p.chunks > 0x7fffffffLL || teams > 0x7fffffffLL) return set_error(TAAC_ERR_UNSUPPORTED, "%s: too many workgroups", name);
  if (p.chunks > 0) hipLaunchKernelGGL((delta_blocks_kernel<DK, COLS>), dim3(static_cast<uint32_t>(heads * p.chunks)), dim3(kWave), 0, s, p);
  if constexpr (COLS) return launch_columns(name, delta_team_back_kernel<DK, NT>, p, teams, L::kBackward, s);
  else if (p.chunk_states != nullptr) return launch_columns(name, delta_team_kernel<DK, NT, true>, p, teams, L::kForward, s);
  else return launch_columns(name, delta_team_kernel<DK, NT, false>, p, teams, L::kForward, s);
}

}  // namespace

int delta_team(const char* name, const DeltaParams& p, bool back, hipStream_t s) {
  if (p.dk <= 32) return back ? launch_team<32, 1, true>(name, p, s) : launch_team<32, 1, false>(name, p, s);
  if (p.dk <= 64) return back ? launch_team<64, 1, true>(name, p, s) : launch_team<64, 1, false>(name, p, s);
  // Two teams run on a CU at once: where there would be more of 16 columns, teams of 32, which read the keys and the blocks half as often.
  if (p.dv > 16 && static_cast<int64_t>(p.B) * p.H * ((p.dv + 15) / 16) > 512)
    return back ? launch_team<128, 2, true>(name, p, s) : launch_team<128, 2, false>(name, p, s);
  return back ? launch_team<128, 1, true>(name, p, s) : launch_team<128, 1, false>(name, p, s);
}

}  // namespace taac
