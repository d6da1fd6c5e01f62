// Gated delta rule, chunked form, for many heads of at most 64 key features (the mathematics, operand order and precision: delta.h).
//
// With many (sample, head) pairs the time is work and memory traffic, not the chain of chunks: a wavefront walks the tokens of one head
// and 32 value columns on its own, without a barrier, and everything it makes for a chunk stays in its registers. It takes 64 tokens
// at a time from memory and walks them as two chunks of 32, which need a third of the fp32 products of one chunk of 64: the four
// diagonal blocks of 16 are still solved at once, a column per lane, but only one block below the diagonal is left per chunk
// instead of six per 64 tokens. Scores are made where they are used.
//
// Bound by instruction issue. 1024 samples x 8 heads of up to 512 tokens (276 at the mean), 32 wide, forward: 246 us in a trace, 3.0 TB/s; two
// wavefronts per SIMD issue in 73 % of the cycles, vector instructions in 55 %, many of those to take fp32 operands apart; the matrix units are busy
// for 23 %. 512 x 4 heads of up to 512, 64 wide: 244 us with the states and misses of training, 197 us backward; there one wavefront per SIMD fills
// the registers (two spill and take 10 % longer), which issues in half of the cycles and waits in a quarter, covered by no other wavefront.
#include "delta.h"

namespace taac {
namespace {

constexpr int kHalf = 32, kSoloCols = 32, kNT = 2;

template <int DK>
struct SoloLds {
  typedef Tile<DK> TK;
  typedef Tile<kSoloCols> TV;
  static constexpr int kTileV = TK::BYTES;
  static constexpr int kTileQ = kTileV + TV::BYTES;  // its first bytes are the scratch of the solution, in front of Q
  static constexpr int kTotal = kTileQ + (TK::BYTES > kScratchFloats * 4 ? TK::BYTES : kScratchFloats * 4);
};

// Floats of the 64 tokens in LDS: G as a pair, beta; e^(G - G in front of the tile of 16), e^(G behind the tile - G) beta; and over the chunk of 32:
// e^(G - G in front of it), beta e^(G behind it - G). Behind them the decay of each chunk.
constexpr int kSoloHi = 0, kSoloLow = 64, kSoloBeta = 128, kSoloIn = 192, kSoloOut = 256, kSoloGrown = 320, kSoloKeep = 384, kSoloTotal = 448,
              kSoloFloats = 452;

template <int DK>
struct SoloTokens {
  bf16x8 kf[4][DK / 32], qf[4][DK / 32], x[4];  // x: pieces of the values (backward: of dO)
  GateBits gates;
};

template <int DK, bool BACK>
struct Solo {
  static constexpr int KB = DK / 32, KA = DK / 16;
  typedef Tile<DK> TK;
  typedef Tile<kSoloCols> TV;
  const DeltaParams& p;
  int lane, l16, grp, col0, h, b, len, groups;
  int64_t unit;
  // The 64 tokens that are requested next: uniform pointers that move by whole groups, and byte offsets of this lane.
  const uint8_t *k_at, *q_at, *x_at;
  int64_t k_step, q_step, x_step;
  int32_t k_ld, q_ld, x_ld, k_less, q_less, x_less;  // bytes from row to row, and what a row is short of that
  int at;
  uint32_t k_off[KB], q_off[KB], state_off[KB], x_off;

  __device__ __forceinline__ Solo(const DeltaParams& params) : p(params) {
    lane = threadIdx.x, l16 = lane % 16, grp = lane / 16;
    const uint32_t col_groups = (p.dv + kSoloCols - 1) / kSoloCols;
    const uint32_t block = xcd_remap(blockIdx.x, gridDim.x);  // the columns of a head, which read the same rows, on one die's L2
    const uint32_t head = block / col_groups;
    unit = head;
    col0 = static_cast<int>(block % col_groups) * kSoloCols;
    h = static_cast<int>(head % static_cast<uint32_t>(p.H));
    b = static_cast<int>(head / static_cast<uint32_t>(p.H));
    len = p.T;
    if (p.lengths != nullptr) {
      len = p.lengths[b];
      len = len < 0 ? 0 : (len > p.T ? p.T : len);
    }
    groups = (len + kChunk - 1) / kChunk;
    const int64_t hk = h / p.group;
    const int64_t* xs = BACK ? p.dos : p.vs;
    at = BACK ? groups - 1 : 0;
    const int64_t first = static_cast<int64_t>(at) * kChunk;
    k_at = reinterpret_cast<const uint8_t*>(p.k + b * p.ks[0] + hk * p.ks[1] + first * p.ks[2]);
    q_at = reinterpret_cast<const uint8_t*>(p.q + b * p.qs[0] + hk * p.qs[1] + first * p.qs[2]);
    x_at = reinterpret_cast<const uint8_t*>((BACK ? p.grad_o : p.v) + b * xs[0] + h * xs[1] + col0 + first * xs[2]);
    constexpr int64_t kMove = (BACK ? -kChunk : kChunk) * 2;
    k_step = kMove * p.ks[2], q_step = kMove * p.qs[2], x_step = kMove * xs[2];
    k_ld = static_cast<int32_t>(p.ks[2]) * 2, q_ld = static_cast<int32_t>(p.qs[2]) * 2, x_ld = static_cast<int32_t>(xs[2]) * 2;
    k_less = k_ld - p.dk * 2, q_less = q_ld - p.dk * 2, x_less = x_ld - (p.dv - col0) * 2;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const bool there = kb * 32 + grp * 8 < p.dk;
      k_off[kb] = there ? l16 * k_ld + kb * 64 + grp * 16 : kNowhere;
      q_off[kb] = there ? l16 * q_ld + kb * 64 + grp * 16 : kNowhere;
      state_off[kb] = there ? static_cast<uint32_t>(l16 * p.dk + 32 * kb + 8 * grp) * 2 : kNowhere;
    }
    const int piece = lane % 4;
    x_off = col0 + piece * 8 < p.dv ? static_cast<uint32_t>(lane / 4 * x_ld) + piece * 16 : kNowhere;
  }
  __device__ __forceinline__ int tokens_of(int group) const {
    const int left = len - group * kChunk;
    return left < kChunk ? left : kChunk;
  }

  // The first n rows at a base; none where n is not positive.
  static __device__ __forceinline__ Buffer rows_at(const uint8_t* base, int n, int32_t ld, int32_t less) {
    const int32_t bytes = n * ld - less;
    return buffer_of(base, bytes > 0 ? bytes : 0);
  }
  // The tokens of a group, then on to the next; behind the last group, zeros.
  __device__ __forceinline__ void fetch(SoloTokens<DK>& c) {
    const int n = at >= 0 ? tokens_of(at) : 0;
    c.gates.request(p, b, h, static_cast<int64_t>(at) * kChunk, n, lane);
    const Buffer k = rows_at(k_at, n, k_ld, k_less), q = rows_at(q_at, n, q_ld, q_less), x = rows_at(x_at, n, x_ld, x_less);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) c.kf[t][kb] = read8(k, k_off[kb] + t * 16 * k_ld);
#pragma unroll
    for (int t = 0; t < 4; ++t) c.x[t] = read8(x, x_off + t * 16 * x_ld);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) c.qf[t][kb] = read8(q, q_off[kb] + t * 16 * q_ld);
    at += BACK ? -1 : 1;
    k_at += k_step, q_at += q_step, x_at += x_step;
  }

  // The tokens' factors and rows into LDS.
  __device__ __forceinline__ void place(const SoloTokens<DK>& c, int n_tok, float* rows, bf16_t* tile_k, bf16_t* tile_x) const {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int at = (16 * t + l16) * TK::STRIDE + kb * 32 + grp * 8;
        *reinterpret_cast<bf16x8*>(tile_k + at) = c.kf[t][kb];
      }
      *reinterpret_cast<bf16x8*>(tile_x + (16 * t + lane / 4) * TV::STRIDE + (lane % 4) * 8) = c.x[t];
    }
    const float beta = c.gates.step(p, lane < n_tok);
    double total = c.gates.decay(p, lane < n_tok);
#pragma unroll
    for (int off = 1; off < kWave; off *= 2) {
      const double up = __shfl_up(total, off, kWave);
      if (lane >= off) total += up;
    }
    const double tile_end = __shfl(total, lane | 15, kWave), half_end = __shfl(total, lane | 31, kWave);
    double tile_start = __shfl(total, lane < 16 ? 0 : (lane & ~15) - 1, kWave), half_start = __shfl(total, 31, kWave);
    if (lane < 16) tile_start = 0.0;
    if (lane < 32) half_start = 0.0;
    const float hi = static_cast<float>(total - half_start);
    const float grown = __builtin_amdgcn_exp2f(hi);
    rows[kSoloHi + lane] = hi;
    rows[kSoloLow + lane] = static_cast<float>(total - half_start - static_cast<double>(hi));
    rows[kSoloBeta + lane] = beta;
    rows[kSoloIn + lane] = __builtin_amdgcn_exp2f(static_cast<float>(total - tile_start));
    rows[kSoloOut + lane] = __builtin_amdgcn_exp2f(static_cast<float>(tile_end - total)) * beta;
    rows[kSoloGrown + lane] = grown;
    rows[kSoloKeep + lane] = __builtin_amdgcn_exp2f(static_cast<float>(half_end - total)) * beta;
    if ((lane & 31) == 31) rows[kSoloTotal + lane / 32] = grown;
    wave_sync();
  }
  // Q's rows, in the place of the solution's scratch; c holds nothing of these tokens any more.
  __device__ __forceinline__ void place_queries(const SoloTokens<DK>& c, bf16_t* tile_q) const {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) *reinterpret_cast<bf16x8*>(tile_q + (16 * t + l16) * TK::STRIDE + kb * 32 + grp * 8) = c.qf[t][kb];
    wave_sync();
  }

  // Gam_ij beta_j of a tile of 16 x 16, by rows (lane: token i = l16 of tile ti, tokens j = 4 grp .. of tile tj); of a diagonal one, whatever for j > i.
  __device__ __forceinline__ f32x4 decays_by_rows(const float* rows, int ti, int tj) const {
    f32x4 gam;
    if (ti > tj) {
      const float in_i = rows[kSoloIn + 16 * ti + l16];
      const f32x4 out_j = *reinterpret_cast<const f32x4*>(rows + kSoloOut + 16 * tj + 4 * grp);
#pragma unroll
      for (int r = 0; r < 4; ++r) gam[r] = in_i * out_j[r];
    } else {
      const float hi_i = rows[kSoloHi + 16 * ti + l16], lo_i = rows[kSoloLow + 16 * ti + l16];
      const f32x4 hi_j = *reinterpret_cast<const f32x4*>(rows + kSoloHi + 16 * tj + 4 * grp);
      const f32x4 lo_j = *reinterpret_cast<const f32x4*>(rows + kSoloLow + 16 * tj + 4 * grp);
      const f32x4 beta_j = *reinterpret_cast<const f32x4*>(rows + kSoloBeta + 16 * tj + 4 * grp);
#pragma unroll
      for (int r = 0; r < 4; ++r) gam[r] = __builtin_amdgcn_exp2f((hi_i - hi_j[r]) + (lo_i - lo_j[r])) * beta_j[r];
    }
    return gam;
  }
  // The same by columns (lane: token j = l16 of tile tj, tokens i = 4 grp .. of tile ti).
  __device__ __forceinline__ f32x4 decays_by_cols(const float* rows, int ti, int tj) const {
    f32x4 gam;
    if (ti > tj) {
      const float out_j = rows[kSoloOut + 16 * tj + l16];
      const f32x4 in_i = *reinterpret_cast<const f32x4*>(rows + kSoloIn + 16 * ti + 4 * grp);
#pragma unroll
      for (int r = 0; r < 4; ++r) gam[r] = out_j * in_i[r];
    } else {
      const float hi_j = rows[kSoloHi + 16 * tj + l16], lo_j = rows[kSoloLow + 16 * tj + l16], beta_j = rows[kSoloBeta + 16 * tj + l16];
      const f32x4 hi_i = *reinterpret_cast<const f32x4*>(rows + kSoloHi + 16 * ti + 4 * grp);
      const f32x4 lo_i = *reinterpret_cast<const f32x4*>(rows + kSoloLow + 16 * ti + 4 * grp);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = __builtin_amdgcn_exp2f((hi_i[r] - hi_j) + (lo_i[r] - lo_j)) * beta_j;
        gam[r] = 4 * grp + r >= l16 ? e : 0.f;
      }
    }
    return gam;
  }

  // The blocks of -M of both chunks, fp32: the diagonal ones of each tile of 16, and the one below them of each chunk. By rows (forward); by columns
  // (backward), which are the rows of its transpose. own: the diagonal tiles' decays, which the forward's scores take too.
  __device__ __forceinline__ void solve(const SoloTokens<DK>& c, const float* rows, float* scratch, f32x4 (&diag)[4], f32x4 (&below)[2],
                                        f32x4 (&own)[4]) const {
    f32x4 low[2];  // the blocks below the diagonal, by rows
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f32x4 kk = zero4();
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) kk = mfma16(c.kf[t][kb], c.kf[t][kb], kk);
      own[t] = decays_by_rows(rows, t, t);
#pragma unroll
      for (int r = 0; r < 4; ++r) kk[r] = l16 > 4 * grp + r ? kk[r] * own[t][r] : 0.f;
      *reinterpret_cast<f32x4*>(scratch + t * kScratchBlock + l16 * kScratchRow + 4 * grp) = kk;
    }
    wave_sync();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      low[s] = zero4();
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) low[s] = mfma16(c.kf[2 * s][kb], c.kf[2 * s + 1][kb], low[s]);
      const f32x4 gam = decays_by_rows(rows, 2 * s + 1, 2 * s);
#pragma unroll
      for (int r = 0; r < 4; ++r) low[s][r] *= gam[r];
    }
    solve_diagonal(scratch, lane);
    f32x4 m_rows[4], m_cols[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      m_rows[t] = *reinterpret_cast<const f32x4*>(scratch + t * kScratchBlock + l16 * kScratchRow + 4 * grp);
#pragma unroll
      for (int r = 0; r < 4; ++r) m_cols[t][r] = scratch[t * kScratchBlock + (4 * grp + r) * kScratchRow + l16];
    }
    wave_sync();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f32x4 t0, t1;  // T of the first block by columns, of the second by rows
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float one = l16 == 4 * grp + r ? 1.f : 0.f;
        t0[r] = one - m_cols[2 * s][r];
        t1[r] = m_rows[2 * s + 1][r] - one;  // negative: gives -M below
      }
      const f32x4 z = mul_cols(low[s], t0, zero4());
      below[s] = BACK ? mul_cols(t1, z, zero4()) : mul_rows(t1, z, zero4());
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) diag[t][r] = BACK ? -m_cols[t][r] : -m_rows[t][r];
  }
  // (I - M) X of a chunk of 32 (backward: of the transposed matrix), in place: fp32 products, since what is lost here stays in the state.
  __device__ __forceinline__ void apply(const f32x4 (&diag)[4], const f32x4 (&below)[2], int half, f32x4 (&x)[2][kNT]) const {
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      const f32x4 x0 = x[0][n], x1 = x[1][n];
      x[0][n] = mul_cols(diag[2 * half], x0, x0);
      x[1][n] = mul_cols(diag[2 * half + 1], x1, x1);
      if (BACK) x[0][n] = mul_cols(below[half], x1, x[0][n]);
      else x[1][n] = mul_cols(below[half], x0, x[1][n]);
    }
  }

  __device__ __forceinline__ void split_state(const f32x4 (&s)[KA][kNT], bf16x8 (&sh)[KB][kNT], bf16x8 (&sl)[KB][kNT]) const {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int n = 0; n < kNT; ++n) split(s[2 * kb][n], s[2 * kb + 1][n], sh[kb][n], sl[kb][n]);
  }
  __device__ __forceinline__ void split_state(const f32x4 (&s)[KA][kNT], bf16x8 (&sh)[KB][kNT], bf16x8 (&sm)[KB][kNT], bf16x8 (&sl)[KB][kNT]) const {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int n = 0; n < kNT; ++n) split3(s[2 * kb][n], s[2 * kb + 1][n], sh[kb][n], sm[kb][n], sl[kb][n]);
  }
  // the state's high parts at dst [dv][dk]
  __device__ __forceinline__ void store_state(bf16_t* dst, const bf16x8 (&sh)[KB][kNT]) const {
    const Buffer to = rows_buffer(dst + col0 * p.dk, p.dk, p.dv - col0, p.dk);
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) write8(to, state_off[kb] + n * p.dk * 32, sh[kb][n]);
  }
  // Rows of one chunk of 32 tokens, held by columns as operands over the tokens, to rows of a group from tile `first` on (off: quads(); pitch: bytes
  // of 16 rows): turned through tile's rows, which have been read.
  __device__ __forceinline__ void store_rows(Buffer to, uint32_t pitch, const uint32_t (&off)[kNT], int first, bf16_t* tile, const bf16x8 (&x)[kNT]) const {
    u32x2 v[2][kNT];
    wave_sync();
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      const u32x4 words = __builtin_bit_cast(u32x4, x[n]);
#pragma unroll
      for (int t = 0; t < 2; ++t) *reinterpret_cast<u32x2*>(tile + (2 * t + n) * 320 + l16 * 20 + grp * 4) = u32x2{words[2 * t], words[2 * t + 1]};
    }
    wave_sync();
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int n = 0; n < kNT; ++n)
        v[t][n] = __builtin_bit_cast(u32x2, TV::read_tr(tile + (2 * t + n) * 320 + (4 * grp + l16 / 4) * 20 + (l16 % 4) * 4));
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int n = 0; n < kNT; ++n) write4(to, off[n] + (first + t) * pitch, v[t][n]);
  }
  // Byte offsets of four columns of token l16 in rows ld elements apart.
  __device__ __forceinline__ void quads(int64_t ld, uint32_t (&off)[kNT]) const {
#pragma unroll
    for (int n = 0; n < kNT; ++n)
      off[n] = col0 + 16 * n + 4 * grp < p.dv ? static_cast<uint32_t>(l16 * ld + 16 * n + 4 * grp) * 2 : kNowhere;
  }
};

template <int DK, bool TRAIN>
__global__ __launch_bounds__(kWave, DK == 32 ? 2 : 1) void delta_solo_kernel(const DeltaParams p) {
  typedef Solo<DK, false> W;
  typedef SoloLds<DK> L;
  typedef Tile<DK> TK;
  typedef Tile<kSoloCols> TV;
  constexpr int KB = W::KB, KA = W::KA;
  __shared__ __attribute__((aligned(64))) uint8_t smem[L::kTotal];
  __shared__ __attribute__((aligned(16))) float rows[kSoloFloats];
  bf16_t* tile_k = reinterpret_cast<bf16_t*>(smem);
  bf16_t* tile_v = reinterpret_cast<bf16_t*>(smem + L::kTileV);
  bf16_t* tile_q = reinterpret_cast<bf16_t*>(smem + L::kTileQ);
  float* scratch = reinterpret_cast<float*>(smem + L::kTileQ);
  W w(p);
  const int lane = w.lane, l16 = w.l16, grp = w.grp, col0 = w.col0;
  bf16_t* o0 = p.o + w.b * p.os[0] + w.h * p.os[1] + col0;
  const uint32_t o_pitch = static_cast<uint32_t>(p.os[2]) * 32;  // bytes of 16 rows
  uint32_t o_off[kNT], n_off[kNT];
  w.quads(p.os[2], o_off);
  w.quads(p.dv, n_off);

  f32x4 s[KA][kNT];
#pragma unroll
  for (int a = 0; a < KA; ++a)
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      s[a][n] = zero4();
      if (p.state_in != nullptr && col0 + 16 * n + l16 < p.dv) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = state_row(a, 4 * grp + r);
          if (row < p.dk) s[a][n][r] = p.state_in[(w.unit * p.dk + row) * p.dv + col0 + 16 * n + l16];
        }
      }
    }

  SoloTokens<DK> c;
  if (w.groups > 0) w.fetch(c);
  for (int group = 0; group < w.groups; ++group) {
    const int64_t token0 = static_cast<int64_t>(group) * kChunk;
    const int n_tok = w.tokens_of(group);
    const Buffer to = rows_buffer(o0 + token0 * p.os[2], p.os[2], n_tok, p.dv - col0);
    const int64_t miss_at = (w.unit * p.T + token0) * p.dv + col0;
    const Buffer misses = rows_buffer(p.misses + miss_at, p.dv, TRAIN ? n_tok : 0, p.dv - col0);
    const Buffer misses_low = rows_buffer(p.misses_low + miss_at, p.dv, TRAIN ? n_tok : 0, p.dv - col0);
    wave_sync();  // the previous tokens' tiles are read
    w.place(c, n_tok, rows, tile_k, tile_v);
    f32x4 diag[4], below[2], own[4];
    w.solve(c, rows, scratch, diag, below, own);
    w.place_queries(c, tile_q);
    w.fetch(c);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half == 1 && n_tok <= kHalf) break;
      bf16x8 sh[KB][kNT], sm[KB][kNT], sl[KB][kNT];
      w.split_state(s, sh, sm, sl);
      if (TRAIN && half == 0) w.store_state(p.chunk_states + (w.unit * p.chunks + group) * static_cast<int64_t>(p.dk) * p.dv, sh);
      // X = V - e^G K S
      f32x4 x[2][kNT];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int ti = 2 * half + t;
        f32x4 y[kNT];
#pragma unroll
        for (int n = 0; n < kNT; ++n) y[n] = zero4();
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const bf16x8 kf = TK::row(tile_k, 16 * ti + l16, kb, grp);
#pragma unroll
          for (int n = 0; n < kNT; ++n) y[n] = mfma16(kf, sl[kb][n], mfma16(kf, sm[kb][n], mfma16(kf, sh[kb][n], y[n])));
        }
        const f32x4 grown = *reinterpret_cast<const f32x4*>(rows + kSoloGrown + 16 * ti + 4 * grp);
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          const bf16x4 v = TV::values(tile_v, 16 * ti, n, l16, grp);
#pragma unroll
          for (int r = 0; r < 4; ++r) x[t][n][r] = fmaf(-grown[r], y[n][r], static_cast<float>(v[r]));
        }
      }
      // N = X - M X
      w.apply(diag, below, half, x);
      bf16x8 xh[kNT], xl[kNT];
#pragma unroll
      for (int n = 0; n < kNT; ++n) split(x[0][n], x[1][n], xh[n], xl[n]);
      if (TRAIN) {
        w.store_rows(misses, p.dv * 32, n_off, 2 * half, tile_v + 32 * half * TV::STRIDE, xh);
        w.store_rows(misses_low, p.dv * 32, n_off, 2 * half, tile_v + 32 * half * TV::STRIDE, xl);
      }
      // the output by columns of tokens: lane = token, four value columns each
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int ti = 2 * half + t;
        bf16x8 qf[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) qf[kb] = TK::row(tile_q, 16 * ti + l16, kb, grp);
        f32x4 score[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          score[u] = zero4();
          if (u > t) continue;
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) score[u] = mfma16(TK::row(tile_k, 16 * (2 * half + u) + l16, kb, grp), qf[kb], score[u]);
          const f32x4 gam = u == t ? own[ti] : w.decays_by_rows(rows, ti, 2 * half + u);
#pragma unroll
          for (int r = 0; r < 4; ++r) score[u][r] = u < t || l16 >= 4 * grp + r ? score[u][r] * (p.scale * gam[r]) : 0.f;
        }
        bf16x8 pf, pl;
        split(score[0], score[1], pf, pl);
        f32x4 out[kNT];
#pragma unroll
        for (int n = 0; n < kNT; ++n) out[n] = zero4();
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int n = 0; n < kNT; ++n) out[n] = mfma16(sm[kb][n], qf[kb], mfma16(sh[kb][n], qf[kb], out[n]));
        const float grown = rows[kSoloGrown + 16 * ti + l16] * p.scale;
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
#pragma unroll
          for (int r = 0; r < 4; ++r) out[n][r] *= grown;
          out[n] = mfma16(xh[n], pl, mfma16(xl[n], pf, mfma16(xh[n], pf, out[n])));
          write4(to, o_off[n] + ti * o_pitch, round4(out[n]));
        }
      }
      // S' = e^G_last S + K^T (beta e^(G_last - G) N)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const f32x4 keep = *reinterpret_cast<const f32x4*>(rows + kSoloKeep + 32 * half + 16 * t + 4 * grp);
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) x[t][n][r] *= keep[r];
      }
      bf16x8 xm[kNT];
#pragma unroll
      for (int n = 0; n < kNT; ++n) split3(x[0][n], x[1][n], xh[n], xm[n], xl[n]);
      const float total = rows[kSoloTotal + half];
#pragma unroll
      for (int a = 0; a < KA; ++a) {
        const bf16x8 kt = TK::keys_frag(tile_k, half, a, l16, grp);
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
#pragma unroll
          for (int r = 0; r < 4; ++r) s[a][n][r] *= total;
          s[a][n] = mfma16(kt, xl[n], mfma16(kt, xm[n], mfma16(kt, xh[n], s[a][n])));
        }
      }
    }
  }

  if (p.state_out != nullptr) {
#pragma unroll
    for (int a = 0; a < KA; ++a)
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = state_row(a, 4 * grp + r);
          if (row < p.dk && col0 + 16 * n + l16 < p.dv) p.state_out[(w.unit * p.dk + row) * p.dv + col0 + 16 * n + l16] = s[a][n][r];
        }
  }
  const bf16x8 none = zero8();
  for (int64_t i = lane; i < static_cast<int64_t>(p.T - w.len) * 4; i += kWave) {
    const int at = static_cast<int>(i % 4) * 8;
    if (col0 + at < p.dv) *reinterpret_cast<bf16x8*>(o0 + (w.len + i / 4) * p.os[2] + at) = none;
  }
}

// The gradient of the state, tokens last to first (the formulas: delta.h).
template <int DK>
__global__ __launch_bounds__(kWave, DK == 32 ? 2 : 1) void delta_solo_back_kernel(const DeltaParams p) {
  typedef Solo<DK, true> W;
  typedef SoloLds<DK> L;
  typedef Tile<DK> TK;
  typedef Tile<kSoloCols> TV;
  constexpr int KB = W::KB, KA = W::KA;
  __shared__ __attribute__((aligned(64))) uint8_t smem[L::kTotal];
  __shared__ __attribute__((aligned(16))) float rows[kSoloFloats];
  bf16_t* tile_k = reinterpret_cast<bf16_t*>(smem);
  bf16_t* tile_q = reinterpret_cast<bf16_t*>(smem + L::kTileQ);
  bf16_t* tile_o = reinterpret_cast<bf16_t*>(smem + L::kTileV);
  float* scratch = reinterpret_cast<float*>(smem + L::kTileQ);
  W w(p);
  const int lane = w.lane, l16 = w.l16, grp = w.grp, col0 = w.col0;
  bf16_t* v0 = p.grad_v + w.b * p.dvs[0] + w.h * p.dvs[1] + col0;
  const uint32_t v_pitch = static_cast<uint32_t>(p.dvs[2]) * 32;
  uint32_t v_off[kNT];
  w.quads(p.dvs[2], v_off);

  f32x4 s[KA][kNT];
#pragma unroll
  for (int a = 0; a < KA; ++a)
#pragma unroll
    for (int n = 0; n < kNT; ++n) s[a][n] = zero4();

  SoloTokens<DK> c;
  if (w.groups > 0) w.fetch(c);
  for (int group = w.groups - 1; group >= 0; --group) {
    const int64_t token0 = static_cast<int64_t>(group) * kChunk;
    const int n_tok = w.tokens_of(group);
    const Buffer to = rows_buffer(v0 + token0 * p.dvs[2], p.dvs[2], n_tok, p.dv - col0);
    wave_sync();
    w.place(c, n_tok, rows, tile_k, tile_o);
    f32x4 diag[4], below[2], own[4];
    w.solve(c, rows, scratch, diag, below, own);
    w.place_queries(c, tile_q);
    w.fetch(c);
#pragma unroll
    for (int back = 0; back < 2; ++back) {
      const int half = 1 - back;
      if (half == 1 && n_tok <= kHalf) continue;
      bf16x8 sh[KB][kNT], sl[KB][kNT], of[kNT];
      w.split_state(s, sh, sl);
      if (half == 1 || n_tok <= kHalf) w.store_state(p.grad_states + (w.unit * p.chunks + group) * static_cast<int64_t>(p.dk) * p.dv, sh);
#pragma unroll
      for (int n = 0; n < kNT; ++n) of[n] = TV::values_frag(tile_o, half, n, l16, grp);
      // beta dU
      f32x4 z[2][kNT];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int tj = 2 * half + t;
        bf16x8 kf[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) kf[kb] = TK::row(tile_k, 16 * tj + l16, kb, grp);
        f32x4 score[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          score[u] = zero4();
          if (u < t) continue;
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) score[u] = mfma16(TK::row(tile_q, 16 * (2 * half + u) + l16, kb, grp), kf[kb], score[u]);
          const f32x4 gam = w.decays_by_cols(rows, 2 * half + u, tj);
#pragma unroll
          for (int r = 0; r < 4; ++r) score[u][r] *= p.scale * gam[r];
        }
        bf16x8 pf, pl;
        split(score[0], score[1], pf, pl);
#pragma unroll
        for (int n = 0; n < kNT; ++n) z[t][n] = zero4();
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int n = 0; n < kNT; ++n) z[t][n] = mfma16(kf[kb], sl[kb][n], mfma16(kf[kb], sh[kb][n], z[t][n]));
        const f32x4 keep = *reinterpret_cast<const f32x4*>(rows + kSoloKeep + 16 * tj + 4 * grp);
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
#pragma unroll
          for (int r = 0; r < 4; ++r) z[t][n][r] *= keep[r];
          z[t][n] = mfma16(pl, of[n], mfma16(pf, of[n], z[t][n]));
        }
      }
      // dX
      w.apply(diag, below, half, z);
      bf16x8 zh[kNT], zl[kNT];
#pragma unroll
      for (int n = 0; n < kNT; ++n) zh[n] = round8(z[0][n], z[1][n]);
      w.store_rows(to, v_pitch, v_off, 2 * half, tile_o + 32 * half * TV::STRIDE, zh);
      // dS
      bf16x8 wh[kNT], wl[kNT];
      const f32x4 g0 = *reinterpret_cast<const f32x4*>(rows + kSoloGrown + 32 * half + 4 * grp);
      const f32x4 g1 = *reinterpret_cast<const f32x4*>(rows + kSoloGrown + 32 * half + 16 + 4 * grp);
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        f32x4 a0, a1;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          a0[r] = -g0[r] * z[0][n][r];
          a1[r] = -g1[r] * z[1][n][r];
        }
        split(a0, a1, zh[n], zl[n]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          a0[r] = p.scale * g0[r] * static_cast<float>(of[n][r]);
          a1[r] = p.scale * g1[r] * static_cast<float>(of[n][4 + r]);
        }
        split(a0, a1, wh[n], wl[n]);
      }
      const float total = rows[kSoloTotal + half];
#pragma unroll
      for (int a = 0; a < KA; ++a) {
        const bf16x8 kt = TK::keys_frag(tile_k, half, a, l16, grp), qt = TK::keys_frag(tile_q, half, a, l16, grp);
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
#pragma unroll
          for (int r = 0; r < 4; ++r) s[a][n][r] *= total;
          s[a][n] = mfma16(kt, zl[n], mfma16(kt, zh[n], s[a][n]));
          s[a][n] = mfma16(qt, wl[n], mfma16(qt, wh[n], s[a][n]));
        }
      }
    }
  }
  const bf16x8 none = zero8();
  for (int64_t i = lane; i < static_cast<int64_t>(p.T - w.len) * 4; i += kWave) {
    const int at = static_cast<int>(i % 4) * 8;
    if (col0 + at < p.dv) *reinterpret_cast<bf16x8*>(v0 + (w.len + i / 4) * p.dvs[2] + at) = none;
  }
}

template <int DK>
int launch_solo(const char* name, const DeltaParams& p, bool back, hipStream_t s) {
  const int64_t waves = static_cast<int64_t>(p.B) * p.H * ((p.dv + kSoloCols - 1) / kSoloCols);
  if (waves > 0x7fffffffLL) return set_error(TAAC_ERR_UNSUPPORTED, "%s: too many workgroups", name);
  const dim3 grid(static_cast<uint32_t>(waves)), threads(kWave);
  if (back) hipLaunchKernelGGL((delta_solo_back_kernel<DK>), grid, threads, 0, s, p);
  else if (p.chunk_states != nullptr) hipLaunchKernelGGL((delta_solo_kernel<DK, true>), grid, threads, 0, s, p);
  else hipLaunchKernelGGL((delta_solo_kernel<DK, false>), grid, threads, 0, s, p);
  return check_launch(name);
}

}  // namespace

int delta_solo(const char* name, const DeltaParams& p, bool back, hipStream_t s) {
  return p.dk <= 32 ? launch_solo<32>(name, p, back, s) : launch_solo<64>(name, p, back, s);
}

}  // namespace taac
