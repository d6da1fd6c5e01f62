// Gated delta rule, chunked form, backward (notation, operand order and precision: delta.h).
//
// With dS' the gradient of the state behind a chunk, X, N as in the forward and T the chunk's 64 tokens:
//   beta dU = diag(beta e^{G_64 - G}) K dS' + P^T dO          (P holds scale, Gam and beta of its column)
//   dX = beta dU - M^T (beta dU) = dV
//   dS = e^{G_64} dS' + Q^T (scale e^G dO) - K^T (e^G dX)
// is a recurrence like the forward's, backwards, column by column of the values: the first kernel, which keeps dS' of every chunk and dX.
// The rest needs all value columns of a chunk but nothing of another chunk: the second kernel, in parallel over the chunks. With
//   B_ij = scale Gam_ij dO_i . N_j (i >= j),   E_ij = -Gam_ij dX_i . N_j (i > j)
//   dQ = scale e^G dO S^T + B diag(beta) K
//   R  = E diag(beta) K - e^G dX S^T
//   C  = B^T Q + E^T K + diag(e^{G_64 - G}) N dS'^T
//   dK = R + diag(beta) C,   dbeta_j = k_j . C_j
//   dG_i = q_i . dQ_i + k_i . R_i - beta_i dbeta_i, and e^{G_64} <S, dS'> + sum_j beta_j e^{G_64 - G_j} k_j . (N dS'^T)_j for G_64
//   dg_t = the sum of dG over t .. 64
// where what a pair (i, j) of tokens adds to a row it takes from a column.
// N, S, dS' and dX are read back in bf16, one rounding each: they only meet the outputs. Key heads that serve several value heads sum
// their gradients in registers, in the order of the heads.
#include "delta.h"

namespace taac {
namespace {

// ---- the state's gradient, chunks last to first -------------------------------------------------------------------
template <int DK, int NT, int NW>
struct BackLds {
  static constexpr int COLS = 16 * NT * NW;
  static constexpr int VCOLS = COLS < 32 ? 32 : COLS;
  static constexpr int kTileK = NW * kBlockBytes;
  static constexpr int kTileQ = kTileK + Tile<DK>::BYTES;
  static constexpr int kTileO = kTileQ + Tile<DK>::BYTES;
  static constexpr int kTotal = kTileO + Tile<VCOLS>::BYTES;
};

template <int DK, int NT, int NW>
__global__ __launch_bounds__(NW * kWave) void delta_back_kernel(const DeltaParams p) {
  constexpr int KB = DK / 32, KA = DK / 16;
  typedef BackLds<DK, NT, NW> L;
  typedef Tile<DK> TK;
  typedef Tile<L::VCOLS> TV;
  extern __shared__ __attribute__((aligned(64))) uint8_t smem[];
  bf16_t* tile_k = reinterpret_cast<bf16_t*>(smem + L::kTileK);
  bf16_t* tile_q = reinterpret_cast<bf16_t*>(smem + L::kTileQ);
  bf16_t* tile_o = reinterpret_cast<bf16_t*>(smem + L::kTileO);

  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, l16 = lane % 16, grp = lane / 16;
  const int col_groups = (p.dv + L::COLS - 1) / L::COLS;
  const int64_t unit = blockIdx.x / col_groups;
  const int col0 = static_cast<int>(blockIdx.x % col_groups) * L::COLS;
  const int h = static_cast<int>(unit % p.H);
  const int b = static_cast<int>(unit / p.H);
  int len = p.T;
  if (p.lengths != nullptr) {
    len = p.lengths[b];
    len = len < 0 ? 0 : (len > p.T ? p.T : len);
  }
  const int chunks = (len + kChunk - 1) / kChunk;
  const int64_t hk = h / p.group;
  const bf16_t* kb0 = p.k + b * p.ks[0] + hk * p.ks[1];
  const bf16_t* qb0 = p.q + b * p.qs[0] + hk * p.qs[1];
  const bf16_t* db0 = p.grad_o + b * p.dos[0] + h * p.dos[1] + col0;
  bf16_t* vb0 = p.grad_v + b * p.dvs[0] + h * p.dvs[1];

  int col[NT];
  bool col_ok[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    col[n] = col0 + (wave * NT + n) * 16;
    col_ok[n] = col[n] + l16 < p.dv;
  }
  f32x4 s[KA][NT];
#pragma unroll
  for (int a = 0; a < KA; ++a)
#pragma unroll
    for (int n = 0; n < NT; ++n) s[a][n] = zero4();

  for (int end = chunks; end > 0; end -= NW) {
    __syncthreads();
    if (end - 1 - wave >= 0) {  // slot w of the round: chunk end - 1 - w
      uint8_t* block = smem + wave * kBlockBytes;
      const int64_t token0 = static_cast<int64_t>(end - 1 - wave) * kChunk;
      const int left = len - static_cast<int>(token0);
      chunk_block<DK, true>(p, b, h, token0, left < kChunk ? left : kChunk, block, reinterpret_cast<float*>(block + kBlockRows),
                            reinterpret_cast<float*>(block));
    }
    const int here = end < NW ? end : NW;
    for (int c = 0; c < here; ++c) {
      const int chunk = end - 1 - c;
      const int64_t token0 = static_cast<int64_t>(chunk) * kChunk;
      const int left = len - static_cast<int>(token0);
      const int n_tok = left < kChunk ? left : kChunk;
      if (c > 0) __syncthreads();
      TK::stage(tile_k, kb0 + token0 * p.ks[2], p.ks[2], n_tok, p.dk, tid, NW * kWave);
      TK::stage(tile_q, qb0 + token0 * p.qs[2], p.qs[2], n_tok, p.dk, tid, NW * kWave);
      TV::stage(tile_o, db0 + token0 * p.dos[2], p.dos[2], n_tok, p.dv - col0, tid, NW * kWave);
      __syncthreads();
      const uint8_t* block = smem + c * kBlockBytes;
      const float* rows = reinterpret_cast<const float*>(block + kBlockRows);

      bf16_t* dst = p.grad_states + (unit * p.chunks + chunk) * static_cast<int64_t>(p.dk) * p.dv;
#pragma unroll
      for (int a = 0; a < KA; ++a)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = state_row(a, 4 * grp + r);
            if (col_ok[n] && row < p.dk) dst[row * p.dv + col[n] + l16] = static_cast<bf16_t>(s[a][n][r]);
          }
      bf16x8 sh[KB][NT], sl[KB][NT];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int n = 0; n < NT; ++n) split(s[2 * kb][n], s[2 * kb + 1][n], sh[kb][n], sl[kb][n]);

      // beta dU
      bf16x8 of[2][NT];
#pragma unroll
      for (int tk = 0; tk < 2; ++tk)
#pragma unroll
        for (int n = 0; n < NT; ++n) of[tk][n] = TV::values_frag(tile_o, tk, wave * NT + n, l16, grp);
      f32x4 z[4][NT];
#pragma unroll
      for (int tj = 0; tj < 4; ++tj) {
#pragma unroll
        for (int n = 0; n < NT; ++n) z[tj][n] = zero4();
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const bf16x8 kf = TK::row(tile_k, 16 * tj + l16, kb, grp);
#pragma unroll
          for (int n = 0; n < NT; ++n) z[tj][n] = mfma16(kf, sl[kb][n], mfma16(kf, sh[kb][n], z[tj][n]));
        }
        const f32x4 keep = *reinterpret_cast<const f32x4*>(rows + kRowKeep + 16 * tj + 4 * grp);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) z[tj][n][r] *= keep[r];
#pragma unroll
        for (int tk = tj / 2; tk < 2; ++tk) {
          const bf16x8 pf = *reinterpret_cast<const bf16x8*>(block + kBlockP + frag_cols(tj, tk) * kFrag + lane * 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) z[tj][n] = mfma16(pf, of[tk][n], z[tj][n]);
        }
      }
      // dX
      bf16x8 zh[2][NT], zl[2][NT];
#pragma unroll
      for (int tk = 0; tk < 2; ++tk)
#pragma unroll
        for (int n = 0; n < NT; ++n) split(z[2 * tk][n], z[2 * tk + 1][n], zh[tk][n], zl[tk][n]);
#pragma unroll
      for (int tj = 0; tj < 4; ++tj)
#pragma unroll
        for (int tk = tj / 2; tk < 2; ++tk) {
          const bf16x8 mh = *reinterpret_cast<const bf16x8*>(block + kBlockM + frag_cols(tj, tk) * kFrag + lane * 16);
          const bf16x8 ml = *reinterpret_cast<const bf16x8*>(block + kBlockLow + frag_cols(tj, tk) * kFrag + lane * 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) z[tj][n] = mfma16(ml, zh[tk][n], mfma16(mh, zl[tk][n], mfma16(mh, zh[tk][n], z[tj][n])));
        }
#pragma unroll
      for (int tj = 0; tj < 4; ++tj)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = 16 * tj + 4 * grp + r;
            if (col_ok[n] && row < n_tok) vb0[(token0 + row) * p.dvs[2] + col[n] + l16] = static_cast<bf16_t>(z[tj][n][r]);
          }
      // dS
      bf16x8 wh[2][NT], wl[2][NT];
#pragma unroll
      for (int tk = 0; tk < 2; ++tk) {
        const f32x4 g0 = *reinterpret_cast<const f32x4*>(rows + kRowGrown + 32 * tk + 4 * grp);
        const f32x4 g1 = *reinterpret_cast<const f32x4*>(rows + kRowGrown + 32 * tk + 16 + 4 * grp);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          f32x4 a, c2;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            a[r] = -g0[r] * z[2 * tk][n][r];
            c2[r] = -g1[r] * z[2 * tk + 1][n][r];
          }
          split(a, c2, zh[tk][n], zl[tk][n]);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            a[r] = p.scale * g0[r] * static_cast<float>(of[tk][n][r]);
            c2[r] = p.scale * g1[r] * static_cast<float>(of[tk][n][4 + r]);
          }
          split(a, c2, wh[tk][n], wl[tk][n]);
        }
      }
      const float total = rows[kRowTotal];
#pragma unroll
      for (int a = 0; a < KA; ++a) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[a][n][r] *= total;
#pragma unroll
        for (int tk = 0; tk < 2; ++tk) {
          const bf16x8 kt = TK::keys_frag(tile_k, tk, a, l16, grp);
          const bf16x8 qt = TK::keys_frag(tile_q, tk, a, l16, grp);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            s[a][n] = mfma16(kt, zl[tk][n], mfma16(kt, zh[tk][n], s[a][n]));
            s[a][n] = mfma16(qt, wl[tk][n], mfma16(qt, wh[tk][n], s[a][n]));
          }
        }
      }
    }
  }
  // padded rows have no gradient
  constexpr int QUADS = L::COLS / 4;
  const bf16x4 none = {};
  for (int64_t i = tid; i < static_cast<int64_t>(p.T - len) * QUADS; i += NW * kWave) {
    const int64_t row = len + i / QUADS;
    const int at = col0 + static_cast<int>(i % QUADS) * 4;
    if (at < p.dv) *reinterpret_cast<bf16x4*>(vb0 + row * p.dvs[2] + at) = none;
  }
}

// ---- gradients of a chunk -----------------------------------------------------------------------------------------
// Four wavefronts; wavefront w owns tokens 16 w .. 16 w + 15 of the chunk, a lane one of them (four key features at a time).
template <int DK, int DV>
struct GradLds {
  static constexpr int kTileK = 0;
  static constexpr int kTileQ = kTileK + Tile<DK>::BYTES;
  static constexpr int kTileO = kTileQ + Tile<DK>::BYTES;
  static constexpr int kTileX = kTileO + Tile<DV>::BYTES;
  static constexpr int kTileN = kTileX + Tile<DV>::BYTES;
  static constexpr int kRows = kTileN + Tile<DV>::BYTES;
  static constexpr int kTotal = kRows + (336 + 64 + 3 * 64 + 16) * 4;
};

__device__ __forceinline__ float group_total(float v) {  // over the four lanes of a token
  v += __shfl_xor(v, 16, kWave);
  return v + __shfl_xor(v, 32, kWave);
}

__device__ __forceinline__ void store_gate(void* p, int64_t at, float v, int f32) {
  if (f32) static_cast<float*>(p)[at] = v;
  else static_cast<bf16_t*>(p)[at] = static_cast<bf16_t>(v);
}

template <int DK, int DV>
__global__ __launch_bounds__(4 * kWave) void delta_grads_kernel(const DeltaParams p) {
  constexpr int KA = DK / 16, VB = DV / 32;
  typedef GradLds<DK, DV> L;
  typedef Tile<DK> TK;
  typedef Tile<DV> TV;
  extern __shared__ __attribute__((aligned(64))) uint8_t smem[];
  bf16_t* tile_k = reinterpret_cast<bf16_t*>(smem + L::kTileK);
  bf16_t* tile_q = reinterpret_cast<bf16_t*>(smem + L::kTileQ);
  bf16_t* tile_o = reinterpret_cast<bf16_t*>(smem + L::kTileO);
  bf16_t* tile_x = reinterpret_cast<bf16_t*>(smem + L::kTileX);
  bf16_t* tile_n = reinterpret_cast<bf16_t*>(smem + L::kTileN);
  float* rows = reinterpret_cast<float*>(smem + L::kRows);
  float* left_over = rows + 336;   // e^(G_last - G)
  float* d_total = left_over + 64; // dG of a token
  float* d_beta = d_total + 64;
  float* d_tail = d_beta + 64;     // its share of dG_64
  float* state_dot = d_tail + 64;  // per wavefront

  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, l16 = lane % 16, grp = lane / 16;
  const int key_heads = p.H / p.group;
  const int chunk = static_cast<int>(blockIdx.x % p.chunks);
  const int64_t pair = blockIdx.x / p.chunks;
  const int hk = static_cast<int>(pair % key_heads);
  const int b = static_cast<int>(pair / key_heads);
  int len = p.T;
  if (p.lengths != nullptr) {
    len = p.lengths[b];
    len = len < 0 ? 0 : (len > p.T ? p.T : len);
  }
  const int64_t token0 = static_cast<int64_t>(chunk) * kChunk;
  const int span = p.T - static_cast<int>(token0) < kChunk ? p.T - static_cast<int>(token0) : kChunk;  // rows of the tensors
  int n_tok = len - static_cast<int>(token0);
  n_tok = n_tok < 0 ? 0 : (n_tok > kChunk ? kChunk : n_tok);

  const int row = 16 * wave + l16;  // this lane's token
  f32x4 dq_sum[KA], dk_sum[KA];
#pragma unroll
  for (int a = 0; a < KA; ++a) dq_sum[a] = dk_sum[a] = zero4();

  if (n_tok > 0) {
    TK::stage(tile_k, p.k + b * p.ks[0] + hk * p.ks[1] + token0 * p.ks[2], p.ks[2], n_tok, p.dk, tid, 4 * kWave);
    TK::stage(tile_q, p.q + b * p.qs[0] + hk * p.qs[1] + token0 * p.qs[2], p.qs[2], n_tok, p.dk, tid, 4 * kWave);
  }
  for (int h = hk * p.group; h < (hk + 1) * p.group; ++h) {
    if (n_tok == 0) {
      for (int i = tid; i < span; i += 4 * kWave) {
        store_gate(p.grad_decay, b * p.dgs[0] + h * p.dgs[1] + (token0 + i) * p.dgs[2], 0.f, p.gates_f32);
        store_gate(p.grad_beta, b * p.dbs[0] + h * p.dbs[1] + (token0 + i) * p.dbs[2], 0.f, p.gates_f32);
      }
      continue;
    }
    const int64_t unit = static_cast<int64_t>(b) * p.H + h;
    __syncthreads();  // the previous head's tiles and sums are no longer read
    TV::stage(tile_o, p.grad_o + b * p.dos[0] + h * p.dos[1] + token0 * p.dos[2], p.dos[2], n_tok, p.dv, tid, 4 * kWave);
    TV::stage(tile_x, p.grad_v + b * p.dvs[0] + h * p.dvs[1] + token0 * p.dvs[2], p.dvs[2], n_tok, p.dv, tid, 4 * kWave);
    TV::stage(tile_n, p.misses + (unit * p.T + token0) * p.dv, p.dv, n_tok, p.dv, tid, 4 * kWave);
    if (wave == 0) chunk_rows(p, b, h, token0, n_tok, rows, left_over);
    __syncthreads();
    const bf16_t* state = p.chunk_states + (unit * p.chunks + chunk) * static_cast<int64_t>(p.dk) * p.dv;
    const bf16_t* grad_state = p.grad_states + (unit * p.chunks + chunk) * static_cast<int64_t>(p.dk) * p.dv;

    bf16x8 o_f[VB], x_f[VB], n_f[VB];
#pragma unroll
    for (int vb = 0; vb < VB; ++vb) {
      o_f[vb] = TV::row(tile_o, row, vb, grp);
      x_f[vb] = TV::row(tile_x, row, vb, grp);
      n_f[vb] = TV::row(tile_n, row, vb, grp);
    }
    const float hi_t = rows[kRowHi + row], lo_t = rows[kRowLow + row], beta_t = rows[kRowBeta + row], grown = rows[kRowGrown + row];
    // This wavefront's tokens as i, then as j. The sums of the pairs' contributions to dG over a row and over a column are taken here, from
    // the same fp32 values: pairs on one side of a token then cancel in dg as they do in the formula.
    bf16x8 k_f[KA / 2], q_f[KA / 2];
#pragma unroll
    for (int kb = 0; kb < KA / 2; ++kb) {
      k_f[kb] = TK::row(tile_k, row, kb, grp);
      q_f[kb] = TK::row(tile_q, row, kb, grp);
    }
    float dot_row = 0.f, dot_col = 0.f;
    f32x4 bi[4], ei[4], bj[4], ej[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      bi[t] = ei[t] = bj[t] = ej[t] = zero4();
      const f32x4 hi_r = *reinterpret_cast<const f32x4*>(rows + kRowHi + 16 * t + 4 * grp);
      const f32x4 lo_r = *reinterpret_cast<const f32x4*>(rows + kRowLow + 16 * t + 4 * grp);
      if (t <= wave) {
        const f32x4 beta_r = *reinterpret_cast<const f32x4*>(rows + kRowBeta + 16 * t + 4 * grp);
        f32x4 qk = zero4(), kk = zero4();
#pragma unroll
        for (int vb = 0; vb < VB; ++vb) {
          const bf16x8 nf = TV::row(tile_n, 16 * t + l16, vb, grp);
          bi[t] = mfma16(nf, o_f[vb], bi[t]);
          ei[t] = mfma16(nf, x_f[vb], ei[t]);
        }
#pragma unroll
        for (int kb = 0; kb < KA / 2; ++kb) {
          const bf16x8 kf = TK::row(tile_k, 16 * t + l16, kb, grp);
          qk = mfma16(kf, q_f[kb], qk);
          kk = mfma16(kf, k_f[kb], kk);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = 16 * t + 4 * grp + r;
          const float gam = __builtin_amdgcn_exp2f((hi_t - hi_r[r]) + (lo_t - lo_r[r]));
          bi[t][r] = row >= j ? p.scale * gam * bi[t][r] : 0.f;
          ei[t][r] = row > j ? -gam * ei[t][r] : 0.f;
          dot_row = fmaf(beta_r[r], fmaf(bi[t][r], qk[r], ei[t][r] * kk[r]), dot_row);
          bi[t][r] *= beta_r[r];
          ei[t][r] *= beta_r[r];
        }
      }
      if (t >= wave) {
        f32x4 qk = zero4(), kk = zero4();
#pragma unroll
        for (int vb = 0; vb < VB; ++vb) {
          bj[t] = mfma16(TV::row(tile_o, 16 * t + l16, vb, grp), n_f[vb], bj[t]);
          ej[t] = mfma16(TV::row(tile_x, 16 * t + l16, vb, grp), n_f[vb], ej[t]);
        }
#pragma unroll
        for (int kb = 0; kb < KA / 2; ++kb) {
          qk = mfma16(TK::row(tile_q, 16 * t + l16, kb, grp), k_f[kb], qk);
          kk = mfma16(TK::row(tile_k, 16 * t + l16, kb, grp), k_f[kb], kk);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * t + 4 * grp + r;
          const float gam = __builtin_amdgcn_exp2f((hi_r[r] - hi_t) + (lo_r[r] - lo_t));
          bj[t][r] = i >= row ? p.scale * gam * bj[t][r] : 0.f;
          ej[t][r] = i > row ? -gam * ej[t][r] : 0.f;
          dot_col += fmaf(bj[t][r], qk[r], ej[t][r] * kk[r]);
        }
      }
    }
    bf16x8 bif[2], eif[2], bjf[2], ejf[2], bil[2], eil[2], bjl[2], ejl[2];
#pragma unroll
    for (int tk = 0; tk < 2; ++tk) {
      split(bi[2 * tk], bi[2 * tk + 1], bif[tk], bil[tk]);
      split(ei[2 * tk], ei[2 * tk + 1], eif[tk], eil[tk]);
      split(bj[2 * tk], bj[2 * tk + 1], bjf[tk], bjl[tk]);
      split(ej[2 * tk], ej[2 * tk + 1], ejf[tk], ejl[tk]);
    }
    float dot_tail = 0.f, dot_state = 0.f;
    const float tail = left_over[row];
#pragma unroll
    for (int a = 0; a < KA; ++a) {
      f32x4 dq = zero4(), dr = zero4(), dc = zero4();
      const int feature = state_row(a, l16);
#pragma unroll
      for (int vb = 0; vb < VB; ++vb) {
        const bf16x8 sf = row_frag(feature < p.dk ? state + feature * p.dv : nullptr, vb, grp, p.dv);
        const bf16x8 gf = row_frag(feature < p.dk ? grad_state + feature * p.dv : nullptr, vb, grp, p.dv);
        dq = mfma16(sf, o_f[vb], dq);
        dr = mfma16(sf, x_f[vb], dr);
        dc = mfma16(gf, n_f[vb], dc);
        if (a % 4 == wave) {
#pragma unroll
          for (int e = 0; e < 8; ++e) dot_state = fmaf(static_cast<float>(sf[e]), static_cast<float>(gf[e]), dot_state);
        }
      }
      const int at = row * TK::STRIDE + (a / 2) * 32 + grp * 8 + (a % 2) * 4;
      const bf16x4 kv = *reinterpret_cast<const bf16x4*>(tile_k + at);
      const bf16x4 qv = *reinterpret_cast<const bf16x4*>(tile_q + at);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        dq[r] *= p.scale * grown;
        dr[r] *= -grown;
        dc[r] *= tail;
        dot_row = fmaf(static_cast<float>(qv[r]), dq[r], fmaf(static_cast<float>(kv[r]), dr[r], dot_row));
        dot_tail = fmaf(static_cast<float>(kv[r]), dc[r], dot_tail);
      }
#pragma unroll
      for (int tk = 0; tk < 2; ++tk) {
        const bf16x8 kt = TK::keys_frag(tile_k, tk, a, l16, grp);
        const bf16x8 qt = TK::keys_frag(tile_q, tk, a, l16, grp);
        dq = mfma16(kt, bil[tk], mfma16(kt, bif[tk], dq));
        dr = mfma16(kt, eil[tk], mfma16(kt, eif[tk], dr));
        dc = mfma16(qt, bjl[tk], mfma16(qt, bjf[tk], dc));
        dc = mfma16(kt, ejl[tk], mfma16(kt, ejf[tk], dc));
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        dq_sum[a][r] += dq[r];
        dk_sum[a][r] += dr[r] + beta_t * dc[r];
      }
    }
    dot_row = group_total(dot_row);
    dot_col = group_total(dot_col);
    dot_tail = group_total(dot_tail);
    dot_state = group_sum<kWave>(dot_state);
    if (grp == 0) {
      d_total[row] = dot_row - beta_t * dot_col;
      d_beta[row] = dot_col + dot_tail;
      d_tail[row] = beta_t * dot_tail;
    }
    if (lane == 0) state_dot[wave] = dot_state;
    __syncthreads();
    if (wave == 0) {
      // the tokens' sums from t on; the tails in front of t, which are what is left of G_64's share
      float sum = d_total[lane], tails = d_tail[lane];
#pragma unroll
      for (int off = 1; off < kWave; off *= 2) {
        const float down = __shfl_down(sum, off, kWave), up = __shfl_up(tails, off, kWave);
        if (lane + off < kWave) sum += down;
        if (lane >= off) tails += up;
      }
      tails = __shfl_up(tails, 1, kWave);
      const float whole = fmaf(rows[kRowTotal], (state_dot[0] + state_dot[1]) + (state_dot[2] + state_dot[3]), lane > 0 ? tails : 0.f);
      if (lane < span) {
        const bool live = lane < n_tok;
        store_gate(p.grad_decay, b * p.dgs[0] + h * p.dgs[1] + (token0 + lane) * p.dgs[2], live ? sum + whole : 0.f, p.gates_f32);
        store_gate(p.grad_beta, b * p.dbs[0] + h * p.dbs[1] + (token0 + lane) * p.dbs[2], live ? d_beta[lane] : 0.f, p.gates_f32);
      }
    }
  }
  if (row < span) {  // rows behind the last token hold zeros
    bf16_t* dq_row = p.grad_q + b * p.dqs[0] + hk * p.dqs[1] + (token0 + row) * p.dqs[2];
    bf16_t* dk_row = p.grad_k + b * p.dks[0] + hk * p.dks[1] + (token0 + row) * p.dks[2];
#pragma unroll
    for (int a = 0; a < KA; ++a) {
      const int at = state_row(a, 4 * grp);
      if (at >= p.dk) continue;
      bf16x4 dq, dk;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        dq[r] = static_cast<bf16_t>(dq_sum[a][r]);
        dk[r] = static_cast<bf16_t>(dk_sum[a][r]);
      }
      *reinterpret_cast<bf16x4*>(dq_row + at) = dq;
      *reinterpret_cast<bf16x4*>(dk_row + at) = dk;
    }
  }
}

template <int DK, int NT, int NW>
int launch_back(const char* name, const DeltaParams& p, hipStream_t s) {
  typedef BackLds<DK, NT, NW> L;
  const int64_t grid = static_cast<int64_t>(p.B) * p.H * ((p.dv + L::COLS - 1) / L::COLS);
  if (grid > 0x7fffffffLL) return set_error(TAAC_ERR_UNSUPPORTED, "%s: too many workgroups", name);
  const void* kernel = reinterpret_cast<const void*>(delta_back_kernel<DK, NT, NW>);
  if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, L::kTotal) != hipSuccess)
    return set_error(TAAC_ERR_LAUNCH, "%s: cannot reserve %d bytes of LDS", name, L::kTotal);
  hipLaunchKernelGGL((delta_back_kernel<DK, NT, NW>), dim3(static_cast<uint32_t>(grid)), dim3(NW * kWave), L::kTotal, s, p);
  return check_launch(name);
}

template <int DK, int DV>
int launch_grads(const char* name, const DeltaParams& p, hipStream_t s) {
  typedef GradLds<DK, DV> L;
  const int64_t grid = static_cast<int64_t>(p.B) * (p.H / p.group) * p.chunks;
  if (grid > 0x7fffffffLL) return set_error(TAAC_ERR_UNSUPPORTED, "%s: too many workgroups", name);
  const void* kernel = reinterpret_cast<const void*>(delta_grads_kernel<DK, DV>);
  if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, L::kTotal) != hipSuccess)
    return set_error(TAAC_ERR_LAUNCH, "%s: cannot reserve %d bytes of LDS", name, L::kTotal);
  hipLaunchKernelGGL((delta_grads_kernel<DK, DV>), dim3(static_cast<uint32_t>(grid)), dim3(4 * kWave), L::kTotal, s, p);
  return check_launch(name);
}

template <int DK>
int dispatch_back(const char* name, const DeltaParams& p, hipStream_t s) {
  int rc;
  if (p.blocks != nullptr) rc = delta_team_back(name, p, s);
  else if (p.dv <= 32) rc = launch_back<DK, 2, 1>(name, p, s);
  else if (p.dv <= 64) rc = launch_back<DK, 2, 2>(name, p, s);
  else rc = launch_back<DK, 2, 4>(name, p, s);
  if (rc != TAAC_OK) return rc;
  if (p.dv <= 32) return launch_grads<DK, 32>(name, p, s);
  if (p.dv <= 64) return launch_grads<DK, 64>(name, p, s);
  return launch_grads<DK, 128>(name, p, s);
}

}  // namespace
}  // namespace taac

extern "C" int taac_delta_rule_bwd(const void* q, const void* k, const void* log_decay, const void* beta, const int32_t* lengths,
                                   const void* chunk_states, const void* misses, const void* grad_o, void* grad_q, void* grad_k,
                                   void* grad_v, void* grad_decay, void* grad_beta, void* grad_states, void* workspace,
                                   int64_t workspace_bytes, int32_t B, int32_t H,
                                   int32_t key_heads, int32_t T, int32_t dk, int32_t dv, const int64_t q_strides[3],
                                   const int64_t k_strides[3], const int64_t decay_strides[3], const int64_t beta_strides[3],
                                   const int64_t go_strides[3], const int64_t gq_strides[3], const int64_t gk_strides[3],
                                   const int64_t gv_strides[3], const int64_t gdecay_strides[3], const int64_t gbeta_strides[3], float scale,
                                   int gate_dtype, void* stream) {
  using namespace taac;
  const char* name = "taac_delta_rule_bwd";
  DeltaParams p{};
  if (key_heads <= 0 || H <= 0 || H % key_heads != 0)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: value heads must be a multiple of the key heads", name);
  p.B = B, p.H = H, p.group = H / key_heads, p.T = T, p.dk = dk, p.dv = dv, p.scale = scale;
  p.chunks = (T + kChunk - 1) / kChunk;
  if (int rc = delta_check(name, p)) return rc;
  if (gate_dtype != TAAC_F32 && gate_dtype != TAAC_BF16)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: gates must be fp32 or bf16 (dtype %d)", name, gate_dtype);
  p.gates_f32 = gate_dtype == TAAC_F32;
  if (B == 0 || T == 0) return TAAC_OK;
  if (!q || !k || !log_decay || !beta || !chunk_states || !misses || !grad_o || !grad_q || !grad_k || !grad_v || !grad_decay || !grad_beta ||
      !grad_states)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: null tensor pointer", name);
  if (int rc = delta_strides(name, "q", q, q_strides, p.qs, true)) return rc;
  if (int rc = delta_strides(name, "k", k, k_strides, p.ks, true)) return rc;
  if (int rc = delta_strides(name, "log_decay", log_decay, decay_strides, p.gs, false)) return rc;
  if (int rc = delta_strides(name, "beta", beta, beta_strides, p.bs, false)) return rc;
  if (int rc = delta_strides(name, "grad_o", grad_o, go_strides, p.dos, true)) return rc;
  if (int rc = delta_strides(name, "grad_q", grad_q, gq_strides, p.dqs, true)) return rc;
  if (int rc = delta_strides(name, "grad_k", grad_k, gk_strides, p.dks, true)) return rc;
  if (int rc = delta_strides(name, "grad_v", grad_v, gv_strides, p.dvs, true)) return rc;
  if (int rc = delta_strides(name, "grad_log_decay", grad_decay, gdecay_strides, p.dgs, false)) return rc;
  if (int rc = delta_strides(name, "grad_beta", grad_beta, gbeta_strides, p.dbs, false)) return rc;
  p.q = static_cast<const bf16_t*>(q), p.k = static_cast<const bf16_t*>(k), p.log_decay = log_decay, p.beta = beta, p.lengths = lengths;
  p.chunk_states = const_cast<bf16_t*>(static_cast<const bf16_t*>(chunk_states));
  p.misses = const_cast<bf16_t*>(static_cast<const bf16_t*>(misses));
  p.grad_o = static_cast<const bf16_t*>(grad_o);
  p.grad_q = static_cast<bf16_t*>(grad_q), p.grad_k = static_cast<bf16_t*>(grad_k), p.grad_v = static_cast<bf16_t*>(grad_v);
  p.grad_decay = grad_decay, p.grad_beta = grad_beta, p.grad_states = static_cast<bf16_t*>(grad_states);
  hipStream_t s = as_stream(stream);
  if (const int64_t bytes = delta_team_bytes(static_cast<int64_t>(B) * H, T, dv)) {
    if (workspace == nullptr || workspace_bytes < bytes || !aligned16(workspace))
      return set_error(TAAC_ERR_INVALID_VALUE, "%s: workspace must hold %lld bytes, 16-byte aligned", name, (long long)bytes);
    p.blocks = static_cast<uint8_t*>(workspace);
  }
  if (dk <= 32) return dispatch_back<32>(name, p, s);
  if (dk <= 64) return dispatch_back<64>(name, p, s);
  return dispatch_back<128>(name, p, s);
}
