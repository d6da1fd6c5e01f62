// Gated delta rule, chunked form, backward: the gradients of a chunk's tokens (notation, operand order and precision, dS' and dX: delta.h),
// in parallel over the chunks. With
//   B_ij = scale Gam_ij dO_i . N_j (i >= j),   E_ij = -Gam_ij dX_i . N_j (i > j)
//   dQ = scale e^G dO S^T + B diag(beta) K
//   R  = E diag(beta) K - e^G dX S^T
//   C  = B^T Q + E^T K + diag(e^{G_64 - G}) N dS'^T
//   dK = R + diag(beta) C,   dbeta_j = k_j . C_j
//   dG_i = q_i . dQ_i + k_i . R_i - beta_i dbeta_i, and e^{G_64} <S, dS'> + sum_j beta_j e^{G_64 - G_j} k_j . (N dS'^T)_j for G_64
//   dg_t = the sum of dG over t .. 64
// where what a pair (i, j) of tokens adds to a row it takes from a column.
//
// All in one workgroup per chunk and key head: the tiles of K, Q, dO, dX, N, S and dS' meet in LDS, where each is read by rows and by columns.
// 512 samples x 4 heads of up to 512 tokens, 64 wide: 389 us in a trace, 3.4 TB/s; two workgroups to a CU by their registers, whose wavefronts wait
// for 41 % of their time and issue vector instructions for 27 %. 128 wide, where the tiles leave room for one: 20 us per chunk and head, 2.0 TB/s; two
// sets of four wavefronts on one chunk (rows and columns at once) took 3 % longer.
//
// S, dS' and dX are read back in bf16, one rounding each: they only meet the outputs, of which they are parts (0.2e-3 to 1.0e-3 of a gradient, whose
// own rounding is 1.7e-3; together 1.7e-3 to 2.2e-3, where nothing is forgotten over hundreds of tokens up to 2.5e-3 and 3.0e-3 for the decays). Two parts
// of S and dS' too would be a fifth more bytes. N, which every pair of tokens has as a factor, is kept in two parts: its one rounding alone cost 1.7e-3. Key heads that serve several value heads sum their gradients in registers, in the order of the heads.
#include "delta.h"

namespace taac {
namespace {

// Four wavefronts; wavefront w owns tokens 16 w .. 16 w + 15 of the chunk, a lane one of them (four key features at a time).
template <int DK, int DV>
struct GradLds {
  static constexpr int kTileK = 0;
  static constexpr int kTileQ = kTileK + Tile<DK>::BYTES;
  static constexpr int kTileO = kTileQ + Tile<DK>::BYTES;
  static constexpr int kTileX = kTileO + Tile<DV>::BYTES;
  static constexpr int kTileN = kTileX + Tile<DV>::BYTES;
  static constexpr int kTileLow = kTileN + Tile<DV>::BYTES;  // what the rounding of N left
  static constexpr int kState = kTileLow + Tile<DV>::BYTES;  // DV rows of DK
  static constexpr bool kTurns = DK > 64 && DV > 64;         // S and dS' take turns: both do not fit
  static constexpr int kGradState = kTurns ? kState : kState + DV * Tile<DK>::STRIDE * 2;
  static constexpr int kRows = kGradState + DV * Tile<DK>::STRIDE * 2;
  static constexpr int kTotal = kRows + (kRowFloats + kTempFloats + 64 + 3 * 64 + 16) * 4;
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
__global__ __launch_bounds__(4 * kWave, DK <= 32 && DV <= 64 ? 3 : DK <= 64 && DV <= 64 ? 2 : 1) void delta_grads_kernel(const DeltaParams p) {
  constexpr int KA = DK / 16, VB = DV / 32, kThreads = 4 * kWave;
  typedef GradLds<DK, DV> L;
  typedef Tile<DK> TK;
  typedef Tile<DV> TV;
  extern __shared__ __attribute__((aligned(64))) uint8_t smem[];
  bf16_t* tile_k = reinterpret_cast<bf16_t*>(smem + L::kTileK);
  bf16_t* tile_q = reinterpret_cast<bf16_t*>(smem + L::kTileQ);
  bf16_t* tile_o = reinterpret_cast<bf16_t*>(smem + L::kTileO);
  bf16_t* tile_x = reinterpret_cast<bf16_t*>(smem + L::kTileX);
  bf16_t* tile_n = reinterpret_cast<bf16_t*>(smem + L::kTileN);
  bf16_t* tile_l = reinterpret_cast<bf16_t*>(smem + L::kTileLow);
  bf16_t* tile_s = reinterpret_cast<bf16_t*>(smem + L::kState);
  bf16_t* tile_g = reinterpret_cast<bf16_t*>(smem + L::kGradState);
  float* rows = reinterpret_cast<float*>(smem + L::kRows);
  float* temp = rows + kRowFloats;
  float* left_over = temp + kTempFloats;  // e^(G_64 - G)
  float* d_total = left_over + 64; // dG of a token
  float* d_beta = d_total + 64;
  float* d_tail = d_beta + 64;     // its share of dG_64
  float* state_dot = d_tail + 64;  // per wavefront

  int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const uint32_t key_heads = static_cast<uint32_t>(p.H) / p.group;
  const int chunk = static_cast<int>(blockIdx.x % static_cast<uint32_t>(p.chunks));
  const uint32_t pair = blockIdx.x / static_cast<uint32_t>(p.chunks);
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

  f32x4 dq_sum[KA], dk_sum[KA];
#pragma unroll
  for (int a = 0; a < KA; ++a) dq_sum[a] = dk_sum[a] = zero4();

  if (n_tok > 0) {
    typename TK::template Piece<kChunk, kThreads> k_in, q_in;
    k_in.load(p.k + b * p.ks[0] + hk * p.ks[1] + token0 * p.ks[2], p.ks[2], n_tok, p.dk, tid);
    q_in.load(p.q + b * p.qs[0] + hk * p.qs[1] + token0 * p.qs[2], p.qs[2], n_tok, p.dk, tid);
    k_in.store(tile_k, tid);
    q_in.store(tile_q, tid);
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
    // opaque to the compiler, which would otherwise keep the LDS addresses of the whole loop body in registers across the heads
    int l16 = lane % 16, grp = lane / 16;
    asm volatile("" : "+v"(l16), "+v"(grp), "+v"(tid));
    const int row = 16 * wave + l16;  // this lane's token
    // everything this head reads is requested before any of it is waited for
    typename TV::template Piece<kChunk, kThreads> o_in, x_in, n_in, l_in;
    typename TK::template Piece<DV, kThreads> s_in, g_in;
    const int64_t at_state = (unit * p.chunks + chunk) * static_cast<int64_t>(p.dk) * p.dv;
    GateBits gates;
    if (wave == 0) gates.request(p, b, h, token0, n_tok, lane);
    o_in.load(p.grad_o + b * p.dos[0] + h * p.dos[1] + token0 * p.dos[2], p.dos[2], n_tok, p.dv, tid);
    x_in.load(p.grad_v + b * p.dvs[0] + h * p.dvs[1] + token0 * p.dvs[2], p.dvs[2], n_tok, p.dv, tid);
    n_in.load(p.misses + (unit * p.T + token0) * p.dv, p.dv, n_tok, p.dv, tid);
    l_in.load(p.misses_low + (unit * p.T + token0) * p.dv, p.dv, n_tok, p.dv, tid);
    s_in.load(p.chunk_states + at_state, p.dk, p.dv, p.dk, tid);
    g_in.load(p.grad_states + at_state, p.dk, p.dv, p.dk, tid);
    float dot_state = s_in.dot(g_in);
    __syncthreads();  // the previous head's tiles and sums are no longer read
    if (wave == 0) chunk_rows(p, gates, n_tok, rows, temp, left_over);
    o_in.store(tile_o, tid);
    x_in.store(tile_x, tid);
    n_in.store(tile_n, tid);
    l_in.store(tile_l, tid);
    s_in.template store<true>(tile_s, tid);
    if (!L::kTurns) g_in.template store<true>(tile_g, tid);
    __syncthreads();

    const float hi_t = temp[kTempHi + row], lo_t = temp[kTempLow + row], beta_t = temp[kTempBeta + row], grown = rows[kRowGrown + row];
    // Gam of this lane's token and the four of tile t that its registers hold; in the own tile this token is the later of a pair (sign 1) or the
    // earlier (sign -1), and pairs in the other order get whatever, to be masked (decays may grow: no sign of a difference says which it is)
    auto decays = [&](int t, float sign) __attribute__((always_inline)) -> f32x4 {
      f32x4 gam;
      if (t == wave) {
        const f32x4 hi_r = *reinterpret_cast<const f32x4*>(temp + kTempHi + 16 * t + 4 * grp);
        const f32x4 lo_r = *reinterpret_cast<const f32x4*>(temp + kTempLow + 16 * t + 4 * grp);
#pragma unroll
        for (int r = 0; r < 4; ++r) gam[r] = __builtin_amdgcn_exp2f(sign * ((hi_t - hi_r[r]) + (lo_t - lo_r[r])));
      } else {
        const f32x4 other = *reinterpret_cast<const f32x4*>(temp + (t < wave ? kTempOut : kTempIn) + 16 * t + 4 * grp);
        const float own = t < wave ? temp[kTempIn + row] * tiles_between(rows, wave, t) : temp[kTempOut + row] * tiles_between(rows, t, wave);
#pragma unroll
        for (int r = 0; r < 4; ++r) gam[r] = own * other[r];
      }
      return gam;
    };
    // The sums of the pairs' contributions to dG over a row and over a column are taken from the same fp32 values: pairs on one side of a
    // token then cancel in dg as they do in the formula, and a token's pair with itself stays out of both, so that a first token's decay, which
    // acts on nothing, has a gradient of zero.
    float dot_row = 0.f, dot_col = 0.f, dot_own = 0.f, dot_tail = 0.f;
    bf16x8 b_hi[2], b_lo[2], e_hi[2], e_lo[2];
    bf16x8 first[VB], second[VB], third[KA / 2], fourth[KA / 2];
    // this wavefront's tokens as i: dQ and R
#pragma unroll
    for (int vb = 0; vb < VB; ++vb) {
      first[vb] = TV::row(tile_o, row, vb, grp);
      second[vb] = TV::row(tile_x, row, vb, grp);
    }
#pragma unroll
    for (int kb = 0; kb < KA / 2; ++kb) {
      third[kb] = TK::row(tile_q, row, kb, grp);
      fourth[kb] = TK::row(tile_k, row, kb, grp);
    }
#pragma unroll
    for (int tk = 0; tk < 2; ++tk) {
      f32x4 bv[2], ev[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int t = 2 * tk + half;
        bv[half] = ev[half] = zero4();
        if (t > wave) continue;
        f32x4 qk = zero4(), kk = zero4();
#pragma unroll
        for (int vb = 0; vb < VB; ++vb) {
          const bf16x8 nf = TV::row(tile_n, 16 * t + l16, vb, grp), lf = TV::row(tile_l, 16 * t + l16, vb, grp);
          bv[half] = mfma16(lf, first[vb], mfma16(nf, first[vb], bv[half]));
          ev[half] = mfma16(lf, second[vb], mfma16(nf, second[vb], ev[half]));
        }
#pragma unroll
        for (int kb = 0; kb < KA / 2; ++kb) {
          const bf16x8 kf = TK::row(tile_k, 16 * t + l16, kb, grp);
          qk = mfma16(kf, third[kb], qk);
          kk = mfma16(kf, fourth[kb], kk);
        }
        const f32x4 gam = decays(t, 1.f), beta_r = *reinterpret_cast<const f32x4*>(temp + kTempBeta + 16 * t + 4 * grp);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = 16 * t + 4 * grp + r;
          const float g = gam[r] * beta_r[r];
          bv[half][r] = row >= j ? p.scale * g * bv[half][r] : 0.f;
          ev[half][r] = row > j ? -g * ev[half][r] : 0.f;
          if (row > j) dot_row += fmaf(bv[half][r], qk[r], ev[half][r] * kk[r]);
        }
      }
      split(bv[0], bv[1], b_hi[tk], b_lo[tk]);
      split(ev[0], ev[1], e_hi[tk], e_lo[tk]);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int a = 0; a < KA; ++a) {
      f32x4 dq = zero4(), dr = zero4();
#pragma unroll
      for (int vb = 0; vb < VB; ++vb) {
        const bf16x8 sf = TK::keys_frag(tile_s, vb, a, l16, grp);
        dq = mfma16(sf, first[vb], dq);
        dr = mfma16(sf, second[vb], dr);
      }
      const int at = row * TK::STRIDE + state_row(a, 4 * grp);
      const bf16x4 kv = *reinterpret_cast<const bf16x4*>(tile_k + at), qv = *reinterpret_cast<const bf16x4*>(tile_q + at);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        dq[r] *= p.scale * grown;
        dr[r] *= -grown;
        dot_row = fmaf(static_cast<float>(qv[r]), dq[r], fmaf(static_cast<float>(kv[r]), dr[r], dot_row));
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        dq_sum[a][r] += dq[r];
        dk_sum[a][r] += dr[r];
      }
#pragma unroll
      for (int tk = 0; tk < 2; ++tk) {
        const bf16x8 kt = TK::keys_frag(tile_k, tk, a, l16, grp);
        dq_sum[a] = mfma16(kt, b_lo[tk], mfma16(kt, b_hi[tk], dq_sum[a]));
        dk_sum[a] = mfma16(kt, e_lo[tk], mfma16(kt, e_hi[tk], dk_sum[a]));
      }
      __builtin_amdgcn_sched_barrier(0);  // keeps the next round's reads, and their registers, behind this one
    }
    if (L::kTurns) {
      __syncthreads();  // S is no longer read
      g_in.template store<true>(tile_g, tid);
      __syncthreads();
    }
    // as j: C
#pragma unroll
    for (int vb = 0; vb < VB; ++vb) {
      first[vb] = TV::row(tile_n, row, vb, grp);
      second[vb] = TV::row(tile_l, row, vb, grp);
    }
#pragma unroll
    for (int tk = 0; tk < 2; ++tk) {
      f32x4 bv[2], ev[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int t = 2 * tk + half;
        bv[half] = ev[half] = zero4();
        if (t < wave) continue;
        f32x4 qk = zero4(), kk = zero4();
#pragma unroll
        for (int vb = 0; vb < VB; ++vb) {
          const bf16x8 of = TV::row(tile_o, 16 * t + l16, vb, grp), xf = TV::row(tile_x, 16 * t + l16, vb, grp);
          bv[half] = mfma16(of, second[vb], mfma16(of, first[vb], bv[half]));
          ev[half] = mfma16(xf, second[vb], mfma16(xf, first[vb], ev[half]));
        }
#pragma unroll
        for (int kb = 0; kb < KA / 2; ++kb) {
          qk = mfma16(TK::row(tile_q, 16 * t + l16, kb, grp), fourth[kb], qk);
          kk = mfma16(TK::row(tile_k, 16 * t + l16, kb, grp), fourth[kb], kk);
        }
        const f32x4 gam = decays(t, -1.f);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * t + 4 * grp + r;
          bv[half][r] = i >= row ? p.scale * gam[r] * bv[half][r] : 0.f;
          ev[half][r] = i > row ? -gam[r] * ev[half][r] : 0.f;
          const float pair = fmaf(bv[half][r], qk[r], ev[half][r] * kk[r]);
          dot_col += i > row ? pair : 0.f;
          dot_own += i == row ? pair : 0.f;
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int r = 0; r < 4; ++r) bv[half][r] *= beta_t, ev[half][r] *= beta_t;
      split(bv[0], bv[1], b_hi[tk], b_lo[tk]);
      split(ev[0], ev[1], e_hi[tk], e_lo[tk]);
      __builtin_amdgcn_sched_barrier(0);
    }
    const float tail = left_over[row];
#pragma unroll
    for (int a = 0; a < KA; ++a) {
      f32x4 dc = zero4();
#pragma unroll
      for (int vb = 0; vb < VB; ++vb) {
        const bf16x8 gf = TK::keys_frag(tile_g, vb, a, l16, grp);
        dc = mfma16(gf, second[vb], mfma16(gf, first[vb], dc));
      }
      const bf16x4 kv = *reinterpret_cast<const bf16x4*>(tile_k + row * TK::STRIDE + state_row(a, 4 * grp));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        dc[r] *= tail;
        dot_tail = fmaf(static_cast<float>(kv[r]), dc[r], dot_tail);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) dk_sum[a][r] = fmaf(beta_t, dc[r], dk_sum[a][r]);
#pragma unroll
      for (int tk = 0; tk < 2; ++tk) {
        const bf16x8 kt = TK::keys_frag(tile_k, tk, a, l16, grp), qt = TK::keys_frag(tile_q, tk, a, l16, grp);
        dk_sum[a] = mfma16(qt, b_lo[tk], mfma16(qt, b_hi[tk], dk_sum[a]));
        dk_sum[a] = mfma16(kt, e_lo[tk], mfma16(kt, e_hi[tk], dk_sum[a]));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    dot_row = group_total(dot_row);
    dot_col = group_total(dot_col);
    dot_own = group_total(dot_own);
    dot_tail = group_total(dot_tail);
    dot_state = group_sum<kWave>(dot_state);
    if (grp == 0) {
      d_total[row] = dot_row - beta_t * dot_col;
      d_beta[row] = dot_col + dot_own + dot_tail;
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
  const int row = 16 * wave + lane % 16, grp = lane / 16;
  if (row < span) {  // rows behind the last token hold zeros
    bf16_t* dq_row = p.grad_q + b * p.dqs[0] + hk * p.dqs[1] + (token0 + row) * p.dqs[2];
    bf16_t* dk_row = p.grad_k + b * p.dks[0] + hk * p.dks[1] + (token0 + row) * p.dks[2];
#pragma unroll
    for (int a = 0; a < KA; ++a) {
      const int at = state_row(a, 4 * grp);
      if (at >= p.dk) continue;
      *reinterpret_cast<u32x2*>(dq_row + at) = round4(dq_sum[a]);
      *reinterpret_cast<u32x2*>(dk_row + at) = round4(dk_sum[a]);
    }
  }
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
int dispatch_grads(const char* name, const DeltaParams& p, hipStream_t s) {
  if (p.dv <= 32) return launch_grads<DK, 32>(name, p, s);
  if (p.dv <= 64) return launch_grads<DK, 64>(name, p, s);
  return launch_grads<DK, 128>(name, p, s);
}

}  // namespace

int delta_grads(const char* name, const DeltaParams& p, hipStream_t s) {
  if (p.dk <= 32) return dispatch_grads<32>(name, p, s);
  if (p.dk <= 64) return dispatch_grads<64>(name, p, s);
  return dispatch_grads<128>(name, p, s);
}

}  // namespace taac
