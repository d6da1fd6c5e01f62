// Gated delta rule, chunked form, backward (notation, operand order and precision: delta.h).
//
// With dS' the gradient of the state behind a chunk, X, N as in the forward and T the chunk's 64 tokens:
//   beta dU = diag(beta e^{G_64 - G}) K dS' + P^T dO          (P holds scale, Gam and beta of its column)
//   dX = beta dU - M^T (beta dU) = dV
//   dS = e^{G_64} dS' + Q^T (scale e^G dO) - K^T (e^G dX)
// is a recurrence like the forward's, backwards, column by column of the values: this kernel (or that of delta_team.hip), which keeps dS' of
// every chunk and dX.
// The other gradients are made from these chunk by chunk (delta_grads.hip).
#include "delta.h"

namespace taac {
namespace {

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

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave, l16 = lane % 16, grp = lane / 16;
  const int col_groups = (p.dv + L::COLS - 1) / L::COLS;
  const uint32_t block_id = xcd_remap(blockIdx.x, gridDim.x);  // the columns of a head, which read the same rows, on one die's L2
  const int64_t unit = block_id / col_groups;
  const int col0 = static_cast<int>(block_id % col_groups) * L::COLS;
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
                            reinterpret_cast<float*>(block + kBlockP), reinterpret_cast<float*>(block));
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

      bf16x8 sh[KB][NT], sl[KB][NT];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int n = 0; n < NT; ++n) split(s[2 * kb][n], s[2 * kb + 1][n], sh[kb][n], sl[kb][n]);
      {
        bf16_t* dst = p.grad_states + (unit * p.chunks + chunk) * static_cast<int64_t>(p.dk) * p.dv;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            if (col_ok[n] && 32 * kb + 8 * grp < p.dk) *reinterpret_cast<bf16x8*>(dst + (col[n] + l16) * p.dk + 32 * kb + 8 * grp) = sh[kb][n];
      }

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

template <int DK>
int dispatch_back(const char* name, const DeltaParams& p, hipStream_t s) {
  int rc;
  if (p.blocks != nullptr) rc = delta_team_back(name, p, s);
  else if (p.dk <= 64) rc = delta_solo(name, p, true, s);
  else if (p.dv <= 32) rc = launch_back<DK, 2, 1>(name, p, s);
  else if (p.dv <= 64) rc = launch_back<DK, 2, 2>(name, p, s);
  else rc = launch_back<DK, 2, 4>(name, p, s);
  return rc == TAAC_OK ? delta_grads(name, p, s) : rc;
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
  if (int rc = delta_strides(name, "q", q, q_strides, p.qs, true, dk)) return rc;
  if (int rc = delta_strides(name, "k", k, k_strides, p.ks, true, dk)) return rc;
  if (int rc = delta_strides(name, "log_decay", log_decay, decay_strides, p.gs, false, 1)) return rc;
  if (int rc = delta_strides(name, "beta", beta, beta_strides, p.bs, false, 1)) return rc;
  if (int rc = delta_strides(name, "grad_o", grad_o, go_strides, p.dos, true, dv)) return rc;
  if (int rc = delta_strides(name, "grad_q", grad_q, gq_strides, p.dqs, true, dk)) return rc;
  if (int rc = delta_strides(name, "grad_k", grad_k, gk_strides, p.dks, true, dk)) return rc;
  if (int rc = delta_strides(name, "grad_v", grad_v, gv_strides, p.dvs, true, dv)) return rc;
  if (int rc = delta_strides(name, "grad_log_decay", grad_decay, gdecay_strides, p.dgs, false, 1)) return rc;
  if (int rc = delta_strides(name, "grad_beta", grad_beta, gbeta_strides, p.dbs, false, 1)) return rc;
  p.q = static_cast<const bf16_t*>(q), p.k = static_cast<const bf16_t*>(k), p.log_decay = log_decay, p.beta = beta, p.lengths = lengths;
  p.chunk_states = const_cast<bf16_t*>(static_cast<const bf16_t*>(chunk_states));
  p.misses = const_cast<bf16_t*>(static_cast<const bf16_t*>(misses));
  p.grad_o = static_cast<const bf16_t*>(grad_o);
  p.grad_q = static_cast<bf16_t*>(grad_q), p.grad_k = static_cast<bf16_t*>(grad_k), p.grad_v = static_cast<bf16_t*>(grad_v);
  p.grad_decay = grad_decay, p.grad_beta = grad_beta, p.grad_states = static_cast<bf16_t*>(grad_states);
  hipStream_t s = as_stream(stream);
  if (const int64_t bytes = delta_team_bytes(static_cast<int64_t>(B) * H, T, dk, dv)) {
    if (workspace == nullptr || workspace_bytes < bytes || !aligned16(workspace))
      return set_error(TAAC_ERR_INVALID_VALUE, "%s: workspace must hold %lld bytes, 16-byte aligned", name, (long long)bytes);
    p.blocks = static_cast<uint8_t*>(workspace);
  }
  return dispatch_back<128>(name, p, s);
}
