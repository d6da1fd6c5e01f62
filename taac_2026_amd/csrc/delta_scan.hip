// Gated delta rule, chunked form, forward (the mathematics, operand order and precision: delta.h).
//
// A workgroup of NW wavefronts walks the chunks of one (sample, head) and 16 NT NW value columns; a wavefront keeps its columns of the
// state in registers. The wavefronts first make the blocks of up to NW chunks, one each (they do not depend on the state), then walk
// these chunks together: K and V through LDS, Q as fragments from memory.
#include "delta.h"

namespace taac {
namespace {

template <int DK, int NT, int NW>
struct ScanLds {
  static constexpr int COLS = 16 * NT * NW;
  static constexpr int VCOLS = COLS < 32 ? 32 : COLS;
  static constexpr int kTileK = NW * kBlockBytes;
  static constexpr int kTileV = kTileK + Tile<DK>::BYTES;
  static constexpr int kTotal = kTileV + Tile<VCOLS>::BYTES;
};

template <int DK, int NT, int NW, bool TRAIN>
__global__ __launch_bounds__(NW * kWave) void delta_scan_kernel(const DeltaParams p) {
  constexpr int KB = DK / 32, KA = DK / 16;
  typedef ScanLds<DK, NT, NW> L;
  typedef Tile<DK> TK;
  typedef Tile<L::VCOLS> TV;
  extern __shared__ __attribute__((aligned(64))) uint8_t smem[];
  bf16_t* tile_k = reinterpret_cast<bf16_t*>(smem + L::kTileK);
  bf16_t* tile_v = reinterpret_cast<bf16_t*>(smem + L::kTileV);

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave, l16 = lane % 16, grp = lane / 16;
  const int col_groups = (p.dv + L::COLS - 1) / L::COLS;
  const uint32_t block_id = xcd_remap(blockIdx.x, gridDim.x);  // the columns of a head, which read the same rows, on one die's L2
  const int64_t unit = block_id / col_groups;
  const int col0 = static_cast<int>(block_id % col_groups) * L::COLS;  // of the workgroup
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
  const bf16_t* vb0 = p.v + b * p.vs[0] + h * p.vs[1] + col0;
  bf16_t* ob0 = p.o + b * p.os[0] + h * p.os[1];

  int col[NT];  // first column of a tile, and whether this lane's column exists
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
    for (int n = 0; n < NT; ++n) {
      s[a][n] = zero4();
      if (p.state_in != nullptr && col_ok[n]) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = state_row(a, 4 * grp + r);
          if (row < p.dk) s[a][n][r] = p.state_in[(unit * p.dk + row) * p.dv + col[n] + l16];
        }
      }
    }

  for (int base = 0; base < chunks; base += NW) {
    __syncthreads();  // the blocks of the previous round are no longer read
    if (base + wave < chunks) {
      uint8_t* block = smem + wave * kBlockBytes;
      const int64_t token0 = static_cast<int64_t>(base + wave) * kChunk;
      const int left = len - static_cast<int>(token0);
      chunk_block<DK, false>(p, b, h, token0, left < kChunk ? left : kChunk, block, reinterpret_cast<float*>(block + kBlockRows),
                             reinterpret_cast<float*>(block + kBlockP), reinterpret_cast<float*>(block));
    }
    const int here = chunks - base < NW ? chunks - base : NW;
    for (int c = 0; c < here; ++c) {
      const int64_t token0 = static_cast<int64_t>(base + c) * kChunk;
      const int left = len - static_cast<int>(token0);
      const int n_tok = left < kChunk ? left : kChunk;
      if (c > 0) __syncthreads();  // the tiles of the previous chunk are no longer read
      TK::stage(tile_k, kb0 + token0 * p.ks[2], p.ks[2], n_tok, p.dk, tid, NW * kWave);
      TV::stage(tile_v, vb0 + token0 * p.vs[2], p.vs[2], n_tok, p.dv - col0, tid, NW * kWave);
      __syncthreads();
      const uint8_t* block = smem + c * kBlockBytes;
      const float* rows = reinterpret_cast<const float*>(block + kBlockRows);

      bf16x8 sh[KB][NT], sl[KB][NT];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int n = 0; n < NT; ++n) split(s[2 * kb][n], s[2 * kb + 1][n], sh[kb][n], sl[kb][n]);
      if (TRAIN) {
        bf16_t* dst = p.chunk_states + (unit * p.chunks + base + c) * static_cast<int64_t>(p.dk) * p.dv;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            if (col_ok[n] && 32 * kb + 8 * grp < p.dk) *reinterpret_cast<bf16x8*>(dst + (col[n] + l16) * p.dk + 32 * kb + 8 * grp) = sh[kb][n];
      }

      // X = V - e^G K S
      f32x4 x[4][NT];
#pragma unroll
      for (int ti = 0; ti < 4; ++ti) {
        f32x4 y[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) y[n] = zero4();
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const bf16x8 kf = TK::row(tile_k, 16 * ti + l16, kb, grp);
#pragma unroll
          for (int n = 0; n < NT; ++n) y[n] = mfma16(kf, sl[kb][n], mfma16(kf, sh[kb][n], y[n]));
        }
        const f32x4 grown = *reinterpret_cast<const f32x4*>(rows + kRowGrown + 16 * ti + 4 * grp);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const bf16x4 v = TV::values(tile_v, 16 * ti, wave * NT + n, l16, grp);
#pragma unroll
          for (int r = 0; r < 4; ++r) x[ti][n][r] = fmaf(-grown[r], y[n][r], static_cast<float>(v[r]));
        }
      }
      // N = X - M X
      bf16x8 xh[2][NT], xl[2][NT];
#pragma unroll
      for (int tk = 0; tk < 2; ++tk)
#pragma unroll
        for (int n = 0; n < NT; ++n) split(x[2 * tk][n], x[2 * tk + 1][n], xh[tk][n], xl[tk][n]);
#pragma unroll
      for (int ti = 0; ti < 4; ++ti)
#pragma unroll
        for (int tk = 0; tk <= ti / 2; ++tk) {
          const bf16x8 mh = *reinterpret_cast<const bf16x8*>(block + kBlockM + frag_rows(ti, tk) * kFrag + lane * 16);
          const bf16x8 ml = *reinterpret_cast<const bf16x8*>(block + kBlockLow + frag_rows(ti, tk) * kFrag + lane * 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) x[ti][n] = mfma16(ml, xh[tk][n], mfma16(mh, xl[tk][n], mfma16(mh, xh[tk][n], x[ti][n])));
        }
      if (TRAIN) {
        bf16_t* dst = p.misses + (unit * p.T + token0) * p.dv;
#pragma unroll
        for (int ti = 0; ti < 4; ++ti)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int row = 16 * ti + 4 * grp + r;
              if (col_ok[n] && row < n_tok) dst[row * p.dv + col[n] + l16] = static_cast<bf16_t>(x[ti][n][r]);
            }
      }
      // O by columns of tokens: lane = token, four value columns each
      bf16x8 nh[2][NT], nl[2][NT];
#pragma unroll
      for (int tk = 0; tk < 2; ++tk)
#pragma unroll
        for (int n = 0; n < NT; ++n) split(x[2 * tk][n], x[2 * tk + 1][n], nh[tk][n], nl[tk][n]);
#pragma unroll
      for (int ti = 0; ti < 4; ++ti) {
        const int row = 16 * ti + l16;
        const bf16_t* q_row = row < n_tok ? qb0 + (token0 + row) * p.qs[2] : nullptr;
        f32x4 out[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) out[n] = zero4();
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const bf16x8 qf = row_frag(q_row, kb, grp, p.dk);
#pragma unroll
          for (int n = 0; n < NT; ++n) out[n] = mfma16(sl[kb][n], qf, mfma16(sh[kb][n], qf, out[n]));
        }
        const float grown = rows[kRowGrown + row] * p.scale;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) out[n][r] *= grown;
#pragma unroll
        for (int tk = 0; tk <= ti / 2; ++tk) {
          const bf16x8 pf = *reinterpret_cast<const bf16x8*>(block + kBlockP + frag_rows(ti, tk) * kFrag + lane * 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) out[n] = mfma16(nl[tk][n], pf, mfma16(nh[tk][n], pf, out[n]));
        }
        if (row < n_tok) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (col[n] + 4 * grp >= p.dv) continue;
            *reinterpret_cast<u32x2*>(ob0 + (token0 + row) * p.os[2] + col[n] + 4 * grp) = round4(out[n]);
          }
        }
      }
      // S' = e^G_last S + K^T (beta e^(G_last - G) N)
#pragma unroll
      for (int ti = 0; ti < 4; ++ti) {
        const f32x4 keep = *reinterpret_cast<const f32x4*>(rows + kRowKeep + 16 * ti + 4 * grp);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) x[ti][n][r] *= keep[r];
      }
#pragma unroll
      for (int tk = 0; tk < 2; ++tk)
#pragma unroll
        for (int n = 0; n < NT; ++n) split(x[2 * tk][n], x[2 * tk + 1][n], xh[tk][n], xl[tk][n]);
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
#pragma unroll
          for (int n = 0; n < NT; ++n) s[a][n] = mfma16(kt, xl[tk][n], mfma16(kt, xh[tk][n], s[a][n]));
        }
      }
    }
  }

  if (p.state_out != nullptr) {
#pragma unroll
    for (int a = 0; a < KA; ++a)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = state_row(a, 4 * grp + r);
          if (col_ok[n] && row < p.dk) p.state_out[(unit * p.dk + row) * p.dv + col[n] + l16] = s[a][n][r];
        }
  }
  // padded rows of the output
  constexpr int QUADS = L::COLS / 4;
  const bf16x4 none = {};
  for (int64_t i = tid; i < static_cast<int64_t>(p.T - len) * QUADS; i += NW * kWave) {
    const int64_t row = len + i / QUADS;
    const int at = col0 + static_cast<int>(i % QUADS) * 4;
    if (at < p.dv) *reinterpret_cast<bf16x4*>(ob0 + row * p.os[2] + at) = none;
  }
}

template <int DK, int NT, int NW, bool TRAIN>
int launch_scan(const char* name, const DeltaParams& p, hipStream_t s) {
  typedef ScanLds<DK, NT, NW> L;
  const int64_t grid = static_cast<int64_t>(p.B) * p.H * ((p.dv + L::COLS - 1) / L::COLS);
  if (grid > 0x7fffffffLL) return set_error(TAAC_ERR_UNSUPPORTED, "%s: too many workgroups", name);
  const void* kernel = reinterpret_cast<const void*>(delta_scan_kernel<DK, NT, NW, TRAIN>);
  if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, L::kTotal) != hipSuccess)
    return set_error(TAAC_ERR_LAUNCH, "%s: cannot reserve %d bytes of LDS", name, L::kTotal);
  hipLaunchKernelGGL((delta_scan_kernel<DK, NT, NW, TRAIN>), dim3(static_cast<uint32_t>(grid)), dim3(NW * kWave), L::kTotal, s, p);
  return check_launch(name);
}

template <int DK, bool TRAIN>
int dispatch_scan(const char* name, const DeltaParams& p, hipStream_t s) {
  if (p.dv <= 32) return launch_scan<DK, 2, 1, TRAIN>(name, p, s);
  if (p.dv <= 64) return launch_scan<DK, 2, 2, TRAIN>(name, p, s);
  return launch_scan<DK, 2, 4, TRAIN>(name, p, s);
}

}  // namespace

int delta_check(const char* name, const DeltaParams& p) {
  if (p.B < 0 || p.H <= 0 || p.T < 0 || p.dk <= 0 || p.dv <= 0 || p.group <= 0)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: batch and tokens must be >= 0, heads and widths > 0", name);
  if (p.dk % 8 != 0 || p.dv % 8 != 0 || p.dk > 128 || p.dv > 128)
    return set_error(TAAC_ERR_UNSUPPORTED, "%s: key and value widths must be multiples of 8, at most 128 (got %d, %d)", name, p.dk, p.dv);
  return TAAC_OK;
}

// Strides of (batch, head, token): multiples of 8 elements for the 16-byte rows.
int delta_strides(const char* name, const char* what, const void* ptr, const int64_t* from, int64_t* to, bool rows, int32_t width) {
  if (from == nullptr) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null strides of %s", name, what);
  for (int i = 0; i < 3; ++i) {
    to[i] = from[i];
    if (from[i] < 0 || (rows && from[i] % 8 != 0))
      return set_error(TAAC_ERR_INVALID_VALUE, "%s: strides of %s must be multiples of 8, not negative", name, what);
  }
  if (rows && from[2] < width)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: the token stride of %s must cover a row", name, what);
  if (rows && from[2] >= (1 << 24)) return set_error(TAAC_ERR_UNSUPPORTED, "%s: the token stride of %s must be below 2^24", name, what);
  if (rows && !aligned16(ptr)) return set_error(TAAC_ERR_INVALID_VALUE, "%s: %s must be 16-byte aligned", name, what);
  return TAAC_OK;
}

}  // namespace taac

extern "C" int taac_delta_rule_fwd(const void* q, const void* k, const void* v, const void* log_decay, const void* beta,
                                   const int32_t* lengths, void* o, const float* state_in, float* state_out, void* chunk_states,
                                   void* misses, void* workspace, int64_t workspace_bytes, int32_t B, int32_t H, int32_t key_heads, int32_t T, int32_t dk, int32_t dv,
                                   const int64_t q_strides[3], const int64_t k_strides[3], const int64_t v_strides[3],
                                   const int64_t o_strides[3], const int64_t decay_strides[3], const int64_t beta_strides[3], float scale,
                                   int gate_dtype, void* stream) {
  using namespace taac;
  const char* name = "taac_delta_rule_fwd";
  DeltaParams p{};
  if (key_heads <= 0 || H <= 0 || H % key_heads != 0)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: value heads must be a multiple of the key heads", name);
  p.B = B, p.H = H, p.group = H / key_heads, p.T = T, p.dk = dk, p.dv = dv, p.scale = scale;
  p.chunks = (T + kChunk - 1) / kChunk;
  if (int rc = delta_check(name, p)) return rc;
  if (gate_dtype != TAAC_F32 && gate_dtype != TAAC_BF16)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: gates must be fp32 or bf16 (dtype %d)", name, gate_dtype);
  p.gates_f32 = gate_dtype == TAAC_F32;
  if ((chunk_states == nullptr) != (misses == nullptr))
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: chunk_states and misses come together", name);
  if (B == 0 || (T == 0 && state_out == nullptr)) return TAAC_OK;
  if (T > 0 && (!q || !k || !v || !log_decay || !beta || !o)) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null tensor pointer", name);
  if (int rc = delta_strides(name, "q", q, q_strides, p.qs, true, dk)) return rc;
  if (int rc = delta_strides(name, "k", k, k_strides, p.ks, true, dk)) return rc;
  if (int rc = delta_strides(name, "v", v, v_strides, p.vs, true, dv)) return rc;
  if (int rc = delta_strides(name, "o", o, o_strides, p.os, true, dv)) return rc;
  if (int rc = delta_strides(name, "log_decay", log_decay, decay_strides, p.gs, false, 1)) return rc;
  if (int rc = delta_strides(name, "beta", beta, beta_strides, p.bs, false, 1)) return rc;
  p.q = static_cast<const bf16_t*>(q), p.k = static_cast<const bf16_t*>(k), p.v = static_cast<const bf16_t*>(v);
  p.o = static_cast<bf16_t*>(o), p.log_decay = log_decay, p.beta = beta, p.lengths = lengths;
  p.state_in = state_in, p.state_out = state_out;
  p.chunk_states = static_cast<bf16_t*>(chunk_states), p.misses = static_cast<bf16_t*>(misses);
  hipStream_t s = as_stream(stream);
  if (const int64_t bytes = delta_team_bytes(static_cast<int64_t>(B) * H, T, dk, dv)) {
    if (workspace == nullptr || workspace_bytes < bytes || !aligned16(workspace))
      return set_error(TAAC_ERR_INVALID_VALUE, "%s: workspace must hold %lld bytes, 16-byte aligned", name, (long long)bytes);
    p.blocks = static_cast<uint8_t*>(workspace);
    return delta_team_fwd(name, p, s);
  }
  if (dk <= 64) return delta_solo(name, p, false, s);
  return chunk_states != nullptr ? dispatch_scan<128, true>(name, p, s) : dispatch_scan<128, false>(name, p, s);
}
