// Gated delta rule, chunked form: the entry points, their checks, and which form takes a call.
#include "delta.h"

namespace taac {
namespace {

// Heads of at most 64 key features walk alone (delta_solo.hip) from more than two teams of 16 columns to a CU on (two and a half of 64 wide ones):
// the chain of chunks no longer counts then, and nothing is left in memory between two kernels. Wider heads always take the teams of
// delta_team.hip: their state does not fit the registers of one wavefront. 2048 tokens, team : solo, by heads times groups of 16 columns:
//   32 wide, forward 131 : 168 us at 384, 170 : 165 at 512, 217 : 168 at 640; with the backward 388 : 446, 463 : 468, 593 : 517
//   64 wide, forward 182 : 205 us at 640, 204 : 205 at 768, 273 : 207 at 1024; with the backward 542 : 556, 626 : 583, 830 : 632
bool uses_teams(int64_t heads, int32_t dk, int32_t dv) { return dk > 64 || heads * ((dv + 15) / 16) <= (dk <= 32 ? 512 : 640); }

int64_t workspace_of(int64_t heads, int32_t T, int32_t dk, int32_t dv) {
  return uses_teams(heads, dk, dv) ? heads * ((static_cast<int64_t>(T) + kChunk - 1) / kChunk) * block_bytes(dk) : 0;
}

int take_workspace(const char* name, DeltaParams& p, void* workspace, int64_t given, bool* team) {
  const int64_t heads = static_cast<int64_t>(p.B) * p.H, bytes = workspace_of(heads, p.T, p.dk, p.dv);
  *team = uses_teams(heads, p.dk, p.dv);
  if (bytes > 0 && (workspace == nullptr || given < bytes || !aligned16(workspace)))
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: workspace must hold %lld bytes, 16-byte aligned", name, (long long)bytes);
  p.blocks = static_cast<uint8_t*>(workspace);
  return TAAC_OK;
}

// Two planes: N rounded, and the rest.
void take_misses(DeltaParams& p, void* misses) {
  p.misses = static_cast<bf16_t*>(misses);
  if (misses != nullptr) p.misses_low = p.misses + static_cast<int64_t>(p.B) * p.H * p.T * p.dv;
}

int check_sizes(const char* name, const DeltaParams& p) {
  if (p.B < 0 || p.H <= 0 || p.T < 0 || p.dk <= 0 || p.dv <= 0 || p.group <= 0)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: batch and tokens must be >= 0, heads and widths > 0", name);
  if (p.T > 1 << 30) return set_error(TAAC_ERR_UNSUPPORTED, "%s: at most 2^30 tokens (got %d)", name, p.T);  // 32-bit token numbers
  if (p.dk % 8 != 0 || p.dv % 8 != 0 || p.dk > 128 || p.dv > 128)
    return set_error(TAAC_ERR_UNSUPPORTED, "%s: key and value widths must be multiples of 8, at most 128 (got %d, %d)", name, p.dk, p.dv);
  return TAAC_OK;
}

// Strides of (batch, head, token): multiples of 8 elements for the 16-byte rows.
int take_strides(const char* name, const char* what, const void* ptr, const int64_t* from, int64_t* to, bool rows, int32_t width) {
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

}  // namespace
}  // namespace taac

extern "C" int taac_delta_rule_fwd(const void* q, const void* k, const void* v, const void* log_decay, const void* beta,
                                   const int32_t* lengths, void* o, const float* state_in, float* state_out, void* chunk_states,
                                   void* misses, void* workspace, int64_t workspace_bytes, int32_t B, int32_t H, int32_t key_heads,
                                   int32_t T, int32_t dk, int32_t dv, const int64_t q_strides[3], const int64_t k_strides[3],
                                   const int64_t v_strides[3], const int64_t o_strides[3], const int64_t decay_strides[3],
                                   const int64_t beta_strides[3], float scale, int gate_dtype, void* stream) {
  using namespace taac;
  const char* name = "taac_delta_rule_fwd";
  DeltaParams p{};
  if (key_heads <= 0 || H <= 0 || H % key_heads != 0)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: value heads must be a multiple of the key heads", name);
  p.B = B, p.H = H, p.group = H / key_heads, p.T = T, p.dk = dk, p.dv = dv, p.scale = scale;
  if (int rc = check_sizes(name, p)) return rc;
  p.chunks = (T + kChunk - 1) / kChunk;
  if (gate_dtype != TAAC_F32 && gate_dtype != TAAC_BF16)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: gates must be fp32 or bf16 (dtype %d)", name, gate_dtype);
  p.gates_f32 = gate_dtype == TAAC_F32;
  if ((chunk_states == nullptr) != (misses == nullptr))
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: chunk_states and misses come together", name);
  if (B == 0 || (T == 0 && state_out == nullptr)) return TAAC_OK;
  if (T > 0 && (!q || !k || !v || !log_decay || !beta || !o)) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null tensor pointer", name);
  if (int rc = take_strides(name, "q", q, q_strides, p.qs, true, dk)) return rc;
  if (int rc = take_strides(name, "k", k, k_strides, p.ks, true, dk)) return rc;
  if (int rc = take_strides(name, "v", v, v_strides, p.vs, true, dv)) return rc;
  if (int rc = take_strides(name, "o", o, o_strides, p.os, true, dv)) return rc;
  if (int rc = take_strides(name, "log_decay", log_decay, decay_strides, p.gs, false, 1)) return rc;
  if (int rc = take_strides(name, "beta", beta, beta_strides, p.bs, false, 1)) return rc;
  p.q = static_cast<const bf16_t*>(q), p.k = static_cast<const bf16_t*>(k), p.v = static_cast<const bf16_t*>(v);
  p.o = static_cast<bf16_t*>(o), p.log_decay = log_decay, p.beta = beta, p.lengths = lengths;
  p.state_in = state_in, p.state_out = state_out;
  p.chunk_states = static_cast<bf16_t*>(chunk_states);
  take_misses(p, misses);
  hipStream_t s = as_stream(stream);
  bool team;
  if (int rc = take_workspace(name, p, workspace, workspace_bytes, &team)) return rc;
  return team ? delta_team(name, p, false, s) : delta_solo(name, p, false, s);
}

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
  if (int rc = check_sizes(name, p)) return rc;
  p.chunks = (T + kChunk - 1) / kChunk;
  if (gate_dtype != TAAC_F32 && gate_dtype != TAAC_BF16)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: gates must be fp32 or bf16 (dtype %d)", name, gate_dtype);
  p.gates_f32 = gate_dtype == TAAC_F32;
  if (B == 0 || T == 0) return TAAC_OK;
  if (!q || !k || !log_decay || !beta || !chunk_states || !misses || !grad_o || !grad_q || !grad_k || !grad_v || !grad_decay || !grad_beta ||
      !grad_states)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: null tensor pointer", name);
  if (int rc = take_strides(name, "q", q, q_strides, p.qs, true, dk)) return rc;
  if (int rc = take_strides(name, "k", k, k_strides, p.ks, true, dk)) return rc;
  if (int rc = take_strides(name, "log_decay", log_decay, decay_strides, p.gs, false, 1)) return rc;
  if (int rc = take_strides(name, "beta", beta, beta_strides, p.bs, false, 1)) return rc;
  if (int rc = take_strides(name, "grad_o", grad_o, go_strides, p.dos, true, dv)) return rc;
  if (int rc = take_strides(name, "grad_q", grad_q, gq_strides, p.dqs, true, dk)) return rc;
  if (int rc = take_strides(name, "grad_k", grad_k, gk_strides, p.dks, true, dk)) return rc;
  if (int rc = take_strides(name, "grad_v", grad_v, gv_strides, p.dvs, true, dv)) return rc;
  if (int rc = take_strides(name, "grad_log_decay", grad_decay, gdecay_strides, p.dgs, false, 1)) return rc;
  if (int rc = take_strides(name, "grad_beta", grad_beta, gbeta_strides, p.dbs, false, 1)) return rc;
  p.q = static_cast<const bf16_t*>(q), p.k = static_cast<const bf16_t*>(k), p.log_decay = log_decay, p.beta = beta, p.lengths = lengths;
  p.chunk_states = const_cast<bf16_t*>(static_cast<const bf16_t*>(chunk_states));
  take_misses(p, const_cast<void*>(misses));
  p.grad_o = static_cast<const bf16_t*>(grad_o);
  p.grad_q = static_cast<bf16_t*>(grad_q), p.grad_k = static_cast<bf16_t*>(grad_k), p.grad_v = static_cast<bf16_t*>(grad_v);
  p.grad_decay = grad_decay, p.grad_beta = grad_beta, p.grad_states = static_cast<bf16_t*>(grad_states);
  hipStream_t s = as_stream(stream);
  bool team;
  if (int rc = take_workspace(name, p, workspace, workspace_bytes, &team)) return rc;
  if (int rc = team ? delta_team(name, p, true, s) : delta_solo(name, p, true, s)) return rc;
  return delta_grads(name, p, s);
}

extern "C" int64_t taac_delta_rule_workspace_bytes(int32_t B, int32_t H, int32_t T, int32_t dk, int32_t dv) {
  if (B < 0 || H <= 0 || T < 0 || dk <= 0 || dv <= 0) return -1;
  return taac::workspace_of(static_cast<int64_t>(B) * H, T, dk, dv);
}
