// Gated delta rule, recurrent form: a few new tokens for states that live in a pool, updated in place (the formulas: delta.h).
//
// Bound by HBM: a state of dk x dv floats is read and written once for however many tokens the call brings; everything else is
// small. A workgroup owns the state of one (sample, head): lanes hold four value columns each of some key rows, so that a row is one
// run of memory, and the whole state stays in registers between its load and its store. A token needs one round of sums over the
// key rows, of k S and q S and q . k at once, since o = scale (S + k u^T)^T q = scale (S^T q + (k . q) u). All arithmetic is fp32.
//
// 1024 samples of 8 heads, 64 x 64, out of 1500 slots, one token: 58 us in a trace, 4.7 TB/s (with the reads of the search for samples of the
// same slot one after the other 19 us more, with the token's inputs requested behind it 27).
//
// Samples that name the same slot are one sequence: their tokens are applied in the order of the batch, by the workgroup of the
// first of them. A slot outside the pool (padding) reads and writes no state and gives zeros. To find samples of the same slot every workgroup
// reads all of them: 8 heads of 32 x 32 take 47 us for 4096 samples without slots and 104 with them, for 16384 samples 205 and 891.
#include "delta.h"

namespace taac {
namespace {

struct StepParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  const void* log_decay;
  const void* beta;
  float* state;             // [slots, H, dk, dv]
  const void* slots;        // [B] int32 or int64, or null: slot b
  const int32_t* lengths;   // [B] or null
  int64_t qs[3], ks[3], vs[3], os[3], gs[3], bs[3];
  int64_t pool;             // number of slots
  int32_t B, H, group, T, dk, dv;
  int32_t gates_f32, slots_int64;
  float scale;
};

// An element of a row as the bits that a read brings, for a conversion after everything is requested.
template <typename T>
__device__ __forceinline__ uint32_t read_bits(Buffer b, uint32_t off) {
  if constexpr (sizeof(T) == 4) return __builtin_amdgcn_raw_buffer_load_b32(b, off, 0, 0);
  else return read1(b, off);
}
template <typename T>
__device__ __forceinline__ float from_bits(uint32_t bits) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, bits);
  else return static_cast<float>(__builtin_bit_cast(T, static_cast<uint16_t>(bits)));
}
// A gate is fp32 or a T, read by halves either way: a branch between two reads would await each.
struct Gate {
  uint32_t low, high;
  __device__ __forceinline__ void request(const void* p, int64_t at, int f32) {
    const Buffer b = buffer_of(static_cast<const uint8_t*>(p) + at * (f32 ? 4 : 2), f32 ? 4 : 2);
    low = read1(b, 0);
    high = read1(b, 2);  // zero behind a gate of two bytes
  }
  template <typename T>
  __device__ __forceinline__ float value(int f32) const {
    const float wide = __builtin_bit_cast(float, high << 16 | low);
    return f32 ? wide : from_bits<T>(low);
  }
};

template <int RPT>
struct Token {
  Gate log_decay, beta;
  uint32_t v[4], k[RPT], q[RPT];
};

// NVP: lanes to a row of value columns (4 columns each); W wavefronts; RPT key rows to a lane.
template <typename T, int NVP, int W, int RPT>
__global__ __launch_bounds__(W * kWave) void delta_step_kernel(const StepParams p) {
  constexpr int ROWS = W * kWave / NVP;  // rows at once
  constexpr int kAhead = W > 1 ? 4 : 8;
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const int vec = tid % NVP, row0 = tid / NVP;
  const int h = static_cast<int>(blockIdx.x % static_cast<uint32_t>(p.H));
  const int first = static_cast<int>(blockIdx.x / static_cast<uint32_t>(p.H));
  __shared__ float red[2][W][NVP][8];
  __shared__ float red_qk[2][W];
  const bool col_ok = vec * 4 < p.dv;
  uint32_t state_off[RPT];  // rows behind the last are behind the end of the state too
#pragma unroll
  for (int i = 0; i < RPT; ++i) state_off[i] = col_ok ? ((row0 + i * ROWS) * p.dv + vec * 4) * 4 : kNowhere;
  const T* q = static_cast<const T*>(p.q);
  const T* k = static_cast<const T*>(p.k);
  const T* v = static_cast<const T*>(p.v);
  T* o = static_cast<T*>(p.o);
  const int hk = h / p.group;

  auto slot_of = [&](int b) -> int64_t {
    return p.slots_int64 ? static_cast<const int64_t*>(p.slots)[b] : static_cast<const int32_t*>(p.slots)[b];
  };
  const int64_t slot = p.slots != nullptr ? slot_of(first) : first;
  auto length_of = [&](int b) -> int {
    if (p.lengths == nullptr) return p.T;
    const int n = p.lengths[b];
    return n < 0 ? 0 : (n > p.T ? p.T : n);
  };
  auto clear = [&](int b, int from) {
    for (int t = from; t < p.T; ++t)
      for (int c = tid; c < p.dv; c += W * kWave) o[b * p.os[0] + h * p.os[1] + t * p.os[2] + c] = static_cast<T>(0.f);
  };
  if (slot < 0 || slot >= p.pool) {
    clear(first, 0);
    return;
  }
  f32x4 s[RPT];
  const uint32_t state_bytes = static_cast<uint32_t>(p.dk * p.dv) * 4;
  const Buffer state = buffer_of(p.state + (slot * p.H + h) * static_cast<int64_t>(p.dk) * p.dv, state_bytes);
#pragma unroll
  for (int i = 0; i < RPT; ++i) s[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(state, state_off[i], 0, 0));
  // A token's inputs, requested one token ahead: the first beside the state, before the search for samples of the same slot.
  Token<RPT> next;
  auto request = [&](int b, int t) __attribute__((always_inline)) {
    next.log_decay.request(p.log_decay, b * p.gs[0] + h * p.gs[1] + t * p.gs[2], p.gates_f32);
    next.beta.request(p.beta, b * p.bs[0] + h * p.bs[1] + t * p.bs[2], p.gates_f32);
    const uint32_t key_bytes = static_cast<uint32_t>(p.dk * sizeof(T));
    const Buffer qt = buffer_of(q + b * p.qs[0] + hk * p.qs[1] + t * p.qs[2], key_bytes);
    const Buffer kt = buffer_of(k + b * p.ks[0] + hk * p.ks[1] + t * p.ks[2], key_bytes);
    const Buffer vt = buffer_of(v + b * p.vs[0] + h * p.vs[1] + t * p.vs[2], static_cast<uint32_t>(p.dv * sizeof(T)));
#pragma unroll
    for (int e = 0; e < 4; ++e) next.v[e] = read_bits<T>(vt, (vec * 4 + e) * sizeof(T));
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      next.k[i] = read_bits<T>(kt, (row0 + i * ROWS) * sizeof(T));
      next.q[i] = read_bits<T>(qt, (row0 + i * ROWS) * sizeof(T));
    }
  };
  request(first, 0);
  bool again = false;  // a later sample has the slot too
  if (p.slots != nullptr && p.B > 1) {
    bool before = false, after = false;
    const uint32_t bytes = p.slots_int64 ? 8 : 4, upper = p.slots_int64 ? 4 : 0;  // of four bytes the lower half stands for both
    const Buffer slots = buffer_of(p.slots, p.B * bytes);
    const uint32_t low = static_cast<uint32_t>(slot), high = p.slots_int64 ? static_cast<uint32_t>(slot >> 32) : low;
    for (int j0 = tid; j0 < p.B; j0 += kAhead * W * kWave) {  // several reads in flight: one after the other they took as long as the state
      uint32_t at_low[kAhead], at_high[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const uint32_t off = (j0 + i * W * kWave) * bytes;
        at_low[i] = __builtin_amdgcn_raw_buffer_load_b32(slots, off, 0, 0);
        at_high[i] = __builtin_amdgcn_raw_buffer_load_b32(slots, off + upper, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int j = j0 + i * W * kWave;
        const bool same = (at_low[i] == low) & (at_high[i] == high) & (j < p.B);
        before |= same & (j < first);
        after |= same & (j > first);
      }
    }
    if (__syncthreads_or(before | after)) {
      if (__syncthreads_or(before)) return;  // that sample's workgroup applies these tokens
      again = true;
    }
  }
  bool touched = false;
  int round = 0;
  for (int b = first; b < p.B;) {
    const int n = length_of(b);
    for (int t = 0; t < n; ++t) {
      const float a = expf(next.log_decay.template value<T>(p.gates_f32)), beta = next.beta.template value<T>(p.gates_f32);
      float kr[RPT], vf[4], qr[RPT];
      float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, qk = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) vf[e] = from_bits<T>(next.v[e]);
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        kr[i] = from_bits<T>(next.k[i]);
        qr[i] = from_bits<T>(next.q[i]);
      }
      if (t + 1 < n) request(b, t + 1);
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        qk = fmaf(qr[i], kr[i], qk);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i][e] *= a;
          sum[e] = fmaf(kr[i], s[i][e], sum[e]);
          sum[4 + e] = fmaf(qr[i], s[i][e], sum[4 + e]);
        }
      }
#pragma unroll
      for (int off = NVP; off < kWave; off *= 2) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += __shfl_xor(sum[e], off, kWave);
        qk += __shfl_xor(qk, off, kWave);
      }
      if (W > 1) {  // two sets of partial sums in turn: a token's are read while the next token's are written
        const int buf = round++ & 1;
        if (lane < NVP) {
#pragma unroll
          for (int e = 0; e < 8; ++e) red[buf][wave][lane][e] = sum[e];
          if (lane == 0) red_qk[buf][wave] = qk;
        }
        __syncthreads();
        qk = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[e] += red[buf][w][vec][e];
          qk += red_qk[buf][w];
        }
      }
      float u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = beta * (vf[e] - sum[e]);
#pragma unroll
      for (int i = 0; i < RPT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = fmaf(kr[i], u[e], s[i][e]);
      if (row0 == 0 && col_ok) {
        T* ot = o + b * p.os[0] + h * p.os[1] + t * p.os[2] + vec * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) ot[e] = static_cast<T>(p.scale * fmaf(qk, u[e], sum[4 + e]));
      }
    }
    touched |= n > 0;
    clear(b, n);
    if (!again) break;
    for (++b; b < p.B && slot_of(b) != slot; ++b) {
    }
    if (b < p.B) request(b, 0);
  }
  if (!touched) return;
#pragma unroll
  for (int i = 0; i < RPT; ++i) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, s[i]), state, state_off[i], 0, 0);
}

template <typename T, int NVP, int W, int RPT>
void launch_step(const StepParams& p, hipStream_t s) {
  hipLaunchKernelGGL((delta_step_kernel<T, NVP, W, RPT>), dim3(static_cast<uint32_t>(p.B) * p.H), dim3(W * kWave), 0, s, p);
}

template <typename T>
void dispatch_step(const StepParams& p, hipStream_t s) {
  // One wavefront while a lane's share is at most four rows of four columns, two while it is at most eight, else four: more wavefronts wait for
  // each other, fewer keep less in flight. Samples of 8 heads, with slots (without), 4096 of 32 x 32: 104 (47) us with one, 170 (119) with four;
  // 1024 of 64 x 64: 55 (44) with two, 57 (45) with one, 60 (49) with four; 1024 of 64 x 32: 32 (26) with two, 29 (24) with one, 43 (38) with four.
#define TAAC_STEP_ROWS(NVP)                                                                                   \
  {                                                                                                           \
    constexpr int ROWS = kWave / NVP;                                                                         \
    if (p.dk <= ROWS) return launch_step<T, NVP, 1, 1>(p, s);                                                 \
    if (p.dk <= 2 * ROWS) return launch_step<T, NVP, 1, 2>(p, s);                                             \
    if (p.dk <= 4 * ROWS) return launch_step<T, NVP, 1, 4>(p, s);                                             \
    if (p.dk <= 8 * ROWS) return launch_step<T, NVP, 2, 4>(p, s);                                             \
    if (p.dk <= 16 * ROWS) return launch_step<T, NVP, 2, 8>(p, s);                                            \
    if constexpr (ROWS < 8) {                                                                                 \
      if (p.dk <= 32 * ROWS) return launch_step<T, NVP, 4, 8>(p, s);                                          \
      if constexpr (ROWS < 4) return launch_step<T, NVP, 4, 16>(p, s);                                        \
    }                                                                                                         \
  }
  if (p.dv <= 16) {
    TAAC_STEP_ROWS(4)
  } else if (p.dv <= 32) {
    TAAC_STEP_ROWS(8)
  } else if (p.dv <= 64) {
    TAAC_STEP_ROWS(16)
  } else {
    TAAC_STEP_ROWS(32)
  }
#undef TAAC_STEP_ROWS
}

int step_strides(const char* name, const char* what, const int64_t* from, int64_t* to) {
  if (from == nullptr) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null strides of %s", name, what);
  for (int i = 0; i < 3; ++i) {
    to[i] = from[i];
    if (from[i] < 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: negative stride of %s", name, what);
  }
  return TAAC_OK;
}

}  // namespace
}  // namespace taac

extern "C" int taac_delta_rule_step(const void* q, const void* k, const void* v, const void* log_decay, const void* beta, float* state,
                                    int64_t pool, const void* slots, int slots_int64, const int32_t* lengths, void* o, int32_t B, int32_t H,
                                    int32_t key_heads, int32_t T, int32_t dk, int32_t dv, const int64_t q_strides[3],
                                    const int64_t k_strides[3], const int64_t v_strides[3], const int64_t o_strides[3],
                                    const int64_t decay_strides[3], const int64_t beta_strides[3], float scale, int dtype, int gate_dtype,
                                    void* stream) {
  using namespace taac;
  const char* name = "taac_delta_rule_step";
  if (B < 0 || T < 0 || H <= 0 || key_heads <= 0 || H % key_heads != 0 || pool < 0)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: value heads must be a multiple of the key heads, sizes not negative", name);
  if (dk <= 0 || dv <= 0 || dk % 8 != 0 || dv % 8 != 0 || dk > 128 || dv > 128)
    return set_error(TAAC_ERR_UNSUPPORTED, "%s: key and value widths must be multiples of 8, at most 128 (got %d, %d)", name, dk, dv);
  if (dtype != TAAC_F32 && dtype != TAAC_BF16 && dtype != TAAC_F16) return set_error(TAAC_ERR_INVALID_VALUE, "%s: unknown dtype %d", name, dtype);
  if (gate_dtype != dtype && gate_dtype != TAAC_F32)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: gates must be fp32 or of the tokens' dtype", name);
  if (slots == nullptr && B > pool) return set_error(TAAC_ERR_INVALID_VALUE, "%s: %d samples without slots and a pool of %lld", name, B, (long long)pool);
  if (B > 1 << 28) return set_error(TAAC_ERR_UNSUPPORTED, "%s: at most 2^28 samples", name);  // 32-bit offsets into the slots
  if (static_cast<int64_t>(B) * H > 0x7fffffffLL) return set_error(TAAC_ERR_UNSUPPORTED, "%s: too many workgroups", name);
  if (B == 0 || T == 0) return TAAC_OK;
  if (!q || !k || !v || !log_decay || !beta || !o || (pool > 0 && !state)) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null tensor pointer", name);
  if (!aligned16(state)) return set_error(TAAC_ERR_INVALID_VALUE, "%s: the state must be 16-byte aligned", name);
  StepParams p{};
  p.q = q, p.k = k, p.v = v, p.o = o, p.log_decay = log_decay, p.beta = beta, p.state = state, p.slots = slots, p.lengths = lengths;
  p.pool = pool, p.B = B, p.H = H, p.group = H / key_heads, p.T = T, p.dk = dk, p.dv = dv, p.scale = scale;
  p.gates_f32 = gate_dtype == TAAC_F32, p.slots_int64 = slots_int64 != 0;
  if (int rc = step_strides(name, "q", q_strides, p.qs)) return rc;
  if (int rc = step_strides(name, "k", k_strides, p.ks)) return rc;
  if (int rc = step_strides(name, "v", v_strides, p.vs)) return rc;
  if (int rc = step_strides(name, "o", o_strides, p.os)) return rc;
  if (int rc = step_strides(name, "log_decay", decay_strides, p.gs)) return rc;
  if (int rc = step_strides(name, "beta", beta_strides, p.bs)) return rc;
  hipStream_t s = as_stream(stream);
  if (dtype == TAAC_F32) dispatch_step<float>(p, s);
  if (dtype == TAAC_BF16) dispatch_step<bf16_t>(p, s);
  if (dtype == TAAC_F16) dispatch_step<f16_t>(p, s);
  return check_launch(name);
}
