// Pieces shared by the kernels of the gated delta rule (delta_solo.hip, delta_team.hip, delta_grads.hip).
//
// Per sample and value head, with a_t = exp(g_t), the state S [key_dim, value_dim] follows
//   N_t = v_t - (a_t S)^T k_t,   S <- a_t S + k_t (beta_t N_t)^T,   o_t = scale S^T q_t.
// Over a chunk of 64 tokens with G_i = g_1 + .. + g_i, Gam_ij = exp(G_i - G_j) and A_ij = Gam_ij (k_i . k_j) beta_j for i > j:
//   X = V - diag(e^G) K S,   (I + A) N = X,   O = scale (diag(e^G) Q S + (Gam * Q K^T * beta) N),
//   S' = e^{G_64} S + (beta e^{G_64 - G} K)^T N.
// The inverse of the unit triangular I + A is written I - M; M and the score matrix P do not depend on the state.
// Backward, with dS' the gradient of the state behind a chunk (P holds scale, Gam and beta of its column),
//   beta dU = diag(beta e^{G_64 - G}) K dS' + P^T dO,   dX = beta dU - M^T (beta dU) = dV,
//   dS = e^{G_64} dS' + Q^T (scale e^G dO) - K^T (e^G dX)
// is a recurrence like the forward's, backwards, column by column of the values. It keeps dX and dS' of every chunk, from which the other
// gradients are made chunk by chunk.
//
// All products run on v_mfma_f32_16x16x32_bf16. With lane = (l16 = lane % 16, grp = lane / 16) its operands hold row (or column)
// l16 and 8 values of the contraction, its result column l16 and rows 4 grp .. 4 grp + 3. The contraction may be walked in any
// order that both operands share, and two results (16 rows each) are an operand of the next product as they stand if element e of
// group grp stands for row 4 grp + e of the first result for e < 4, of the second for e >= 4: a chain X -> N -> S' -> next X never
// leaves the registers. Over tokens the two results are tokens 0 .. 15 and 16 .. 31 of a block of 32. Over key features an operand
// holds 8 neighbours of a row of memory, feature 8 grp + e of a block of 32, so row 4 g + r of result a of the state is feature
// 32 (a / 2) + 8 g + 4 (a % 2) + r (state_row).
//
// Precision: q, k, v are bf16 and exact operands. What reaches the state (S itself, X, M, and what is added to S) is fp32 and enters a product
// with all 24 bits, as hi + mid + lo of bf16: three matrix instructions where one factor is exact, six where none is (the products whose parts
// together stand 24 bits below the first are left out); or M and X in fp32 products. The state behind a history is then as near 64 bits as in a
// plain fp32 evaluation, 0.8e-7 to 2.5e-7 of its norm against 0.8e-7 to 3e-7 (all four in hi + lo: 2.8e-6, S alone where decays are slow: 1.3e-6).
// What only meets outputs enters as hi + lo (16 bits): S, N and P for O (of wide heads P once rounded, see the blocks below), and the backward's
// recurrence, whose results are bf16.
// Cumulative decays are summed in 64 bits and kept as pairs, so that G_i - G_j of a fast decaying head keeps fp32 precision.
#pragma once

#include "common.h"

namespace taac {

struct DeltaParams {
  const bf16_t* q;
  const bf16_t* k;
  const bf16_t* v;
  bf16_t* o;
  const void* log_decay;
  const void* beta;
  const int32_t* lengths;    // [B] or null: every sample has T tokens
  const float* state_in;     // [B, H, dk, dv] or null: zeros
  float* state_out;          // [B, H, dk, dv] or null
  bf16_t* chunk_states;      // [B, H, chunks, dv, dk] or null: the state in front of every chunk, transposed
  bf16_t* misses;            // [B, H, T, dv] or null: N
  bf16_t* misses_low;        // [B, H, T, dv]: what the rounding of N left
  uint8_t* blocks;           // [B, H, chunks] blocks in memory (the form for few heads)
  // backward
  const bf16_t* grad_o;
  bf16_t* grad_q;
  bf16_t* grad_k;
  bf16_t* grad_v;            // also dX, which the last kernel reads
  void* grad_decay;
  void* grad_beta;
  bf16_t* grad_states;       // [B, H, chunks, dv, dk]: the gradient of the state behind every chunk, transposed
  int64_t dos[3], dqs[3], dks[3], dvs[3], dgs[3], dbs[3];
  // element strides of (batch, head, token)
  int64_t qs[3], ks[3], vs[3], os[3], gs[3], bs[3];
  int32_t B, H, group, T, dk, dv, chunks;  // group: value heads per key head
  int32_t gates_f32;
  float scale;
};

// The two forms of the recurrence, forward (o, the last state; chunk_states and misses where they are wanted) and backward (grad_v,
// grad_states): with the chunks' blocks in p.blocks (delta_team.hip), and for heads of at most 64 key features without (delta_solo.hip).
int delta_team(const char* name, const DeltaParams& p, bool back, hipStream_t s);
int delta_solo(const char* name, const DeltaParams& p, bool back, hipStream_t s);
// The second half of the backward (delta_grads.hip).
int delta_grads(const char* name, const DeltaParams& p, hipStream_t s);

namespace {

constexpr int kChunk = 64;
constexpr int kFrag = 1024;              // bytes of one operand fragment of a wavefront
// A block in memory: the tokens' factors, M in three parts, P, and what the rounding of P left (the backward, whose M has two parts, has that in the
// place of the third). The forward of wide heads has P rounded once: there that leaves outputs 2.3e-3 from 64 bits, of which 1.7e-3 is their own
// rounding, and six fragments more a block take 2 x 16 heads x 8192 tokens, 128 wide, from 255 to 280 us. Of narrow heads, where pairs within a chunk
// make more of an output, it would be up to 2.5e-3.
constexpr int kBlockRows = 0, kBlockM = 640, kBlockMid = kBlockM + 6 * kFrag, kBlockLow = kBlockM + 12 * kFrag, kBlockP = kBlockM + 18 * kFrag,
              kBlockPLow = kBlockM + 24 * kFrag;
__host__ __device__ constexpr bool low_scores(int dk) { return dk <= 64; }
__host__ __device__ constexpr int block_bytes(int dk) { return kBlockM + (low_scores(dk) ? 30 : 24) * kFrag; }
// the floats of a block: e^G, beta e^(G_64 - G), e^G_64 (then e^ of the second and third tile's own decays)
constexpr int kRowGrown = 0, kRowKeep = 64, kRowTotal = 128, kRowFloats = 144;
static_assert(kRowFloats * 4 <= kBlockM);
// floats that only the maker of a block needs: G as a pair, beta; e^(G - G in front of the tile of 16), e^(G behind the tile - G), that times beta
constexpr int kTempHi = 0, kTempLow = 64, kTempBeta = 128, kTempIn = 192, kTempOut = 256, kTempOutBeta = 320, kTempFloats = 384;
// Scratch for the diagonal blocks: rows of 20 floats, blocks 16 banks apart.
constexpr int kScratchRow = 20, kScratchBlock = 16 * kScratchRow + 16, kScratchFloats = 4 * kScratchBlock;

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// LDS written by some lanes of a wavefront and read by others: the operations of a wavefront complete in order; this keeps the
// compiler from reordering them.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Two values to bf16 in one instruction; and what that left of them.
__device__ __forceinline__ uint32_t round2(float a, float b) {
  typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2;
  typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t rounded) {
  return round2(a - __builtin_bit_cast(float, rounded << 16), b - __builtin_bit_cast(float, rounded & 0xffff0000u));
}
__device__ __forceinline__ u32x2 round4(const f32x4& v) { return u32x2{round2(v[0], v[1]), round2(v[2], v[3])}; }
__device__ __forceinline__ u32x2 rest4(const f32x4& v, const u32x2& r) { return u32x2{rest2(v[0], v[1], r[0]), rest2(v[2], v[3], r[1])}; }
__device__ __forceinline__ void split(const f32x4& a, const f32x4& b, bf16x8& hi, bf16x8& lo) {
  const u32x2 ha = round4(a), hb = round4(b), la = rest4(a, ha), lb = rest4(b, hb);
  hi = __builtin_bit_cast(bf16x8, (u32x4{ha[0], ha[1], hb[0], hb[1]}));
  lo = __builtin_bit_cast(bf16x8, (u32x4{la[0], la[1], lb[0], lb[1]}));
}
// In three parts, which are all of a float's 24 bits.
__device__ __forceinline__ f32x4 left4(const f32x4& v, const u32x2& r) {
  return f32x4{v[0] - __builtin_bit_cast(float, r[0] << 16), v[1] - __builtin_bit_cast(float, r[0] & 0xffff0000u),
               v[2] - __builtin_bit_cast(float, r[1] << 16), v[3] - __builtin_bit_cast(float, r[1] & 0xffff0000u)};
}
__device__ __forceinline__ void split3(const f32x4& a, const f32x4& b, bf16x8& hi, bf16x8& mid, bf16x8& lo) {
  const u32x2 ha = round4(a), hb = round4(b);
  const f32x4 da = left4(a, ha), db = left4(b, hb);
  const u32x2 ma = round4(da), mb = round4(db), la = rest4(da, ma), lb = rest4(db, mb);
  hi = __builtin_bit_cast(bf16x8, (u32x4{ha[0], ha[1], hb[0], hb[1]}));
  mid = __builtin_bit_cast(bf16x8, (u32x4{ma[0], ma[1], mb[0], mb[1]}));
  lo = __builtin_bit_cast(bf16x8, (u32x4{la[0], la[1], lb[0], lb[1]}));
}
__device__ __forceinline__ bf16x8 round8(const f32x4& a, const f32x4& b) {
  const u32x2 ha = round4(a), hb = round4(b);
  return __builtin_bit_cast(bf16x8, (u32x4{ha[0], ha[1], hb[0], hb[1]}));
}
__device__ __forceinline__ f32x4 zero4() { return f32x4{0.f, 0.f, 0.f, 0.f}; }
__device__ __forceinline__ bf16x8 zero8() {
  const u32x4 z = {0u, 0u, 0u, 0u};
  return __builtin_bit_cast(bf16x8, z);
}

// Reads and writes through a buffer descriptor: bytes at or beyond its end read as zero and are not written, so that rows behind the last
// token need neither a branch nor a mask, and a wait for one read counts everything requested since. kNowhere: an offset behind every end (64
// rows of less than 2^24 elements end below it), so also for features or columns that there are not.
typedef __amdgpu_buffer_rsrc_t Buffer;
constexpr uint32_t kNowhere = 0x80000000u;
__device__ __forceinline__ Buffer buffer_of(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, static_cast<int>(bytes), 0x00027000);
}
// n rows of `width` elements, ld elements apart (at least width)
__device__ __forceinline__ Buffer rows_buffer(const bf16_t* base, int64_t ld, int n, int width) {
  return buffer_of(base, n > 0 ? static_cast<uint32_t>((n - 1) * ld + width) * 2 : 0);
}
// off: of the lane; further: the same for all lanes.
__device__ __forceinline__ bf16x8 read8(Buffer b, uint32_t off, uint32_t further = 0) {
  return __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(b, off, further, 0));
}
__device__ __forceinline__ f32x4 read_floats(Buffer b, uint32_t off, uint32_t further = 0) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(b, off, further, 0));
}
__device__ __forceinline__ u32x2 read4(Buffer b, uint32_t off) { return __builtin_amdgcn_raw_buffer_load_b64(b, off, 0, 0); }
__device__ __forceinline__ float read_float(Buffer b, uint32_t off, uint32_t further = 0) {
  return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(b, off, further, 0));
}
__device__ __forceinline__ void write4(Buffer b, uint32_t off, const u32x2& v) { __builtin_amdgcn_raw_buffer_store_b64(v, b, off, 0, 0); }
__device__ __forceinline__ void write8(Buffer b, uint32_t off, const bf16x8& v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), b, off, 0, 0);
}
__device__ __forceinline__ uint32_t read1(Buffer b, uint32_t off) {
  return static_cast<uint16_t>(__builtin_amdgcn_raw_buffer_load_b16(b, off, 0, 0));
}

__device__ __forceinline__ int state_row(int a, int m) { return 32 * (a / 2) + 8 * (m / 4) + 4 * (a % 2) + m % 4; }

// Tiles of 64 token rows in LDS. Rows are 16 bytes longer than their contents, which puts the 16 rows of a read on different banks.
template <int WIDTH>
struct Tile {
  static constexpr int STRIDE = WIDTH + 8;  // elements
  static constexpr int BYTES = kChunk * STRIDE * 2;
  // ROWS rows of memory (n of them valid, `width` valid features) on their way into LDS by THREADS threads: requested for several tiles before any of
  // them is stored
  template <int ROWS, int THREADS>
  struct Piece {
    static constexpr int PIECES = WIDTH / 8, COUNT = (ROWS * PIECES + THREADS - 1) / THREADS;
    bf16x8 v[COUNT];
    __device__ __forceinline__ void load(const bf16_t* src, int64_t ld, int n, int width, int tid) {
      static_assert(THREADS % PIECES == 0);
      const Buffer rows = rows_buffer(src, ld, n, width);
      const int row = tid / PIECES, piece = tid % PIECES;
      const uint32_t pitch = static_cast<uint32_t>(ld) * 2, off = piece * 8 < width ? row * pitch + piece * 16 : kNowhere;
#pragma unroll
      for (int i = 0; i < COUNT; ++i) v[i] = read8(rows, off + i * (THREADS / PIECES) * pitch);
    }
    // the sum of the products of this lane's elements with those of another piece
    __device__ __forceinline__ float dot(const Piece& other) const {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < COUNT; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(static_cast<float>(v[i][e]), static_cast<float>(other.v[i][e]), sum);
      return sum;
    }
    // PAIRED: row 8 g + e of a block of 32 goes to row 4 g + e (e < 4) or 12 + 4 g + e, so that a keys_frag() over the rows has them in order
    template <bool PAIRED = false>
    __device__ __forceinline__ void store(bf16_t* dst, int tid) const {
#pragma unroll
      for (int i = 0; i < COUNT; ++i) {
        int row = (tid + i * THREADS) / PIECES;
        const int piece = (tid + i * THREADS) % PIECES;
        if (row >= ROWS) continue;
        if (PAIRED) row = (row & ~31) + (row & 4) * 4 + ((row & 24) >> 1) + (row & 3);
        *reinterpret_cast<bf16x8*>(dst + row * STRIDE + piece * 8) = v[i];
      }
    }
  };
  static __device__ __forceinline__ bf16x8 row(const bf16_t* tile, int row, int kb, int grp) {
    return *reinterpret_cast<const bf16x8*>(tile + row * STRIDE + kb * 32 + grp * 8);
  }
  // Transposed reads: lane 4 e + q of a group of 16 gives the address of 8 bytes (four features) of token e, lane j receives element j % 4 of
  // what lanes 4 e + j / 4 gave. Tokens token0 + 4 grp .. of feature 16 a + l16 (values), of feature state_row(a, l16) (key features).
  static __device__ __forceinline__ bf16x4 read_tr(const bf16_t* at) {
    typedef __attribute__((address_space(3))) bf16x4 lds_vec;
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_vec*)(at));
  }
  static __device__ __forceinline__ bf16x4 values(const bf16_t* tile, int token0, int a, int l16, int grp) {
    return read_tr(tile + (token0 + 4 * grp + l16 / 4) * STRIDE + a * 16 + (l16 % 4) * 4);
  }
  static __device__ __forceinline__ bf16x4 keys(const bf16_t* tile, int token0, int a, int l16, int grp) {
    return read_tr(tile + (token0 + 4 * grp + l16 / 4) * STRIDE + (a / 2) * 32 + (l16 % 4) * 8 + (a % 2) * 4);
  }
  static __device__ __forceinline__ bf16x8 join(const bf16x4& lo, const bf16x4& hi) {
    bf16x8 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      r[e] = lo[e];
      r[4 + e] = hi[e];
    }
    return r;
  }
  // operand fragments over the tokens of block tk
  static __device__ __forceinline__ bf16x8 values_frag(const bf16_t* tile, int tk, int a, int l16, int grp) {
    return join(values(tile, 32 * tk, a, l16, grp), values(tile, 32 * tk + 16, a, l16, grp));
  }
  static __device__ __forceinline__ bf16x8 keys_frag(const bf16_t* tile, int tk, int a, int l16, int grp) {
    return join(keys(tile, 32 * tk, a, l16, grp), keys(tile, 32 * tk + 16, a, l16, grp));
  }
};

// 16 x 16 fp32 products on v_mfma_f32_16x16x4_f32, contraction index 4 grp + step. A matrix Y is held "by rows" (lane: row l16, columns
// 4 grp ..) or "by columns" (lane: column l16, rows 4 grp ..).
__device__ __forceinline__ f32x4 mul_cols(const f32x4& x_rows, const f32x4& y_cols, f32x4 acc) {  // X Y by columns
#pragma unroll
  for (int r = 0; r < 4; ++r) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x_rows[r], y_cols[r], acc, 0, 0, 0);
  return acc;
}
__device__ __forceinline__ f32x4 mul_rows(const f32x4& x_rows, const f32x4& y_cols, f32x4 acc) {  // X Y by rows
#pragma unroll
  for (int r = 0; r < 4; ++r) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(y_cols[r], x_rows[r], acc, 0, 0, 0);
  return acc;
}

// M of the four diagonal blocks of 16 in scratch, in the place of A, all four at once: M_ic = A_ic - sum over c < j < i of A_ij M_jc, a column
// c per lane. Every lane of the wavefront has written its part of A before a wave_sync().
__device__ __forceinline__ void solve_diagonal(float* scratch, int lane) {
  float* mine = scratch + lane / 16 * kScratchBlock;
  const int l16 = lane % 16;
  float m[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float acc = mine[i * kScratchRow + l16];
#pragma unroll
    for (int j4 = 0; j4 * 4 < i; ++j4) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(mine + i * kScratchRow + 4 * j4);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * j4 + e < i) acc = fmaf(-a[e], m[4 * j4 + e], acc);
    }
    m[i] = acc;
  }
  wave_sync();
#pragma unroll
  for (int i = 0; i < 16; ++i) mine[i * kScratchRow + l16] = m[i];
  wave_sync();
}

// The gates of a lane's token as the bits that the reads bring, by halves: a branch between fp32 and bf16 would await each.
struct GateBits {
  uint32_t g[2], beta[2];
  // token `lane` of the n behind token0 (n may be 0: nothing is used then)
  __device__ __forceinline__ void request(const DeltaParams& p, int b, int h, int64_t token0, int n, int lane) {
    const int64_t token = lane < n ? token0 + lane : 0;
    const int64_t at_g = b * p.gs[0] + h * p.gs[1] + token * p.gs[2], at_beta = b * p.bs[0] + h * p.bs[1] + token * p.bs[2];
    const uint16_t* from_g = static_cast<const uint16_t*>(p.log_decay) + (at_g << p.gates_f32);
    const uint16_t* from_beta = static_cast<const uint16_t*>(p.beta) + (at_beta << p.gates_f32);
    g[0] = from_g[0], g[1] = from_g[p.gates_f32];
    beta[0] = from_beta[0], beta[1] = from_beta[p.gates_f32];
  }
  static __device__ __forceinline__ float value(const uint32_t (&bits)[2], int f32, bool live) {
    const float v = __builtin_bit_cast(float, bits[1] << 16 | (f32 ? bits[0] : 0));  // a bf16 is the upper half of a float
    return live ? v : 0.f;
  }
  // A decay in powers of two; an exponent below -1e5 is a decay of zero, and stays finite in the sums.
  __device__ __forceinline__ double decay(const DeltaParams& p, bool live) const {
    const float v = value(g, p.gates_f32, live);
    return static_cast<double>(v < -1e5f ? -1e5f : v) * 1.4426950408889634;
  }
  __device__ __forceinline__ float step(const DeltaParams& p, bool live) const { return value(beta, p.gates_f32, live); }
};

// The factors of a chunk's n tokens, by one wavefront. last_minus: null, or receives e^(G_64 - G) of every token.
__device__ __forceinline__ void chunk_rows(const DeltaParams& p, const GateBits& gates, int n, float* rows, float* temp,
                                           float* last_minus = nullptr) {
  const int lane = threadIdx.x % kWave;
  double total = gates.decay(p, lane < n);
  const float beta = gates.step(p, lane < n);
#pragma unroll
  for (int off = 1; off < kWave; off *= 2) {
    const double up = __shfl_up(total, off, kWave);
    if (lane >= off) total += up;
  }
  const double last = __shfl(total, kWave - 1, kWave);
  const double behind = __shfl(total, lane | 15, kWave);
  const double before = __shfl(total, lane < 16 ? 0 : (lane & ~15) - 1, kWave);
  const float hi = static_cast<float>(total);
  temp[kTempHi + lane] = hi;
  temp[kTempLow + lane] = static_cast<float>(total - static_cast<double>(hi));
  temp[kTempBeta + lane] = beta;
  temp[kTempIn + lane] = __builtin_amdgcn_exp2f(static_cast<float>(lane < 16 ? total : total - before));
  const float out = __builtin_amdgcn_exp2f(static_cast<float>(behind - total));
  temp[kTempOut + lane] = out;
  temp[kTempOutBeta + lane] = out * beta;
  rows[kRowGrown + lane] = __builtin_amdgcn_exp2f(hi);
  const float left = __builtin_amdgcn_exp2f(static_cast<float>(last - total));
  rows[kRowKeep + lane] = beta * left;
  if (last_minus != nullptr) last_minus[lane] = left;
  if (lane == 63) rows[kRowTotal] = __builtin_amdgcn_exp2f(hi);
  if (lane == 31 || lane == 47) rows[kRowTotal + lane / 16] = __builtin_amdgcn_exp2f(static_cast<float>(total - before));
}

// e^(G in front of tile ti - G behind tile tj), ti > tj: the decay of the whole tiles between them. Gam of a token i of tile ti and a token
// j of tile tj is this times In_i times Out_j, one exponential per token instead of one per pair; three factors of at most one where states decay.
__device__ __forceinline__ float tiles_between(const float* rows, int ti, int tj) {
  const float second = rows[kRowTotal + 1], third = rows[kRowTotal + 2];
  return ti - tj < 2 ? 1.f : (ti - tj == 3 ? second * third : (tj == 0 ? second : third));
}

}  // namespace
}  // namespace taac
