// Quantising keys and values on their way into a pool of pages, and reading them back (the format: kv_cache.h).
//
// Bound by HBM, or by latency for a few tokens: a value is read once and leaves as 4 or 8 bits, or the other way round, and needs a maximum over 32 and a
// conversion.
//
// Measured: 512 histories of up to 512 tokens, 8 heads of 32 features in 4 bits: written in 55 us (183 MB, 3.3 TB/s), read in 54 (301 MB with the zeros, 5.6). 16 x 8000 tokens of 8
// heads of 128 in 8 bits: 165 us (4.8 TB/s) and 154 (5.2). Writing was 58 and 180 when numbers became fp32 first and lanes exchanged through LDS: 281 and 740 vector
// instructions of a wavefront, now 222 and 549. Two records of a wavefront at a time (122 us for both directions of the first, 115 then with one), the heads of a chunk in
// turn at one address (122 to 139), more and fewer wavefronts were slower.
#include "kv_cache.h"

namespace taac {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMostGroups = 1 << 14;  // of four chunks at a time: a wavefront asks for its next chunk's place while the rows of one are on their way
// Rows of tokens one by one below, chunks from here on: 512 samples of 8 heads of 32 features in 4 bits, written and read, take 11 : 15 us with 8 tokens, 17 : 15 with 16;
// 64 samples of 128 features in 8 bits 9 : 11 and 12 : 11.
constexpr int kChunksFrom = 12;

constexpr int64_t kMostRows = 1 << 27;  // of a launch row by row, whose numbers have 32 bits

struct CacheParams {
  KvPool pool;
  const void* k;
  const void* v;
  void* k_out;
  void* v_out;
  const void* starts;      // [B] int32 or int64 or null: zeros
  const int32_t* lengths;  // [B] or null: T
  int64_t ks[3], vs[3];    // element strides of (batch, head, token)
  int64_t rows;            // B * T * heads
  int64_t units;           // B * chunks * heads
  Divisor by_heads, by_chunks, by_tokens;
  int32_t T, chunks, starts_int64;
};

typedef __attribute__((__vector_size__(2 * sizeof(short)))) short s16x2;
typedef __attribute__((__vector_size__(2 * sizeof(unsigned short)))) unsigned short u16x2;
typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
typedef __attribute__((__vector_size__(2 * sizeof(_Float16)))) _Float16 f16x2;
typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2;

// Eight neighbouring features as they lie in memory.
template <typename T>
struct Eight {
  static constexpr int WORDS = 2 * sizeof(T);
  uint32_t w[WORDS];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < WORDS / 4; ++i) {
      const u32x4 v = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[4 * i + j] = v[j];
    }
  }
  // The largest magnitude, found among the bits without the sign, whose order is that of the numbers, then infinity, then NaN. finite: none of the last two.
  __device__ __forceinline__ float most(bool& finite) const {
    if constexpr (sizeof(T) == 4) {
      uint32_t m = w[0] & 0x7fffffffu;
#pragma unroll
      for (int i = 1; i < WORDS; ++i) m = max(m, w[i] & 0x7fffffffu);
      finite &= m < 0x7f800000u;
      return __builtin_bit_cast(float, m);
    } else {
      u16x2 m = __builtin_bit_cast(u16x2, w[0] & 0x7fff7fffu);
#pragma unroll
      for (int i = 1; i < WORDS; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
      const uint32_t both = __builtin_bit_cast(uint32_t, m), top = max(both & 0xffffu, both >> 16);
      if constexpr (__is_same(T, bf16_t)) {
        finite &= top < 0x7f80u;
        return __builtin_bit_cast(float, top << 16);
      } else {
        finite &= top < 0x7c00u;
        return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(top)));
      }
    }
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, static_cast<uint32_t>(w[i]));
    else if constexpr (__is_same(T, bf16_t)) return __builtin_bit_cast(float, i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i / 2] >> (16 * (i % 2)))));
  }
};
template <typename T>
__device__ __forceinline__ void store_eight(T* p, const float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<f32x4*>(p)[0] = f32x4{f[0], f[1], f[2], f[3]};
    reinterpret_cast<f32x4*>(p)[1] = f32x4{f[4], f[5], f[6], f[7]};
  } else {
    typename Vec8<T>::type a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = static_cast<T>(f[i]);
    *reinterpret_cast<typename Vec8<T>::type*>(p) = a;
  }
}

// The value of lane l ^ XOR, by the operands' own lane patterns: quads, sixteen lanes turned by eight, and for four eight lanes mirrored, then their quads.
template <int XOR>
__device__ __forceinline__ uint32_t across(uint32_t v) {
  static_assert(XOR == 1 || XOR == 2 || XOR == 4 || XOR == 8);
  constexpr int PATTERN = XOR == 1 ? 0xb1 : XOR == 2 ? 0x4e : XOR == 4 ? 0x141 : 0x128;
  const uint32_t r = __builtin_amdgcn_update_dpp(v, v, PATTERN, 0xf, 0xf, false);
  return XOR == 4 ? __builtin_amdgcn_update_dpp(r, r, 0x1b, 0xf, 0xf, false) : r;
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __builtin_bit_cast(float, across<1>(__builtin_bit_cast(uint32_t, v))));
  return fmaxf(v, __builtin_bit_cast(float, across<2>(__builtin_bit_cast(uint32_t, v))));
}

// The least power of two 2^e with max < 7 2^e (464 2^e), as e + 127, for a finite max. The carry out of the fraction is the step to the next power: 7 and 464
// are 1.75 and 1.8125 of one. Kept between 2^-117, under which the smallest code would be subnormal, and what keeps the largest code finite.
template <int BITS>
constexpr int kMostScale = BITS == 4 ? 252 : 246;
template <int BITS>
__device__ __forceinline__ int scale_byte(float most) {
  const uint32_t up = BITS == 4 ? 0x200000u : 0x180000u;
  const int e = static_cast<int>((__builtin_bit_cast(uint32_t, most) + up) >> 23) - (BITS == 4 ? 2 : 8);
  return min(max(e, 10), kMostScale<BITS>);
}

// Codes of eight values in order: one word of 4 bits, two of 8.
template <int BITS>
struct Codes {
  uint32_t w[BITS / 4];
};
// Two features, x / scale, to the nearest code, in one instruction from the type that they have.
template <int BITS, int I, typename T>
__device__ __forceinline__ void two_codes(Codes<BITS>& c, const Eight<T>& x, float scale) {
  if constexpr (BITS == 4) {
    if constexpr (sizeof(T) == 4) {
      c.w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c.w[0], x.at(2 * I), x.at(2 * I + 1), scale, I);
    } else if constexpr (__is_same(T, bf16_t)) {
      c.w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c.w[0], __builtin_bit_cast(bf16x2, static_cast<uint32_t>(x.w[I])), scale, I);
    } else {
      c.w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c.w[0], __builtin_bit_cast(f16x2, static_cast<uint32_t>(x.w[I])), scale, I);
    }
  } else {
    s16x2 w = __builtin_bit_cast(s16x2, static_cast<uint32_t>(c.w[I / 2]));
    if constexpr (sizeof(T) == 4) w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x.at(2 * I), x.at(2 * I + 1), scale, I % 2 != 0);
    else if constexpr (__is_same(T, bf16_t)) w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2, static_cast<uint32_t>(x.w[I])), scale, I % 2 != 0);
    else w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, __builtin_bit_cast(f16x2, static_cast<uint32_t>(x.w[I])), scale, I % 2 != 0);
    c.w[I / 2] = __builtin_bit_cast(uint32_t, w);
  }
}
// Codes of eight features under the scale 2^e that they share, e + 127 = byte.
template <int BITS, typename T>
__device__ __forceinline__ Codes<BITS> encode(const Eight<T>& x, int byte) {
  const float scale = kv_scale(byte);
  Codes<BITS> c;
#pragma unroll
  for (int i = 0; i < BITS / 4; ++i) c.w[i] = 0;
  if (__is_same(T, f16_t) || byte < kMostScale<BITS>) {
    two_codes<BITS, 0>(c, x, scale), two_codes<BITS, 1>(c, x, scale), two_codes<BITS, 2>(c, x, scale), two_codes<BITS, 3>(c, x, scale);
  } else {  // under the largest scale a number may be beyond the largest code
    const float end = (BITS == 4 ? 6.f : 448.f) * scale;
    Eight<float> f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f.w[i] = __builtin_bit_cast(uint32_t, fminf(fmaxf(x.at(i), -end), end));
    two_codes<BITS, 0>(c, f, scale), two_codes<BITS, 1>(c, f, scale), two_codes<BITS, 2>(c, f, scale), two_codes<BITS, 3>(c, f, scale);
  }
  return c;
}
template <int BITS>
__device__ __forceinline__ void decode(const Codes<BITS>& c, float scale, float (&f)[8]) {
  f32x2 p[4];
  if constexpr (BITS == 4) {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.w[0], scale, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.w[0], scale, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.w[0], scale, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.w[0], scale, 3);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      p[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.w[i], scale, false);
      p[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.w[i], scale, true);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) f[2 * i] = p[i][0], f[2 * i + 1] = p[i][1];
}

// ---- a few tokens: row by row --------------------------------------------------------------------------------------

// A row (sample, token, head) and where it belongs: D / 8 lanes, eight features each.
struct Row {
  int64_t b, position;
  int t, h;
  bool there;
  __device__ __forceinline__ Row(const CacheParams& p, int row) {
    const int token = p.by_heads.over(row), sample = p.by_tokens.over(token);
    h = row - token * p.pool.heads;
    t = token - sample * p.T;
    b = sample;
    there = p.lengths == nullptr || t < p.lengths[b];
    const int64_t start = p.starts == nullptr ? 0 : (p.starts_int64 ? static_cast<const int64_t*>(p.starts)[b] : static_cast<const int32_t*>(p.starts)[b]);
    there &= start >= 0 && start < (int64_t{1} << 40);
    position = start + t;
  }
};

template <typename T, int D, int BITS>
__global__ __launch_bounds__(kThreads) void kv_write_rows_kernel(const CacheParams p) {
  constexpr int LANES = D / 8, ROWS = kThreads / LANES, BLOCKS = D / kKvBlock;
  const int row = blockIdx.x * ROWS + threadIdx.x / LANES;
  if (row >= p.rows) return;
  const int s = threadIdx.x % LANES, block = s / 4, sub = s % 4;
  const Row at(p, row);
  const int64_t page = at.there ? kv_page(p.pool, at.b, at.position >> p.pool.page_shift) : -1;
  if (page < 0) return;
  Eight<T> k, v;
  k.load(static_cast<const T*>(p.k) + at.b * p.ks[0] + at.h * p.ks[1] + at.t * p.ks[2] + 8 * s);
  v.load(static_cast<const T*>(p.v) + at.b * p.vs[0] + at.h * p.vs[1] + at.t * p.vs[2] + 8 * s);
  const int in_page = static_cast<int>(at.position & ((1 << p.pool.page_shift) - 1)), token = in_page % kKvChunk;
  uint8_t* record = p.pool.data + kv_record(p.pool, page, at.h, in_page / kKvChunk, kv_record_bytes(D, BITS));
  bool finite = true;
  const float k_most = quad_max(k.most(finite)), v_most = quad_max(v.most(finite));
  int bad = !finite;
#pragma unroll
  for (int off = LANES / 2; off > 0; off /= 2) bad |= __shfl_xor(bad, off, kWave);
  int k_scale = scale_byte<BITS>(k_most), v_scale = scale_byte<BITS>(v_most);
  if (bad) {
    k_scale = v_scale = 127;
    k.clear(), v.clear();
  }
  const Codes<BITS> kc = encode<BITS>(k, k_scale), vc = encode<BITS>(v, v_scale);
  if (bad) k_scale = kKvNotFinite;
  uint8_t* keys = record + block * (kKvChunk * kKvBlock * BITS / 8) + token * (kKvBlock * BITS / 8) + sub * BITS;
  if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(keys) = kc.w[0];
  else *reinterpret_cast<u32x2*>(keys) = u32x2{kc.w[0], kc.w[1]};
  uint8_t* values = record + kv_value_at(D, BITS);
  const int group = token / 4, of4 = token % 4;
  if constexpr (BITS == 4) {
    const uint32_t mine = vc.w[0], other = across<2>(mine);
    if (sub < 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        values[(((8 * sub + i) * 4 + group) * BLOCKS + block) * 4 + of4] = static_cast<uint8_t>((mine >> (4 * i) & 15u) | (other >> (4 * i) & 15u) << 4);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      values[(((8 * (sub % 2) + i) * 4 + group) * BLOCKS + block) * 8 + of4 * 2 + sub / 2] = static_cast<uint8_t>(vc.w[i / 4] >> (8 * (i % 4)));
  }
  if (sub == 0) {
    record[kv_key_scale_at(D, BITS) + token * BLOCKS + block] = static_cast<uint8_t>(k_scale);
    record[kv_value_scale_at(D, BITS) + (group * BLOCKS + block) * 4 + of4] = static_cast<uint8_t>(v_scale);
  }
}

template <typename T, int D, int BITS>
__global__ __launch_bounds__(kThreads) void kv_read_rows_kernel(const CacheParams p) {
  constexpr int LANES = D / 8, ROWS = kThreads / LANES, BLOCKS = D / kKvBlock;
  const int row = blockIdx.x * ROWS + threadIdx.x / LANES;
  if (row >= p.rows) return;
  const int s = threadIdx.x % LANES, block = s / 4, sub = s % 4;
  const Row at(p, row);
  const int64_t page = at.there ? kv_page(p.pool, at.b, at.position >> p.pool.page_shift) : -1;
  float k[8], v[8];
  if (page < 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = v[i] = 0.f;
  } else {
    const int in_page = static_cast<int>(at.position & ((1 << p.pool.page_shift) - 1)), token = in_page % kKvChunk;
    const uint8_t* record = p.pool.data + kv_record(p.pool, page, at.h, in_page / kKvChunk, kv_record_bytes(D, BITS));
    const uint8_t* keys = record + block * (kKvChunk * kKvBlock * BITS / 8) + token * (kKvBlock * BITS / 8) + sub * BITS;
    Codes<BITS> kc, vc;
    if constexpr (BITS == 4) {
      kc.w[0] = *reinterpret_cast<const uint32_t*>(keys);
    } else {
      const u32x2 w = *reinterpret_cast<const u32x2*>(keys);
      kc.w[0] = w[0], kc.w[1] = w[1];
    }
    const uint8_t* values = record + kv_value_at(D, BITS);
    const int group = token / 4, of4 = token % 4;
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int place = ((8 * (sub % 2) + i) * 4 + group) * BLOCKS + block;
      b[i] = BITS == 4 ? values[place * 4 + of4] >> (4 * (sub / 2)) & 15u : values[place * 8 + of4 * 2 + sub / 2];
    }
#pragma unroll
    for (int j = 0; j < BITS / 4; ++j) {
      vc.w[j] = 0;
#pragma unroll
      for (int i = 0; i < 32 / BITS; ++i) vc.w[j] |= b[j * 4 + i] << (BITS * i);
    }
    const uint32_t k_scale = record[kv_key_scale_at(D, BITS) + token * BLOCKS + block];
    const uint32_t v_scale = k_scale == kKvNotFinite ? kKvNotFinite : record[kv_value_scale_at(D, BITS) + (group * BLOCKS + block) * 4 + of4];
    decode<BITS>(kc, kv_scale(k_scale), k);
    decode<BITS>(vc, kv_scale(v_scale), v);
  }
  store_eight(static_cast<T*>(p.k_out) + at.b * p.ks[0] + at.h * p.ks[1] + at.t * p.ks[2] + 8 * s, k);
  store_eight(static_cast<T*>(p.v_out) + at.b * p.vs[0] + at.h * p.vs[1] + at.t * p.vs[2] + 8 * s, v);
}

// ---- many tokens: chunk by chunk -----------------------------------------------------------------------------------
//
// A wavefront has the sixteen tokens of a record: lane = (token, sub), features 8 sub .. 8 sub + 7 of every block of 32. Keys leave as they lie. Values of four tokens and
// two features turn into a word in two exchanges of lanes, between the sixteens of a block's features and between the tokens of a group, so that all
// of a record is written and read in whole words, side by side.

// One of a call's integers. SCALAR: by a scalar read, which counts apart from a chunk's rows and does not wait for them. For heads of 32 features, whose chunks are
// small, that is a sixth faster (512 ragged histories of 512 tokens, 8 heads, written and read: 124 against 147 us), for wider ones a tenth slower
// (16 x 8000 tokens of 8 heads of 128 in 8 bits: 361 against 324).
template <bool SCALAR>
__device__ __forceinline__ int64_t integer_at(const void* p, int64_t i, bool wide) {
  if constexpr (SCALAR) {
    typedef const __attribute__((address_space(4))) int32_t* Narrow;
    typedef const __attribute__((address_space(4))) int64_t* Wide;
    return wide ? ((Wide)(reinterpret_cast<uint64_t>(p)))[i] : ((Narrow)(reinterpret_cast<uint64_t>(p)))[i];
  }
  return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// Sample, head and chunk of a wavefront: which of the chunk's tokens are the call's, and which of them there are. The same in all
// lanes.
template <bool SCALAR>
struct Chunk {
  int64_t b;
  int h;
  int t0;               // the call's token that would be the chunk's first
  int first, end;       // tokens first .. end - 1 of the chunk are written (read)
  uint8_t* record;      // null: in no page, or nothing to do there
  Chunk() = default;
  __device__ __forceinline__ Chunk(const CacheParams& p, int64_t unit, int record_bytes) {
    int64_t rest;
    if (p.units < 0x7fffffff) {
      rest = p.by_heads.over(static_cast<int>(unit));
      b = p.by_chunks.over(static_cast<int>(rest));
    } else {
      rest = unit / p.pool.heads;
      b = rest / p.chunks;
    }
    h = static_cast<int>(unit - rest * p.pool.heads);
    int64_t start = p.starts == nullptr ? 0 : integer_at<SCALAR>(p.starts, b, p.starts_int64);
    int n = p.lengths == nullptr ? p.T : min(max(static_cast<int>(integer_at<SCALAR>(p.lengths, b, false)), 0), p.T);
    if (start < 0 || start >= int64_t{1} << 40) start = 0, n = 0;
    const int64_t chunk = (start / kKvChunk) + (rest - b * p.chunks), from = chunk * kKvChunk, behind = start + n - from;
    t0 = static_cast<int>(from - start);
    first = t0 < 0 ? -t0 : 0;
    end = behind < kKvChunk ? static_cast<int>(behind) : kKvChunk;  // not above first: nothing
    const int64_t index = from >> p.pool.page_shift;
    record = nullptr;
    if (first < end && index < p.pool.table_pages) {
      const int64_t page = integer_at<SCALAR>(p.pool.table, b * p.pool.table_stride + index, p.pool.int64);
      if (page >= 0 && page < p.pool.pages)
        record = p.pool.data + kv_record(p.pool, page, h, static_cast<int>(chunk & ((1 << (p.pool.page_shift - 4)) - 1)), record_bytes);
    }
  }
};

// Lanes of four tokens (bits 2 and 3 of the lane) hold four bytes each: byte i of lane j becomes byte j of lane i. Its own inverse.
__device__ __forceinline__ uint32_t turn_bytes(uint32_t w, int token) {
  uint32_t other = across<4>(w);
  w = __builtin_amdgcn_perm(other, w, token & 1 ? 0x03070105u : 0x06020400u);
  other = across<8>(w);
  return __builtin_amdgcn_perm(other, w, token & 2 ? 0x03020706u : 0x05040100u);
}
// The same of four halves of 16 bits.
__device__ __forceinline__ void turn_halves(uint32_t (&w)[2], int token) {
  const uint32_t a = across<4>(w[0]), b = across<4>(w[1]), pick = token & 1 ? 0x03020706u : 0x05040100u;
  const uint32_t x = __builtin_amdgcn_perm(a, w[0], pick), y = __builtin_amdgcn_perm(b, w[1], pick);
  const uint32_t other = across<8>(token & 2 ? x : y);
  w[0] = token & 2 ? other : x;
  w[1] = token & 2 ? y : other;
}

__device__ __forceinline__ uint32_t spread_nibbles(uint32_t x) {  // four in the low half, a byte each
  x = (x | x << 8) & 0x00ff00ffu;
  return (x | x << 4) & 0x0f0f0f0fu;
}
__device__ __forceinline__ uint32_t gather_nibbles(uint32_t x) {
  x = (x | x >> 4) & 0x00ff00ffu;
  return (x | x >> 8) & 0xffffu;
}

// Codes of eight features of a token -> the words of the record that this lane writes: features n = 8 (sub % 2) + 4 (sub / 2) + token % 4 and n + 16, tokens 4 (token / 4) ..
template <int BITS>
__device__ __forceinline__ Codes<BITS> to_record(const Codes<BITS>& c, int token, int sub) {
  Codes<BITS> r;
  if constexpr (BITS == 4) {
    const uint32_t w = c.w[0], other = across<2>(sub < 2 ? w >> 16 : w & 0xffffu);
    r.w[0] = turn_bytes(spread_nibbles(sub < 2 ? w & 0xffffu : other) | spread_nibbles(sub < 2 ? other : w >> 16) << 4, token);
  } else {
    const uint32_t other = across<2>(sub < 2 ? c.w[1] : c.w[0]), low = sub < 2 ? c.w[0] : other, high = sub < 2 ? other : c.w[1];
    r.w[0] = __builtin_amdgcn_perm(high, low, 0x05010400u), r.w[1] = __builtin_amdgcn_perm(high, low, 0x07030602u);
    turn_halves(r.w, token);
  }
  return r;
}
template <int BITS>
__device__ __forceinline__ Codes<BITS> from_record(const Codes<BITS>& c, int token, int sub) {
  Codes<BITS> r;
  if constexpr (BITS == 4) {
    const uint32_t w = turn_bytes(c.w[0], token), low = gather_nibbles(w & 0x0f0f0f0fu), high = gather_nibbles(w >> 4 & 0x0f0f0f0fu);
    const uint32_t other = across<2>(sub < 2 ? high : low);
    r.w[0] = sub < 2 ? low | other << 16 : other | high << 16;
  } else {
    uint32_t w[2] = {c.w[0], c.w[1]};
    turn_halves(w, token);
    const uint32_t low = __builtin_amdgcn_perm(w[1], w[0], 0x06040200u), high = __builtin_amdgcn_perm(w[1], w[0], 0x07050301u);
    const uint32_t other = across<2>(sub < 2 ? high : low);
    r.w[0] = sub < 2 ? low : other, r.w[1] = sub < 2 ? other : high;
  }
  return r;
}

template <int N>
__device__ __forceinline__ void store_words(uint8_t* p, const uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) reinterpret_cast<u32x4*>(p)[i] = u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
  } else if constexpr (N == 2) {
    *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
  } else {
    *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u32x4 v = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[4 * i + j] = v[j];
    }
  } else if constexpr (N == 2) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
    w[0] = v[0], w[1] = v[1];
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

template <typename T, int D, int BITS>
__global__ __launch_bounds__(kThreads) void kv_write_chunks_kernel(const CacheParams p) {
  constexpr int BLOCKS = D / kKvBlock, EACH = BITS / 4;
  constexpr bool SCALAR = D == 32;
  const int lane = threadIdx.x % kWave, token = lane / 4, sub = lane % 4;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / kWave);
  int64_t unit = static_cast<int64_t>(blockIdx.x) * (kThreads / kWave) + (SCALAR ? __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) : threadIdx.x / kWave);
  Chunk<SCALAR> at, next;
  if (unit < p.units) next = Chunk<SCALAR>(p, unit, kv_record_bytes(D, BITS));
  for (; unit < p.units; unit += step) {
    at = next;
    if (at.record == nullptr) {
      if (unit + step < p.units) next = Chunk<SCALAR>(p, unit + step, kv_record_bytes(D, BITS));
      continue;
    }
    const bool there = token >= at.first && token < at.end;
    Eight<T> k[BLOCKS], v[BLOCKS];
    const T* kp = static_cast<const T*>(p.k) + at.b * p.ks[0] + at.h * p.ks[1] + (at.t0 + token) * p.ks[2] + 8 * sub;
    const T* vp = static_cast<const T*>(p.v) + at.b * p.vs[0] + at.h * p.vs[1] + (at.t0 + token) * p.vs[2] + 8 * sub;
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) {
      k[j].clear(), v[j].clear();
      if (there) {
        k[j].load(kp + kKvBlock * j);
        v[j].load(vp + kKvBlock * j);
      }
    }
    if (unit + step < p.units) next = Chunk<SCALAR>(p, unit + step, kv_record_bytes(D, BITS));
    int k_scale[BLOCKS], v_scale[BLOCKS];
    bool finite = true;
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) {
      k_scale[j] = scale_byte<BITS>(quad_max(k[j].most(finite)));
      v_scale[j] = scale_byte<BITS>(quad_max(v[j].most(finite)));
    }
    int bad = !finite;
    bad |= across<1>(bad);
    bad |= across<2>(bad);
    uint32_t values[BLOCKS * EACH];
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) {
      if (bad) {
        k_scale[j] = v_scale[j] = 127;
        k[j].clear(), v[j].clear();
      }
      const Codes<BITS> kc = encode<BITS>(k[j], k_scale[j]), vc = to_record<BITS>(encode<BITS>(v[j], v_scale[j]), token, sub);
      if (bad) k_scale[j] = kKvNotFinite;
      if (there) store_words(at.record + j * (kKvChunk * 4 * BITS) + token * 4 * BITS + sub * BITS, kc.w);
#pragma unroll
      for (int i = 0; i < EACH; ++i) values[j * EACH + i] = vc.w[i];
    }
    const int n = 8 * (sub % 2) + 4 * (sub / 2) + token % 4, group = token / 4;
    uint8_t* to = at.record + kv_value_at(D, BITS) + (n * 4 + group) * BLOCKS * BITS;
    if (4 * group >= at.first && 4 * group + 4 <= at.end) {
      store_words(to, values);
    } else {
#pragma unroll
      for (int j = 0; j < BLOCKS; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (4 * group + e < at.first || 4 * group + e >= at.end) continue;
          if constexpr (BITS == 4) to[j * 4 + e] = static_cast<uint8_t>(values[j] >> (8 * e));
          else *reinterpret_cast<uint16_t*>(to + j * 8 + 2 * e) = static_cast<uint16_t>(values[2 * j + e / 2] >> (16 * (e % 2)));
        }
    }
    if (there && sub == 0) {
#pragma unroll
      for (int j = 0; j < BLOCKS; ++j) {
        at.record[kv_key_scale_at(D, BITS) + token * BLOCKS + j] = static_cast<uint8_t>(k_scale[j]);
        at.record[kv_value_scale_at(D, BITS) + (group * BLOCKS + j) * 4 + token % 4] = static_cast<uint8_t>(v_scale[j]);
      }
    }
  }
}

template <typename T, int D, int BITS>
__global__ __launch_bounds__(kThreads) void kv_read_chunks_kernel(const CacheParams p) {
  constexpr int BLOCKS = D / kKvBlock, EACH = BITS / 4;
  constexpr bool SCALAR = D == 32;
  const int lane = threadIdx.x % kWave, token = lane / 4, sub = lane % 4;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / kWave);
  int64_t unit = static_cast<int64_t>(blockIdx.x) * (kThreads / kWave) + (SCALAR ? __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) : threadIdx.x / kWave);
  Chunk<SCALAR> at, next;
  if (unit < p.units) next = Chunk<SCALAR>(p, unit, kv_record_bytes(D, BITS));
  for (; unit < p.units; unit += step) {
    at = next;
    const bool there = at.record != nullptr && token >= at.first && token < at.end;
    Codes<BITS> keys[BLOCKS];
    uint32_t values[BLOCKS * EACH], k_scale[BLOCKS], v_scale[BLOCKS];
    const int n = 8 * (sub % 2) + 4 * (sub / 2) + token % 4, group = token / 4;
    if (at.record != nullptr) {
#pragma unroll
      for (int j = 0; j < BLOCKS; ++j) {
        load_words(at.record + j * (kKvChunk * 4 * BITS) + token * 4 * BITS + sub * BITS, keys[j].w);
        k_scale[j] = at.record[kv_key_scale_at(D, BITS) + token * BLOCKS + j];
        v_scale[j] = at.record[kv_value_scale_at(D, BITS) + (group * BLOCKS + j) * 4 + token % 4];
      }
      load_words(at.record + kv_value_at(D, BITS) + (n * 4 + group) * BLOCKS * BITS, values);
    }
    if (unit + step < p.units) next = Chunk<SCALAR>(p, unit + step, kv_record_bytes(D, BITS));
    const int t = at.t0 + token;
    T* kp = static_cast<T*>(p.k_out) + at.b * p.ks[0] + at.h * p.ks[1] + t * p.ks[2] + 8 * sub;
    T* vp = static_cast<T*>(p.v_out) + at.b * p.vs[0] + at.h * p.vs[1] + t * p.vs[2] + 8 * sub;
    const bool asked = t >= 0 && t < p.T;
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) {
      float k[8], v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) k[i] = v[i] = 0.f;
      if (at.record != nullptr) {
        Codes<BITS> c;
#pragma unroll
        for (int i = 0; i < EACH; ++i) c.w[i] = values[j * EACH + i];
        c = from_record<BITS>(c, token, sub);
        if (there) {
          decode<BITS>(keys[j], kv_scale(k_scale[j]), k);
          decode<BITS>(c, kv_scale(k_scale[j] == kKvNotFinite ? kKvNotFinite : v_scale[j]), v);
        }
      }
      if (asked) {
        store_eight(kp + kKvBlock * j, k);
        store_eight(vp + kKvBlock * j, v);
      }
    }
  }
}

template <typename T, int D, int BITS>
void launch_cache(const CacheParams& p, bool write, hipStream_t s) {
  if (p.chunks > 0) {
    const int64_t groups = (p.units + kThreads / kWave - 1) / (kThreads / kWave);
    const dim3 grid(static_cast<uint32_t>(groups < kMostGroups ? groups : kMostGroups));
    if (write) hipLaunchKernelGGL((kv_write_chunks_kernel<T, D, BITS>), grid, dim3(kThreads), 0, s, p);
    else hipLaunchKernelGGL((kv_read_chunks_kernel<T, D, BITS>), grid, dim3(kThreads), 0, s, p);
    return;
  }
  constexpr int ROWS = kThreads / (D / 8);
  const dim3 grid(static_cast<uint32_t>((p.rows + ROWS - 1) / ROWS));
  if (write) hipLaunchKernelGGL((kv_write_rows_kernel<T, D, BITS>), grid, dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL((kv_read_rows_kernel<T, D, BITS>), grid, dim3(kThreads), 0, s, p);
}
template <typename T>
void dispatch_cache(const CacheParams& p, int d, int bits, bool write, hipStream_t s) {
#define TAAC_KV(D)                                                             \
  if (d == D) bits == 4 ? launch_cache<T, D, 4>(p, write, s) : launch_cache<T, D, 8>(p, write, s);
  TAAC_KV(32) TAAC_KV(64) TAAC_KV(128)
#undef TAAC_KV
}

int run_cache(const char* name, CacheParams& p, bool write, const void* k, const void* v, int32_t B, int32_t T, int32_t d, int bits, const int64_t* ks,
              const int64_t* vs, int dtype, hipStream_t s) {
  if (dtype != TAAC_F32 && dtype != TAAC_BF16 && dtype != TAAC_F16) return set_error(TAAC_ERR_INVALID_VALUE, "%s: unknown dtype %d", name, dtype);
  const int64_t size = dtype == TAAC_F32 ? 4 : 2;
  if (ks == nullptr || vs == nullptr) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null strides", name);
  for (int i = 0; i < 3; ++i) {
    p.ks[i] = ks[i], p.vs[i] = vs[i];
    if (ks[i] * size % 16 != 0 || vs[i] * size % 16 != 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: strides must be multiples of 16 bytes", name);
  }
  if (B == 0 || T == 0) return TAAC_OK;
  if (!k || !v) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null tensor pointer", name);
  if (!aligned16(k) || !aligned16(v)) return set_error(TAAC_ERR_INVALID_VALUE, "%s: tensors must be 16-byte aligned", name);
  p.T = T;
  p.rows = static_cast<int64_t>(B) * T * p.pool.heads;
  // chunks that T tokens meet at most, wherever they start
  const int chunks = static_cast<int>((static_cast<int64_t>(T) + 2 * kKvChunk - 2) / kKvChunk);
  if (T >= kChunksFrom || p.rows > kMostRows) p.chunks = chunks;
  p.units = static_cast<int64_t>(B) * chunks * p.pool.heads;
  p.by_heads = divisor(p.pool.heads), p.by_chunks = divisor(chunks), p.by_tokens = divisor(T);
  if (dtype == TAAC_F32) dispatch_cache<float>(p, d, bits, write, s);
  if (dtype == TAAC_BF16) dispatch_cache<bf16_t>(p, d, bits, write, s);
  if (dtype == TAAC_F16) dispatch_cache<f16_t>(p, d, bits, write, s);
  return check_launch(name);
}

}  // namespace

int take_kv_pool(const char* name, KvPool& pool, void* data, int64_t pages, int32_t heads, int32_t page_tokens, int32_t d, int bits, const void* table,
                 int table_int64, int64_t table_stride, int32_t table_pages, bool has_samples) {
  if (pages < 0 || heads <= 0 || table_pages < 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: sizes of the cache must not be negative, heads > 0", name);
  if (d != 32 && d != 64 && d != 128) return set_error(TAAC_ERR_UNSUPPORTED, "%s: a cached head has 32, 64 or 128 features (got %d)", name, d);
  if (bits != 4 && bits != 8) return set_error(TAAC_ERR_UNSUPPORTED, "%s: a cache has 4 or 8 bits (got %d)", name, bits);
  if (page_tokens < 16 || page_tokens > 1 << 16 || (page_tokens & (page_tokens - 1)) != 0)
    return set_error(TAAC_ERR_UNSUPPORTED, "%s: a page has a power of two of tokens, 16 to 65536 (got %d)", name, page_tokens);
  if (heads > 1 << 16) return set_error(TAAC_ERR_UNSUPPORTED, "%s: at most 2^16 heads", name);
  if ((pages > 0 && data == nullptr) || !aligned16(data)) return set_error(TAAC_ERR_INVALID_VALUE, "%s: the cache must be 16-byte aligned", name);
  if (has_samples && table_pages > 0 && table == nullptr) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null table of pages", name);
  pool.data = static_cast<uint8_t*>(data), pool.pages = pages, pool.table = table, pool.table_stride = table_stride;
  pool.table_pages = table_pages, pool.heads = heads, pool.page_shift = __builtin_ctz(page_tokens), pool.int64 = table_int64 != 0;
  return TAAC_OK;
}

}  // namespace taac

extern "C" int64_t taac_kv_cache_bytes(int64_t pages, int32_t heads, int32_t page_tokens, int32_t d, int bits) {
  using namespace taac;
  KvPool pool{};
  if (take_kv_pool("taac_kv_cache_bytes", pool, pages > 0 ? reinterpret_cast<void*>(16) : nullptr, pages, heads, page_tokens, d, bits, nullptr, 0, 0, 0, false) !=
      TAAC_OK)
    return -1;
  return pages * heads * (page_tokens / kKvChunk) * kv_record_bytes(d, bits);
}

extern "C" int taac_kv_cache_write(void* cache, int64_t pages, int32_t heads, int32_t page_tokens, int32_t d, int bits, const void* table, int table_int64,
                                   int64_t table_stride, int32_t table_pages, const void* k, const void* v, const void* starts, int starts_int64,
                                   const int32_t* lengths, int32_t B, int32_t T, const int64_t k_strides[3], const int64_t v_strides[3], int dtype,
                                   void* stream) {
  using namespace taac;
  const char* name = "taac_kv_cache_write";
  CacheParams p{};
  if (B < 0 || T < 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: batch and tokens must be >= 0", name);
  if (int rc = take_kv_pool(name, p.pool, cache, pages, heads, page_tokens, d, bits, table, table_int64, table_stride, table_pages, B > 0)) return rc;
  p.k = k, p.v = v, p.starts = starts, p.starts_int64 = starts_int64 != 0, p.lengths = lengths;
  return run_cache(name, p, true, k, v, B, T, d, bits, k_strides, v_strides, dtype, as_stream(stream));
}

extern "C" int taac_kv_cache_read(const void* cache, int64_t pages, int32_t heads, int32_t page_tokens, int32_t d, int bits, const void* table, int table_int64,
                                  int64_t table_stride, int32_t table_pages, void* k, void* v, const void* starts, int starts_int64, const int32_t* lengths,
                                  int32_t B, int32_t T, const int64_t k_strides[3], const int64_t v_strides[3], int dtype, void* stream) {
  using namespace taac;
  const char* name = "taac_kv_cache_read";
  CacheParams p{};
  if (B < 0 || T < 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: batch and tokens must be >= 0", name);
  if (int rc = take_kv_pool(name, p.pool, const_cast<void*>(cache), pages, heads, page_tokens, d, bits, table, table_int64, table_stride, table_pages, B > 0))
    return rc;
  p.k_out = k, p.v_out = v, p.starts = starts, p.starts_int64 = starts_int64 != 0, p.lengths = lengths;
  return run_cache(name, p, false, k, v, B, T, d, bits, k_strides, v_strides, dtype, as_stream(stream));
}
