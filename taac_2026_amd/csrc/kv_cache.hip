// Quantising keys and values on their way into a pool of pages, and reading them back (the format: kv_cache.h).
//
// Bound by HBM, or by latency for a few tokens: a value is read once and leaves as 4 or 8 bits, or the other way round, and needs a maximum over 32 and a
// conversion.
#include "kv_cache.h"

namespace taac {
namespace {

constexpr int kThreads = 256;

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
  int32_t B, T, starts_int64;
};

template <typename T>
struct Eight {  // eight neighbouring features
  float f[8];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(T) == 4) {
      const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = a[i], f[4 + i] = b[i];
    } else {
      const typename Vec8<T>::type a = *reinterpret_cast<const typename Vec8<T>::type*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(a[i]);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
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
};

// The least power of two 2^e with max < 7 2^e (464 2^e), as e + 127, for a finite max. The carry out of the fraction is the step to the next power: 7 and 464
// are 1.75 and 1.8125 of one. Kept between 2^-117, under which the smallest code would be subnormal, and what keeps the largest code finite.
template <int BITS>
__device__ __forceinline__ int scale_byte(float most) {
  const uint32_t up = BITS == 4 ? 0x200000u : 0x180000u;
  const int e = static_cast<int>((__builtin_bit_cast(uint32_t, most) + up) >> 23) - (BITS == 4 ? 2 : 8);
  return min(max(e, 10), BITS == 4 ? 252 : 246);
}

// Codes of eight values in order: one word of 4 bits, two of 8.
template <int BITS>
struct Codes {
  uint32_t w[BITS / 4];
};
template <int BITS>
__device__ __forceinline__ Codes<BITS> encode(const float (&f)[8], int byte) {
  typedef __attribute__((__vector_size__(2 * sizeof(short)))) short s16x2;
  const float back = __builtin_bit_cast(float, static_cast<uint32_t>(254 - byte) << 23);  // 2^-e
  float y[8];
  constexpr float kMost = BITS == 4 ? 6.f : 448.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = fminf(fmaxf(f[i] * back, -kMost), kMost);
  Codes<BITS> c;
  if constexpr (BITS == 4) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], 1.f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], 1.f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], 1.f, 3);
    c.w[0] = w;
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s16x2 w = {0, 0};
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, y[4 * i], y[4 * i + 1], 1.f, false);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, y[4 * i + 2], y[4 * i + 3], 1.f, true);
      c.w[i] = __builtin_bit_cast(uint32_t, w);
    }
  }
  return c;
}
template <int BITS>
__device__ __forceinline__ void decode(const Codes<BITS>& c, float scale, float (&f)[8]) {
  typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2;
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

// A row (sample, token, head) and where it belongs: D / 8 lanes, eight features each.
struct Row {
  int64_t b, position;
  int t, h;
  bool there;
  __device__ __forceinline__ Row(const CacheParams& p, int64_t row) {
    const int64_t token = row / p.pool.heads;
    h = static_cast<int>(row - token * p.pool.heads);
    b = token / p.T;
    t = static_cast<int>(token - b * p.T);
    there = p.lengths == nullptr || t < p.lengths[b];
    const int64_t start = p.starts == nullptr ? 0 : (p.starts_int64 ? static_cast<const int64_t*>(p.starts)[b] : static_cast<const int32_t*>(p.starts)[b]);
    there &= start >= 0 && start < (int64_t{1} << 40);
    position = start + t;
  }
};

template <typename T, int D, int BITS>
__global__ __launch_bounds__(kThreads) void kv_write_rows_kernel(const CacheParams p) {
  constexpr int LANES = D / 8, ROWS = kThreads / LANES, BLOCKS = D / kKvBlock;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / LANES;
  if (row >= p.rows) return;
  const int s = threadIdx.x % LANES, block = s / 4, sub = s % 4;
  const Row at(p, row);
  if (!at.there) return;
  const int64_t page = kv_page(p.pool, at.b, at.position >> p.pool.page_shift);
  if (page < 0) return;
  Eight<T> k, v;
  k.load(static_cast<const T*>(p.k) + at.b * p.ks[0] + at.h * p.ks[1] + at.t * p.ks[2] + 8 * s);
  v.load(static_cast<const T*>(p.v) + at.b * p.vs[0] + at.h * p.vs[1] + at.t * p.vs[2] + 8 * s);
  const int in_page = static_cast<int>(at.position & ((1 << p.pool.page_shift) - 1)), token = in_page % kKvChunk;
  uint8_t* record = p.pool.data + kv_record(p.pool, page, at.h, in_page / kKvChunk, kv_record_bytes(D, BITS));
  float k_most = 0.f, v_most = 0.f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    k_most = fmaxf(k_most, fabsf(k.f[i]));
    v_most = fmaxf(v_most, fabsf(v.f[i]));
    finite &= fabsf(k.f[i]) <= 3.4028235e38f && fabsf(v.f[i]) <= 3.4028235e38f;
  }
  k_most = group_max<4>(k_most);
  v_most = group_max<4>(v_most);
  int bad = !finite;
#pragma unroll
  for (int off = LANES / 2; off > 0; off /= 2) bad |= __shfl_xor(bad, off, kWave);
  int k_scale = scale_byte<BITS>(k_most), v_scale = scale_byte<BITS>(v_most);
  if (bad) {
    k_scale = kKvNotFinite, v_scale = 127;
#pragma unroll
    for (int i = 0; i < 8; ++i) k.f[i] = v.f[i] = 0.f;
  }
  const Codes<BITS> kc = encode<BITS>(k.f, bad ? 127 : k_scale), vc = encode<BITS>(v.f, v_scale);
  uint8_t* keys = record + block * (kKvChunk * kKvBlock * BITS / 8) + token * (kKvBlock * BITS / 8) + sub * BITS;
  if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(keys) = kc.w[0];
  else *reinterpret_cast<u32x2*>(keys) = u32x2{kc.w[0], kc.w[1]};
  uint8_t* values = record + kv_value_at(D, BITS);
  const int group = token / 4, of4 = token % 4;
  if constexpr (BITS == 4) {
    const uint32_t mine = vc.w[0], other = __shfl_xor(mine, 2, kWave);
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
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / LANES;
  if (row >= p.rows) return;
  const int s = threadIdx.x % LANES, block = s / 4, sub = s % 4;
  const Row at(p, row);
  const int64_t page = at.there ? kv_page(p.pool, at.b, at.position >> p.pool.page_shift) : -1;
  Eight<T> k, v;
  if (page < 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) k.f[i] = v.f[i] = 0.f;
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
    decode<BITS>(kc, kv_scale(k_scale), k.f);
    decode<BITS>(vc, kv_scale(v_scale), v.f);
  }
  k.store(static_cast<T*>(p.k_out) + at.b * p.ks[0] + at.h * p.ks[1] + at.t * p.ks[2] + 8 * s);
  v.store(static_cast<T*>(p.v_out) + at.b * p.vs[0] + at.h * p.vs[1] + at.t * p.vs[2] + 8 * s);
}

template <typename T, int D, int BITS>
void launch_cache(const CacheParams& p, bool write, hipStream_t s) {
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
  p.B = B, p.T = T;
  p.rows = static_cast<int64_t>(B) * T * p.pool.heads;
  if (p.rows > int64_t{0x7fffffff} * 16) return set_error(TAAC_ERR_UNSUPPORTED, "%s: too many rows for one call", name);
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
