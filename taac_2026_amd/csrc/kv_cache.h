// Keys and values of many sequences, quantised, in a pool of pages (kv_cache.hip writes and reads them, cached_attention.hip attends to them).
//
// A value is stored as x ~ code * 2^e with one e per 32 consecutive features of a token's head: codes are e2m1 (4 bits: 0, 0.5, 1, 1.5, 2, 3, 4, 6) or
// e4m3 (8 bits), rounded to nearest even; 2^e is the least power of two with max |x| < 7 2^e (464 2^e), so that no code is further off than half a step:
// 7 is as far above 6 as a half step, 464 above 448. e is kept as a byte e + 127. The conversion instructions of CDNA4 multiply by a power of two on
// their way, so that reading a scale costs a shift. A token with a NaN or an infinity in its key or value is stored as e = 128 (byte 255, which these
// instructions turn into NaN) for its key, and zeros for its value: it reads back as NaN, and where a mask hides it from a query it adds 0 * 0.
//
// A page holds page_tokens tokens of every head: [page][head][chunk of 16 tokens][record]. A record is laid out for the matrix instructions
// (v_mfma_f32_16x16x32, operand lane = row l16 + 16 * group, eight values of the contraction each), so that a wavefront's reads are runs of memory
// which arrive as operands:
//   key codes     [block of 32 features][token 16][feature 32]     a lane of a token reads features in order
//   value codes   [feature n of 16][group of 4 tokens][block][token of 4][features n, n + 16]      a lane of feature n reads four tokens of two features
//   key scales    [token 16][block]
//   value scales  [group of 4 tokens][block][token of 4]
// 4 bits: two features to a byte, the first in the low half.
#pragma once

#include "common.h"

namespace taac {

constexpr int kKvChunk = 16;  // tokens of a record
constexpr int kKvBlock = 32;  // features that share a scale

__host__ __device__ constexpr int kv_key_bytes(int d, int bits) { return kKvChunk * d * bits / 8; }
__host__ __device__ constexpr int kv_value_at(int d, int bits) { return kv_key_bytes(d, bits); }
__host__ __device__ constexpr int kv_key_scale_at(int d, int bits) { return 2 * kv_key_bytes(d, bits); }
__host__ __device__ constexpr int kv_value_scale_at(int d, int bits) { return kv_key_scale_at(d, bits) + kKvChunk * d / kKvBlock; }
__host__ __device__ constexpr int kv_record_bytes(int d, int bits) { return kv_value_scale_at(d, bits) + kKvChunk * d / kKvBlock; }

constexpr int kKvNotFinite = 255;  // the scale of a key that holds a NaN or an infinity, or whose value does

// n / d of n below 2^31 by a product: divisions are most of a short call's scalar instructions.
struct Divisor {
  uint32_t factor, shift;
  int32_t d;
  __device__ __forceinline__ int over(int n) const { return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * factor) >> shift); }
};
inline Divisor divisor(int32_t d) {
  uint32_t bits = 0;
  while ((int64_t{1} << bits) < d) ++bits;
  // factor = ceil(2^(31 + bits) / d) is off by less than one in 2^(31 + bits) / d, i.e. n / d by less than 1 / d
  return {static_cast<uint32_t>(((uint64_t{1} << (31 + bits)) + d - 1) / d), 31 + bits, d};
}

struct KvPool {
  uint8_t* data;
  int64_t pages;          // in the pool
  const void* table;      // [B][table_pages] int32 or int64: the page of a sample's positions page_tokens i .. page_tokens (i + 1) - 1
  int64_t table_stride;   // of a sample, elements
  int32_t table_pages, heads, page_shift, int64;
};

// The page of a position's index in the table; -1: there is none.
__device__ __forceinline__ int64_t kv_page(const KvPool& pool, int64_t sample, int64_t index) {
  if (index < 0 || index >= pool.table_pages) return -1;
  const int64_t at = sample * pool.table_stride + index;
  const int64_t page = pool.int64 ? static_cast<const int64_t*>(pool.table)[at] : static_cast<const int32_t*>(pool.table)[at];
  return page >= 0 && page < pool.pages ? page : -1;
}
// Byte offset of the record of a page's chunk.
__device__ __forceinline__ int64_t kv_record(const KvPool& pool, int64_t page, int head, int chunk, int record_bytes) {
  return ((page * pool.heads + head) * (int64_t{1} << (pool.page_shift - 4)) + chunk) * record_bytes;
}

// A scale for the conversion instructions, which only look at its exponent.
__device__ __forceinline__ float kv_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

int take_kv_pool(const char* name, KvPool& pool, void* data, int64_t pages, int32_t heads, int32_t page_tokens, int32_t d, int bits, const void* table,
                 int table_int64, int64_t table_stride, int32_t table_pages, bool has_samples);

}  // namespace taac
