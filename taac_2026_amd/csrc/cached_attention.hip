// Attention of a few new tokens of many sequences over keys and values that lie quantised in a pool of pages (the format: kv_cache.h).
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j   over the positions j that query i sees: up to its own, with a window only the last of them.
//
// The new tokens of a sample are the last of its cached ones. Queries of the heads that share a key head are rows of one product.
//
// Bound by HBM: every code is read once per key head. A wavefront walks tiles of 64 tokens, one tile ahead in registers, with the running maximum and sum
// of a softmax; the wavefronts of a workgroup take the tiles in turn and meet at its end; long histories of few heads are split over workgroups, whose parts
// a second kernel joins. Codes become bf16 operands by the conversion instructions, two values an issue, scales included.
//
// Two forms, lane = (l16 = lane % 16, grp = lane / 16):
//  * up to 4 rows: scores come out with a lane to a token, whatever the number of rows, so that the softmax's instructions are not spent on rows that there are
//    not. Operand rows 4 g + r of the queries hold row r in the lanes of group g and zeros in the others, and the keys' lane holds its own token's
//    features: result row 4 g + r, column l16 is the score of row r with token 16 g + l16. The probabilities turn through LDS into an operand.
//  * 16 rows at a time: keys are the first operand, so that a lane has 4 tokens of each 16 for one row, as they stand an operand of the product with the values.
// Values enter as their transpose: features are rows, queries columns, and a row's rescaling stays in its lanes.
//
// Precision: all operands are bf16, exact for keys and values of either size, whatever their scales, and for queries (fp16 ones in two parts); scores, statistics
// and sums are fp32; probabilities enter as two parts (16 bits), in the first form in columns that would be empty. The maximum moves when a score exceeds it
// by a factor of 2^8, which cancels.
#include "kv_cache.h"
#include "ts_common.h"

namespace taac {
namespace {

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

struct AttendParams {
  KvPool pool;
  const void* q;
  void* o;
  const int32_t* lengths;        // [B]: cached tokens, the new ones among them
  const int32_t* query_lengths;  // [B] or null: T
  float* partial;                // [row][split][D], then [row][split] of (maximum, sum)
  int64_t qs[3], os[3];          // element strides of (batch, head, token)
  int64_t all_rows;              // B * heads * T
  Divisor group, splits, row_tiles, heads;
  int32_t H, T, rows, window;
  float scale;                   // times log2 e: powers of two
};

constexpr int kTile = 64;          // tokens
constexpr float kNothing = -3e38f; // the maximum of no scores
constexpr float kSlack = 8.f;

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// Two values of a word of codes.
template <int BITS, int I>
__device__ __forceinline__ uint32_t two(uint32_t w, float scale) {
  if constexpr (BITS == 4) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, I));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, I != 0));
}

// Eight neighbours of a row of queries, in one part of bf16, or two for fp16, whose eleven bits they hold.
template <typename T>
constexpr int kParts = sizeof(T) == 2 && !__is_same(T, bf16_t) ? 2 : 1;
template <typename T>
__device__ __forceinline__ bf16x8 query_part(const T* p, int part) {
  const typename Vec8<T>::type v = *reinterpret_cast<const typename Vec8<T>::type*>(p);
  if constexpr (kParts<T> == 1) {
    return v;
  } else {
    bf16x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = static_cast<float>(v[i]);
      const bf16_t high = static_cast<bf16_t>(x);
      r[i] = part == 0 ? high : static_cast<bf16_t>(x - static_cast<float>(high));
    }
    return r;
  }
}

__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Byte i of a word of scales as the conversions' factor, which is the exponent alone: what is left of its neighbours does not count.
template <int I>
__device__ __forceinline__ float scale_of(uint32_t w) {
  return __builtin_bit_cast(float, I == 0 ? w << 23 : I == 1 ? w << 15 : I == 2 ? w << 7 : w >> 1);
}

template <int N>
struct Words {
  uint32_t w[N];
  __device__ __forceinline__ void load(const uint8_t* p) {
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
      static_assert(N == 1);
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
  }
};

// Eight values in order: one word of 4 bits, two of 8.
template <int BITS>
__device__ __forceinline__ bf16x8 eight(const uint32_t* w, float scale) {
  u32x4 r;
  if constexpr (BITS == 4) r = u32x4{two<4, 0>(w[0], scale), two<4, 1>(w[0], scale), two<4, 2>(w[0], scale), two<4, 3>(w[0], scale)};
  else r = u32x4{two<8, 0>(w[0], scale), two<8, 1>(w[0], scale), two<8, 0>(w[1], scale), two<8, 1>(w[1], scale)};
  return __builtin_bit_cast(bf16x8, r);
}

// Four tokens of features n and n + 16: a pair of words for each feature.
template <int BITS>
__device__ __forceinline__ void four_tokens(const uint32_t* w, uint32_t scales, uint32_t (&first)[2], uint32_t (&second)[2]) {
  uint32_t x[4];
  if constexpr (BITS == 4) {
    x[0] = two<4, 0>(w[0], scale_of<0>(scales)), x[1] = two<4, 1>(w[0], scale_of<1>(scales));
    x[2] = two<4, 2>(w[0], scale_of<2>(scales)), x[3] = two<4, 3>(w[0], scale_of<3>(scales));
  } else {
    x[0] = two<8, 0>(w[0], scale_of<0>(scales)), x[1] = two<8, 1>(w[0], scale_of<1>(scales));
    x[2] = two<8, 0>(w[1], scale_of<2>(scales)), x[3] = two<8, 1>(w[1], scale_of<3>(scales));
  }
  first[0] = __builtin_amdgcn_perm(x[1], x[0], 0x05040100u), first[1] = __builtin_amdgcn_perm(x[3], x[2], 0x05040100u);
  second[0] = __builtin_amdgcn_perm(x[1], x[0], 0x07060302u), second[1] = __builtin_amdgcn_perm(x[3], x[2], 0x07060302u);
}

// What a row tile of a sample sees, and the part of it that a split takes, in tiles of 64 tokens.
struct Span {
  int length, news;   // of the sample: tokens, and how many of them are queries
  int first, end;     // tiles of the split
  int active;         // splits that have tiles
};
__device__ __forceinline__ Span span_of(const AttendParams& p, int b, int row0, int rows, int split, int waves) {
  Span s;
  s.length = max(p.lengths[b], 0);
  s.news = p.query_lengths == nullptr ? p.T : min(max(p.query_lengths[b], 0), p.T);
  const int64_t held = static_cast<int64_t>(p.pool.table_pages) << p.pool.page_shift;
  const int t0 = p.group.over(row0), t1 = min(p.group.over(row0 + rows - 1), s.news - 1);
  const int base = s.length - s.news;  // of the sample's first query; below zero where it has more queries than tokens
  int64_t high = static_cast<int64_t>(base) + t1 + 1, low = p.window > 0 ? static_cast<int64_t>(base) + t0 + 1 - p.window : 0;
  high = high < held ? high : held;
  low = low > 0 ? low : 0;
  if (t1 < t0 || high <= low) {
    s.first = s.end = s.active = 0;
    return s;
  }
  const int t_first = static_cast<int>(low / kTile), t_end = static_cast<int>((high + kTile - 1) / kTile);
  // a multiple of the wavefronts' number, a power of two
  const int each = (p.splits.over(t_end - t_first + p.splits.d - 1) + waves - 1) & -waves;
  s.active = 1;
  if (each < t_end - t_first) s.active = (t_end - t_first + each - 1) / each;
  s.first = min(t_first + split * each, t_end);
  s.end = min(s.first + each, t_end);
  return s;
}
// The positions that a row sees.
struct Seen {
  int low, high;
  __device__ __forceinline__ Seen(const AttendParams& p, const Span& s, int row) {
    const int t = p.group.over(row), place = s.length - s.news + t;
    const bool there = row < p.rows && t < s.news;
    high = there ? place + 1 : 0;
    low = p.window > 0 && place + 1 > p.window ? place + 1 - p.window : 0;
  }
};

// Which workgroup is which: splits next to each other, then row tiles, key heads, samples.
struct Job {
  int b, head, row0, split;
  Job() = default;
  __device__ __forceinline__ Job(const AttendParams& p, int rows) {
    int id = blockIdx.x, over = p.splits.over(id);
    split = id - over * p.splits.d;
    id = over, over = p.row_tiles.over(id);
    row0 = (id - over * p.row_tiles.d) * rows;
    b = p.heads.over(over);
    head = over - b * p.heads.d;
  }
};

// Where a row's query is, and its output or the split's part of it.
struct Place {
  int t, h;
  __device__ __forceinline__ Place(const AttendParams& p, const Job& job, int row) {
    t = p.group.over(row);
    h = job.head * p.group.d + row - t * p.group.d;
  }
  template <typename T>
  __device__ __forceinline__ const T* query(const AttendParams& p, const Job& job) const {
    return static_cast<const T*>(p.q) + job.b * p.qs[0] + h * p.qs[1] + t * p.qs[2];
  }
  // four features, their sum of weights, and the maximum that both refer to
  template <typename T, int D>
  __device__ __forceinline__ void leave(const AttendParams& p, const Job& job, const Span& span, int c, const f32x4& total, float l, float top) const {
    if (span.active > 1) {
      const int64_t row = ((static_cast<int64_t>(job.b) * p.H + h) * p.T + t) * p.splits.d + job.split;
      *reinterpret_cast<f32x4*>(p.partial + row * D + c) = total;
      if (c == 0) {
        float* stats = p.partial + p.all_rows * p.splits.d * D + row * 2;
        stats[0] = top, stats[1] = l;
      }
      return;
    }
    store<T>(p, job.b, c, total, l);
  }
  template <typename T>
  __device__ __forceinline__ void store(const AttendParams& p, int b, int c, const f32x4& total, float l) const {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    typename Vec8<T>::half_type v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = static_cast<T>(total[e] * inv);
    *reinterpret_cast<typename Vec8<T>::half_type*>(static_cast<T*>(p.o) + b * p.os[0] + h * p.os[1] + t * p.os[2] + c) = v;
  }
};

template <typename T, int D, int ROWS, int THREADS>
__device__ __forceinline__ void clear_rows(const AttendParams& p, const Job& job) {
  for (int i = threadIdx.x; i < ROWS * (D / 4); i += THREADS) {
    const int row = job.row0 + i / (D / 4);
    if (row < p.rows) Place(p, job, row).template store<T>(p, job.b, i % (D / 4) * 4, f32x4{0.f, 0.f, 0.f, 0.f}, 0.f);
  }
}

// Rows [ROWS][D] of every wavefront meet in LDS and leave as outputs, or as a split's part.
template <typename T, int D, int ROWS, int W>
struct Meeting {
  float acc[W][ROWS][D + 4];
  float most[W][ROWS], sum[W][ROWS];

  __device__ __forceinline__ void leave(const AttendParams& p, const Job& job, const Span& span) {
    for (int i = threadIdx.x; i < ROWS * (D / 4); i += W * kWave) {
      const int r = i / (D / 4), c = i % (D / 4) * 4, row = job.row0 + r;
      if (row >= p.rows) continue;
      float top = most[0][r];
#pragma unroll
      for (int w = 1; w < W; ++w) top = fmaxf(top, most[w][r]);
      f32x4 total = {0.f, 0.f, 0.f, 0.f};
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = __builtin_amdgcn_exp2f(most[w][r] - top);
        l = fmaf(f, sum[w][r], l);
        const f32x4 part = *reinterpret_cast<const f32x4*>(&acc[w][r][c]);
#pragma unroll
        for (int e = 0; e < 4; ++e) total[e] = fmaf(f, part[e], total[e]);
      }
      Place(p, job, row).template leave<T, D>(p, job, span, c, total, l, top);
    }
  }
};

// Maximum over a wavefront, for every lane: within quads, eights and rows of sixteen by the operands' own lane patterns, then across.
template <int PATTERN>
__device__ __forceinline__ float max_with(float v) {
  const int bits = __builtin_bit_cast(int, v);
  return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(bits, bits, PATTERN, 0xf, 0xf, false)));
}
__device__ __forceinline__ float max_over_rows(float v) {  // across the four rows of sixteen
  const uint32_t bits = __builtin_bit_cast(uint32_t, v);
  const auto a = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);
  const uint32_t a0 = a[0], a1 = a[1], pair = __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
  const auto b = __builtin_amdgcn_permlane32_swap(pair, pair, false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return fmaxf(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}
__device__ __forceinline__ float wave_max(float v) {
  v = max_with<0xb1>(v);   // quads: lanes 1, 0, 3, 2
  v = max_with<0x4e>(v);   // 2, 3, 0, 1
  v = max_with<0x141>(v);  // eight lanes mirrored
  v = max_with<0x140>(v);  // sixteen
  return max_over_rows(v);
}

// The pages of a tile's four chunks, read as scalars one tile before they are needed. WHOLE: pages of at least a tile, one for all four.
template <bool WHOLE>
struct Pages {
  static constexpr int N = WHOLE ? 1 : 4;
  int32_t low[N], high[N];
  __device__ __forceinline__ void find(const KvPool& pool, int64_t row, int tile) {
    typedef const __attribute__((address_space(4))) int32_t* Scalars;
    const Scalars table = (Scalars)(reinterpret_cast<uint64_t>(pool.table) + row * (pool.int64 ? 8 : 4));
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int index = min((tile * (kTile / kKvChunk) + c) >> (pool.page_shift - 4), pool.table_pages - 1);
      if (pool.int64) {
        low[c] = table[2 * static_cast<int64_t>(index)], high[c] = table[2 * static_cast<int64_t>(index) + 1];
      } else {
        low[c] = table[index], high[c] = low[c] >> 31;
      }
    }
  }
};

// A tile in LDS: the records of its chunks, brought there without registers, sixteen bytes to a lane.
template <int D, int BITS>
struct Staged {
  static constexpr int RECORD = kv_record_bytes(D, BITS), PIECES = 4 * RECORD / 16, REQUESTS = (PIECES + kWave - 1) / kWave, BYTES = REQUESTS * kWave * 16;
  static constexpr int BLOCKS = D / kKvBlock;

  // Which chunks there are, a bit each. In the place of one that there is not: the first of the pool, whose tokens are then masked.
  template <bool WHOLE>
  static __device__ __forceinline__ uint32_t request(const KvPool& pool, const Pages<WHOLE>& pages, int head, int tile, uint8_t* to, int lane) {
    constexpr int N = Pages<WHOLE>::N;
    uint32_t held = 0;
    const uint8_t* record[N];
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int chunk = tile * (kTile / kKvChunk) + c;
      const int64_t page = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(pages.high[c])) << 32 | static_cast<uint32_t>(pages.low[c]));
      const bool there = (chunk >> (pool.page_shift - 4)) < pool.table_pages && page >= 0 && page < pool.pages;
      held |= there ? (WHOLE ? 15u : 1u << c) : 0u;
      record[c] = pool.data + (there ? kv_record(pool, page, head, chunk & ((1 << (pool.page_shift - 4)) - 1), RECORD) : 0);
    }
    if constexpr (WHOLE) {
#pragma unroll
      for (int i = 0; i < REQUESTS; ++i) lds_dma16_offset(record[0], min(i * kWave + lane, PIECES - 1) * 16, to + i * kWave * 16);
      return held;
    }
#pragma unroll
    for (int i = 0; i < REQUESTS; ++i) {
      const int piece = min(i * kWave + lane, PIECES - 1);
      // the lane's chunk is one of those that these sixty-four pieces meet
      const uint8_t* from = record[i * kWave * 16 / RECORD % N] - i * kWave * 16 / RECORD * RECORD;
#pragma unroll
      for (int c = i * kWave * 16 / RECORD + 1; c < 4; ++c) {
        if (c * RECORD >= (i + 1) * kWave * 16) break;
        from = piece >= c * (RECORD / 16) ? record[c % N] - c * RECORD : from;
      }
      lds_dma16(from + piece * 16, to + i * kWave * 16);
    }
    return held;
  }
};

// acc[rows of 16 features] += values^T p: probs[n][part][half]: of 32 tokens, group grp those of chunk 2 half at 4 grp, then those of the next chunk.
template <int D, int BITS, int RT, int PARTS>
__device__ __forceinline__ void times_values(const uint8_t* tile, int l16, int grp, const bf16x8 (&probs)[RT][PARTS][2], f32x4 (&acc)[RT][D / 16]) {
  constexpr int BLOCKS = D / kKvBlock, EACH = BITS / 4, RECORD = kv_record_bytes(D, BITS);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    Words<BLOCKS * EACH> codes[2];
    Words<BLOCKS> scales[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      codes[c].load(tile + (2 * half + c) * RECORD + kv_value_at(D, BITS) + (l16 * 4 + grp) * BLOCKS * BITS);
      scales[c].load(tile + (2 * half + c) * RECORD + kv_value_scale_at(D, BITS) + grp * BLOCKS * 4);
    }
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) {
      uint32_t a0[2], a1[2], b0[2], b1[2];
      four_tokens<BITS>(codes[0].w + j * EACH, scales[0].w[j], a0, a1);
      four_tokens<BITS>(codes[1].w + j * EACH, scales[1].w[j], b0, b1);
      const auto first = __builtin_bit_cast(bf16x8, (u32x4{a0[0], a0[1], b0[0], b0[1]}));
      const auto second = __builtin_bit_cast(bf16x8, (u32x4{a1[0], a1[1], b1[0], b1[1]}));
#pragma unroll
      for (int n = 0; n < RT; ++n)
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          acc[n][2 * j] = mfma(first, probs[n][part][half], acc[n][2 * j]);
          acc[n][2 * j + 1] = mfma(second, probs[n][part][half], acc[n][2 * j + 1]);
        }
    }
  }
}

// A wavefront's tiles, S of them in LDS: S - 1 on their way while one is taken. Its only vector-memory operations are the transfers, so that their count says
// what has arrived.
template <int D, int BITS, int W, int S, bool WHOLE, typename Take>
__device__ __forceinline__ void walk(const AttendParams& p, const Job& job, const Span& span, int wave, int lane, uint8_t* stages, Take&& take) {
  typedef Staged<D, BITS> Tile;
  const int64_t row = job.b * p.pool.table_stride;
  uint32_t held[S];
  Pages<WHOLE> pages;
  int next = span.first + wave, tile = next;
  if (next >= span.end) return;
  pages.find(p.pool, row, next);
#pragma unroll
  for (int i = 0; i < S - 1; ++i) {
    if (next < span.end) {
      held[i] = Tile::request(p.pool, pages, job.head, next, stages + i * Tile::BYTES, lane);
      next += W;
      pages.find(p.pool, row, next);
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // what the compiler asked for before, which it would otherwise await in every round
  while (tile < span.end) {
#pragma unroll
    for (int i = 0; i < S; ++i) {
      if (tile >= span.end) break;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the reads of the tile that lay there
      if (next < span.end) {
        held[(i + S - 1) % S] = Tile::request(p.pool, pages, job.head, next, stages + (i + S - 1) % S * Tile::BYTES, lane);
        next += W;
        pages.find(p.pool, row, next);
        vm_wait<(S - 1) * Tile::REQUESTS>();
      } else if (S > 2 && next - tile > W) {
        vm_wait<Tile::REQUESTS>();
      } else {
        vm_wait<0>();
      }
      take(stages + i * Tile::BYTES, held[i], tile);
      tile += W;
    }
  }
}

// Lane l + 4's value, within a row of sixteen.
__device__ __forceinline__ float from_four_on(float v) {
  const int bits = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(bits, bits, 0x104, 0xf, 0xf, false));
}

// ---- up to four rows ----------------------------------------------------------------------------------------------

template <typename T, int D, int BITS, int ROWS, int W, int S>
__global__ __launch_bounds__(W * kWave) void cached_attention_few_kernel(const AttendParams p) {
  constexpr int BLOCKS = D / kKvBlock, SLOT = kTile + 8, PARTS = kParts<T>;
  typedef Staged<D, BITS> Tile;
  typedef Meeting<T, D, ROWS, W> Met;
  extern __shared__ __align__(16) uint8_t memory[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave, l16 = lane % 16, grp = lane / 16;
  const Job job(p, ROWS);
  const Span span = span_of(p, job.b, job.row0, ROWS, job.split, W);
  if (job.split >= span.active) {
    if (job.split == 0) clear_rows<T, D, ROWS, W * kWave>(p, job);
    return;
  }
  uint8_t* const stages = memory + wave * (S * Tile::BYTES);
  bf16_t (*const turned)[SLOT] = reinterpret_cast<bf16_t (*)[SLOT]>(memory + W * S * Tile::BYTES) + wave * 8;
  int low[ROWS], high[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const Seen seen(p, span, job.row0 + r);
    low[r] = seen.low, high[r] = seen.high;
  }
  bf16x8 q[D / 8];
  {
    static_assert(ROWS * PARTS <= 4);
    const int slot = l16 % 4, part = PARTS == 2 ? slot / 2 : 0, r = PARTS == 2 ? slot % 2 : slot, row = job.row0 + r;
    const bool mine = l16 / 4 == grp && r < ROWS && row < p.rows;
    const T* src = Place(p, job, min(row, p.rows - 1)).query<T>(p, job);
#pragma unroll
    for (int o = 0; o < D / 8; ++o) {
      q[o] = bf16x8{};
      if (mine) q[o] = query_part<T>(src + 8 * o, part);
    }
  }
  float most[ROWS];
  f32x4 acc[1][D / 16], sum = {0.f, 0.f, 0.f, 0.f};  // sums are products with ones: their columns are those of acc
#pragma unroll
  for (int r = 0; r < ROWS; ++r) most[r] = kNothing;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) acc[0][i] = f32x4{0.f, 0.f, 0.f, 0.f};

  const bf16x8 ones = __builtin_bit_cast(bf16x8, (u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}));
  auto take = [&](const uint8_t* tile, uint32_t chunks, int number) __attribute__((always_inline)) {
    const uint8_t* mine = tile + grp * Tile::RECORD;
    const uint8_t* scale_bytes = mine + kv_key_scale_at(D, BITS) + l16 * BLOCKS;
    const uint32_t key_scales = BLOCKS == 1 ? *scale_bytes : BLOCKS == 2 ? *reinterpret_cast<const uint16_t*>(scale_bytes) : *reinterpret_cast<const uint32_t*>(scale_bytes);
    const bool held = chunks >> grp & 1;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    f32x4 chain[BLOCKS];  // a block each, which do not wait for each other
    // a NaN would reach the lanes of the other groups, whose products with it are zeros: it waits for the scores
    const bool finite = (key_scales & 255u) != kKvNotFinite;
    const uint32_t scales = finite ? key_scales : 0u;
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) {
      const float scale = j == 0 ? scale_of<0>(scales) : j == 1 ? scale_of<1>(scales) : j == 2 ? scale_of<2>(scales) : scale_of<3>(scales);
      Words<BITS> keys;
      keys.load(mine + j * (kKvChunk * 4 * BITS) + l16 * 4 * BITS);
#pragma unroll
      for (int i = 0; i < 4; ++i) chain[j] = mfma(q[4 * j + i], eight<BITS>(keys.w + i * (BITS / 4), scale), i == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : chain[j]);
    }
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] += chain[j][r];
    const int position = number * kTile + lane;
    float score[ROWS];
    bool above = false;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float x = finite ? (PARTS == 2 ? s[r] + s[2 + r] : s[r]) * p.scale : __builtin_nanf("");
      score[r] = held && position >= low[r] && position < high[r] ? x : -INFINITY;
      above |= score[r] > most[r] + kSlack;
    }
    if (__any(above)) {
      float mine = 1.f;  // the factor of this lane's column of acc
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const float top = fmaxf(most[r], wave_max(score[r])), f = __builtin_amdgcn_exp2f(most[r] - top);
        most[r] = top;
        mine = l16 % 4 == r ? f : mine;
      }
      sum[0] *= mine;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[0][i][e] *= mine;
    }
    // token 16 grp + l16 lies in chunk grp, group l16 / 4
    bf16_t* to = &turned[0][l16 / 4 * 16 + grp * 4 + l16 % 4];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float x = __builtin_amdgcn_exp2f(score[r] - most[r]);
      const bf16_t rounded = static_cast<bf16_t>(x);
      to[r * SLOT] = rounded;
      to[(4 + r) * SLOT] = static_cast<bf16_t>(x - static_cast<float>(rounded));
    }
    wave_sync();
    bf16x8 probs[1][1][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) probs[0][0][half] = *reinterpret_cast<const bf16x8*>(&turned[l16 % 8][grp * 16 + half * 8]);
    wave_sync();
    sum = mfma(ones, probs[0][0][0], sum);
    sum = mfma(ones, probs[0][0][1], sum);
    times_values<D, BITS, 1, 1>(tile, l16, grp, probs, acc);
  };

  p.pool.page_shift >= 6 ? walk<D, BITS, W, S, true>(p, job, span, wave, lane, stages, take) : walk<D, BITS, W, S, false>(p, job, span, wave, lane, stages, take);
  // the two parts of the probabilities stand in columns r and 4 + r
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[0][i][e] += from_four_on(acc[0][i][e]);
  sum[0] += from_four_on(sum[0]);
  float top = most[0];
#pragma unroll
  for (int r = 1; r < ROWS; ++r) top = l16 == r ? most[r] : top;
  if constexpr (W == 1) {
    if (l16 >= ROWS || job.row0 + l16 >= p.rows) return;
    const Place place(p, job, job.row0 + l16);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) place.leave<T, D>(p, job, span, 16 * i + 4 * grp, acc[0][i], sum[0], top);
  } else {
    Met& meeting = *reinterpret_cast<Met*>(memory);  // in the place of the tiles
    __syncthreads();
    if (l16 < ROWS) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) *reinterpret_cast<f32x4*>(&meeting.acc[wave][l16][16 * i + 4 * grp]) = acc[0][i];
      if (grp == 0) meeting.most[wave][l16] = top, meeting.sum[wave][l16] = sum[0];
    }
    __syncthreads();
    meeting.leave(p, job, span);
  }
}

// ---- sixteen rows at a time ---------------------------------------------------------------------------------------

template <typename T, int D, int BITS, int RT, int W, int S>
__global__ __launch_bounds__(W * kWave) void cached_attention_many_kernel(const AttendParams p) {
  constexpr int BLOCKS = D / kKvBlock, ROWS = 16 * RT, PARTS = kParts<T>;
  typedef Staged<D, BITS> Tile;
  typedef Meeting<T, D, ROWS, W> Met;
  extern __shared__ __align__(16) uint8_t memory[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave, l16 = lane % 16, grp = lane / 16;
  const Job job(p, ROWS);
  const Span span = span_of(p, job.b, job.row0, min(ROWS, p.rows - job.row0), job.split, W);
  if (job.split >= span.active) {
    if (job.split == 0) clear_rows<T, D, ROWS, W * kWave>(p, job);
    return;
  }
  uint8_t* const stages = memory + wave * (S * Tile::BYTES);
  int low[RT], high[RT];
  bf16x8 q[RT][PARTS][BLOCKS];
#pragma unroll
  for (int n = 0; n < RT; ++n) {
    const int row = job.row0 + 16 * n + l16;
    const Seen seen(p, span, row);
    low[n] = seen.low, high[n] = seen.high;
    const T* src = Place(p, job, min(row, p.rows - 1)).query<T>(p, job);
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j)
#pragma unroll
      for (int part = 0; part < PARTS; ++part) {
        q[n][part][j] = bf16x8{};
        if (row < p.rows) q[n][part][j] = query_part<T>(src + 8 * (grp * BLOCKS + j), part);
      }
  }
  float most[RT], sum[RT];
  f32x4 acc[RT][D / 16];
#pragma unroll
  for (int n = 0; n < RT; ++n) {
    most[n] = kNothing, sum[n] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) acc[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int octet = grp * BLOCKS, block = octet / 4;  // of the lane's features
  auto take = [&](const uint8_t* tile, uint32_t chunks, int number) __attribute__((always_inline)) {
    f32x4 s[RT][4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int n = 0; n < RT; ++n) s[n][c] = f32x4{0.f, 0.f, 0.f, 0.f};
      const uint8_t* record = tile + c * Tile::RECORD;
      Words<BLOCKS * BITS / 4> keys;
      keys.load(record + block * (kKvChunk * 4 * BITS) + l16 * 4 * BITS + octet % 4 * BITS);
      const float scale = scale_of<0>(record[kv_key_scale_at(D, BITS) + l16 * BLOCKS + block]);
#pragma unroll
      for (int j = 0; j < BLOCKS; ++j) {
        const bf16x8 key = eight<BITS>(keys.w + j * (BITS / 4), scale);
#pragma unroll
        for (int n = 0; n < RT; ++n)
#pragma unroll
          for (int part = 0; part < PARTS; ++part) s[n][c] = mfma(key, q[n][part][j], s[n][c]);
      }
    }
    bool above = false;
    float top[RT];
#pragma unroll
    for (int n = 0; n < RT; ++n) {
      top[n] = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool held = chunks >> c & 1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int position = number * kTile + 16 * c + 4 * grp + e;
          s[n][c][e] = held && position >= low[n] && position < high[n] ? s[n][c][e] * p.scale : -INFINITY;
          top[n] = fmaxf(top[n], s[n][c][e]);
        }
      }
      above |= top[n] > most[n] + kSlack;
    }
    if (__any(above)) {
#pragma unroll
      for (int n = 0; n < RT; ++n) {
        const float t = fmaxf(most[n], max_over_rows(top[n]));
        const float f = __builtin_amdgcn_exp2f(most[n] - t);
        most[n] = t;
        sum[n] *= f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][i][e] *= f;
      }
    }
    bf16x8 probs[RT][2][2];
#pragma unroll
    for (int n = 0; n < RT; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = __builtin_amdgcn_exp2f(s[n][c][e] - most[n]);
          sum[n] += x;
          const bf16_t rounded = static_cast<bf16_t>(x);
          probs[n][0][c / 2][c % 2 * 4 + e] = rounded;
          probs[n][1][c / 2][c % 2 * 4 + e] = static_cast<bf16_t>(x - static_cast<float>(rounded));
        }
    times_values<D, BITS, RT, 2>(tile, l16, grp, probs, acc);
  };

  p.pool.page_shift >= 6 ? walk<D, BITS, W, S, true>(p, job, span, wave, lane, stages, take) : walk<D, BITS, W, S, false>(p, job, span, wave, lane, stages, take);
  Met& meeting = *reinterpret_cast<Met*>(memory);  // in the place of the tiles
  __syncthreads();
#pragma unroll
  for (int n = 0; n < RT; ++n) {
    sum[n] += __shfl_xor(sum[n], 16, kWave);
    sum[n] += __shfl_xor(sum[n], 32, kWave);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) *reinterpret_cast<f32x4*>(&meeting.acc[wave][16 * n + l16][16 * i + 4 * grp]) = acc[n][i];
    if (grp == 0) meeting.most[wave][16 * n + l16] = most[n], meeting.sum[wave][16 * n + l16] = sum[n];
  }
  __syncthreads();
  meeting.leave(p, job, span);
}

// ---- the splits' parts --------------------------------------------------------------------------------------------

// A wavefront to a row: its lanes are 64 / (D / 4) groups that take the splits in turn.
template <typename T, int D>
__global__ __launch_bounds__(256) void cached_attention_join_kernel(const AttendParams p, int tile_rows, int waves) {
  constexpr int LANES = D / 4, GROUPS = kWave / LANES, AT_ONCE = 8;
  const int64_t out_row = static_cast<int64_t>(blockIdx.x) * (256 / kWave) + threadIdx.x / kWave;
  if (out_row >= p.all_rows) return;
  const int lane = threadIdx.x % kWave, c = lane % LANES * 4, group = lane / LANES;
  const int64_t token = out_row / p.T;
  const int t = static_cast<int>(out_row - token * p.T), b = static_cast<int>(token / p.H), h = static_cast<int>(token - static_cast<int64_t>(b) * p.H);
  const int head = p.group.over(h), row = t * p.group.d + h - head * p.group.d, row0 = row / tile_rows * tile_rows;
  const Span span = span_of(p, b, row0, min(tile_rows, p.rows - row0), 0, waves);
  if (span.active <= 1) return;
  const float* part = p.partial + out_row * p.splits.d * D + c;
  const float* stats = p.partial + p.all_rows * p.splits.d * D + out_row * p.splits.d * 2;
  float top = kNothing, l = 0.f;
  f32x4 total = {0.f, 0.f, 0.f, 0.f};
  for (int first = group; first < span.active; first += GROUPS * AT_ONCE) {
    f32x4 v[AT_ONCE];
    float most[AT_ONCE], sum[AT_ONCE], up = top;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {  // those behind the last count as the last once more, with no weight
      const int split = min(first + i * GROUPS, span.active - 1);
      v[i] = *reinterpret_cast<const f32x4*>(part + static_cast<int64_t>(split) * D);
      most[i] = stats[2 * split], sum[i] = stats[2 * split + 1];
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) up = fmaxf(up, most[i]);
    const float f = __builtin_amdgcn_exp2f(top - up);
    top = up, l *= f;
#pragma unroll
    for (int e = 0; e < 4; ++e) total[e] *= f;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const bool there = first + i * GROUPS < span.active;
      const float w = __builtin_amdgcn_exp2f(most[i] - top);
      l = there ? fmaf(w, sum[i], l) : l;
#pragma unroll
      for (int e = 0; e < 4; ++e) total[e] = there ? fmaf(w, v[i][e], total[e]) : total[e];
    }
  }
#pragma unroll
  for (int off = LANES; off < kWave; off *= 2) {
    const float other = __shfl_xor(top, off, kWave), up = fmaxf(top, other), f = __builtin_amdgcn_exp2f(top - up), g = __builtin_amdgcn_exp2f(other - up);
    const float other_l = __shfl_xor(l, off, kWave);
    top = up, l = l * f + other_l * g;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float other_total = __shfl_xor(total[e], off, kWave);
      total[e] = total[e] * f + other_total * g;
    }
  }
  Job job;
  job.head = head;
  if (group == 0) Place(p, job, row).template store<T>(p, b, c, total, l);
}

// ---- the host -----------------------------------------------------------------------------------------------------

#ifndef KALONE
#define KALONE 2048
#endif
constexpr int64_t kAlone = KALONE;
struct Plan {
  int tile_rows, row_tiles, splits, waves;
  uint32_t groups;
};
// The number of rows at a time decides nothing else: up to 4 rows are one tile in either form.
// Splits until there are four workgroups to a compute unit, as long as a split has a tile for each of its wavefronts.
Plan plan_of(int64_t B, int32_t heads, int32_t group, int32_t T, int64_t held, bool parts) {
  Plan plan;
  const int64_t rows = static_cast<int64_t>(group) * T;
  plan.tile_rows = rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 && !parts ? 4 : 16;
  plan.row_tiles = static_cast<int>((rows + plan.tile_rows - 1) / plan.tile_rows);
  const int64_t units = B * heads * plan.row_tiles;
  plan.waves = units >= kAlone ? 1 : 4;
  const int64_t most = held / (kTile * plan.waves),
                wanted = (4096 / plan.waves + units - 1) / (units > 0 ? units : 1);
  const int64_t splits = wanted < most ? wanted : most;
  plan.splits = static_cast<int>(splits < 1 ? 1 : splits);
  return plan;
}

// More than the 64 KB of LDS that a launch may have unasked.
template <typename Kernel>
void launch_with(Kernel* kernel, dim3 grid, int threads, int bytes, const AttendParams& p, hipStream_t s) {
  if (bytes > 65536) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  hipLaunchKernelGGL(kernel, grid, dim3(threads), bytes, s, p);
}
template <typename T, int D, int BITS, int ROWS, int W>
void launch_few(const AttendParams& p, dim3 grid, hipStream_t s) {
  constexpr int S = 2, BYTES = W * S * Staged<D, BITS>::BYTES + W * 8 * (kTile + 8) * 2;
  static_assert(sizeof(Meeting<T, D, ROWS, W>) <= W * S * Staged<D, BITS>::BYTES);
  launch_with(cached_attention_few_kernel<T, D, BITS, ROWS, W, S>, grid, W * kWave, BYTES, p, s);
}
template <typename T, int D, int BITS, int RT, int W>
void launch_many(const AttendParams& p, dim3 grid, hipStream_t s) {
  constexpr int S = 2, TILES = W * S * Staged<D, BITS>::BYTES, MET = sizeof(Meeting<T, D, 16 * RT, W>);
  launch_with(cached_attention_many_kernel<T, D, BITS, RT, W, S>, grid, W * kWave, TILES > MET ? TILES : MET, p, s);
}
template <typename T, int D, int BITS, int W>
void launch_attend(const AttendParams& p, const Plan& plan, hipStream_t s) {
  const dim3 grid(plan.groups);
  if (plan.tile_rows == 1) launch_few<T, D, BITS, 1, W>(p, grid, s);
  if (plan.tile_rows == 2) launch_few<T, D, BITS, 2, W>(p, grid, s);
  if constexpr (kParts<T> == 1) {
    if (plan.tile_rows == 4) launch_few<T, D, BITS, 4, W>(p, grid, s);
  }
  if (plan.tile_rows == 16) launch_many<T, D, BITS, 1, W>(p, grid, s);
}
template <typename T, int D, int BITS>
void launch_attend(const AttendParams& p, const Plan& plan, hipStream_t s) {
  if (plan.waves == 1) launch_attend<T, D, BITS, 1>(p, plan, s);
  if (plan.waves == 4) launch_attend<T, D, BITS, 4>(p, plan, s);
  if (p.splits.d > 1) {
    constexpr int ROWS = 256 / kWave;
    hipLaunchKernelGGL((cached_attention_join_kernel<T, D>), dim3(static_cast<uint32_t>((p.all_rows + ROWS - 1) / ROWS)), dim3(256), 0, s, p, plan.tile_rows, plan.waves);
  }
}
template <typename T>
void dispatch_attend(const AttendParams& p, const Plan& plan, int d, int bits, hipStream_t s) {
#define TAAC_ATTEND(D) \
  if (d == D) bits == 4 ? launch_attend<T, D, 4>(p, plan, s) : launch_attend<T, D, 8>(p, plan, s);
  TAAC_ATTEND(32) TAAC_ATTEND(64) TAAC_ATTEND(128)
#undef TAAC_ATTEND
}

}  // namespace
}  // namespace taac

extern "C" int64_t taac_cached_attention_workspace_bytes(int32_t B, int32_t H, int32_t heads, int32_t T, int32_t d, int64_t table_tokens) {
  using namespace taac;
  if (B < 0 || T < 0 || heads <= 0 || H <= 0 || H % heads != 0 || d <= 0 || table_tokens < 0) return -1;
  const Plan plan = plan_of(B, heads, H / heads, T, table_tokens, false);
  return plan.splits > 1 ? static_cast<int64_t>(B) * H * T * plan.splits * (d + 2) * 4 : 0;
}

extern "C" int taac_cached_attention_fwd(const void* q, void* o, const void* cache, int64_t pages, int32_t heads, int32_t page_tokens, int32_t d, int bits,
                                         const void* table, int table_int64, int64_t table_stride, int32_t table_pages, const int32_t* lengths,
                                         const int32_t* query_lengths, int32_t window, float scale, void* workspace, int64_t workspace_bytes, int32_t B,
                                         int32_t H, int32_t T, const int64_t q_strides[3], const int64_t o_strides[3], int dtype, void* stream) {
  using namespace taac;
  const char* name = "taac_cached_attention_fwd";
  AttendParams p{};
  if (B < 0 || T < 0 || H <= 0 || heads <= 0 || H % heads != 0)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: query heads must be a multiple of the cache's, sizes not negative", name);
  if (int rc = take_kv_pool(name, p.pool, const_cast<void*>(cache), pages, heads, page_tokens, d, bits, table, table_int64, table_stride, table_pages, B > 0))
    return rc;
  if (dtype != TAAC_BF16 && dtype != TAAC_F16) return set_error(TAAC_ERR_INVALID_VALUE, "%s: queries must be bf16 or fp16 (dtype %d)", name, dtype);
  if (window < 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: the window must not be negative", name);
  if (q_strides == nullptr || o_strides == nullptr) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null strides", name);
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = q_strides[i], p.os[i] = o_strides[i];
    if (p.qs[i] % 8 != 0 || p.os[i] % 4 != 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: strides of q must be multiples of 8, those of o of 4", name);
  }
  if (B == 0 || T == 0) return TAAC_OK;
  if (!q || !o || !lengths) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null tensor pointer", name);
  if (!aligned16(q) || reinterpret_cast<uintptr_t>(o) % 8 != 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: q must be 16-byte aligned, o 8-byte", name);
  if (pages == 0) p.pool.table_pages = 0;  // nothing is cached
  const int64_t held = static_cast<int64_t>(p.pool.table_pages) * page_tokens;
  const int group = H / heads;
  // token numbers of 32 bits, a wavefront's tiles behind the last among them
  if (held > int64_t{1} << 30) return set_error(TAAC_ERR_UNSUPPORTED, "%s: at most 2^30 tokens to a sample", name);
  if (static_cast<int64_t>(group) * T > 1 << 24) return set_error(TAAC_ERR_UNSUPPORTED, "%s: too many queries to a key head", name);
  Plan plan = plan_of(B, heads, group, T, held, dtype == TAAC_F16);
  const int64_t groups = static_cast<int64_t>(B) * heads * plan.row_tiles * plan.splits;
  if (groups > 1 << 23) return set_error(TAAC_ERR_UNSUPPORTED, "%s: too many workgroups", name);
  plan.groups = static_cast<uint32_t>(groups);
  p.all_rows = static_cast<int64_t>(B) * H * T;
  const int64_t need = plan.splits > 1 ? p.all_rows * plan.splits * (d + 2) * 4 : 0;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: workspace must hold %lld bytes, 16-byte aligned", name, (long long)need);
  p.q = q, p.o = o, p.lengths = lengths, p.query_lengths = query_lengths, p.partial = static_cast<float*>(workspace);
  p.group = divisor(group), p.splits = divisor(plan.splits), p.row_tiles = divisor(plan.row_tiles), p.heads = divisor(heads);
  p.H = H, p.T = T, p.rows = group * T, p.window = window;
  p.scale = scale * 1.4426950408889634f;
  if (dtype == TAAC_BF16) dispatch_attend<bf16_t>(p, plan, d, bits, as_stream(stream));
  else dispatch_attend<f16_t>(p, plan, d, bits, as_stream(stream));
  return check_launch(name);
}
