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

namespace taac {
namespace {

struct AttendParams {
  KvPool pool;
  const void* q;
  void* o;
  const int32_t* lengths;        // [B]: cached tokens, the new ones among them
  const int32_t* query_lengths;  // [B] or null: T
  float* partial;                // [row][split][D], then [row][split] of (maximum, sum)
  int64_t qs[3], os[3];          // element strides of (batch, head, token)
  int64_t all_rows;              // B * heads * T
  int32_t B, H, group, T, rows, row_tiles, splits, window;
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
  const int t0 = row0 / p.group, t1 = min((row0 + rows - 1) / p.group, s.news - 1);
  const int base = s.length - s.news;  // of the sample's first query; below zero where it has more queries than tokens
  int64_t high = static_cast<int64_t>(base) + t1 + 1, low = p.window > 0 ? static_cast<int64_t>(base) + t0 + 1 - p.window : 0;
  high = high < held ? high : held;
  low = low > 0 ? low : 0;
  if (t1 < t0 || high <= low) {
    s.first = s.end = s.active = 0;
    return s;
  }
  const int t_first = static_cast<int>(low / kTile), t_end = static_cast<int>((high + kTile - 1) / kTile);
  int each = (t_end - t_first + p.splits - 1) / p.splits;
  each = (each + waves - 1) / waves * waves;
  s.active = (t_end - t_first + each - 1) / each;
  s.first = min(t_first + split * each, t_end);
  s.end = min(s.first + each, t_end);
  return s;
}
// The positions that a row sees.
struct Seen {
  int low, high;
  __device__ __forceinline__ Seen(const AttendParams& p, const Span& s, int row) {
    const int t = row / p.group, place = s.length - s.news + t;
    const bool there = row < p.rows && t < s.news;
    high = there ? place + 1 : 0;
    low = p.window > 0 && place + 1 > p.window ? place + 1 - p.window : 0;
  }
};

// Which workgroup is which: splits next to each other, then row tiles, key heads, samples.
struct Job {
  int b, head, row0, split;
  __device__ __forceinline__ Job(const AttendParams& p, int rows) {
    uint32_t id = blockIdx.x;
    split = id % p.splits;
    id /= p.splits;
    row0 = static_cast<int>(id % p.row_tiles) * rows;
    id /= p.row_tiles;
    head = id % p.pool.heads;
    b = id / p.pool.heads;
  }
};

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
        const float f = W == 1 ? 1.f : exp2f(most[w][r] - top);
        l += f * sum[w][r];
#pragma unroll
        for (int e = 0; e < 4; ++e) total[e] = fmaf(f, acc[w][r][c + e], total[e]);
      }
      const int t = row / p.group, h = job.head * p.group + row % p.group;
      const int64_t out_row = (static_cast<int64_t>(job.b) * p.H + h) * p.T + t;
      if (span.active > 1) {
        float* part = p.partial + (out_row * p.splits + job.split) * D + c;
        *reinterpret_cast<f32x4*>(part) = total;
        if (c == 0) {
          float* stats = p.partial + p.all_rows * p.splits * D + (out_row * p.splits + job.split) * 2;
          stats[0] = top, stats[1] = l;
        }
        continue;
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      typename Vec8<T>::half_type v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = static_cast<T>(total[e] * inv);
      *reinterpret_cast<typename Vec8<T>::half_type*>(static_cast<T*>(p.o) + job.b * p.os[0] + h * p.os[1] + t * p.os[2] + c) = v;
    }
  }
  __device__ __forceinline__ void clear(const AttendParams& p, const Job& job) {
    for (int i = threadIdx.x; i < ROWS * (D / 4); i += W * kWave) {
      const int r = i / (D / 4), c = i % (D / 4) * 4, row = job.row0 + r;
      if (row >= p.rows) continue;
      const int t = row / p.group, h = job.head * p.group + row % p.group;
      const typename Vec8<T>::half_type v = {};
      *reinterpret_cast<typename Vec8<T>::half_type*>(static_cast<T*>(p.o) + job.b * p.os[0] + h * p.os[1] + t * p.os[2] + c) = v;
    }
  }
};

// Where the records of a tile's four chunks are: a lane of group g knows that of chunk g.
struct Records {
  int64_t page;  // of the lane's chunk
  __device__ __forceinline__ void find(const AttendParams& p, int b, int tile, int grp) {
    page = kv_page(p.pool, b, (static_cast<int64_t>(tile) * kTile + kKvChunk * grp) >> p.pool.page_shift);
  }
  // In the place of a record that there is not: the first one of the pool, whose tokens are then masked.
  __device__ __forceinline__ int64_t offset(const AttendParams& p, int head, int tile, int grp, int record_bytes) const {
    const int chunk = (tile * (kTile / kKvChunk) + grp) & ((1 << (p.pool.page_shift - 4)) - 1);
    return page < 0 ? 0 : kv_record(p.pool, page, head, chunk, record_bytes);
  }
};
__device__ __forceinline__ int64_t from_lane(int64_t v, int lane) {
  const uint32_t low = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), lane), high = __builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), lane);
  return static_cast<int64_t>(static_cast<uint64_t>(high) << 32 | low);
}

template <int D, int BITS>
struct Values {
  static constexpr int BLOCKS = D / kKvBlock;
  Words<BLOCKS * BITS / 4> codes[4];
  Words<BLOCKS> scales[4];
  __device__ __forceinline__ void load(int c, const uint8_t* record, int l16, int grp) {
    codes[c].load(record + kv_value_at(D, BITS) + (l16 * 4 + grp) * BLOCKS * BITS);
    scales[c].load(record + kv_value_scale_at(D, BITS) + grp * BLOCKS * 4);
  }
};

// acc[rows of 16 features] += values^T p: probs[n][part][half]: of 32 tokens, group grp those of chunk 2 half at 4 grp, then those of the next chunk.
template <int D, int BITS, int RT, int PARTS>
__device__ __forceinline__ void times_values(const Values<D, BITS>& v, const bf16x8 (&probs)[RT][PARTS][2], f32x4 (&acc)[RT][D / 16]) {
  constexpr int BLOCKS = D / kKvBlock, EACH = BITS / 4;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) {
      uint32_t a0[2], a1[2], b0[2], b1[2];
      four_tokens<BITS>(v.codes[2 * half].w + j * EACH, v.scales[2 * half].w[j], a0, a1);
      four_tokens<BITS>(v.codes[2 * half + 1].w + j * EACH, v.scales[2 * half + 1].w[j], b0, b1);
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

// ---- up to four rows ----------------------------------------------------------------------------------------------

template <int D, int BITS>
struct FewTile {
  static constexpr int BLOCKS = D / kKvBlock;
  Words<BITS> keys[BLOCKS];  // the lane's token
  uint32_t key_scales;
  Values<D, BITS> values;
  bool held;
  __device__ __forceinline__ void load(const AttendParams& p, const Records& at, int head, int tile, int l16, int grp) {
    constexpr int RECORD = kv_record_bytes(D, BITS);
    held = at.page >= 0;
    const int64_t mine = at.offset(p, head, tile, grp, RECORD);
    const uint8_t* record = p.pool.data + mine;
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) keys[j].load(record + j * (kKvChunk * 4 * BITS) + l16 * 4 * BITS);
    const uint8_t* scales = record + kv_key_scale_at(D, BITS) + l16 * BLOCKS;
    if constexpr (BLOCKS == 1) key_scales = *scales;
    if constexpr (BLOCKS == 2) key_scales = *reinterpret_cast<const uint16_t*>(scales);
    if constexpr (BLOCKS == 4) key_scales = *reinterpret_cast<const uint32_t*>(scales);
#pragma unroll
    for (int c = 0; c < 4; ++c) values.load(c, p.pool.data + from_lane(mine, 16 * c), l16, grp);
  }
};

template <typename T, int D, int BITS, int ROWS, int W>
__global__ __launch_bounds__(W * kWave) void cached_attention_few_kernel(const AttendParams p) {
  constexpr int BLOCKS = D / kKvBlock, SLOT = kTile + 8, PARTS = kParts<T>;
  __shared__ Meeting<T, D, ROWS, W> meeting;
  __shared__ bf16_t turned[W][8][SLOT];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, l16 = lane % 16, grp = lane / 16;
  const Job job(p, ROWS);
  const Span span = span_of(p, job.b, job.row0, ROWS, job.split, W);
  if (job.split >= span.active) {
    if (job.split == 0) meeting.clear(p, job);
    return;
  }
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
    const T* src = static_cast<const T*>(p.q);
    if (mine) src += job.b * p.qs[0] + (job.head * p.group + row % p.group) * p.qs[1] + (row / p.group) * p.qs[2];
#pragma unroll
    for (int o = 0; o < D / 8; ++o) {
      q[o] = bf16x8{};
      if (mine) q[o] = query_part<T>(src + 8 * o, part);
    }
  }
  float most[ROWS], sum[ROWS];
  f32x4 acc[1][D / 16];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) most[r] = kNothing, sum[r] = 0.f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) acc[0][i] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto take = [&](const FewTile<D, BITS>& tile, int number) __attribute__((always_inline)) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    // a NaN would reach the lanes of the other groups, whose products with it are zeros: it waits for the scores
    const bool finite = (tile.key_scales & 255u) != kKvNotFinite;
    const uint32_t scales = finite ? tile.key_scales : 0u;
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) {
      const float scale = j == 0 ? scale_of<0>(scales) : j == 1 ? scale_of<1>(scales) : j == 2 ? scale_of<2>(scales) : scale_of<3>(scales);
#pragma unroll
      for (int i = 0; i < 4; ++i) s = mfma(q[4 * j + i], eight<BITS>(tile.keys[j].w + i * (BITS / 4), scale), s);
    }
    const int position = number * kTile + lane;
    float score[ROWS];
    bool above = false;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float x = finite ? (PARTS == 2 ? s[r] + s[2 + r] : s[r]) * p.scale : __builtin_nanf("");
      score[r] = tile.held && position >= low[r] && position < high[r] ? x : -INFINITY;
      above |= score[r] > most[r] + kSlack;
    }
    if (__any(above)) {
      float mine = 1.f;  // the factor of this lane's column of acc
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const float top = fmaxf(most[r], group_max<kWave>(score[r])), f = exp2f(most[r] - top);
        most[r] = top;
        sum[r] *= f;
        mine = l16 % 4 == r ? f : mine;
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[0][i][e] *= mine;
    }
    // token 16 grp + l16 lies in chunk grp, group l16 / 4
    bf16_t* to = &turned[wave][0][l16 / 4 * 16 + grp * 4 + l16 % 4];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float x = exp2f(score[r] - most[r]);
      sum[r] += x;
      const bf16_t rounded = static_cast<bf16_t>(x);
      to[r * SLOT] = rounded;
      to[(4 + r) * SLOT] = static_cast<bf16_t>(x - static_cast<float>(rounded));
    }
    wave_sync();
    bf16x8 probs[1][1][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) probs[0][0][half] = *reinterpret_cast<const bf16x8*>(&turned[wave][l16 % 8][grp * 16 + half * 8]);
    wave_sync();
    times_values<D, BITS, 1, 1>(tile.values, probs, acc);
  };

  FewTile<D, BITS> even, odd;
  Records at;
  int tile = span.first + wave;
  if (tile < span.end) {
    at.find(p, job.b, tile, grp);
    even.load(p, at, job.head, tile, l16, grp);
    at.find(p, job.b, tile + W, grp);
  }
  while (tile < span.end) {
    if (tile + W < span.end) odd.load(p, at, job.head, tile + W, l16, grp);
    at.find(p, job.b, tile + 2 * W, grp);
    take(even, tile);
    tile += W;
    if (tile >= span.end) break;
    if (tile + W < span.end) even.load(p, at, job.head, tile + W, l16, grp);
    at.find(p, job.b, tile + 2 * W, grp);
    take(odd, tile);
    tile += W;
  }
  // the two parts of the probabilities stand in columns r and 4 + r
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[0][i][e] += __shfl_xor(acc[0][i][e], 4, kWave);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) sum[r] = group_sum<kWave>(sum[r]);
  if (l16 < ROWS) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) *reinterpret_cast<f32x4*>(&meeting.acc[wave][l16][16 * i + 4 * grp]) = acc[0][i];
  }
  if (lane == 0) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) meeting.most[wave][r] = most[r], meeting.sum[wave][r] = sum[r];
  }
  __syncthreads();
  meeting.leave(p, job, span);
}

// ---- sixteen rows at a time ---------------------------------------------------------------------------------------

template <int D, int BITS>
struct ManyTile {
  static constexpr int BLOCKS = D / kKvBlock;
  Words<BLOCKS * BITS / 4> keys[4];  // of token l16 of each chunk: features D / 4 grp ..
  uint32_t key_scales[4];
  Values<D, BITS> values;
  uint64_t held;
  __device__ __forceinline__ void load(const AttendParams& p, const Records& at, int head, int tile, int l16, int grp) {
    constexpr int RECORD = kv_record_bytes(D, BITS);
    held = __ballot(at.page >= 0);
    const int64_t mine = at.offset(p, head, tile, grp, RECORD);
    const int octet = grp * BLOCKS, block = octet / 4;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint8_t* record = p.pool.data + from_lane(mine, 16 * c);
      keys[c].load(record + block * (kKvChunk * 4 * BITS) + l16 * 4 * BITS + octet % 4 * BITS);
      key_scales[c] = record[kv_key_scale_at(D, BITS) + l16 * BLOCKS + block];
      values.load(c, record, l16, grp);
    }
  }
};

template <typename T, int D, int BITS, int RT, int W>
__global__ __launch_bounds__(W * kWave) void cached_attention_many_kernel(const AttendParams p) {
  constexpr int BLOCKS = D / kKvBlock, ROWS = 16 * RT, PARTS = kParts<T>;
  __shared__ Meeting<T, D, ROWS, W> meeting;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, l16 = lane % 16, grp = lane / 16;
  const Job job(p, ROWS);
  const Span span = span_of(p, job.b, job.row0, min(ROWS, p.rows - job.row0), job.split, W);
  if (job.split >= span.active) {
    if (job.split == 0) meeting.clear(p, job);
    return;
  }
  int low[RT], high[RT];
  bf16x8 q[RT][PARTS][BLOCKS];
#pragma unroll
  for (int n = 0; n < RT; ++n) {
    const int row = job.row0 + 16 * n + l16;
    const Seen seen(p, span, row);
    low[n] = seen.low, high[n] = seen.high;
    const T* src = static_cast<const T*>(p.q);
    if (row < p.rows) src += job.b * p.qs[0] + (job.head * p.group + row % p.group) * p.qs[1] + (row / p.group) * p.qs[2];
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

  auto take = [&](const ManyTile<D, BITS>& tile, int number) __attribute__((always_inline)) {
    f32x4 s[RT][4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int n = 0; n < RT; ++n) s[n][c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < BLOCKS; ++j) {
        const bf16x8 key = eight<BITS>(tile.keys[c].w + j * (BITS / 4), scale_of<0>(tile.key_scales[c]));
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
        const bool held = tile.held >> (16 * c) & 1;
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
        float t = fmaxf(top[n], __shfl_xor(top[n], 16, kWave));
        t = fmaxf(most[n], fmaxf(t, __shfl_xor(t, 32, kWave)));
        const float f = exp2f(most[n] - t);
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
          const float x = exp2f(s[n][c][e] - most[n]);
          sum[n] += x;
          const bf16_t rounded = static_cast<bf16_t>(x);
          probs[n][0][c / 2][c % 2 * 4 + e] = rounded;
          probs[n][1][c / 2][c % 2 * 4 + e] = static_cast<bf16_t>(x - static_cast<float>(rounded));
        }
    times_values<D, BITS, RT, 2>(tile.values, probs, acc);
  };

  ManyTile<D, BITS> even, odd;
  Records at;
  int tile = span.first + wave;
  if (tile < span.end) {
    at.find(p, job.b, tile, grp);
    even.load(p, at, job.head, tile, l16, grp);
    at.find(p, job.b, tile + W, grp);
  }
  while (tile < span.end) {
    if (tile + W < span.end) odd.load(p, at, job.head, tile + W, l16, grp);
    at.find(p, job.b, tile + 2 * W, grp);
    take(even, tile);
    tile += W;
    if (tile >= span.end) break;
    if (tile + W < span.end) even.load(p, at, job.head, tile + W, l16, grp);
    at.find(p, job.b, tile + 2 * W, grp);
    take(odd, tile);
    tile += W;
  }
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

template <typename T, int D>
__global__ __launch_bounds__(256) void cached_attention_join_kernel(const AttendParams p, int tile_rows, int waves) {
  constexpr int LANES = D / 4;
  const int64_t out_row = static_cast<int64_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
  if (out_row >= p.all_rows) return;
  const int c = threadIdx.x % LANES * 4, t = static_cast<int>(out_row % p.T), h = static_cast<int>(out_row / p.T % p.H), b = static_cast<int>(out_row / p.T / p.H);
  const int row0 = (t * p.group + h % p.group) / tile_rows * tile_rows;
  const Span span = span_of(p, b, row0, min(tile_rows, p.rows - row0), 0, waves);
  if (span.active <= 1) return;
  const float* part = p.partial + out_row * p.splits * D + c;
  const float* stats = p.partial + p.all_rows * p.splits * D + out_row * p.splits * 2;
  float top = kNothing, l = 0.f;
  for (int i = 0; i < span.active; ++i) top = fmaxf(top, stats[2 * i]);
  f32x4 total = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < span.active; ++i) {
    const float f = exp2f(stats[2 * i] - top);
    const f32x4 v = *reinterpret_cast<const f32x4*>(part + static_cast<int64_t>(i) * D);
    l = fmaf(f, stats[2 * i + 1], l);
#pragma unroll
    for (int e = 0; e < 4; ++e) total[e] = fmaf(f, v[e], total[e]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  typename Vec8<T>::half_type v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = static_cast<T>(total[e] * inv);
  *reinterpret_cast<typename Vec8<T>::half_type*>(static_cast<T*>(p.o) + b * p.os[0] + h * p.os[1] + t * p.os[2] + c) = v;
}

// ---- the host -----------------------------------------------------------------------------------------------------

constexpr int kWaves = 4;

struct Plan {
  int tile_rows, row_tiles, splits;
};
// The number of rows at a time decides nothing else: up to 4 rows are one tile in either form.
// Splits until there are four workgroups to a compute unit, as long as a split has a tile for each of its wavefronts.
Plan plan_of(int64_t B, int32_t heads, int32_t group, int32_t T, int64_t held, bool parts) {
  Plan plan;
  const int64_t rows = static_cast<int64_t>(group) * T;
  plan.tile_rows = rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 && !parts ? 4 : 16;
  plan.row_tiles = static_cast<int>((rows + plan.tile_rows - 1) / plan.tile_rows);
  const int64_t units = B * heads * plan.row_tiles, most = held / (kTile * kWaves), wanted = (1024 + units - 1) / (units > 0 ? units : 1);
  const int64_t splits = wanted < most ? wanted : most;
  plan.splits = static_cast<int>(splits < 1 ? 1 : splits);
  return plan;
}

template <typename T, int D, int BITS>
void launch_attend(const AttendParams& p, const Plan& plan, hipStream_t s) {
  const dim3 grid(static_cast<uint32_t>(static_cast<int64_t>(p.B) * p.pool.heads * p.row_tiles * p.splits)), block(kWaves * kWave);
  if (plan.tile_rows == 1) hipLaunchKernelGGL((cached_attention_few_kernel<T, D, BITS, 1, kWaves>), grid, block, 0, s, p);
  if (plan.tile_rows == 2) hipLaunchKernelGGL((cached_attention_few_kernel<T, D, BITS, 2, kWaves>), grid, block, 0, s, p);
  if constexpr (kParts<T> == 1) {
    if (plan.tile_rows == 4) hipLaunchKernelGGL((cached_attention_few_kernel<T, D, BITS, 4, kWaves>), grid, block, 0, s, p);
  }
  if (plan.tile_rows == 16) hipLaunchKernelGGL((cached_attention_many_kernel<T, D, BITS, 1, kWaves>), grid, block, 0, s, p);
  if (p.splits > 1) {
    constexpr int ROWS = 256 / (D / 4);
    hipLaunchKernelGGL((cached_attention_join_kernel<T, D>), dim3(static_cast<uint32_t>((p.all_rows + ROWS - 1) / ROWS)), dim3(256), 0, s, p, plan.tile_rows, kWaves);
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
  const Plan plan = plan_of(B, heads, group, T, held, dtype == TAAC_F16);
  const int64_t groups = static_cast<int64_t>(B) * heads * plan.row_tiles * plan.splits;
  if (groups > 1 << 23) return set_error(TAAC_ERR_UNSUPPORTED, "%s: too many workgroups", name);
  p.all_rows = static_cast<int64_t>(B) * H * T;
  const int64_t need = plan.splits > 1 ? p.all_rows * plan.splits * (d + 2) * 4 : 0;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: workspace must hold %lld bytes, 16-byte aligned", name, (long long)need);
  p.q = q, p.o = o, p.lengths = lengths, p.query_lengths = query_lengths, p.partial = static_cast<float*>(workspace);
  p.B = B, p.H = H, p.group = group, p.T = T, p.rows = group * T, p.row_tiles = plan.row_tiles, p.splits = plan.splits, p.window = window;
  p.scale = scale * 1.4426950408889634f;
  if (dtype == TAAC_BF16) dispatch_attend<bf16_t>(p, plan, d, bits, as_stream(stream));
  else dispatch_attend<f16_t>(p, plan, d, bits, as_stream(stream));
  return check_launch(name);
}
