// Attention of a few new tokens of many sequences over keys and values that lie quantised in a pool of pages (the format: kv_cache.h).
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j   over the positions j that query i sees: up to its own, with a window only the last of them.
//
// The new tokens of a sample are the last of its cached ones. Queries of the heads that share a key head are rows of one product.
//
// Bound by HBM: every code is read once per key head. A wavefront walks tiles of 64 tokens, which come into LDS without registers, with the running maximum and sum of a
// softmax; the wavefronts of a workgroup take the tiles in turn and meet at its end; long histories of few heads are split over workgroups, whose parts
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
// and sums are fp32. Probabilities enter as parts of eight bits: three in the first form, in columns that would be empty, so that they keep the digits of fp32; two in the
// other, where a third would be half as many products with the values again, and outputs of 16 bits are off by their own rounding either way. The maximum moves when a score exceeds it
// by a factor of 2^8, which cancels.
//
// Measured: 4 samples of 65536 tokens, 32 heads over 8 of 128 features in 4 bits: 51 us and 5 for the join, 5.6 TB/s of the cache (tiles in registers, one ahead: 101, for the
// registers left one wavefront to a SIMD, and page numbers that wait behind the rows). 1024 samples of up to 512 tokens, 8 heads of 32: 23 us; of one tile each 9.5,
// and 2.8 every tile more, 6.4 TB/s. 64 samples of 2048 tokens, 24 queries of 8 heads over 4 of 128 in 8 bits: 34 us, of up to 2048 tokens and up to 24
// queries 27. A tile of 32 rows has 104 matrix and some 530 vector instructions there, of which 270 convert the codes; those of one wavefront do not overlap (six products with three
// additions behind each take 184 cycles, the products alone 120, the additions alone 72), those of two do in part. The end of a
// workgroup (its wavefronts' sums joined, divided, written) is shared by all of them: done by the first one it took half of a call with one tile of 48 rows, 7 of 15 us.
#pragma once

#include "kv_cache.h"
#include "ts_common.h"

namespace taac {

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
  int32_t first;                 // sample of the launch
  float scale;                   // times log2 e: powers of two; its size
  uint32_t flip, keep;           // its sign, which the queries take, of two of their elements; nothing of them where it is zero (scale is one then)
};

namespace {

constexpr int kTile = 64;          // tokens
// A kernel's shape, by the rows of a workgroup - 1, 2 or 4 (one form), 16, 32 or 48 (the other) - and its wavefronts: 1, 4, or 8.
struct Shape {
  int waves;
  int stages;    // tiles of a wavefront in LDS; one: keys and values by themselves
  int per_simd;  // wavefronts that the registers leave room for
};
__host__ __device__ constexpr Shape shape_of(int rows, int d, int waves) {
  if (rows <= 4) return {waves, 2, d == 32 ? 6 : d == 64 ? 4 : 2};
  if (waves == 8) return {waves, 1, 2};
  if (rows == 16) return {waves, 1, d == 32 ? 6 : d == 64 ? 4 : 3};
  return {waves, 1, d == 32 ? 4 : d == 64 ? 3 : 2};
}
__host__ __device__ constexpr int tile_bytes(int d, int bits) { return (4 * kv_record_bytes(d, bits) + 1023) / 1024 * 1024; }
__host__ __device__ constexpr int half_bytes(int d, int bits) { return 4 * kv_key_bytes(d, bits) + 4 * kWave; }
// Queries of more than sixteen rows lie in LDS: their registers are what a second wavefront to a SIMD needs. Not those in two parts: twice the bytes are what a second
// workgroup needs.
__host__ __device__ constexpr bool queries_in_lds(int rows, int parts) { return rows > 16 && parts == 1; }
// Bytes that `waves` wavefronts with n fours of features in each lane leave for each other where they meet, in the first of two places and every second time, or in
// the second.
__host__ __device__ constexpr int meeting_bytes(int n, int waves, bool second) {
  int most = 0;
  for (int half = waves / 2, level = 0; half > 0; half /= 2, ++level) {
    const int given = n % 2 == 0 ? n / 2 : n;
    if ((level % 2 == 1) == second && waves * given * kWave * 16 > most) most = waves * given * kWave * 16;
    n = given;
  }
  return most;
}
// Whether fewer columns than a workgroup's find room where all of them do.
__host__ __device__ constexpr bool meeting_fits(int n, int waves, int each, int bytes) {
  for (; n > 0; n -= each)
    if (meeting_bytes(n, waves, false) + meeting_bytes(n, waves, true) > bytes) return false;
  return true;
}
__host__ __device__ constexpr int stats_bytes(int rows, int waves) { return waves > 1 ? waves * (rows <= 16 ? 16 : rows) * 8 : 0; }
// of the tiles, or of the meeting behind them; then the queries and the statistics
__host__ __device__ constexpr int working_bytes(int rows, int d, int bits, int waves) {
  const Shape shape = shape_of(rows, d, waves);
  const int tiles = shape.waves * (rows <= 4 ? shape.stages * tile_bytes(d, bits) + 3 * rows * (kTile + 8) * 2 : 2 * half_bytes(d, bits));
  const int fours = (rows <= 16 ? 1 : rows / 16) * (d / 16), meeting = meeting_bytes(fours, shape.waves, false) + meeting_bytes(fours, shape.waves, true);
  return tiles > meeting ? tiles : meeting;
}
__host__ __device__ constexpr int lds_bytes(int rows, int d, int bits, int parts, int waves) {
  return working_bytes(rows, d, bits, waves) + (queries_in_lds(rows, parts) ? rows * d * 2 : 0) + stats_bytes(rows, shape_of(rows, d, waves).waves);
}
constexpr float kNothing = -3.402823466e38f;  // the maximum of no scores: no finite one is below
constexpr float kSlack = 8.f;
constexpr float kFar = 1048576.f;  // a maximum whose own rounding, half of 2^-3, is what a product that is not rounded may differ by from it

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// Two values of a word of codes.
template <int BITS, int I>
__device__ __forceinline__ uint32_t two(uint32_t w, float scale) {
  if constexpr (BITS == 4) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, I));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, I != 0));
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
// Eight probabilities as two parts of bf16.
__device__ __forceinline__ void two_parts(const f32x4& a, const f32x4& b, bf16x8& high, bf16x8& low) {
  const u32x4 h = {round2(a[0], a[1]), round2(a[2], a[3]), round2(b[0], b[1]), round2(b[2], b[3])};
  const u32x4 l = {rest2(a[0], a[1], h[0]), rest2(a[2], a[3], h[1]), rest2(b[0], b[1], h[2]), rest2(b[2], b[3], h[3])};
  high = __builtin_bit_cast(bf16x8, h), low = __builtin_bit_cast(bf16x8, l);
}

// Eight neighbours of a row of queries, in one part of bf16, or two for fp16, whose eleven bits they hold.
template <typename T>
constexpr int kParts = sizeof(T) == 2 && !__is_same(T, bf16_t) ? 2 : 1;
template <typename T>
__device__ __forceinline__ bf16x8 query_part(const T* p, int part, uint32_t flip, uint32_t keep) {
  const typename Vec8<T>::type v = __builtin_bit_cast(typename Vec8<T>::type, (*reinterpret_cast<const u32x4*>(p) ^ flip) & keep);
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
    // row tiles of a key head read the same records: on one die they meet in its L2
    int id = p.row_tiles.d > 1 ? xcd_remap(blockIdx.x, gridDim.x) : blockIdx.x, over = p.splits.over(id);
    split = id - over * p.splits.d;
    id = over, over = p.row_tiles.over(id);
    row0 = (id - over * p.row_tiles.d) * rows;
    b = p.heads.over(over);
    head = over - b * p.heads.d;
    b += p.first;
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
  template <typename T>
  __device__ __forceinline__ T* output(const AttendParams& p, int b) const {
    return static_cast<T*>(p.o) + b * p.os[0] + h * p.os[1] + t * p.os[2];
  }
};
template <typename T>
__device__ __forceinline__ void store_four(T* to, const f32x4& total, float inv) {
  typename Vec8<T>::half_type v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = static_cast<T>(total[e] * inv);
  *reinterpret_cast<typename Vec8<T>::half_type*>(to) = v;
}

// C fours of features of a lane's columns, from the `from`th of RT columns' D / 16 on: to the output, or to the split's part. sum, top: the columns' sums of weights and the
// maxima that all refer to.
template <typename T, int D, int RT, int C>
__device__ __forceinline__ void leave(const AttendParams& p, const Job& job, const Span& span, int from, int l16, int grp, const f32x4* part, const float (&sum)[RT],
                                      const float (&top)[RT]) {
  const float sum1 = sum[RT > 1 ? 1 : 0], sum2 = sum[RT > 2 ? 2 : 0], top1 = top[RT > 1 ? 1 : 0], top2 = top[RT > 2 ? 2 : 0];
  constexpr int EACH = C < D / 16 ? C : D / 16, FOURS = D / 16 % C == 0 || C % (D / 16) == 0 ? EACH : 1;  // of the same column
#pragma unroll
  for (int e = 0; e < C; e += FOURS) {
    const int n = (from + e) / (D / 16), row = job.row0 + 16 * n + l16, c = (from + e) % (D / 16) * 16 + 4 * grp;
    if (row >= p.rows) continue;
    const float l = n == 0 ? sum[0] : n == 1 ? sum1 : sum2, most = n == 0 ? top[0] : n == 1 ? top1 : top2;
    const Place place(p, job, row);
    if (span.active > 1 && place.t < span.news) {  // rows of no query are zeros whoever writes them
      const int64_t at = ((static_cast<int64_t>(job.b) * p.H + place.h) * p.T + place.t) * p.splits.d + job.split;
#pragma unroll
      for (int i = 0; i < FOURS; ++i) *reinterpret_cast<f32x4*>(p.partial + at * D + c + 16 * i) = part[e + i];
      if (c == 0) {
        float* stats = p.partial + p.all_rows * p.splits.d * D + at * 2;
        stats[0] = most, stats[1] = l;
      }
    } else {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      T* to = place.output<T>(p, job.b) + c;
#pragma unroll
      for (int i = 0; i < FOURS; ++i) store_four<T>(to + 16 * i, part[e + i], inv);
    }
  }
}

// The wavefronts' sums of the same rows. Those HALF apart give each other the half that the other one keeps, so that each ends with a part of its own, from
// the `from`th four on; an odd number is given as a whole, and the giver is done.
template <int N, int HALF, int M>
__device__ __forceinline__ void gather(f32x4* place, f32x4* other_place, int wave, int lane, f32x4 (&acc)[M], int& from, bool& there) {
  if constexpr (HALF > 0) {
    constexpr bool SPLIT = N % 2 == 0;
    constexpr int GIVEN = SPLIT ? N / 2 : N;
    const bool upper = wave & HALF;
    if (there && (SPLIT || upper)) {
#pragma unroll
      for (int i = 0; i < GIVEN; ++i) {
        const f32x4 low = acc[i], high = acc[SPLIT ? GIVEN + i : i];
        place[(wave * GIVEN + i) * kWave + lane] = upper ? low : high;
      }
    }
    __syncthreads();
    there &= SPLIT || !upper;
    if (there) {
#pragma unroll
      for (int i = 0; i < GIVEN; ++i) {
        const f32x4 other = place[((wave ^ HALF) * GIVEN + i) * kWave + lane], low = acc[i], high = acc[SPLIT ? GIVEN + i : i];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] = (upper ? high[e] : low[e]) + other[e];
      }
    }
    if (SPLIT && upper) from += GIVEN;
    gather<GIVEN, HALF / 2>(other_place, place, wave, lane, acc, from, there);
  }
}
__host__ __device__ constexpr int gathered(int n, int waves) {
  for (int half = waves / 2; half > 0; half /= 2) n = n % 2 == 0 ? n / 2 : n;
  return n;
}

// A workgroup's end: its wavefronts' statistics, then their sums under the common maxima, then what each leaves of them.
template <typename T, int D, int RT, int W>
__device__ __forceinline__ void finish(const AttendParams& p, const Job& job, const Span& span, uint8_t* memory, float* stats, int wave, int lane, f32x4 (&acc)[RT * (D / 16)],
                                       float (&sum)[RT], float (&top)[RT]) {
  constexpr int N = RT * (D / 16), C = gathered(N, W);
  const int l16 = lane % 16, grp = lane / 16;
  int from = 0;
  bool there = true;
  if constexpr (W > 1) {
    typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2;
    f32x2* const all = reinterpret_cast<f32x2*>(stats);  // [wavefront][row]
    if (grp == 0) {
#pragma unroll
      for (int n = 0; n < RT; ++n) all[wave * (RT * 16) + n * 16 + l16] = f32x2{sum[n], top[n]};
    }
    __syncthreads();  // all tiles are done with, too
#pragma unroll
    for (int n = 0; n < RT; ++n) {
      f32x2 each[W];
      float most = kNothing, total = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        each[w] = all[w * (RT * 16) + n * 16 + l16];
        most = fmaxf(most, each[w][1]);
      }
#pragma unroll
      for (int w = 0; w < W; ++w) total = fmaf(each[w][0], __builtin_amdgcn_exp2f(each[w][1] - most), total);
      const float f = __builtin_amdgcn_exp2f(top[n] - most);
      top[n] = most, sum[n] = total;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n * (D / 16) + i][e] *= f;
    }
    gather<N, W / 2>(reinterpret_cast<f32x4*>(memory), reinterpret_cast<f32x4*>(memory + meeting_bytes(N, W, false)), wave, lane, acc, from, there);
  }
  if (there) leave<T, D, RT, C>(p, job, span, from, l16, grp, acc, sum, top);
}

// Zeros for a workgroup's rows from its `from`th on.
template <typename T, int D, int ROWS, int THREADS>
__device__ __forceinline__ void clear_rows(const AttendParams& p, const Job& job, int from) {
  for (int i = from * (D / 4) + threadIdx.x; i < ROWS * (D / 4); i += THREADS) {
    const int row = job.row0 + i / (D / 4);
    if (row < p.rows) store_four<T>(Place(p, job, row).output<T>(p, job.b) + i % (D / 4) * 4, f32x4{0.f, 0.f, 0.f, 0.f}, 0.f);
  }
}

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
  static __device__ __forceinline__ uint32_t find(const KvPool& pool, const Pages<WHOLE>& pages, int head, int tile, const uint8_t* (&record)[Pages<WHOLE>::N]) {
    uint32_t held = 0;
#pragma unroll
    for (int c = 0; c < Pages<WHOLE>::N; ++c) {
      const int chunk = tile * (kTile / kKvChunk) + c;
      const int64_t page = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(pages.high[c])) << 32 | static_cast<uint32_t>(pages.low[c]));
      const bool there = (chunk >> (pool.page_shift - 4)) < pool.table_pages && page >= 0 && page < pool.pages;
      held |= there ? (WHOLE ? 15u : 1u << c) : 0u;
      record[c] = pool.data + (there ? kv_record(pool, page, head, chunk & ((1 << (pool.page_shift - 4)) - 1), RECORD) : 0);
    }
    return held;
  }
  template <bool WHOLE>
  static __device__ __forceinline__ uint32_t request(const KvPool& pool, const Pages<WHOLE>& pages, int head, int tile, uint8_t* to, int lane) {
    constexpr int N = Pages<WHOLE>::N;
    const uint8_t* record[N];
    const uint32_t held = find<WHOLE>(pool, pages, head, tile, record);
    if constexpr (WHOLE) {
#pragma unroll
      for (int i = 0; i < REQUESTS; ++i)
        lds_dma16_offset(record[0], min(i * kWave + lane, PIECES - 1) * 16, to + i * kWave * 16);
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

// The same of the keys or the values alone: the codes of the four chunks, then their scales, four bytes to a lane.
template <int D, int BITS>
struct StagedHalf {
  static constexpr int RECORD = kv_record_bytes(D, BITS), CODES = kv_key_bytes(D, BITS), SCALES = kKvChunk * D / kKvBlock;
  static constexpr int PIECES = 4 * CODES / (kWave * 16), REQUESTS = PIECES + 1, BYTES = 4 * CODES + 4 * kWave;
  template <bool WHOLE>
  static __device__ __forceinline__ void request(const uint8_t* const (&record)[Pages<WHOLE>::N], bool values, uint8_t* to, int lane) {
    const int codes_at = values ? kv_value_at(D, BITS) : 0, scales_at = values ? kv_value_scale_at(D, BITS) : kv_key_scale_at(D, BITS);
    const int scale = min(lane, SCALES - 1), scale_chunk = scale / (SCALES / 4), scale_in = scale % (SCALES / 4) * 4;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      // of chunk i * 1024 / CODES, or of as many from there on as 1024 bytes hold
      constexpr int LANES = CODES / 16 < kWave ? CODES / 16 : kWave;  // of a chunk
      const int first = i * kWave * 16 / CODES, of = lane / LANES, in = i * kWave * 16 % CODES + lane % LANES * 16;
      if constexpr (WHOLE) {
        lds_dma16_offset(record[0] + first * RECORD + codes_at, of * RECORD + in, to + i * kWave * 16);
      } else {
        const uint8_t* from = record[first];
        if constexpr (kWave / LANES == 2) {
          from = of >= 1 ? record[first + 1] : from;
        } else if constexpr (kWave / LANES == 4) {
          const uint8_t *r1 = record[1], *r2 = record[2], *r3 = record[3];
          from = of >= 2 ? (of == 3 ? r3 : r2) : (of == 1 ? r1 : from);
        }
        lds_dma16(from + codes_at + in, to + i * kWave * 16);
      }
    }
    if constexpr (WHOLE) {
      lds_dma4_offset(record[0] + scales_at, scale_chunk * RECORD + scale_in, to + 4 * CODES);
    } else {
      const uint8_t *r0 = record[0], *r1 = record[1], *r2 = record[2], *r3 = record[3];
      const uint8_t* from = scale_chunk >= 2 ? (scale_chunk == 3 ? r3 : r2) : (scale_chunk == 1 ? r1 : r0);
      lds_dma4(from + scales_at + scale_in, to + 4 * CODES);
    }
  }
};

// acc[rows of 16 features] += values^T p: probs[n][part][half]: of 32 tokens, group grp those of chunk 2 half at 4 grp, then those of the next chunk.
// code_bytes, scale_bytes: of the tile's first chunk, CODES_STEP and SCALES_STEP before the next one's.
template <int D, int BITS, int CODES_STEP, int SCALES_STEP, int RT, int PARTS>
__device__ __forceinline__ void times_values(const uint8_t* code_bytes, const uint8_t* scale_bytes, int l16, int grp, const bf16x8 (&probs)[RT][PARTS][2], f32x4 (&acc)[RT * (D / 16)]) {
  constexpr int BLOCKS = D / kKvBlock, EACH = BITS / 4;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    Words<BLOCKS * EACH> codes[2];
    Words<BLOCKS> scales[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      codes[c].load(code_bytes + (2 * half + c) * CODES_STEP + (l16 * 4 + grp) * BLOCKS * BITS);
      scales[c].load(scale_bytes + (2 * half + c) * SCALES_STEP + grp * BLOCKS * 4);
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
          acc[n * (D / 16) + 2 * j] = mfma(first, probs[n][part][half], acc[n * (D / 16) + 2 * j]);
          acc[n * (D / 16) + 2 * j + 1] = mfma(second, probs[n][part][half], acc[n * (D / 16) + 2 * j + 1]);
        }
    }
  }
}

// A wavefront's tiles, two of them in LDS: one on its way while the other is taken. Its only vector-memory operations are the transfers, so that their count says
// what has arrived. No barrier: a wavefront reads what it brought itself, with loads of the compiler's, which the waits in front of them keep in place (ts_common.h).
template <int D, int BITS, int W, int S, bool WHOLE, typename Take>
__device__ __forceinline__ void walk(const AttendParams& p, const Job& job, const Span& span, int wave, int lane, uint8_t* stages, Take&& take) {
  static_assert(S == 2, "the waits below count the requests of one tile");
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
        vm_wait<Tile::REQUESTS>();
      } else {
        vm_wait<0>();
      }
      take(stages + i * Tile::BYTES, held[i], tile);
      tile += W;
    }
  }
}

// A wavefront's tiles, one in LDS, keys and values by themselves: the next keys are on their way from when the scores are made, the next values from when the
// products with these are. Two whole tiles would leave half of the wavefronts no room in LDS, and one whole tile nothing on its way while it is taken.
template <int D, int BITS, int W, bool WHOLE, typename Scores, typename Softmax, typename Values>
__device__ __forceinline__ void walk_halves(const AttendParams& p, const Job& job, const Span& span, int wave, int lane, uint8_t* keys, Scores&& scores,
                                            Softmax&& softmax, Values&& take_values) {
  typedef StagedHalf<D, BITS> Half;
  const int64_t row = job.b * p.pool.table_stride;
  uint8_t* const values = keys + Half::BYTES;
  const uint8_t* record[Pages<WHOLE>::N];
  Pages<WHOLE> pages;
  int tile = span.first + wave;
  if (tile >= span.end) return;
  pages.find(p.pool, row, tile);
  uint32_t held = Staged<D, BITS>::template find<WHOLE>(p.pool, pages, job.head, tile, record);
  pages.find(p.pool, row, tile + W);
  __builtin_amdgcn_s_waitcnt(0x0f70);  // what the compiler asked for before, which it would otherwise await in every round
  Half::template request<WHOLE>(record, false, keys, lane);
  Half::template request<WHOLE>(record, true, values, lane);
  while (true) {
    vm_wait<Half::REQUESTS>();
    scores(keys);
    const int next = tile + W;
    const bool more = next < span.end;
    const uint32_t chunks = held;
    if (more) {
      held = Staged<D, BITS>::template find<WHOLE>(p.pool, pages, job.head, next, record);
      pages.find(p.pool, row, next + W);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the reads of the keys that lay there
      Half::template request<WHOLE>(record, false, keys, lane);
    }
    softmax(chunks, tile);
    if (more) vm_wait<Half::REQUESTS>();
    else vm_wait<0>();
    take_values(values);
    if (!more) return;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    Half::template request<WHOLE>(record, true, values, lane);
    tile = next;
  }
}

// The sum of lanes l, l + 4 and l + 8, within a row of sixteen, for its first four.
__device__ __forceinline__ float three_parts(float v) {
  const int bits = __builtin_bit_cast(int, v);
  return v + (__builtin_bit_cast(float, __builtin_amdgcn_update_dpp(bits, bits, 0x104, 0xf, 0xf, false)) +
              __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(bits, bits, 0x108, 0xf, 0xf, false)));
}

// ---- up to four rows ----------------------------------------------------------------------------------------------

template <typename T, int D, int BITS, int ROWS, int W, int S>
__global__ __launch_bounds__(W * kWave, shape_of(ROWS, D, W).per_simd) void cached_attention_few_kernel(const AttendParams p) {
  constexpr int BLOCKS = D / kKvBlock, SLOT = kTile + 8, PARTS = kParts<T>;
  typedef Staged<D, BITS> Tile;
  extern __shared__ __align__(16) uint8_t memory[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave, l16 = lane % 16, grp = lane / 16;
  const Job job(p, ROWS);
  const Span span = span_of(p, job.b, job.row0, ROWS, job.split, W);
  if (job.split >= span.active) {
    if (job.split == 0) clear_rows<T, D, ROWS, W * kWave>(p, job, 0);
    return;
  }
  uint8_t* const stages = memory + wave * (S * Tile::BYTES);
  bf16_t (*const turned)[SLOT] = reinterpret_cast<bf16_t (*)[SLOT]>(memory + W * S * Tile::BYTES) + wave * (3 * ROWS);  // [part][row]
  // column 4 i + r of the operand: part i of row r; the columns that are left hold one of the others', which nothing reads
  const int column = min(l16 / 4, 2) * ROWS + min(l16 % 4, ROWS - 1);
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
      if (mine) q[o] = query_part<T>(src + 8 * o, part, p.flip, p.keep);
    }
  }
  float most[ROWS];
  f32x4 acc[D / 16], sum = {0.f, 0.f, 0.f, 0.f};  // sums are products with ones: their columns are those of acc
#pragma unroll
  for (int r = 0; r < ROWS; ++r) most[r] = kNothing;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};

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
        for (int e = 0; e < 4; ++e) acc[i][e] *= mine;
    }
    // token 16 grp + l16 lies in chunk grp, group l16 / 4
    bf16_t* to = &turned[0][l16 / 4 * 16 + grp * 4 + l16 % 4];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float x = __builtin_amdgcn_exp2f(score[r] - most[r]);
#pragma unroll
      for (int part = 0; part < 3; ++part) {
        const bf16_t rounded = static_cast<bf16_t>(x);
        to[(part * ROWS + r) * SLOT] = rounded;
        x -= static_cast<float>(rounded);
      }
    }
    wave_sync();
    bf16x8 probs[1][1][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) probs[0][0][half] = *reinterpret_cast<const bf16x8*>(&turned[column][grp * 16 + half * 8]);
    wave_sync();
    sum = mfma(ones, probs[0][0][0], sum);
    sum = mfma(ones, probs[0][0][1], sum);
    times_values<D, BITS, Tile::RECORD, Tile::RECORD>(tile + kv_value_at(D, BITS), tile + kv_value_scale_at(D, BITS), l16, grp, probs, acc);
  };

  p.pool.page_shift >= 6 ? walk<D, BITS, W, S, true>(p, job, span, wave, lane, stages, take) : walk<D, BITS, W, S, false>(p, job, span, wave, lane, stages, take);
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = three_parts(acc[i][e]);
  sum[0] = three_parts(sum[0]);
  float top[1] = {most[0]}, total[1] = {sum[0]};
#pragma unroll
  for (int r = 1; r < ROWS; ++r) top[0] = l16 == r ? most[r] : top[0];
  finish<T, D, 1, W>(p, job, span, memory, reinterpret_cast<float*>(memory + working_bytes(ROWS, D, BITS, W)), wave, lane, acc, total, top);
}

// ---- sixteen rows at a time ---------------------------------------------------------------------------------------

// shared_queries: their place in LDS, or null: in registers.
template <typename T, int D, int BITS, int RT, int W, bool SHARED>
__device__ __forceinline__ void attend_many(const AttendParams& p, const Job& job, const Span& span, int rows, uint8_t* memory, uint8_t* shared_queries, float* stats) {
  constexpr int BLOCKS = D / kKvBlock, PARTS = kParts<T>;
  typedef StagedHalf<D, BITS> Half;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave, l16 = lane % 16, grp = lane / 16;
  uint8_t* const stages = memory + wave * (2 * Half::BYTES);
  int low[RT], high[RT];
  bool empty[RT];  // rows that see nothing are taken along, and cleared at the end
  bf16x8 own[SHARED ? 1 : BLOCKS * RT * PARTS];  // queries: [block][sixteen][part]
  bf16x8* const shared = reinterpret_cast<bf16x8*>(shared_queries) + lane;
  auto query = [&](int i) __attribute__((always_inline)) {
    const int row = job.row0 + 16 * (i / PARTS % RT) + l16;
    const T* src = Place(p, job, min(row, p.rows - 1)).query<T>(p, job);
    bf16x8 q = {};
    if (row < p.rows) q = query_part<T>(src + 8 * (grp * BLOCKS + i / (PARTS * RT)), i % PARTS, p.flip, p.keep);
    return q;
  };
  if constexpr (SHARED) {
    for (int i = wave; i < BLOCKS * RT * PARTS; i += W) shared[i * kWave] = query(i);
    __syncthreads();
  } else {
#pragma unroll
    for (int i = 0; i < BLOCKS * RT * PARTS; ++i) own[i] = query(i);
  }
#pragma unroll
  for (int n = 0; n < RT; ++n) {
    const Seen seen(p, span, job.row0 + 16 * n + l16);
    empty[n] = seen.high <= 0;
    low[n] = seen.low, high[n] = empty[n] ? 0x7fffffff : seen.high;
  }
  // the positions that all of them see
  const int all_low = Seen(p, span, job.row0 + rows - 1).low, all_high = Seen(p, span, job.row0).high;
  float most[RT];
  f32x4 acc[RT * (D / 16)], sums[RT];
#pragma unroll
  for (int n = 0; n < RT; ++n) {
    most[n] = kNothing, sums[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D / 16; ++i) acc[n * (D / 16) + i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int octet = grp * BLOCKS, block = octet / 4;  // of the lane's features
  const bf16x8 ones = __builtin_bit_cast(bf16x8, (u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}));
  f32x4 s[RT][4];
  bf16x8 probs[RT][2][2];
  bool far = false;  // the same in all lanes
  auto scores = [&](const uint8_t* keys_at) __attribute__((always_inline)) {
    Words<BLOCKS * BITS / 4> keys[4];
    float scale[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      keys[c].load(keys_at + c * Half::CODES + block * (kKvChunk * 4 * BITS) + l16 * 4 * BITS + octet % 4 * BITS);
      scale[c] = scale_of<0>(keys_at[4 * Half::CODES + c * Half::SCALES + l16 * BLOCKS + block]);
#pragma unroll
      for (int n = 0; n < RT; ++n) s[n][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int j = 0; j < BLOCKS; ++j) {  // sums that do not wait for each other side by side
      bf16x8 q[RT * PARTS];
#pragma unroll
      for (int i = 0; i < RT * PARTS; ++i) q[i] = SHARED ? shared[(j * RT * PARTS + i) * kWave] : own[SHARED ? 0 : j * RT * PARTS + i];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bf16x8 key = eight<BITS>(keys[c].w + j * (BITS / 4), scale[c]);
#pragma unroll
        for (int i = 0; i < RT * PARTS; ++i) s[i / PARTS][c] = mfma(key, q[i], s[i / PARTS][c]);
      }
    }
  };
  auto softmax = [&](uint32_t chunks, int number) __attribute__((always_inline)) {
    if (chunks != 15u || number * kTile < all_low || number * kTile + kTile > all_high) {
#pragma unroll
      for (int n = 0; n < RT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int position = number * kTile + 16 * c + 4 * grp + e;
            s[n][c][e] = (chunks >> c & 1) && position >= low[n] && position < high[n] ? s[n][c][e] : -INFINITY;
          }
    }
    bool above = false;
    float top[RT];
#pragma unroll
    for (int n = 0; n < RT; ++n) {
      top[n] = s[n][0][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top[n] = fmaxf(top[n], s[n][i / 4][i % 4]);
      top[n] *= p.scale;
      above |= top[n] > most[n] + kSlack;
    }
    if (__any(above)) {
      bool beyond = false;
#pragma unroll
      for (int n = 0; n < RT; ++n) {
        const float t = fmaxf(most[n], max_over_rows(top[n]));
        const float f = __builtin_amdgcn_exp2f(most[n] - t);
        most[n] = t;
        beyond |= t > kNothing && fabsf(t) > kFar;
        sums[n][0] *= f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n * (D / 16) + i][e] *= f;
      }
      far = __any(beyond);
    }
    // Product and difference are one instruction, whose product is not rounded as the maximum is. Scores in the billions would differ from their own maximum by that: such
    // are rounded first.
    if (far) {
#pragma clang fp contract(off)
#pragma unroll
      for (int n = 0; n < RT; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][i / 4][i % 4] *= p.scale;
    }
    const float factor = far ? 1.f : p.scale;
#pragma unroll
    for (int n = 0; n < RT; ++n)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        f32x4 x[2];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[c][e] = __builtin_amdgcn_exp2f(fmaf(s[n][2 * half + c][e], factor, -most[n]));
        two_parts(x[0], x[1], probs[n][0][half], probs[n][1][half]);
        sums[n] = mfma(ones, probs[n][0][half], sums[n]);
        sums[n] = mfma(ones, probs[n][1][half], sums[n]);
      }
  };
  auto take_values = [&](const uint8_t* values) __attribute__((always_inline)) {
    times_values<D, BITS, Half::CODES, Half::SCALES>(values, values + 4 * Half::CODES, l16, grp, probs, acc);
  };

  p.pool.page_shift >= 6 ? walk_halves<D, BITS, W, true>(p, job, span, wave, lane, stages, scores, softmax, take_values)
                         : walk_halves<D, BITS, W, false>(p, job, span, wave, lane, stages, scores, softmax, take_values);
  float sum[RT];
#pragma unroll
  for (int n = 0; n < RT; ++n) {
    sum[n] = empty[n] ? 0.f : sums[n][0], most[n] = empty[n] ? kNothing : most[n];
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n * (D / 16) + i][e] = empty[n] ? 0.f : acc[n * (D / 16) + i][e];
  }
  finish<T, D, RT, W>(p, job, span, memory, stats, wave, lane, acc, sum, most);
}

// Rows of queries that a sample has not, whole sixteens of them, are cleared and not taken along.
template <typename T, int D, int BITS, int ROWS, int W>
__global__ __launch_bounds__(W * kWave, shape_of(ROWS, D, W).per_simd) void cached_attention_many_kernel(const AttendParams p) {
  constexpr bool SHARED = queries_in_lds(ROWS, kParts<T>);
  extern __shared__ __align__(16) uint8_t memory[];
  constexpr int WORKING = working_bytes(ROWS, D, BITS, W);
  static_assert(meeting_fits(ROWS / 16 * (D / 16), W, D / 16, WORKING));
  uint8_t* const queries = memory + WORKING;
  float* const stats = reinterpret_cast<float*>(queries + (SHARED ? ROWS * D * 2 : 0));
  const Job job(p, ROWS);
  const int row_end = min(job.row0 + ROWS, p.rows);
  const Span span = span_of(p, job.b, job.row0, row_end - job.row0, job.split, W);
  const bool mine = job.split < span.active;
  const int rows = mine ? min(row_end, p.group.d * span.news) - job.row0 : 0, taken = (rows + 15) & ~15;  // rows that there are
  if (job.split == 0 && taken < ROWS) clear_rows<T, D, ROWS, W * kWave>(p, job, taken);
  if (!mine) return;
  if (ROWS == 16 || taken == 16) attend_many<T, D, BITS, 1, W, SHARED>(p, job, span, rows, memory, queries, stats);
  else if (ROWS == 32 || taken == 32) attend_many<T, D, BITS, 2, W, SHARED>(p, job, span, rows, memory, queries, stats);
  else attend_many<T, D, BITS, ROWS / 16, W, SHARED>(p, job, span, rows, memory, queries, stats);
}

// More than the 64 KB of LDS that a launch may have unasked.
template <typename Kernel>
void launch_with(Kernel* kernel, uint32_t groups, int threads, int bytes, const AttendParams& p, hipStream_t s) {
  if (bytes > 65536) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  hipLaunchKernelGGL(kernel, dim3(groups), dim3(threads), bytes, s, p);
}
template <typename T, int D, int BITS, int ROWS, int W>
void launch_rows(const AttendParams& p, uint32_t groups, hipStream_t s) {
  constexpr Shape shape = shape_of(ROWS, D, W);
  static_assert(Staged<D, BITS>::BYTES == tile_bytes(D, BITS) && StagedHalf<D, BITS>::BYTES == half_bytes(D, BITS));
  constexpr int bytes = lds_bytes(ROWS, D, BITS, kParts<T>, W), threads = W * kWave;
  if constexpr (ROWS <= 4) launch_with(cached_attention_few_kernel<T, D, BITS, ROWS, W, shape.stages>, groups, threads, bytes, p, s);
  else launch_with(cached_attention_many_kernel<T, D, BITS, ROWS, W>, groups, threads, bytes, p, s);
}
template <typename T, int D, int BITS>
void launch_attend(const AttendParams& p, int rows, int waves, uint32_t groups, hipStream_t s) {
  if (rows == 1) waves == 1 ? launch_rows<T, D, BITS, 1, 1>(p, groups, s) : launch_rows<T, D, BITS, 1, 4>(p, groups, s);
  if (rows == 2) waves == 1 ? launch_rows<T, D, BITS, 2, 1>(p, groups, s) : launch_rows<T, D, BITS, 2, 4>(p, groups, s);
  if constexpr (kParts<T> == 1) {
    if (rows == 4) waves == 1 ? launch_rows<T, D, BITS, 4, 1>(p, groups, s) : launch_rows<T, D, BITS, 4, 4>(p, groups, s);
  }
  if (rows == 16) waves == 1 ? launch_rows<T, D, BITS, 16, 1>(p, groups, s) : waves == 4 ? launch_rows<T, D, BITS, 16, 4>(p, groups, s) : launch_rows<T, D, BITS, 16, 8>(p, groups, s);
  if (rows == 32) launch_rows<T, D, BITS, 32, 4>(p, groups, s);
  if constexpr (kParts<T> == 1) {
    if (rows == 48) launch_rows<T, D, BITS, 48, 8>(p, groups, s);
  }
}
template <int BITS>
void dispatch_attend(const AttendParams& p, int d, bool f16, int rows, int waves, uint32_t groups, hipStream_t s) {
#define TAAC_ATTEND(D) \
  if (d == D) f16 ? launch_attend<f16_t, D, BITS>(p, rows, waves, groups, s) : launch_attend<bf16_t, D, BITS>(p, rows, waves, groups, s);
  TAAC_ATTEND(32) TAAC_ATTEND(64) TAAC_ATTEND(128)
#undef TAAC_ATTEND
}

}  // namespace

// Of caches of 4 bits and of 8 (cached_attention_4.hip, cached_attention_8.hip): a unit each, which build side by side.
void attend_4(const AttendParams& p, int d, bool f16, int rows, int waves, uint32_t groups, hipStream_t s);
void attend_8(const AttendParams& p, int d, bool f16, int rows, int waves, uint32_t groups, hipStream_t s);

}  // namespace taac
