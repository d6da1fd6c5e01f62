// Attention over a cache: the entry points, how a call is cut into workgroups, and the kernel that joins the parts of histories that were split (the kernels
// that attend: cached_attention.h).
#include <cmath>

#include "cached_attention.h"

namespace taac {
namespace {

// ---- the splits' parts --------------------------------------------------------------------------------------------

// Lanes of four features to a row. Of many splits a whole wavefront: its lanes are 64 / (D / 4) groups that take them in turn. Bound by latency: calls of two
// splits, 64 samples of 1024 tokens, 32 rows, take 28.3 us with wavefronts, 24.9 with lanes; of eight, 4 samples of 2000 tokens, 48 rows, 13.1 and 13.7.
template <typename T, int D, bool MANY>
__global__ __launch_bounds__(256) void cached_attention_join_kernel(const AttendParams p, int tile_rows, int waves) {
  typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2;
  constexpr int LANES = D / 4, GROUPS = MANY ? kWave / LANES : 1, AT_ONCE = MANY ? 8 : 2;
  const int64_t out_row = static_cast<int64_t>(blockIdx.x) * (256 / (LANES * GROUPS)) + threadIdx.x / (LANES * GROUPS);
  if (out_row >= p.all_rows) return;
  const int c = threadIdx.x % LANES * 4, group = threadIdx.x % (LANES * GROUPS) / LANES;
  const int64_t token = out_row / p.T;
  const int t = static_cast<int>(out_row - token * p.T), b = static_cast<int>(token / p.H), h = static_cast<int>(token - static_cast<int64_t>(b) * p.H);
  const int head = p.group.over(h), row = t * p.group.d + h - head * p.group.d, row0 = row / tile_rows * tile_rows;
  const Span span = span_of(p, b, row0, min(tile_rows, p.rows - row0), 0, waves);
  if (span.active <= 1 || t >= span.news) return;  // whole already, or zeros
  const float* part = p.partial + out_row * p.splits.d * D + c;
  const f32x2* stats = reinterpret_cast<const f32x2*>(p.partial + p.all_rows * p.splits.d * D) + out_row * p.splits.d;
  float top = kNothing, l = 0.f;
  f32x4 total = {0.f, 0.f, 0.f, 0.f};
  for (int first = group; first < span.active; first += GROUPS * AT_ONCE) {
    f32x4 v[AT_ONCE];
    float most[AT_ONCE], sum[AT_ONCE], up = top;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {  // those behind the last count as the last once more, with no weight
      const int split = min(first + i * GROUPS, span.active - 1);
      v[i] = *reinterpret_cast<const f32x4*>(part + static_cast<int64_t>(split) * D);
      const f32x2 both = stats[split];
      most[i] = both[0], sum[i] = both[1];
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
  for (int off = LANES; off < LANES * GROUPS; off *= 2) {
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
  if (group == 0) store_four<T>(Place(p, job, row).output<T>(p, b) + c, total, l == 0.f ? 0.f : 1.f / l);
}

// ---- the host -----------------------------------------------------------------------------------------------------

constexpr int64_t kOccupied = 192;  // units: most of 256 CUs have one
constexpr int64_t kMostGroups = 1 << 23;  // of a launch: at most 2^31 threads in workgroups of four wavefronts, of the 2^32 - 1 that a launch may have; eight are for 256 units

// How a call is cut. A unit is a tile of rows of a key head of a sample.
struct Plan {
  int rows;       // of a tile: 1, 2, 4, 16, 32 or 48
  int row_tiles;  // of a key head
  int splits;     // of a history
  int waves;      // of a workgroup: 1, 4 or 8
};

// From so many units on a wavefront takes one alone, without the meeting; below, four share its tokens. Ragged histories, alone : shared, in us:
//   up to 4 rows, 32 features: 9.9 : 14.0 at 4096 units of up to 256 tokens, 23.6 : 24.2 of 1024; 7.0 : 8.7 and 18.4 : 14.9 at 2048
//   64 features: 9.5 : 14.9 at 2048 units of 256, 23.3 : 25.8 of 1024; 7.3 : 9.4 and 17.9 : 17.0 at 1024
//   128 features: 16.0 : 28.5 at 2048 units of 256, 39.3 : 45.2 of 1024; 10.3 : 15.2 and 25.6 : 28.0 at 1024
//   16 rows, 64 features: 26.0 : 37.2 at 8192 units of 256, 40.0 : 47.6 of 512; 16.6 : 21.2 of 256 and 45.0 : 39.1 of 1024 at 4096
// Below the lines short histories are faster alone still, and with 128 features both; what long ones lose there decided.
int64_t alone_from(int rows, int32_t d) { return rows > 4 ? 8192 : d == 32 ? 4096 : 2048; }

// Tiles of so many rows. held: the table's tokens, whether a window sees them or not; splits that a window leaves without a tile end at once.
Plan cut(int64_t B, int32_t heads, int64_t rows, int tile, bool wide, int32_t d, int bits, int64_t held, bool parts) {
  Plan plan{};
  plan.rows = tile;
  plan.row_tiles = static_cast<int>((rows + tile - 1) / (tile > 0 ? tile : 1));
  const int64_t units = B * heads * plan.row_tiles;
  plan.waves = wide ? 8 : tile <= 16 && units >= alone_from(tile, d) ? 1 : 4;
  const Shape shape = shape_of(tile, d, plan.waves);
  // Histories are split until the card is full, by LDS and registers; twice as many workgroups cost more than a better balance gives back (4 x 8 key heads of 128 features,
  // 65536 tokens: 56 us, 60 with twice as many). A split has a tile for each of its wavefronts, and below four (six of narrower heads) the kernel that joins them
  // takes longer than the tiles would: one sample of 768 tokens 5.7 us as a whole, of 1024 in four 7.9. Where whole histories occupy three quarters of the CUs, only from 16 tiles
  // to a wavefront on, and not of 128 features. One query of 4 key heads, split : whole, 64 samples of 2500 tokens: 32 features 11.8 : 10.4, 64 17.2 : 15.0, 128 24.8 : 20.5;
  // of 8000: 20.8 : 26.5, 31.7 : 34.7, 53.0 : 48.2; 48 of 2500 11.5 : 9.8, 15.0 : 14.1, 22.1 : 20.0.
  const int by_lds = 163840 / lds_bytes(tile, d, bits, parts ? 2 : 1, plan.waves), by_registers = 4 * shape.per_simd / shape.waves;
  const int64_t resident = 256 * (by_lds < by_registers ? by_lds : by_registers), most = held / (kTile * shape.waves);
  int64_t splits = resident / (units > 0 ? units : 1);
  splits = splits < most ? splits : most;
  const bool long_enough = units < kOccupied ? most >= (d == 128 ? 4 : 6) : most >= 16 && d < 128;
  plan.splits = static_cast<int>(!long_enough || splits < 1 ? 1 : splits);
  return plan;
}

Plan plan_of(int64_t B, int32_t heads, int32_t group, int32_t T, int32_t d, int bits, int64_t held, bool parts) {
  const int64_t rows = static_cast<int64_t>(group) * T;
  // up to 4 rows (2 in two parts) in the one form
  if (rows <= 2 || (rows <= 4 && !parts)) return cut(B, heads, rows, rows <= 2 ? static_cast<int>(rows) : 4, false, d, bits, held, parts);
  // 16 rows where a workgroup to a CU fills the card: eight wavefronts, and no splits. 8 rows of 4 key heads, ragged histories, four with splits : eight, in us, at
  //                                 128 units     192           256           288           384
  //   32 features, 4 bits,  2500 tokens   10.5 :  9.5   12.3 :  9.7   12.4 :  9.7   13.2 : 11.5   14.8 : 13.2
  //   64 features, 8 bits,   500           6.0 :  6.0    6.0 :  6.1    6.1 :  6.1    7.2 :  7.6    7.3 :  7.8
  //                         1000           8.2 :  7.4    8.3 :  7.4    8.5 :  7.8    9.9 : 10.0   10.1 : 10.2
  //                         2500          12.8 : 11.7   15.4 : 13.0   16.2 : 14.4   18.4 : 19.2   18.7 : 20.0
  //                         8000          24.8 : 22.9   29.2 : 28.3   31.5 : 30.8   38.3 : 45.3
  //   64 features, 4 bits,  8000          19.6 : 20.8   24.1 : 27.1   25.2 : 27.7   29.0 : 37.0
  //   128 features, 8 bits, 1000          12.2 : 10.3   11.4 : 11.3   12.1 : 12.3   16.2 : 17.5   17.0 : 19.9
  //                         2500          19.7 : 19.1   21.3 : 20.4   22.3 : 21.9   32.5 : 30.5   33.2 : 32.3
  // Beyond 256 units a second round begins, which eight fill worse. Down to 128 they would be as fast or faster, but for the longest histories.
  if (rows <= 16) return cut(B, heads, rows, 16, B * heads >= kOccupied && B * heads <= 256, d, bits, held, parts);
  // In the other 16, or 32, which share the conversion of the codes. Where a workgroup of eight wavefronts to a CU just fills the card, up to 48 rows in one, which need no
  // splits and no joining; of four sixteens the sums would leave no registers. 4 key heads, 2000 tokens, 48 rows : 32: of 128 features in 8 bits, 18 rows, 48 samples 25.1 : 29.6
  // us, 64 samples 29.8 : 32.3, 100 samples 47.8 : 43.2; 48 rows, 64 samples 32.9 : 36.8, 100 samples 56.5 : 65.9; of 64 in 4 bits, 18 rows, 64 samples 16.3 : 19.7, 100 samples
  // 29.6 : 24.1; 48 rows 20.8 : 23.9 and 38.7 : 37.2. Of 500 tokens 16.2 : 16.3 and 29.1 : 26.6, 11.0 : 10.3 and 20.0 : 14.8.
  if (rows <= 48 && !parts && held >= 1024 && B * heads <= 256) {
    const Plan wide = cut(B, heads, rows, 48, true, d, bits, held, parts);
    if (B * heads * wide.splits >= kOccupied) return wide;
  }
  return cut(B, heads, rows, 32, false, d, bits, held, parts);
}

template <typename T, int D>
void launch_join(const AttendParams& p, const Plan& plan, hipStream_t s) {
  const bool many = plan.splits > 4;
  const int64_t at_once = 256 / (many ? kWave : D / 4);
  const dim3 grid(static_cast<uint32_t>((p.all_rows + at_once - 1) / at_once));
  if (many) hipLaunchKernelGGL((cached_attention_join_kernel<T, D, true>), grid, dim3(256), 0, s, p, plan.rows, plan.waves);
  else hipLaunchKernelGGL((cached_attention_join_kernel<T, D, false>), grid, dim3(256), 0, s, p, plan.rows, plan.waves);
}
template <typename T>
void join(const AttendParams& p, const Plan& plan, int d, hipStream_t s) {
  if (d == 32) launch_join<T, 32>(p, plan, s);
  if (d == 64) launch_join<T, 64>(p, plan, s);
  if (d == 128) launch_join<T, 128>(p, plan, s);
}

}  // namespace
}  // namespace taac

extern "C" int64_t taac_cached_attention_workspace_bytes(int32_t B, int32_t H, int32_t heads, int32_t T, int32_t d, int bits, int64_t table_tokens) {
  using namespace taac;
  if (B < 0 || T < 0 || heads <= 0 || H <= 0 || H % heads != 0 || d <= 0 || (bits != 4 && bits != 8) || table_tokens < 0) return -1;
  // of either type of queries: three and four rows in two parts take the other form
  const int one = plan_of(B, heads, H / heads, T, d, bits, table_tokens, false).splits, two = plan_of(B, heads, H / heads, T, d, bits, table_tokens, true).splits;
  const int splits = one > two ? one : two;
  return splits > 1 ? static_cast<int64_t>(B) * H * T * splits * (d + 2) * 4 : 0;
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
  Plan plan = plan_of(B, heads, group, T, d, bits, held, dtype == TAAC_F16);
  const int64_t each = static_cast<int64_t>(heads) * plan.row_tiles * plan.splits, at_once = kMostGroups / each;  // workgroups of a sample, samples of a launch
  if (at_once < 1) return set_error(TAAC_ERR_UNSUPPORTED, "%s: too many workgroups to a sample", name);
  p.all_rows = static_cast<int64_t>(B) * H * T;
  const int64_t need = plan.splits > 1 ? p.all_rows * plan.splits * (d + 2) * 4 : 0;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: workspace must hold %lld bytes, 16-byte aligned", name, (long long)need);
  p.q = q, p.o = o, p.lengths = lengths, p.query_lengths = query_lengths, p.partial = static_cast<float*>(workspace);
  p.group = divisor(group), p.splits = divisor(plan.splits), p.row_tiles = divisor(plan.row_tiles), p.heads = divisor(heads);
  p.H = H, p.T = T, p.rows = group * T, p.window = window;
  p.scale = scale * 1.4426950408889634f;
  p.scale = scale == 0.f ? 1.f : fabsf(p.scale);
  p.keep = scale == 0.f ? 0u : 0xffffffffu;
  p.flip = scale < 0.f ? 0x80008000u : 0u;
  const bool f16 = dtype == TAAC_F16;
  hipStream_t s = as_stream(stream);
  for (int64_t first = 0; first < B; first += at_once) {
    p.first = static_cast<int32_t>(first);
    const uint32_t groups = static_cast<uint32_t>((B - first < at_once ? B - first : at_once) * each);
    bits == 4 ? attend_4(p, d, f16, plan.rows, plan.waves, groups, s) : attend_8(p, d, f16, plan.rows, plan.waves, groups, s);
  }
  if (plan.splits > 1) f16 ? join<f16_t>(p, plan, d, s) : join<bf16_t>(p, plan, d, s);
  return check_launch(name);
}
