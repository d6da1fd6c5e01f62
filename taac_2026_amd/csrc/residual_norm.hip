// RMSNorm of a sum, h = x + residual, for gfx950: the seam between the two halves of a pre-norm block.
//
//   h = round(x + residual)                 written in the storage type: the residual stream
//   y = h * rsqrt(mean(h^2) + eps) * w      from the rounded h, so that it is the norm of what is stored
//   y leaves in the storage type, or as e4m3 with one maximum per row: amax = max |y|, q = e4m3(y * 448 / amax)
//
// Backward, with r = rsqrt(mean(h^2) + eps) recomputed from h (one more reduction in registers instead of a vector of factors):
//   dh = ds + r (w dy - h r^2 mean(h w dy)),   dx = dresidual = dh,   dw = sum over the rows of dy h r
//
// All of it is bound by HBM: the forward reads x and residual and writes h and y, the backward reads h, dy and ds and writes dh,
// each exactly once. As in the plain norm kernels a group of G consecutive lanes owns a row in NV 128-bit vectors per lane and
// everything is requested before anything is used. Arithmetic is fp32; h is rounded because it is an output, y once at the end.
// A NaN in a row reaches the row's maximum and its e4m3 values (no max instruction that would drop it).
#include "norm_rows.h"

namespace taac {
namespace {

constexpr int kFwdMaxNV = 8, kBwdMaxNV = 4;

template <typename T>
struct RawPack {  // the storage type's bits of one vector of e4m3 values: one byte per element
  static constexpr int WORDS = Pack<T>::VEC / 4;
};

__device__ __forceinline__ float nan_max(float m, float a) { return (a > m || a != a) ? a : m; }

template <int G>
__device__ __forceinline__ float group_nan_max(float v) {
#pragma unroll
  for (int off = G / 2; off > 0; off >>= 1) v = nan_max(v, __shfl_xor(v, off, kWave));
  return v;
}

__device__ __forceinline__ float clamp_e4m3(float f) { return f > 448.f ? 448.f : (f < -448.f ? -448.f : f); }  // keeps NaN

// Four fp32 values -> four e4m3 bytes, round to nearest even.
__device__ __forceinline__ uint32_t pack_e4m3(const float* f, float inv_scale) {
  int r = 0;
  r = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(f[0] * inv_scale), clamp_e4m3(f[1] * inv_scale), r, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(f[2] * inv_scale), clamp_e4m3(f[3] * inv_scale), r, true);
  return static_cast<uint32_t>(r);
}

// 448 / amax with the smallest amax that quantize_fp8 uses (rows of zeros give zeros).
__device__ __forceinline__ float inverse_scale(float amax) { return 448.0f / (amax < 1e-12f ? 1e-12f : amax); }

// x and residual may be the tensor that `summed` names: a lane writes what it alone has read.
template <typename T, int G, int NV, int R, bool FP8>
__global__ __launch_bounds__(kBlock) void residual_norm_vec_kernel(const T* x, const T* residual, const T* __restrict__ w, T* summed,
                                                                   void* __restrict__ out, float* __restrict__ row_amax,
                                                                   int64_t rows, int cols, int nvec, float eps) {
  typedef Pack<T> P;
  typedef typename P::vec vec_t;
  constexpr int VEC = P::VEC;
  constexpr int GPB = kBlock / G;
  const int lane = threadIdx.x % G;
  const int gid = threadIdx.x / G;

  vec_t xr[R][NV], rr[R][NV];
  bool row_ok[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * R + r) * GPB + gid;
    row_ok[r] = row < rows;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = lane + i * G;
      if (row_ok[r] && v < nvec) {
        xr[r][i] = __builtin_nontemporal_load(reinterpret_cast<const vec_t*>(x + row * cols) + v);
        rr[r][i] = __builtin_nontemporal_load(reinterpret_cast<const vec_t*>(residual + row * cols) + v);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) xr[r][i][e] = rr[r][i][e] = 0;
      }
    }
  }
  float wf[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = lane + i * G;
    if (v < nvec) {
      P::unpack(reinterpret_cast<const vec_t*>(w)[v], wf[i]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) wf[i][e] = 0.f;
    }
  }

  const float inv_cols = 1.0f / static_cast<float>(cols);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * R + r) * GPB + gid;
    float hf[NV][VEC];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = lane + i * G;
      float xf[VEC], rf[VEC];
      P::unpack(xr[r][i], xf);
      P::unpack(rr[r][i], rf);
#pragma unroll
      for (int e = 0; e < VEC; ++e) xf[e] += rf[e];
      const vec_t h = P::pack(xf);
      P::unpack(h, hf[i]);
      if (row_ok[r] && v < nvec) __builtin_nontemporal_store(h, reinterpret_cast<vec_t*>(summed + row * cols) + v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) ss += hf[i][e] * hf[i][e];
    }
    const float scale = rsqrtf(group_sum<G>(ss) * inv_cols + eps);
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        hf[i][e] = hf[i][e] * scale * wf[i][e];
        if (FP8 && lane + i * G < nvec) amax = nan_max(amax, __builtin_fabsf(hf[i][e]));
      }
    if (FP8) {
      amax = group_nan_max<G>(amax);
      const float inv = inverse_scale(amax);
      if (row_ok[r] && lane == 0) row_amax[row] = amax;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * G;
        if (!(row_ok[r] && v < nvec)) continue;
        uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(out) + row * cols) + v * RawPack<T>::WORDS;
        if constexpr (VEC == 8) {
          const u32x2 q = {pack_e4m3(hf[i], inv), pack_e4m3(hf[i] + 4, inv)};
          __builtin_nontemporal_store(q, reinterpret_cast<u32x2*>(dst));
        } else {
          __builtin_nontemporal_store(pack_e4m3(hf[i], inv), dst);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * G;
        if (row_ok[r] && v < nvec)
          __builtin_nontemporal_store(P::pack(hf[i]), reinterpret_cast<vec_t*>(static_cast<T*>(out) + row * cols) + v);
      }
    }
  }
}

// Rows that are not whole aligned 128-bit vectors, or longer than the registers of a wavefront hold: one wavefront per row, element by
// element; the sweeps after the first read h back through the cache (written and read by the same lane).
template <typename T, bool FP8>
__global__ __launch_bounds__(kBlock) void residual_norm_generic_kernel(const T* x, const T* residual, const T* __restrict__ w, T* summed,
                                                                       void* __restrict__ out, float* __restrict__ row_amax,
                                                                       int64_t rows, int cols, float eps) {
  const int lane = threadIdx.x % kWave;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kBlock / kWave) + threadIdx.x / kWave;
  if (row >= rows) return;
  const T* xr = x + row * cols;
  const T* rr = residual + row * cols;
  T* hr = summed + row * cols;
  float ss = 0.f;
  for (int c = lane; c < cols; c += kWave) {
    const T h = static_cast<T>(static_cast<float>(xr[c]) + static_cast<float>(rr[c]));
    hr[c] = h;
    ss += static_cast<float>(h) * static_cast<float>(h);
  }
  const float scale = rsqrtf(group_sum<kWave>(ss) / static_cast<float>(cols) + eps);
  if (FP8) {
    float amax = 0.f;
    for (int c = lane; c < cols; c += kWave)
      amax = nan_max(amax, __builtin_fabsf(static_cast<float>(hr[c]) * scale * static_cast<float>(w[c])));
    amax = group_nan_max<kWave>(amax);
    const float inv = inverse_scale(amax);
    if (lane == 0) row_amax[row] = amax;
    uint8_t* q = static_cast<uint8_t*>(out) + row * cols;
    for (int c = lane; c < cols; c += kWave) {
      const float f = clamp_e4m3(static_cast<float>(hr[c]) * scale * static_cast<float>(w[c]) * inv);
      q[c] = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(f, 0.f, 0, false) & 0xff);
    }
  } else {
    T* y = static_cast<T*>(out) + row * cols;
    for (int c = lane; c < cols; c += kWave)
      y[c] = static_cast<T>(static_cast<float>(hr[c]) * scale * static_cast<float>(w[c]));
  }
}

// ds null: the sum itself has no gradient.
template <typename T, int G, int NV>
__global__ __launch_bounds__(kBlock) void residual_norm_bwd_vec_kernel(const T* __restrict__ h, const T* __restrict__ w,
                                                                       const T* __restrict__ dy, const T* __restrict__ ds,
                                                                       T* __restrict__ dh, float* __restrict__ partial, int64_t rows,
                                                                       int cols, int nvec, float eps) {
  typedef Pack<T> P;
  typedef typename P::vec vec_t;
  constexpr int VEC = P::VEC;
  constexpr int GPB = kBlock / G;
  __shared__ float red[GPB][G * VEC];
  const int lane = threadIdx.x % G;
  const int gid = threadIdx.x / G;
  const float inv_cols = 1.0f / static_cast<float>(cols);

  float wf[NV][VEC], dwacc[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = lane + i * G;
#pragma unroll
    for (int e = 0; e < VEC; ++e) wf[i][e] = dwacc[i][e] = 0.f;
    if (v < nvec) P::unpack(reinterpret_cast<const vec_t*>(w)[v], wf[i]);
  }
  constexpr int R = NV == 1 ? 2 : 1;  // rows in flight per lane group
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * (GPB * R); row0 < rows; row0 += static_cast<int64_t>(gridDim.x) * (GPB * R)) {
    vec_t hr[R][NV], gr[R][NV], sr[R][NV];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r * GPB + gid;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * G;
        const bool live = row < rows && v < nvec;
#pragma unroll
        for (int e = 0; e < VEC; ++e) hr[r][i][e] = gr[r][i][e] = sr[r][i][e] = 0;
        if (live) {
          hr[r][i] = __builtin_nontemporal_load(reinterpret_cast<const vec_t*>(h + row * cols) + v);
          gr[r][i] = __builtin_nontemporal_load(reinterpret_cast<const vec_t*>(dy + row * cols) + v);
          if (ds != nullptr) sr[r][i] = __builtin_nontemporal_load(reinterpret_cast<const vec_t*>(ds + row * cols) + v);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r * GPB + gid;
      float hf[NV][VEC], gf[NV][VEC];
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        P::unpack(hr[r][i], hf[i]);
        P::unpack(gr[r][i], gf[i]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) ss += hf[i][e] * hf[i][e];
      }
      const float rstd = rsqrtf(group_sum<G>(ss) * inv_cols + eps);
      float proj = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          hf[i][e] *= rstd;
          proj += gf[i][e] * wf[i][e] * hf[i][e];
        }
      const float mean = group_sum<G>(proj) * inv_cols;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = lane + i * G;
        float sf[VEC], of[VEC];
        P::unpack(sr[r][i], sf);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          of[e] = sf[e] + rstd * (gf[i][e] * wf[i][e] - hf[i][e] * mean);
          dwacc[i][e] += gf[i][e] * hf[i][e];  // rows beyond the end contribute zeros
        }
        if (row < rows && v < nvec) __builtin_nontemporal_store(P::pack(of), reinterpret_cast<vec_t*>(dh + row * cols) + v);
      }
    }
  }
  // partial row of this workgroup: the lane groups meet in LDS and are added in their order
  float* out_w = partial + static_cast<int64_t>(blockIdx.x) * cols;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) red[gid][lane * VEC + e] = dwacc[i][e];
    __syncthreads();
    for (int t = threadIdx.x; t < G * VEC; t += kBlock) {
      float sum = 0.f;
#pragma unroll
      for (int g = 0; g < GPB; ++g) sum += red[g][t];
      const int col = i * G * VEC + t;
      if (col < cols) out_w[col] = sum;
    }
  }
}

// As the generic backward of the plain norms: a workgroup per row at a time, its partial row of dw kept in the workspace by the threads
// that own the columns.
template <typename T>
__global__ __launch_bounds__(kBlock) void residual_norm_bwd_generic_kernel(const T* __restrict__ h, const T* __restrict__ w,
                                                                           const T* __restrict__ dy, const T* __restrict__ ds,
                                                                           T* __restrict__ dh, float* __restrict__ partial,
                                                                           int64_t rows, int cols, float eps) {
  __shared__ float red[1][kBlock / kWave];
  const int tid = threadIdx.x;
  const float inv_cols = 1.0f / static_cast<float>(cols);
  float* out_w = partial + static_cast<int64_t>(blockIdx.x) * cols;
  for (int c = tid; c < cols; c += kBlock) out_w[c] = 0.f;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* hr = h + row * cols;
    const T* gr = dy + row * cols;
    float ss[1] = {0.f};
    for (int c = tid; c < cols; c += kBlock) ss[0] += static_cast<float>(hr[c]) * static_cast<float>(hr[c]);
    block_sum<1>(ss, red);
    const float rstd = rsqrtf(ss[0] * inv_cols + eps);
    float proj[1] = {0.f};
    for (int c = tid; c < cols; c += kBlock)
      proj[0] += static_cast<float>(gr[c]) * static_cast<float>(w[c]) * (static_cast<float>(hr[c]) * rstd);
    block_sum<1>(proj, red);
    const float mean = proj[0] * inv_cols;
    for (int c = tid; c < cols; c += kBlock) {
      const float gy = static_cast<float>(gr[c]), unit = static_cast<float>(hr[c]) * rstd;
      const float s = ds != nullptr ? static_cast<float>(ds[row * cols + c]) : 0.f;
      dh[row * cols + c] = static_cast<T>(s + rstd * (gy * static_cast<float>(w[c]) - unit * mean));
      out_w[c] += gy * unit;
    }
  }
}

template <typename T, int G, int NV, bool FP8>
void launch_fwd(const T* x, const T* r, const T* w, T* h, void* out, float* amax, int64_t rows, int cols, int nvec, float eps,
                hipStream_t s) {
  constexpr int R = NV == 1 ? 2 : 1;
  const int64_t rows_per_block = static_cast<int64_t>(kBlock / G) * R;
  hipLaunchKernelGGL((residual_norm_vec_kernel<T, G, NV, R, FP8>), dim3(static_cast<uint32_t>((rows + rows_per_block - 1) / rows_per_block)),
                     dim3(kBlock), 0, s, x, r, w, h, out, amax, rows, cols, nvec, eps);
}

template <typename T, bool FP8>
void dispatch_fwd(const void* xv, const void* rv, const void* wv, void* hv, void* out, float* amax, int64_t rows, int cols, float eps,
                  hipStream_t s) {
  const T *x = static_cast<const T*>(xv), *r = static_cast<const T*>(rv), *w = static_cast<const T*>(wv);
  T* h = static_cast<T*>(hv);
  constexpr int VEC = Pack<T>::VEC;
  const int nvec = cols / VEC;
  if (cols % VEC != 0 || !aligned16(x) || !aligned16(r) || !aligned16(w) || !aligned16(h) || !aligned16(out) || nvec > kWave * kFwdMaxNV) {
    const int64_t grid = (rows + (kBlock / kWave) - 1) / (kBlock / kWave);
    hipLaunchKernelGGL((residual_norm_generic_kernel<T, FP8>), dim3(static_cast<uint32_t>(grid)), dim3(kBlock), 0, s, x, r, w, h, out,
                       amax, rows, cols, eps);
    return;
  }
#define TAAC_RESIDUAL_NORM(G, NV) return launch_fwd<T, G, NV, FP8>(x, r, w, h, out, amax, rows, cols, nvec, eps, s)
  if (nvec <= 2) TAAC_RESIDUAL_NORM(2, 1);
  if (nvec <= 4) TAAC_RESIDUAL_NORM(4, 1);
  if (nvec <= 8) TAAC_RESIDUAL_NORM(8, 1);
  if (nvec <= 16) TAAC_RESIDUAL_NORM(16, 1);
  if (nvec <= 32) TAAC_RESIDUAL_NORM(32, 1);
  if (nvec <= 64) TAAC_RESIDUAL_NORM(64, 1);
  if (nvec <= 128) TAAC_RESIDUAL_NORM(64, 2);
  if (nvec <= 256) TAAC_RESIDUAL_NORM(64, 4);
  TAAC_RESIDUAL_NORM(64, 8);
#undef TAAC_RESIDUAL_NORM
}

template <typename T>
int dispatch_residual_bwd(const char* name, const void* hv, const void* wv, const void* dyv, const void* dsv, void* dhv, void* dwv,
                          float* workspace, int64_t workspace_floats, int64_t rows, int cols, float eps, hipStream_t s) {
  const T *h = static_cast<const T*>(hv), *w = static_cast<const T*>(wv), *dy = static_cast<const T*>(dyv), *ds = static_cast<const T*>(dsv);
  T* dh = static_cast<T*>(dhv);
  constexpr int VEC = Pack<T>::VEC;
  const int nvec = cols / VEC;
  const bool vec = cols % VEC == 0 && aligned16(h) && aligned16(w) && aligned16(dy) && aligned16(ds) && aligned16(dh) &&
                   nvec <= kWave * kBwdMaxNV;
  int G = 1;
  while (G < nvec && G < kWave) G *= 2;
  const int64_t rows_at_once = vec ? static_cast<int64_t>(kBlock / G) * (nvec <= kWave ? 2 : 1) : 1;
  int64_t blocks = (rows + rows_at_once - 1) / rows_at_once;
  if (blocks > kBwdMaxBlocks) blocks = kBwdMaxBlocks;
  if (workspace == nullptr || workspace_floats < blocks * cols)
    return set_error(TAAC_ERR_INVALID_VALUE, "%s: workspace must hold %lld floats", name, (long long)(blocks * cols));
  const dim3 grid(static_cast<uint32_t>(blocks));
#define TAAC_RESIDUAL_BWD(GG, NV)                                                                                                  \
  hipLaunchKernelGGL((residual_norm_bwd_vec_kernel<T, GG, NV>), grid, dim3(kBlock), 0, s, h, w, dy, ds, dh, workspace, rows, cols, \
                     nvec, eps);                                                                                                   \
  break
  if (rows > 0 && !vec) {
    hipLaunchKernelGGL((residual_norm_bwd_generic_kernel<T>), grid, dim3(kBlock), 0, s, h, w, dy, ds, dh, workspace, rows, cols, eps);
  } else if (rows > 0) {
    switch (G) {
      case 1: TAAC_RESIDUAL_BWD(1, 1);
      case 2: TAAC_RESIDUAL_BWD(2, 1);
      case 4: TAAC_RESIDUAL_BWD(4, 1);
      case 8: TAAC_RESIDUAL_BWD(8, 1);
      case 16: TAAC_RESIDUAL_BWD(16, 1);
      case 32: TAAC_RESIDUAL_BWD(32, 1);
      default:
        if (nvec <= 64) { TAAC_RESIDUAL_BWD(64, 1); }
        if (nvec <= 128) { TAAC_RESIDUAL_BWD(64, 2); }
        TAAC_RESIDUAL_BWD(64, 4);
    }
  }
#undef TAAC_RESIDUAL_BWD
  hipLaunchKernelGGL((norm_bwd_reduce_kernel<T>), dim3((cols + 15) / 16), dim3(kBlock), 0, s, workspace, static_cast<int>(blocks), cols, 1,
                     static_cast<T*>(dwv), static_cast<T*>(nullptr));
  return TAAC_OK;
}

int check_rows(const char* name, int64_t rows, int32_t cols) {
  if (rows < 0 || cols <= 0) return set_error(TAAC_ERR_INVALID_VALUE, "%s: rows must be >= 0 and cols > 0", name);
  if (rows > 0x7fffffffLL) return set_error(TAAC_ERR_UNSUPPORTED, "%s: more than 2^31-1 rows", name);
  return TAAC_OK;
}

template <bool FP8>
int fwd_entry(const char* name, const void* x, const void* residual, const void* w, void* summed, void* out, float* row_amax, int64_t rows,
              int32_t cols, float eps, int dtype, void* stream) {
  if (int rc = check_rows(name, rows, cols)) return rc;
  if (dtype != TAAC_F32 && dtype != TAAC_BF16 && dtype != TAAC_F16) return set_error(TAAC_ERR_INVALID_VALUE, "%s: unknown dtype %d", name, dtype);
  if (rows == 0) return TAAC_OK;
  if (!x || !residual || !w || !summed || !out || (FP8 && !row_amax)) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null tensor pointer", name);
  hipStream_t s = as_stream(stream);
  if (dtype == TAAC_F32) dispatch_fwd<float, FP8>(x, residual, w, summed, out, row_amax, rows, cols, eps, s);
  if (dtype == TAAC_BF16) dispatch_fwd<bf16_t, FP8>(x, residual, w, summed, out, row_amax, rows, cols, eps, s);
  if (dtype == TAAC_F16) dispatch_fwd<f16_t, FP8>(x, residual, w, summed, out, row_amax, rows, cols, eps, s);
  return check_launch(name);
}

}  // namespace
}  // namespace taac

extern "C" int taac_residual_rmsnorm_fwd(const void* x, const void* residual, const void* w, void* summed, void* y, int64_t rows,
                                         int32_t cols, float eps, int dtype, void* stream) {
  return taac::fwd_entry<false>("taac_residual_rmsnorm_fwd", x, residual, w, summed, y, nullptr, rows, cols, eps, dtype, stream);
}

extern "C" int taac_residual_rmsnorm_fp8_fwd(const void* x, const void* residual, const void* w, void* summed, void* q, float* row_amax,
                                             int64_t rows, int32_t cols, float eps, int dtype, void* stream) {
  return taac::fwd_entry<true>("taac_residual_rmsnorm_fp8_fwd", x, residual, w, summed, q, row_amax, rows, cols, eps, dtype, stream);
}

extern "C" int taac_residual_rmsnorm_bwd(const void* summed, const void* w, const void* dy, const void* dsummed, void* dx, void* dw,
                                         float* workspace, int64_t workspace_floats, int64_t rows, int32_t cols, float eps, int dtype,
                                         void* stream) {
  using namespace taac;
  const char* name = "taac_residual_rmsnorm_bwd";
  if (int rc = check_rows(name, rows, cols)) return rc;
  if (!dw || (rows > 0 && (!summed || !w || !dy || !dx))) return set_error(TAAC_ERR_INVALID_VALUE, "%s: null tensor pointer", name);
  hipStream_t s = as_stream(stream);
  int rc;
  switch (dtype) {
    case TAAC_F32: rc = dispatch_residual_bwd<float>(name, summed, w, dy, dsummed, dx, dw, workspace, workspace_floats, rows, cols, eps, s); break;
    case TAAC_BF16: rc = dispatch_residual_bwd<bf16_t>(name, summed, w, dy, dsummed, dx, dw, workspace, workspace_floats, rows, cols, eps, s); break;
    case TAAC_F16: rc = dispatch_residual_bwd<f16_t>(name, summed, w, dy, dsummed, dx, dw, workspace, workspace_floats, rows, cols, eps, s); break;
    default: return set_error(TAAC_ERR_INVALID_VALUE, "%s: unknown dtype %d", name, dtype);
  }
  if (rc != TAAC_OK) return rc;
  return check_launch(name);
}
