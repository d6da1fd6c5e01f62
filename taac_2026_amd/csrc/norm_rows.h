// Pieces shared by the row kernels of the norms (norm.hip, residual_norm.hip): 128-bit vectors of a row, sums over a workgroup,
// and the reduction of the workgroups' partial weight gradients.
#pragma once

#include "common.h"

namespace taac {
namespace {

constexpr int kBlock = 256;
constexpr int kBwdMaxBlocks = 1024;  // workgroups of a backward pass, one partial row of dw each

template <typename T>
struct Pack;
template <>
struct Pack<float> {
  static constexpr int VEC = 4;
  typedef f32x4 vec;
  static __device__ __forceinline__ void unpack(const vec& v, float* f) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = v[i];
  }
  static __device__ __forceinline__ vec pack(const float* f) {
    vec v;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = f[i];
    return v;
  }
};
template <>
struct Pack<bf16_t> {
  static constexpr int VEC = 8;
  typedef bf16x8 vec;
  static __device__ __forceinline__ void unpack(const vec& v, float* f) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = static_cast<float>(v[i]);
  }
  static __device__ __forceinline__ vec pack(const float* f) {
    vec v;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = static_cast<bf16_t>(f[i]);
    return v;
  }
};
template <>
struct Pack<f16_t> {
  static constexpr int VEC = 8;
  typedef f16x8 vec;
  static __device__ __forceinline__ void unpack(const vec& v, float* f) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = static_cast<float>(v[i]);
  }
  static __device__ __forceinline__ vec pack(const float* f) {
    vec v;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = static_cast<f16_t>(f[i]);
    return v;
  }
};

// dw[c] (and db[c]) = sum over the workgroups' partial rows in a fixed order: a workgroup owns 16 columns, thread
// (column, slice) adds the partial rows slice, slice + 16, ... and the 16 slice sums of a column are added in slice order.
template <typename T>
__global__ __launch_bounds__(kBlock) void norm_bwd_reduce_kernel(const float* __restrict__ partial, int nblocks, int cols,
                                                                  int parts, T* __restrict__ dw, T* __restrict__ db) {
  constexpr int CPB = 16, SLICES = kBlock / CPB;
  __shared__ float red[SLICES][CPB];
  const int cl = threadIdx.x % CPB, slice = threadIdx.x / CPB;
  const int c = blockIdx.x * CPB + cl;
  for (int part = 0; part < parts; ++part) {
    float sum = 0.f;
    if (c < cols) {
#pragma unroll 4
      for (int b = slice; b < nblocks; b += SLICES) sum += partial[(static_cast<int64_t>(b) * parts + part) * cols + c];
    }
    __syncthreads();
    red[slice][cl] = sum;
    __syncthreads();
    if (slice == 0 && c < cols) {
      float total = 0.f;
#pragma unroll
      for (int sl = 0; sl < SLICES; ++sl) total += red[sl][cl];
      T* dst = part == 0 ? dw : db;
      if (dst != nullptr) dst[c] = static_cast<T>(total);
    }
  }
}

// Sum over the workgroup of up to three values at once (wavefront shuffles, then one LDS round over the wavefronts);
// every thread gets the totals. `red` is reused by consecutive calls: the leading barrier protects the previous round.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float (*red)[kBlock / kWave]) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = group_sum<kWave>(v[i]);
  __syncthreads();
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) red[i][wave] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < kBlock / kWave; ++w) total += red[i][w];
    v[i] = total;
  }
}

}  // namespace
}  // namespace taac
