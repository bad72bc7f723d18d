// Layer norm of rows of any width, forward and backward (sm_100a).
//
//   xh = (x - mean) * rstd,  y = xh * w + b      (biased variance, float32)
//   gh = gy * w,  gx = rstd (gh - mean(gh) - xh mean(gh xh))
//   gw = sum_rows gy xh,  gb = sum_rows gy
// Two passes over the row for the statistics (mean, then centred squares).
#pragma once

#include "row_io.cuh"

namespace wkv {

constexpr int kNormThreads = 256;
constexpr int kNormMaxC = 16384;

struct NormArgs {
  const void* x;
  const float* w;  // [C] or null (ones)
  const float* b;  // [C] or null (zeros)
  const void* gy;
  void* y;  // y; gx in the backward
  float* mean;
  float* rstd;
  float* partial;  // [grid][2][C]
  int64_t rows, x_s, gy_s;
  int C;
  float eps;
};

__device__ __forceinline__ float norm_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) s += red[i];
  return s;
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads) layer_norm_fwd_kernel(NormArgs a) {
  __shared__ float red[32];
  const int64_t r = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + r * a.x_s;
  T* y = static_cast<T*>(a.y) + r * a.C;
  float s = 0.f;
  for (int c = threadIdx.x; c < a.C; c += blockDim.x) s += Pair<T>::scalar(x[c]);
  const float mu = norm_sum(s, red) / a.C;
  s = 0.f;
  for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
    const float d = Pair<T>::scalar(x[c]) - mu;
    s = fmaf(d, d, s);
  }
  const float rs = rsqrtf(norm_sum(s, red) / a.C + a.eps);
  for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
    const float h = (Pair<T>::scalar(x[c]) - mu) * rs;
    y[c] = Pair<T>::from_float(fmaf(h, a.w ? a.w[c] : 1.f, a.b ? a.b[c] : 0.f));
  }
  if (threadIdx.x == 0) {
    a.mean[r] = mu;
    a.rstd[r] = rs;
  }
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads) layer_norm_bwd_kernel(NormArgs a) {
  extern __shared__ float acc[];  // [2][C]
  __shared__ float red[32];
  for (int c = threadIdx.x; c < 2 * a.C; c += blockDim.x) acc[c] = 0.f;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.x_s;
    const T* g = static_cast<const T*>(a.gy) + r * a.gy_s;
    T* gx = static_cast<T*>(a.y) + r * a.C;
    const float mu = a.mean[r], rs = a.rstd[r];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
      const float h = (Pair<T>::scalar(x[c]) - mu) * rs, gy = Pair<T>::scalar(g[c]);
      const float gh = gy * (a.w ? a.w[c] : 1.f);
      s1 += gh;
      s2 = fmaf(gh, h, s2);
      acc[c] = fmaf(gy, h, acc[c]);
      acc[a.C + c] += gy;
    }
    const float m1 = norm_sum(s1, red) / a.C, m2 = norm_sum(s2, red) / a.C;
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
      const float h = (Pair<T>::scalar(x[c]) - mu) * rs;
      const float gh = Pair<T>::scalar(g[c]) * (a.w ? a.w[c] : 1.f);
      gx[c] = Pair<T>::from_float(rs * (gh - m1 - h * m2));
    }
  }
  float* part = a.partial + (int64_t)blockIdx.x * 2 * a.C;
  for (int c = threadIdx.x; c < 2 * a.C; c += blockDim.x) part[c] = acc[c];
}

}  // namespace wkv
