// Matrix-vector products with 4-bit weights and group scales (sm_100a).
//
//   y[m][n] = sum_k x[m][k] * scale[n][k / G] * (q[n][k] - zero[n][k / G]) (+ bias[n])
// q holds two weights a byte (even k in the low nibble), rows of ceil(K / 32) * 16
// bytes; scales bfloat16, zeros one byte each (8 without them). float32 sums.
#pragma once

#include "row_io.cuh"

namespace wkv {

constexpr int kQ4Threads = 128;
constexpr int kQ4Tokens = 8;

struct Q4Args {
  const void* x;  // [M][K]
  const uint8_t* q;
  const __nv_bfloat16* scale;
  const uint8_t* zero;  // or null
  const float* bias;    // [N] or null
  void* y;              // [M][N]
  int64_t x_s;
  int M, N, K, G, groups, pitch;
};

template <typename T>
__global__ void __launch_bounds__(kQ4Threads) q4_matvec_kernel(Q4Args a) {
  const int n = blockIdx.x * (kQ4Threads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (n >= a.N) return;
  const int m0 = blockIdx.y * kQ4Tokens, mc = min(kQ4Tokens, a.M - m0);
  const T* x = static_cast<const T*>(a.x) + m0 * a.x_s;
  float acc[kQ4Tokens] = {};
  for (int k = lane; k < a.K; k += 32) {
    const int byte = a.q[(int64_t)n * a.pitch + k / 2], g = k / a.G;
    const int q = (k & 1) ? byte >> 4 : byte & 15;
    const int z = a.zero ? a.zero[(int64_t)n * a.groups + g] : 8;
    const float w = (float)(q - z) * __bfloat162float(a.scale[(int64_t)n * a.groups + g]);
    for (int m = 0; m < mc; ++m) acc[m] = fmaf(Pair<T>::scalar(x[m * a.x_s + k]), w, acc[m]);
  }
  for (int m = 0; m < mc; ++m) {
    float s = acc[m];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
    if (lane == 0)
      static_cast<T*>(a.y)[(int64_t)(m0 + m) * a.N + n] = Pair<T>::from_float(s + (a.bias ? a.bias[n] : 0.f));
  }
}

}  // namespace wkv
