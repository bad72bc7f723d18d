// Typed vector access for the mixer kernels: V adjacent elements of float,
// bfloat16 or float16 moved as one word and widened to float32.
#pragma once

#include "wkv_device.cuh"

namespace wkv {

template <int kBytes>
struct Word;
template <>
struct Word<2> {
  using type = uint16_t;
};
template <>
struct Word<4> {
  using type = uint32_t;
};
template <>
struct Word<8> {
  using type = uint2;
};
template <>
struct Word<16> {
  using type = uint4;
};

// V elements of T as they lie in memory (V * sizeof(T) is 2, 4, 8 or 16 bytes,
// and addresses are multiples of that).
template <typename T, int V>
struct Vec {
  using word = typename Word<V * static_cast<int>(sizeof(T))>::type;
  union {
    word w;
    T e[V];
  };
  __device__ __forceinline__ Vec() {}
  __device__ __forceinline__ static Vec load(const T* p) {
    Vec r;
    r.w = *reinterpret_cast<const word*>(p);
    return r;
  }
  __device__ __forceinline__ static Vec load_once(const T* p) {  // read-only data that no other thread reads again
    Vec r;
    if constexpr (V * sizeof(T) == 2)
      r.w = __ldcs(reinterpret_cast<const unsigned short*>(p));
    else
      r.w = __ldcs(reinterpret_cast<const word*>(p));
    return r;
  }
  __device__ __forceinline__ static Vec zero() {
    Vec r;
    r.w = word{};
    return r;
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<word*>(p) = w; }
  __device__ __forceinline__ void get(float (&f)[V]) const {
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
      const uint32_t* u = reinterpret_cast<const uint32_t*>(&w);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const f2 p = Pair<T>::unpack(u[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = Pair<T>::scalar(e[i]);
    }
  }
  __device__ __forceinline__ void set(const float (&f)[V]) {
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
      uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) u[i] = Pair<T>::pack(f2{f[2 * i], f[2 * i + 1]});
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = Pair<T>::from_float(f[i]);
    }
  }
};

// 1 / (1 + e^-v) for results of type T; 0 and 1 at the infinities. The product v log2(e)
// is off by up to half an ulp of itself, which the exponential turns into a relative
// error of |v| 2^-24: nothing next to a 16-bit type's rounding. For float32 what is
// missing, -v less the product times ln(2), corrects the exponential. (Where the product
// overflows that is no number, and the maximum leaves the infinity or zero as it is.)
template <typename T>
__device__ __forceinline__ float sigmoid1(float v) {
  const float p = -v * kL2E;
  if constexpr (sizeof(T) == 2) return rcp(1.f + ex2(p));
  return rcp(fmaf(ex2(p), fmaxf(1.f + fmaf(p, -0.6931471806f, -v), 0.5f), 1.f));
}
template <typename T>
__device__ __forceinline__ f2 sigmoid2(f2 v) {
  const f2 p = mul2(v, splat(-kL2E));
  if constexpr (sizeof(T) == 2) return rcpx2(add2(ex2x2(p), splat(1.f)));
  const f2 c = add2(fma2(p, splat(-0.6931471806f), f2{-v.x, -v.y}), splat(1.f));
  return rcpx2(fma2(ex2x2(p), f2{fmaxf(c.x, 0.5f), fmaxf(c.y, 0.5f)}, splat(1.f)));
}

// Column sums of `rows` float32 rows of `blocks` groups of C columns, in row order
// within each of kRows strides and then over the strides in order, so the result does
// not depend on timing. Group k goes to out[k][c * step[k]]. A CTA of 32 kRows threads
// sums 32 columns; neighbouring lanes read neighbouring columns.
constexpr int kSumGroups = 6;
struct ColSumArgs {
  const float* in;
  float* out[kSumGroups];
  int step[kSumGroups];
  int rows, blocks;
  int64_t C;
};

template <int kRows>
__device__ __forceinline__ void column_sums(const ColSumArgs& a, int64_t block) {
  __shared__ float red[kRows][33];
  const int x = threadIdx.x % 32, y = threadIdx.x / 32;
  const int64_t width = a.C * a.blocks, col = block * 32 + x;
  float s = 0.f;
  if (col < width) {
    const float* p = a.in + col;
    for (int r = y; r < a.rows; r += kRows * 10) {  // ten rows under way at a time
      float v[10];
#pragma unroll
      for (int i = 0; i < 10; ++i) v[i] = r + i * kRows < a.rows ? p[(int64_t)(r + i * kRows) * width] : 0.f;
#pragma unroll
      for (int i = 0; i < 10; ++i) s += v[i];
    }
  }
  red[y][x] = s;
  __syncthreads();
  if (y == 0 && col < width) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) t += red[i][x];
    const int k = (int)(col / a.C);
    const int64_t c = col - (int64_t)k * a.C;
    if (a.out[k]) a.out[k][c * a.step[k]] = t;
  }
}

__global__ void __launch_bounds__(1024) column_sum_kernel(ColSumArgs a) { column_sums<32>(a, blockIdx.x); }

}  // namespace wkv
