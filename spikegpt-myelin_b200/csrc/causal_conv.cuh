// Short causal convolution of every channel with its own W <= 4 taps, and its
// gradient and single-token step (sm_100a).
//
//   u[t] = bias + sum_j w[j] x[t - W + 1 + j],   y[t] = silu(u[t]) or u[t]
// with the rows before t = 0 taken from a cached window (or zero). With lengths,
// row t >= length gives y = 0 and reads nothing, whatever lies there, and the new
// window holds the last W - 1 rows inside the length. Gradient:
//   gu = gy * silu'(u),  gx[t] = sum_j w[j] gu[t + W - 1 - j],
//   gw[j] = sum gu[t] x[t - W + 1 + j],  gb = sum gu
// float32 arithmetic; x, y and their gradients in the tensor's type.
//
// Memory-bound: the forward reads x and writes y once (2 e bytes per element of
// size e), the backward reads x and gy and writes gx. A thread holds V adjacent
// channels and walks kConvSteps rows with the window in registers, so a row is
// read once but for the W - 1 rows shared by neighbouring walks. The per-tap
// sums of a walk go to a partial row and are added in a fixed order. Measured at
// 8 x 1024 x 1024 bfloat16: forward 16 us (2.0 TB/s), backward 30 us (1.7 TB/s), sums
// 8 us: at this size the walks are short of warps (1024 CTAs of two) and bound by the
// latency of their rows and the float32 arithmetic (about 10 operations an element
// forward, 25 backward), not by memory; 5 x 1003 x 1536 float32 forward 16 us. Longer
// walks would re-read less and leave SMs idle; shorter ones re-read more.
#pragma once

#include "row_io.cuh"

namespace wkv {

constexpr int kConvMaxTaps = 4;
constexpr int kConvSteps = 32;  // rows of a walk
constexpr int kConvAhead = 4;   // rows under way
constexpr int kConvThreads = 64;

struct ConvArgs {
  const void* x;
  const float* w;      // [C][W]
  const float* bias;   // [C] or null
  const void* front;   // [B][W-1][C] or null
  const int* lengths;  // [B] or null
  const void* gy;      // [B][T][C]
  void* y;             // [B][T][C]; gx in the backward
  void* window;        // [B][W-1][C] or null: the new window; gradient of `front` in the backward
  float* partial;      // [B * chunks][W + 1][C]
  int64_t x_sb, x_st;  // strides of x, in elements
  int64_t gy_sb, gy_st;
  int B, T, C;
  int chunks, cblocks;
  int silu;
  int wide_w;  // the four taps of a channel can be read as one word
};

__device__ __forceinline__ int conv_length(const ConvArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
}

// Row t of sequence b (t may lie in the window before it).
template <typename T, int V, int W>
__device__ __forceinline__ Vec<T, V> conv_row(const ConvArgs& a, int b, int t, int c, int len) {
  if (t >= 0)
    return t < len ? Vec<T, V>::load(static_cast<const T*>(a.x) + b * a.x_sb + t * a.x_st + c) : Vec<T, V>::zero();
  if (a.front == nullptr || t < 1 - W) return Vec<T, V>::zero();
  return Vec<T, V>::load(static_cast<const T*>(a.front) + ((int64_t)b * (W - 1) + (W - 1 + t)) * a.C + c);
}

template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads) causal_conv_fwd_kernel(ConvArgs a) {
  const int cb = blockIdx.x % a.cblocks;
  const int chunk = blockIdx.x / a.cblocks % a.chunks;
  const int b = blockIdx.x / a.cblocks / a.chunks;
  const int c = (cb * kConvThreads + threadIdx.x) * V;
  if (c >= a.C) return;
  const int len = conv_length(a, b);
  if (chunk == 0 && a.window != nullptr) {
#pragma unroll
    for (int i = 0; i < W - 1; ++i)
      conv_row<T, V, W>(a, b, len - (W - 1) + i, c, len)
          .store(static_cast<T*>(a.window) + ((int64_t)b * (W - 1) + i) * a.C + c);
  }
  const int t0 = chunk * kConvSteps, t1 = min(t0 + kConvSteps, a.T);
  if (t0 >= t1) return;
  float w[W][V], bias[V], win[W][V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][v] = a.w[(int64_t)(c + v) * W + j];
    bias[v] = a.bias ? a.bias[c + v] : 0.f;
  }
#pragma unroll
  for (int i = 1; i < W; ++i) conv_row<T, V, W>(a, b, t0 - W + i, c, len).get(win[i]);
  // kConvAhead rows are under way while as many are worked on
  Vec<T, V> next[kConvAhead];
  const T* x = static_cast<const T*>(a.x) + b * a.x_sb + c;
  auto fetch = [&](int t) {
#pragma unroll
    for (int i = 0; i < kConvAhead; ++i)
      next[i] = t + i < min(t1, len) ? Vec<T, V>::load(x + (t + i) * a.x_st) : Vec<T, V>::zero();
  };
  fetch(t0);
  T* y = static_cast<T*>(a.y) + ((int64_t)b * a.T + t0) * a.C + c;
  for (int t = t0; t < t1; t += kConvAhead) {
    Vec<T, V> cur[kConvAhead];
#pragma unroll
    for (int i = 0; i < kConvAhead; ++i) cur[i] = next[i];
    fetch(t + kConvAhead);
#pragma unroll
    for (int k = 0; k < kConvAhead; ++k, y += a.C) {
      if (t + k >= t1) break;
#pragma unroll
      for (int i = 0; i + 1 < W; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) win[i][v] = win[i + 1][v];
      cur[k].get(win[W - 1]);
      float f[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float u = bias[v];
#pragma unroll
        for (int j = 0; j < W; ++j) u = fmaf(w[j][v], win[j][v], u);
        f[v] = a.silu ? u * sigmoid1<T>(u) : u;
      }
      Vec<T, V> out;
      out.set(f);
      if (t + k >= len) out = Vec<T, V>::zero();
      out.store(y);
    }
  }
}

// A walk visits rows t0 .. t1 + W - 2: gx[t] needs gu[t] .. gu[t + W - 1]. The
// walk of the first rows starts with the window's rows, whose gradient it writes.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads) causal_conv_bwd_kernel(ConvArgs a) {
  const int cb = blockIdx.x % a.cblocks;
  const int chunk = blockIdx.x / a.cblocks % a.chunks;
  const int b = blockIdx.x / a.cblocks / a.chunks;
  const int c = (cb * kConvThreads + threadIdx.x) * V;
  if (c >= a.C) return;
  const int len = conv_length(a, b);
  const int t0 = chunk * kConvSteps, t1 = min(t0 + kConvSteps, a.T);
  float w[W][V], bias[V], win[W][V], gu[W][V], gw[W + 1][V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][v] = a.w[(int64_t)(c + v) * W + j];
    bias[v] = a.bias ? a.bias[c + v] : 0.f;
#pragma unroll
    for (int j = 0; j <= W; ++j) gw[j][v] = 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) gu[j][v] = 0.f;
  }
#pragma unroll
  for (int i = 1; i < W; ++i) conv_row<T, V, W>(a, b, t0 - W + i, c, len).get(win[i]);
  T* gx = static_cast<T*>(a.y) + (int64_t)b * a.T * a.C + c;
  const T* gy = static_cast<const T*>(a.gy) + b * a.gy_sb + c;
  const int t_end = t1 + W - 1;
  Vec<T, V> nx[kConvAhead], ng[kConvAhead];
  const T* x = static_cast<const T*>(a.x) + b * a.x_sb + c;
  auto fetch = [&](int t) {
#pragma unroll
    for (int i = 0; i < kConvAhead; ++i) {
      const bool on = t + i < min(t_end, len);
      nx[i] = on ? Vec<T, V>::load(x + (t + i) * a.x_st) : Vec<T, V>::zero();
      ng[i] = on ? Vec<T, V>::load(gy + (t + i) * a.gy_st) : Vec<T, V>::zero();
    }
  };
  fetch(t0);
  for (int tt = t0; tt < t_end; tt += kConvAhead) {
    Vec<T, V> cx[kConvAhead], cg[kConvAhead];
#pragma unroll
    for (int i = 0; i < kConvAhead; ++i) {
      cx[i] = nx[i];
      cg[i] = ng[i];
    }
    fetch(tt + kConvAhead);
#pragma unroll
    for (int k = 0; k < kConvAhead; ++k) {
      const int t = tt + k;
      if (t >= t_end) break;
#pragma unroll
      for (int i = 0; i + 1 < W; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          win[i][v] = win[i + 1][v];
          gu[i][v] = gu[i + 1][v];
        }
      cx[k].get(win[W - 1]);
      float g[V];
      cg[k].get(g);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (a.silu) {
          float u = bias[v];
#pragma unroll
          for (int j = 0; j < W; ++j) u = fmaf(w[j][v], win[j][v], u);
          const float s = sigmoid1<T>(u);
          g[v] *= s * fmaf(u, 1.f - s, 1.f);
        }
        if (t >= len) g[v] = 0.f;  // a window of infinities gives its row no gradient
        gu[W - 1][v] = g[v];
      }
      if (t < min(t1, len)) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
          for (int j = 0; j < W; ++j) gw[j][v] = fmaf(g[v], win[j][v], gw[j][v]);
          gw[W][v] += g[v];
        }
      }
      const int at = t - W + 1;  // the row whose gradient is complete now
      if (at >= t0 || (chunk == 0 && a.window != nullptr && at < 0)) {
        float f[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          f[v] = 0.f;
#pragma unroll
          for (int j = 0; j < W; ++j) f[v] = fmaf(w[j][v], gu[W - 1 - j][v], f[v]);
        }
        Vec<T, V> out;
        out.set(f);
        if (at >= 0)
          out.store(gx + (int64_t)at * a.C);
        else
          out.store(static_cast<T*>(a.window) + ((int64_t)b * (W - 1) + (W - 1 + at)) * a.C + c);
      }
    }
  }
  float* part = a.partial + ((int64_t)b * a.chunks + chunk) * (W + 1) * a.C + c;
#pragma unroll
  for (int j = 0; j <= W; ++j)
#pragma unroll
    for (int v = 0; v < V; ++v) part[(int64_t)j * a.C + v] = gw[j][v];
}

// One token: y from the window and x, and the window moved on by x, in place.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads) causal_conv_step_kernel(ConvArgs a) {
  const int cb = blockIdx.x % a.cblocks;
  const int b = blockIdx.x / a.cblocks;
  const int c = (cb * kConvThreads + threadIdx.x) * V;
  if (c >= a.C) return;
  T* window = static_cast<T*>(a.window) + (int64_t)b * (W - 1) * a.C + c;
  Vec<T, V> row[W];
#pragma unroll
  for (int i = 0; i < W - 1; ++i) row[i] = Vec<T, V>::load(window + (int64_t)i * a.C);
  row[W - 1] = Vec<T, V>::load(static_cast<const T*>(a.x) + b * a.x_sb + c);
  float u[V], w[W][V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (W == 4 && a.wide_w) {
      const float4 f = *reinterpret_cast<const float4*>(a.w + (int64_t)(c + v) * 4);
      w[0][v] = f.x, w[1 % W][v] = f.y, w[2 % W][v] = f.z, w[3 % W][v] = f.w;
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) w[j][v] = a.w[(int64_t)(c + v) * W + j];
    }
    u[v] = a.bias ? a.bias[c + v] : 0.f;
  }
#pragma unroll
  for (int j = 0; j < W; ++j) {
    float f[V];
    row[j].get(f);
#pragma unroll
    for (int v = 0; v < V; ++v) u[v] = fmaf(w[j][v], f[v], u[v]);
    if (j > 0) row[j].store(window + (int64_t)(j - 1) * a.C);
  }
  if (a.silu) {
#pragma unroll
    for (int v = 0; v < V; ++v) u[v] *= sigmoid1<T>(u[v]);
  }
  Vec<T, V> out;
  out.set(u);
  out.store(static_cast<T*>(a.y) + (int64_t)b * a.C + c);
}

}  // namespace wkv
