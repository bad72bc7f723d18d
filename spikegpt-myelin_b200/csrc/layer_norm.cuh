// Layer norm of rows of any width, forward and backward (sm_100a).
//
//   xh = (x - mean) * rstd,  y = xh * w + b      (biased variance, float32)
//   gh = gy * w,  gx = rstd (gh - mean(gh) - xh mean(gh xh))
//   gw = sum_rows gy xh,  gb = sum_rows gy
//
// Memory-bound: the forward reads x and writes y once, the backward reads x and gy
// and writes gx. A team of `span` threads (a warp to 1024 threads) holds a row in
// registers, 16 values each as granules of 16 bytes, so the statistics take two passes
// over the registers (mean, then centred squares) and one over memory. A CTA of at
// least 256 threads has several teams where rows are short, walks the rows with a
// grid-wide stride, and has the next row's words under way while it works on one: that
// is what keeps the memory busy. Row sums go through a warp butterfly and, for wider
// teams, the warps' sums in warp order through shared memory, two buffers in turn so
// that one barrier a sum is enough. The backward keeps gw and gb of its columns in
// registers over all its rows, adds its teams' in team order and leaves one partial row
// a CTA.
//
// Rows that are not 16-byte aligned (odd widths, odd pitches) move as words of V
// values, neighbouring lanes' side by side, and are re-ordered into the same granules
// through shared memory (where w and b lie as well): a row's result does not depend on
// how it lies in memory.
#pragma once

#include "row_io.cuh"

namespace wkv {

constexpr int kNormValues = 16;  // of a thread
constexpr int kNormMaxC = 1024 * kNormValues;

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
  int span;  // threads of a row, a power of two from 32
  float eps;
};

// Rows and parameters as the kernels see them. kStaged: through shared memory.
template <typename T, int V>
struct NormIo {
  static constexpr int kGran = 16 / (int)sizeof(T), kGrans = kNormValues / kGran, kWords = kNormValues / V;
  static constexpr bool kStaged = V < kGran;

  struct Row {
    Vec<T, V> w[kWords];
    __device__ __forceinline__ void load(const T* row, int lane, int span, int C, bool live) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const int c = (i * span + lane) * V;
        w[i] = live && c < C ? Vec<T, V>::load_once(row + c) : Vec<T, V>::zero();
      }
    }
  };
  static __device__ __forceinline__ void sync(int span) {
    if (span == 32)
      __syncwarp();
    else
      __syncthreads();
  }
  // The granules of a row. Staged rows go through `buf` (span * 16 values of the team).
  static __device__ __forceinline__ void spread(const Row& r, T* buf, int lane, int span) {
    if constexpr (kStaged)
#pragma unroll
      for (int i = 0; i < kWords; ++i) r.w[i].store(buf + (i * span + lane) * V);
  }
  static __device__ __forceinline__ void gather(Row& r, const T* buf, int lane, int span) {
    if constexpr (kStaged)
#pragma unroll
      for (int i = 0; i < kGrans; ++i) {
        const Vec<T, kGran> g = Vec<T, kGran>::load(buf + (i * span + lane) * kGran);
#pragma unroll
        for (int k = 0; k < kGran / V; ++k)
#pragma unroll
          for (int v = 0; v < V; ++v) r.w[i * (kGran / V) + k].e[v] = g.e[k * V + v];
      }
  }
  // Values of granule i of a gathered row.
  static __device__ __forceinline__ void get(const Row& r, int i, float (&f)[kGran]) {
#pragma unroll
    for (int k = 0; k < kGran / V; ++k) {
      float p[V];
      r.w[i * (kGran / V) + k].get(p);
#pragma unroll
      for (int v = 0; v < V; ++v) f[k * V + v] = p[v];
    }
  }
  // A parameter's granule: from shared memory where rows are staged (padded there), else
  // from the parameter itself, whose C is then a multiple of the granule.
  static __device__ __forceinline__ void param(const float* p, const float* staged, int c, float fill,
                                               float (&f)[kGran]) {
    const float* from = kStaged ? staged : p;
    if (!kStaged && p == nullptr) {
#pragma unroll
      for (int v = 0; v < kGran; ++v) f[v] = fill;
    } else {
#pragma unroll
      for (int v = 0; v < kGran; v += 4) {
        const float4 u = *reinterpret_cast<const float4*>(from + c + v);
        f[v] = u.x, f[v + 1] = u.y, f[v + 2] = u.z, f[v + 3] = u.w;
      }
    }
  }
  static __device__ __forceinline__ void stage_param(const float* p, float* to, int C, int span, float fill) {
    for (int c = threadIdx.x; c < span * kNormValues; c += blockDim.x) to[c] = c < C ? (p ? p[c] : fill) : 0.f;
  }
  // Writes a row given by granules.
  static __device__ __forceinline__ void store(T* row, T* buf, int lane, int span, int C, bool live,
                                               const float (&f)[kGrans][kGran]) {
#pragma unroll
    for (int i = 0; i < kGrans; ++i) {
      const int c = (i * span + lane) * kGran;
      Vec<T, kGran> o;
      o.set(f[i]);
      if constexpr (kStaged)
        o.store(buf + c);
      else if (live && c < C)
        o.store(row + c);
    }
    if constexpr (kStaged) {
      sync(span);
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const int c = (i * span + lane) * V;
        if (live && c < C) Vec<T, V>::load(buf + c).store(row + c);
      }
    }
  }
};

// Shared memory of the kernels, in bytes: staged parameters and rows, and the
// backward's sums where a CTA has several teams.
inline size_t norm_smem(bool backward, bool staged, size_t es, int span, int threads, int64_t C) {
  size_t n = backward && threads > span ? (2 * C * sizeof(float) + 15) / 16 * 16 : 0;
  if (staged) n += (size_t)span * kNormValues * sizeof(float) * (backward ? 1 : 2) + threads * kNormValues * es * (backward ? 2 : 1);
  return n;
}

// The sums of u and v over the threads of a row (teams of `span` threads); `slot`
// alternates between calls.
__device__ __forceinline__ float2 norm_sums(float u, float v, int span, float2 (*red)[32], int slot) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    u += __shfl_xor_sync(kFull, u, o);
    v += __shfl_xor_sync(kFull, v, o);
  }
  if (span == 32) return make_float2(u, v);
  if ((threadIdx.x & 31) == 0) red[slot][threadIdx.x >> 5] = make_float2(u, v);
  __syncthreads();
  const int warps = span >> 5, first = (threadIdx.x >> 5) / warps * warps;
  float2 s = make_float2(0.f, 0.f);
  for (int i = 0; i < warps; ++i) {
    const float2 r = red[slot][first + i];
    s.x += r.x;
    s.y += r.y;
  }
  return s;
}

// kThr: the CTA's threads, 256, 512 (rows past 4096) or 1024 (past 8192, where 64
// registers a thread make the backward spill: such rows are rare).
template <typename T, int V, int kThr>
__global__ void __launch_bounds__(kThr, kThr == 256 ? 2 : 1) layer_norm_fwd_kernel(NormArgs a) {
  using Io = NormIo<T, V>;
  constexpr int G = Io::kGran, kGrans = Io::kGrans;
  extern __shared__ __align__(16) char smem[];
  __shared__ float2 red[2][32];
  const int lane = threadIdx.x & (a.span - 1), teams = blockDim.x / a.span, team = threadIdx.x / a.span;
  float* sw = reinterpret_cast<float*>(smem);
  float* sb = sw + a.span * kNormValues;
  T* buf = reinterpret_cast<T*>(sb + a.span * kNormValues) + team * a.span * kNormValues;
  const int64_t first = (int64_t)blockIdx.x * teams, step = (int64_t)gridDim.x * teams;
  const float inv = 1.f / a.C;
  typename Io::Row row;
  row.load(static_cast<const T*>(a.x) + (first + team) * a.x_s, lane, a.span, a.C, first + team < a.rows);
  if constexpr (Io::kStaged) {
    Io::stage_param(a.w, sw, a.C, a.span, 1.f);
    Io::stage_param(a.b, sb, a.C, a.span, 0.f);
    __syncthreads();
  }
  for (int64_t r0 = first; r0 < a.rows; r0 += step) {
    const int64_t r = r0 + team;
    if constexpr (Io::kStaged) {
      Io::spread(row, buf, lane, a.span);
      Io::sync(a.span);
      Io::gather(row, buf, lane, a.span);
    }
    float f[kGrans][G], s = 0.f;
#pragma unroll
    for (int i = 0; i < kGrans; ++i) {
      Io::get(row, i, f[i]);
#pragma unroll
      for (int v = 0; v < G; ++v) s += f[i][v];
    }
    row.load(static_cast<const T*>(a.x) + (r + step) * a.x_s, lane, a.span, a.C, r + step < a.rows);
    const float mu = norm_sums(s, 0.f, a.span, red, 0).x * inv;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < kGrans; ++i)
#pragma unroll
      for (int v = 0; v < G; ++v) {
        f[i][v] -= mu;
        if ((i * a.span + lane) * G + (Io::kStaged ? v : 0) < a.C) s = fmaf(f[i][v], f[i][v], s);
      }
    const float rs = rsqrtf(norm_sums(s, 0.f, a.span, red, 1).x * inv + a.eps);
#pragma unroll
    for (int i = 0; i < kGrans; ++i) {
      const int c = (i * a.span + lane) * G;
      if (Io::kStaged || c < a.C) {
        float w[G], b[G];
        Io::param(a.w, sw, c, 1.f, w);
        Io::param(a.b, sb, c, 0.f, b);
#pragma unroll
        for (int v = 0; v < G; ++v) f[i][v] = fmaf(f[i][v] * rs, w[v], b[v]);
      }
    }
    Io::store(static_cast<T*>(a.y) + r * a.C, buf, lane, a.span, a.C, r < a.rows, f);
    if constexpr (Io::kStaged) Io::sync(a.span);  // buf is rewritten
    if (r < a.rows && lane == 0) {
      a.mean[r] = mu;
      a.rstd[r] = rs;
    }
  }
}

template <typename T, int V, int kThr>
__global__ void __launch_bounds__(kThr, kThr == 256 ? 2 : 1) layer_norm_bwd_kernel(NormArgs a) {
  using Io = NormIo<T, V>;
  constexpr int G = Io::kGran, kGrans = Io::kGrans;
  extern __shared__ __align__(16) char smem[];  // [2][C] sums where a CTA has several teams, then what is staged
  __shared__ float2 red[2][32];
  const int lane = threadIdx.x & (a.span - 1), teams = blockDim.x / a.span, team = threadIdx.x / a.span;
  float* acc = reinterpret_cast<float*>(smem);
  float* sw = reinterpret_cast<float*>(smem + (teams > 1 ? (2 * a.C * sizeof(float) + 15) / 16 * 16 : 0));
  T* bx = reinterpret_cast<T*>(sw + a.span * kNormValues) + team * 2 * a.span * kNormValues;
  T* bg = bx + a.span * kNormValues;
  const int64_t first = (int64_t)blockIdx.x * teams, step = (int64_t)gridDim.x * teams;
  const float inv = 1.f / a.C;
  float gw[kGrans][G], gb[kGrans][G];
#pragma unroll
  for (int i = 0; i < kGrans; ++i)
#pragma unroll
    for (int v = 0; v < G; ++v) gw[i][v] = gb[i][v] = 0.f;
  typename Io::Row nx, ng;
  float nmu = 0.f, nrs = 0.f;
  auto fetch = [&](int64_t r) {
    const bool live = r < a.rows;
    nx.load(static_cast<const T*>(a.x) + r * a.x_s, lane, a.span, a.C, live);
    ng.load(static_cast<const T*>(a.gy) + r * a.gy_s, lane, a.span, a.C, live);
    nmu = live ? a.mean[r] : 0.f;
    nrs = live ? a.rstd[r] : 0.f;
  };
  fetch(first + team);
  if constexpr (Io::kStaged) {
    Io::stage_param(a.w, sw, a.C, a.span, 1.f);
    __syncthreads();
  }
  int slot = 0;
  for (int64_t r0 = first; r0 < a.rows; r0 += step, slot ^= 1) {
    const int64_t r = r0 + team;
    typename Io::Row x = nx, g = ng;
    const float mu = nmu, rs = nrs;
    if constexpr (Io::kStaged) {
      Io::spread(x, bx, lane, a.span);
      Io::spread(g, bg, lane, a.span);
      Io::sync(a.span);
    }
    fetch(r + step);
    if constexpr (Io::kStaged) {
      Io::gather(x, bx, lane, a.span);
      Io::gather(g, bg, lane, a.span);
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < kGrans; ++i) {
      const int c = (i * a.span + lane) * G;
      if (Io::kStaged || c < a.C) {  // what is staged past C has w = gy = 0
        float xv[G], gv[G], w[G];
        Io::get(x, i, xv);
        Io::get(g, i, gv);
        Io::param(a.w, sw, c, 1.f, w);
#pragma unroll
        for (int v = 0; v < G; ++v) {
          const float h = (xv[v] - mu) * rs, gh = gv[v] * w[v];
          s1 += gh;
          s2 = fmaf(gh, h, s2);
          gw[i][v] = fmaf(gv[v], h, gw[i][v]);
          gb[i][v] += gv[v];
        }
      }
    }
    const float2 m = norm_sums(s1, s2, a.span, red, slot);
    const float m1 = m.x * inv, m2 = m.y * inv;
    float o[kGrans][G];
#pragma unroll
    for (int i = 0; i < kGrans; ++i) {
      const int c = (i * a.span + lane) * G;
      if (Io::kStaged || c < a.C) {
        float xv[G], gv[G], w[G];
        Io::get(x, i, xv);
        Io::get(g, i, gv);
        Io::param(a.w, sw, c, 1.f, w);
#pragma unroll
        for (int v = 0; v < G; ++v) o[i][v] = rs * (fmaf(gv[v], w[v], -m1) - (xv[v] - mu) * rs * m2);
      }
    }
    if constexpr (Io::kStaged) Io::sync(a.span);  // every lane has gathered from bx
    Io::store(static_cast<T*>(a.y) + r * a.C, bx, lane, a.span, a.C, r < a.rows, o);
    if constexpr (Io::kStaged) Io::sync(a.span);
  }
  float* part = a.partial + (int64_t)blockIdx.x * 2 * a.C;
  float* to = teams > 1 ? acc : part;
  for (int k = 0; k < teams; ++k) {
    if (team == k) {
#pragma unroll
      for (int i = 0; i < kGrans; ++i) {
        const int c = (i * a.span + lane) * G;
#pragma unroll
        for (int v = 0; v < G; ++v)
          if (c + v < a.C) {
            to[c + v] = (k ? to[c + v] : 0.f) + gw[i][v];
            to[a.C + c + v] = (k ? to[a.C + c + v] : 0.f) + gb[i][v];
          }
      }
    }
    if (teams > 1) __syncthreads();
  }
  if (teams > 1)
    for (int c = threadIdx.x; c < 2 * a.C; c += blockDim.x) part[c] = acc[c];
}

}  // namespace wkv
