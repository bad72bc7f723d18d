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
// a CTA. Measured, launches included: 16384 x 4096 bfloat16 forward 62 us (4.3 TB/s),
// backward 88 us (4.6 TB/s) and its column sums 11 us; 8192 x 512 float32 14, 23 and 9 us;
// 8192 x 16384 bfloat16 133, 368 and 21 us.
// The instructions between a row's arrival and the next one's bound it (issue slots half
// busy, memory 42 to 51 % of its nominal rate), which is why the arithmetic is packed.
//
// Rows that are not 16-byte aligned (odd widths, odd pitches) move as words of V
// values, neighbouring lanes' side by side, and are re-ordered into the same granules
// through shared memory: a row's result does not depend on how it lies in memory.
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
  static constexpr int kPairs = kNormValues / 2;
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
  // The pairs of a gathered row, in granule order.
  static __device__ __forceinline__ void get(const Row& r, f2 (&f)[kPairs]) {
    if constexpr (V == 1) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) f[i] = f2{Pair<T>::scalar(r.w[2 * i].e[0]), Pair<T>::scalar(r.w[2 * i + 1].e[0])};
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        float p[V];
        r.w[i].get(p);
#pragma unroll
        for (int v = 0; v < V; v += 2) f[(i * V + v) / 2] = f2{p[v], p[v + 1]};
      }
    }
  }
  // A parameter's pairs, held for all the rows; zeros past C, `fill` without one.
  static __device__ __forceinline__ void param(const float* p, int lane, int span, int C, float fill, f2 (&f)[kPairs]) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const int c = (i * 2 / kGran * span + lane) * kGran + i * 2 % kGran;
      f[i] = f2{c < C ? (p ? p[c] : fill) : 0.f, c + 1 < C ? (p ? p[c + 1] : fill) : 0.f};
    }
  }
  static __device__ __forceinline__ bool inside(int i, int e, int lane, int span, int C) {
    const int c = (i * 2 / kGran * span + lane) * kGran;
    return kStaged ? c + i * 2 % kGran + e < C : c < C;
  }
  // Writes a row given by pairs.
  static __device__ __forceinline__ void store(T* row, T* buf, int lane, int span, int C, bool live, const f2 (&f)[kPairs]) {
#pragma unroll
    for (int i = 0; i < kGrans; ++i) {
      const int c = (i * span + lane) * kGran;
      float p[kGran];
#pragma unroll
      for (int v = 0; v < kGran; v += 2) {
        p[v] = f[(i * kGran + v) / 2].x;
        p[v + 1] = f[(i * kGran + v) / 2].y;
      }
      Vec<T, kGran> o;
      o.set(p);
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

// Shared memory of the kernels, in bytes: the backward's sums where a CTA has several
// teams, and staged rows.
inline size_t norm_smem(bool backward, bool staged, size_t es, int span, int threads, int64_t C) {
  size_t n = backward && threads > span ? (2 * C * sizeof(float) + 15) / 16 * 16 : 0;
  if (staged) n += threads * kNormValues * es * (backward ? 2 : 1);
  return n;
}

// The sum of u (and of v: kTwo) over the threads of a row (teams of `span` threads);
// `slot` alternates between calls.
template <bool kTwo>
__device__ __forceinline__ float2 norm_sums(float u, float v, int span, float2 (*red)[32], int slot) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    u += __shfl_xor_sync(kFull, u, o);
    if (kTwo) v += __shfl_xor_sync(kFull, v, o);
  }
  if (span == 32) return make_float2(u, v);
  if ((threadIdx.x & 31) == 0) red[slot][threadIdx.x >> 5] = make_float2(u, v);
  __syncthreads();
  const int warps = span >> 5;  // lane i takes warp i's (the team's warps in turn, as often as they fit)
  const float2 r = red[slot][((threadIdx.x >> 5) & ~(warps - 1)) + (threadIdx.x & (warps - 1))];
  u = r.x;
  v = r.y;
  for (int o = warps >> 1; o > 0; o >>= 1) {
    u += __shfl_xor_sync(kFull, u, o);
    if (kTwo) v += __shfl_xor_sync(kFull, v, o);
  }
  return make_float2(u, v);
}

// CTAs of the forward that share an SM: three of 256 threads where their 80 registers
// hold a row without spilling, which is for whole aligned words of 16 bits (16384 x 4096
// 61 us, with two 67; float32 rows of 1003 22 us with two, 29 with three).
template <typename T, int V, int kThr>
__host__ __device__ constexpr int norm_fwd_ctas() {
  return kThr != 256 ? 1 : sizeof(T) == 2 && !NormIo<T, V>::kStaged ? 3 : 2;
}
// kThr: the CTA's threads, 256, 512 (rows past 4096) or 1024 (past 8192, where 64
// registers a thread make both kernels spill, 28 to 872 bytes: such rows are rare). Below
// that, 16-bit rows of whole words do not spill; the backward of aligned float32 rows
// spills 56 bytes of its 128 registers' worth, that of unaligned rows up to 296, and the
// forward of rows that move value by value 40 to 64.
template <typename T, int V, int kThr>
__global__ void __launch_bounds__(kThr, (norm_fwd_ctas<T, V, kThr>())) layer_norm_fwd_kernel(NormArgs a) {
  using Io = NormIo<T, V>;
  constexpr int P = Io::kPairs;
  extern __shared__ __align__(16) char smem[];
  __shared__ float2 red[2][32];
  const int lane = threadIdx.x & (a.span - 1), teams = blockDim.x / a.span, team = threadIdx.x / a.span;
  T* buf = reinterpret_cast<T*>(smem) + team * a.span * kNormValues;
  const int64_t first = (int64_t)blockIdx.x * teams, step = (int64_t)gridDim.x * teams;
  const float inv = 1.f / a.C;
  typename Io::Row row;
  row.load(static_cast<const T*>(a.x) + (first + team) * a.x_s, lane, a.span, a.C, first + team < a.rows);
  f2 w[P], b[P];
  Io::param(a.w, lane, a.span, a.C, 1.f, w);
  Io::param(a.b, lane, a.span, a.C, 0.f, b);
  for (int64_t r0 = first; r0 < a.rows; r0 += step) {
    const int64_t r = r0 + team;
    if constexpr (Io::kStaged) {
      Io::spread(row, buf, lane, a.span);
      Io::sync(a.span);
      Io::gather(row, buf, lane, a.span);
    }
    f2 f[P], s{0.f, 0.f};
    Io::get(row, f);
    row.load(static_cast<const T*>(a.x) + (r + step) * a.x_s, lane, a.span, a.C, r + step < a.rows);
#pragma unroll
    for (int i = 0; i < P; ++i) s = add2(s, f[i]);
    const float mu = norm_sums<false>(s.x + s.y, 0.f, a.span, red, 0).x * inv;
    s = f2{0.f, 0.f};
#pragma unroll
    for (int i = 0; i < P; ++i) {
      f[i] = sub2(f[i], splat(mu));
      if constexpr (Io::kStaged) {  // the values past C are zeros less the mean
        if (!Io::inside(i, 0, lane, a.span, a.C)) f[i].x = 0.f;
        if (!Io::inside(i, 1, lane, a.span, a.C)) f[i].y = 0.f;
      } else {
        if (!Io::inside(i, 0, lane, a.span, a.C)) f[i] = f2{0.f, 0.f};
      }
      s = fma2(f[i], f[i], s);
    }
    const float rs = rsqrtf(norm_sums<false>(s.x + s.y, 0.f, a.span, red, 1).x * inv + a.eps);
#pragma unroll
    for (int i = 0; i < P; ++i) f[i] = fma2(mul2(f[i], splat(rs)), w[i], b[i]);
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
  constexpr int P = Io::kPairs, G = Io::kGran;
  extern __shared__ __align__(16) char smem[];  // [2][C] sums where a CTA has several teams, then staged rows
  __shared__ float2 red[2][32];
  const int lane = threadIdx.x & (a.span - 1), teams = blockDim.x / a.span, team = threadIdx.x / a.span;
  float* acc = reinterpret_cast<float*>(smem);
  T* bx = reinterpret_cast<T*>(smem + (teams > 1 ? (2 * a.C * sizeof(float) + 15) / 16 * 16 : 0)) +
          team * 2 * a.span * kNormValues;
  T* bg = bx + a.span * kNormValues;
  const int64_t first = (int64_t)blockIdx.x * teams, step = (int64_t)gridDim.x * teams;
  const float inv = 1.f / a.C;
  f2 gw[P], gb[P], w[P];
#pragma unroll
  for (int i = 0; i < P; ++i) gw[i] = gb[i] = f2{0.f, 0.f};
  Io::param(a.w, lane, a.span, a.C, 1.f, w);
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
  int slot = 0;
  for (int64_t r0 = first; r0 < a.rows; r0 += step, slot ^= 1) {
    const int64_t r = r0 + team;
    f2 h[P], g[P];
    if constexpr (Io::kStaged) {
      Io::spread(nx, bx, lane, a.span);
      Io::spread(ng, bg, lane, a.span);
      Io::sync(a.span);
      Io::gather(nx, bx, lane, a.span);
      Io::gather(ng, bg, lane, a.span);
    }
    Io::get(nx, h);
    Io::get(ng, g);
    const f2 mu = splat(nmu), rs = splat(nrs);
    fetch(r + step);
    f2 s1{0.f, 0.f}, s2{0.f, 0.f};
#pragma unroll
    for (int i = 0; i < P; ++i) {  // past C w and gy are zeros
      h[i] = mul2(sub2(h[i], mu), rs);
      gw[i] = fma2(g[i], h[i], gw[i]);
      gb[i] = add2(gb[i], g[i]);
      g[i] = mul2(g[i], w[i]);
      s1 = add2(s1, g[i]);
      s2 = fma2(g[i], h[i], s2);
    }
    const float2 m = norm_sums<true>(s1.x + s1.y, s2.x + s2.y, a.span, red, slot);
    const f2 m1 = splat(m.x * inv), m2 = splat(-m.y * inv);
#pragma unroll
    for (int i = 0; i < P; ++i) g[i] = mul2(fma2(h[i], m2, sub2(g[i], m1)), rs);
    if constexpr (Io::kStaged) Io::sync(a.span);  // every lane has gathered from bx
    Io::store(static_cast<T*>(a.y) + r * a.C, bx, lane, a.span, a.C, r < a.rows, g);
    if constexpr (Io::kStaged) Io::sync(a.span);
  }
  float* part = a.partial + (int64_t)blockIdx.x * 2 * a.C;
  float* to = teams > 1 ? acc : part;
  for (int k = 0; k < teams; ++k) {
    if (team == k) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = (i * 2 / G * a.span + lane) * G + i * 2 % G;
        const float vw[2] = {gw[i].x, gw[i].y}, vb[2] = {gb[i].x, gb[i].y};
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (c + e < a.C) {
            to[c + e] = (k ? to[c + e] : 0.f) + vw[e];
            to[a.C + c + e] = (k ? to[a.C + c + e] : 0.f) + vb[e];
          }
      }
    }
    if (teams > 1) __syncthreads();
  }
  if (teams > 1)
    for (int c = threadIdx.x; c < 2 * a.C; c += blockDim.x) part[c] = acc[c];
}

}  // namespace wkv
