// Selective state-space scan, forward, backward and single-token step (sm_100a).
//
// Per sequence b, channel c and state n (N <= 64), with d = softplus(dt + bias):
//   h_t = a_t h_{t-1} + d_t B_t[n] x_t,  a_t = exp(d_t A[c][n])
//   y_t = sum_n C_t[n] h_t + D[c] x_t,   out_t = y_t silu(z_t)
// Gradient, with gy = gout silu(z), g_t = dL/dh_t and p_t = a_t h_{t-1}:
//   g_t = C_t gy_t + a_{t+1} g_{t+1}
//   gC_t[n] = sum_c gy_t h_t,            gB_t[n] = sum_c g_t d_t x_t
//   gx_t = d_t sum_n g_t B_t + D gy_t,   gd_t = x_t sum_n g_t B_t + sum_n A g_t p_t
//   gA = sum g_t d_t p_t,  gD = sum gy_t x_t,  gz_t = gout_t y_t silu'(z_t)
//   gdt = gd softplus'(dt + bias)
// The state and every sum are float32. A row t >= length leaves the state as it
// is (d = 0), gives out = 0 and reads nothing.
#pragma once

#include "row_io.cuh"

namespace wkv {

constexpr int kScanMaxN = 64;
constexpr int kScanCkpt = 8;       // steps between the states the forward keeps for the backward
constexpr int kScanThreads = 128;  // threads of a CTA
constexpr int kScanRows = 32;      // steps of a staged tile, at most: segments are multiples of it

struct ScanArgs {
  const void *x, *dt, *Bm, *Cm, *z, *gout;
  const float *A, *D, *bias;  // [C][N], [C] or null, [C] or null
  const float* h0;            // [B][C][N] or null
  const int* lengths;         // [B] or null
  void* out;                  // [B][T][C]
  float* h_last;              // [B][C][N] or null
  float* ckpt;                // [B][ceil(T / kScanCkpt)][C][N] or null: the state before each group of steps
  // segments of the time axis (nseg > 1): what a segment adds to a zero state, and its sum of d
  float* seg_h;  // [B][nseg][C][N]
  float* seg_d;  // [B][nseg][C]
  // backward
  const float* gh_last;  // [B][C][N] or null
  void *gx, *gdt, *gz;   // [B][T][C]
  float* gh0;            // [B][C][N] or null
  float* part_bc;        // [slices][B][T][2][N]
  float* part_a;         // [B * nseg][C][N]
  float* part_d;         // [B * nseg][2][C]: gD, gbias
  int64_t x_sb, x_st, dt_sb, dt_st, z_sb, z_st, b_sb, b_st, c_sb, c_st, g_sb, g_st;
  int B, T, C, N;
  int nseg, seg_len, cblocks;
  int groups;   // backward: channel groups of a CTA
  int wide;     // rows of x, dt, z, gout move as aligned 16-byte words
  int wide_bc;  // four adjacent states of B and C move as one aligned word
  int wide_n;   // four adjacent float32 states move as one aligned word (N % 4 == 0)
  int softplus;
};

// softplus and its slope; log1p keeps the small values' relative accuracy.
__device__ __forceinline__ float scan_delta(float v, int softplus) {
  return softplus ? fmaxf(v, 0.f) + log1pf(expf(-fabsf(v))) : v;
}
__device__ __forceinline__ float scan_delta_slope(float v, int softplus) { return softplus ? sigmoid1(v) : 1.f; }

__device__ __forceinline__ int scan_length(const ScanArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
}

// Sums v[0 .. NV) over L lanes (a power of two; lane bits kStride * 1, 2, ...),
// scattered: the lane of index l among the L keeps the sums of v[l * NV / L ..] in
// v[0 .. NV / L) (NV >= L), or of v[l / (L / NV)] in v[0] (NV < L). Each halving
// exchanges half of the values, so NV sums cost about NV shuffles, not NV log2 L.
template <int NV, int L, int kStride>
__device__ __forceinline__ void reduce_scatter(float* v) {
  if constexpr (L > 1) {
    constexpr int mask = kStride * (L / 2);
    if constexpr (NV > 1) {
      const bool upper = (threadIdx.x & mask) != 0;
#pragma unroll
      for (int i = 0; i < NV / 2; ++i) {
        const float send = upper ? v[i] : v[i + NV / 2], keep = upper ? v[i + NV / 2] : v[i];
        v[i] = keep + __shfl_xor_sync(kFull, send, mask);
      }
      reduce_scatter<NV / 2, L / 2, kStride>(v);
    } else {
      v[0] += __shfl_xor_sync(kFull, v[0], mask);
      reduce_scatter<1, L / 2, kStride>(v);
    }
  }
}

// Four adjacent states of one channel, as two packed pairs.
struct Quad {
  f2 lo, hi;
};
__device__ __forceinline__ Quad quad(float4 v) { return Quad{f2{v.x, v.y}, f2{v.z, v.w}}; }
__device__ __forceinline__ float4 quad4(Quad q) { return make_float4(q.lo.x, q.lo.y, q.hi.x, q.hi.y); }
__device__ __forceinline__ Quad load_quad(const float* p, int n, int N, int wide) {
  if (n >= N) return Quad{f2{0.f, 0.f}, f2{0.f, 0.f}};
  if (wide) return quad(*reinterpret_cast<const float4*>(p + n));
  return Quad{f2{p[n], n + 1 < N ? p[n + 1] : 0.f}, f2{n + 2 < N ? p[n + 2] : 0.f, n + 3 < N ? p[n + 3] : 0.f}};
}
__device__ __forceinline__ void store_quad(float* p, int n, int N, int wide, Quad q) {
  if (n >= N) return;
  if (wide) {
    *reinterpret_cast<float4*>(p + n) = quad4(q);
    return;
  }
  p[n] = q.lo.x;
  if (n + 1 < N) p[n + 1] = q.lo.y;
  if (n + 2 < N) p[n + 2] = q.hi.x;
  if (n + 3 < N) p[n + 3] = q.hi.y;
}
// exp(d A) of four states: A2 is A log2(e).
__device__ __forceinline__ Quad decay(Quad A2, f2 d) { return Quad{ex2x2(mul2(A2.lo, d)), ex2x2(mul2(A2.hi, d))}; }

// Eight adjacent channels of one row; `live` false or channels past C: zeros.
template <typename T>
struct Eight {
  alignas(16) T e[8];
  __device__ __forceinline__ void load(const T* row, int c, int C, bool live, int wide) {
    uint4* w = reinterpret_cast<uint4*>(e);
    if (wide) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        w[i] = live && c < C ? reinterpret_cast<const uint4*>(row + c)[i] : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = live && c + i < C ? row[c + i] : Pair<T>::from_float(0.f);
    }
  }
  __device__ __forceinline__ void store(T* row, int c, int C, int wide) const {
    if (wide) {
      const uint4* w = reinterpret_cast<const uint4*>(e);
      if (c < C)
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(row + c)[i] = w[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < C) row[c + i] = e[i];
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = Pair<T>::scalar(e[i]);
  }
};

// Four adjacent states of a row of B or C; past N: zeros.
template <typename T>
__device__ __forceinline__ Vec<T, 4> load_bc(const T* row, int n, int N, bool live, int wide) {
  Vec<T, 4> r = Vec<T, 4>::zero();
  if (!live || n >= N) return r;
  if (wide) return Vec<T, 4>::load(row + n);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < N) r.e[i] = row[n + i];
  return r;
}

// The layout of a CTA's work, by the lanes that share a channel (four states each).
template <int LPC>
struct ScanShape {
  static constexpr int NP = 4 * LPC;               // states, padded
  static constexpr int CH = kScanThreads / LPC;    // channels of a CTA (of a group in the backward)
  static constexpr int TT = LPC < 4 ? 8 * LPC : kScanRows;  // steps of a staged tile: TT * CH <= 1024
  static constexpr int VPR = CH / 8;               // eights of a row
};

// The state a segment starts from: the earlier segments' contributions in order
// (forward), or the adjoint that the later segments hand back.
__device__ __forceinline__ Quad scan_carry(const ScanArgs& a, int b, int c, int n, Quad h, Quad A2, int from, int to,
                                           int step) {
  for (int s = from; s != to; s += step) {
    const int64_t at = ((int64_t)b * a.nseg + s) * a.C + c;
    const Quad add = load_quad(a.seg_h + at * a.N, n, a.N, a.wide_n);
    const Quad e = decay(A2, splat(a.seg_d[at]));
    h.lo = fma2(e.lo, h.lo, add.lo);
    h.hi = fma2(e.hi, h.hi, add.hi);
  }
  return h;
}

// What a segment adds to a zero state (kAdjoint: to a zero adjoint, walking back:
// g <- a (g + C gy)), and its sum of d: the decay across it is exp(A sum d).
template <typename T, int LPC, bool kAdjoint>
__global__ void __launch_bounds__(kScanThreads) scan_summary_kernel(ScanArgs a) {
  using S = ScanShape<LPC>;
  __shared__ float2 sdx[S::TT][S::CH];
  __shared__ __align__(16) float sn[S::TT][S::NP];
  // the last segment's sum serves no later one (the first's, walking back)
  const int cb = blockIdx.x % a.cblocks, seg = blockIdx.x / a.cblocks % (a.nseg - 1) + (kAdjoint ? 1 : 0);
  const int b = blockIdx.x / a.cblocks / (a.nseg - 1);
  const int q = threadIdx.x % LPC, ch = threadIdx.x / LPC, c = cb * S::CH + ch;
  const int t_begin = seg * a.seg_len, t_end = min(t_begin + a.seg_len, scan_length(a, b));
  Quad A2 = load_quad(a.A + (int64_t)min(c, a.C - 1) * a.N, 4 * q, a.N, a.wide_n);
  A2.lo = mul2(A2.lo, splat(kL2E));
  A2.hi = mul2(A2.hi, splat(kL2E));
  Quad h{f2{0.f, 0.f}, f2{0.f, 0.f}};
  float dsum = 0.f;
  const int row = threadIdx.x / S::VPR, vc = threadIdx.x % S::VPR * 8;
  const int tiles = t_end > t_begin ? (t_end - t_begin + S::TT - 1) / S::TT : 0;
  float bias[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) bias[i] = a.bias && cb * S::CH + vc + i < a.C ? a.bias[cb * S::CH + vc + i] : 0.f;
  for (int k = 0; k < tiles; ++k) {
    const int t0 = t_begin + (kAdjoint ? tiles - 1 - k : k) * S::TT;
    if (row < S::TT) {
      const int t = t0 + row;
      const bool live = t < t_end;
      Eight<T> r;
      float f[8], d[8], w[8];
      r.load(static_cast<const T*>(a.dt) + b * a.dt_sb + (int64_t)t * a.dt_st + cb * S::CH, vc, a.C - cb * S::CH, live,
             a.wide);
      r.get(f);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = live ? scan_delta(f[i] + bias[i], a.softplus) : 0.f;
      if constexpr (kAdjoint) {
        r.load(static_cast<const T*>(a.gout) + b * a.g_sb + (int64_t)t * a.g_st + cb * S::CH, vc, a.C - cb * S::CH,
               live, a.wide);
        r.get(w);
        if (a.z) {
          r.load(static_cast<const T*>(a.z) + b * a.z_sb + (int64_t)t * a.z_st + cb * S::CH, vc, a.C - cb * S::CH, live,
                 a.wide);
          r.get(f);
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] *= f[i] * sigmoid1(f[i]);
        }
      } else {
        r.load(static_cast<const T*>(a.x) + b * a.x_sb + (int64_t)t * a.x_st + cb * S::CH, vc, a.C - cb * S::CH, live,
               a.wide);
        r.get(f);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = d[i] * f[i];
      }
#pragma unroll
      for (int i = 0; i < 8; i += 2)
        *reinterpret_cast<float4*>(&sdx[row][vc + i]) = make_float4(d[i], w[i], d[i + 1], w[i + 1]);
    }
    for (int i = threadIdx.x; i < S::TT * LPC; i += kScanThreads) {
      const int t = t0 + i / LPC, n = i % LPC * 4;
      const T* p = kAdjoint ? static_cast<const T*>(a.Cm) + b * a.c_sb + (int64_t)t * a.c_st
                            : static_cast<const T*>(a.Bm) + b * a.b_sb + (int64_t)t * a.b_st;
      float f[4];
      load_bc(p, n, a.N, t < t_end, a.wide_bc).get(f);
      *reinterpret_cast<float4*>(&sn[i / LPC][n]) = make_float4(f[0], f[1], f[2], f[3]);
    }
    __syncthreads();
#pragma unroll 8
    for (int j = 0; j < S::TT; ++j) {
      const int i = kAdjoint ? S::TT - 1 - j : j;
      const float2 s = sdx[i][ch];
      const Quad v = quad(*reinterpret_cast<const float4*>(&sn[i][4 * q]));
      const Quad e = decay(A2, splat(s.x));
      if constexpr (kAdjoint) {
        h.lo = mul2(e.lo, fma2(v.lo, splat(s.y), h.lo));
        h.hi = mul2(e.hi, fma2(v.hi, splat(s.y), h.hi));
      } else {
        h.lo = fma2(e.lo, h.lo, mul2(v.lo, splat(s.y)));
        h.hi = fma2(e.hi, h.hi, mul2(v.hi, splat(s.y)));
      }
      dsum += s.x;
    }
    __syncthreads();
  }
  if (c >= a.C) return;
  const int64_t at = ((int64_t)b * a.nseg + seg) * a.C + c;
  store_quad(a.seg_h + at * a.N, 4 * q, a.N, a.wide_n, h);
  if (q == 0) a.seg_d[at] = dsum;
}

// A CTA walks one segment of CH channels of one sequence; LPC lanes share a
// channel, four states each. Tiles of TT steps are staged: d and d x of every
// (step, channel) and B, C in float32, while the next tile's raw rows are already
// under way to registers. The lanes' parts of y are summed by an exchange of four
// steps at a time, and the gate and the output are done by whole rows again.
template <typename T, int LPC>
__global__ void __launch_bounds__(kScanThreads) scan_fwd_kernel(ScanArgs a) {
  using S = ScanShape<LPC>;
  __shared__ float2 sdx[S::TT][S::CH];
  __shared__ __align__(16) float sbc[S::TT][2 * S::NP];
  __shared__ __align__(16) float sy[S::TT][S::CH + 8];
  const int cb = blockIdx.x % a.cblocks, seg = blockIdx.x / a.cblocks % a.nseg, b = blockIdx.x / a.cblocks / a.nseg;
  const int q = threadIdx.x % LPC, ch = threadIdx.x / LPC, c0 = cb * S::CH, c = c0 + ch;
  const int len = scan_length(a, b);
  const int t_begin = seg * a.seg_len, t_end = min(t_begin + a.seg_len, a.T), t_live = min(t_end, len);
  const int64_t hc = ((int64_t)b * a.C + c) * a.N;
  const bool mine = c < a.C;
  Quad A2 = load_quad(a.A + (int64_t)min(c, a.C - 1) * a.N, 4 * q, a.N, a.wide_n);
  A2.lo = mul2(A2.lo, splat(kL2E));
  A2.hi = mul2(A2.hi, splat(kL2E));
  Quad h{f2{0.f, 0.f}, f2{0.f, 0.f}};
  if (mine && a.h0) h = load_quad(a.h0 + hc, 4 * q, a.N, a.wide_n);
  if (mine) h = scan_carry(a, b, c, 4 * q, h, A2, 0, seg, 1);

  const int row = threadIdx.x / S::VPR, vc = threadIdx.x % S::VPR * 8;
  const bool stager = row < S::TT;
  constexpr int kBC = (S::TT * 2 * LPC + kScanThreads - 1) / kScanThreads;
  Eight<T> rx, rd, rz;
  Vec<T, 4> rbc[kBC];
  auto fetch = [&](int t0) {
    const int t = t0 + row;
    const bool live = stager && t < t_live;
    rx.load(static_cast<const T*>(a.x) + b * a.x_sb + (int64_t)t * a.x_st + c0, vc, a.C - c0, live, a.wide);
    rd.load(static_cast<const T*>(a.dt) + b * a.dt_sb + (int64_t)t * a.dt_st + c0, vc, a.C - c0, live, a.wide);
    if (a.z)
      rz.load(static_cast<const T*>(a.z) + b * a.z_sb + (int64_t)t * a.z_st + c0, vc, a.C - c0, live, a.wide);
#pragma unroll
    for (int k = 0; k < kBC; ++k) {
      const int i = k * kScanThreads + threadIdx.x, tb = t0 + i / (2 * LPC), n = i % LPC * 4;
      const bool on = i < S::TT * 2 * LPC && tb < t_live;
      const T* p = i % (2 * LPC) < LPC ? static_cast<const T*>(a.Bm) + b * a.b_sb + (int64_t)tb * a.b_st
                                       : static_cast<const T*>(a.Cm) + b * a.c_sb + (int64_t)tb * a.c_st;
      rbc[k] = load_bc(p, n, a.N, on, a.wide_bc);
    }
  };
  const int nck = (a.T + kScanCkpt - 1) / kScanCkpt;
  if (t_begin < t_live) fetch(t_begin);
  for (int t0 = t_begin; t0 < t_live; t0 += S::TT) {
    const Eight<T> cx = rx, cz = rz;
    if (stager) {
      float f[8], d[8];
      rd.get(d);
      rx.get(f);
      const bool live = t0 + row < t_live;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        d[i] = live ? scan_delta(d[i] + (a.bias && c0 + vc + i < a.C ? a.bias[c0 + vc + i] : 0.f), a.softplus) : 0.f;
#pragma unroll
      for (int i = 0; i < 8; i += 2)
        *reinterpret_cast<float4*>(&sdx[row][vc + i]) = make_float4(d[i], d[i] * f[i], d[i + 1], d[i + 1] * f[i + 1]);
    }
#pragma unroll
    for (int k = 0; k < kBC; ++k) {
      const int i = k * kScanThreads + threadIdx.x;
      float f[4];
      rbc[k].get(f);
      if (i < S::TT * 2 * LPC)
        *reinterpret_cast<float4*>(&sbc[i / (2 * LPC)][i % (2 * LPC) * 4]) = make_float4(f[0], f[1], f[2], f[3]);
    }
    __syncthreads();
    if (t0 + S::TT < t_live) fetch(t0 + S::TT);
#pragma unroll 2
    for (int j = 0; j < S::TT; j += 4) {
      if (j % kScanCkpt == 0 && a.ckpt && mine && t0 + j < t_live)
        store_quad(a.ckpt + (((int64_t)b * nck + (t0 + j) / kScanCkpt) * a.C + c) * a.N, 4 * q, a.N, a.wide_n, h);
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 s = sdx[j + i][ch];
        const Quad Bt = quad(*reinterpret_cast<const float4*>(&sbc[j + i][4 * q]));
        const Quad Ct = quad(*reinterpret_cast<const float4*>(&sbc[j + i][S::NP + 4 * q]));
        const Quad e = decay(A2, splat(s.x));
        h.lo = fma2(e.lo, h.lo, mul2(Bt.lo, splat(s.y)));
        h.hi = fma2(e.hi, h.hi, mul2(Bt.hi, splat(s.y)));
        const f2 p = fma2(h.hi, Ct.hi, mul2(h.lo, Ct.lo));
        y[i] = p.x + p.y;
      }
      reduce_scatter<4, LPC, 1>(y);
      if constexpr (LPC <= 4) {
#pragma unroll
        for (int i = 0; i < 4 / LPC; ++i) sy[j + q * (4 / LPC) + i][ch] = y[i];
      } else {
        if (q % (LPC / 4) == 0) sy[j + q / (LPC / 4)][ch] = y[0];
      }
    }
    __syncthreads();
    if (stager && t0 + row < t_live) {
      float f[8], y[8], z[8];
      cx.get(f);
      cz.get(z);
      Eight<T> o;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = fmaf(a.D && c0 + vc + i < a.C ? a.D[c0 + vc + i] : 0.f, f[i], sy[row][vc + i]);
        if (a.z) y[i] *= z[i] * sigmoid1(z[i]);
        o.e[i] = Pair<T>::from_float(y[i]);
      }
      o.store(static_cast<T*>(a.out) + ((int64_t)b * a.T + t0 + row) * a.C + c0, vc, a.C - c0, a.wide);
    }
  }
  // the rows past the sequence's length
  for (int i = threadIdx.x; i < (t_end - max(t_begin, t_live)) * S::CH; i += kScanThreads) {
    const int t = max(t_begin, t_live) + i / S::CH, k = c0 + i % S::CH;
    if (k < a.C) static_cast<T*>(a.out)[((int64_t)b * a.T + t) * a.C + k] = Pair<T>::from_float(0.f);
  }
  if (a.h_last && mine && seg == a.nseg - 1) store_quad(a.h_last + hc, 4 * q, a.N, a.wide_n, h);
}

__device__ __forceinline__ void copy16(void* dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0)
               : "memory");
}

// Shared memory of the backward kernel (see there), in bytes from the start.
template <typename T, int LPC>
struct ScanBwdSmem {
  using S = ScanShape<LPC>;
  static constexpr int M = LPC < 4 ? LPC : 4;     // groups x sub-chunks of a tile
  static constexpr int kCells = 8 * M * S::CH;    // (step, channel) pairs of a tile, <= 1024
  static constexpr int kRaw = kCells * 16;                        // after the slots, float4 [kCells]: T [2][4][kCells]
  static constexpr int kBC = kRaw + 8 * kCells * (int)sizeof(T);  // float [8 subs][2 NP]
  static constexpr int kSub = 8 * 2 * S::NP * 4 * 5;              // bytes a sub-chunk: its B, C, and a partial row a warp
  // float [subs][4 warps][8][2 NP], then float4 [3][groups][threads]: A log2 e, adjoint, gA
  static constexpr int bytes(int groups) { return kBC + M / groups * kSub + 3 * groups * kScanThreads * 16; }
};

// A CTA walks one segment of `groups` x CH channels of one sequence backwards, in
// tiles of 8 * (M / groups) steps. Per sub-chunk of 8 steps and group of CH
// channels, a thread runs its channel's four states forward from the kept state,
// with a_t and p_t = a_t h_{t-1} in registers, and then back with the adjoint. The
// sums over states (for gx, gdt, gz) are exchanged among the channel's lanes; the
// sums over channels (gB, gC) gather in registers over the groups, are exchanged
// once for all of them, then added over the warps and left as one partial row of
// the CTA's channels.
template <typename T, int LPC>
__global__ void __launch_bounds__(kScanThreads, LPC <= 4 ? 3 : 2) scan_bwd_kernel(ScanArgs a) {
  using S = ScanShape<LPC>;
  using L = ScanBwdSmem<T, LPC>;
  extern __shared__ __align__(16) char smem[];
  constexpr int NP = S::NP, CH = S::CH, M = L::M, kCells = L::kCells;
  const int G = a.groups, subs = M / G, TS = 8 * subs, CHB = CH * G;
  float4* slot = reinterpret_cast<float4*>(smem);
  T* raw = reinterpret_cast<T*>(smem + L::kRaw);
  float* sbc = reinterpret_cast<float*>(smem + L::kBC);
  float* part = sbc + TS * 2 * NP;
  float4* sgrp = reinterpret_cast<float4*>(part + subs * 4 * 8 * 2 * NP);
  const int tid = threadIdx.x, q = tid % LPC, ch = tid / LPC, warp = tid / 32;
  const int cb = blockIdx.x % a.cblocks, seg = blockIdx.x / a.cblocks % a.nseg, b = blockIdx.x / a.cblocks / a.nseg;
  const int c0 = cb * CHB;
  const int len = scan_length(a, b);
  const int t_begin = seg * a.seg_len, t_end = min(t_begin + a.seg_len, a.T), t_live = min(t_end, len);
  const int nck = (a.T + kScanCkpt - 1) / kScanCkpt;

  for (int k = 0; k < G; ++k) {
    const int c = c0 + k * CH + ch;
    Quad A2{f2{0.f, 0.f}, f2{0.f, 0.f}}, g = A2;
    sgrp[(2 * G + k) * kScanThreads + tid] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < a.C) {
      A2 = load_quad(a.A + (int64_t)c * a.N, 4 * q, a.N, a.wide_n);
      A2.lo = mul2(A2.lo, splat(kL2E));
      A2.hi = mul2(A2.hi, splat(kL2E));
      if (a.gh_last) g = load_quad(a.gh_last + ((int64_t)b * a.C + c) * a.N, 4 * q, a.N, a.wide_n);
      g = scan_carry(a, b, c, 4 * q, g, A2, a.nseg - 1, seg, -1);
    }
    sgrp[k * kScanThreads + tid] = quad4(A2);
    sgrp[(G + k) * kScanThreads + tid] = quad4(g);
  }

  // rows past the length: zero gradients
  for (int i = tid; i < (t_end - max(t_begin, t_live)) * CHB; i += kScanThreads) {
    const int t = max(t_begin, t_live) + i / CHB, c = c0 + i % CHB;
    if (c < a.C) {
      const int64_t at = ((int64_t)b * a.T + t) * a.C + c;
      static_cast<T*>(a.gx)[at] = Pair<T>::from_float(0.f);
      static_cast<T*>(a.gdt)[at] = Pair<T>::from_float(0.f);
      if (a.gz) static_cast<T*>(a.gz)[at] = Pair<T>::from_float(0.f);
    }
  }
  float* pbc = a.part_bc + ((int64_t)cb * a.B + b) * a.T * 2 * a.N;
  for (int i = tid; i < (t_end - max(t_begin, t_live)) * 2 * a.N; i += kScanThreads)
    pbc[(int64_t)max(t_begin, t_live) * 2 * a.N + i] = 0.f;

  // a thread's cells in the staging and in the row-wise end: two adjacent channels
  // (always the same ones) of every row_step-th row
  const int pairs = CHB / 2, cp = tid % pairs * 2, row0 = tid / pairs, row_step = kScanThreads / pairs;
  float Dp[2], bp[2], gD[2] = {0.f, 0.f}, gb[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = c0 + cp + i;
    Dp[i] = a.D && c < a.C ? a.D[c] : 0.f;
    bp[i] = a.bias && c < a.C ? a.bias[c] : 0.f;
  }
  const T* src[4] = {static_cast<const T*>(a.x) + b * a.x_sb, static_cast<const T*>(a.dt) + b * a.dt_sb,
                     static_cast<const T*>(a.gout) + b * a.g_sb,
                     a.z ? static_cast<const T*>(a.z) + b * a.z_sb : nullptr};
  const int64_t pitch[4] = {a.x_st, a.dt_st, a.g_st, a.z_st};
  auto fetch = [&](int t0, int stage) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k == 3 && !a.z) break;
      T* dst = raw + (stage * 4 + k) * kCells;
      if (a.wide) {
        constexpr int E = 16 / (int)sizeof(T);
        for (int i = tid * E; i < kCells; i += kScanThreads * E) {
          const int t = t0 + i / CHB, c = c0 + i % CHB;
          const bool on = t < t_live && c < a.C;
          copy16(dst + i, on ? src[k] + t * pitch[k] + c : src[k], on);
        }
      } else {
        for (int i = tid; i < kCells; i += kScanThreads) {
          const int t = t0 + i / CHB, c = c0 + i % CHB;
          dst[i] = t < t_live && c < a.C ? src[k][t * pitch[k] + c] : Pair<T>::from_float(0.f);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  constexpr int kBC = (8 * M * 2 * LPC + kScanThreads - 1) / kScanThreads;
  Vec<T, 4> rbc[kBC];
  auto fetch_bc = [&](int t0) {
#pragma unroll
    for (int k = 0; k < kBC; ++k) {
      const int i = k * kScanThreads + tid, t = t0 + i / (2 * LPC), n = i % LPC * 4;
      const bool on = i < TS * 2 * LPC && t < t_live;
      const T* p = i % (2 * LPC) < LPC ? static_cast<const T*>(a.Bm) + b * a.b_sb + (int64_t)t * a.b_st
                                       : static_cast<const T*>(a.Cm) + b * a.c_sb + (int64_t)t * a.c_st;
      rbc[k] = load_bc(p, n, a.N, on, a.wide_bc);
    }
  };
  auto kept = [&](int t, int k) {  // the state before step t (a multiple of 8) of group k
    const int c = c0 + k * CH + ch;
    if (c >= a.C || t >= t_live || t < t_begin) return Quad{f2{0.f, 0.f}, f2{0.f, 0.f}};
    return load_quad(a.ckpt + (((int64_t)b * nck + t / kScanCkpt) * a.C + c) * a.N, 4 * q, a.N, a.wide_n);
  };

  const int tiles = t_live > t_begin ? (t_live - t_begin + TS - 1) / TS : 0;
  if (tiles > 0) {
    fetch(t_begin + (tiles - 1) * TS, 0);
    fetch_bc(t_begin + (tiles - 1) * TS);
  }
  Quad next = kept(t_begin + (tiles - 1) * TS + (subs - 1) * 8, 0);
  int stage = 0;
  for (int tile = tiles - 1; tile >= 0; --tile, stage ^= 1) {
    const int t0 = t_begin + tile * TS;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    const T* cur = raw + stage * 4 * kCells;
    for (int r = row0; r < TS; r += row_step) {
      const int at = r * CHB + cp;
      const bool live = t0 + r < t_live;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float x = Pair<T>::scalar(cur[at + i]);
        const float d = live ? scan_delta(Pair<T>::scalar(cur[kCells + at + i]) + bp[i], a.softplus) : 0.f;
        float gy = Pair<T>::scalar(cur[2 * kCells + at + i]);
        if (a.z) {
          const float z = Pair<T>::scalar(cur[3 * kCells + at + i]);
          gy *= z * sigmoid1(z);
        }
        slot[at + i] = make_float4(d, d * x, gy, 0.f);
      }
    }
#pragma unroll
    for (int k = 0; k < kBC; ++k) {
      const int i = k * kScanThreads + tid;
      float f[4];
      rbc[k].get(f);
      if (i < TS * 2 * LPC)
        *reinterpret_cast<float4*>(sbc + i / (2 * LPC) * 2 * NP + i % (2 * LPC) * 4) =
            make_float4(f[0], f[1], f[2], f[3]);
    }
    __syncthreads();
    if (tile > 0) {
      fetch(t0 - TS, stage ^ 1);
      fetch_bc(t0 - TS);
    }
    for (int sub = subs - 1; sub >= 0; --sub) {
      f2 accB[8][2], accC[8][2];
#pragma unroll
      for (int i = 0; i < 8; ++i) accB[i][0] = accB[i][1] = accC[i][0] = accC[i][1] = f2{0.f, 0.f};
      const float* bc = sbc + sub * 8 * 2 * NP + 4 * q;
      for (int k = 0; k < G; ++k) {
        float4* sl = slot + sub * 8 * CHB + k * CH + ch;
        const Quad A2 = quad(sgrp[k * kScanThreads + tid]);
        Quad h = next;
        {  // the state that the next group or sub-chunk starts from
          const int nk = k + 1 < G ? k + 1 : 0;
          next = kept(t0 + (nk ? sub : sub - 1) * 8, nk);
        }
        Quad e[8], p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 s = *reinterpret_cast<const float2*>(sl + i * CHB);
          const Quad Bt = quad(*reinterpret_cast<const float4*>(bc + i * 2 * NP));
          e[i] = decay(A2, splat(s.x));
          p[i] = Quad{mul2(e[i].lo, h.lo), mul2(e[i].hi, h.hi)};
          h.lo = fma2(Bt.lo, splat(s.y), p[i].lo);
          h.hi = fma2(Bt.hi, splat(s.y), p[i].hi);
        }
        Quad g = quad(sgrp[(G + k) * kScanThreads + tid]);
        Quad gA{f2{0.f, 0.f}, f2{0.f, 0.f}};
#pragma unroll
        for (int half = 1; half >= 0; --half) {
          float along[4], gd[4], y[4];
#pragma unroll
          for (int ii = 3; ii >= 0; --ii) {
            const int i = half * 4 + ii;
            const float4 s = sl[i * CHB];
            const Quad Bt = quad(*reinterpret_cast<const float4*>(bc + i * 2 * NP));
            const Quad Ct = quad(*reinterpret_cast<const float4*>(bc + i * 2 * NP + NP));
            const Quad hn{fma2(Bt.lo, splat(s.y), p[i].lo), fma2(Bt.hi, splat(s.y), p[i].hi)};
            g.lo = fma2(Ct.lo, splat(s.z), g.lo);
            g.hi = fma2(Ct.hi, splat(s.z), g.hi);
            const f2 al = fma2(g.hi, Bt.hi, mul2(g.lo, Bt.lo));
            const f2 yy = fma2(hn.hi, Ct.hi, mul2(hn.lo, Ct.lo));
            accB[i][0] = fma2(g.lo, splat(s.y), accB[i][0]);
            accB[i][1] = fma2(g.hi, splat(s.y), accB[i][1]);
            accC[i][0] = fma2(hn.lo, splat(s.z), accC[i][0]);
            accC[i][1] = fma2(hn.hi, splat(s.z), accC[i][1]);
            const Quad w{mul2(g.lo, p[i].lo), mul2(g.hi, p[i].hi)};
            const f2 dd = fma2(w.hi, A2.hi, mul2(w.lo, A2.lo));
            gA.lo = fma2(w.lo, splat(s.x), gA.lo);
            gA.hi = fma2(w.hi, splat(s.x), gA.hi);
            g.lo = mul2(g.lo, e[i].lo);
            g.hi = mul2(g.hi, e[i].hi);
            along[ii] = al.x + al.y;
            y[ii] = yy.x + yy.y;
            gd[ii] = dd.x + dd.y;
          }
          reduce_scatter<4, LPC, 1>(along);
          reduce_scatter<4, LPC, 1>(gd);
          reduce_scatter<4, LPC, 1>(y);
          __syncwarp();  // every lane has read the slots that are now reused
          if constexpr (LPC <= 4) {
#pragma unroll
            for (int i = 0; i < 4 / LPC; ++i) {
              float4* to = sl + (half * 4 + q * (4 / LPC) + i) * CHB;
              to->y = along[i];
              to->z = gd[i];
              to->w = y[i];
            }
          } else {
            if (q % (LPC / 4) == 0) {
              float4* to = sl + (half * 4 + q / (LPC / 4)) * CHB;
              to->y = along[0];
              to->z = gd[0];
              to->w = y[0];
            }
          }
        }
        sgrp[(G + k) * kScanThreads + tid] = quad4(g);
        float4& tot = sgrp[(2 * G + k) * kScanThreads + tid];
        tot = make_float4(tot.x + gA.lo.x, tot.y + gA.lo.y, tot.z + gA.hi.x, tot.w + gA.hi.y);
      }
      // the warp's sums over its channels: value v = step * 8 + (0..3: B, 4..7: C)
      constexpr int CL = 32 / LPC;
      float v[64];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i * 8 + 0] = accB[i][0].x, v[i * 8 + 1] = accB[i][0].y, v[i * 8 + 2] = accB[i][1].x;
        v[i * 8 + 3] = accB[i][1].y, v[i * 8 + 4] = accC[i][0].x, v[i * 8 + 5] = accC[i][0].y;
        v[i * 8 + 6] = accC[i][1].x, v[i * 8 + 7] = accC[i][1].y;
      }
      reduce_scatter<64, CL, LPC>(v);
      const int own = tid % 32 / LPC * (64 / CL);
      float* pw = part + (sub * 4 + warp) * 8 * 2 * NP;
#pragma unroll
      for (int i = 0; i < 64 / CL; ++i) {
        const int k = own + i;
        pw[k / 8 * 2 * NP + (k % 8 < 4 ? 0 : NP) + 4 * q + k % 4] = v[i];
      }
    }
    __syncthreads();
    for (int r = row0; r < TS; r += row_step) {
      const int at = r * CHB + cp, t = t0 + r;
      if (t >= t_live) continue;
      float fx[2], fd[2], fz[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 s = slot[at + i];
        const float x = Pair<T>::scalar(cur[at + i]), v = Pair<T>::scalar(cur[kCells + at + i]) + bp[i];
        const float go = Pair<T>::scalar(cur[2 * kCells + at + i]);
        float gy = go;
        fz[i] = 0.f;
        if (a.z) {
          const float z = Pair<T>::scalar(cur[3 * kCells + at + i]), sz = sigmoid1(z);
          gy = go * z * sz;
          fz[i] = go * fmaf(Dp[i], x, s.w) * sz * fmaf(z, 1.f - sz, 1.f);
        }
        fx[i] = fmaf(s.x, s.y, Dp[i] * gy);
        fd[i] = fmaf(x, s.y, s.z * 0.6931471805599453f) * scan_delta_slope(v, a.softplus);
        gD[i] = fmaf(gy, x, gD[i]);
        gb[i] += fd[i];
      }
      const int64_t to = ((int64_t)b * a.T + t) * a.C + c0 + cp;
      if (a.wide) {
        if (c0 + cp < a.C) {
          Vec<T, 2> o;
          o.set(fx);
          o.store(static_cast<T*>(a.gx) + to);
          o.set(fd);
          o.store(static_cast<T*>(a.gdt) + to);
          if (a.gz) {
            o.set(fz);
            o.store(static_cast<T*>(a.gz) + to);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (c0 + cp + i < a.C) {
            static_cast<T*>(a.gx)[to + i] = Pair<T>::from_float(fx[i]);
            static_cast<T*>(a.gdt)[to + i] = Pair<T>::from_float(fd[i]);
            if (a.gz) static_cast<T*>(a.gz)[to + i] = Pair<T>::from_float(fz[i]);
          }
      }
    }
    for (int i = tid; i < TS * 2 * NP; i += kScanThreads) {
      const int r = i / (2 * NP), j = i % (2 * NP), n = j < NP ? j : j - NP;
      if (t0 + r >= t_live || n >= a.N) continue;
      const float* p = part + (r / 8 * 4 * 8 + r % 8) * 2 * NP + j;
      pbc[(int64_t)(t0 + r) * 2 * a.N + (j < NP ? n : a.N + n)] =
          (p[0] + p[8 * 2 * NP]) + (p[2 * 8 * 2 * NP] + p[3 * 8 * 2 * NP]);
    }
  }
  __syncthreads();
  for (int k = 0; k < G; ++k) {
    const int c = c0 + k * CH + ch;
    if (c >= a.C) continue;
    store_quad(a.part_a + (((int64_t)b * a.nseg + seg) * a.C + c) * a.N, 4 * q, a.N, a.wide_n,
               quad(sgrp[(2 * G + k) * kScanThreads + tid]));
    if (a.gh0 && seg == 0)
      store_quad(a.gh0 + ((int64_t)b * a.C + c) * a.N, 4 * q, a.N, a.wide_n, quad(sgrp[(G + k) * kScanThreads + tid]));
  }
  // gD and gbias over the rows of the thread's channels
  float* red = reinterpret_cast<float*>(slot);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    red[(row0 * 2 + 0) * CHB + cp + i] = gD[i];
    red[(row0 * 2 + 1) * CHB + cp + i] = gb[i];
  }
  __syncthreads();
  for (int i = tid; i < 2 * CHB; i += kScanThreads) {
    const int c = c0 + i % CHB;
    if (c >= a.C) continue;
    float s = 0.f;
    for (int r = 0; r < row_step; ++r) s += red[(r * 2 + i / CHB) * CHB + i % CHB];
    a.part_d[(((int64_t)b * a.nseg + seg) * 2 + i / CHB) * a.C + c] = s;
  }
}

// gB and gC: the slices' partial sums in slice order, in the tensors' type.
template <typename T>
__global__ void __launch_bounds__(256) scan_reduce_kernel(const float* part, int slices, int64_t rows, int N, void* gB,
                                                          void* gC) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, width = rows * 2 * N;
  if (i >= width) return;
  float s = 0.f;
  for (int k = 0; k < slices; ++k) s += part[k * width + i];
  const int64_t row = i / (2 * N);
  const int j = (int)(i - row * 2 * N);
  T* to = static_cast<T*>(j < N ? gB : gC);
  to[row * N + (j < N ? j : j - N)] = Pair<T>::from_float(s);
}

// One token: x, dt, z [B][C] and B, C [B][N]; the state is updated in place.
template <typename T>
__global__ void __launch_bounds__(128) scan_step_kernel(ScanArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
  if (i >= (int64_t)a.B * a.C) return;
  const int b = (int)(i / a.C), c = (int)(i - (int64_t)b * a.C);
  const float x = Pair<T>::scalar(static_cast<const T*>(a.x)[b * a.x_sb + c]);
  const float d = scan_delta(
      Pair<T>::scalar(static_cast<const T*>(a.dt)[b * a.dt_sb + c]) + (a.bias ? a.bias[c] : 0.f), a.softplus);
  const T* Bt = static_cast<const T*>(a.Bm) + b * a.b_sb;
  const T* Ct = static_cast<const T*>(a.Cm) + b * a.c_sb;
  float y = (a.D ? a.D[c] : 0.f) * x;
  float* h = a.h_last + i * a.N;
  for (int n = 0; n < a.N; ++n) {
    const float v = fmaf(ex2(d * a.A[(int64_t)c * a.N + n] * kL2E), h[n], d * x * Pair<T>::scalar(Bt[n]));
    h[n] = v;
    y = fmaf(v, Pair<T>::scalar(Ct[n]), y);
  }
  if (a.z) {
    const float z = Pair<T>::scalar(static_cast<const T*>(a.z)[b * a.z_sb + c]);
    y *= z * sigmoid1(z);
  }
  static_cast<T*>(a.out)[i] = Pair<T>::from_float(y);
}

}  // namespace wkv
