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
//
// What it cannot do without is one exponential a state and step in each direction (16 a
// clock and SM), which at 16 states outweighs the bytes; sequential in time, parallel
// over channels and states, and over segments of the time axis where those are too few.
// Measured at 16 x 1024 x 1536, 16 states, bfloat16: forward 243 us (1.7e12
// exponentials a second, 37 % of the unit's rate; 232 us without the kept states),
// backward 714 us, sums 20 us; float32 242, 1045 and 21 us. 1 x 8191 x 1536: summaries
// 72 us, forward 113 us.
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
  int wide;     // rows of x, dt, z, gout move as aligned 16-byte words
  int pairs;    // two adjacent channels of every row move as one aligned word
  int near;     // a tile's rows lie within 2^31 elements
  int wide_bc;  // four adjacent states of B and C move as one aligned word
  int wide_n;   // four adjacent float32 states move as one aligned word (N % 4 == 0)
  int softplus;
};

// softplus(v) = max(v, 0) + log1p(u), u = e^-|v|. The exponent v log2(e) is split in
// two floats so that u keeps float32's relative accuracy at large |v|, and log1p(u) =
// 2 atanh(u / (2 + u)) is its power series: the argument is at most 1/3, so seven
// terms leave 2e-8 of the value, small steps' relative accuracy included. About 17
// instructions a value against about 45 for the library's exp and log1p, which took
// as many issue slots as the scan itself.
__device__ __forceinline__ f2 softplus2(f2 v) {
  const f2 n{fmaxf(-fabsf(v.x), -100.f), fmaxf(-fabsf(v.y), -100.f)};
  const f2 hi = mul2(n, splat(kL2E));
  const f2 lo = fma2(n, splat(1.9259629911e-8f), fma2(n, splat(kL2E), f2{-hi.x, -hi.y}));  // log2(e) - kL2E
  f2 u = ex2x2(hi);
  u = fma2(mul2(u, splat(0.6931471806f)), lo, u);
  const f2 s = mul2(u, rcpx2(add2(u, splat(2.f)))), w = mul2(s, s);
  f2 p = fma2(w, splat(1.f / 13.f), splat(1.f / 11.f));
  p = fma2(w, p, splat(1.f / 9.f));
  p = fma2(w, p, splat(1.f / 7.f));
  p = fma2(w, p, splat(1.f / 5.f));
  p = fma2(w, p, splat(1.f / 3.f));
  const f2 s2 = add2(s, s);
  p = fma2(mul2(s2, w), p, s2);
  return add2(f2{v.x < 0.f ? 0.f : v.x, v.y < 0.f ? 0.f : v.y}, p);  // a NaN stays one
}
__device__ __forceinline__ f2 scan_delta(f2 v, int softplus) { return softplus ? softplus2(v) : v; }

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

// exp(d A) of a pair of states, A2 = A log2(e). The exponential unit's 2^x comes out
// low by about 2e-8 of the value on average for x in [-0.3, 0) (measured over 4e6
// arguments a decade), and a recurrence multiplies by it once a step, so the mean
// counts for as many steps as the state remembers: kDecayShift in the argument takes
// most of it back (the gradient of A of 2 x 1024 steps: 1.1e-6 off without it). It
// costs nothing (a fused multiply-add for the product), is below the rounding of x
// where decays are strong, and leaves 2^0 at exactly 1.
constexpr float kDecayShift = 2.4e-8f;
__device__ __forceinline__ f2 decay2(f2 A2, f2 d) { return ex2x2(fma2(A2, d, splat(kDecayShift))); }

// kS states of one channel, as packed pairs: groups of four adjacent ones, kGap apart.
// Where lanes share a channel their groups alternate (kGap = 4 lanes), so that a group
// of all lanes is one contiguous read of shared memory and whole sectors of the kept
// states (eight adjacent states a lane met in the banks: forward of 16 x 1024 x 1536
// with 64 states 1043 us).
template <int kS, int kGap = 4>
struct States {
  f2 p[kS / 2];
  __device__ __forceinline__ static States zero() {
    States r;
#pragma unroll
    for (int i = 0; i < kS / 2; ++i) r.p[i] = f2{0.f, 0.f};
    return r;
  }
  // the states from n on of a row of N float32 states; past N: zeros. `wide`: four
  // adjacent states move as one aligned word, and N is a multiple of 4.
  __device__ __forceinline__ static States load(const float* row, int n, int N, int wide) {
    States r;
#pragma unroll
    for (int i = 0; i < kS; i += 4) {
      const int m = n + i / 4 * kGap;
      if (wide) {
        const float4 v = m < N ? *reinterpret_cast<const float4*>(row + m) : make_float4(0.f, 0.f, 0.f, 0.f);
        r.p[i / 2] = f2{v.x, v.y};
        r.p[i / 2 + 1] = f2{v.z, v.w};
      } else {
#pragma unroll
        for (int j = 0; j < 4; j += 2)
          r.p[(i + j) / 2] = f2{m + j < N ? row[m + j] : 0.f, m + j + 1 < N ? row[m + j + 1] : 0.f};
      }
    }
    return r;
  }
  __device__ __forceinline__ void store(float* row, int n, int N, int wide) const {
#pragma unroll
    for (int i = 0; i < kS; i += 4) {
      const int m = n + i / 4 * kGap;
      const f2 u = p[i / 2], v = p[i / 2 + 1];
      if (wide) {
        if (m < N) *reinterpret_cast<float4*>(row + m) = make_float4(u.x, u.y, v.x, v.y);
      } else {
        if (m < N) row[m] = u.x;
        if (m + 1 < N) row[m + 1] = u.y;
        if (m + 2 < N) row[m + 2] = v.x;
        if (m + 3 < N) row[m + 3] = v.y;
      }
    }
  }
  // A row of B or C in shared memory.
  __device__ __forceinline__ static States shared(const float* row) {
    States r;
#pragma unroll
    for (int i = 0; i < kS; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(row + i / 4 * kGap);
      r.p[i / 2] = f2{v.x, v.y};
      r.p[i / 2 + 1] = f2{v.z, v.w};
    }
    return r;
  }
  __device__ __forceinline__ void scale(float k) {
#pragma unroll
    for (int i = 0; i < kS / 2; ++i) p[i] = mul2(p[i], splat(k));
  }
};

// Two adjacent channels of one row; `live` false or channels past C: zeros. `pairs`:
// the rows allow a word for both.
template <typename T>
__device__ __forceinline__ Vec<T, 2> load_pair(const T* row, int c, int C, bool live, int pairs) {
  Vec<T, 2> r = Vec<T, 2>::zero();
  if (!live || c >= C) return r;
  if (pairs) return Vec<T, 2>::load(row + c);
  r.e[0] = row[c];
  if (c + 1 < C) r.e[1] = row[c + 1];
  return r;
}
template <typename T>
__device__ __forceinline__ void store_pair(T* row, int c, int C, int pairs, f2 v) {
  if (c >= C) return;
  Vec<T, 2> r;
  r.set({v.x, v.y});
  if (pairs) {
    r.store(row + c);
    return;
  }
  row[c] = r.e[0];
  if (c + 1 < C) row[c + 1] = r.e[1];
}
template <typename T>
__device__ __forceinline__ f2 pair_of(const Vec<T, 2>& r) {
  float f[2];
  r.get(f);
  return f2{f[0], f[1]};
}
__device__ __forceinline__ f2 param_pair(const float* p, int c, int C) {
  return f2{p && c < C ? p[c] : 0.f, p && c + 1 < C ? p[c + 1] : 0.f};
}

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

// The layout of a CTA's work, by the lanes that share a channel and the states of
// a lane. A thread stages pairs of channels: always the same pair, of every kStep-th
// row.
template <int LPC, int kS, int kThr, int kTT, int kPer = 1>
struct ScanShape {
  static constexpr int NP = kS * LPC;           // states, padded
  static constexpr int CH = kThr / LPC * kPer;  // channels of a CTA, kPer of them a lane group's
  static constexpr int TT = kTT;         // steps of a staged tile
  static constexpr int kPairs = CH / 2;
  static constexpr int kStep = kThr / kPairs;
  static constexpr int kRows = TT / kStep;
  static_assert(kRows * kStep == TT, "whole rows a thread");
};

// The forward's and the summaries': kS states a lane, 1024 cells a tile.
template <int LPC, int kS>
using FwdShape = ScanShape<LPC, kS, kScanThreads, 8 * LPC < kScanRows ? 8 * LPC : kScanRows>;

// The state a segment starts from: the earlier segments' contributions in order
// (forward), or the adjoint that the later segments hand back.
template <int kS, int kGap>
__device__ __forceinline__ States<kS, kGap> scan_carry(const ScanArgs& a, int b, int c, int n, States<kS, kGap> h,
                                                       const States<kS, kGap>& A2, int from, int to, int step) {
  for (int s = from; s != to; s += step) {
    const int64_t at = ((int64_t)b * a.nseg + s) * a.C + c;
    const auto add = States<kS, kGap>::load(a.seg_h + at * a.N, n, a.N, a.wide_n);
    const f2 d = splat(a.seg_d[at]);
#pragma unroll
    for (int i = 0; i < kS / 2; ++i) h.p[i] = fma2(ex2x2(mul2(A2.p[i], d)), h.p[i], add.p[i]);
  }
  return h;
}

// Rows of one sequence as a thread stages them: its channel pair of kRows rows.
// `plain`: the CTA's channels all exist, pairs move as words and offsets within a
// tile fit 32 bits; a whole tile is then read without a test per row.
template <typename T, class S>
struct RowSource {
  const T* base;  // channel 0 of row 0
  int64_t pitch;
  __device__ __forceinline__ void fetch(Vec<T, 2> (&to)[S::kRows], int t0, int row0, int cp, const ScanArgs& a, int t_end,
                                        bool plain) const {
    if (plain && t0 + S::TT <= t_end) {
      const T* tile = base + t0 * pitch;
      const uint32_t p = (uint32_t)pitch, at = row0 * p + cp;
#pragma unroll
      for (int k = 0; k < S::kRows; ++k) to[k] = Vec<T, 2>::load(tile + (at + k * S::kStep * p));
    } else {
#pragma unroll
      for (int k = 0; k < S::kRows; ++k) {
        const int t = t0 + row0 + k * S::kStep;
        to[k] = load_pair(base + t * pitch, cp, a.C, t < t_end, a.pairs);
      }
    }
  }
};
__device__ __forceinline__ bool scan_plain(const ScanArgs& a, int c_end) {
  return a.pairs && a.near && c_end <= a.C;
}

// What a segment adds to a zero state (kAdjoint: to a zero adjoint, walking back:
// g <- a (g + C gy)), and its sum of d: the decay across it is exp(A sum d).
template <typename T, int LPC, int kS, bool kAdjoint>
__global__ void __launch_bounds__(kScanThreads) scan_summary_kernel(ScanArgs a) {
  using S = FwdShape<LPC, kS>;
  using St = States<kS, 4 * LPC>;
  __shared__ float4 sdx[S::TT][S::CH];  // d, d, w, w: pairs as the packed arithmetic reads them
  __shared__ __align__(16) float sn[S::TT][S::NP];
  // the last segment's sum serves no later one (the first's, walking back)
  const int cb = blockIdx.x % a.cblocks, seg = blockIdx.x / a.cblocks % (a.nseg - 1) + (kAdjoint ? 1 : 0);
  const int b = blockIdx.x / a.cblocks / (a.nseg - 1);
  const int q = threadIdx.x % LPC, ch = threadIdx.x / LPC, c0 = cb * S::CH, c = c0 + ch;
  const int t_begin = seg * a.seg_len, t_end = min(t_begin + a.seg_len, scan_length(a, b));
  St A2 = St::load(a.A + (int64_t)min(c, a.C - 1) * a.N, 4 * q, a.N, a.wide_n);
  A2.scale(kL2E);
  St h = St::zero();
  f2 dsum{0.f, 0.f};
  const int row0 = threadIdx.x / S::kPairs, cp = c0 + threadIdx.x % S::kPairs * 2;
  const bool plain = scan_plain(a, c0 + S::CH);
  const f2 bias = param_pair(a.bias, cp, a.C);
  const RowSource<T, S> px{static_cast<const T*>(kAdjoint ? a.gout : a.x) + b * (kAdjoint ? a.g_sb : a.x_sb),
                           kAdjoint ? a.g_st : a.x_st};
  const RowSource<T, S> pd{static_cast<const T*>(a.dt) + b * a.dt_sb, a.dt_st};
  const RowSource<T, S> pz{static_cast<const T*>(a.z) + (a.z ? b * a.z_sb : 0), a.z_st};
  const T* pn = static_cast<const T*>(kAdjoint ? a.Cm : a.Bm) + b * (kAdjoint ? a.c_sb : a.b_sb);
  const int64_t sbc = kAdjoint ? a.c_st : a.b_st;
  const int tiles = t_end > t_begin ? (t_end - t_begin + S::TT - 1) / S::TT : 0;
  constexpr int kQ = S::NP / 4, kN = (S::TT * kQ + kScanThreads - 1) / kScanThreads;
  Vec<T, 2> rx[S::kRows], rd[S::kRows], rz[S::kRows];
  Vec<T, 4> rn[kN];
  auto fetch = [&](int t0) {
    px.fetch(rx, t0, row0, cp, a, t_end, plain);
    pd.fetch(rd, t0, row0, cp, a, t_end, plain);
    if (kAdjoint && a.z) pz.fetch(rz, t0, row0, cp, a, t_end, plain);
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      const int i = k * kScanThreads + threadIdx.x, t = t0 + i / kQ;
      rn[k] = load_bc(pn + (int64_t)t * sbc, i % kQ * 4, a.N, i < S::TT * kQ && t < t_end, a.wide_bc);
    }
  };
  if (tiles > 0) fetch(t_begin + (kAdjoint ? tiles - 1 : 0) * S::TT);
  for (int tile = 0; tile < tiles; ++tile) {
    const int t0 = t_begin + (kAdjoint ? tiles - 1 - tile : tile) * S::TT;
#pragma unroll
    for (int k = 0; k < S::kRows; ++k) {
      const int r = row0 + k * S::kStep;
      f2 d = scan_delta(add2(pair_of(rd[k]), bias), a.softplus), w = pair_of(rx[k]);
      if (t0 + r >= t_end) d = f2{0.f, 0.f};
      if constexpr (kAdjoint) {
        if (a.z) {
          const f2 z = pair_of(rz[k]);
          w = mul2(w, mul2(z, sigmoid2<T>(z)));
        }
      } else {
        w = mul2(d, w);
      }
      sdx[r][cp - c0] = make_float4(d.x, d.x, w.x, w.x);
      sdx[r][cp - c0 + 1] = make_float4(d.y, d.y, w.y, w.y);
    }
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      const int i = k * kScanThreads + threadIdx.x;
      float f[4];
      rn[k].get(f);
      if (i < S::TT * kQ) *reinterpret_cast<float4*>(&sn[i / kQ][i % kQ * 4]) = make_float4(f[0], f[1], f[2], f[3]);
    }
    __syncthreads();
    if (tile + 1 < tiles) fetch(t0 + (kAdjoint ? -S::TT : S::TT));
#pragma unroll 4
    for (int j = 0; j < S::TT; ++j) {
      const int i = kAdjoint ? S::TT - 1 - j : j;
      const float4 s = sdx[i][ch];
      const f2 d{s.x, s.y}, w{s.z, s.w};
      const St v = St::shared(&sn[i][4 * q]);
#pragma unroll
      for (int n = 0; n < kS / 2; ++n) {
        const f2 e = decay2(A2.p[n], d);
        h.p[n] = kAdjoint ? mul2(e, fma2(v.p[n], w, h.p[n])) : fma2(e, h.p[n], mul2(v.p[n], w));
      }
      dsum = add2(dsum, d);
    }
    __syncthreads();
  }
  if (c >= a.C) return;
  const int64_t at = ((int64_t)b * a.nseg + seg) * a.C + c;
  h.store(a.seg_h + at * a.N, 4 * q, a.N, a.wide_n);
  if (q == 0) a.seg_d[at] = dsum.x;
}

// Forward. Bound by the latency of a warp's own work at the 2.6 warps a scheduler that
// 384 CTAs give (16 x 1024 x 1536: issue slots 44 % busy, the exponential unit 49 %); at
// 1024 CTAs, where all slots are full, it reaches 50 % of that unit (509 us for 64 x
// 1024 x 1024). About half of the instructions are a cell's own (softplus, gate, staging),
// spread over its 16 states.
//
// A CTA walks one segment of CH channels of one sequence; LPC lanes share a
// channel, kS states each. Tiles of TT steps are staged: d and d x of every
// (step, channel) and B, C in float32, while the next tile's raw rows are already
// under way to registers. The lanes' parts of y are summed by an exchange of four
// steps at a time, and the gate and the output are done by whole rows again.
template <typename T, int LPC, int kS>
__global__ void __launch_bounds__(kScanThreads) scan_fwd_kernel(ScanArgs a) {
  using S = FwdShape<LPC, kS>;
  using St = States<kS, 4 * LPC>;
  __shared__ float4 sdx[S::TT][S::CH];  // d, d, d x, d x: pairs as the packed arithmetic reads them
  __shared__ __align__(16) float sbc[S::TT][2 * S::NP];
  __shared__ __align__(16) float sy[S::TT][S::CH + 8];
  const int cb = blockIdx.x % a.cblocks, seg = blockIdx.x / a.cblocks % a.nseg, b = blockIdx.x / a.cblocks / a.nseg;
  const int q = threadIdx.x % LPC, ch = threadIdx.x / LPC, c0 = cb * S::CH, c = c0 + ch;
  const int len = scan_length(a, b);
  const int t_begin = seg * a.seg_len, t_end = min(t_begin + a.seg_len, a.T), t_live = min(t_end, len);
  const int64_t hc = ((int64_t)b * a.C + c) * a.N;
  const bool mine = c < a.C;
  St A2 = St::load(a.A + (int64_t)min(c, a.C - 1) * a.N, 4 * q, a.N, a.wide_n);
  A2.scale(kL2E);
  St h = St::zero();
  if (mine && a.h0) h = St::load(a.h0 + hc, 4 * q, a.N, a.wide_n);
  if (mine) h = scan_carry(a, b, c, 4 * q, h, A2, 0, seg, 1);

  const int row0 = threadIdx.x / S::kPairs, cp = c0 + threadIdx.x % S::kPairs * 2;
  const bool plain = scan_plain(a, c0 + S::CH);
  const f2 bias = param_pair(a.bias, cp, a.C), D = param_pair(a.D, cp, a.C);
  const RowSource<T, S> px{static_cast<const T*>(a.x) + b * a.x_sb, a.x_st};
  const RowSource<T, S> pd{static_cast<const T*>(a.dt) + b * a.dt_sb, a.dt_st};
  const RowSource<T, S> pz{static_cast<const T*>(a.z) + (a.z ? b * a.z_sb : 0), a.z_st};
  constexpr int kQ = S::NP / 4, kBC = (S::TT * 2 * kQ + kScanThreads - 1) / kScanThreads;
  Vec<T, 2> rx[S::kRows], rd[S::kRows], rz[S::kRows];
  Vec<T, 4> rbc[kBC];
  auto fetch = [&](int t0) {
    px.fetch(rx, t0, row0, cp, a, t_live, plain);
    pd.fetch(rd, t0, row0, cp, a, t_live, plain);
    if (a.z) pz.fetch(rz, t0, row0, cp, a, t_live, plain);
#pragma unroll
    for (int k = 0; k < kBC; ++k) {
      const int i = k * kScanThreads + threadIdx.x, tb = t0 + i / (2 * kQ), n = i % kQ * 4;
      const bool on = i < S::TT * 2 * kQ && tb < t_live;
      const T* p = i % (2 * kQ) < kQ ? static_cast<const T*>(a.Bm) + b * a.b_sb + (int64_t)tb * a.b_st
                                     : static_cast<const T*>(a.Cm) + b * a.c_sb + (int64_t)tb * a.c_st;
      rbc[k] = load_bc(p, n, a.N, on, a.wide_bc);
    }
  };
  const int nck = (a.T + kScanCkpt - 1) / kScanCkpt;
  float* ckpt = a.ckpt && mine ? a.ckpt + ((int64_t)b * nck * a.C + c) * a.N : nullptr;
  T* out = static_cast<T*>(a.out) + (int64_t)b * a.T * a.C;
  if (t_begin < t_live) fetch(t_begin);
  for (int t0 = t_begin; t0 < t_live; t0 += S::TT) {
    Vec<T, 2> cx[S::kRows], cz[S::kRows];
#pragma unroll
    for (int k = 0; k < S::kRows; ++k) {
      const int r = row0 + k * S::kStep;
      cx[k] = rx[k];
      cz[k] = rz[k];
      f2 d = scan_delta(add2(pair_of(rd[k]), bias), a.softplus);
      if (t0 + r >= t_live) d = f2{0.f, 0.f};
      const f2 w = mul2(d, pair_of(rx[k]));
      sdx[r][cp - c0] = make_float4(d.x, d.x, w.x, w.x);
      sdx[r][cp - c0 + 1] = make_float4(d.y, d.y, w.y, w.y);
    }
#pragma unroll
    for (int k = 0; k < kBC; ++k) {
      const int i = k * kScanThreads + threadIdx.x;
      float f[4];
      rbc[k].get(f);
      if (i < S::TT * 2 * kQ)
        *reinterpret_cast<float4*>(&sbc[i / (2 * kQ)][i % (2 * kQ) * 4]) = make_float4(f[0], f[1], f[2], f[3]);
    }
    __syncthreads();
    if (t0 + S::TT < t_live) fetch(t0 + S::TT);
#pragma unroll 2
    for (int j = 0; j < S::TT; j += 4) {
      if (j % kScanCkpt == 0 && ckpt && t0 + j < t_live)
        h.store(ckpt + (int64_t)((t0 + j) / kScanCkpt) * a.C * a.N, 4 * q, a.N, a.wide_n);
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 s = sdx[j + i][ch];
        const f2 d{s.x, s.y}, w{s.z, s.w};
        const St Bt = St::shared(&sbc[j + i][4 * q]), Ct = St::shared(&sbc[j + i][S::NP + 4 * q]);
        f2 v[2];
#pragma unroll
        for (int n = 0; n < kS / 2; ++n) {
          h.p[n] = fma2(decay2(A2.p[n], d), h.p[n], mul2(Bt.p[n], w));
          v[n % 2] = n < 2 ? mul2(h.p[n], Ct.p[n]) : fma2(h.p[n], Ct.p[n], v[n % 2]);
        }
        const f2 u = add2(v[0], v[1]);
        y[i] = u.x + u.y;
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
    const bool whole = plain && t0 + S::TT <= t_live;
    T* tile = out + (int64_t)t0 * a.C;
#pragma unroll
    for (int k = 0; k < S::kRows; ++k) {
      const int r = row0 + k * S::kStep;
      const float2 v = *reinterpret_cast<const float2*>(&sy[r][cp - c0]);
      f2 y = fma2(D, pair_of(cx[k]), f2{v.x, v.y});
      if (a.z) {
        const f2 z = pair_of(cz[k]);
        y = mul2(y, mul2(z, sigmoid2<T>(z)));
      }
      if (whole) {
        Vec<T, 2> o;
        o.set({y.x, y.y});
        o.store(tile + (r * (uint32_t)a.C + cp));
      } else if (t0 + r < t_live) {
        store_pair(tile + (int64_t)r * a.C, cp, a.C, a.pairs, y);
      }
    }
  }
  // the rows past the sequence's length
  for (int i = threadIdx.x; i < (t_end - max(t_begin, t_live)) * S::CH; i += kScanThreads) {
    const int t = max(t_begin, t_live) + i / S::CH, k = c0 + i % S::CH;
    if (k < a.C) out[(int64_t)t * a.C + k] = Pair<T>::from_float(0.f);
  }
  if (a.h_last && mine && seg == a.nseg - 1) h.store(a.h_last + hc, 4 * q, a.N, a.wide_n);
}

__device__ __forceinline__ void copy16(void* dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0)
               : "memory");
}

// D = A B + C for one m16n8k8 tile of tf32 factors with float32 sums.
__device__ __forceinline__ void mma_tf32(float (&d)[4], float a0, float a1, float a2, float a3, uint32_t b0,
                                         uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)), "r"(__float_as_uint(a2)), "r"(__float_as_uint(a3)),
        "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// Sums over the lanes of a channel with the tensor core, where at least four lanes
// share one. The four lanes of a tile's k group belong to one channel and a column is
// a lane group: a channel, or a half or quarter of one. A pair of values is a B
// operand as it lies in its two registers; the A operand is a 0/1 matrix that adds
// value r of four into row 2 r. Two A operands serve all tiles, because the rows from
// 8 on may hold anything: they get value r in row 2 r + 9, from where the odd lane
// groups read it. A step's three sums of two channels take 16 instructions this way,
// by shuffles 36.
//
// A term enters as the sum of two tf32 values of 11 bits, its upper ones and the rest
// (rounded once to 11 bits, a sum that cancels would lose more than the result's own
// rounding to bfloat16 does). For 16-bit tensors the upper ones are cut off, which keeps 22
// bits of the term. For float32 tensors they are rounded: the rest is then half as large and
// of either sign, at most the last of float32's 24 bits is lost, and the gradients' errors
// are those of sums in float32 (of the step's 2.3e-7 -> 1.9e-7, 16 states), for 2.7 % of the
// kernel's time at 16 x 1024 x 1536 (a third value, which keeps all bits, gave the same
// errors for 7 %).
// A term that is infinite or NaN makes all rows of its tile NaN: the caller then adds by
// shuffles instead.
template <typename T>
struct StateSums {
  float sel[8];  // two A operands: for the values 0, 1 and for 2, 3

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      sel[r] = threadIdx.x % 32 / 4 == r ? 1.f : 0.f;
      asm volatile("" : "+f"(sel[r]));  // stays in its register: rebuilding an operand costs more than its product
    }
  }
  static __device__ __forceinline__ float upper(float v) {
    return __uint_as_float((__float_as_uint(v) + (sizeof(T) == 2 ? 0u : 0x1000u)) & 0xffffe000u);
  }
  // the tile of four values
  __device__ __forceinline__ void sum(float (&d)[4], f2 v, f2 w) const {
    const f2 vh{upper(v.x), upper(v.y)}, wh{upper(w.x), upper(w.y)};
    const f2 vl = sub2(v, vh), wl = sub2(w, wh);
    const float none[4] = {0.f, 0.f, 0.f, 0.f};
    mma_tf32(d, sel[0], sel[1], sel[2], sel[3], __float_as_uint(vh.x), __float_as_uint(vh.y), none);
    mma_tf32(d, sel[4], sel[5], sel[6], sel[7], __float_as_uint(wh.x), __float_as_uint(wh.y), d);
    mma_tf32(d, sel[0], sel[1], sel[2], sel[3], __float_as_uint(vl.x), __float_as_uint(vl.y), d);
    mma_tf32(d, sel[4], sel[5], sel[6], sel[7], __float_as_uint(wl.x), __float_as_uint(wl.y), d);
  }
};
// The lane's pair of columns of value (lane / 8) of two tiles: the even lane groups'
// from tile a, the odd ones' from tile b.
__device__ __forceinline__ f2 tile_pair(const float (&a)[4], const float (&b)[4]) {
  return threadIdx.x & 4 ? f2{b[2], b[3]} : f2{a[0], a[1]};
}

// Shared memory of the backward kernel (see there), in bytes from the start.
constexpr int kScanBwdThreads = 128;
// Channels of a thread: two share the reads of B and C and a tile's columns, where the
// tensor core sums; with two lanes a channel one is faster (16 x 1024 x 1536 with 8
// states 443 us, with two 488 and a pass over segments of 82).
__host__ __device__ constexpr int scan_bwd_per(int lanes) { return lanes >= 4 ? 2 : 1; }
template <typename T, int LPC>
struct ScanBwdSmem {
  using S = ScanShape<LPC, 4, kScanBwdThreads, 16, scan_bwd_per(LPC)>;
  static constexpr int kWarps = kScanBwdThreads / 32;
  static constexpr int TS = S::TT;              // steps of a tile
  static constexpr int kCells = TS * S::CH;     // (step, channel) pairs of a tile
  static constexpr int kPitch = S::CH + 8;
  static constexpr int kGy = kCells * 16;       // after d, d, d x, d x (float4 [kCells]): gy, gy (float2 [kCells])
  static constexpr int kRaw = kGy + kCells * 8;                      // T [2][4][kCells]
  static constexpr int kBC = kRaw + 8 * kCells * (int)sizeof(T);     // float [TS][2 NP]
  static constexpr int kRes = kBC + TS * 2 * S::NP * 4;              // float [3][TS][kPitch]
  static constexpr int kPart = kRes + 3 * TS * kPitch * 4;           // float [TS][warps][2 NP]
  static constexpr int kHeld = kPart + TS * kWarps * 2 * S::NP * 4;  // float [threads][4 kPer]
  static constexpr int kBytes = kHeld + (LPC >= 4 ? kScanBwdThreads * 4 * scan_bwd_per(LPC) * 4 : 0);
};

// A CTA walks one segment of CH channels of one sequence backwards, in tiles of TS
// steps. Per sub-chunk of 8 steps a thread runs four states of each of its channels
// forward from the kept states, with p_t = a_t h_{t-1} in registers, and then back
// with the adjoint (a_t again from the exponential unit, which has the time: held in
// registers it would cost a quarter of the resident warps). The sums over states (for
// gx, gdt, gz) go through the tensor core, the sums over channels (gB, gC) are
// exchanged among the lanes, added over the warps and left as one partial row of the
// CTA's channels. Bound by issue and latency at 2.6 warps a scheduler: 26 instructions for
// 32 state updates, of which 8 are staging and the epilogue. 255 registers a thread, longer
// and shorter tiles and a delayed read of the tensor core's sums were no faster. The bounds
// and the plan are for three CTAs an SM, which 16-bit tensors have (32 to 44 bytes spilled);
// float32 with 9 to 16 states takes 85,504 bytes of shared memory, so two fit, and spills 124
// bytes for a third that does not come.
template <typename T, int LPC>
__global__ void __launch_bounds__(kScanBwdThreads, 3) scan_bwd_kernel(ScanArgs a) {
  using L = ScanBwdSmem<T, LPC>;
  using S = typename L::S;
  using St = States<4>;
  constexpr int NP = S::NP, CH = S::CH, TS = L::TS, kCells = L::kCells, kThr = kScanBwdThreads, kLane = 32 / LPC;
  constexpr int kPer = scan_bwd_per(LPC);
  extern __shared__ __align__(16) char smem[];
  float4* slot = reinterpret_cast<float4*>(smem);             // d, d, d x, d x of a cell
  float2* sgy = reinterpret_cast<float2*>(smem + L::kGy);     // gy, gy
  T* raw = reinterpret_cast<T*>(smem + L::kRaw);              // x, dt, gout, z of this tile and the next
  float* sbc = reinterpret_cast<float*>(smem + L::kBC);
  float* res = reinterpret_cast<float*>(smem + L::kRes);      // sum g B, sum A g p log2(e), sum C h of a cell
  float* part = reinterpret_cast<float*>(smem + L::kPart);
  const int tid = threadIdx.x, warp = tid / 32, q = tid % LPC, ch = warp * kLane * kPer + tid % 32 / LPC;
  const int cb = blockIdx.x % a.cblocks, seg = blockIdx.x / a.cblocks % a.nseg, b = blockIdx.x / a.cblocks / a.nseg;
  const int c0 = cb * CH, c = c0 + ch;  // and c + kLane
  const int len = scan_length(a, b);
  const int t_begin = seg * a.seg_len, t_end = min(t_begin + a.seg_len, a.T), t_live = min(t_end, len);
  const int nck = (a.T + kScanCkpt - 1) / kScanCkpt;

  St A2[kPer], g[kPer], gA[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const int k = c + u * kLane;
    A2[u] = g[u] = gA[u] = St::zero();
    if (k < a.C) {
      A2[u] = St::load(a.A + (int64_t)k * a.N, 4 * q, a.N, a.wide_n);
      A2[u].scale(kL2E);
      if (a.gh_last) g[u] = St::load(a.gh_last + ((int64_t)b * a.C + k) * a.N, 4 * q, a.N, a.wide_n);
      g[u] = scan_carry(a, b, k, 4 * q, g[u], A2[u], a.nseg - 1, seg, -1);
    }
  }

  // rows past the length: zero gradients
  for (int i = tid; i < (t_end - max(t_begin, t_live)) * CH; i += kThr) {
    const int t = max(t_begin, t_live) + i / CH, k = c0 + i % CH;
    if (k < a.C) {
      const int64_t at = ((int64_t)b * a.T + t) * a.C + k;
      static_cast<T*>(a.gx)[at] = Pair<T>::from_float(0.f);
      static_cast<T*>(a.gdt)[at] = Pair<T>::from_float(0.f);
      if (a.gz) static_cast<T*>(a.gz)[at] = Pair<T>::from_float(0.f);
    }
  }
  float* pbc = a.part_bc + ((int64_t)cb * a.B + b) * a.T * 2 * a.N;
  for (int i = tid; i < (t_end - max(t_begin, t_live)) * 2 * a.N; i += kThr)
    pbc[(int64_t)max(t_begin, t_live) * 2 * a.N + i] = 0.f;

  const int row0 = tid / S::kPairs, cl = tid % S::kPairs * 2, cp = c0 + cl;
  const bool plain = scan_plain(a, c0 + CH);
  const f2 bias = param_pair(a.bias, cp, a.C), D = param_pair(a.D, cp, a.C);
  f2 gD{0.f, 0.f}, gb{0.f, 0.f};

  // Raw rows come by asynchronous copies of 16 bytes, one thread always the same
  // word of its tensors' tiles; rows without that alignment by plain loads. A copy that
  // only writes zeros names a source all the same, which has to be aligned like any
  // other: x's first word (`wide` says nothing of A).
  constexpr int E = 16 / (int)sizeof(T), kWords = kCells / E, kCopies = (4 * kWords + kThr - 1) / kThr;
  const T* src[kCopies];
  int64_t back[kCopies];
#pragma unroll
  for (int j = 0; j < kCopies; ++j) {
    const int i = j * kThr + tid, k = i / kWords, cell = i % kWords * E;
    const T* p = static_cast<const T*>(k == 0 ? a.x : k == 1 ? a.dt : k == 2 ? a.gout : a.z);
    const int64_t sb = k == 0 ? a.x_sb : k == 1 ? a.dt_sb : k == 2 ? a.g_sb : a.z_sb;
    const int64_t st = k == 0 ? a.x_st : k == 1 ? a.dt_st : k == 2 ? a.g_st : a.z_st;
    src[j] = k < 4 && p && c0 + cell % CH < a.C ? p + b * sb + cell / CH * st + c0 + cell % CH : nullptr;
    back[j] = st;
  }
  auto fetch = [&](int t0, int stage) {
    T* dst = raw + stage * 4 * kCells;
    if (a.wide) {
#pragma unroll
      for (int j = 0; j < kCopies; ++j) {
        const int i = j * kThr + tid;
        if (kCopies * kThr > 4 * kWords && i >= 4 * kWords) break;
        const bool on = src[j] != nullptr && t0 + i % kWords * E / CH < t_live;
        copy16(dst + i * E, on ? static_cast<const void*>(src[j] + t0 * back[j]) : a.x, on);
      }
    } else {
      for (int k = 0; k < (a.z ? 4 : 3); ++k) {
        const T* p = static_cast<const T*>(k == 0 ? a.x : k == 1 ? a.dt : k == 2 ? a.gout : a.z) +
                     b * (k == 0 ? a.x_sb : k == 1 ? a.dt_sb : k == 2 ? a.g_sb : a.z_sb);
        const int64_t st = k == 0 ? a.x_st : k == 1 ? a.dt_st : k == 2 ? a.g_st : a.z_st;
#pragma unroll 4
        for (int i = tid; i < kCells; i += kThr) {
          const int t = t0 + i / CH, k0 = c0 + i % CH;
          dst[k * kCells + i] = t < t_live && k0 < a.C ? p[t * st + k0] : Pair<T>::from_float(0.f);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  constexpr int kBC = (TS * 2 * LPC + kThr - 1) / kThr;
  Vec<T, 4> rbc[kBC];
  auto fetch_bc = [&](int t0) {
#pragma unroll
    for (int k = 0; k < kBC; ++k) {
      const int i = k * kThr + tid, t = t0 + i / (2 * LPC), n = i % LPC * 4;
      const bool on = i < TS * 2 * LPC && t < t_live;
      const T* p = i % (2 * LPC) < LPC ? static_cast<const T*>(a.Bm) + b * a.b_sb + (int64_t)t * a.b_st
                                       : static_cast<const T*>(a.Cm) + b * a.c_sb + (int64_t)t * a.c_st;
      rbc[k] = load_bc(p, n, a.N, on, a.wide_bc);
    }
  };
  auto kept = [&](int t, int u) {  // the state before step t, a multiple of 8, of the thread's channel u
    if (t >= t_live || t < t_begin) return St::zero();
    const int64_t row = ((int64_t)b * nck + t / kScanCkpt) * a.C + min(c + u * kLane, a.C - 1);
    return St::load(a.ckpt + row * a.N, 4 * q, a.N, a.wide_n);
  };

  const int tiles = t_live > t_begin ? (t_live - t_begin + TS - 1) / TS : 0;
  StateSums<T> sums;
  sums.init();
  if (tiles > 0) {
    fetch(t_begin + (tiles - 1) * TS, 0);
    fetch_bc(t_begin + (tiles - 1) * TS);
  }
  St next[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) next[u] = kept(t_begin + tiles * TS - 8, u);
  int stage = 0;
  for (int tile = tiles - 1; tile >= 0; --tile, stage ^= 1) {
    const int t0 = t_begin + tile * TS;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    const T* cur = raw + stage * 4 * kCells;
#pragma unroll
    for (int k = 0; k < S::kRows; ++k) {
      const int r = row0 + k * S::kStep, at = r * CH + cl;
      const f2 x = pair_of(Vec<T, 2>::load(cur + at));
      f2 d = scan_delta(add2(pair_of(Vec<T, 2>::load(cur + kCells + at)), bias), a.softplus);
      if (t0 + r >= t_live) d = f2{0.f, 0.f};
      f2 gy = pair_of(Vec<T, 2>::load(cur + 2 * kCells + at));
      if (a.z) {
        const f2 z = pair_of(Vec<T, 2>::load(cur + 3 * kCells + at));
        gy = mul2(gy, mul2(z, sigmoid2<T>(z)));
      }
      const f2 dx = mul2(d, x);
      slot[at] = make_float4(d.x, d.x, dx.x, dx.x);
      slot[at + 1] = make_float4(d.y, d.y, dx.y, dx.y);
      *reinterpret_cast<float4*>(sgy + at) = make_float4(gy.x, gy.x, gy.y, gy.y);
    }
#pragma unroll
    for (int k = 0; k < kBC; ++k) {
      const int i = k * kThr + tid;
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
#pragma unroll 1
    for (int sub = TS / 8 - 1; sub >= 0; --sub) {
      const float* bc = sbc + sub * 8 * 2 * NP + 4 * q;
      const float4* sl = slot + sub * 8 * CH + ch;
      const float2* sg = sgy + sub * 8 * CH + ch;
      St p[8][kPer];
      {
        St h[kPer];
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
          h[u] = next[u];
          next[u] = kept(t0 + (sub - 1) * 8, u);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const St Bt = St::shared(bc + i * 2 * NP);
#pragma unroll
          for (int u = 0; u < kPer; ++u) {
            const float4 s = sl[i * CH + u * kLane];
            const f2 d{s.x, s.y}, w{s.z, s.w};
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              p[i][u].p[n] = mul2(decay2(A2[u].p[n], d), h[u].p[n]);
              h[u].p[n] = fma2(Bt.p[n], w, p[i][u].p[n]);
            }
          }
        }
      }
      St gAs[kPer];
      f2 check{0.f, 0.f};
      float* held = reinterpret_cast<float*>(smem + L::kHeld) + tid * 4 * kPer;  // the adjoint as these steps get it
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        gAs[u] = St::zero();
        if constexpr (LPC >= 4) g[u].store(held + u * 4, 0, 4, 1);
      }
#pragma unroll
      for (int two = 3; two >= 0; --two) {  // two steps at a time
        f2 along[2], gd[2], y[2];           // of the thread's two channels
#pragma unroll
        for (int ii = 1; ii >= 0; --ii) {
          const int i = two * 2 + ii;
          const St Bt = St::shared(bc + i * 2 * NP), Ct = St::shared(bc + i * 2 * NP + NP);
          f2 sumB[2], sumC[2];
          float ra[2] = {}, rg[2] = {}, ry[2] = {};
#pragma unroll
          for (int u = 0; u < kPer; ++u) {
            const float4 s = sl[i * CH + u * kLane];
            const float2 s2 = sg[i * CH + u * kLane];
            const f2 d{s.x, s.y}, w{s.z, s.w}, gy{s2.x, s2.y};
            f2 al, yy, dd;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const f2 hn = fma2(Bt.p[n], w, p[i][u].p[n]), gn = fma2(Ct.p[n], gy, g[u].p[n]);
              const f2 v = mul2(gn, p[i][u].p[n]);
              sumB[n] = u == 0 ? mul2(gn, w) : fma2(gn, w, sumB[n]);
              sumC[n] = u == 0 ? mul2(hn, gy) : fma2(hn, gy, sumC[n]);
              al = n == 0 ? mul2(gn, Bt.p[n]) : fma2(gn, Bt.p[n], al);
              yy = n == 0 ? mul2(hn, Ct.p[n]) : fma2(hn, Ct.p[n], yy);
              dd = n == 0 ? mul2(v, A2[u].p[n]) : fma2(v, A2[u].p[n], dd);
              gAs[u].p[n] = fma2(v, d, gAs[u].p[n]);
              g[u].p[n] = mul2(gn, decay2(A2[u].p[n], d));
            }
            ra[u] = al.x + al.y;
            ry[u] = yy.x + yy.y;
            rg[u] = dd.x + dd.y;
          }
          along[ii] = f2{ra[0], ra[1]};
          gd[ii] = f2{rg[0], rg[1]};
          y[ii] = f2{ry[0], ry[1]};
          // over the warp's channels: lane group l keeps sum l of (B: 0..3, C: 4..7) of its quad
          float v[8] = {sumB[0].x, sumB[0].y, sumB[1].x, sumB[1].y, sumC[0].x, sumC[0].y, sumC[1].x, sumC[1].y};
          reduce_scatter<8, kLane, LPC>(v);
          constexpr int kOwn = kLane < 8 ? 8 / kLane : 1, kSkip = kLane < 8 ? 1 : kLane / 8;
          const int l = tid % 32 / LPC;
          if (l % kSkip == 0) {
            float* pw = part + ((sub * 8 + i) * L::kWarps + warp) * 2 * NP + 4 * q;
#pragma unroll
            for (int k = 0; k < kOwn; ++k) {
              const int at = l / kSkip * kOwn + k;
              pw[at < 4 ? at : NP + at - 4] = v[k];
            }
          }
        }
        float* to = res + (sub * 8 + two * 2) * L::kPitch;  // step two * 2; the other is a row on
        if constexpr (LPC >= 4) {
          float t0_[4], t1_[4], ty[4];
          sums.sum(t0_, along[0], gd[0]);
          sums.sum(t1_, along[1], gd[1]);
          sums.sum(ty, y[0], y[1]);
          f2 s = tile_pair(t0_, t1_), r = tile_pair(ty, ty);
          // value (lane / 8): along of channel 0, of channel 1, gd of each; y of each at step 0, at step 1
          const int k = tid % 32 / 8, step = tid / 4 % 2, col = tid % 4 * 2, c8 = warp * kLane * kPer + k % 2 * kLane;
          check = add2(check, mul2(add2(s, r), splat(0.f)));  // NaN if one of them is not finite
          float* ps = to + k / 2 * TS * L::kPitch + step * L::kPitch + c8;
          float* pr = to + 2 * TS * L::kPitch + k / 2 * L::kPitch + c8;
          if constexpr (LPC == 4) {  // a column is a channel
            *reinterpret_cast<float2*>(ps + col) = make_float2(s.x, s.y);
            if (step == 0) *reinterpret_cast<float2*>(pr + col) = make_float2(r.x, r.y);
          } else {
            float su = s.x + s.y, ru = r.x + r.y;  // two columns a channel, or four
            if constexpr (LPC == 16) {
              su += __shfl_xor_sync(kFull, su, 1);
              ru += __shfl_xor_sync(kFull, ru, 1);
            }
            if (LPC == 8 || tid % 2 == 0) {
              ps[col / (LPC / 4)] = su;
              if (step == 0) pr[col / (LPC / 4)] = ru;
            }
          }
        } else {
#pragma unroll
          for (int ii = 0; ii < 2; ++ii)
#pragma unroll
            for (int u = 0; u < kPer; ++u) {
              float v[3] = {u ? along[ii].y : along[ii].x, u ? gd[ii].y : gd[ii].x, u ? y[ii].y : y[ii].x};
#pragma unroll
              for (int k = 0; k < 3; ++k) {
                v[k] += __shfl_xor_sync(kFull, v[k], 1);
                if (q == 0) to[k * TS * L::kPitch + ii * L::kPitch + ch + u * kLane] = v[k];
              }
            }
        }
      }
      if constexpr (LPC >= 4) {
        if (__any_sync(kFull, check.x + check.y != 0.f)) {
          // A value is not finite: these sums once more, each channel's for itself, so that
          // it stays in its channel. Not for speed: the loops are rolled.
          __syncwarp();
          St h[kPer], back[kPer], q8[8][kPer];
#pragma unroll
          for (int u = 0; u < kPer; ++u) {
            h[u] = kept(t0 + sub * 8, u);
            back[u] = St::shared(held + u * 4);
          }
#pragma unroll 1
          for (int i = 0; i < 8; ++i) {
            const St Bt = St::shared(bc + i * 2 * NP);
#pragma unroll
            for (int u = 0; u < kPer; ++u) {
              const float4 s = sl[i * CH + u * kLane];
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                q8[i][u].p[n] = mul2(decay2(A2[u].p[n], f2{s.x, s.y}), h[u].p[n]);
                h[u].p[n] = fma2(Bt.p[n], f2{s.z, s.w}, q8[i][u].p[n]);
              }
            }
          }
#pragma unroll 1
          for (int i = 7; i >= 0; --i) {
            const St Bt = St::shared(bc + i * 2 * NP), Ct = St::shared(bc + i * 2 * NP + NP);
#pragma unroll
            for (int u = 0; u < kPer; ++u) {
              const float4 s = sl[i * CH + u * kLane];
              const float2 s2 = sg[i * CH + u * kLane];
              f2 v[3] = {f2{0.f, 0.f}, f2{0.f, 0.f}, f2{0.f, 0.f}};
#pragma unroll
              for (int n = 0; n < 2; ++n) {
                const f2 hn = fma2(Bt.p[n], f2{s.z, s.w}, q8[i][u].p[n]), gn = fma2(Ct.p[n], f2{s2.x, s2.y}, back[u].p[n]);
                v[0] = fma2(gn, Bt.p[n], v[0]);
                v[1] = fma2(mul2(gn, q8[i][u].p[n]), A2[u].p[n], v[1]);
                v[2] = fma2(hn, Ct.p[n], v[2]);
                back[u].p[n] = mul2(gn, decay2(A2[u].p[n], f2{s.x, s.y}));
              }
#pragma unroll
              for (int e = 0; e < 3; ++e) {
                float w = v[e].x + v[e].y;
#pragma unroll
                for (int o = LPC / 2; o > 0; o >>= 1) w += __shfl_xor_sync(kFull, w, o);
                if (q == 0) res[(e * TS + sub * 8 + i) * L::kPitch + ch + u * kLane] = w;
              }
            }
          }
        }
      }
      // gA: eight steps' sum at a time, which keeps the long sum's rounding small
#pragma unroll
      for (int u = 0; u < kPer; ++u) {
        gA[u].p[0] = add2(gA[u].p[0], gAs[u].p[0]);
        gA[u].p[1] = add2(gA[u].p[1], gAs[u].p[1]);
      }
    }
    __syncthreads();
    const bool whole = plain && t0 + TS <= t_live;
    const int64_t to = ((int64_t)b * a.T + t0) * a.C;
    T *tx = static_cast<T*>(a.gx) + to, *td = static_cast<T*>(a.gdt) + to, *tz = static_cast<T*>(a.gz) + (a.gz ? to : 0);
#pragma unroll
    for (int k = 0; k < S::kRows; ++k) {
      const int r = row0 + k * S::kStep, at = r * CH + cl;
      const f2 d{slot[at].x, slot[at + 1].x};
      const float* v = res + r * L::kPitch + cl;
      const float2 al = *reinterpret_cast<const float2*>(v), ga = *reinterpret_cast<const float2*>(v + TS * L::kPitch);
      const f2 along{al.x, al.y}, x = pair_of(Vec<T, 2>::load(cur + at));
      const f2 go = pair_of(Vec<T, 2>::load(cur + 2 * kCells + at));
      f2 gy = go, gz{0.f, 0.f};
      if (a.z) {
        const f2 z = pair_of(Vec<T, 2>::load(cur + 3 * kCells + at)), sz = sigmoid2<T>(z);
        const float2 yv = *reinterpret_cast<const float2*>(v + 2 * TS * L::kPitch);
        const f2 gs = mul2(go, sz), y = fma2(D, x, f2{yv.x, yv.y});
        gy = mul2(gs, z);
        gz = mul2(mul2(gs, y), fma2(z, sub2(splat(1.f), sz), splat(1.f)));
      }
      f2 gdt = fma2(x, along, mul2(f2{ga.x, ga.y}, splat(0.6931471806f)));
      if (a.softplus) gdt = mul2(gdt, sigmoid2<T>(add2(pair_of(Vec<T, 2>::load(cur + kCells + at)), bias)));
      const f2 gx = fma2(d, along, mul2(D, gy));
      if (whole) {
        const uint32_t off = r * (uint32_t)a.C + cp;
        Vec<T, 2> o;
        o.set({gx.x, gx.y});
        o.store(tx + off);
        o.set({gdt.x, gdt.y});
        o.store(td + off);
        if (a.gz) {
          o.set({gz.x, gz.y});
          o.store(tz + off);
        }
      } else if (t0 + r < t_live) {
        const int64_t off = (int64_t)r * a.C;
        store_pair(tx + off, cp, a.C, a.pairs, gx);
        store_pair(td + off, cp, a.C, a.pairs, gdt);
        if (a.gz) store_pair(tz + off, cp, a.C, a.pairs, gz);
      }
      if (t0 + r < t_live) {
        gD = fma2(gy, x, gD);
        gb = add2(gb, gdt);
      }
    }
#pragma unroll
    for (int k = 0; k < (TS * 2 * LPC + kThr - 1) / kThr; ++k) {
      const int i = k * kThr + tid, r = i / (2 * LPC), j = i % (2 * LPC) * 4, n = j < NP ? j : j - NP;
      if (i >= TS * 2 * LPC || t0 + r >= t_live) break;
      const float* p = part + r * L::kWarps * 2 * NP + j;
      States<4> s = States<4>::shared(p);
#pragma unroll
      for (int w = 1; w < L::kWarps; ++w) {
        const States<4> o = States<4>::shared(p + w * 2 * NP);
        s.p[0] = add2(s.p[0], o.p[0]);
        s.p[1] = add2(s.p[1], o.p[1]);
      }
      s.store(pbc + (int64_t)(t0 + r) * 2 * a.N + (j < NP ? 0 : a.N), n, a.N, a.wide_n);
    }
  }
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const int k = c + u * kLane;
    if (k >= a.C) continue;
    gA[u].store(a.part_a + (((int64_t)b * a.nseg + seg) * a.C + k) * a.N, 4 * q, a.N, a.wide_n);
    if (a.gh0 && seg == 0) g[u].store(a.gh0 + ((int64_t)b * a.C + k) * a.N, 4 * q, a.N, a.wide_n);
  }
  // gD and gbias over the rows of the thread's channels
  float* red = reinterpret_cast<float*>(slot);
  static_assert(kCells * 4 >= 4 * kThr, "the slots hold the channel sums");
  __syncthreads();
  *reinterpret_cast<float2*>(red + (row0 * 2 + 0) * CH + cl) = make_float2(gD.x, gD.y);
  *reinterpret_cast<float2*>(red + (row0 * 2 + 1) * CH + cl) = make_float2(gb.x, gb.y);
  __syncthreads();
  for (int i = tid; i < 2 * CH; i += kThr) {
    const int k = c0 + i % CH;
    if (k >= a.C) continue;
    float s = 0.f;
    for (int r = 0; r < S::kStep; ++r) s += red[(r * 2 + i / CH) * CH + i % CH];
    a.part_d[(((int64_t)b * a.nseg + seg) * 2 + i / CH) * a.C + k] = s;
  }
}

// The sums over CTAs, in one launch (as three 14 us more at 2 x 1024 x 1024): gB and gC, the channel
// slices' partial rows in slice order, in the tensors' type; then gA, and gD and
// gbias, over sequences and segments.
struct ScanReduceArgs {
  const float* bc;  // [slices][rows][2][N]
  int slices, N;
  int64_t rows;
  void *gB, *gC;
  int64_t bc_blocks, a_blocks;  // CTAs of the first two parts
  ColSumArgs a, d;
};
constexpr int kScanReduceThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kScanReduceThreads) scan_reduce_kernel(ScanReduceArgs r) {
  if (blockIdx.x >= r.bc_blocks) {
    const int64_t block = blockIdx.x - r.bc_blocks;
    column_sums<kScanReduceThreads / 32>(block < r.a_blocks ? r.a : r.d, block < r.a_blocks ? block : block - r.a_blocks);
    return;
  }
  const int64_t i = (int64_t)blockIdx.x * kScanReduceThreads + threadIdx.x, width = r.rows * 2 * r.N;
  if (i >= width) return;
  float s = 0.f;
#pragma unroll 8
  for (int k = 0; k < r.slices; ++k) s += r.bc[k * width + i];
  const int64_t row = i / (2 * r.N);
  const int j = (int)(i - row * 2 * r.N);
  T* to = static_cast<T*>(j < r.N ? r.gB : r.gC);
  to[row * r.N + (j < r.N ? j : j - r.N)] = Pair<T>::from_float(s);
}

// One token: x, dt, z [B][C] and B, C [B][N]; the state is updated in place. LPC
// lanes share a channel, four states each, so a warp reads and writes 512 contiguous
// bytes of the state, which is nearly all the traffic there is. The lanes take LPC
// sequences together: each works out one sequence's step (its softplus and its gate)
// and hands it to the others.
constexpr int kScanStepThreads = 128;
template <typename T, int LPC>
__global__ void __launch_bounds__(kScanStepThreads) scan_step_kernel(ScanArgs a) {
  constexpr int kChannels = kScanStepThreads / LPC;
  const int q = threadIdx.x % LPC, b0 = blockIdx.x / a.cblocks * LPC;
  const int c0 = blockIdx.x % a.cblocks * kChannels + threadIdx.x / LPC;
  const bool mine = c0 < a.C;
  const int c = mine ? c0 : a.C - 1, own = min(b0 + q, a.B - 1), rows = min(LPC, a.B - b0);
  float* hp = a.h_last + ((int64_t)b0 * a.C + c) * a.N;
  const int64_t pitch = (int64_t)a.C * a.N;
  constexpr int kAhead = LPC < 4 ? LPC : 4;  // sequences whose states are under way at a time
  States<4> A2 = States<4>::load(a.A + (int64_t)c * a.N, 4 * q, a.N, a.wide_n);
  const float x = Pair<T>::scalar(static_cast<const T*>(a.x)[own * a.x_sb + c]);
  const float raw = Pair<T>::scalar(static_cast<const T*>(a.dt)[own * a.dt_sb + c]);
  const float z = a.z ? Pair<T>::scalar(static_cast<const T*>(a.z)[own * a.z_sb + c]) : 0.f;
  const float D = a.D ? a.D[c] : 0.f, bias = a.bias ? a.bias[c] : 0.f;
  float y[LPC];
  f2 d, w;
  A2.scale(kL2E);
#pragma unroll
  for (int r0 = 0; r0 < LPC; r0 += kAhead) {
    States<4> h[kAhead];
    Vec<T, 4> rB[kAhead], rC[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int r = r0 + i;
      h[i] = States<4>::zero();
      rB[i] = rC[i] = Vec<T, 4>::zero();
      if (r < rows) {
        h[i] = States<4>::load(hp + r * pitch, 4 * q, a.N, a.wide_n);
        rB[i] = load_bc(static_cast<const T*>(a.Bm) + (b0 + r) * a.b_sb, 4 * q, a.N, true, a.wide_bc);
        rC[i] = load_bc(static_cast<const T*>(a.Cm) + (b0 + r) * a.c_sb, 4 * q, a.N, true, a.wide_bc);
      }
    }
    if (r0 == 0) {
      d = scan_delta(splat(raw + bias), a.softplus);
      w = mul2(d, splat(x));
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int r = r0 + i;
      const f2 dr = splat(__shfl_sync(kFull, d.x, r, LPC)), wr = splat(__shfl_sync(kFull, w.x, r, LPC));
      float fB[4], fC[4];
      rB[i].get(fB);
      rC[i].get(fC);
      f2 v{0.f, 0.f};
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        h[i].p[n] = fma2(decay2(A2.p[n], dr), h[i].p[n], mul2(f2{fB[2 * n], fB[2 * n + 1]}, wr));
        v = fma2(h[i].p[n], f2{fC[2 * n], fC[2 * n + 1]}, v);
      }
      y[r] = v.x + v.y;
      if (mine && r < rows) h[i].store(hp + r * pitch, 4 * q, a.N, a.wide_n);
    }
  }
  reduce_scatter<LPC, LPC, 1>(y);
  if (!mine || q >= rows) return;
  float s = fmaf(D, x, y[0]);
  if (a.z) s *= z * sigmoid1<T>(z);
  static_cast<T*>(a.out)[(int64_t)own * a.C + c] = Pair<T>::from_float(s);
}

}  // namespace wkv
