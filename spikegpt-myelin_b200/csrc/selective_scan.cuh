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
constexpr int kScanCkpt = 16;  // steps between the states the forward keeps for the backward

struct ScanArgs {
  const void *x, *dt, *Bm, *Cm, *z, *gout;
  const float *A, *D, *bias;  // [C][N], [C] or null, [C] or null
  const float* h0;            // [B][C][N] or null
  const int* lengths;         // [B] or null
  void* out;                  // [B][T][C]
  float* h_last;              // [B][C][N] or null
  float* ckpt;                // [B][ceil(T / kScanCkpt)][C][N] or null: the state before each group of steps
  // backward
  const float* gh_last;  // [B][C][N] or null
  void *gx, *gdt, *gz;   // [B][T][C]
  float* gh0;            // [B][C][N] or null
  float* part_bc;        // [slices][B][T][2][N]
  float* part_a;         // [B][C][N]
  float* part_d;         // [B][2][C]: gD, gbias
  int64_t x_sb, x_st, dt_sb, dt_st, z_sb, z_st, b_sb, b_st, c_sb, c_st, g_sb, g_st;
  int B, T, C, N;
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

template <typename T, int NP>
__global__ void __launch_bounds__(32) scan_fwd_kernel(ScanArgs a) {
  const int blocks = (a.C + 31) / 32;
  const int b = blockIdx.x / blocks, c = blockIdx.x % blocks * 32 + threadIdx.x;
  if (c >= a.C) return;
  const int len = scan_length(a, b);
  const int64_t hc = ((int64_t)b * a.C + c) * a.N;
  float A[NP], h[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    A[n] = n < a.N ? a.A[(int64_t)c * a.N + n] * kL2E : 0.f;
    h[n] = n < a.N && a.h0 ? a.h0[hc + n] : 0.f;
  }
  const float D = a.D ? a.D[c] : 0.f, bias = a.bias ? a.bias[c] : 0.f;
  for (int t = 0; t < a.T; ++t) {
    if (a.ckpt && t % kScanCkpt == 0) {
      float* p = a.ckpt + (((int64_t)b * ((a.T + kScanCkpt - 1) / kScanCkpt) + t / kScanCkpt) * a.C + c) * a.N;
#pragma unroll
      for (int n = 0; n < NP; ++n)
        if (n < a.N) p[n] = h[n];
    }
    T* out = static_cast<T*>(a.out) + ((int64_t)b * a.T + t) * a.C + c;
    if (t >= len) {
      *out = Pair<T>::from_float(0.f);
      continue;
    }
    const float x = Pair<T>::scalar(static_cast<const T*>(a.x)[b * a.x_sb + t * a.x_st + c]);
    const float d =
        scan_delta(Pair<T>::scalar(static_cast<const T*>(a.dt)[b * a.dt_sb + t * a.dt_st + c]) + bias, a.softplus);
    const T* Bt = static_cast<const T*>(a.Bm) + b * a.b_sb + t * a.b_st;
    const T* Ct = static_cast<const T*>(a.Cm) + b * a.c_sb + t * a.c_st;
    float y = D * x;
    const float dx = d * x;
#pragma unroll
    for (int n = 0; n < NP; ++n)
      if (n < a.N) {
        h[n] = fmaf(ex2(d * A[n]), h[n], dx * Pair<T>::scalar(Bt[n]));
        y = fmaf(h[n], Pair<T>::scalar(Ct[n]), y);
      }
    if (a.z) {
      const float z = Pair<T>::scalar(static_cast<const T*>(a.z)[b * a.z_sb + t * a.z_st + c]);
      y *= z * sigmoid1(z);
    }
    *out = Pair<T>::from_float(y);
  }
  if (a.h_last)
#pragma unroll
    for (int n = 0; n < NP; ++n)
      if (n < a.N) a.h_last[hc + n] = h[n];
}

__device__ __forceinline__ float lane_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

template <typename T, int NP>
__global__ void __launch_bounds__(32) scan_bwd_kernel(ScanArgs a) {
  const int blocks = (a.C + 31) / 32;
  const int b = blockIdx.x / blocks, slice = blockIdx.x % blocks, c0 = slice * 32 + threadIdx.x;
  const bool live = c0 < a.C;
  const int c = live ? c0 : a.C - 1;
  const int len = scan_length(a, b);
  const int64_t hc = ((int64_t)b * a.C + c) * a.N;
  const int nck = (a.T + kScanCkpt - 1) / kScanCkpt;
  float A[NP], g[NP], gA[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    A[n] = n < a.N ? a.A[(int64_t)c * a.N + n] : 0.f;
    g[n] = n < a.N && a.gh_last ? a.gh_last[hc + n] : 0.f;
    gA[n] = 0.f;
  }
  const float D = a.D ? a.D[c] : 0.f, bias = a.bias ? a.bias[c] : 0.f;
  float gD = 0.f, gbias = 0.f;
  for (int ck = nck - 1; ck >= 0; --ck) {
    const float* p0 = a.ckpt + (((int64_t)b * nck + ck) * a.C + c) * a.N;
    for (int i = min(kScanCkpt, a.T - ck * kScanCkpt) - 1; i >= 0; --i) {
      const int t = ck * kScanCkpt + i;
      const int64_t at = ((int64_t)b * a.T + t) * a.C + c;
      float* pbc = a.part_bc + (((int64_t)slice * a.B + b) * a.T + t) * 2 * a.N;
      if (t >= len) {
        if (live) {
          static_cast<T*>(a.gx)[at] = Pair<T>::from_float(0.f);
          static_cast<T*>(a.gdt)[at] = Pair<T>::from_float(0.f);
          if (a.gz) static_cast<T*>(a.gz)[at] = Pair<T>::from_float(0.f);
        }
        for (int n = threadIdx.x; n < 2 * a.N; n += 32) pbc[n] = 0.f;
        continue;
      }
      // the state before step t, from the kept one
      float h[NP];
#pragma unroll
      for (int n = 0; n < NP; ++n) h[n] = n < a.N ? p0[n] : 0.f;
      float x = 0.f, d = 0.f, raw = 0.f, y = 0.f, along = 0.f, gd = 0.f, gy = 0.f, gout = 0.f, z = 0.f, sz = 1.f;
      for (int s = ck * kScanCkpt; s < t; ++s) {
        const float xs = Pair<T>::scalar(static_cast<const T*>(a.x)[b * a.x_sb + s * a.x_st + c]);
        const float ds = scan_delta(
            Pair<T>::scalar(static_cast<const T*>(a.dt)[b * a.dt_sb + s * a.dt_st + c]) + bias, a.softplus);
        const T* Bs = static_cast<const T*>(a.Bm) + b * a.b_sb + s * a.b_st;
#pragma unroll
        for (int n = 0; n < NP; ++n)
          if (n < a.N) h[n] = fmaf(ex2(ds * A[n] * kL2E), h[n], ds * xs * Pair<T>::scalar(Bs[n]));
      }
      x = Pair<T>::scalar(static_cast<const T*>(a.x)[b * a.x_sb + t * a.x_st + c]);
      raw = Pair<T>::scalar(static_cast<const T*>(a.dt)[b * a.dt_sb + t * a.dt_st + c]) + bias;
      d = scan_delta(raw, a.softplus);
      gout = Pair<T>::scalar(static_cast<const T*>(a.gout)[b * a.g_sb + t * a.g_st + c]);
      gy = gout;
      if (a.z) {
        z = Pair<T>::scalar(static_cast<const T*>(a.z)[b * a.z_sb + t * a.z_st + c]);
        sz = sigmoid1(z);
        gy = gout * z * sz;
      }
      y = D * x;
      const T* Bt = static_cast<const T*>(a.Bm) + b * a.b_sb + t * a.b_st;
      const T* Ct = static_cast<const T*>(a.Cm) + b * a.c_sb + t * a.c_st;
#pragma unroll
      for (int n = 0; n < NP; ++n)
        if (n < a.N) {
          const float Bv = Pair<T>::scalar(Bt[n]), Cv = Pair<T>::scalar(Ct[n]);
          const float decay = ex2(d * A[n] * kL2E), p = decay * h[n], hn = fmaf(d * x, Bv, p);
          g[n] = fmaf(Cv, gy, g[n]);
          y = fmaf(Cv, hn, y);
          along = fmaf(g[n], Bv, along);
          const float q = g[n] * p;
          gd = fmaf(A[n], q, gd);
          gA[n] = fmaf(d, q, gA[n]);
          const float sb = lane_sum(live ? g[n] * d * x : 0.f), sc = lane_sum(live ? gy * hn : 0.f);
          if (threadIdx.x == 0) {
            pbc[n] = sb;
            pbc[a.N + n] = sc;
          }
          g[n] *= decay;
        }
      gd = fmaf(x, along, gd) * scan_delta_slope(raw, a.softplus);
      gD = fmaf(gy, x, gD);
      gbias += gd;
      if (live) {
        static_cast<T*>(a.gx)[at] = Pair<T>::from_float(fmaf(d, along, D * gy));
        static_cast<T*>(a.gdt)[at] = Pair<T>::from_float(gd);
        if (a.gz) static_cast<T*>(a.gz)[at] = Pair<T>::from_float(gout * y * sz * fmaf(z, 1.f - sz, 1.f));
      }
    }
  }
  if (!live) return;
#pragma unroll
  for (int n = 0; n < NP; ++n)
    if (n < a.N) {
      a.part_a[hc + n] = gA[n];
      if (a.gh0) a.gh0[hc + n] = g[n];
    }
  a.part_d[((int64_t)b * 2 + 0) * a.C + c] = gD;
  a.part_d[((int64_t)b * 2 + 1) * a.C + c] = gbias;
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
template <typename T, int NP>
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
