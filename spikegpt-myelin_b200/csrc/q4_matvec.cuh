// Matrix-vector products with 4-bit weights and group scales (sm_100a).
//
//   y[m][n] = sum_k x[m][k] * scale[n][k / G] * (q[n][k] - zero[n][k / G]) (+ bias[n])
// q holds two weights a byte (even k in the low nibble), rows of ceil(K / 32) * 16
// bytes; scales bfloat16, zeros one byte each (8 without them; any value). float32 sums.
//
// The least it can do is to read the weights once, for up to 16 tokens (8 in float32):
// they come by asynchronous copies kQ4Stages deep in a ring of the warp's own, 16 R rows
// x 128 inputs a stage. Decoding is a logical operation and a packed subtraction for two
// weights (and a shift for three of four): a nibble or-ed into the mantissa of a 16-bit
// float stands for 2^m + q, and less 2^m + zero it is exact (in bfloat16 up to a zero of
// 127; for the others see q4_far_zeros). The products go to
// m16n8k16 tiles (A the weights, B the tokens), whose k order is free: the pairs that a
// word of eight nibbles gives, (0, 4), (1, 5), (2, 6), (3, 7), are taken as they come
// and x is paired the same way. Four lanes' words make 32 inputs (64 or 128 where the
// group allows), always of one group, whose sums are scaled in float32. float32 tokens
// enter as three bfloat16 terms (8 + 8 + 8 bits, exact) in three columns that are added
// at the end.
//
// Measured: 6 x 8192 x 16384 bfloat16, groups of 128: 28.7 us, 2.5 TB/s of weights; 1 x 768
// x 50257, groups of 64: 10.3 us. What bounds it is latency: 512 CTAs of four warps, 13
// warps an SM, issue in 51 % of their slots and keep the integer pipe 54 % busy (about 1.4
// integer and packed operations a weight), and wait most (1.6 warps an issue) for global
// loads, which the scales, zero points and tokens are, one stage ahead, next to the
// weights' ring. 64 rows a warp and six stages were no faster.
//
// The warps of a CTA are `wk` along the inputs (every wk-th 128 of them) by the
// others along the rows; the sums along the inputs meet in shared memory in warp order.
#pragma once

#include "row_io.cuh"

namespace wkv {

constexpr int kQ4MaxWarps = 8;  // of a CTA: 4 or 8
constexpr int kQ4Chunk = 128;  // inputs of a stage
constexpr int kQ4Stages = 4;
// Bytes of a staged row of weights, 64 and a shift: lanes read 4 GW bytes of eight rows
// side by side, and no two rows of an access may meet in a bank.
__host__ __device__ constexpr int q4_row_bytes(int GW) { return GW == 4 ? 64 : GW == 2 ? 96 : 80; }

struct Q4Args {
  const void* x;  // [M][K]
  const uint8_t* q;
  const __nv_bfloat16* scale;
  const uint8_t* zero;  // or null
  const float* bias;    // [N] or null
  void* y;              // [M][N]
  int64_t x_s;
  int M, N, K, G, groups, pitch;
  int tokens;  // of a CTA
  int wk;      // warps along the inputs
  uint32_t group_magic;  // the upper word of its product with k / 32 is the group (0: k / 32 is)
};

// Columns that a token takes, and the 16-bit type the products run in.
template <typename T>
struct Q4Type {
  using half = T;
  static constexpr int kTerms = 1;
};
template <>
struct Q4Type<float> {
  using half = __nv_bfloat16;
  static constexpr int kTerms = 3;
};

// Packed arithmetic of the 16-bit type: kBase or-ed to a nibble is 2^m + nibble.
template <typename H>
struct Q4Math;
template <>
struct Q4Math<__nv_bfloat16> {
  static constexpr uint32_t kBase = 0x43004300u;  // 128: a nibble fills the mantissa's last bits
  static constexpr int kMostZero = 127;           // 128 + zero keeps the exponent
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
};
template <>
struct Q4Math<__half> {
  static constexpr uint32_t kBase = 0x64006400u;  // 1024
  static constexpr int kMostZero = 255;           // any byte
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
};

// (a & mask) | base: one operation with both constants in registers.
__device__ __forceinline__ uint32_t q4_nibbles(uint32_t a, uint32_t mask, uint32_t base) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(a), "r"(mask), "r"(base));
  return d;
}

// A stage's inputs come to registers a stage ahead. One tile of 16-bit tokens goes from
// there to the products as each lane reads it (its rows of x are short and stay in the
// L1 cache: 31 us for 8 x 8192 x 16384, through shared memory 39); more tokens (whose
// registers would not do) and float32 ones (whose values are split once a warp) go
// through shared memory.
template <typename T, int NT>
__host__ __device__ constexpr bool q4_direct() {
  return NT == 1 && sizeof(T) == 2;
}
// Bytes of a column's inputs of a stage: a shift of half the banks from one to the next.
constexpr int kQ4ColumnBytes = kQ4Chunk * 2 + 64;
template <int R, int GW>
__host__ __device__ constexpr int q4_stage_bytes() {
  return R * 16 * q4_row_bytes(GW);
}
// A warp's ring, its scales and zeros (float, uint32_t) [2][16 R][4 / GW] and its
// columns' inputs.
template <typename T, int R, int NT, int GW>
__host__ __device__ constexpr int q4_warp_bytes(int tokens) {
  return kQ4Stages * q4_stage_bytes<R, GW>() + 2 * R * 16 * (4 / GW) * 8 +
         (q4_direct<T, NT>() ? 0 : Q4Type<T>::kTerms * tokens * kQ4ColumnBytes);
}
template <int R, int NT>
constexpr int q4_sum_bytes(int warps) {
  return warps * R * 16 * (8 * NT + 1) * 4;
}

__device__ __forceinline__ void q4_copy(void* dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0)
               : "memory");
}

// B operands of a column's eight inputs: word i holds inputs i and i + 4.
__device__ __forceinline__ void q4_pairs(uint4 u, uint32_t (&b)[4]) {
  b[0] = __byte_perm(u.x, u.z, 0x5410);
  b[1] = __byte_perm(u.x, u.z, 0x7632);
  b[2] = __byte_perm(u.y, u.w, 0x5410);
  b[3] = __byte_perm(u.y, u.w, 0x7632);
}
// Four float32 values as three bfloat16 terms of 8 bits each (the upper half of a
// float32 is its value cut to bfloat16), exactly; term e's four words side by side.
__device__ __forceinline__ void q4_split(uint4 v, uint2 (&t)[3]) {
  const float f[4] = {__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
  uint32_t u[3][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float h = __uint_as_float(__float_as_uint(f[i]) & 0xffff0000u);
    const float r = h == f[i] ? 0.f : f[i] - h;  // an infinity stays in the first term
    u[0][i] = __float_as_uint(f[i]);
    u[1][i] = __float_as_uint(r);
    u[2][i] = __float_as_uint(r - __uint_as_float(__float_as_uint(r) & 0xffff0000u));
  }
#pragma unroll
  for (int e = 0; e < 3; ++e)
    t[e] = make_uint2(__byte_perm(u[e][0], u[e][1], 0x7632), __byte_perm(u[e][2], u[e][3], 0x7632));
}

// The product of token m and row n once more, if one of the row's zero points has no room
// next to kBase. Zero points of 4-bit weights are 0 to 15, so this is made to cost the
// usual path nothing, not for speed.
template <typename T>
__device__ __forceinline__ void q4_far_zeros(const Q4Args& a, int m, int n, int most) {
  const uint8_t *zero = a.zero + (int64_t)n * a.groups, *q = a.q + (int64_t)n * a.pitch;
  const T* x = static_cast<const T*>(a.x) + m * a.x_s;
  bool far = false;
  for (int g = 0; g < a.groups; ++g) far |= zero[g] > most;
  if (!far) return;
  float y = a.bias ? a.bias[n] : 0.f;
  for (int g = 0, k = 0; g < a.groups; ++g) {
    float sum = 0.f;
    for (const int end = k + min(a.K - k, a.G); k < end; ++k)
      sum = fmaf((float)((q[k >> 1] >> (k & 1) * 4 & 15) - zero[g]), Pair<T>::scalar(x[k]), sum);
    y = fmaf(__bfloat162float(a.scale[(int64_t)n * a.groups + g]), sum, y);
  }
  static_cast<T*>(a.y)[(int64_t)m * a.N + n] = Pair<T>::from_float(y);
}

// GW: words of eight weights that a lane takes side by side, 1, 2 or 4: the four lanes'
// 32, 64 or 128 inputs lie in one group, and are scaled at a time.
// kWide: rows of x are whole aligned 16-byte words (8-byte ones are enough for more than
// one tile of 16-bit tokens).
template <typename T, int R, int NT, int GW, bool kWide>
__global__ void __launch_bounds__(kQ4MaxWarps * 32, 2) q4_matvec_kernel(Q4Args a) {
  using H = typename Q4Type<T>::half;
  using Math = Q4Math<H>;
  constexpr int kTerms = Q4Type<T>::kTerms, kTok = kQ4ColumnBytes, kRow = q4_row_bytes(GW);
  constexpr int kSpans = 4 / GW, kEntries = 16 * R * kSpans, kPer = (kEntries + 31) / 32;
  constexpr bool kDirect = q4_direct<T, NT>();
  constexpr int kFetches = kDirect ? 4 : 8 * NT / kTerms;
  extern __shared__ __align__(16) char smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, j = lane % 4;
  const int wk = warp % a.wk, wn = warp / a.wk;
  constexpr int rows = 16 * R;
  const int cta_rows = rows * ((int)blockDim.x / 32 / a.wk);
  const int n0 = blockIdx.x * cta_rows + wn * rows, m0 = blockIdx.y * a.tokens;
  const int tokens = min(a.tokens, a.M - m0);
  constexpr int stage_bytes = q4_stage_bytes<R, GW>();
  char* ring = smem + warp * q4_warp_bytes<T, R, NT, GW>(a.tokens);
  float2* sz = reinterpret_cast<float2*>(ring + kQ4Stages * stage_bytes);
  char* columns = reinterpret_cast<char*>(sz + 2 * kEntries);
  const int chunks = (a.K + kQ4Chunk - 1) / kQ4Chunk;
  const int mine = n0 < a.N && chunks > wk ? (chunks - wk + a.wk - 1) / a.wk : 0;
  const T* x = static_cast<const T*>(a.x) + m0 * a.x_s;

  // What the lane copies: its quarter of each stage's inputs of rows p * 8 + g. Rows past N
  // stand in for the last one; inputs past K are zeros.
  const uint8_t* pq[2 * R];
#pragma unroll
  for (int p = 0; p < 2 * R; ++p) pq[p] = a.q + (int64_t)min(n0 + p * 8 + g, a.N - 1) * a.pitch;
  int copy_k = wk * kQ4Chunk + j * 32, copy_stage = 0;
  auto issue = [&](int i) {
    if (i < mine) {
      char* to = ring + copy_stage * stage_bytes;
      const bool on = copy_k < a.K;
      const int off = on ? copy_k >> 1 : 0;
#pragma unroll
      for (int p = 0; p < 2 * R; ++p) q4_copy(to + (p * 8 + g) * kRow + j * 16, pq[p] + off, on);
      copy_k += a.wk * kQ4Chunk;
      copy_stage = copy_stage + 1 == kQ4Stages ? 0 : copy_stage + 1;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // The next stage's scales and zeros, kPer (row, span) pairs a lane, and its inputs: the
  // lane's column of eight at a time (direct), or four of each token.
  uint16_t fs[kPer];
  uint8_t fz[kPer];
  Vec<T, kDirect ? 8 : 4> fx[kFetches];
  const T* px = x + (g < tokens ? g * a.x_s : 0);  // columns past the tokens are not written
  int fetch_k = wk * kQ4Chunk;
  auto fetch = [&]() {  // past the last stage: of inputs that exist, and are not used
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const int entry = p * 32 + lane, row = min(n0 + entry / kSpans % rows, a.N - 1);
      const int k32 = (min(fetch_k + entry % kSpans * (32 * GW), a.K - 1)) >> 5;
      const int64_t at = (int64_t)row * a.groups + (a.group_magic ? __umulhi(k32, a.group_magic) : k32);
      fs[p] = reinterpret_cast<const uint16_t*>(a.scale)[at];
      fz[p] = a.zero ? a.zero[at] : 8;
    }
    if constexpr (kDirect) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int k = fetch_k + j * 8 * GW + w / GW * (32 * GW) + w % GW * 8;
        if constexpr (kWide) {
          fx[w] = Vec<T, 8>::load(px + min(k, a.K - 8));
        } else {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(px) + k;
          uint32_t u[4];
#pragma unroll
          for (int n = 0; n < 4; ++n)
            u[n] = (k + 2 * n < a.K ? h[2 * n] : 0u) | (k + 2 * n + 1 < a.K ? (uint32_t)h[2 * n + 1] << 16 : 0u);
          fx[w].w = make_uint4(u[0], u[1], u[2], u[3]);
        }
      }
      if (kWide && fetch_k + kQ4Chunk > a.K) {
#pragma unroll
        for (int w = 0; w < 4; ++w)
          if (fetch_k + j * 8 * GW + w / GW * (32 * GW) + w % GW * 8 >= a.K) fx[w] = Vec<T, 8>::zero();
      }
    } else {
      const int k = fetch_k + lane * 4;
#pragma unroll
      for (int t = 0; t < kFetches; ++t) {
        fx[t] = Vec<T, 4>::zero();
        if (t < tokens && k < a.K) {
          const T* p = x + t * a.x_s + k;
          if constexpr (kWide) {
            fx[t] = Vec<T, 4>::load(p);
          } else {
#pragma unroll
            for (int n = 0; n < 4; ++n)
              if (k + n < a.K) fx[t].e[n] = p[n];
          }
        }
      }
    }
    fetch_k += a.wk * kQ4Chunk;
  };
  auto keep = [&](int i) {
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      if (fz[p] > Math::kMostZero) fs[p] = 0xffff;  // a NaN: the row is worked out again at the end
      if (kEntries % 32 == 0 || lane < kEntries)
        sz[(i & 1) * kEntries + p * 32 + lane] =
            make_float2(__uint_as_float((uint32_t)fs[p] << 16), __uint_as_float(Math::kBase + fz[p] * 0x10001u));
    }
  };

  float acc[R][NT][4];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[r][t][0] = acc[r][t][1] = acc[r][t][2] = acc[r][t][3] = 0.f;
  const float none[4] = {0.f, 0.f, 0.f, 0.f};
  uint32_t mask = 0x000f000fu, base = Math::kBase;
  asm volatile("" : "+r"(mask), "+r"(base));  // in registers: an instruction holds one constant
  if (mine > 0) fetch();
#pragma unroll
  for (int i = 0; i < kQ4Stages - 1; ++i) issue(i);
  if (mine > 0) keep(0);
  int stage = 0;
  for (int i = 0; i < mine; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kQ4Stages - 2) : "memory");
    __syncwarp();  // the stage and its scales are there, and every lane is done with the stage before
    issue(i + kQ4Stages - 1);
    uint32_t bx[4][4];  // direct operands: their words are free for the next stage's
    if constexpr (kDirect) {
#pragma unroll
      for (int w = 0; w < 4; ++w) q4_pairs(fx[w].w, bx[w]);
    } else {
#pragma unroll
      for (int t = 0; t < kFetches; ++t)
        if (t < tokens) {
          uint2 u[kTerms];
          if constexpr (kTerms == 1)
            u[0] = fx[t].w;
          else
            q4_split(fx[t].w, u);
#pragma unroll
          for (int e = 0; e < kTerms; ++e)
            *reinterpret_cast<uint2*>(columns + (kTerms * t + e) * kTok + lane * 8) = u[e];
        }
      __syncwarp();
    }
    fetch();
    const char* from = ring + stage * stage_bytes + g * kRow + j * 4 * GW;
    const char* tx = columns + j * 8 * GW * 2;
    const float2* sc = sz + (i & 1) * kEntries + g * kSpans;
    stage = stage + 1 == kQ4Stages ? 0 : stage + 1;
#pragma unroll
    for (int span = 0; span < kSpans; ++span) {
      uint32_t b[GW][NT][4];
#pragma unroll
      for (int w = 0; w < GW; ++w)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int column = t * 8 + g;
          if constexpr (kDirect) {
#pragma unroll
            for (int n = 0; n < 4; ++n) b[w][t][n] = bx[span * GW + w][n];
          } else if (column < tokens * kTerms)
            q4_pairs(*reinterpret_cast<const uint4*>(tx + column * kTok + (span * 32 * GW + w * 8) * 2), b[w][t]);
          else
            b[w][t][0] = b[w][t][1] = b[w][t][2] = b[w][t][3] = 0;
        }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        using Words = Vec<uint32_t, GW>;
        const Words u = Words::load(reinterpret_cast<const uint32_t*>(from + r * 16 * kRow + span * 16 * GW));
        const Words v = Words::load(reinterpret_cast<const uint32_t*>(from + (r * 16 + 8) * kRow + span * 16 * GW));
        const float2 su = sc[r * 16 * kSpans + span], sv = sc[(r * 16 + 8) * kSpans + span];
        float d[NT][4];
#pragma unroll
        for (int w = 0; w < GW; ++w) {
          uint32_t p[4], q[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            p[n] = Math::sub(q4_nibbles(u.e[w] >> (4 * n), mask, base), __float_as_uint(su.y));
            q[n] = Math::sub(q4_nibbles(v.e[w] >> (4 * n), mask, base), __float_as_uint(sv.y));
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if (w == 0)
              Math::mma(d[t], p[0], q[0], p[1], q[1], b[w][t][0], b[w][t][1], none);
            else
              Math::mma(d[t], p[0], q[0], p[1], q[1], b[w][t][0], b[w][t][1], d[t]);
            Math::mma(d[t], p[2], q[2], p[3], q[3], b[w][t][2], b[w][t][3], d[t]);
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          acc[r][t][0] = fmaf(su.x, d[t][0], acc[r][t][0]);
          acc[r][t][1] = fmaf(su.x, d[t][1], acc[r][t][1]);
          acc[r][t][2] = fmaf(sv.x, d[t][2], acc[r][t][2]);
          acc[r][t][3] = fmaf(sv.x, d[t][3], acc[r][t][3]);
        }
      }
    }
    keep(i + 1);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();  // the rings become the sums [warp][rows][8 NT + 1]
  float* sum = reinterpret_cast<float*>(smem);
  constexpr int kPitch = 8 * NT + 1;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sum[(warp * rows + r * 16 + g + i / 2 * 8) * kPitch + t * 8 + j * 2 + i % 2] = acc[r][t][i];
  __syncthreads();
  bool bad = false;
  for (int i = threadIdx.x; i < cta_rows * tokens; i += blockDim.x) {
    const int row = i % cta_rows, t = i / cta_rows, n = blockIdx.x * cta_rows + row;
    if (n >= a.N) continue;
    float s = 0.f;
    for (int k = 0; k < a.wk; ++k)
#pragma unroll
      for (int e = 0; e < kTerms; ++e)
        s += sum[((row / rows * a.wk + k) * rows + row % rows) * kPitch + t * kTerms + e];
    bad |= isnan(s);
    if (a.bias) s += a.bias[n];
    static_cast<T*>(a.y)[(int64_t)(m0 + t) * a.N + n] = Pair<T>::from_float(s);
  }
  // the rows with a NaN for a scale, in a loop of their own: the one above is pipelined
  if constexpr (Math::kMostZero < 255) {
    if (!bad || a.zero == nullptr) return;
    for (int i = threadIdx.x; i < cta_rows * tokens; i += blockDim.x) {
      const int t = i / cta_rows, n = blockIdx.x * cta_rows + i % cta_rows;
      if (n < a.N) q4_far_zeros<T>(a, m0 + t, n, Math::kMostZero);
    }
  }
}

}  // namespace wkv
