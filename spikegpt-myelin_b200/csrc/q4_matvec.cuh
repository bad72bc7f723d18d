// Matrix-vector products with 4-bit weights and group scales (sm_100a).
//
//   y[m][n] = sum_k x[m][k] * scale[n][k / G] * (q[n][k] - zero[n][k / G]) (+ bias[n])
// q holds two weights a byte (even k in the low nibble), rows of ceil(K / 32) * 16
// bytes; scales bfloat16, zeros one byte each (8 without them). float32 sums.
//
// Bound by the bytes of the weights while the tokens are few, so the weights are
// read once for up to 16 tokens (8 in float32), by asynchronous copies kQ4Stages deep in a
// ring of the warp's own: 16 R rows x 128 inputs a stage. Decoding is a logical operation and a packed subtraction for two
// weights (and a shift for three of four): a nibble or-ed into the mantissa of a 16-bit
// float stands for 2^m + q, and less 2^m + zero it is exact. The products go to
// m16n8k16 tiles (A the weights, B the tokens), whose k order is free: the pairs that a
// word of eight nibbles gives, (0, 4), (1, 5), (2, 6), (3, 7), are taken as they come
// and x is paired the same way. Four lanes' words make 32 inputs, always of one group,
// whose sums are scaled in float32. float32 tokens enter as three bfloat16 terms
// (8 + 8 + 8 bits, exact) in three columns that are added at the end.
//
// The warps of a CTA are `wk` along the inputs (every wk-th 128 of them) by 8 / wk
// along the rows; the sums along the inputs meet in shared memory in warp order.
#pragma once

#include "row_io.cuh"

namespace wkv {

constexpr int kQ4Warps = 8;
constexpr int kQ4Chunk = 128;  // inputs of a stage
constexpr int kQ4Stages = 4;
constexpr int kQ4Row = 80;  // bytes of a staged row of weights: 64 and a shift of the banks

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
  int wide;    // rows of x are whole aligned 16-byte words
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

template <typename H>
struct Q4Math;
template <>
struct Q4Math<__nv_bfloat16> {
  static constexpr uint32_t kBase = 0x43004300u;  // 128: a nibble fills the mantissa's last bits
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <>
struct Q4Math<__half> {
  static constexpr uint32_t kBase = 0x64006400u;  // 1024
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// One tile of 16-bit tokens is read straight to registers a stage ahead (the rows of x
// are short and stay in the L1 cache); more tokens, and float32 ones, are staged.
template <typename T, int NT>
__host__ __device__ constexpr bool q4_staged() {
  return NT > 1 || sizeof(T) > 2;
}
// Bytes of a staged token's inputs: a shift of half the banks from token to token.
template <typename T>
__host__ __device__ constexpr int q4_token_bytes() {
  return kQ4Chunk * (int)sizeof(T) + 64;
}
template <typename T, int R, int NT>
__host__ __device__ constexpr int q4_stage_bytes(int tokens) {
  return R * 16 * kQ4Row + (q4_staged<T, NT>() ? tokens * q4_token_bytes<T>() : 0);
}
// A warp's ring and its scales and zeros (float, uint32_t) [2][16 R][4].
template <typename T, int R, int NT>
__host__ __device__ constexpr int q4_warp_bytes(int tokens) {
  return kQ4Stages * q4_stage_bytes<T, R, NT>(tokens) + 2 * R * 16 * 4 * 8;
}
template <int R, int NT>
constexpr int q4_sum_bytes() {
  return kQ4Warps * R * 16 * (8 * NT + 1) * 4;
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
template <typename T>
__device__ __forceinline__ void q4_inputs(const T* p, int term, uint32_t (&b)[4]) {
  if constexpr (sizeof(T) == 2) {
    q4_pairs(*reinterpret_cast<const uint4*>(p), b);
  } else {
    const float4 u = reinterpret_cast<const float4*>(p)[0], v = reinterpret_cast<const float4*>(p)[1];
    const float f[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
    uint32_t t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // the upper half of a float32 is its value cut to bfloat16
      const float h = __uint_as_float(__float_as_uint(f[i]) & 0xffff0000u);
      const float r = h == f[i] ? 0.f : f[i] - h;  // an infinity stays in the first term
      const float r2 = r - __uint_as_float(__float_as_uint(r) & 0xffff0000u);
      t[i] = __float_as_uint(term == 0 ? f[i] : term == 1 ? r : r2);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __byte_perm(t[i], t[i + 4], 0x7632);
  }
}

template <typename T, int R, int NT>
__global__ void __launch_bounds__(kQ4Warps * 32) q4_matvec_kernel(Q4Args a) {
  using H = typename Q4Type<T>::half;
  using Math = Q4Math<H>;
  constexpr int kTerms = Q4Type<T>::kTerms, kTok = q4_token_bytes<T>();
  extern __shared__ __align__(16) char smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, j = lane % 4;
  const int wk = warp % a.wk, wn = warp / a.wk;
  const int rows = 16 * R, cta_rows = rows * (kQ4Warps / a.wk);
  const int n0 = blockIdx.x * cta_rows + wn * rows, m0 = blockIdx.y * a.tokens;
  const int tokens = min(a.tokens, a.M - m0);
  const int stage_bytes = q4_stage_bytes<T, R, NT>(a.tokens);
  char* ring = smem + warp * q4_warp_bytes<T, R, NT>(a.tokens);
  float2* sz = reinterpret_cast<float2*>(ring + kQ4Stages * stage_bytes);
  const int chunks = (a.K + kQ4Chunk - 1) / kQ4Chunk;
  const int mine = n0 < a.N && chunks > wk ? (chunks - wk + a.wk - 1) / a.wk : 0;
  const T* x = static_cast<const T*>(a.x) + m0 * a.x_s;

  // where the lane reads: rows p * 8 + g, its quarter of each stage's inputs
  const uint8_t* pq[2 * R];
  const uint16_t* ps[2 * R];
  const uint8_t* pz[2 * R];
#pragma unroll
  for (int p = 0; p < 2 * R; ++p) {
    const int64_t row = min(n0 + p * 8 + g, a.N - 1);
    pq[p] = a.q + row * a.pitch + wk * (kQ4Chunk / 2) + j * 16;
    ps[p] = reinterpret_cast<const uint16_t*>(a.scale) + row * a.groups;
    pz[p] = a.zero ? a.zero + row * a.groups : nullptr;
  }
  const int last32 = (a.K - 1) / 32;  // the row's last 32 inputs
  auto issue = [&](int i) {
    if (i < mine) {
      const int k0 = (wk + i * a.wk) * kQ4Chunk;
      char* to = ring + i % kQ4Stages * stage_bytes;
      const bool on = k0 + j * 32 < a.K;
      const int64_t at = (int64_t)i * a.wk * (kQ4Chunk / 2);
#pragma unroll
      for (int p = 0; p < 2 * R; ++p)
        q4_copy(to + (p * 8 + g) * kQ4Row + j * 16, on ? pq[p] + at : a.q, on);
      if constexpr (q4_staged<T, NT>()) {
        char* tx = to + rows * kQ4Row;
        constexpr int kWords = kQ4Chunk * (int)sizeof(T) / 16, E = 16 / (int)sizeof(T);
        if (a.wide) {
          for (int p = lane; p < tokens * kWords; p += 32) {
            const int k = k0 + p % kWords * E;
            q4_copy(tx + p / kWords * kTok + p % kWords * 16, x + p / kWords * a.x_s + (k < a.K ? k : 0), k < a.K);
          }
        } else {
          for (int p = lane; p < tokens * kQ4Chunk; p += 32) {
            const int k = k0 + p % kQ4Chunk;
            reinterpret_cast<T*>(tx + p / kQ4Chunk * kTok)[p % kQ4Chunk] =
                k < a.K ? x[p / kQ4Chunk * a.x_s + k] : Pair<T>::from_float(0.f);
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // scales and zeros of the next stage, 32 inputs of a row each, and unstaged tokens
  uint16_t fs[2 * R];
  uint8_t fz[2 * R];
  uint4 fx[4];
  const bool token = g < tokens;  // the lane's column is a token (one tile of 16-bit tokens)
  const T* px = x + (token ? g * a.x_s : 0) + wk * kQ4Chunk + j * 8;
  auto fetch = [&](int i) {
    if (i >= mine) return;
    const int k32 = min((wk + i * a.wk) * 4 + j, last32), group = a.group_magic ? __umulhi(k32, a.group_magic) : k32;
#pragma unroll
    for (int p = 0; p < 2 * R; ++p) {
      fs[p] = ps[p][group];
      fz[p] = a.zero ? pz[p][group] : 8;
    }
    if constexpr (!q4_staged<T, NT>()) {
      const T* from = px + (int64_t)i * a.wk * kQ4Chunk;
      const int k0 = (wk + i * a.wk) * kQ4Chunk + j * 8;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int k = k0 + w * 32;
        fx[w] = make_uint4(0, 0, 0, 0);
        if (token && k < a.K) {
          if (a.wide) {
            fx[w] = *reinterpret_cast<const uint4*>(from + w * 32);
          } else {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(from + w * 32);
            uint32_t u[4];
#pragma unroll
            for (int n = 0; n < 4; ++n)
              u[n] = (k + 2 * n < a.K ? h[2 * n] : 0u) | (k + 2 * n + 1 < a.K ? (uint32_t)h[2 * n + 1] << 16 : 0u);
            fx[w] = make_uint4(u[0], u[1], u[2], u[3]);
          }
        }
      }
    }
  };
  auto keep = [&](int i) {
    if (i >= mine) return;
#pragma unroll
    for (int p = 0; p < 2 * R; ++p)
      sz[((i & 1) * rows + p * 8 + g) * 4 + j] =
          make_float2(__uint_as_float((uint32_t)fs[p] << 16), __uint_as_float(Math::kBase + fz[p] * 0x10001u));
  };

  float acc[R][NT][4];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[r][t][0] = acc[r][t][1] = acc[r][t][2] = acc[r][t][3] = 0.f;
  fetch(0);
#pragma unroll
  for (int i = 0; i < kQ4Stages - 1; ++i) issue(i);
  keep(0);
  for (int i = 0; i < mine; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kQ4Stages - 2) : "memory");
    __syncwarp();  // the stage and its scales are there, and every lane is done with the stage before
    issue(i + kQ4Stages - 1);
    const uint4 cx[4] = {fx[0], fx[1], fx[2], fx[3]};
    fetch(i + 1);
    const char* from = ring + i % kQ4Stages * stage_bytes;
    const float2* sc = sz + (i & 1) * rows * 4;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t b[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int column = t * 8 + g;
        if constexpr (!q4_staged<T, NT>())
          q4_pairs(cx[w], b[t]);
        else if (column < tokens * kTerms)
          q4_inputs(reinterpret_cast<const T*>(from + rows * kQ4Row + column / kTerms * kTok) + w * 32 + j * 8,
                    column % kTerms, b[t]);
        else
          b[t][0] = b[t][1] = b[t][2] = b[t][3] = 0;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int row = r * 16 + g;
        const uint32_t u = *reinterpret_cast<const uint32_t*>(from + row * kQ4Row + w * 16 + j * 4);
        const uint32_t v = *reinterpret_cast<const uint32_t*>(from + (row + 8) * kQ4Row + w * 16 + j * 4);
        const float2 su = sc[row * 4 + w], sv = sc[(row + 8) * 4 + w];
        uint32_t p[4], q[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          p[n] = Math::sub((u >> (4 * n) & 0x000f000fu) | Math::kBase, __float_as_uint(su.y));
          q[n] = Math::sub((v >> (4 * n) & 0x000f000fu) | Math::kBase, __float_as_uint(sv.y));
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          Math::mma(d, p[0], q[0], p[1], q[1], b[t][0], b[t][1]);
          Math::mma(d, p[2], q[2], p[3], q[3], b[t][2], b[t][3]);
          acc[r][t][0] = fmaf(su.x, d[0], acc[r][t][0]);
          acc[r][t][1] = fmaf(su.x, d[1], acc[r][t][1]);
          acc[r][t][2] = fmaf(sv.x, d[2], acc[r][t][2]);
          acc[r][t][3] = fmaf(sv.x, d[3], acc[r][t][3]);
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
  for (int i = threadIdx.x; i < cta_rows * tokens; i += kQ4Warps * 32) {
    const int row = i % cta_rows, token = i / cta_rows, n = blockIdx.x * cta_rows + row;
    if (n >= a.N) continue;
    float s = 0.f;
    for (int k = 0; k < a.wk; ++k)
#pragma unroll
      for (int t = 0; t < kTerms; ++t)
        s += sum[((row / rows * a.wk + k) * rows + row % rows) * kPitch + token * kTerms + t];
    if (a.bias) s += a.bias[n];
    static_cast<T*>(a.y)[(int64_t)(m0 + token) * a.N + n] = Pair<T>::from_float(s);
  }
}

}  // namespace wkv
