// C ABI of the selective-mixer operators (declared in include/spikegpt_wkv.h):
// the short causal convolution, the selective scan, their single-token steps,
// layer norm, and the matrix-vector product with 4-bit weights. Argument checks,
// workspace layout, the choice of kernel variants and the launches; every entry
// point is asynchronous on the caller's stream and allocates nothing.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <initializer_list>
#include <type_traits>

#include "capi_host.cuh"
#include "causal_conv.cuh"
#include "layer_norm.cuh"
#include "q4_matvec.cuh"
#include "selective_scan.cuh"

namespace {

using namespace wkv;
using namespace wkv_host;

constexpr int64_t kMaxDim = 1ll << 30;
constexpr int kScanMaxSegments = 64;
constexpr int kScanMinSegment = 32;

// Calls f with a value of the dtype's element type.
template <class F>
int with_type(int dtype, F&& f) {
  switch (dtype) {
    case WKV_DTYPE_F32: return f(float{});
    case WKV_DTYPE_BF16: return f(__nv_bfloat16{});
    default: return f(__half{});
  }
}

int check_type(int dtype) {
  return dtype_size(dtype) == 0 ? fail(WKV_ERR_INVALID_ARGUMENT, "unknown dtype code %d", dtype) : WKV_OK;
}

int check_sizes(std::initializer_list<int64_t> sizes) {
  for (int64_t v : sizes) {
    if (v < 0) return fail(WKV_ERR_INVALID_ARGUMENT, "negative size %lld", (long long)v);
    if (v > kMaxDim) return fail(WKV_ERR_INVALID_ARGUMENT, "size out of range: %lld", (long long)v);
  }
  return WKV_OK;
}

int check_pointers(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (!p) return fail(WKV_ERR_INVALID_ARGUMENT, "null pointer");
  return WKV_OK;
}

// The largest number of adjacent elements (a power of two up to `most`) that
// every pointer and row pitch lets a thread move as one aligned word.
int vector_width(size_t es, int most, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> pitches) {
  int v = most;
  for (const void* p : ptrs)
    while (v > 1 && reinterpret_cast<uintptr_t>(p) % (v * es) != 0) v /= 2;
  for (int64_t s : pitches)
    while (v > 1 && s % v != 0) v /= 2;
  return v;
}

int launch_column_sums(ColSumArgs a, cudaStream_t st) {
  const int64_t width = a.C * a.blocks;
  if (width == 0) return WKV_OK;
  launch(K_COL_SUM, st, [&] { column_sum_kernel<<<(unsigned)((width + 31) / 32), 1024, 0, st>>>(a); });
  return launched("column sum launch");
}

// ----------------------------------------------------------- causal convolution

int conv_check(int dtype, int64_t B, int64_t T, int64_t C, int W) {
  if (int rc = check_type(dtype)) return rc;
  if (int rc = check_sizes({B, T, C})) return rc;
  if (W < 1 || W > kConvMaxTaps)
    return fail(WKV_ERR_INVALID_ARGUMENT, "the convolution's width must be 1..%d, got %d", kConvMaxTaps, W);
  if (B > 0 && C > 0 && ((T + kConvSteps - 1) / kConvSteps + 1) * ((C + kConvThreads - 1) / kConvThreads) > INT_MAX / B)
    return fail(WKV_ERR_INVALID_ARGUMENT, "sizes out of range B=%lld T=%lld C=%lld", (long long)B, (long long)T,
                (long long)C);
  return WKV_OK;
}

int conv_chunks(int64_t T) { return (int)std::max<int64_t>(1, (T + kConvSteps - 1) / kConvSteps); }

// Calls f(element, integral constant V, integral constant W).
template <class F>
int conv_dispatch(int dtype, int V, int W, F&& f) {
  return with_type(dtype, [&](auto e) {
    using T = decltype(e);
    auto taps = [&](auto v) {
      switch (W) {
        case 1: return f(e, v, std::integral_constant<int, 1>{});
        case 2: return f(e, v, std::integral_constant<int, 2>{});
        case 3: return f(e, v, std::integral_constant<int, 3>{});
        default: return f(e, v, std::integral_constant<int, 4>{});
      }
    };
    if (V >= 4) return taps(std::integral_constant<int, 4>{});
    if (V >= 2) return taps(std::integral_constant<int, 2>{});
    return taps(std::integral_constant<int, 1>{});
  });
}

ConvArgs conv_args(const void* x, const float* w, const float* bias, const void* front, const int* lengths,
                   int64_t B, int64_t T, int64_t C, int64_t x_sb, int64_t x_st, int silu) {
  ConvArgs a{};
  a.x = x;
  a.w = w;
  a.bias = bias;
  a.front = front;
  a.lengths = lengths;
  a.x_sb = x_sb;
  a.x_st = x_st;
  a.B = (int)B;
  a.T = (int)T;
  a.C = (int)C;
  a.chunks = conv_chunks(T);
  a.silu = silu;
  return a;
}

// ---------------------------------------------------------------- layer norm

int norm_check(int dtype, int64_t rows, int64_t C) {
  if (int rc = check_type(dtype)) return rc;
  if (int rc = check_sizes({rows, C})) return rc;
  if (C > kNormMaxC) return fail(WKV_ERR_INVALID_ARGUMENT, "layer norm takes rows of up to %d, got %lld", kNormMaxC, (long long)C);
  return WKV_OK;
}

// Threads of a row and of a CTA (several rows' where they are short), and CTAs: about
// what is resident at a time, so that every CTA walks several rows. (512 threads an SM, and
// one CTA where it is larger: 8192 x 16384 bfloat16 backward 368 us, with a CTA on every
// other SM 677.)
struct NormPlan {
  int span, threads, grid;
};
NormPlan norm_plan(int64_t rows, int64_t C) {
  NormPlan p{32, 256, 0};
  while (p.span * kNormValues < C) p.span *= 2;
  p.threads = std::max(p.threads, p.span);
  const int64_t teams = p.threads / p.span;
  p.grid = (int)std::min<int64_t>((rows + teams - 1) / teams, (int64_t)sm_count() * std::max(1, 512 / p.threads));
  return p;
}

// Calls f(element, V, threads): the widest words of x, y (and their gradients) that all
// rows allow. The parameters are float32 [C]: words of four where x has words of 16 bytes.
template <class F>
int norm_dispatch(int dtype, int threads, std::initializer_list<const void*> ptrs,
                  std::initializer_list<int64_t> pitches, F&& f) {
  const int es = (int)dtype_size(dtype), v = vector_width(es, 16 / es, ptrs, pitches);
  return with_type(dtype, [&](auto e) {
    constexpr int kMost = 16 / (int)sizeof(e);
    auto sized = [&](auto n) {
      switch (threads) {
        case 256: return f(e, n, std::integral_constant<int, 256>{});
        case 512: return f(e, n, std::integral_constant<int, 512>{});
        default: return f(e, n, std::integral_constant<int, 1024>{});
      }
    };
    if (v == kMost) return sized(std::integral_constant<int, kMost>{});
    if (v >= 2) return sized(std::integral_constant<int, 2>{});
    return sized(std::integral_constant<int, 1>{});
  });
}

// --------------------------------------------------------------------- scan

int scan_check(int dtype, int64_t B, int64_t T, int64_t C, int64_t N) {
  if (int rc = check_type(dtype)) return rc;
  if (int rc = check_sizes({B, T, C, N})) return rc;
  if (N < 1 || N > kScanMaxN)
    return fail(WKV_ERR_INVALID_ARGUMENT, "the state size must be 1..%d, got %lld", kScanMaxN, (long long)N);
  if (T > (1 << 23) || (B > 0 && ((C + 7) / 8 * kScanMaxSegments > INT_MAX / B || T > INT_MAX / B)))
    return fail(WKV_ERR_INVALID_ARGUMENT, "sizes out of range B=%lld T=%lld C=%lld", (long long)B, (long long)T,
                (long long)C);
  return WKV_OK;
}

// Lanes that share a channel with four states each: a power of two.
int scan_lanes(int64_t N) {
  int lanes = 1;
  while (lanes * 4 < N) lanes *= 2;
  return lanes;
}

// The forward's and the summaries' lanes and states a lane: eight share the reads of d,
// d x and the exchange of y best, but up to eight states a channel two lanes of four are
// faster than one lane of eight or of four, with twice the CTAs and so fewer segments (16 x
// 1024 x 1536 with 8 states 173 us and 89 + 152 us, with 4 states 173 and 70 + 125).
int scan_forward_lanes(int64_t N) { return N <= 16 ? 2 : N <= 32 ? 4 : 8; }
template <class F>
int scan_forward_dispatch(int dtype, int64_t N, F f) {
  return with_type(dtype, [&](auto e) {
    constexpr std::integral_constant<int, 2> two;
    constexpr std::integral_constant<int, 4> four;
    constexpr std::integral_constant<int, 8> eight;
    if (N <= 8) return f(e, two, four);
    if (N <= 16) return f(e, two, eight);
    if (N <= 32) return f(e, four, eight);
    return f(e, eight, eight);
  });
}

// Lanes of four states each that share a channel in the backward, which needs two at
// least (one, of 128 channels a CTA, spills its registers: 657 us for 16 x 1024 x 1536
// with 4 states, two lanes 443).
int scan_backward_lanes(int64_t N) { return std::max(2, scan_lanes(N)); }

int64_t scan_ckpts(int64_t T) { return (T + kScanCkpt - 1) / kScanCkpt; }

// How a call is cut: CTAs of `channels` channels and segments of seg_len steps.
struct ScanPlan {
  int cblocks, nseg, seg_len;
};
// Segments where the channels alone give fewer than two CTAs an SM: as many as make
// `want` CTAs. A segment is a multiple of kScanRows steps and at least
// kScanMinSegment of them. The first pass over the segments takes about half as long
// as the scan, which pays only where SMs would idle: 128 channel blocks of 2000 steps
// 308 us in one piece and 220 us in seven, 384 blocks of 1024 steps 245 us in one
// piece and 320 us in two.
ScanPlan scan_plan(int64_t B, int64_t T, int64_t C, int channels, int64_t want) {
  ScanPlan p{(int)((C + channels - 1) / channels), 1, 0};
  const int64_t sets = B * p.cblocks;
  int64_t nseg = sets > 0 && sets < 2 * sm_count() ? (want + sets - 1) / sets : 1;
  nseg = std::max<int64_t>(1, std::min<int64_t>({nseg, T / kScanMinSegment, kScanMaxSegments}));
  const int64_t len = ((T + nseg - 1) / nseg + kScanRows - 1) / kScanRows * kScanRows;
  p.seg_len = (int)std::max<int64_t>(len, kScanRows);
  p.nseg = (int)std::max<int64_t>(1, (T + p.seg_len - 1) / p.seg_len);
  return p;
}
ScanPlan scan_forward_plan(int64_t B, int64_t T, int64_t C, int64_t N) {
  return scan_plan(B, T, C, kScanThreads / scan_forward_lanes(N), 6 * sm_count());
}
ScanPlan scan_backward_plan(int64_t B, int64_t T, int64_t C, int64_t N) {
  const int lanes = scan_backward_lanes(N);
  return scan_plan(B, T, C, scan_bwd_per(lanes) * kScanBwdThreads / lanes, 3 * sm_count());
}

struct ScanWs {
  float *seg_h, *seg_d, *bc, *a, *d;
  size_t bytes;
};
ScanWs scan_ws(const ScanPlan& p, bool backward, int64_t B, int64_t T, int64_t C, int64_t N, void* base) {
  ScanWs w{};
  char* cur = static_cast<char*>(base);
  auto take = [&](size_t n) {
    float* r = reinterpret_cast<float*>(cur);
    const size_t sz = round_up(n * sizeof(float));
    if (cur) cur += sz;
    w.bytes += sz;
    return r;
  };
  if (p.nseg > 1) {
    w.seg_h = take((size_t)B * p.nseg * C * N);
    w.seg_d = take((size_t)B * p.nseg * C);
  }
  if (backward) {
    w.bc = take((size_t)p.cblocks * B * T * 2 * N);
    w.a = take((size_t)B * p.nseg * C * N);
    w.d = take((size_t)B * p.nseg * 2 * C);
  }
  return w;
}

void scan_layout(ScanArgs& a, const ScanPlan& p, const ScanWs& w, int dtype, std::initializer_list<const void*> rows,
                 std::initializer_list<const void*> states) {
  a.cblocks = p.cblocks;
  a.nseg = p.nseg;
  a.seg_len = p.seg_len;
  a.seg_h = w.seg_h;
  a.seg_d = w.seg_d;
  const int es = (int)dtype_size(dtype);
  const int width =
      vector_width(es, 16 / es, rows, {a.C, a.x_sb, a.x_st, a.dt_sb, a.dt_st, a.z_sb, a.z_st, a.g_sb, a.g_st});
  a.wide = width == 16 / es;
  a.pairs = width >= 2;
  a.near = 1;
  for (int64_t s : {a.x_st, a.dt_st, a.z_st, a.g_st, (int64_t)a.C}) a.near = a.near && s >= 0 && s < (1 << 25);
  a.wide_bc = a.N % 4 == 0 && vector_width(es, 4, {a.Bm, a.Cm}, {a.b_sb, a.b_st, a.c_sb, a.c_st}) == 4;
  a.wide_n = a.N % 4 == 0 && vector_width(4, 4, states, {}) == 4;
}

// --------------------------------------------------------------- 4-bit weights

// The most shared memory a launch of the kernel takes: the widest tile of tokens.
template <class E, int R, int NT, int GW>
constexpr size_t q4_smem_max() {
  constexpr int tokens = 8 * NT / Q4Type<E>::kTerms;
  constexpr int a = kQ4MaxWarps * q4_warp_bytes<E, R, NT, GW>(tokens), b = q4_sum_bytes<R, NT>(kQ4MaxWarps);
  return a > b ? a : b;
}

int q4_check(int dtype, int64_t M, int64_t N, int64_t K, int64_t G) {
  if (int rc = check_type(dtype)) return rc;
  if (int rc = check_sizes({M, N, K})) return rc;
  if (K > (1 << 21)) return fail(WKV_ERR_INVALID_ARGUMENT, "size out of range: %lld", (long long)K);
  if (G < 32 || G % 32 != 0 || G > kMaxDim)
    return fail(WKV_ERR_INVALID_ARGUMENT, "the group size must be a positive multiple of 32, got %lld", (long long)G);
  return WKV_OK;
}

}  // namespace

extern "C" {

int causal_conv_forward(int dtype, const void* x, const float* weight, const float* bias, const void* window_in,
                        const int* lengths, void* y, void* window_out, int64_t B, int64_t T, int64_t C, int W,
                        int64_t x_stride_b, int64_t x_stride_t, int silu, void* stream) {
  g_last_error[0] = '\0';
  if (int rc = conv_check(dtype, B, T, C, W)) return rc;
  if (B == 0 || C == 0 || (T == 0 && !window_out)) return WKV_OK;
  if (int rc = check_pointers({weight})) return rc;
  if (T > 0)
    if (int rc = check_pointers({x, y})) return rc;
  ConvArgs a = conv_args(x, weight, bias, window_in, lengths, B, T, C, x_stride_b, x_stride_t, silu);
  a.y = y;
  a.window = W > 1 ? window_out : nullptr;
  const int V = vector_width(dtype_size(dtype), 4, {x, y, window_in, window_out}, {C, x_stride_b, x_stride_t});
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return conv_dispatch(dtype, V, W, [&](auto e, auto v, auto w) {
    constexpr int kV = decltype(v)::value;
    a.cblocks = (int)((C + kConvThreads * kV - 1) / (kConvThreads * kV));
    launch(K_CONV_FWD, st, [&] {
      causal_conv_fwd_kernel<decltype(e), kV, decltype(w)::value>
          <<<(unsigned)(a.cblocks * (int64_t)a.chunks * B), kConvThreads, 0, st>>>(a);
    });
    return launched("causal_conv forward launch");
  });
}

size_t causal_conv_workspace_size(int64_t B, int64_t T, int64_t C, int W) {
  if (conv_check(WKV_DTYPE_F32, B, T, C, W)) return 0;
  return round_up((size_t)B * conv_chunks(T) * (W + 1) * C * sizeof(float));
}

int causal_conv_backward(int dtype, const void* grad_y, const void* x, const float* weight, const float* bias,
                         const void* window_in, const int* lengths, void* grad_x, float* grad_weight,
                         float* grad_bias, void* grad_window, void* workspace, size_t workspace_bytes, int64_t B,
                         int64_t T, int64_t C, int W, int64_t g_stride_b, int64_t g_stride_t, int64_t x_stride_b,
                         int64_t x_stride_t, int silu, void* stream) {
  g_last_error[0] = '\0';
  if (int rc = conv_check(dtype, B, T, C, W)) return rc;
  if (C == 0) return WKV_OK;
  if (int rc = check_pointers({weight, grad_weight})) return rc;
  if (T > 0 && B > 0)
    if (int rc = check_pointers({grad_y, x, grad_x})) return rc;
  const size_t need = causal_conv_workspace_size(B, T, C, W);
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(WKV_ERR_WORKSPACE_TOO_SMALL, "causal_conv backward needs %zu workspace bytes, got %zu", need,
                workspace_bytes);
  ConvArgs a = conv_args(x, weight, bias, window_in, lengths, B, T, C, x_stride_b, x_stride_t, silu);
  a.gy = grad_y;
  a.gy_sb = g_stride_b;
  a.gy_st = g_stride_t;
  a.y = grad_x;
  a.window = W > 1 ? grad_window : nullptr;
  a.partial = static_cast<float*>(workspace);
  const int V = vector_width(dtype_size(dtype), 4, {x, grad_y, grad_x, window_in, grad_window},
                             {C, x_stride_b, x_stride_t, g_stride_b, g_stride_t});
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (B > 0) {
    const int rc = conv_dispatch(dtype, V, W, [&](auto e, auto v, auto w) {
      constexpr int kV = decltype(v)::value;
      a.cblocks = (int)((C + kConvThreads * kV - 1) / (kConvThreads * kV));
      launch(K_CONV_BWD, st, [&] {
        causal_conv_bwd_kernel<decltype(e), kV, decltype(w)::value>
            <<<(unsigned)(a.cblocks * (int64_t)a.chunks * B), kConvThreads, 0, st>>>(a);
      });
      return launched("causal_conv backward launch");
    });
    if (rc) return rc;
  }
  ColSumArgs s{};
  s.in = a.partial;
  s.rows = (int)(B * a.chunks);
  s.blocks = W + 1;
  s.C = C;
  for (int j = 0; j < W; ++j) {
    s.out[j] = grad_weight + j;
    s.step[j] = W;
  }
  s.out[W] = grad_bias;
  s.step[W] = 1;
  return launch_column_sums(s, st);
}

int causal_conv_step(int dtype, const void* x, const float* weight, const float* bias, void* window, void* y,
                     int64_t B, int64_t C, int W, int64_t x_stride_b, int silu, void* stream) {
  g_last_error[0] = '\0';
  if (int rc = conv_check(dtype, B, 1, C, W)) return rc;
  if (B == 0 || C == 0) return WKV_OK;
  if (int rc = check_pointers({x, weight, y})) return rc;
  if (W > 1 && !window) return fail(WKV_ERR_INVALID_ARGUMENT, "null pointer");
  ConvArgs a = conv_args(x, weight, bias, nullptr, nullptr, B, 1, C, x_stride_b, C, silu);
  a.y = y;
  a.window = window;
  a.wide_w = aligned16(weight);
  const int V = vector_width(dtype_size(dtype), 4, {x, y, window}, {C, x_stride_b});
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return conv_dispatch(dtype, V, W, [&](auto e, auto v, auto w) {
    constexpr int kV = decltype(v)::value;
    a.cblocks = (int)((C + kConvThreads * kV - 1) / (kConvThreads * kV));
    launch(K_CONV_STEP, st, [&] {
      causal_conv_step_kernel<decltype(e), kV, decltype(w)::value>
          <<<(unsigned)(a.cblocks * B), kConvThreads, 0, st>>>(a);
    });
    return launched("causal_conv step launch");
  });
}

size_t selective_scan_state_size(int64_t B, int64_t T, int64_t C, int64_t N) {
  if (scan_check(WKV_DTYPE_F32, B, T, C, N)) return 0;
  return (size_t)B * scan_ckpts(T) * C * N * sizeof(float);
}

int selective_scan_forward(int dtype, const void* x, const void* dt, const float* A, const void* Bm, const void* Cm,
                           const float* D, const void* z, const float* dt_bias, const float* state_in,
                           const int* lengths, void* out, float* state_out, float* kept, size_t kept_bytes,
                           void* workspace, size_t workspace_bytes, int64_t B, int64_t T, int64_t C, int64_t N,
                           int64_t x_sb, int64_t x_st, int64_t dt_sb, int64_t dt_st, int64_t b_sb, int64_t b_st,
                           int64_t c_sb, int64_t c_st, int64_t z_sb, int64_t z_st, int softplus, void* stream) {
  g_last_error[0] = '\0';
  if (int rc = scan_check(dtype, B, T, C, N)) return rc;
  if (B == 0 || C == 0 || (T == 0 && !state_out)) return WKV_OK;
  if (int rc = check_pointers({A})) return rc;
  if (T > 0)
    if (int rc = check_pointers({x, dt, Bm, Cm, out})) return rc;
  if (kept && kept_bytes < selective_scan_state_size(B, T, C, N))
    return fail(WKV_ERR_WORKSPACE_TOO_SMALL, "selective_scan keeps %zu bytes of states, got %zu",
                selective_scan_state_size(B, T, C, N), kept_bytes);
  ScanArgs a{};
  a.x = x;
  a.dt = dt;
  a.A = A;
  a.Bm = Bm;
  a.Cm = Cm;
  a.D = D;
  a.z = z;
  a.bias = dt_bias;
  a.h0 = state_in;
  a.lengths = lengths;
  a.out = out;
  a.h_last = state_out;
  a.ckpt = kept;
  a.x_sb = x_sb, a.x_st = x_st, a.dt_sb = dt_sb, a.dt_st = dt_st, a.b_sb = b_sb, a.b_st = b_st;
  a.c_sb = c_sb, a.c_st = c_st, a.z_sb = z_sb, a.z_st = z_st;
  a.B = (int)B, a.T = (int)T, a.C = (int)C, a.N = (int)N;
  a.softplus = softplus;
  const ScanPlan p = scan_forward_plan(B, T, C, N);
  const size_t need = scan_ws(p, false, B, T, C, N, nullptr).bytes;
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(WKV_ERR_WORKSPACE_TOO_SMALL, "selective_scan forward needs %zu workspace bytes, got %zu", need,
                workspace_bytes);
  if (need > 0 && !aligned16(workspace)) return fail(WKV_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
  scan_layout(a, p, scan_ws(p, false, B, T, C, N, workspace), dtype, {x, dt, z, out}, {A, state_in, state_out, kept});
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return scan_forward_dispatch(dtype, N, [&](auto e, auto lanes, auto states) {
    using E = decltype(e);
    constexpr int kLanesPer = decltype(lanes)::value, kStates = decltype(states)::value;
    if (p.nseg > 1) {
      launch(K_SCAN_SUM, st, [&] {
        scan_summary_kernel<E, kLanesPer, kStates, false>
            <<<(unsigned)(B * p.cblocks * (p.nseg - 1)), kScanThreads, 0, st>>>(a);
      });
      if (int rc = launched("selective_scan summary launch")) return rc;
    }
    launch(K_SCAN_FWD, st, [&] {
      scan_fwd_kernel<E, kLanesPer, kStates><<<(unsigned)(B * p.cblocks * p.nseg), kScanThreads, 0, st>>>(a);
    });
    return launched("selective_scan forward launch");
  });
}

size_t selective_scan_forward_workspace_size(int dtype, int64_t B, int64_t T, int64_t C, int64_t N) {
  if (scan_check(dtype, B, T, C, N)) return 0;
  return scan_ws(scan_forward_plan(B, T, C, N), false, B, T, C, N, nullptr).bytes;
}

size_t selective_scan_backward_workspace_size(int dtype, int64_t B, int64_t T, int64_t C, int64_t N) {
  if (scan_check(dtype, B, T, C, N)) return 0;
  return scan_ws(scan_backward_plan(B, T, C, N), true, B, T, C, N, nullptr).bytes;
}

int selective_scan_backward(int dtype, const void* grad_out, const void* x, const void* dt, const float* A,
                            const void* Bm, const void* Cm, const float* D, const void* z, const float* dt_bias,
                            const float* kept, const int* lengths, const float* grad_state_out, void* grad_x,
                            void* grad_dt, float* grad_A, void* grad_B, void* grad_C, float* grad_D, void* grad_z,
                            float* grad_dt_bias, float* grad_state_in, void* workspace, size_t workspace_bytes,
                            int64_t B, int64_t T, int64_t C, int64_t N, int64_t g_sb, int64_t g_st, int64_t x_sb,
                            int64_t x_st, int64_t dt_sb, int64_t dt_st, int64_t b_sb, int64_t b_st, int64_t c_sb,
                            int64_t c_st, int64_t z_sb, int64_t z_st, int softplus, void* stream) {
  g_last_error[0] = '\0';
  if (int rc = scan_check(dtype, B, T, C, N)) return rc;
  if (C == 0) {  // the sums over channels are there all the same
    const size_t bytes = (size_t)B * T * N * dtype_size(dtype);
    if (bytes == 0) return WKV_OK;
    if (int rc = check_pointers({grad_B, grad_C})) return rc;
    cudaError_t e = cudaMemsetAsync(grad_B, 0, bytes, static_cast<cudaStream_t>(stream));
    if (e == cudaSuccess) e = cudaMemsetAsync(grad_C, 0, bytes, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? WKV_OK : cuda_fail(e, "zeroing the gradients of B and C");
  }
  if (int rc = check_pointers({A, grad_A})) return rc;
  if (B > 0 && T > 0)
    if (int rc = check_pointers({grad_out, x, dt, Bm, Cm, kept, grad_x, grad_dt, grad_B, grad_C})) return rc;
  if (B > 0 && T > 0 && (z != nullptr) != (grad_z != nullptr))
    return fail(WKV_ERR_INVALID_ARGUMENT, "z and grad_z go together");
  const ScanPlan p = scan_backward_plan(B, T, C, N);
  const size_t need = scan_ws(p, true, B, T, C, N, nullptr).bytes;
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(WKV_ERR_WORKSPACE_TOO_SMALL, "selective_scan backward needs %zu workspace bytes, got %zu", need,
                workspace_bytes);
  if (need > 0 && !aligned16(workspace)) return fail(WKV_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
  const ScanWs ws = scan_ws(p, true, B, T, C, N, workspace);
  ScanArgs a{};
  a.gout = grad_out;
  a.x = x;
  a.dt = dt;
  a.A = A;
  a.Bm = Bm;
  a.Cm = Cm;
  a.D = D;
  a.z = z;
  a.bias = dt_bias;
  a.ckpt = const_cast<float*>(kept);
  a.lengths = lengths;
  a.gh_last = grad_state_out;
  a.gx = grad_x;
  a.gdt = grad_dt;
  a.gz = grad_z;
  a.gh0 = grad_state_in;
  a.part_bc = ws.bc;
  a.part_a = ws.a;
  a.part_d = ws.d;
  a.x_sb = x_sb, a.x_st = x_st, a.dt_sb = dt_sb, a.dt_st = dt_st, a.b_sb = b_sb, a.b_st = b_st;
  a.c_sb = c_sb, a.c_st = c_st, a.z_sb = z_sb, a.z_st = z_st, a.g_sb = g_sb, a.g_st = g_st;
  a.B = (int)B, a.T = (int)T, a.C = (int)C, a.N = (int)N;
  a.softplus = softplus;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  scan_layout(a, p, ws, dtype, {grad_out, x, dt, z, grad_x, grad_dt, grad_z},
              {A, kept, grad_state_out, grad_state_in});
  if (B > 0) {
    int rc = WKV_OK;
    if (p.nseg > 1) {
      rc = scan_forward_dispatch(dtype, N, [&](auto e, auto lanes, auto states) {
        constexpr int kLanesPer = decltype(lanes)::value, kStates = decltype(states)::value;
        constexpr int kChannels = kScanThreads / kLanesPer;
        ScanArgs s = a;
        s.cblocks = (int)((C + kChannels - 1) / kChannels);
        launch(K_SCAN_ADJ, st, [&] {
          scan_summary_kernel<decltype(e), kLanesPer, kStates, true>
              <<<(unsigned)(B * s.cblocks * (p.nseg - 1)), kScanThreads, 0, st>>>(s);
        });
        return launched("selective_scan adjoint launch");
      });
      if (rc) return rc;
    }
    auto main = [&](auto e, auto lanes) {
      using E = decltype(e);
      constexpr int kLanesPer = decltype(lanes)::value;
      const cudaError_t err = allow_smem(scan_bwd_kernel<E, kLanesPer>, ScanBwdSmem<E, kLanesPer>::kBytes);
      if (err != cudaSuccess) return cuda_fail(err, "setting the selective_scan backward kernel's shared memory size");
      launch(K_SCAN_BWD, st, [&] {
        scan_bwd_kernel<E, kLanesPer><<<(unsigned)(B * p.cblocks * p.nseg), kScanBwdThreads,
                                        ScanBwdSmem<E, kLanesPer>::kBytes, st>>>(a);
      });
      return launched("selective_scan backward launch");
    };
    rc = with_type(dtype, [&](auto e) {
      switch (scan_backward_lanes(N)) {
        case 2: return main(e, std::integral_constant<int, 2>{});
        case 4: return main(e, std::integral_constant<int, 4>{});
        case 8: return main(e, std::integral_constant<int, 8>{});
        default: return main(e, std::integral_constant<int, 16>{});
      }
    });
    if (rc) return rc;
  }
  const int64_t cells = B * T * 2 * N;
  ScanReduceArgs r{};
  r.bc = ws.bc;
  r.slices = p.cblocks;
  r.N = (int)N;
  r.rows = B * T;
  r.gB = grad_B;
  r.gC = grad_C;
  r.bc_blocks = (cells + kScanReduceThreads - 1) / kScanReduceThreads;
  r.a_blocks = (C * N + 31) / 32;
  r.a.in = ws.a;
  r.a.out[0] = grad_A;
  r.a.step[0] = 1;
  r.a.C = C * N;
  r.a.blocks = 1;
  r.d.in = ws.d;
  r.d.out[0] = grad_D;
  r.d.out[1] = grad_dt_bias;
  r.d.step[0] = r.d.step[1] = 1;
  r.d.C = C;
  r.d.blocks = 2;
  r.a.rows = r.d.rows = (int)(B * p.nseg);
  const int64_t d_blocks = grad_D || grad_dt_bias ? (2 * C + 31) / 32 : 0;
  return with_type(dtype, [&](auto e) {
    launch(K_SCAN_RED, st, [&] {
      scan_reduce_kernel<decltype(e)>
          <<<(unsigned)(r.bc_blocks + r.a_blocks + d_blocks), kScanReduceThreads, 0, st>>>(r);
    });
    return launched("selective_scan reduction launch");
  });
}

int selective_scan_step(int dtype, const void* x, const void* dt, const float* A, const void* Bm, const void* Cm,
                        float* state, const float* D, const void* z, const float* dt_bias, void* out, int64_t B,
                        int64_t C, int64_t N, int64_t x_sb, int64_t dt_sb, int64_t b_sb, int64_t c_sb, int64_t z_sb,
                        int softplus, void* stream) {
  g_last_error[0] = '\0';
  if (int rc = scan_check(dtype, B, 1, C, N)) return rc;
  if (B == 0 || C == 0) return WKV_OK;
  if (int rc = check_pointers({x, dt, A, Bm, Cm, state, out})) return rc;
  ScanArgs a{};
  a.x = x;
  a.dt = dt;
  a.A = A;
  a.Bm = Bm;
  a.Cm = Cm;
  a.D = D;
  a.z = z;
  a.bias = dt_bias;
  a.out = out;
  a.h_last = state;
  a.x_sb = x_sb, a.dt_sb = dt_sb, a.b_sb = b_sb, a.c_sb = c_sb, a.z_sb = z_sb;
  a.B = (int)B, a.T = 1, a.C = (int)C, a.N = (int)N;
  a.softplus = softplus;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int es = (int)dtype_size(dtype), lanes = scan_lanes(N);
  a.wide_bc = N % 4 == 0 && vector_width(es, 4, {Bm, Cm}, {b_sb, c_sb}) == 4;
  a.wide_n = N % 4 == 0 && vector_width(4, 4, {A, state}, {}) == 4;
  auto go = [&](auto e, auto lanes_) {
    constexpr int kLanesPer = decltype(lanes_)::value, kChannels = kScanStepThreads / kLanesPer;
    a.cblocks = (int)((C + kChannels - 1) / kChannels);
    launch(K_SCAN_STEP, st, [&] {
      scan_step_kernel<decltype(e), kLanesPer>
          <<<(unsigned)((B + kLanesPer - 1) / kLanesPer * a.cblocks), kScanStepThreads, 0, st>>>(a);
    });
    return launched("selective_scan step launch");
  };
  return with_type(dtype, [&](auto e) {
    switch (lanes) {
      case 1: return go(e, std::integral_constant<int, 1>{});
      case 2: return go(e, std::integral_constant<int, 2>{});
      case 4: return go(e, std::integral_constant<int, 4>{});
      case 8: return go(e, std::integral_constant<int, 8>{});
      default: return go(e, std::integral_constant<int, 16>{});
    }
  });
}

int layer_norm_forward(int dtype, const void* x, const float* weight, const float* bias, void* y, float* mean,
                       float* rstd, int64_t rows, int64_t C, int64_t x_stride, float eps, void* stream) {
  g_last_error[0] = '\0';
  if (int rc = norm_check(dtype, rows, C)) return rc;
  if (rows == 0 || C == 0) return WKV_OK;
  if (int rc = check_pointers({x, y, mean, rstd})) return rc;
  NormArgs a{};
  a.x = x;
  a.w = weight;
  a.b = bias;
  a.y = y;
  a.mean = mean;
  a.rstd = rstd;
  a.rows = rows;
  a.C = (int)C;
  a.x_s = x_stride;
  a.eps = eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const NormPlan p = norm_plan(rows, C);
  a.span = p.span;
  return norm_dispatch(dtype, p.threads, {x, y, weight, bias}, {C, x_stride}, [&](auto e, auto v, auto n) {
    using E = decltype(e);
    constexpr int V = decltype(v)::value, kThr = decltype(n)::value;
    constexpr bool kStaged = NormIo<E, V>::kStaged;
    auto kernel = layer_norm_fwd_kernel<E, V, kThr>;
    const cudaError_t err = allow_smem(kernel, kStaged ? norm_smem(false, true, sizeof(E), kThr, kThr, kThr * kNormValues) : 0);
    if (err != cudaSuccess) return cuda_fail(err, "setting the layer_norm kernel's shared memory size");
    // where three CTAs share an SM, those; elsewhere twice as many as the plan has, which
    // evens out the rows (16384 x 8192 70 us, with three quarters of them 83), but of 1024
    // threads what is resident (8192 x 16384 133 us, with twice as many 138)
    const unsigned grid = norm_fwd_ctas<E, V, kThr>() == 3 ? p.grid * 3 / 2
                          : kThr < 1024                    ? p.grid * 2
                                                           : (unsigned)std::min<int64_t>(2 * rows, sm_count());
    launch(K_LN_FWD, st, [&] {
      kernel<<<grid, p.threads, norm_smem(false, kStaged, sizeof(E), p.span, p.threads, C), st>>>(a);
    });
    return launched("layer_norm forward launch");
  });
}

size_t layer_norm_workspace_size(int dtype, int64_t rows, int64_t C) {
  if (norm_check(dtype, rows, C)) return 0;
  return round_up((size_t)norm_plan(rows, C).grid * 2 * C * sizeof(float));
}

int layer_norm_backward(int dtype, const void* grad_y, const void* x, const float* weight, const float* mean,
                        const float* rstd, void* grad_x, float* grad_weight, float* grad_bias, void* workspace,
                        size_t workspace_bytes, int64_t rows, int64_t C, int64_t g_stride, int64_t x_stride,
                        void* stream) {
  g_last_error[0] = '\0';
  if (int rc = norm_check(dtype, rows, C)) return rc;
  if (C == 0) return WKV_OK;
  if (rows > 0)
    if (int rc = check_pointers({grad_y, x, mean, rstd, grad_x})) return rc;
  const size_t need = layer_norm_workspace_size(dtype, rows, C);
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(WKV_ERR_WORKSPACE_TOO_SMALL, "layer_norm backward needs %zu workspace bytes, got %zu", need,
                workspace_bytes);
  NormArgs a{};
  a.x = x;
  a.w = weight;
  a.gy = grad_y;
  a.y = grad_x;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.partial = static_cast<float*>(workspace);
  a.rows = rows;
  a.C = (int)C;
  a.x_s = x_stride;
  a.gy_s = g_stride;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const NormPlan p = norm_plan(rows, C);
  a.span = p.span;
  if (rows > 0) {
    const int rc =
        norm_dispatch(dtype, p.threads, {grad_y, x, grad_x, weight}, {C, g_stride, x_stride}, [&](auto e, auto v, auto n) {
          using E = decltype(e);
          constexpr int V = decltype(v)::value, kThr = decltype(n)::value;
          constexpr bool kStaged = NormIo<E, V>::kStaged;
          auto kernel = layer_norm_bwd_kernel<E, V, kThr>;
          const cudaError_t err =
              allow_smem(kernel, (kThr == 256 ? 2 * kThr * kNormValues * sizeof(float) : 0) +
                                     (kStaged ? norm_smem(true, true, sizeof(E), kThr, kThr, kThr * kNormValues) : 0));
          if (err != cudaSuccess) return cuda_fail(err, "setting the layer_norm kernel's shared memory size");
          launch(K_LN_BWD, st, [&] {
            kernel<<<(unsigned)p.grid, p.threads, norm_smem(true, kStaged, sizeof(E), p.span, p.threads, C), st>>>(a);
          });
          return launched("layer_norm backward launch");
        });
    if (rc) return rc;
  }
  if (!grad_weight && !grad_bias) return WKV_OK;
  ColSumArgs s{};
  s.in = a.partial;
  s.rows = p.grid;
  s.blocks = 2;
  s.C = C;
  s.out[0] = grad_weight;
  s.out[1] = grad_bias;
  s.step[0] = s.step[1] = 1;
  return launch_column_sums(s, st);
}

int q4_matvec(int dtype, const void* x, const uint8_t* packed, const void* scales, const uint8_t* zeros,
              const float* bias, void* y, int64_t M, int64_t N, int64_t K, int64_t group, int64_t x_stride,
              void* stream) {
  g_last_error[0] = '\0';
  if (int rc = q4_check(dtype, M, N, K, group)) return rc;
  if (M == 0 || N == 0) return WKV_OK;
  if (int rc = check_pointers({y})) return rc;
  if (K > 0) {
    if (int rc = check_pointers({x, packed, scales})) return rc;
    if (!aligned16(packed)) return fail(WKV_ERR_INVALID_ARGUMENT, "packed must be 16-byte aligned");
  }
  Q4Args a{};
  a.x = x;
  a.q = packed;
  a.scale = static_cast<const __nv_bfloat16*>(scales);
  a.zero = zeros;
  a.bias = bias;
  a.y = y;
  a.x_s = x_stride;
  a.M = (int)M;
  a.N = (int)N;
  a.K = (int)K;
  a.G = (int)group;
  a.groups = (int)((K + group - 1) / group);
  a.pitch = (int)((K + 31) / 32 * 16);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int es = (int)dtype_size(dtype);
  const int vector = vector_width(es, 16 / es, {x}, {x_stride, K});
  // floor(i / d) is the upper word of i * (floor(2^32 / d) + 1) while i * d < 2^32
  const int64_t d = std::min(group, (K + 31) / 32 * 32) / 32;
  a.group_magic = d > 1 ? (uint32_t)((1ull << 32) / d + 1) : 0;
  return with_type(dtype, [&](auto e) {
    using E = decltype(e);
    constexpr int kTerms = Q4Type<E>::kTerms;
    a.tokens = (int)std::min<int64_t>(M, kTerms == 1 ? 16 : 8);  // what a lane's registers hold of a stage
    const int tiles = (a.tokens * kTerms + 7) / 8;
    const int64_t my = (M + a.tokens - 1) / a.tokens;
    if (my > 65535) return fail(WKV_ERR_INVALID_ARGUMENT, "too many tokens: %lld", (long long)M);
    auto launch_one = [&](auto r, auto nt, auto gw) {
      constexpr int R = decltype(r)::value, NT = decltype(nt)::value, GW = decltype(gw)::value;
      // Four warps a CTA where the rows alone make two such CTAs an SM, else eight; all of
      // them along the inputs as long as each has three stages or rows are short of SMs.
      // With one tile of tokens fewer are along the inputs still while that leaves two
      // CTAs an SM: 393 CTAs of six stages a warp run at once where 786 of three take two
      // turns (1 x 768 x 50257 10.3 and 11.4 us a call back to back; with three tiles, whose
      // CTAs are fewer an SM, 6 x 2048 x 16384 float32 22 and 20 us).
      const int64_t chunks = (K + kQ4Chunk - 1) / kQ4Chunk;
      const int warps = N >= 16 * R * 2 * sm_count() ? 4 : 8;
      auto ctas = [&](int wk) { return (N + 16 * R * (warps / wk) - 1) / (16 * R * (warps / wk)); };
      a.wk = warps;
      while (a.wk > 1 && ((chunks < 3 * a.wk && ctas(a.wk / 2) >= sm_count()) ||
                          (NT == 1 && chunks < 6 * a.wk && ctas(a.wk / 2) >= 2 * sm_count())))
        a.wk /= 2;
      const int bytes = std::max(warps * q4_warp_bytes<E, R, NT, GW>(a.tokens), q4_sum_bytes<R, NT>(warps));
      const bool wide = vector >= (q4_direct<E, NT>() ? 8 : 4);
      auto kernel = wide ? q4_matvec_kernel<E, R, NT, GW, true> : q4_matvec_kernel<E, R, NT, GW, false>;
      const cudaError_t err = allow_smem(kernel, q4_smem_max<E, R, NT, GW>());
      if (err != cudaSuccess) return cuda_fail(err, "setting the q4_matvec kernel's shared memory size");
      launch(K_Q4, st, [&] {
        kernel<<<dim3((unsigned)ctas(a.wk), (unsigned)my), warps * 32, bytes, st>>>(a);
      });
      return launched("q4_matvec launch");
    };
    // Inputs scaled at a time: 128, 64 or 32, that always lie in one group.
    auto go = [&](auto r, auto nt) {
      if (a.groups == 1 || group % 128 == 0) return launch_one(r, nt, std::integral_constant<int, 4>{});
      if (group % 64 == 0) return launch_one(r, nt, std::integral_constant<int, 2>{});
      return launch_one(r, nt, std::integral_constant<int, 1>{});
    };
    // 32 rows a warp where that still gives two CTAs an SM, so that the inputs are read and
    // paired half as often: 16 x 768 x 50257 31 us with 16 rows, 29 with 32; 16 x 8192 x 16384
    // 76 and 66, though with groups of 128 the kernel spills 108 bytes. (Three tiles' sums and
    // operands leave no registers for 32 rows.)
    if (tiles == 2) {
      if (N >= 64 * sm_count()) return go(std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
      return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{});
    }
    if constexpr (kTerms > 1)
      if (tiles == 3) return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 3>{});
    if (N >= 64 * sm_count()) return go(std::integral_constant<int, 2>{}, std::integral_constant<int, 1>{});
    return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
  });
}

}  // extern "C"
