// C-ABI implementation (include/tha4_hip.h) of the transformer block operators for MI355X (gfx950): argument checks and launches.
// The kernels live in transformer_{norm,linear,attention}_kernels.h.  Nothing here allocates, synchronises or keeps state between calls.
#include "tha4_hip.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <utility>

#include "tha4_host.h"
#include "transformer_attention_kernels.h"
#include "transformer_linear_kernels.h"
#include "transformer_norm_kernels.h"

using namespace tha4;
using namespace tha4::xf;

namespace {

constexpr int64_t kMaxGrid = 0x7fffffff;
constexpr float kLog2e = 1.44269504088896340736f;

int64_t size_of(int dtype) { return dtype == THA4_F32 ? 4 : 2; }
bool known(int dtype) { return dtype == THA4_F32 || dtype == THA4_F16 || dtype == THA4_BF16; }
bool aligned(const void* p, int64_t row_stride, int64_t size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row_stride * size % 16 == 0; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// the GPU all the pointers (NULL ones aside) live on, or -1
template <int N>
int one_device(const void* const (&p)[N]) {
  int dev = -1;
  for (const void* x : p) {
    if (!x) continue;
    const int d = device_of(x);
    if (d < 0 || (dev >= 0 && d != dev)) return -1;
    dev = d;
  }
  return dev;
}

int bad(const char* msg) { return fail(THA4_ERR_INVALID_ARGUMENT, msg); }

// A launch has fewer than 2^32 threads in a direction: the most workgroups of one.  What needs more is cut into several launches.
constexpr int64_t most_workgroups(int threads) { return 0xffffffffLL / threads; }

template <class K, class A>
int launch(K kernel, int64_t grid, int64_t grid_y, int threads, const A& a, void* stream) {
  if (grid > most_workgroups(threads) || grid_y > 65535) return bad("too many workgroups for one launch");
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid, (unsigned)grid_y), dim3(threads), 0, static_cast<hipStream_t>(stream), a);
  HIP_TRY(hipGetLastError());
  return THA4_OK;
}

// kernels that work on rows, `per` of them a workgroup
template <class K, class A>
int launch_rows(K kernel, int per, int threads, A a, void* stream) {
  const int64_t step = most_workgroups(threads) * per;
  for (a.first = 0; a.first < a.rows; a.first += step) {
    const int st = launch(kernel, ceil_div(std::min(a.rows - a.first, step), per), 1, threads, a, stream);
    if (st != THA4_OK) return st;
  }
  return THA4_OK;
}

// ---- quantisation ----
template <class T>
int quantize(const QuantArgs& a, void* stream) {
  if (a.cols % 8 || !aligned(a.x, a.x_stride, sizeof(T)) || reinterpret_cast<uintptr_t>(a.q) % 8 || a.q_stride % 8 || a.cols > 16384)
    return launch_rows(quantize_any_kernel<T>, 1, 256, a, stream);
  if (a.cols <= 512) return launch_rows(quantize_kernel<T, 64, 1>, 4, 256, a, stream);
  if (a.cols <= 2048) return launch_rows(quantize_kernel<T, 256, 1>, 1, 256, a, stream);
  if (a.cols <= 4096) return launch_rows(quantize_kernel<T, 256, 2>, 1, 256, a, stream);
  if (a.cols <= 8192) return launch_rows(quantize_kernel<T, 256, 4>, 1, 256, a, stream);
  return launch_rows(quantize_kernel<T, 1024, 2>, 1, 1024, a, stream);
}

// ---- product ----
const char* check_linear(const tha4_linear_i8_args& g) {
  if (g.x_dtype != THA4_I8 && !known(g.x_dtype)) return "x_dtype must be i8, f32, f16 or bf16";
  if (!known(g.y_dtype)) return "y_dtype must be f32, f16 or bf16";
  if (g.m < 0 || g.n < 0 || g.k < 1) return "m / n must not be negative and k must be positive";
  if (g.k > 131071) return "k must be at most 131071 (the sums are 32-bit integers)";
  if (g.m > kMaxGrid || g.n > kMaxGrid) return "m / n must be below 2^31";
  return nullptr;
}
// float tokens that every workgroup of the product quantises for itself (linear_few_kernel)
bool inline_tokens(const tha4_linear_i8_args& g) { return g.m <= kInlineTokens && g.m * g.k <= kInlineBytes; }
int64_t token_stride(const tha4_linear_i8_args& g) { return ceil_div(g.k, 16) * 16; }

// m tokens from m0 on, n channels from n0 on
LinearArgs part_of(const LinearArgs& a, int64_t m0, int64_t m, int64_t n0, int64_t n) {
  LinearArgs b = a;
  if (m0) {                                                              // (int8 tokens: the forms for few tokens take them all)
    b.x = static_cast<const int8_t*>(a.x) + m0 * a.x_stride;
    b.xs += m0;
  }
  b.w += n0 * a.w_stride;
  b.ws += n0;
  if (b.bias) b.bias += n0;
  b.y = static_cast<char*>(a.y) + (m0 * a.y_stride + n0) * size_of(a.y_dtype);
  b.m = std::min(a.m - m0, m);
  b.n = std::min(a.n - n0, n);
  return b;
}

template <class XT, int NT, int MT, bool INLINE>
int few(const LinearArgs& a, bool al, void* stream) {
  const int64_t step = most_workgroups(512) * 16 * NT, mb = ceil_div(a.m, 16 * MT);
  for (int64_t n0 = 0; n0 < a.n; n0 += step) {
    const LinearArgs b = part_of(a, 0, a.m, n0, step);
    const int64_t nb = ceil_div(b.n, 16 * NT);
    int st = THA4_OK;
    if constexpr (NT == 1) st = al ? launch(linear_few_kernel<XT, NT, MT, true, INLINE>, nb, mb, 512, b, stream) : launch(linear_few_kernel<XT, NT, MT, false, INLINE>, nb, mb, 512, b, stream);
    else st = launch(linear_few_kernel<XT, NT, MT, true, INLINE>, nb, mb, 512, b, stream);
    if (st != THA4_OK) return st;
  }
  return THA4_OK;
}
template <int BM, int BN, int WM, int WN, int G, int STAGES>
int tile(const LinearArgs& a, bool al, void* stream) {
  constexpr int threads = 64 * WM * WN * G;
  const int64_t most = most_workgroups(threads), step_n = most * BN, step_m = most / std::min(ceil_div(a.n, BN), most) * BM;
  for (int64_t n0 = 0; n0 < a.n; n0 += step_n)
    for (int64_t m0 = 0; m0 < a.m; m0 += step_m) {
      const LinearArgs b = part_of(a, m0, step_m, n0, step_n);
      const int64_t tiles = ceil_div(b.m, BM) * ceil_div(b.n, BN);
      const int st = al ? launch(linear_tile_kernel<BM, BN, 128, WM, WN, G, STAGES, true>, tiles, 1, threads, b, stream)
                        : launch(linear_tile_kernel<BM, BN, 128, WM, WN, G, STAGES, false>, tiles, 1, threads, b, stream);
      if (st != THA4_OK) return st;
    }
  return THA4_OK;
}
// Which kernel: by the number of tokens, then the largest tile whose grid still covers most of the 256 CUs (us, w one of three in turn, bf16 out):
//   m <= 32  weights straight into operands, wide tiles of channels where they fill the GPU:  32 x 16384 x 4096: 30.9 (NT 1), 20.3 (2), 17.2 (4);  32 x 8192 x 8192: 26.9, 21.9, 25.3
//                                                32 x 4096 x 4096: 11.2 against 13.7 on 64 x 64 tiles;  64 x 8192 x 8192: 40.2 against 20.8 - tiles from 33 tokens on
//   256 x 256 from 192 tiles on                  8192^3: 531 against 781 on 128 x 128
//   64 x 64 at most 256 tiles: four groups       256 x 4096 x 4096: 12.2 against 14.9 with one group;  320 x 4096 x 4096 (320 tiles): 22.9 against 17.0
int product(const LinearArgs& a, bool al, void* stream) {
  if (a.m <= 16) return al && a.m > kInlineTokens && a.n >= 16384 ? few<float, 4, 1, false>(a, al, stream) : few<float, 1, 1, false>(a, al, stream);
  if (a.m <= 32) return al && a.n >= 16384 ? few<float, 4, 2, false>(a, al, stream) : al && a.n >= 8192 ? few<float, 2, 2, false>(a, al, stream) : few<float, 1, 2, false>(a, al, stream);
  if (ceil_div(a.m, 256) * ceil_div(a.n, 256) >= 192) return tile<256, 256, 4, 2, 1, 2>(a, al, stream);
  if (ceil_div(a.m, 128) * ceil_div(a.n, 128) >= 192) return tile<128, 128, 2, 2, 1, 2>(a, al, stream);
  if (ceil_div(a.m, 64) * ceil_div(a.n, 64) > 256) return tile<64, 64, 2, 2, 1, 4>(a, al, stream);
  return tile<64, 64, 2, 2, 4, 2>(a, al, stream);
}

// ---- norms ----
template <class T, class R>
int norm(const NormArgs& a, bool vector, void* stream) {
  if (!vector || a.cols > 16384) return launch_rows(residual_norm_any_kernel<T, R>, 1, 256, a, stream);
  if (a.cols <= 512) return launch_rows(residual_norm_kernel<T, R, 64, 1>, 4, 256, a, stream);
  if (a.cols <= 1024) return launch_rows(residual_norm_kernel<T, R, 64, 2>, 4, 256, a, stream);
  if (a.cols <= 2048) return launch_rows(residual_norm_kernel<T, R, 256, 1>, 1, 256, a, stream);
  if (a.cols <= 4096) return launch_rows(residual_norm_kernel<T, R, 256, 2>, 1, 256, a, stream);
  if (a.cols <= 8192) return launch_rows(residual_norm_kernel<T, R, 512, 2>, 1, 512, a, stream);
  return launch_rows(residual_norm_kernel<T, R, 1024, 2>, 1, 1024, a, stream);
}

// ---- attention ----
// How the keys are divided among workgroups when there are few queries.  A pure function of the sizes: the workspace query and the launch agree.
struct Plan {
  bool few;
  int row_tiles, splits, chunk, part_rows;
};
Plan plan_of(const tha4_diff_attention_args& a) {
  Plan p{};
  const int64_t rows = (int64_t)a.q_len * (a.heads / a.kv_heads);
  // A prompt's workgroup walks through all the keys alone (4.6e-4 us a key and channel behind 10 us: 128 x 8192, d = 64: 262 us however few queries there are); the path for few queries
  // divides the keys but repeats them for every 16 rows (290 TFLOP/s behind two launches).  It is taken where it is clearly the shorter (prompt path / few path, us):
  // 128 x 8192, 8 heads, d = 64: 262 / 35;  64 x 32768, 8 on 2 heads, d = 128: 1813 / 110;  512 x 4096, 8 heads, d = 64: 134 / 61;  1024 x 8192, 8 heads, d = 128: 468 / 367;
  // 128 x 1024, 8 heads, d = 64: 44 / 17;  8 x 32 x 512, 8 heads, d = 64: 25 / 20;  512 x 512, 8 heads, d = 64: 26 / 32;  24 x 300, 8 heads, d = 32: 12.6 / 16.8
  const double keys_d = (double)a.k_len * a.head_dim;
  const double prompt_us = 10.0 + 4.6e-4 * keys_d * (double)ceil_div((int64_t)a.batch * a.heads * ceil_div(a.q_len, 128), 256);
  const double few_us = 16.0 + 12.0 / 2.9e8 * keys_d * (double)a.batch * a.kv_heads * (double)(ceil_div(rows, kRows) * kRows);
  p.few = rows <= kRows || 1.3 * few_us < prompt_us;
  p.splits = 1;
  p.chunk = a.k_len;
  if (!p.few) return p;
  p.row_tiles = (int)ceil_div(rows, kRows);
  p.part_rows = (int)std::min<int64_t>(rows, kRows);
  const int64_t wgs = std::max<int64_t>((int64_t)a.batch * a.kv_heads * p.row_tiles, 1);
  // Workgroups to aim for.  Full caches: what the GPU holds at once (256 CUs, one workgroup each at d = 128, two below; 131072 keys, d = 128, 8 heads on 2: 256 -> 63 us, 512 ->
  // 71 us, 1024 -> 90 us: the parts to join grow).  Caches of their own lengths: many more, for the short ones end at once (32 x 16384 keys: 512 -> 138 us, 1024 -> 146 us, 2048 -> 131 us, 8192 -> 132 us).
  const int64_t aim = a.kv_lengths_dev ? 2048 : a.head_dim == 128 ? 256 : 512;
  const int64_t want = std::min<int64_t>(ceil_div(aim, wgs), kMaxSplits);
  const int64_t chunk = std::max<int64_t>(ceil_div(ceil_div(a.k_len, want), 128) * 128, 256);
  p.splits = (int)std::max<int64_t>(ceil_div(a.k_len, chunk), 1);
  p.chunk = (int)chunk;
  return p;
}
int64_t part_floats(int d) { return d == 32 ? Few<32>::PART : d == 64 ? Few<64>::PART : Few<128>::PART; }

const char* check_shape(const tha4_diff_attention_args& a) {
  if (a.batch < 0 || a.q_len < 0 || a.k_len < 0 || a.heads < 1 || a.kv_heads < 1) return "batch / q_len / k_len must not be negative, heads / kv_heads must be positive";
  if (a.heads % a.kv_heads) return "heads must be a multiple of kv_heads";
  if (a.head_dim != 32 && a.head_dim != 64 && a.head_dim != 128) return "head_dim must be 32, 64 or 128";
  if (a.dtype != THA4_F16 && a.dtype != THA4_BF16) return "dtype must be f16 or bf16";
  if (a.q_len > (1 << 30) || a.k_len > (1 << 30)) return "q_len / k_len must be at most 2^30";
  if ((int64_t)a.q_len * (a.heads / a.kv_heads) > kMaxGrid) return "too many queries for one launch";
  return nullptr;
}

// whether the rows of `out` that (batch, token, head) address share elements: every stride has to step over what the smaller ones span
bool overlaps_itself(const tha4_diff_attention_args& g) {
  int64_t n[3] = {g.batch, g.q_len, g.heads}, s[3] = {g.out_stride[0], g.out_stride[1], g.out_stride[2]}, span = 2 * g.head_dim;
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2 - i; ++j)
      if (s[j] > s[j + 1]) {
        std::swap(s[j], s[j + 1]);
        std::swap(n[j], n[j + 1]);
      }
  for (int i = 0; i < 3; ++i) {
    if (n[i] == 1) continue;
    if (s[i] < span) return true;
    span += s[i] * (n[i] - 1);
  }
  return false;
}

template <class T, int D>
int attention_launch(const AttnArgs& a, const Plan& p, bool narrow, void* stream) {
  if (!p.few) {
    const int64_t heads = (int64_t)a.batch * a.heads;
    if constexpr (D == 32)
      if (narrow) return launch(diff_prompt_kernel<T, D, 2>, heads * ceil_div(a.q_len, 64), 1, 256, a, stream);
    return launch(diff_prompt_kernel<T, D, 4>, heads * ceil_div(a.q_len, 128), 1, 512, a, stream);
  }
  const int64_t tiles = (int64_t)a.batch * a.kv_heads * p.row_tiles;
  const int st = launch(diff_few_kernel<T, D>, tiles * p.splits, 1, 256, a, stream);
  if (st != THA4_OK || p.splits == 1) return st;
  return launch(diff_join_kernel<T, D>, tiles * p.part_rows, 1, 512, a, stream);
}
template <class T, int D>
int attention(const AttnArgs& a, const Plan& p, void* stream) {
  // d = 32: workgroups of 64 queries where those of 128 leave CUs without one (8 frames of 256 tokens: 11.4 us against 15.7, in a graph; at d = 64 the wider ones are as fast or faster)
  const bool narrow = D == 32 && (int64_t)a.batch * a.heads * ceil_div(a.q_len, 128) < 256;
  // sequences of one launch: by the kernel that has the most threads for each
  const int64_t tiles = (int64_t)a.kv_heads * p.row_tiles;
  const int64_t threads = !p.few ? 512 * (a.heads * ceil_div(a.q_len, 128)) : std::max<int64_t>(256 * tiles * p.splits, p.splits == 1 ? 0 : 512 * tiles * p.part_rows);
  const int64_t step = std::max<int64_t>(0xffffffffLL / std::max<int64_t>(threads, 1), 1);
  for (int64_t b0 = 0; b0 < a.batch; b0 += step) {
    AttnArgs c = a;
    c.batch = (int32_t)std::min<int64_t>(a.batch - b0, step);
    c.q = static_cast<const T*>(a.q) + b0 * a.qs[0];
    c.k = static_cast<const T*>(a.k) + b0 * a.ks[0];
    c.v = static_cast<const T*>(a.v) + b0 * a.vs[0];
    c.out = static_cast<T*>(a.out) + b0 * a.os[0];
    if (a.mask) c.mask = a.mask + b0 * a.ms[0];
    if (a.q_lengths) c.q_lengths = a.q_lengths + b0;
    if (a.kv_lengths) c.kv_lengths = a.kv_lengths + b0;
    if (a.work) c.work = a.work + b0 * tiles * p.part_rows * p.splits * part_floats(D);
    const int st = attention_launch<T, D>(c, p, narrow, stream);
    if (st != THA4_OK) return st;
  }
  return THA4_OK;
}
template <class T>
int attention(const AttnArgs& a, int d, const Plan& p, void* stream) {
  return d == 32 ? attention<T, 32>(a, p, stream) : d == 64 ? attention<T, 64>(a, p, stream) : attention<T, 128>(a, p, stream);
}

}  // namespace

extern "C" {

int tha4_quantize_tokens_i8(const void* x_dev, int x_dtype, int64_t rows, int64_t cols, int64_t x_row_stride, int8_t* q_dev, int64_t q_row_stride,
                            float* scale_dev, void* stream) {
  if (!known(x_dtype)) return bad("x_dtype must be f32, f16 or bf16");
  if (rows < 0 || cols < 1) return bad("rows must not be negative and cols must be positive");
  if (rows == 0) return THA4_OK;
  if (!x_dev || !q_dev || !scale_dev) return bad("x / q / scale must not be NULL");
  if (x_row_stride < 0 || q_row_stride < cols) return bad("x_row_stride must not be negative and q_row_stride must be at least cols");
  const int dev = one_device({x_dev, q_dev, scale_dev});
  if (dev < 0) return bad("x / q / scale must be device pointers of one GPU");
  DeviceGuard guard(dev);
  const QuantArgs a{x_dev, q_dev, scale_dev, rows, cols, x_row_stride, q_row_stride, 0};
  return x_dtype == THA4_F32 ? quantize<float>(a, stream) : x_dtype == THA4_F16 ? quantize<f16>(a, stream) : quantize<bf16>(a, stream);
}

int64_t tha4_linear_i8_workspace(const tha4_linear_i8_args* args) {
  if (!args) return bad("args must not be NULL");
  if (const char* e = check_linear(*args)) return bad(e);
  return args->x_dtype == THA4_I8 || inline_tokens(*args) ? 0 : args->m * (token_stride(*args) + 4);
}

int tha4_linear_i8(const tha4_linear_i8_args* args, void* stream) {
  if (!args) return bad("args must not be NULL");
  const tha4_linear_i8_args& g = *args;
  if (const char* e = check_linear(g)) return bad(e);
  if (g.m == 0 || g.n == 0) return THA4_OK;
  const bool quantised = g.x_dtype == THA4_I8;
  if (!g.x_dev || !g.w_dev || !g.w_scale_dev || !g.y_dev) return bad("x / w / w_scale / y must not be NULL");
  if (quantised != (g.x_scale_dev != nullptr)) return bad("x_scale belongs to an int8 x, and only there");
  if (g.x_row_stride < 0 || g.w_row_stride < 0 || g.y_row_stride < g.n) return bad("row strides must not be negative and y_row_stride must be at least n");
  const int64_t need = tha4_linear_i8_workspace(args);
  if (need && (!g.workspace_dev || g.workspace_bytes < need || reinterpret_cast<uintptr_t>(g.workspace_dev) % 16))
    return bad("workspace is smaller than tha4_linear_i8_workspace() or not 16-byte aligned");
  const int dev = one_device({g.x_dev, g.x_scale_dev, g.w_dev, g.w_scale_dev, g.bias_dev, g.y_dev, need ? g.workspace_dev : nullptr});
  if (dev < 0) return bad("x / x_scale / w / w_scale / bias / y / workspace must be device pointers of one GPU");
  DeviceGuard guard(dev);
  LinearArgs a{g.x_dev, g.w_dev, g.x_scale_dev, g.w_scale_dev, g.bias_dev, g.y_dev, g.m, g.n, g.k, g.x_row_stride, g.w_row_stride, g.y_row_stride, g.x_dtype, g.y_dtype};
  const bool w16 = g.k % 16 == 0 && aligned(g.w_dev, g.w_row_stride, 1);
  if (!quantised) {
    if (inline_tokens(g))
      return g.x_dtype == THA4_F32 ? few<float, 1, 1, true>(a, w16, stream) : g.x_dtype == THA4_F16 ? few<f16, 1, 1, true>(a, w16, stream) : few<bf16, 1, 1, true>(a, w16, stream);
    const int64_t stride = token_stride(g);
    int8_t* q = static_cast<int8_t*>(g.workspace_dev);
    float* scale = reinterpret_cast<float*>(q + g.m * stride);
    const QuantArgs t{g.x_dev, q, scale, g.m, g.k, g.x_row_stride, stride, 0};
    const int st = g.x_dtype == THA4_F32 ? quantize<float>(t, stream) : g.x_dtype == THA4_F16 ? quantize<f16>(t, stream) : quantize<bf16>(t, stream);
    if (st != THA4_OK) return st;
    a.x = q;
    a.xs = scale;
    a.x_stride = stride;
  }
  return product(a, w16 && aligned(a.x, a.x_stride, 1), stream);
}

int tha4_residual_norm(const tha4_residual_norm_args* args, void* stream) {
  if (!args) return bad("args must not be NULL");
  const tha4_residual_norm_args& g = *args;
  if (!known(g.dtype)) return bad("dtype must be f32, f16 or bf16");
  for (int t : {g.residual_dtype, g.gate_dtype, g.params_dtype})
    if (t != THA4_F32 && t != g.dtype) return bad("residual_dtype / gate_dtype / params_dtype must be f32 or dtype");
  for (int t : {g.post_norm, g.pre_norm})
    if (t != THA4_NORM_NONE && t != THA4_NORM_RMS && t != THA4_NORM_LAYER) return bad("unknown norm");
  if (g.gate_activation != THA4_GATE_LINEAR && g.gate_activation != THA4_GATE_SIGMOID) return bad("unknown gate activation");
  if (g.rows < 0 || g.cols < 1) return bad("rows must not be negative and cols must be positive");
  if (!(g.eps >= 0.0f) || !std::isfinite(g.residual_scale)) return bad("eps must not be negative and residual_scale must be finite");
  if (!g.residual_dev && g.rows) return bad("residual must not be NULL");
  if (!g.branch_dev && (g.gate_dev || g.post_weight_dev || g.post_bias_dev)) return bad("a gate or a post norm's weights need a branch");
  if (!g.film_scale_dev != !g.film_shift_dev) return bad("film_scale and film_shift come together");
  if (!g.y_dev && (g.film_scale_dev || g.pre_weight_dev || g.pre_bias_dev)) return bad("a pre norm's weights or FiLM need y");
  if (!g.h_dev && !g.y_dev && g.rows) return bad("one of h and y must be given");
  if (g.rows == 0) return THA4_OK;
  if ((g.gate_dev && g.gate_rows < 1) || (g.film_scale_dev && g.film_rows < 1)) return bad("gate_rows / film_rows must be positive");
  if (g.residual_row_stride < 0 || g.branch_row_stride < 0 || g.gate_row_stride < 0 || g.film_row_stride < 0) return bad("row strides must not be negative");
  if ((g.h_dev && g.h_row_stride < g.cols) || (g.y_dev && g.y_row_stride < g.cols)) return bad("output row strides must be at least cols");
  const int dev = one_device({g.residual_dev, g.branch_dev, g.gate_dev, g.residual_scale_vector_dev, g.post_weight_dev, g.post_bias_dev, g.pre_weight_dev,
                              g.pre_bias_dev, g.film_scale_dev, g.film_shift_dev, g.h_dev, g.y_dev});
  if (dev < 0) return bad("residual / branch / gate / weights / film / h / y must be device pointers of one GPU");
  DeviceGuard guard(dev);
  NormArgs a{g.residual_dev, g.branch_dev, g.gate_dev, g.residual_scale_vector_dev, g.post_weight_dev, g.post_bias_dev, g.pre_weight_dev, g.pre_bias_dev,
             g.film_scale_dev, g.film_shift_dev, g.h_dev, g.y_dev, g.rows, g.cols, g.residual_row_stride, g.branch_row_stride, g.gate_row_stride, g.film_row_stride,
             g.h_row_stride, g.y_row_stride, g.gate_rows, g.film_rows, 0, g.gate_dtype == THA4_F32, g.params_dtype == THA4_F32, g.post_norm, g.pre_norm,
             g.gate_activation == THA4_GATE_SIGMOID, g.residual_scale, g.eps, 1.0f / (float)g.cols};
  const int64_t st = size_of(g.dtype), sr = size_of(g.residual_dtype), sg = size_of(g.gate_dtype), sp = size_of(g.params_dtype);
  const bool vector = g.cols % 8 == 0 && aligned(g.residual_dev, g.residual_row_stride, sr) && aligned(g.branch_dev, g.branch_row_stride, st) &&
                      aligned(g.gate_dev, g.gate_dev ? g.gate_row_stride : 0, sg) && aligned(g.film_scale_dev, g.film_scale_dev ? g.film_row_stride : 0, sp) &&
                      aligned(g.film_shift_dev, 0, sp) && aligned(g.h_dev, g.h_dev ? g.h_row_stride : 0, sr) && aligned(g.y_dev, g.y_dev ? g.y_row_stride : 0, st) &&
                      aligned(g.residual_scale_vector_dev, 0, sp) && aligned(g.post_weight_dev, 0, sp) && aligned(g.post_bias_dev, 0, sp) &&
                      aligned(g.pre_weight_dev, 0, sp) && aligned(g.pre_bias_dev, 0, sp);
  if (g.dtype == THA4_F32) return norm<float, float>(a, vector, stream);
  if (g.dtype == THA4_F16) return g.residual_dtype == THA4_F32 ? norm<f16, float>(a, vector, stream) : norm<f16, f16>(a, vector, stream);
  return g.residual_dtype == THA4_F32 ? norm<bf16, float>(a, vector, stream) : norm<bf16, bf16>(a, vector, stream);
}

int64_t tha4_diff_attention_workspace(const tha4_diff_attention_args* args) {
  if (!args) return bad("args must not be NULL");
  if (const char* e = check_shape(*args)) return bad(e);
  const Plan p = plan_of(*args);
  return p.splits == 1 ? 0 : (int64_t)args->batch * args->kv_heads * p.row_tiles * p.part_rows * p.splits * part_floats(args->head_dim) * 4;
}

int tha4_diff_attention(const tha4_diff_attention_args* args, void* stream) {
  if (!args) return bad("args must not be NULL");
  const tha4_diff_attention_args& g = *args;
  if (const char* e = check_shape(g)) return bad(e);
  if (!(g.scale > 0.0f) || !std::isfinite(g.scale * kLog2e)) return bad("scale must be positive and finite, times log2(e) too");
  if (!(g.eps >= 0.0f) || !std::isfinite(g.lambda_init)) return bad("eps must not be negative and lambda_init must be finite");
  if (g.batch == 0 || g.q_len == 0) return THA4_OK;
  if (!g.q_dev || !g.out_dev || !g.lambda_vectors_dev) return bad("q / out / lambda_vectors must not be NULL");
  if (g.k_len && (!g.k_dev || !g.v_dev)) return bad("k / v must not be NULL");
  if (reinterpret_cast<uintptr_t>(g.q_dev) % 16 || reinterpret_cast<uintptr_t>(g.k_dev) % 16 || reinterpret_cast<uintptr_t>(g.v_dev) % 16 || reinterpret_cast<uintptr_t>(g.out_dev) % 8)
    return bad("q / k / v must be 16-byte aligned, out 8-byte");
  for (int i = 0; i < 3; ++i) {
    if (g.q_stride[i] % 8 || g.k_stride[i] % 8 || g.v_stride[i] % 8 || g.out_stride[i] % 4) return bad("strides of q / k / v must be multiples of 8 elements, of out of 4");
    if (i == 1 && (g.k_stride[i] >= (1 << 24) || g.v_stride[i] >= (1 << 24))) return bad("token strides of k / v must be below 2^24 elements");
    if (g.q_stride[i] < 0 || g.k_stride[i] < 0 || g.v_stride[i] < 0 || g.out_stride[i] < 0) return bad("strides must not be negative");
  }
  for (int i = 0; i < 4; ++i)
    if (g.mask_dev && g.mask_stride[i] < 0) return bad("strides must not be negative");
  if (g.lambda_vector_stride < 0 || g.lambda_head_stride < 0) return bad("strides must not be negative");
  if (overlaps_itself(g)) return bad("rows of out overlap each other");
  const Plan p = plan_of(g);
  const int64_t need = tha4_diff_attention_workspace(args);
  if (need && (!g.workspace_dev || g.workspace_bytes < need || reinterpret_cast<uintptr_t>(g.workspace_dev) % 16))
    return bad("workspace is smaller than tha4_diff_attention_workspace() or not 16-byte aligned");
  const int dev = one_device({g.q_dev, g.k_len ? g.k_dev : nullptr, g.k_len ? g.v_dev : nullptr, g.out_dev, g.lambda_vectors_dev, g.norm_weight_dev, g.q_lengths_dev,
                              g.kv_lengths_dev, g.k_len ? g.mask_dev : nullptr, need ? g.workspace_dev : nullptr});
  if (dev < 0) return bad("q / k / v / out / weights / lengths / mask / workspace must be device pointers of one GPU");
  DeviceGuard guard(dev);
  AttnArgs a{};
  a.q = g.q_dev; a.k = g.k_dev; a.v = g.v_dev; a.out = g.out_dev;
  a.lambdas = g.lambda_vectors_dev; a.norm_w = g.norm_weight_dev;
  a.q_lengths = g.q_lengths_dev; a.kv_lengths = g.kv_lengths_dev;
  a.mask = g.k_len ? g.mask_dev : nullptr;
  a.work = static_cast<float*>(g.workspace_dev);
  for (int i = 0; i < 3; ++i) { a.qs[i] = g.q_stride[i]; a.ks[i] = g.k_stride[i]; a.vs[i] = g.v_stride[i]; a.os[i] = g.out_stride[i]; }
  for (int i = 0; i < 4; ++i) a.ms[i] = g.mask_stride[i];
  a.lambda_vs = g.lambda_vector_stride; a.lambda_hs = g.lambda_head_stride;
  a.batch = g.batch; a.q_len = g.q_len; a.k_len = g.k_len; a.heads = g.heads; a.kv_heads = g.kv_heads; a.group = g.heads / g.kv_heads;
  a.causal = g.causal; a.norm = g.norm;
  a.row_tiles = p.row_tiles; a.splits = p.splits; a.chunk = p.chunk; a.part_rows = p.part_rows;
  a.c = g.scale * kLog2e; a.slack = (g.dtype == THA4_F16 ? Mat<f16>::SLACK : Mat<bf16>::SLACK) / a.c; a.lambda_init = g.lambda_init; a.eps = g.eps;
  return g.dtype == THA4_F16 ? attention<f16>(a, g.head_dim, p, stream) : attention<bf16>(a, g.head_dim, p, stream);
}

}  // extern "C"
