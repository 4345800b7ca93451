// The norms around a block, fused with its gate, the residual sum and FiLM (tha4_residual_norm):
//   h = rs * residual + act(gate) * (post(branch) * wp + bp),   y = (pre(h) * wq + bq) * (1 + s) + t
// A row's two means depend on each other (the second norm is of h, which needs the first), so a row stays in registers from its first load to
// its last store: every input is read once and every output written once, which is the floor of a memory-bound operator.
#pragma once
#include "transformer_types.h"

namespace tha4 {
namespace xf {

struct NormArgs {
  const void *residual, *branch, *gate, *rsv, *post_w, *post_b, *pre_w, *pre_b, *film_s, *film_t;
  void *h, *y;
  int64_t rows, cols;
  int64_t residual_stride, branch_stride, gate_stride, film_stride, h_stride, y_stride;
  int64_t gate_rows, film_rows;
  int64_t first;               // row of the launch's first workgroup
  int32_t gate_f32, params_f32, post_norm, pre_norm, sigmoid;
  float residual_scale, eps, inv_cols;
};

THA4_DEV float sigmoid(float v) { return 1.0f / (1.0f + __expf(-v)); }     // v -> -inf: 1 / inf = 0

// TPR threads share a row; thread t of the row owns elements 8 (j TPR + t) .. + 7, j < NV (a wave's loads are contiguous runs of 1 KiB).
// Measured (rows x cols, bytes over time; a large copy moves 5.1 TB/s): 16384 x 8192 bf16 with a full gate 255 us, 5.3 TB/s; 65536 x 1024 5.5 TB/s on one wave a row (3.9 on
// four); 262144 x 256 fp32 5.5 TB/s.  8192 x 16384 4.1 TB/s: one workgroup of 16 waves fills a CU's registers, and nothing runs under its reductions.  8192 columns on 512
// threads rather than 256: 307 -> 255 us (registers: five waves a SIMD instead of three).
// Statistics: the sum of squares (rms), or the mean first and the squares of the differences then (layer): no cancellation.
template <class T, class R, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) residual_norm_kernel(NormArgs a) {
  warm_kernarg<(int)sizeof(NormArgs)>();
  constexpr int WAVES = TPR / 64, RPW = TPR < 256 ? 256 / TPR : 1;
  __shared__ float slots[4][RPW][WAVES];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, wave = t / 64;
  const int64_t row_ = a.first + (int64_t)blockIdx.x * RPW + sub;
  const bool live = row_ < a.rows;                       // a row behind the last: the same work on the last row, no stores (the barriers stay uniform)
  const int64_t row = live ? row_ : a.rows - 1;
  const T* branch = static_cast<const T*>(a.branch) + row * a.branch_stride;
  const R* residual = static_cast<const R*>(a.residual) + row * a.residual_stride;
  const int64_t gate_at = a.gate ? (row / a.gate_rows) * a.gate_stride : 0;
  const int64_t film_at = a.film_s ? (row / a.film_rows) * a.film_stride : 0;
  const bool pf = a.params_f32 != 0;

  float h[NV][8];
  Raw8<R> res[NV];
  Raw8<T> gate[NV];                                      // (of the gate's own type only if that is T; an fp32 gate beside 16-bit rows is read where it is used)
  bool in[NV];
  int c[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    c[j] = 8 * (j * TPR + t);
    in[j] = c[j] < a.cols;
    if (!in[j]) c[j] = 0;                                // (a valid place; its values are zeroed below)
  }
  if (a.branch) {
    Raw8<T> raw[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) raw[j] = fetch8(branch + c[j]);
#pragma unroll
    for (int j = 0; j < NV; ++j) res[j] = fetch8(residual + c[j]);
    const bool gate_here = a.gate && (std::is_same<T, float>::value || !a.gate_f32);
    if (gate_here) {
#pragma unroll
      for (int j = 0; j < NV; ++j) gate[j] = fetch8(static_cast<const T*>(a.gate) + gate_at + c[j]);
    }
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      unpack8(raw[j], h[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) { h[j][e] = in[j] ? h[j][e] : 0.0f; }
    }
    if (a.post_norm == 2) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += h[j][e];
      const float mean = row_reduce<WAVES>(sum, Add(), slots[0][sub], wave) * a.inv_cols;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) h[j][e] = in[j] ? h[j][e] - mean : 0.0f;
    }
    float k = 1.0f;
    if (a.post_norm) {
      sum = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(h[j][e], h[j][e], sum);
      k = 1.0f / sqrtf(row_reduce<WAVES>(sum, Add(), slots[1][sub], wave) * a.inv_cols + a.eps);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float w[8], b[8], r[8], g[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) { w[e] = 1.0f; b[e] = 0.0f; }
      if (a.post_w) param8<T>(a.post_w, c[j], pf, w);
      if (a.post_b) param8<T>(a.post_b, c[j], pf, b);
      unpack8(res[j], r);
      if (gate_here) unpack8(gate[j], g);
      else if (a.gate) unpack8(fetch8(static_cast<const float*>(a.gate) + gate_at + c[j]), g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = fmaf(h[j][e] * k, w[e], b[e]);
        if (a.gate) v *= a.sigmoid ? sigmoid(g[e]) : g[e];
        h[j][e] = v;
        r[e] *= a.residual_scale;
      }
      if (a.rsv) {
        param8<T>(a.rsv, c[j], pf, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] *= w[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) h[j][e] = in[j] ? h[j][e] + r[e] : 0.0f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) res[j] = fetch8(residual + c[j]);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      unpack8(res[j], h[j]);
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 1.0f;
      if (a.rsv) param8<T>(a.rsv, c[j], pf, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[j][e] = in[j] ? h[j][e] * a.residual_scale * w[e] : 0.0f;
    }
  }
  if (a.h && live) {
    R* out = static_cast<R*>(a.h) + row * a.h_stride;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (in[j]) put8(out + c[j], h[j]);
  }
  if (!a.y) return;
  float sum = 0.0f, k = 1.0f;
  if (a.pre_norm == 2) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += h[j][e];
    const float mean = row_reduce<WAVES>(sum, Add(), slots[2][sub], wave) * a.inv_cols;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[j][e] = in[j] ? h[j][e] - mean : 0.0f;
  }
  if (a.pre_norm) {
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(h[j][e], h[j][e], sum);
    k = 1.0f / sqrtf(row_reduce<WAVES>(sum, Add(), slots[3][sub], wave) * a.inv_cols + a.eps);
  }
  if (!live) return;
  T* out = static_cast<T*>(a.y) + row * a.y_stride;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (!in[j]) continue;
    float w[8], b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) { w[e] = 1.0f; b[e] = 0.0f; }
    if (a.pre_w) param8<T>(a.pre_w, c[j], pf, w);
    if (a.pre_b) param8<T>(a.pre_b, c[j], pf, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[j][e] = fmaf(h[j][e] * k, w[e], b[e]);
    if (a.film_s) {
      param8<T>(a.film_s, film_at + c[j], pf, w);
      param8<T>(a.film_t, film_at + c[j], pf, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[j][e] = fmaf(h[j][e], w[e], h[j][e] + b[e]);
    }
    put8(out + c[j], h[j]);
  }
}

// Rows that are not 16-byte aligned or multiples of 8 long, or longer than the registers of a workgroup hold: element by element, the row read again in each
// pass (from the caches: a row is at most a few hundred KiB).  h is recomputed from the inputs, so nothing depends on h having been stored.
template <class T, class R>
__global__ void __launch_bounds__(256) residual_norm_any_kernel(NormArgs a) {
  warm_kernarg<(int)sizeof(NormArgs)>();
  __shared__ float slots[4][4];
  const int64_t row = a.first + blockIdx.x;
  const int t = threadIdx.x, wave = t / 64;
  const T* branch = static_cast<const T*>(a.branch) + row * a.branch_stride;
  const R* residual = static_cast<const R*>(a.residual) + row * a.residual_stride;
  const int64_t gate_at = a.gate ? (row / a.gate_rows) * a.gate_stride : 0;
  const int64_t film_at = a.film_s ? (row / a.film_rows) * a.film_stride : 0;
  const bool pf = a.params_f32 != 0;
  float mean = 0.0f, k = 1.0f, sum;
  if (a.branch && a.post_norm == 2) {
    sum = 0.0f;
    for (int64_t c = t; c < a.cols; c += 256) sum += (float)branch[c];
    mean = row_reduce<4>(sum, Add(), slots[0], wave) * a.inv_cols;
  }
  if (a.branch && a.post_norm) {
    sum = 0.0f;
    for (int64_t c = t; c < a.cols; c += 256) { const float v = (float)branch[c] - mean; sum = fmaf(v, v, sum); }
    k = 1.0f / sqrtf(row_reduce<4>(sum, Add(), slots[1], wave) * a.inv_cols + a.eps);
  }
  auto h_at = [&](int64_t c) {
    float r = (float)residual[c] * a.residual_scale;
    if (a.rsv) r *= param1<T>(a.rsv, c, pf);
    if (!a.branch) return r;
    float v = ((float)branch[c] - mean) * k;
    v = fmaf(v, a.post_w ? param1<T>(a.post_w, c, pf) : 1.0f, a.post_b ? param1<T>(a.post_b, c, pf) : 0.0f);
    if (a.gate) {
      const float g = param1<T>(a.gate, gate_at + c, a.gate_f32 != 0);
      v *= a.sigmoid ? sigmoid(g) : g;
    }
    return v + r;
  };
  sum = 0.0f;
  R* hout = static_cast<R*>(a.h) + row * a.h_stride;
  for (int64_t c = t; c < a.cols; c += 256) {
    const float v = h_at(c);
    if (a.h) hout[c] = (R)v;
    sum += a.pre_norm == 2 ? v : v * v;
  }
  if (!a.y) return;
  float mean2 = 0.0f, k2 = 1.0f;
  if (a.pre_norm) {
    sum = row_reduce<4>(sum, Add(), slots[2], wave) * a.inv_cols;
    if (a.pre_norm == 2) {
      mean2 = sum;
      sum = 0.0f;
      for (int64_t c = t; c < a.cols; c += 256) { const float v = h_at(c) - mean2; sum = fmaf(v, v, sum); }
      sum = row_reduce<4>(sum, Add(), slots[3], wave) * a.inv_cols;
    }
    k2 = 1.0f / sqrtf(sum + a.eps);
  }
  T* out = static_cast<T*>(a.y) + row * a.y_stride;
  for (int64_t c = t; c < a.cols; c += 256) {
    float v = (h_at(c) - mean2) * k2;
    v = fmaf(v, a.pre_w ? param1<T>(a.pre_w, c, pf) : 1.0f, a.pre_b ? param1<T>(a.pre_b, c, pf) : 0.0f);
    if (a.film_s) v = fmaf(v, param1<T>(a.film_s, film_at + c, pf), v + param1<T>(a.film_t, film_at + c, pf));
    out[c] = (T)v;
  }
}

}  // namespace xf
}  // namespace tha4
