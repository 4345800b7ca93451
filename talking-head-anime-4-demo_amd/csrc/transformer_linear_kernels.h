// Quantisation of tokens to int8 (tha4_quantize_tokens_i8) and the int8 x int8 product with a scale for each token and channel (tha4_linear_i8):
//   y[i][j] = xs[i] ws[j] sum_k xq[i][k] wq[j][k] + b[j]
// The sums are exact integers (v_mfma_i32_*_i8), so neither the order of k nor a split of k over waves changes a result: both operands are read with k contiguous
// and any assignment of k to matrix-instruction slots is right as long as both operands use the same one.
#pragma once
#include "transformer_types.h"

namespace tha4 {
namespace xf {

// ---- quantisation ------------------------------------------------------------------------------------------------------------------------
struct QuantArgs {
  const void* x;
  int8_t* q;
  float* scale;
  int64_t rows, cols, x_stride, q_stride;
};

struct MaxU32 { THA4_DEV float operator()(float a, float b) const {          // of bit patterns without sign: orders inf and NaN behind every number
  const unsigned u = __float_as_uint(a), v = __float_as_uint(b);
  return __uint_as_float(u > v ? u : v);
} };
THA4_DEV float abs_bits(float v) { return __uint_as_float(__float_as_uint(v) & 0x7fffffffu); }

struct Step {                 // one row's scale, prepared for division
  float scale, s, inv, mul;
};
THA4_DEV Step make_step(float amax) {
  Step r;
  r.scale = __float_as_uint(amax) >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : amax / 127.0f;
  r.mul = r.scale < 7.9e-31f ? 18446744073709551616.0f : 1.0f;              // 2^64, exact: a scale near the subnormals has no finite reciprocal
  r.s = r.scale * r.mul;
  r.inv = r.s > 0.0f ? 1.0f / r.s : 0.0f;                                   // zero rows and NaN scales: zeros
  return r;
}
// the integer nearest to the exact quotient x / s, ties to even.  x * inv is off by at most a few 2^-17 at |127|; only where that could decide,
// the remainder x - q s settles it (one fma: exact, it has no more bits than x).
THA4_DEV int quantize1(float x, const Step& k) {
  if (!(k.inv > 0.0f)) return 0;
  x *= k.mul;
  const float t = x * k.inv;
  float q = rintf(t);
  if (fabsf(t - q) > 0.4998f) {
    const float r = fmaf(-q, k.s, x), half = 0.5f * k.s;
    if (r > half || (r == half && ((int)q & 1))) q += 1.0f;
    else if (r < -half || (r == -half && ((int)q & 1))) q -= 1.0f;
  }
  return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

// TPR threads share a row that stays in registers between the maximum and the rounding: read once
template <class T, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) quantize_kernel(QuantArgs a) {
  warm_kernarg<(int)sizeof(QuantArgs)>();
  constexpr int WAVES = TPR / 64, RPW = TPR < 256 ? 256 / TPR : 1;
  __shared__ float slots[RPW][WAVES];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int64_t row_ = (int64_t)blockIdx.x * RPW + sub;
  const bool live = row_ < a.rows;
  const int64_t row = live ? row_ : a.rows - 1;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  Raw8<T> raw[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = 8 * (j * TPR + t);
    raw[j] = fetch8(x + (c < a.cols ? c : 0));           // (a place behind the row reads the row's head again: no new maximum)
  }
  float m = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    float v[8];
    unpack8(raw[j], v);
#pragma unroll
    for (int e = 0; e < 8; ++e) m = MaxU32()(m, abs_bits(v[e]));
  }
  const Step k = make_step(row_reduce<WAVES>(m, MaxU32(), slots[sub], t / 64));
  if (!live) return;
  if (t == 0) a.scale[row] = k.scale;
  int8_t* q = a.q + row * a.q_stride;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = 8 * (j * TPR + t);
    if (c >= a.cols) continue;
    float v[8];
    unpack8(raw[j], v);
    unsigned w[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e / 4] |= ((unsigned)quantize1(v[e], k) & 255u) << (8 * (e % 4));
    *reinterpret_cast<uint2*>(q + c) = make_uint2(w[0], w[1]);
  }
}

// any alignment, any length: two passes over the row
template <class T>
__global__ void __launch_bounds__(256) quantize_any_kernel(QuantArgs a) {
  warm_kernarg<(int)sizeof(QuantArgs)>();
  __shared__ float slot[4];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  float m = 0.0f;
  for (int64_t c = threadIdx.x; c < a.cols; c += 256) m = MaxU32()(m, abs_bits((float)x[c]));
  const Step k = make_step(row_reduce<4>(m, MaxU32(), slot, threadIdx.x / 64));
  if (threadIdx.x == 0) a.scale[row] = k.scale;
  int8_t* q = a.q + row * a.q_stride;
  for (int64_t c = threadIdx.x; c < a.cols; c += 256) q[c] = (int8_t)quantize1((float)x[c], k);
}

// ---- product -----------------------------------------------------------------------------------------------------------------------------
struct LinearArgs {
  const int8_t *x, *w;
  const float *xs, *ws, *bias;
  void* y;
  int64_t m, n, k, x_stride, w_stride, y_stride;
  int32_t y_dtype;
};

THA4_DEV void store_y(void* y, int dtype, int64_t at, float v) {
  if (dtype == 0) static_cast<float*>(y)[at] = v;
  else if (dtype == 1) static_cast<f16*>(y)[at] = (f16)v;
  else static_cast<bf16*>(y)[at] = (bf16)v;
}

// 16 bytes of row `p` from element k on; elements at or behind `n` (the row's length) are zero.  ALIGNED: every 16-byte piece lies wholly inside or
// outside and is aligned; otherwise single bytes where the row ends inside the piece.
template <bool ALIGNED>
THA4_DEV i32x4 piece16(const int8_t* p, int64_t k, int64_t n) {
  i32x4 v = {0, 0, 0, 0};
  if (k >= n) return v;
  if (ALIGNED) return *reinterpret_cast<const i32x4*>(p + k);
  if (k + 16 <= n) {
    __builtin_memcpy(&v, p + k, 16);
    return v;
  }
#pragma unroll
  for (int i = 0; i < 15; ++i)
    if (k + i < n) v[i / 4] |= (int)(((unsigned)p[k + i] & 255u) << (8 * (i % 4)));
  return v;
}

// Few tokens: the weights are the traffic.  A workgroup owns 16 channels x 16 MT tokens; its 8 waves take turns of 128 k, weights straight from memory into matrix-instruction
// operands (nothing else would reuse them), and their exact partial sums meet in LDS.
template <int MT, bool ALIGNED>
__global__ void __launch_bounds__(512) linear_few_kernel(LinearArgs a) {
  warm_kernarg<(int)sizeof(LinearArgs)>();
  constexpr int WAVES = 8;
  __shared__ i32x4 part[WAVES][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * (16 * MT);
  const int64_t wr = n0 + r < a.n ? n0 + r : a.n - 1;                       // (a channel behind the last: the last again, not stored)
  const int8_t* w = a.w + wr * a.w_stride;
  const int8_t* x[MT];
  int64_t xk[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t row = m0 + 16 * i + r;
    xk[i] = row < a.m ? a.k : 0;                                            // a token behind the last: zeros, nothing is read
    x[i] = a.x + (row < a.m ? row : 0) * a.x_stride;
  }
  i32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = i32x4{0, 0, 0, 0};
  for (int64_t k0 = wave * 128; k0 < a.k; k0 += WAVES * 128) {
    i32x4 wf[2], xf[2][MT];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      wf[s] = piece16<ALIGNED>(w, k0 + 64 * s + 16 * g, a.k);
#pragma unroll
      for (int i = 0; i < MT; ++i) xf[s][i] = piece16<ALIGNED>(x[i], k0 + 64 * s + 16 * g, xk[i]);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[s], xf[s][i], acc[i], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) part[wave][i][lane] = acc[i];
  __syncthreads();
  for (int u = threadIdx.x; u < MT * 64; u += 512) {
    const int i = u >> 6, l = u & 63;
    i32x4 s = part[0][i][l];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) s += part[v][i][l];
    const int64_t row = m0 + 16 * i + (l & 15);
    if (row >= a.m) continue;
    const float xs = a.xs[row];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t col = n0 + 4 * (l >> 4) + e;
      if (col >= a.n) continue;
      float v = (float)s[e] * xs * a.ws[col];
      if (a.bias) v += a.bias[col];
      store_y(a.y, a.y_dtype, row * a.y_stride + col, v);
    }
  }
}

// Many tokens: 128 x 128 outputs a workgroup, four waves of 64 x 64 (2 x 2 matrix tiles of 32 x 32), operands through LDS in steps of 64 k.
// 16-byte pieces of a row are permuted by (row / 4) mod 4, so that the 16 lanes the LDS serves together hit 16 different 16-byte slots.
template <bool ALIGNED>
__global__ void __launch_bounds__(256) linear_tile_kernel(LinearArgs a) {
  warm_kernarg<(int)sizeof(LinearArgs)>();
  constexpr int BM = 128, BN = 128, BK = 64;
  __shared__ __attribute__((aligned(16))) char lx[BM * BK], lw[BN * BK];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t m0 = (int64_t)blockIdx.y * BM, n0 = (int64_t)blockIdx.x * BN;
  const int wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
  i32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = i32x16{0};
  for (int64_t k0 = 0; k0 < a.k; k0 += BK) {
    i32x4 fx[2], fw[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int id = threadIdx.x + 256 * u, row = id >> 2, p = (id & 3) ^ ((row >> 2) & 3);
      const int64_t rx = m0 + row < a.m ? m0 + row : a.m - 1, rw = n0 + row < a.n ? n0 + row : a.n - 1;
      fx[u] = piece16<ALIGNED>(a.x + rx * a.x_stride, k0 + 16 * p, a.k);
      fw[u] = piece16<ALIGNED>(a.w + rw * a.w_stride, k0 + 16 * p, a.k);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      *reinterpret_cast<i32x4*>(lx + 16 * (threadIdx.x + 256 * u)) = fx[u];
      *reinterpret_cast<i32x4*>(lw + 16 * (threadIdx.x + 256 * u)) = fw[u];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      i32x4 xf[2], wf[2];
      const int c = 2 * s + (lane >> 5);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int rx = wm + 32 * i + (lane & 31), rw = wn + 32 * i + (lane & 31);
        xf[i] = *reinterpret_cast<const i32x4*>(lx + rx * BK + 16 * (c ^ ((rx >> 2) & 3)));
        wf[i] = *reinterpret_cast<const i32x4*>(lw + rw * BK + 16 * (c ^ ((rw >> 2) & 3)));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xf[i], wf[j], acc[i][j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t col = n0 + wn + 32 * j + (lane & 31);
    if (col >= a.n) continue;
    const float ws = a.ws[col], b = a.bias ? a.bias[col] : 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t row = m0 + wm + 32 * i + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
        if (row < a.m) store_y(a.y, a.y_dtype, row * a.y_stride + col, (float)acc[i][j][e] * a.xs[row] * ws + b);
      }
  }
}

}  // namespace xf
}  // namespace tha4
