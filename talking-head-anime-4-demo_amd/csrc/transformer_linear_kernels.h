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
  int64_t first;               // row of the launch's first workgroup
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

THA4_DEV uint2 quantize8(const float (&v)[8], const Step& k) {
  unsigned w[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e / 4] |= ((unsigned)quantize1(v[e], k) & 255u) << (8 * (e % 4));
  return make_uint2(w[0], w[1]);
}

// TPR threads share a row that stays in registers between the maximum and the rounding: read once (8192 x 8192: bf16 37 us, fp32 60 us, 5.4 - 5.6 TB/s: a copy's rate)
template <class T, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) quantize_kernel(QuantArgs a) {
  warm_kernarg<(int)sizeof(QuantArgs)>();
  constexpr int WAVES = TPR / 64, RPW = TPR < 256 ? 256 / TPR : 1;
  __shared__ float slots[RPW][WAVES];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int64_t row_ = a.first + (int64_t)blockIdx.x * RPW + sub;
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
    *reinterpret_cast<uint2*>(q + c) = quantize8(v, k);
  }
}

// any alignment, any length: two passes over the row
template <class T>
__global__ void __launch_bounds__(256) quantize_any_kernel(QuantArgs a) {
  warm_kernarg<(int)sizeof(QuantArgs)>();
  __shared__ float slot[4];
  const int64_t row = a.first + blockIdx.x;
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
  const void* x;               // int8 [m][k], or (linear_few_kernel<.., INLINE>) the float tokens themselves
  const int8_t* w;
  const float *xs, *ws, *bias;
  void* y;
  int64_t m, n, k, x_stride, w_stride, y_stride;
  int32_t x_dtype, y_dtype;
};

THA4_DEV void store_y(void* y, int dtype, int64_t at, float v) {
  if (dtype == 0) static_cast<float*>(y)[at] = v;
  else if (dtype == 1) static_cast<f16*>(y)[at] = (f16)v;
  else static_cast<bf16*>(y)[at] = (bf16)v;
}

// 16 bytes of row `p` from element k on; elements at or behind `n` (the row's length) are zero.  ALIGNED: every 16-byte piece lies wholly inside or
// outside and is aligned.  Otherwise a piece that the row ends in is the row's last 16 bytes, shifted: one load either way (777 x 1001 x 1111 from fp32: 20.3 us, byte by byte 20.6).
template <bool ALIGNED>
THA4_DEV i32x4 piece16(const int8_t* p, int64_t k, int64_t n) {
  i32x4 v = {0, 0, 0, 0};
  if (k >= n) return v;
  if (ALIGNED) return *reinterpret_cast<const i32x4*>(p + k);
  if (n >= 16) {
    const int64_t at = k + 16 <= n ? k : n - 16;
    unsigned __int128 t;
    __builtin_memcpy(&t, p + at, 16);
    return __builtin_bit_cast(i32x4, t >> (8 * (int)(k - at)));              // (0 <= k - at < 16)
  }
#pragma unroll
  for (int i = 0; i < 15; ++i)                                               // rows shorter than a piece
    if (k + i < n) v[i / 4] |= (int)(((unsigned)p[k + i] & 255u) << (8 * (i % 4)));
  return v;
}

// Few tokens: the weights are the traffic.  A workgroup owns 16 NT channels x 16 MT tokens; its 8 waves take turns of 128 k, weights straight from memory into
// matrix-instruction operands (nothing else would reuse them), AHEAD turns of them on their way at any time, and their exact partial sums meet in LDS.  Every workgroup reads all the tokens, through L2: with 16 of them and one tile of channels that is as much again as the weights.
// NT tiles for each token operand where there are channels enough to fill the GPU (16 x 16384 x 8192: NT 1 38.9 us, 2 35.6, 4 32.7 = 4.1 TB/s; one token: NT 1 28.1 us = 4.8 TB/s, 4 30.6).
// INLINE: x is float (XT), m <= kInlineTokens and m k <= kInlineBytes (one token may have 32768 elements): every workgroup quantises the tokens itself, into LDS, while its first weights are on their
// way - a few hundred instructions against a launch of their own.
constexpr int kInlineTokens = 4, kInlineBytes = 32768;

template <class XT, int NT, int MT, bool ALIGNED, bool INLINE>
__global__ void __launch_bounds__(512) linear_few_kernel(LinearArgs a) {
  warm_kernarg<(int)sizeof(LinearArgs)>();
  constexpr int WAVES = 8, AHEAD = NT * MT >= 4 ? 1 : NT * MT == 2 ? 2 : 4;
  __shared__ i32x4 part[WAVES][NT * MT][64];
  __shared__ __attribute__((aligned(16))) int8_t xq[INLINE ? kInlineBytes : 16];
  __shared__ float xscale[INLINE ? kInlineTokens : 1], slot[WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), m0 = (int64_t)blockIdx.y * (16 * MT);
  const int8_t* w[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) w[i] = a.w + (n0 + 16 * i + r < a.n ? n0 + 16 * i + r : a.n - 1) * a.w_stride;   // (a channel behind the last: the last again, not stored)
  const int8_t* x[MT];
  int64_t xk[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t row = m0 + 16 * i + r;
    xk[i] = row < a.m ? a.k : 0;                                            // a token behind the last: zeros, nothing is read
    x[i] = INLINE ? xq + (row < a.m ? row : 0) * a.k : static_cast<const int8_t*>(a.x) + (row < a.m ? row : 0) * a.x_stride;
  }
  i32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT * MT; ++i) acc[i / MT][i % MT] = i32x4{0, 0, 0, 0};
  i32x4 wf[AHEAD][2][NT], xf[AHEAD][2][MT];
  auto weights = [&](int t, int64_t k0) {                                   // (behind the row's end: zeros, nothing is read)
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < NT; ++i) wf[t][s][i] = piece16<ALIGNED>(w[i], k0 + 64 * s + 16 * g, a.k);
  };
  auto tokens = [&](int t, int64_t k0) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < MT; ++i) xf[t][s][i] = piece16<ALIGNED>(x[i], k0 + 64 * s + 16 * g, xk[i]);
  };
#pragma unroll
  for (int t = 0; t < AHEAD; ++t) {
    weights(t, (t * WAVES + wave) * 128);
    if constexpr (!INLINE) tokens(t, (t * WAVES + wave) * 128);
  }
  if constexpr (INLINE) {
    // 16-byte aligned tokens of at most 8 x 512 elements stay in registers between their maximum and their rounding
    const bool vec = a.k % 8 == 0 && a.k <= 8 * 512 && reinterpret_cast<size_t>(a.x) % 16 == 0 && a.x_stride * sizeof(XT) % 16 == 0;
    const int c8 = 8 * (int)threadIdx.x;
    for (int row = 0; row < a.m; ++row) {
      const XT* from = static_cast<const XT*>(a.x) + row * a.x_stride;
      float m = 0.0f, v[8];
      if (vec) {
        unpack8(fetch8(from + (c8 < a.k ? c8 : 0)), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = MaxU32()(m, abs_bits(v[e]));
      } else {
        for (int c = threadIdx.x; c < a.k; c += 512) m = MaxU32()(m, abs_bits((float)from[c]));
      }
      const Step k = make_step(row_reduce<WAVES>(m, MaxU32(), slot, wave));
      if (threadIdx.x == 0) xscale[row] = k.scale;
      if (!vec) {
        for (int c = threadIdx.x; c < a.k; c += 512) xq[row * a.k + c] = (int8_t)quantize1((float)from[c], k);
      } else if (c8 < a.k) {
        *reinterpret_cast<uint2*>(xq + row * a.k + c8) = quantize8(v, k);
      }
      __syncthreads();                                                      // (slot is free again; after the last row: everything is there)
    }
  }
  for (int64_t k0 = wave * 128; k0 < a.k; k0 += AHEAD * WAVES * 128) {
#pragma unroll
    for (int t = 0; t < AHEAD; ++t) {
      const int64_t at = k0 + t * (WAVES * 128), next = at + AHEAD * WAVES * 128;
      if constexpr (INLINE) tokens(t, at);
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < NT * MT; ++i) acc[i / MT][i % MT] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[t][s][i / MT], xf[t][s][i % MT], acc[i / MT][i % MT], 0, 0, 0);
      weights(t, next);
      if constexpr (!INLINE) tokens(t, next);
    }
  }
#pragma unroll
  for (int i = 0; i < NT * MT; ++i) part[wave][i][lane] = acc[i / MT][i % MT];
  __syncthreads();
  for (int u = threadIdx.x; u < NT * MT * 64; u += 512) {
    const int i = u >> 6, l = u & 63;
    i32x4 s = part[0][i][l];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) s += part[v][i][l];
    const int64_t row = m0 + 16 * (i % MT) + (l & 15);
    if (row >= a.m) continue;
    const float xs = INLINE ? xscale[row] : a.xs[row];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t col = n0 + 16 * (i / MT) + 4 * (l >> 4) + e;
      if (col >= a.n) continue;
      float v = (float)s[e] * xs * a.ws[col];
      if (a.bias) v += a.bias[col];
      store_y(a.y, a.y_dtype, row * a.y_stride + col, v);
    }
  }
}

// Many tokens: BM tokens x BN channels a workgroup of WM x WN waves (times G groups that take turns along k: where there are few tiles, more of a row is on its way at once), operands through LDS in stages of BK k.
//  * 16-byte pieces of a row are permuted (swizzle), so that the 16 lanes the LDS serves together hit 16 different 16-byte slots.
//  * DMA (aligned rows): STAGES stages of LDS, filled by asynchronous copies up to three stages ahead behind counted waits - one barrier a stage, which both
//    publishes the next stage and frees this one.  Otherwise rows go through registers, one stage ahead.
//  * Stages of 128 k: a copy moves whole 128-byte lines (8192^3: stages of 64 k 577 us, of 128 k 531 us, tokens' quantisation included).
//  * 256 x 256 tiles: 8192^3 in 488 us, 2250 TOP/s, beside 490 - 530 us of the library's int8 product without scales.  Matrix pipes 52 % busy by the counters, at 1.9 - 2.0 GHz: power
//    sets the clock (an earlier form took 620 us on random numbers and 458 on zeros), the rest is the wait for LDS and the barrier at a stage's head.
//  * Channels are the matrix tile's rows, dealt so that a lane ends with 16 consecutive channels of one token: the result leaves in 16-byte stores.
__device__ const i32x4 g_zero16 = {0, 0, 0, 0};                              // what a copy reads behind a row's end

constexpr int kBand = 4;

template <int BM, int BN, int BK, int WM, int WN, int G, int STAGES, bool DMA>
__global__ void __launch_bounds__(64 * WM * WN * G) linear_tile_kernel(LinearArgs a) {
  warm_kernarg<(int)sizeof(LinearArgs)>();
  constexpr int WAVES = WM * WN, FM = BM / WM / 32, FN = BN / WN / 32;      // 32 x 32 tiles of a wave
  constexpr int STAGE = (BM + BN) * BK, PIECES = STAGE / 1024 / WAVES;               // 1-KiB copies of a wave and stage
  static_assert(PIECES * WAVES * 1024 == STAGE && (BM * BK / 1024) % WAVES == 0, "a copy moves rows of one operand");
  constexpr int RING = (DMA ? STAGES : 1) * STAGE;                                    // bytes of one group's stages
  __shared__ __attribute__((aligned(16))) char lds_all[G * RING];
  static_assert(G == 1 || (G - 1) * BM * BN * 4 <= G * RING, "the groups' sums meet in the stages");
  const int lane = threadIdx.x & 63, wave = uniform_i32(threadIdx.x >> 6) % WAVES, group_k = uniform_i32(threadIdx.x >> 6) / WAVES, h = lane >> 5;
  char* lds = lds_all + group_k * RING;
  // Order of the tiles: blockIdx.x goes round the eight XCDs, so each gets a contiguous eighth of an order in which kBand bands of tokens run together, column by column: the tiles
  // an XCD has in flight (32 CUs) form a block of 4 x 8, whose rows of x and w its L2 reads once for all of them (8192^3: 1 band 608 us, 4 bands 579 us, 8 585 us, 16 600 us).
  const int tiles_n = (int)((a.n + BN - 1) / BN), tiles_m = (int)((a.m + BM - 1) / BM);
  int id = blockIdx.x;
  const int even = tiles_m * tiles_n / 8 * 8;
  if (id < even) id = (id % 8) * (even / 8) + id / 8;
  const int group = id / (kBand * tiles_n), bands = min(kBand, tiles_m - group * kBand);
  id -= group * kBand * tiles_n;
  const int64_t m0 = (int64_t)(group * kBand + id % bands) * BM, n0 = (int64_t)(id / bands) * BN;
  const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);

  // this lane's place in each copy: rows of P 16-byte pieces, 64 pieces a copy
  constexpr int P = BK / 16;
  static_assert((P == 4 || P == 8) && WAVES * (64 / P) % 16 == 0, "a 256-byte line of LDS holds four or two rows; a wave's copies lie 16 rows apart or a multiple");
  auto swizzle = [](int row) { return (row / (16 / P)) & (P - 1); };
  const int8_t* from[PIECES];
#pragma unroll
  for (int u = 0; u < PIECES; ++u) {
    const int row = (u * WAVES + wave) * (64 / P) + lane / P;
    const int64_t rx = m0 + row < a.m ? m0 + row : a.m - 1, rw = n0 + row - BM < a.n ? n0 + row - BM : a.n - 1;
    from[u] = u * WAVES * (64 / P) < BM ? static_cast<const int8_t*>(a.x) + rx * a.x_stride : a.w + rw * a.w_stride;
  }
  const int piece = 16 * ((lane % P) ^ swizzle(wave * (64 / P) + lane / P));           // (the permutation repeats after 16 rows: the same in every copy of the wave)
  const int stages = (int)((a.k + BK * G - 1) / (BK * G));                            // of each group; one behind the row's end is zeros

  i32x16 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = i32x16{0};
  const int ch = 16 * ((lane >> 2) & 1) + 4 * ((lane & 31) >> 3) + (lane & 3);         // row of the matrix tile -> channel
  struct Operands { i32x4 x[FM], w[FN]; };
  auto fetch = [&](const char* stage, int s, Operands& f) {                            // step s (32 k) of a stage
    const int c = 2 * s + h;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int row = wm + 32 * j + (lane & 31);
      f.x[j] = *reinterpret_cast<const i32x4*>(stage + row * BK + 16 * (c ^ swizzle(row)));
    }
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      const int row = wn + 32 * i + ch;
      f.w[i] = *reinterpret_cast<const i32x4*>(stage + (BM + row) * BK + 16 * (c ^ swizzle(row)));
    }
  };
  auto multiply = [&](const Operands& f) {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[i], f.x[j], acc[i][j], 0, 0, 0);
  };

  if constexpr (DMA) {
    const unsigned base = lds_address(lds);
    auto request = [&](int t) {
      const int64_t at = ((int64_t)t * G + group_k) * BK + piece;
#pragma unroll
      for (int u = 0; u < PIECES; ++u)
        copy16_async(at < a.k ? (const void*)(from[u] + at) : (const void*)&g_zero16, base + (t % STAGES) * STAGE + (u * WAVES + wave) * 1024);
    };
#pragma unroll
    for (int t = 0; t < STAGES; ++t)
      if (t < stages) request(t);
    THA4_BARRIER_KEEP(min(stages - 1, STAGES - 1) * PIECES);                           // stage 0 is there
    // Operands of a step are read from LDS under the products of the step before; the barrier that publishes the next stage stands in front of the last products of this one, behind
    // this wave's last reads of it, so a wave never waits for a barrier and for LDS with nothing to multiply
    Operands f[2];
    fetch(lds, 0, f[0]);
    for (int t = 0; t < stages; ++t) {
#pragma unroll
      for (int u = 0; u < BK / 32; ++u) {
        if (u + 1 < BK / 32) {
          fetch(lds + (t % STAGES) * STAGE, u + 1, f[(u + 1) & 1]);
        } else if (t + 1 < stages) {
          THA4_BARRIER_KEEP(min(stages - 2 - t, STAGES - 2) * PIECES);
          if (t + STAGES < stages) request(t + STAGES);                                // into the stage that everybody has read
          fetch(lds + ((t + 1) % STAGES) * STAGE, 0, f[0]);
        }
        THA4_SCHED_FENCE();
        multiply(f[u & 1]);
      }
    }
  } else {
    i32x4 hold[PIECES];
    auto request = [&](int t) {
#pragma unroll
      for (int u = 0; u < PIECES; ++u) hold[u] = piece16<false>(from[u], ((int64_t)t * G + group_k) * BK + piece, a.k);
    };
    request(0);
    for (int t = 0; t < stages; ++t) {
      __syncthreads();
#pragma unroll
      for (int u = 0; u < PIECES; ++u) *reinterpret_cast<i32x4*>(lds + (u * WAVES + wave) * 1024 + 16 * lane) = hold[u];
      __syncthreads();
      if (t + 1 < stages) request(t + 1);
#pragma unroll
      for (int u = 0; u < BK / 32; ++u) {
        Operands f;
        fetch(lds, u, f);
        multiply(f);
      }
    }
  }

  if constexpr (G > 1) {                                                               // integer sums: no order to keep
    i32x4* meet = reinterpret_cast<i32x4*>(lds_all) + wave * (FN * FM * 4 * 64) + lane;
    constexpr int SET = WAVES * FN * FM * 4 * 64;
    __syncthreads();
    if (group_k) {
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            meet[(group_k - 1) * SET + ((i * FM + j) * 4 + e) * 64] = i32x4{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
    }
    __syncthreads();
    if (group_k) return;
#pragma unroll
    for (int v = 0; v < G - 1; ++v)
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const i32x4 o = meet[v * SET + ((i * FM + j) * 4 + e) * 64];
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][4 * e + r] += o[r];
            THA4_SCHED_FENCE();
          }
  }
  const bool vec = a.n % 8 == 0 && a.y_stride % 8 == 0 && (reinterpret_cast<size_t>(a.y) & 15) == 0;
#pragma unroll
  for (int i = 0; i < FN; ++i) {
#pragma unroll
    for (int o = 0; o < 16; o += 8) {
      const int64_t col = n0 + wn + 32 * i + 16 * h + o;
      float ws[8], b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int64_t c = col + e < a.n ? col + e : a.n - 1;
        ws[e] = a.ws[c];
        b[e] = a.bias ? a.bias[c] : 0.0f;
      }
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        const int64_t row = m0 + wm + 32 * j + (lane & 31);
        if (row >= a.m) continue;
        const float xs = a.xs[row];
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf((float)acc[i][j][o + e] * xs, ws[e], b[e]);
        const int64_t at = row * a.y_stride + col;
        if (vec && col < a.n) {
          if (a.y_dtype == 0) put8(static_cast<float*>(a.y) + at, v);
          else if (a.y_dtype == 1) put8(static_cast<f16*>(a.y) + at, v);
          else put8(static_cast<bf16*>(a.y) + at, v);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (col + e < a.n) store_y(a.y, a.y_dtype, at + e, v[e]);
        }
      }
    }
  }
}

}  // namespace xf
}  // namespace tha4
