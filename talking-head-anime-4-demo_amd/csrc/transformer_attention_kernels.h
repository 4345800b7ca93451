// Differential attention (tha4_diff_attention): for each head two softmax maps over the same keys and one value matrix of twice the width,
//   o = softmax(s q1 k1^T) v - lambda softmax(s q2 k2^T) v,   out = (1 - lambda_init) o / sqrt(mean(o^2) + eps) w
// One pass over the keys with the running maximum m and sum l of each map:  p = exp(s x - m), l = sum p, O = sum p v, out of which O / l.
//
// Every product is written transposed, with the queries along the matrix instruction's columns:  S^T = K Q^T and O^T = V^T P^T.  A lane then holds scores of ONE
// query (column lane % 32 or lane % 16): maxima and sums are registers of the lane plus one exchange with the lanes of the same column, a
// rescale is one multiplier a lane, and the accumulator layout of S^T is already an operand layout for P^T - which key sits in which k slot of the
// product with V is free as long as V^T uses the same order, so P never leaves its registers.  V^T operands come from row-major V in LDS by the transposing read
// ds_read_b64_tr_b16 (four keys of one column a lane).
//
// Precision: scores, maxima, sums, accumulators, lambda and the norm are fp32.  A weight p is an operand of the product with V as the sum of two numbers of the inputs' type, hi and p - hi: off by 2^-16 (bf16)
// or 2^-22 (fp16) of itself, where one number would be off by 2^-8 or 2^-11 - which the difference of the maps and the norm behind it enlarge by |A1| + lambda |A2| over |A1 - lambda A2|: seven times what
// the result's own rounding costs where the maps see nearly the same.  The second product of a pair costs nothing where the cache is the traffic (one token) and 5 / 3 of the matrix work
// elsewhere: 8192 x 8192, d = 128: 588 us instead of 416; d = 64, padded: 78 instead of 61; 8 frames of 256 tokens, d = 32: the kernel 13.9 instead of 11.6, the call 11.9 instead of 11.7.
#pragma once
#include "transformer_types.h"

namespace tha4 {
namespace xf {

struct AttnArgs {
  const void *q, *k, *v;
  void* out;
  const float *lambdas, *norm_w;
  const int32_t *q_lengths, *kv_lengths;
  const uint8_t* mask;
  float* work;
  int64_t qs[3], ks[3], vs[3], os[3], ms[4];
  int64_t lambda_vs, lambda_hs;
  int32_t batch, q_len, k_len, heads, kv_heads, group, causal, norm;
  int32_t row_tiles, splits, chunk, part_rows;
  float c, slack, lambda_init, eps;            // c = scale * log2(e): the softmax is taken in powers of two; slack = SLACK / c
};

// A weight is held as 2^BIAS p in two parts, hi and what its rounding left.  BIAS: p <= 1 (few queries), p <= 2^SLACK (prompts, whose reference point follows the maximum lazily).  fp16 has no
// exponents to spare: its weights are raised to just below its largest number (2^15), so that only those below 2^-40 or 2^-37 of the largest lose their last bits to its subnormals.
template <class T> struct Mat;
template <> struct Mat<f16> {
  static constexpr float SLACK = 3.0f, BIAS_PROMPT = 12.0f, BIAS_FEW = 15.0f;
  typedef f16x8 v8;
  static THA4_DEV f32x16 mma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static THA4_DEV f32x4 mma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mat<bf16> {
  static constexpr float SLACK = 8.0f, BIAS_PROMPT = 0.0f, BIAS_FEW = 0.0f;
  typedef bf16x8 v8;
  static THA4_DEV f32x16 mma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static THA4_DEV f32x4 mma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// lane i of each 16 receives column i of the 4 x 16 block of 16-bit values whose row r the lanes 4r .. 4r+3 address (8 bytes each)
THA4_DEV s16x4 read_transposed(const char* lds) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds));
}
template <class V8>
THA4_DEV V8 join(s16x4 a, s16x4 b) { return __builtin_bit_cast(V8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7)); }

THA4_DEV float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }
// p as the sum of two numbers of the operands' type
template <class T>
THA4_DEV void in_two(float p, T& hi, T& lo) {
  hi = (T)p;
  lo = (T)(p - (float)hi);
}
// f of the values that lanes i and i + 32 hold, in both: v_permlane32_swap of v with itself leaves the lower half's values in one result, the upper half's in the other
template <class F>
THA4_DEV float both_halves(float v, F f) {
  const unsigned u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// whether one of the 16-bit numbers in a 16-byte piece is an infinity or a NaN (all ones in the exponent: one more there carries into the sign's place)
template <class T>
THA4_DEV bool not_finite(const u32x4& p) {
  constexpr unsigned M = std::is_same<T, bf16>::value ? 0x7f807f80u : 0x7c007c00u, one = std::is_same<T, bf16>::value ? 0x00800080u : 0x04000400u;
  unsigned r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) r |= (p[i] & M) + one;
  return (r & 0x80008000u) != 0;
}
template <class T>
THA4_DEV bool not_finite(T v) { return (__builtin_bit_cast(unsigned short, v) & (std::is_same<T, bf16>::value ? 0x7f80 : 0x7c00)) == (std::is_same<T, bf16>::value ? 0x7f80 : 0x7c00); }
// zeros in their places, in the pieces `first`, `first + step`, ... of `bytes` bytes of LDS
template <class T>
THA4_DEV void clear_not_finite(char* lds, int bytes, int first, int step) {
  for (int p = first; p < bytes / 16; p += step) {
    u32x4 v = reinterpret_cast<u32x4*>(lds)[p];
    if (!not_finite<T>(v)) continue;
    T* e = reinterpret_cast<T*>(lds) + 8 * p;
    for (int i = 0; i < 8; ++i)
      if (not_finite(e[i])) e[i] = (T)0.0f;
  }
}

struct Lengths { int q, k; };
THA4_DEV Lengths lengths_of(const AttnArgs& a, int b) {
  Lengths n;
  n.q = a.q_lengths ? min(max(a.q_lengths[b], 0), a.q_len) : a.q_len;
  n.k = a.kv_lengths ? min(max(a.kv_lengths[b], 0), a.k_len) : a.k_len;
  return n;
}
// exp(l0 . l1) - exp(l2 . l3) + lambda_init of a head, by one wave
template <int D>
THA4_DEV float lambda_of(const AttnArgs& a, int head) {
  const float* l = a.lambdas + head * a.lambda_hs;
  float s = 0.0f, t = 0.0f;
  for (int i = threadIdx.x & 63; i < D; i += 64) {
    s = fmaf(l[i], l[a.lambda_vs + i], s);
    t = fmaf(l[2 * a.lambda_vs + i], l[3 * a.lambda_vs + i], t);
  }
  return expf(wave_reduce(s, Add())) - expf(wave_reduce(t, Add())) + a.lambda_init;
}

// the norm's factor of a row whose squares sum to ss: zero for a row of zeros also where eps is zero (a query that sees no key answers zero)
template <int D>
THA4_DEV float norm_factor(const AttnArgs& a, float ss) { return !a.norm ? 1.0f : ss == 0.0f ? 0.0f : (1.0f - a.lambda_init) / sqrtf(ss * (1.0f / (2 * D)) + a.eps); }

// ---- prompts: many queries ---------------------------------------------------------------------------------------------------------------
// A workgroup owns 32 RG queries of one head: 2 RG waves, wave w the queries 32 (w % RG) .. + 31 of map w / RG (the maps meet once, at the end: each wave carries one
// map's accumulator, which is what lets 2 x 2d columns fit the registers).  Keys go through LDS in groups, K of both maps and V, through a ring of four groups:
// copies are asynchronous and have two to three groups' time to arrive.
// The 16-byte pieces of a K row are permuted so that the 16 lanes the LDS serves together read 16 different slots, those of a V row so that
// the four rows of a transposing read lie in different quarters of the banks (no conflicts by the counters).
//
// Two waves share a SIMD: one of each map.  A group costs a wave a stretch of matrix products (with V of the group before, then with K of this one) and a stretch of
// vector arithmetic (the softmax); the two waves run them in opposite phases, a barrier between the phases, so that one's arithmetic runs under the other's products.
// Measured, causal: 8192 x 8192, 8 heads, d = 128: 588 - 607 us (in step, without the phases: 637): 700 TFLOP/s of the 12 d operations a pair that the formula has, 1170 of
// the 20 d that run;  4096 x 4096, 16 heads on 4, d = 64: 177 us (fp16 186), 970 TFLOP/s of what runs.
template <int D>
struct Tile {
  static constexpr int J = D == 128 ? 1 : 2, KEYS = 32 * J, SLOTS = 4;  // 32-key tiles of a group: one where the accumulator leaves no registers for two
  static constexpr int KP = D / 8, VP = D / 4;                         // 16-byte pieces of a K row (one map), of a V row
  static constexpr int K_BYTES = 2 * KEYS * KP * 16, V_BYTES = KEYS * VP * 16, BYTES = K_BYTES + V_BYTES;
  static THA4_DEV int k_swizzle(int row) { return (row / (16 / KP)) & (KP - 1); }
  static THA4_DEV int v_swizzle(int row) { return VP == 8 ? ((row >> 1) & 1) * 4 : (row & 3) * 4; }
};

// Request K (of both maps) or V of a group into LDS: per copy a wave moves 64 pieces, 64 / KP rows of K or 64 / VP rows of V; keys behind row `left` repeat it.
// kb, vb: the group's first rows (scalar); offsets inside a group fit 32 bits (the host bounds the strides).
template <class T, int D, int WAVES>
THA4_DEV void request_group_k(const AttnArgs& a, const T* kb, int left, unsigned lds) {
  typedef Tile<D> L;
  const int lane = threadIdx.x & 63, wave = uniform_i32(threadIdx.x >> 6);
  constexpr int KR = WAVES * 64 / L::KP;                               // rows that the waves move together: a multiple of 16, after which the swizzle repeats
  static_assert(KR % 16 == 0 && (KR >= L::KEYS ? KR % L::KEYS == 0 : L::KEYS % KR == 0), "every copy of a wave has the same column permutation and one map");
  const int kw = wave * (KR / WAVES), row = kw % L::KEYS + lane / L::KP;
  const unsigned col = 8 * ((lane % L::KP) ^ L::k_swizzle(row));
#pragma unroll
  for (int u = 0; u < L::K_BYTES / 1024 / WAVES; ++u)
    copy16_async(kb + (u * KR / L::KEYS + kw / L::KEYS) * a.ks[2] + ((unsigned)min(row + (u * KR) % L::KEYS, left) * (unsigned)a.ks[1] + col), lds + (u * WAVES + wave) * 1024);
}
template <class T, int D, int WAVES>
THA4_DEV void request_group_v(const AttnArgs& a, const T* vb, int left, unsigned lds) {
  typedef Tile<D> L;
  const int lane = threadIdx.x & 63, wave = uniform_i32(threadIdx.x >> 6);
  constexpr int VR = WAVES * 64 / L::VP;
  static_assert(VR % 4 == 0, "every copy of a wave has the same column permutation");
  const int row = wave * (VR / WAVES) + lane / L::VP;
  const unsigned col = 8 * ((lane % L::VP) ^ L::v_swizzle(row));
#pragma unroll
  for (int u = 0; u < L::V_BYTES / 1024 / WAVES; ++u)
    copy16_async(vb + ((unsigned)min(row + u * VR, left) * (unsigned)a.vs[1] + col), lds + L::K_BYTES + (u * WAVES + wave) * 1024);
}

// A group of which some query sees only a part, with an infinity or a NaN in V: 0 * inf must not reach a query that does not see that key.  The value is added
// to the accumulators that do see it, and taken out of the group.  Rare: written for size.
template <class T, int D, int THREADS>
THA4_DEV void quarantine(const AttnArgs& a, char* vt, f32x16 (&acc)[D / 16], int k0, int limit, const uint8_t* mask, int* flag) {
  typedef Tile<D> L;
  const int lane = threadIdx.x & 63;
  bool bad = false;
  for (int p = threadIdx.x; p < L::V_BYTES / 16; p += THREADS) bad |= not_finite<T>(reinterpret_cast<const u32x4*>(vt)[p]);
  if (bad) *flag = 1;
  __syncthreads();
  if (*flag == 0) return;                                              // (set again behind another barrier at the earliest)
  for (int key = 0; key < L::KEYS; ++key) {
    const bool seen = k0 + key < limit && (!mask || mask[(int64_t)(k0 + key) * a.ms[3]]);
    const T* row = reinterpret_cast<const T*>(vt + key * L::VP * 16);
    int h = lane >> 5;
    asm volatile("" : "+v"(h));                                        // (addresses computed here, not kept from the loop's head: they would cost the main loop registers)
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int dv = 32 * t + 8 * (r / 4) + 4 * h + r % 4;
        const T val = row[8 * ((dv / 8) ^ L::v_swizzle(key)) + dv % 8];
        if (seen && not_finite(val)) acc[t][r] += (float)val;
      }
      THA4_SCHED_FENCE();                                              // (a few values at a time: nothing here may cost the main loop registers)
    }
  }
  __syncthreads();
  clear_not_finite<T>(vt, L::V_BYTES, threadIdx.x, THREADS);
  if (threadIdx.x == 0) *flag = 0;
  __syncthreads();
}

template <class T, int D, int RG>
__global__ void __launch_bounds__(128 * RG, 2) diff_prompt_kernel(AttnArgs a) {
  warm_kernarg<(int)sizeof(AttnArgs)>();
  typedef Tile<D> L;
  typedef typename Mat<T>::v8 v8;
  constexpr int VT = D / 16;                                           // tiles of 32 value columns
  constexpr int J = L::J, KS = D / 16, AHEAD = D == 64 ? 8 : 4;        // products of 32 keys with K; operands on their way from LDS
  constexpr int JOIN = RG * VT * 16 * 64 * 4;                          // bytes in which the second maps' results meet the first's
  constexpr int BATCH = L::BYTES / 1024 / (2 * RG);                    // copies of a wave and group
  constexpr int kQueries = 32 * RG;
  __shared__ __attribute__((aligned(16))) char lds[L::SLOTS * L::BYTES > JOIN ? L::SLOTS * L::BYTES : JOIN];
  __shared__ int flag;
  const int lane = threadIdx.x & 63, wave = uniform_i32(threadIdx.x >> 6), map = wave / RG, h = lane >> 5;
  const int bh = blockIdx.x % (a.batch * a.heads), b = bh / a.heads, head = bh % a.heads;
  const int q0 = ((int)(gridDim.x / (a.batch * a.heads)) - 1 - (int)(blockIdx.x / (a.batch * a.heads))) * kQueries;     // the longest rows of a causal map first
  const Lengths n = lengths_of(a, b);
  if (q0 >= n.q) return;
  if (threadIdx.x == 0) flag = 0;
  const int kv = head / a.group, off = n.k - n.q;
  const int qw = q0 + 32 * (wave % RG), row = min(qw + (lane & 31), n.q - 1);
  const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + row * a.qs[1] + (2 * head + map) * a.qs[2];
  const T* k = static_cast<const T*>(a.k) + b * a.ks[0] + 2 * kv * a.ks[2];
  const T* v = static_cast<const T*>(a.v) + b * a.vs[0] + kv * a.vs[2];
  const uint8_t* mask = a.mask ? a.mask + b * a.ms[0] + head * a.ms[1] + row * a.ms[2] : nullptr;
  v8 qf[D / 16];
#pragma unroll
  for (int s = 0; s < D / 16; ++s) qf[s] = *reinterpret_cast<const v8*>(q + 16 * s + 8 * h);
  const int limit = a.causal ? min(n.k, row + off + 1) : n.k;          // this query sees keys below it
  const int wg_end = a.causal ? min(n.k, min(q0 + kQueries, n.q) + off) : n.k;
  const int wg_full = a.mask ? 0 : a.causal ? min(n.k, q0 + off + 1) : n.k;      // every query of the workgroup sees the keys below it
  f32x16 acc[VT];
#pragma unroll
  for (int t = 0; t < VT; ++t) acc[t] = f32x16{0};
  float m = -INFINITY, l = 0.0f;

  const unsigned lds_at = lds_address(lds);
  const int groups = (max(wg_end, 0) + L::KEYS - 1) / L::KEYS, whole = max(wg_full, 0) / L::KEYS;      // the first `whole` groups are seen wholly by everybody
  auto request_k = [&](int g) {
    if (g < groups) request_group_k<T, D, 2 * RG>(a, k + (int64_t)g * L::KEYS * a.ks[1], n.k - 1 - g * L::KEYS, lds_at + g % L::SLOTS * L::BYTES);
  };
  auto request_v = [&](int g) {
    if (g < groups) request_group_v<T, D, 2 * RG>(a, v + (int64_t)g * L::KEYS * a.vs[1], n.k - 1 - g * L::KEYS, lds_at + g % L::SLOTS * L::BYTES);
  };
  auto v_operand = [&](const char* vt, int ln, int u, int t) {         // k slot (h, e) of step u holds key 16 u + 8 (e / 4) + 4 h + e % 4: the accumulator layout of S^T
    const int r0 = 16 * u + 4 * (ln >> 5) + ((ln & 15) >> 2), piece = 4 * t + 2 * ((ln >> 4) & 1) + ((ln & 3) >> 1), in = 8 * (ln & 1);
    const s16x4 lo = read_transposed(vt + (r0 * L::VP + (piece ^ L::v_swizzle(r0))) * 16 + in);
    const s16x4 hi = read_transposed(vt + ((r0 + 8) * L::VP + (piece ^ L::v_swizzle(r0 + 8))) * 16 + in);
    return join<v8>(lo, hi);
  };
  auto k_operand = [&](const char* kt, int ln, int i, int u) {
    const int r = 32 * i + (ln & 31);
    return *reinterpret_cast<const v8*>(kt + (r * L::KP + ((2 * u + (ln >> 5)) ^ L::k_swizzle(r))) * 16);
  };
  f32x16 s[J];
  v8 pf[2 * J], pr[2 * J];                                             // weights, and what their rounding left
  // The scores of a group.  The next AHEAD operands are always on their way, each requested right behind the product that frees its registers: LDS answers in the time of
  // several products (8192 x 8192, d = 128: 607 us with 4 ahead, 609 with 6, which need every register)
  auto scores = [&](int g, int ln) {
    const char* kt = lds + g % L::SLOTS * L::BYTES + map * (L::K_BYTES / 2);
    v8 kf[AHEAD];
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) kf[p] = k_operand(kt, ln, p / KS, p % KS);
#pragma unroll
    for (int i = 0; i < J; ++i) s[i] = f32x16{0};
#pragma unroll
    for (int p = 0; p < J * KS; ++p) {
      s[p / KS] = Mat<T>::mma32(kf[p % AHEAD], qf[p % KS], s[p / KS]);
      if (p + AHEAD < J * KS) kf[p % AHEAD] = k_operand(kt, ln, (p + AHEAD) / KS, (p + AHEAD) % KS);
      if (p % 2) THA4_SCHED_FENCE();
    }
  };
  auto add_values = [&](int g, int ln) {
    const char* vt = lds + g % L::SLOTS * L::BYTES + L::K_BYTES;
    v8 vf[AHEAD];
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) vf[p] = v_operand(vt, ln, p / VT, p % VT);
#pragma unroll
    for (int p = 0; p < 2 * J * VT; p += 2) {                          // (two tiles in turn: a product never waits for the one before)
#pragma unroll
      for (int e = 0; e < 2; ++e) acc[(p + e) % VT] = Mat<T>::mma32(vf[(p + e) % AHEAD], pf[p / VT], acc[(p + e) % VT]);
#pragma unroll
      for (int e = 0; e < 2; ++e) acc[(p + e) % VT] = Mat<T>::mma32(vf[(p + e) % AHEAD], pr[p / VT], acc[(p + e) % VT]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int next = p + e + AHEAD;
        if (next < 2 * J * VT) vf[(p + e) % AHEAD] = v_operand(vt, ln, next / VT, next % VT);
      }
      THA4_SCHED_FENCE();
    }
  };
  auto softmax = [&]() {
    float top = s[0][0];
#pragma unroll
    for (int i = 0; i < J; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[i][r]);
    top = both_halves(top, Max());
    // The reference point of the exponents follows the maximum only when that has outgrown it by 2^SLACK (in the first groups of nearly every row, seldom later): the accumulator is left
    // alone in most groups (8192 x 8192, d = 128, one product a weight: 462 -> 443 us)
    const float now = top - m > a.slack ? top : m;                      // (the difference: exact where it is small, whatever the size of the scores)
    if (__any(now != m)) {
      const float w = now == -INFINITY ? 1.0f : exp2_((m - now) * a.c);
      l *= w;
#pragma unroll
      for (int t = 0; t < VT; ++t) acc[t] *= w;
      m = now;
    }
    const float from = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < J; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = exp2_(fmaf(s[i][r] - from, a.c, Mat<T>::BIAS_PROMPT));
        T hi, lo;
        in_two(p, hi, lo);
        l += p;
        pf[2 * i + r / 8][r % 8] = hi;
        pr[2 * i + r / 8][r % 8] = lo;
      }
  };

  // a group that some query sees only a part of
  auto part_group = [&](int g) {
    quarantine<T, D, 128 * RG>(a, lds + g % L::SLOTS * L::BYTES + L::K_BYTES, acc, g * L::KEYS, limit, mask, &flag);
    int ln = lane;
    asm volatile("" : "+v"(ln));                                       // (addresses computed here: kept from the kernel's head they would cost the loop above registers)
    scores(g, ln);
#pragma unroll
    for (int i = 0; i < J; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = g * L::KEYS + 32 * i + 8 * (r / 4) + 4 * h + r % 4;
        bool seen = key < limit;
        if (mask) {
          seen = seen && mask[(int64_t)min(key, a.k_len - 1) * a.ms[3]];
          if (r % 4 == 3) THA4_SCHED_FENCE();
        }
        s[i][r] = seen ? s[i][r] : -INFINITY;
      }
    softmax();
    THA4_SCHED_FENCE();
    add_values(g, ln);
  };

  if constexpr (RG == 2) {
    // Four waves, each alone on its SIMD (or beside another workgroup's): no partner to take turns with (8 frames of 256 tokens, d = 32, in a graph: 11.4 us in step, 13.7 us in phases)
#pragma unroll
    for (int g = 0; g < 3; ++g) { request_k(g); request_v(g); }
    auto enter = [&](int g) {
      THA4_BARRIER_KEEP(min(2, groups - 1 - g) * BATCH);               // this group is there, and everybody has left the one before
      request_k(g + 3);
      request_v(g + 3);
    };
    for (int g = 0; g < whole; ++g) {
      enter(g);
      scores(g, lane);
      softmax();
      THA4_SCHED_FENCE();
      add_values(g, lane);
    }
    for (int g = whole; g < groups; ++g) {
      enter(g);
      part_group(g);
    }
  } else {
    // Whole groups in phases.  In phase 2 i the first map's waves multiply (values of group i - 1, scores of group i) while the second's take the softmax of group i - 1; in phase
    // 2 i + 1 the other way round.  K of a group is read in phases 2 i and 2 i + 1, V in 2 i + 2 and 2 i + 3; so at the head of phase 2 i the slots of K (i - 1) and V (i - 2) are
    // free and take K (i + 3) and V (i + 2), and behind phase 2 i + 1 K (i + 1) and V (i) have to be there: everything but the two newest batches.
    auto batch = [&](int i) { request_k(i + 3); request_v(i + 2); };
    auto even_end = [&]() { THA4_SCHED_FENCE(); THA4_BARRIER_LDS(); THA4_SCHED_FENCE(); };
    auto odd_end = [&](int i) { THA4_SCHED_FENCE(); THA4_BARRIER_KEEP(i + 3 < groups ? 2 * BATCH : 0); THA4_SCHED_FENCE(); };
    request_k(0);
    request_k(1); request_v(0);
    request_k(2); request_v(1);
    if (whole > 0) {                                                   // (both maps pass 2 whole + 3 barriers)
      odd_end(-1);
      if (map == 1) { batch(0); even_end(); }
      for (int i = 0; i <= whole; ++i) {
        if (map == 0) batch(i);
        if (i > 0) add_values(i - 1, lane);
        if (i < whole) scores(i, lane);
        if (map == 0) even_end(); else odd_end(i);
        if (i < whole) {
          if (map == 1) batch(i + 1);
          softmax();
        }
        if (map == 0) odd_end(i); else if (i < whole) even_end();
      }
    } else {
      batch(0);
    }
    for (int g = whole; g < groups; ++g) {                             // the rest in step
      THA4_BARRIER_KEEP(0);                                            // this group is there, and everybody has left the one before
      if (g > whole) request_k(g + 3);
      request_v(g + 3);
      part_group(g);
    }
  }

  l = both_halves(l, Add());
  float* meet = reinterpret_cast<float*>(lds) + (wave % RG) * (VT * 16 * 64) + lane;
  __syncthreads();
  if (map == 1) {
    const float lam = lambda_of<D>(a, head), w = l > 0.0f || l != l ? lam / l : 0.0f;      // (no key seen: nothing)
#pragma unroll
    for (int t = 0; t < VT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) meet[(t * 16 + r) * 64] = acc[t][r] * w;
  }
  __syncthreads();
  if (map == 1) return;
  const float w = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  float ss = 0.0f;
#pragma unroll
  for (int t = 0; t < VT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      acc[t][r] = fmaf(acc[t][r], w, -meet[(t * 16 + r) * 64]);
      ss = fmaf(acc[t][r], acc[t][r], ss);
    }
  ss = both_halves(ss, Add());
  int le = threadIdx.x & 63;
  asm volatile("" : "+v"(le));                                        // (the query's number again: not worth a register throughout the loop)
  const int qi = qw + (le & 31);
  if (qi >= n.q) return;
  const float g = norm_factor<D>(a, ss);
  T* out = static_cast<T*>(a.out) + b * a.os[0] + qi * a.os[1] + head * a.os[2];
  typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int t = 0; t < VT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int dv = 32 * t + 8 * r + 4 * h;
      T4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (T)(acc[t][4 * r + e] * g * (a.norm && a.norm_w ? a.norm_w[dv + e] : 1.0f));
      *reinterpret_cast<T4*>(out + dv) = o;
    }
}

// ---- few queries over a long cache -------------------------------------------------------------------------------------------------------
// The cache is the traffic: 4 d elements a key and kv head, read once for all queries and heads that share it (up to 16 rows, the columns of the 16 x 16 x 32 products).
// A workgroup owns a range of the keys; its four waves take turns of 32 keys, each with running statistics and LDS of its own and without barriers.  The next turn's K is
// requested as soon as this turn's has been read into operands, the next V behind the product with this one: a wave always has one of the two in flight,
// asynchronously and straight into LDS, behind counted waits.  The waves meet in LDS, the ranges in a second launch.
// Measured: 32 caches of up to 16384 keys, 16 heads on 4, d = 64 (544 MB): 116 us + 6.5 us for the join, 4.7 TB/s;  131072 keys, 8 heads on 2, d = 128 (268 MB): 51 + 8 us, 5.3 TB/s.
constexpr int kTurn = 32, kRows = 16, kMaxSplits = 512;

template <int D>
struct Few {
  static constexpr int KP = D / 8, VP = D / 4, VT = D / 8;             // 16-byte pieces of a K row (one map), of a V row; tiles of 16 value columns
  static constexpr int K_COPIES = KP, V_COPIES = VP / 2;               // KiB of a turn's K (both maps), V
  static constexpr int WAVE_BYTES = (K_COPIES + V_COPIES) * 1024;
  static constexpr int SET = 2 * VT * 4 * 64;                          // floats of one wave's two accumulators
  static constexpr int PART = 4 * D + 4;                               // floats that a range leaves for each row: O1, O2, m1, l1, m2, l2
  // slots of the 16 lanes that the LDS serves together (rows 0 - 3 and 12 - 15 of one piece, 4 - 11 of the next one) all differ
  static THA4_DEV int k_swizzle(int row) { return KP == 4 ? (4 - (row >> 2)) & 3 : (row / (16 / KP)) & (KP - 1); }
  static THA4_DEV int v_swizzle(int row) { return VP == 8 ? ((row >> 1) & 3) * 2 : (row & 7) * 2; }
};

// A query's value columns: o = O1 w1 - O2 w2, normalised and stored, 4 columns a lane and step.  `ss` sums over the lanes that share the query.
template <class T, int D>
THA4_DEV void store_columns(const AttnArgs& a, T* out, int dv, const f32x4& o, float g) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  T4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = (T)(o[e] * g * (a.norm && a.norm_w ? a.norm_w[dv + e] : 1.0f));
  *reinterpret_cast<T4*>(out + dv) = r;
}
THA4_DEV float weight_of(float top, float l) { return l > 0.0f || l != l ? top / l : 0.0f; }      // (no key seen: nothing)

// out of O1, l1, O2, l2 (accumulator layout: row lane % 16, value columns 16 t + 4 (lane / 16) + e)
template <class T, int D>
THA4_DEV void finish_few(const AttnArgs& a, f32x4 (&o)[2][D / 8], float l1, float l2, int b, int kv, int R, int rows, int q_valid) {
  const int lane = threadIdx.x & 63, head = kv * a.group + R % a.group, qi = R / a.group;
  // (every lane takes part in the sums of lambda: the heads of a wave's rows differ)
  const float* l = a.lambdas + head * a.lambda_hs;
  float s = 0.0f, t2 = 0.0f;
  for (int i = lane >> 4; i < D; i += 4) {
    s = fmaf(l[i], l[a.lambda_vs + i], s);
    t2 = fmaf(l[2 * a.lambda_vs + i], l[3 * a.lambda_vs + i], t2);
  }
  s += __shfl_xor(s, 16, 64); s += __shfl_xor(s, 32, 64);
  t2 += __shfl_xor(t2, 16, 64); t2 += __shfl_xor(t2, 32, 64);
  const float w1 = weight_of(1.0f, l1), w2 = weight_of(expf(s) - expf(t2) + a.lambda_init, l2);
  float ss = 0.0f;
#pragma unroll
  for (int t = 0; t < D / 8; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[0][t][e] = o[0][t][e] * w1 - o[1][t][e] * w2;
      ss = fmaf(o[0][t][e], o[0][t][e], ss);
    }
  ss += __shfl_xor(ss, 16, 64);
  ss += __shfl_xor(ss, 32, 64);
  if (R >= rows || qi >= q_valid) return;
  const float g = norm_factor<D>(a, ss);
  T* out = static_cast<T*>(a.out) + b * a.os[0] + qi * a.os[1] + head * a.os[2];
#pragma unroll
  for (int t = 0; t < D / 8; ++t) store_columns<T, D>(a, out, 16 * t + 4 * (lane >> 4), o[0][t], g);
}

// One wave's K or V of a turn: `left` is the last valid row (rows behind it repeat it).  Offsets inside a turn fit 32 bits (the host bounds the strides).
template <class T, int D>
THA4_DEV void request_k(const AttnArgs& a, const T* k, int left, unsigned lds) {
  typedef Few<D> L;
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int u = 0; u < L::K_COPIES; ++u) {
    const int p = u * 64 + lane, map = p / (kTurn * L::KP), row = (p / L::KP) % kTurn, pos = p % L::KP;
    copy16_async(k + map * a.ks[2] + ((unsigned)min(row, left) * (unsigned)a.ks[1] + 8 * (pos ^ L::k_swizzle(row % 16))), lds + u * 1024);
  }
}
template <class T, int D>
THA4_DEV void request_v(const AttnArgs& a, const T* v, int left, unsigned lds) {
  typedef Few<D> L;
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int u = 0; u < L::V_COPIES; ++u) {
    const int p = u * 64 + lane, row = p / L::VP, pos = p % L::VP;
    copy16_async(v + ((unsigned)min(row, left) * (unsigned)a.vs[1] + 8 * (pos ^ L::v_swizzle(row))), lds + u * 1024);
  }
}
template <int N>
THA4_DEV void wait_copies() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }       // at most the N newest requests of this wave are on their way
THA4_DEV void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }               // what this wave read from LDS has arrived: it may be overwritten

template <class T, int D>
__global__ void __launch_bounds__(256, D == 128 ? 1 : 2) diff_few_kernel(AttnArgs a) {
  warm_kernarg<(int)sizeof(AttnArgs)>();
  typedef Few<D> L;
  typedef typename Mat<T>::v8 v8;
  constexpr int LDS = 4 * L::WAVE_BYTES > 2 * L::SET * 4 ? 4 * L::WAVE_BYTES : 2 * L::SET * 4;
  __shared__ __attribute__((aligned(16))) char lds[LDS];
  __shared__ float stat[4][4][kRows];
  const int lane = threadIdx.x & 63, wave = uniform_i32(threadIdx.x >> 6), g = lane >> 4;
  int id = blockIdx.x;
  // kv heads next to each other: their rows of a token are neighbours in memory (32 x 16384 keys, 4 kv heads, d = 64: 131 -> 122 us against ranges next to each other)
  const int kv = id % a.kv_heads; id /= a.kv_heads;
  const int split = id % a.splits; id /= a.splits;
  const int rt = id % a.row_tiles, b = id / a.row_tiles, tile = (b * a.kv_heads + kv) * a.row_tiles + rt;
  const Lengths n = lengths_of(a, b);
  const int rows = a.q_len * a.group, R = rt * kRows + (lane & 15), Rc = min(R, rows - 1);
  const int qi = min(Rc / a.group, max(n.q - 1, 0)), head = kv * a.group + Rc % a.group;
  const int begin = split * a.chunk, end = min(n.k, begin + a.chunk);
  if (a.splits > 1 && begin >= n.k) return;                              // (the join knows the length too)
  const int limit = a.causal ? min(n.k, qi + (n.k - n.q) + 1) : n.k;
  const int q_first = (rt * kRows) / a.group;
  const int full = a.mask ? 0 : a.causal ? min(n.k, q_first + (n.k - n.q) + 1) : n.k;
  const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + qi * a.qs[1] + 2 * head * a.qs[2];
  const T* k = static_cast<const T*>(a.k) + b * a.ks[0] + 2 * kv * a.ks[2];
  const T* v = static_cast<const T*>(a.v) + b * a.vs[0] + kv * a.vs[2];
  const uint8_t* mask = a.mask ? a.mask + b * a.ms[0] + head * a.ms[1] + qi * a.ms[2] : nullptr;
  char* kt = lds + wave * L::WAVE_BYTES;
  char* vt = kt + L::K_COPIES * 1024;
  const unsigned kt_at = lds_address(kt), vt_at = lds_address(vt);
  int k0 = begin + wave * kTurn;
  if (k0 < end) {
    request_k<T, D>(a, k + (int64_t)k0 * a.ks[1], n.k - 1 - k0, kt_at);
    request_v<T, D>(a, v + (int64_t)k0 * a.vs[1], n.k - 1 - k0, vt_at);
  }
  v8 qf[2][D / 32];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int u = 0; u < D / 32; ++u) qf[i][u] = *reinterpret_cast<const v8*>(q + i * a.qs[2] + 32 * u + 8 * g);
  f32x4 acc[2][L::VT];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int t = 0; t < L::VT; ++t) acc[i][t] = f32x4{0, 0, 0, 0};
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

  for (; k0 < end; k0 += 4 * kTurn) {
    const int next = k0 + 4 * kTurn;
    wait_copies<L::V_COPIES>();                                          // K is here, V may be on its way
    f32x4 s[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[i][j] = f32x4{0, 0, 0, 0};
        const int r = lane & 15;
#pragma unroll
        for (int u = 0; u < D / 32; ++u) {
          const v8 kf = *reinterpret_cast<const v8*>(kt + ((i * kTurn + 16 * j + r) * L::KP + ((4 * u + g) ^ L::k_swizzle(r))) * 16);
          s[i][j] = Mat<T>::mma16(kf, qf[i][u], s[i][j]);
        }
      }
    wait_reads();
    if (next < end) request_k<T, D>(a, k + (int64_t)next * a.ks[1], n.k - 1 - next, kt_at);
    v8 pf[2], pr[2];                                                     // weights, and what their rounding left
    const bool part = k0 + kTurn > full;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (part) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = k0 + 16 * j + 4 * g + e;
            bool seen = key < limit;
            if (mask) seen = seen && mask[(int64_t)min(key, a.k_len - 1) * a.ms[3]];
            s[i][j][e] = seen ? s[i][j][e] : -INFINITY;
          }
      }
      float top = s[i][0][0];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, s[i][j][e]);
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      if (__any(top > m[i])) {
        const float now = fmaxf(m[i], top), w = now == -INFINITY ? 1.0f : exp2_((m[i] - now) * a.c);
        l[i] *= w;
#pragma unroll
        for (int t = 0; t < L::VT; ++t) acc[i][t] *= w;
        m[i] = now;
      }
      const float from = m[i] == -INFINITY ? 0.0f : m[i];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = exp2_(fmaf(s[i][j][e] - from, a.c, Mat<T>::BIAS_FEW));
          T hi, lo;
          in_two(p, hi, lo);
          l[i] += p;
          pf[i][4 * j + e] = hi;
          pr[i][4 * j + e] = lo;
        }
    }
    if (next < end) wait_copies<L::K_COPIES>();                          // V is here, the next K may be on its way
    else wait_copies<0>();
    if (part) {                                                          // infinities and NaN that a row does not see (see quarantine above)
      bool bad = false;
      for (int p = lane; p < L::V_COPIES * 64; p += 64) bad |= not_finite<T>(reinterpret_cast<const u32x4*>(vt)[p]);
      if (__any(bad)) {
        for (int key = 0; key < kTurn; ++key) {
          const bool seen = k0 + key < limit && (!mask || mask[(int64_t)(k0 + key) * a.ms[3]]);
          int gg = g;
          asm volatile("" : "+v"(gg));                                   // (addresses computed here, not kept from the loop's head)
#pragma unroll
          for (int t = 0; t < L::VT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int dv = 16 * t + 4 * gg + e;
              const T val = reinterpret_cast<const T*>(vt + key * L::VP * 16)[8 * ((dv / 8) ^ L::v_swizzle(key)) + dv % 8];
              if (seen && not_finite(val)) { acc[0][t][e] += (float)val; acc[1][t][e] += (float)val; }
            }
        }
        wait_reads();
        clear_not_finite<T>(vt, L::V_COPIES * 1024, lane, 64);
        wait_reads();
      }
    }
    // k slot (g, e) of the product holds key 16 (e / 4) + 4 g + e % 4: the accumulator layout of the two tiles of S^T
#pragma unroll
    for (int t = 0; t < L::VT; ++t) {
      const int r0 = 4 * g + ((lane & 15) >> 2), piece = 2 * t + ((lane & 3) >> 1), in = 8 * (lane & 1);
      const s16x4 lo = read_transposed(vt + (r0 * L::VP + (piece ^ L::v_swizzle(r0))) * 16 + in);
      const s16x4 hi = read_transposed(vt + ((r0 + 16) * L::VP + (piece ^ L::v_swizzle(r0 + 16))) * 16 + in);
      const v8 vf = join<v8>(lo, hi);
      acc[0][t] = Mat<T>::mma16(vf, pf[0], acc[0][t]);
      acc[1][t] = Mat<T>::mma16(vf, pf[1], acc[1][t]);
      acc[0][t] = Mat<T>::mma16(vf, pr[0], acc[0][t]);
      acc[1][t] = Mat<T>::mma16(vf, pr[1], acc[1][t]);
    }
    wait_reads();
    if (next < end) request_v<T, D>(a, v + (int64_t)next * a.vs[1], n.k - 1 - next, vt_at);
  }

  // the four waves meet: common maxima, then two rounds of sums
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor(l[i], 16, 64);
    l[i] += __shfl_xor(l[i], 32, 64);
    if (lane < kRows) { stat[wave][2 * i][lane] = m[i]; stat[wave][2 * i + 1][lane] = l[i]; }
  }
  __syncthreads();
  float M[2], S[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = lane & 15;
    M[i] = fmaxf(fmaxf(stat[0][2 * i][r], stat[1][2 * i][r]), fmaxf(stat[2][2 * i][r], stat[3][2 * i][r]));
    S[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) S[i] += stat[w][2 * i][r] == -INFINITY ? stat[w][2 * i + 1][r] : stat[w][2 * i + 1][r] * exp2_((stat[w][2 * i][r] - M[i]) * a.c);
    const float w = m[i] == -INFINITY ? 1.0f : exp2_((m[i] - M[i]) * a.c);
#pragma unroll
    for (int t = 0; t < L::VT; ++t) acc[i][t] *= w;
  }
  f32x4* meet = reinterpret_cast<f32x4*>(lds) + (wave & 1) * (L::SET / 4) + lane;
#pragma unroll
  for (int round = 0; round < 2; ++round) {
    const int givers = round == 0 ? 2 : 1;                               // waves 2, 3 give to 0, 1; then 1 gives to 0
    if (wave >= givers && wave < 2 * givers) {
      f32x4* to = reinterpret_cast<f32x4*>(lds) + (wave - givers) * (L::SET / 4) + lane;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < L::VT; ++t) to[(i * L::VT + t) * 64] = acc[i][t];
    }
    __syncthreads();
    if (wave < givers) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < L::VT; ++t) acc[i][t] += meet[(i * L::VT + t) * 64];
    }
    __syncthreads();
  }
  if (wave) return;
  if (a.splits == 1) {
    finish_few<T, D>(a, acc, S[0], S[1], b, kv, R, rows, n.q);
    return;
  }
  if (R >= rows) return;
  float* part = a.work + (((int64_t)tile * a.part_rows + (lane & 15)) * a.splits + split) * L::PART;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int t = 0; t < L::VT; ++t) *reinterpret_cast<f32x4*>(part + i * 2 * D + 16 * t + 4 * g) = acc[i][t];
  if (g == 0) *reinterpret_cast<f32x4*>(part + 4 * D) = f32x4{M[0], S[0], M[1], S[1]};
}

// Joins the ranges of the keys: a workgroup for each query and head, the same rescaled sums over the ranges that hold keys.  512 threads: 16-byte pieces of O1 and O2
// side by side, 512 / D ranges at a time (one workgroup reads the parts of one row only: with few rows the parts are what takes the time).
template <class T, int D>
__global__ void __launch_bounds__(512) diff_join_kernel(AttnArgs a) {
  warm_kernarg<(int)sizeof(AttnArgs)>();
  typedef Few<D> L;
  constexpr int SIDE = 512 / D;
  __shared__ float stat[4][kMaxSplits];                                  // m1, l1, m2, l2 of each range
  __shared__ f32x4 sum[SIDE][D];
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x % a.part_rows, tile = blockIdx.x / a.part_rows;
  int id = tile;
  const int R = (id % a.row_tiles) * kRows + row; id /= a.row_tiles;
  const int kv = id % a.kv_heads, b = id / a.kv_heads;
  if (R >= a.q_len * a.group) return;
  const int head = kv * a.group + R % a.group, qi = R / a.group;
  const Lengths n = lengths_of(a, b);
  if (qi >= n.q) return;
  const int used = (n.k + a.chunk - 1) / a.chunk;
  const float* part = a.work + ((int64_t)tile * a.part_rows + row) * a.splits * L::PART;
  for (int s = threadIdx.x; s < used; s += 512) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(part + (int64_t)s * L::PART + 4 * D);
#pragma unroll
    for (int i = 0; i < 4; ++i) stat[i][s] = v[i];
  }
  const int slot = threadIdx.x % D, side = threadIdx.x / D, map = slot / (D / 2);
  __syncthreads();
  float M[2] = {-INFINITY, -INFINITY}, S[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    for (int s = lane; s < used; s += 64) M[i] = fmaxf(M[i], stat[2 * i][s]);
    M[i] = wave_reduce(M[i], Max());
    for (int s = lane; s < used; s += 64) S[i] += stat[2 * i][s] == -INFINITY ? stat[2 * i + 1][s] : stat[2 * i + 1][s] * exp2_((stat[2 * i][s] - M[i]) * a.c);
    S[i] = wave_reduce(S[i], Add());
  }
  f32x4 acc = {0, 0, 0, 0};
#pragma unroll 4
  for (int s = side; s < used; s += SIDE) {
    const float m = stat[2 * map][s], w = m == -INFINITY ? 1.0f : exp2_((m - (map ? M[1] : M[0])) * a.c);
    acc += w * *reinterpret_cast<const f32x4*>(part + (int64_t)s * L::PART + 4 * slot);
  }
  sum[side][slot] = acc;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const float lam = lambda_of<D>(a, head);
  const int at = min(lane, D / 2 - 1);
  f32x4 o[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    o[i] = sum[0][i * (D / 2) + at];
#pragma unroll
    for (int s = 1; s < SIDE; ++s) o[i] += sum[s][i * (D / 2) + at];
  }
  o[0] = o[0] * weight_of(1.0f, S[0]) - o[1] * weight_of(lam, S[1]);
  float ss = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; ++e) ss = fmaf(o[0][e], o[0][e], ss);
  ss = wave_reduce(lane < D / 2 ? ss : 0.0f, Add());
  if (lane < D / 2) store_columns<T, D>(a, static_cast<T*>(a.out) + b * a.os[0] + qi * a.os[1] + head * a.os[2], 4 * lane, o[0], norm_factor<D>(a, ss));
}

}  // namespace xf
}  // namespace tha4
