// Element types, vector loads and wave reductions shared by the transformer block operators (transformer_*_kernels.h, tha4_transformer.hip).
#pragma once
#include <cstdint>

#include "tha4_platform.h"

namespace tha4 {
namespace xf {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

THA4_DEV float as_f32(unsigned u) { return __builtin_bit_cast(float, u); }

// 8 consecutive elements as fetched (16 bytes, 32 for fp32): kept packed between the load and its use, so that many rows can be in flight
template <class T>
struct Raw8 { u32x4 a; };
template <>
struct Raw8<float> { f32x4 a, b; };

template <class T>
THA4_DEV Raw8<T> fetch8(const T* p) { return Raw8<T>{*reinterpret_cast<const u32x4*>(p)}; }
template <>
THA4_DEV Raw8<float> fetch8<float>(const float* p) { return Raw8<float>{reinterpret_cast<const f32x4*>(p)[0], reinterpret_cast<const f32x4*>(p)[1]}; }

THA4_DEV void unpack8(const Raw8<float>& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[i] = r.a[i]; v[4 + i] = r.b[i]; }
}
THA4_DEV void unpack8(const Raw8<bf16>& r, float (&v)[8]) {      // bf16 is the upper half of an fp32
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = as_f32(r.a[i] << 16); v[2 * i + 1] = as_f32(r.a[i] & 0xffff0000u); }
}
THA4_DEV void unpack8(const Raw8<f16>& r, float (&v)[8]) {
  const f16x8 h = __builtin_bit_cast(f16x8, r.a);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
}

THA4_DEV void put8(float* p, const float (&v)[8]) {
  reinterpret_cast<f32x4*>(p)[0] = f32x4{v[0], v[1], v[2], v[3]};
  reinterpret_cast<f32x4*>(p)[1] = f32x4{v[4], v[5], v[6], v[7]};
}
template <class T>
THA4_DEV void put8(T* p, const float (&v)[8]) {                  // rounded once, to the nearest
  typedef T T8 __attribute__((ext_vector_type(8)));
  T8 o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = (T)v[i];
  *reinterpret_cast<T8*>(p) = o;
}

// 8 elements of a vector whose type is chosen at run time (the branch is uniform over the launch): fp32, or T
template <class T>
THA4_DEV void param8(const void* p, int64_t at, bool is_f32, float (&v)[8]) {
  if (is_f32) unpack8(fetch8(static_cast<const float*>(p) + at), v);
  else unpack8(fetch8(static_cast<const T*>(p) + at), v);
}
template <class T>
THA4_DEV float param1(const void* p, int64_t at, bool is_f32) {
  return is_f32 ? static_cast<const float*>(p)[at] : (float)static_cast<const T*>(p)[at];
}

struct Add { THA4_DEV float operator()(float a, float b) const { return a + b; } };
struct Max { THA4_DEV float operator()(float a, float b) const { return fmaxf(a, b); } };

template <class F>
THA4_DEV float wave_reduce(float v, F f) {                       // a butterfly: every lane ends with the same bits
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = f(v, __shfl_xor(v, m, 64));
  return v;
}

// The reduction of a row that WAVES waves share; `slot` is LDS of WAVES floats that no other reduction of the kernel uses (one barrier each)
template <int WAVES, class F>
THA4_DEV float row_reduce(float v, F f, float* slot, int wave_of_row) {
  v = wave_reduce(v, f);
  if constexpr (WAVES == 1) return v;
  if ((threadIdx.x & 63) == 0) slot[wave_of_row] = v;
  __syncthreads();
  float r = slot[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) r = f(r, slot[w]);
  return r;
}

// 16 bytes a lane from memory to LDS (base + 16 lane), asynchronous and unknown to the compiler's own wait counting: with copies in flight that it knows of it waits for
// all of them in front of every LDS read.  The caller orders it: THA4_BARRIER_KEEP, or an explicit vmcnt wait.
THA4_DEV void copy16_async(const void* from_lane, unsigned lds_base_uniform) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from_lane), "s"(lds_base_uniform) : "memory", "m0");
}
THA4_DEV unsigned lds_address(const void* p) { return (unsigned)(size_t)(const __attribute__((address_space(3))) char*)p; }

}  // namespace xf
}  // namespace tha4
