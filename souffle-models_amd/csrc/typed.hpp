// Activations of three element types (fp16, bf16, fp32) for kernels that compute in fp32: vectors of 8 elements that are
// loaded and stored in 16-byte pieces wherever a row starts, their conversion, and wave reductions without LDS traffic.
#pragma once
#include "common.hpp"
#include "../../include/souffle_hip.h"

namespace souffle {

typedef __bf16 bf16_t;

template <class T>
struct Vec8 {
  typedef T type __attribute__((ext_vector_type(8)));
  // Rows may start at any multiple of the element's size (an odd width, a slice): the unaligned form is one
  // global_load_dwordx4 / global_store_dwordx4 all the same, the memory unit splits it where it crosses a line.
  typedef T unaligned __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

// How the length n of a row goes into vectors: a multiple of 8, with a rest, or shorter than one vector.
enum RowForm { kWhole = 0, kRagged = 1, kShort = 2 };
// Elements c .. c+7 of a row of n, in two steps that both run without a branch around the load: load_row takes the eight
// elements from min(c, n - 8) on (all lanes load, also those behind the row's end), and settle_row, where the data is used, moves the
// row's last elements into place and zeroes what lies behind it.  (A lane that skips a load by a branch makes
// the whole wave wait for every load it has in flight, at each such branch.)
template <RowForm FORM, class T>
__device__ __forceinline__ typename Vec8<T>::type load_row(const T *row, int c, int n) {
  if constexpr (FORM != kShort) {
    return *(const __attribute__((address_space(1))) typename Vec8<T>::unaligned *)(row + min(c, n - 8));
  } else {
    typename Vec8<T>::type v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = *(const __attribute__((address_space(1))) T *)(row + min(c + e, n - 1));
    return v;
  }
}
template <RowForm FORM, class T>
__device__ __forceinline__ typename Vec8<T>::type settle_row(typename Vec8<T>::type v, int c, int n) {
  if constexpr (FORM != kShort) {
    constexpr int kWords = sizeof(T) * 2, kHalf = sizeof(T) == 2;      // 32-bit words of a vector; two elements a word
    typedef unsigned W __attribute__((ext_vector_type(kWords)));
    W w = __builtin_bit_cast(W, v);
    if constexpr (FORM == kRagged) {
      const int by = c - min(c, n - 8);      // elements to move down
#pragma unroll
      for (int step = 4; step >= 1; step >>= 1) {
        const bool on = by & step;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          unsigned moved;
          if (kHalf && step == 1) {
            moved = i + 1 < kWords ? __builtin_amdgcn_alignbit(w[i + 1 < kWords ? i + 1 : i], w[i], 16) : w[i] >> 16;
          } else {
            const int d = kHalf ? step / 2 : step;
            moved = i + d < kWords ? w[i + d < kWords ? i + d : i] : 0u;
          }
          w[i] = on ? moved : w[i];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = c < n ? w[i] : 0u;
    return __builtin_bit_cast(typename Vec8<T>::type, w);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < n ? v[e] : (T)0.f;
    return v;
  }
}
// The same at once, for a lane that may be the only one with something to load.
template <class T>
__device__ __forceinline__ typename Vec8<T>::type load8(const T *row, int c, int n) {
  typedef typename Vec8<T>::type V;
  if (c + 8 <= n) return *(const __attribute__((address_space(1))) typename Vec8<T>::unaligned *)(row + c);
  V v = {};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (c + e < n) v[e] = *(const __attribute__((address_space(1))) T *)(row + c + e);
  return v;
}
template <RowForm FORM, class T>
__device__ __forceinline__ void store_row(T *row, int c, int n, typename Vec8<T>::type v) {
  if (c + 8 <= n) *(__attribute__((address_space(1))) typename Vec8<T>::unaligned *)(row + c) = v;
  if constexpr (FORM != kWhole)
    if (c + 8 > n)
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (c + e < n) *(__attribute__((address_space(1))) T *)(row + c + e) = v[e];
}
// The vector as a value that the optimiser cannot see through: what is computed from it in a loop stays there (conversions of
// a loop's constants to fp32, moved out of it, take twice the registers of the constants).
template <class V>
__device__ __forceinline__ V opaque(V v) {
  typedef unsigned W __attribute__((ext_vector_type(sizeof(V) / 4)));
  W w = __builtin_bit_cast(W, v);
#pragma unroll
  for (int i = 0; i < (int)(sizeof(V) / 4); ++i) asm volatile("" : "+v"(w[i]));
  return __builtin_bit_cast(V, w);
}
template <class V>
__device__ __forceinline__ void to_f32(float (&f)[8], V v) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (float)v[e];
}
// One rounding to nearest even per element (the compiler's conversions; fp32 passes through).
template <class T>
__device__ __forceinline__ typename Vec8<T>::type from_f32(const float (&f)[8]) {
  typename Vec8<T>::type v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (T)f[e];
  return v;
}

// Reductions over the 64 lanes by DPP moves inside the vector unit (rows of 16, then across the rows); the result is
// the same in every lane.  A shuffle goes through the LDS unit instead, at some 60 cycles a step, six steps a reduction.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float v, float identity) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, identity), __builtin_bit_cast(int, v), CTRL, ROWS, 15, false));
}
__device__ __forceinline__ float lane63(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ float wave_sum_dpp(float v) {
  v += dpp<0x111, 15>(v, 0.f);      // row_shr:1
  v += dpp<0x112, 15>(v, 0.f);      // row_shr:2
  v += dpp<0x114, 15>(v, 0.f);      // row_shr:4
  v += dpp<0x118, 15>(v, 0.f);      // row_shr:8: lane 15 of each row of 16 holds the row's sum
  v += dpp<0x142, 10>(v, 0.f);      // row_bcast:15 into rows 1 and 3
  v += dpp<0x143, 12>(v, 0.f);      // row_bcast:31 into rows 2 and 3
  return lane63(v);
}
// Two sums in one chain: after the halves of both change places, one half of the wave sums v0 and the other v1.
__device__ __forceinline__ void wave_sum2_dpp(float &v0, float &v1) {
  const auto p = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v0), __builtin_bit_cast(unsigned, v1), false, false);
  float v = __builtin_bit_cast(float, (unsigned)p[0]) + __builtin_bit_cast(float, (unsigned)p[1]);
  v += dpp<0x111, 15>(v, 0.f);
  v += dpp<0x112, 15>(v, 0.f);
  v += dpp<0x114, 15>(v, 0.f);
  v += dpp<0x118, 15>(v, 0.f);
  v += dpp<0x142, 10>(v, 0.f);
  v0 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 31));
  v1 = lane63(v);
}
// The same over each row of 16 lanes by rotations (every step adds two values that both lanes have, so all lanes get the same bits).
__device__ __forceinline__ float row16_sum_dpp(float v) {
  v += dpp<0x128, 15>(v, 0.f);      // row_ror:8
  v += dpp<0x124, 15>(v, 0.f);
  v += dpp<0x122, 15>(v, 0.f);
  return v + dpp<0x121, 15>(v, 0.f);
}
__device__ __forceinline__ unsigned row16_umax_dpp(unsigned v) {
#define SOUFFLE_STEP(CTRL) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 15, 15, false))
  SOUFFLE_STEP(0x128);
  SOUFFLE_STEP(0x124);
  SOUFFLE_STEP(0x122);
  SOUFFLE_STEP(0x121);
#undef SOUFFLE_STEP
  return v;
}
// Largest of non-negative floats or NaNs, as bit patterns: NaN > infinity > finite, so a NaN is never lost.
__device__ __forceinline__ unsigned wave_umax_dpp(unsigned v) {
#define SOUFFLE_STEP(CTRL, ROWS) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 15, false))
  SOUFFLE_STEP(0x111, 15);
  SOUFFLE_STEP(0x112, 15);
  SOUFFLE_STEP(0x114, 15);
  SOUFFLE_STEP(0x118, 15);
  SOUFFLE_STEP(0x142, 10);
  SOUFFLE_STEP(0x143, 12);
#undef SOUFFLE_STEP
  return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}

// ------------------------------------------------------------------ rows of 8-bit integers ----
// A row x is held as q = round_half_even(x / s), s = max(fp32(max|x| / 127), 2^-100): |q| <= 127, and the bound keeps
// 1 / s finite.  A row that holds a NaN or an infinity gets q = 0 and s = NaN, so that everything computed from it is NaN.
struct RowScale {
  float scale, inverse;
  bool finite;
};
__device__ __forceinline__ unsigned abs_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }
__device__ __forceinline__ RowScale row_scale(unsigned amax_bits) {
  RowScale r;
  r.finite = amax_bits < 0x7f800000u;
  const float s = fmaxf(__builtin_bit_cast(float, amax_bits) / 127.0f, 0x1p-100f);
  r.scale = r.finite ? s : __builtin_nanf("");
  r.inverse = r.finite ? 1.0f / s : 0.0f;
  return r;
}
// The rounding is that of the real quotient, not of a rounded one: halves are common (any value that is half its row's
// largest is 63.5 s), and a product in fp32 would fall on either side of them.  Added to 1.5 * 2^23 in a fused multiply-add, x times
// 1/s is rounded to a whole number q that stands in the sum's low bits in two's complement; it is off by one at most, and
// e = x - q s, which the second fused multiply-add gives exactly (x and q s are multiples of a power of two that
// |e| <= s holds fewer than 2^24 of), says where: beyond half a step, or at half a step from an odd q.
__device__ __forceinline__ unsigned quantize_bits(float x, const RowScale &r) {      // the low byte counts
  constexpr float kShift = 12582912.0f;
  const float sum = __builtin_fmaf(x, r.inverse, kShift);
  const unsigned bits = __builtin_bit_cast(unsigned, sum);
  const float e = __builtin_fmaf(kShift - sum, r.scale, x);
  const float half = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, 0.5f * r.scale) - (bits & 1u));      // odd: the next number below, so that half a step itself is beyond it
  return bits + (e > half ? 1u : 0u) - (e < -half ? 1u : 0u);
}
__device__ __forceinline__ int quantize(float x, const RowScale &r) { return r.finite ? (int)(int8_t)quantize_bits(x, r) : 0; }
__device__ __forceinline__ u2 quantize8(const float (&f)[8], const RowScale &r) {
  u2 p;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    unsigned b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = quantize_bits(f[4 * h + e], r);
    const unsigned lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    p[h] = r.finite ? lo | hi : 0u;
  }
  return p;
}

}  // namespace souffle
