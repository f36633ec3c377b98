// e4m3 blocks: what the kernels that write or read 8-bit operands share.
//
// A matrix is held as e4m3 values in rows of `pitch` bytes (a multiple of 128,
// zero behind the last column) with one scale for each 1x128 or 128x128 block.
// The scale is a power of two (one e8m0 byte) or a 32-bit float; with
// a = max|v| of the block, at least 2^-110:
//   e8m0: scale = the smallest 2^e with a <= 448 * 2^e,  code = v * 2^-e
//   f32:  scale = a / 448,                               code = v * (448 / a)
// A block that holds an infinity or a NaN gets a NaN scale and NaN codes.
#pragma once

#include "al_common.h"
#include <hip/hip_fp16.h>

#include <type_traits>

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4v __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4v __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8v __attribute__((ext_vector_type(8)));

constexpr int kQB = 128;  // values along a row that share a scale

enum ScaleKind { kE8M0 = 0, kF32 = 1 };
enum { kTypeBF16 = 0, kTypeF16 = 1, kTypeF32 = 2 };

// Eight values at an address that is aligned to one value only: rows of odd
// length start anywhere. gfx950 takes such 16-byte accesses in hardware.
template <typename T> struct Vec8;
template <> struct Vec8<__bf16> { typedef bf16x8v V; };
template <> struct Vec8<_Float16> { typedef f16x8v V; };
template <> struct Vec8<float> { typedef f32x8 V; };

template <typename T> AL_DEV f32x8 load8(const T* p) {
  typename Vec8<T>::V v;
  __builtin_memcpy(&v, p, sizeof(v));
  return __builtin_convertvector(v, f32x8);
}
template <typename T> AL_DEV void store8(T* p, f32x8 f) {
  typename Vec8<T>::V v = __builtin_convertvector(f, typename Vec8<T>::V);
  __builtin_memcpy(p, &v, sizeof(v));
}
// the first `left` of eight values, zero behind them
template <typename T> AL_DEV f32x8 load8_upto(const T* p, int left) {
  if (left >= 8) return load8(p);
  f32x8 f = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < left) f[i] = (float)p[i];
  return f;
}
template <typename T> AL_DEV void store8_upto(T* p, f32x8 f, int left) {
  if (left >= 8) { store8(p, f); return; }
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < left) p[i] = (T)f[i];
}

// max of |v| as bits: an infinity or NaN stays the largest (fmaxf drops NaN)
AL_DEV unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
AL_DEV unsigned amax8(f32x8 f) {
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, abs_bits(f[i]));
  return m;
}

struct BlockScale {
  float inv;      // codes are value * inv
  unsigned code;  // e8m0 byte, or the bits of the 32-bit scale
};
AL_DEV float e8m0_value(unsigned code) {
  return __uint_as_float(code == 255u ? 0x7fc00000u : code << 23);
}

template <int KIND> AL_DEV BlockScale block_scale(unsigned amax) {
  BlockScale s;
  if (amax >= 0x7f800000u) {  // infinity or NaN in the block
    s.inv = __uint_as_float(0x7fc00000u);
    s.code = KIND == kE8M0 ? 255u : 0x7fc00000u;
    return s;
  }
  amax = max(amax, 17u << 23);  // 2^-110: scale and its inverse stay normal
  if (KIND == kE8M0) {
    // 448 = 1.75 * 2^8: a mantissa above 1.75 carries into the exponent
    s.code = ((amax + 0x1fffffu) >> 23) - 8;
    s.inv = __uint_as_float((254 - s.code) << 23);
  } else {
    const float a = __uint_as_float(amax);
    s.inv = 448.f / a;
    s.code = __float_as_uint(a / 448.f);
  }
  return s;
}

template <int KIND> AL_DEV void store_scale(void* p, long at, unsigned code) {
  if (KIND == kE8M0) ((unsigned char*)p)[at] = (unsigned char)code;
  else ((unsigned*)p)[at] = code;
}

// Eight values as they are in memory, and the work on them that needs no unpacking:
// 16-bit magnitudes are compared as whole numbers, two at a time, and the conversion
// to e4m3 takes them, and a power of two to divide by, directly.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));
template <typename T> struct Raw8 { typedef i32x4 V; };
template <> struct Raw8<float> { typedef f32x8 V; };

template <typename T> AL_DEV typename Raw8<T>::V raw8(const T* p) {
  typename Raw8<T>::V v;
  __builtin_memcpy(&v, p, sizeof(T) * 8);
  return v;
}
template <typename T> AL_DEV typename Raw8<T>::V raw8_upto(const T* p, int left) {
  if (left >= 8) return raw8(p);
  typename Vec8<T>::V v = (typename Vec8<T>::V)(T)0;
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < left) v[i] = p[i];
  return __builtin_bit_cast(typename Raw8<T>::V, v);
}
template <typename T> AL_DEV f32x8 unpack(typename Raw8<T>::V v) {
  return __builtin_convertvector(__builtin_bit_cast(typename Vec8<T>::V, v), f32x8);
}

// the largest magnitude so far
template <typename T> struct Top {
  u16x2 m = {0, 0};
  AL_DEV void add(int two) { m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, two & 0x7fff7fff)); }
  AL_DEV void add(i32x4 v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) add(v[i]);
  }
  // as the bits of a 32-bit float
  AL_DEV static unsigned bits(unsigned short v) {
    return abs_bits((float)__builtin_bit_cast(T, v));
  }
  AL_DEV unsigned bits() const { return bits(m[0] > m[1] ? m[0] : m[1]); }
};
template <> struct Top<float> {
  unsigned m = 0;
  AL_DEV void add(f32x8 v) { m = max(m, amax8(v)); }
  AL_DEV unsigned bits() const { return m; }
};

// two values' codes into the lower or upper half of `to`; e8m0: divided by a power of two
template <bool HIGH> AL_DEV int two_codes(int to, float x, float y, float scale) {
  return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(__builtin_bit_cast(s16x2, to), x, y, scale, HIGH));
}
template <typename T, bool HIGH> AL_DEV int two_codes(int to, int two, float scale) {
  const s16x2 t = __builtin_bit_cast(s16x2, to);
  if constexpr (std::is_same<T, __bf16>::value)
    return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(t, __builtin_bit_cast(bf16x2v, two), scale, HIGH));
  else
    return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(t, __builtin_bit_cast(f16x2v, two), scale, HIGH));
}

// eight values to eight e4m3 codes, rounded to nearest even
template <int KIND> AL_DEV i32x2 to_fp8(f32x8 f, BlockScale s) {
  i32x2 r;
  if (KIND == kE8M0) {
    const float by = e8m0_value(s.code);
    r[0] = two_codes<true>(two_codes<false>(0, f[0], f[1], by), f[2], f[3], by);
    r[1] = two_codes<true>(two_codes<false>(0, f[4], f[5], by), f[6], f[7], by);
    return r;
  }
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] * s.inv, f[1] * s.inv, 0, false);
  r[0] = __builtin_amdgcn_cvt_pk_fp8_f32(f[2] * s.inv, f[3] * s.inv, lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4] * s.inv, f[5] * s.inv, 0, false);
  r[1] = __builtin_amdgcn_cvt_pk_fp8_f32(f[6] * s.inv, f[7] * s.inv, hi, true);
  return r;
}
template <typename T, int KIND> AL_DEV i32x2 raw_to_fp8(typename Raw8<T>::V v, BlockScale s) {
  if constexpr (std::is_same<T, float>::value) {
    return to_fp8<KIND>(v, s);
  } else if constexpr (KIND == kF32) {
    return to_fp8<KIND>(unpack<T>(v), s);
  } else {
    const float by = e8m0_value(s.code);
    i32x2 r;
    r[0] = two_codes<T, true>(two_codes<T, false>(0, v[0], by), v[1], by);
    r[1] = two_codes<T, true>(two_codes<T, false>(0, v[2], by), v[3], by);
    return r;
  }
}

// the first `left` of eight codes, zero behind them (also where the codes are NaN)
AL_DEV i32x2 keep_upto(i32x2 codes, int left) {
  if (left >= 8) return codes;
  if (left <= 0) return i32x2{0, 0};
  return __builtin_bit_cast(i32x2, __builtin_bit_cast(unsigned long, codes) &
                                       ((1ul << (left * 8)) - 1));
}

// A lane's partner for the reductions over 16 lanes: within pairs, pairs of pairs,
// halves, and the whole. Once the groups below agree, a mirror reaches the other one.
template <int STEP> AL_DEV int partner(int v) {
  constexpr int kCtrl[4] = {0xb1, 0x4e, 0x141, 0x140};  // swap 1, swap 2, mirror 8, mirror 16
  return __builtin_amdgcn_update_dpp(0, v, kCtrl[STEP], 0xf, 0xf, true);
}
template <int STEP> AL_DEV float partner(float v) { return __int_as_float(partner<STEP>(__float_as_int(v))); }
template <int STEP> AL_DEV double partner(double v) {
  return __hiloint2double(partner<STEP>(__double2hiint(v)), partner<STEP>(__double2loint(v)));
}
// over the 16 lanes that hold one block's 128 values, eight each
AL_DEV unsigned max_over_16(unsigned m) {
  m = max(m, (unsigned)partner<0>((int)m));
  m = max(m, (unsigned)partner<1>((int)m));
  m = max(m, (unsigned)partner<2>((int)m));
  return max(m, (unsigned)partner<3>((int)m));
}
// the sum over a wave, in every lane
template <typename F> AL_DEV F wave_total(F v) {
  v += partner<0>(v);
  v += partner<1>(v);
  v += partner<2>(v);
  v += partner<3>(v);
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}
