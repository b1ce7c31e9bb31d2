// 8-bit blocks: 128 consecutive elements of a row share one power of two s = 2^q, the smallest with max |x| <= 448 s over the
// block's finite elements (q >= -126; 0 for a block of zeros), and each is kept as the e4m3 code nearest to x / s, ties to
// even.  The division by a power of two is exact, so a code is off by half a step of its own binade: 2^-4 of the value, or
// 2^-10 s where the value is below 2^-6 s.  A NaN or an infinity is kept as NaN (code 0x7f) and leaves its neighbours' scale
// alone; a finite element stays finite: with the topmost scale, 2^120, codes end at 240 (256 2^120 is no fp32 number).  A scale is kept as the byte q + 127 - the form in which the scaled matrix instructions take it.
#pragma once
#include "hecka_vec.hpp"

namespace hecka {

static constexpr int kBlock = 128;

// max |.| with non-finite elements left out
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;      // false for NaN
}

// scale byte of a block whose largest finite magnitude is `amax`: 448 = 0.875 * 2^9
__device__ __forceinline__ int scale_byte(float amax) {
  int e;
  const float m = frexpf(amax, &e);
  const int q = e - 9 + (m > 0.875f ? 1 : 0);
  return amax > 0.f ? (q < -126 ? 1 : q + 127) : 127;
}
__device__ __forceinline__ float scale_of(int byte) { return __uint_as_float((unsigned)byte << 23); }            // 2^q
__device__ __forceinline__ float inverse_scale(int byte) { return __uint_as_float((unsigned)(254 - byte) << 23); }  // 2^-q

// four elements as codes, `inv` = 2^-q; |x inv| <= 448, so the conversion never meets its overflow
__device__ __forceinline__ unsigned encode4(float a, float b, float c, float d, float inv) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, r, true);
  return (unsigned)r;
}
// What the conversion is given for x: an infinity must not reach it (it may clamp), so NaN takes its place, and magnitudes past
// 240 2^120 - which only the topmost scale meets - are held there.
__device__ __forceinline__ float encodable(float x) {
  const float top = 0x1.ep+127f;      // 240 2^120
  const float a = fabsf(x);
  return a <= top ? x : a <= 3.402823466e38f ? copysignf(top, x) : __uint_as_float(0x7fc00000u);
}

// A lane's E elements of a block (Piece<T>s) as codes, four a dword, and the block's scale byte; across(bits) is the largest of a
// number over the lanes that hold the block.  Magnitudes are compared as integers (two 16-bit ones at a time), which finds NaN and infinities on
// the way; without any, and below 240 2^120, the conversion takes the elements as they are and divides by the scale itself.
template <class T> struct Magnitude { static constexpr unsigned kLast = 0x7f70; };      // of bf16: 240 2^120
template <> struct Magnitude<float> { static constexpr unsigned kLast = 0x7f700000; };
template <> struct Magnitude<F16> { static constexpr unsigned kLast = 0x7bff; };
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
typedef short i16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

template <class T, int E, class Across>
__device__ __forceinline__ int encode(const Piece<T> (&p)[E / Piece<T>::N], unsigned (&codes)[E / 4], const Across& across) {
  constexpr int D = E * (int)sizeof(T) / 4;      // dwords
  const unsigned* raw = reinterpret_cast<const unsigned*>(&p[0]);
  unsigned big = 0;
#pragma unroll
  for (int i = 0; i < D; ++i) {
    if constexpr (sizeof(T) == 4) {
      const unsigned a = raw[i] & 0x7fffffffu;
      big = a > big ? a : big;
    } else {
      const u16x2_t a = __builtin_bit_cast(u16x2_t, raw[i] & 0x7fff7fffu);
      big = __builtin_bit_cast(unsigned, __builtin_elementwise_max(a, __builtin_bit_cast(u16x2_t, big)));
    }
  }
  if constexpr (sizeof(T) == 2) {
    const unsigned hi = big >> 16, lo = big & 0xffffu;
    big = hi > lo ? hi : lo;
  }
  big = across(big);
  if (__any(big > Magnitude<T>::kLast)) {
    float v[E], a = 0.f;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      v[k] = widen(p[k / Piece<T>::N].e[k % Piece<T>::N]);
      a = fmaxf(a, finite_abs(v[k]));
      v[k] = encodable(v[k]);
    }
    const int byte = scale_byte(__uint_as_float(across(__float_as_uint(a))));      // magnitudes order as their bits do
#pragma unroll
    for (int i = 0; i < E / 4; ++i) codes[i] = encode4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], inverse_scale(byte));
    return byte;
  }
  T top;
  if constexpr (sizeof(T) == 4) top = __uint_as_float(big);
  else top = __builtin_bit_cast(T, (unsigned short)big);
  const int byte = scale_byte(widen(top));
  const float s = scale_of(byte);
#pragma unroll
  for (int i = 0; i < E / 4; ++i) {
    i16x2_t c = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (sizeof(T) == 4) {
        const float a = __uint_as_float(raw[4 * i + 2 * h]), b = __uint_as_float(raw[4 * i + 2 * h + 1]);
        c = h ? __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, a, b, s, true) : __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, a, b, s, false);
      } else if constexpr (__is_same(T, Bf16)) {
        const bf16x2_t a = __builtin_bit_cast(bf16x2_t, raw[2 * i + h]);
        c = h ? __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, a, s, true) : __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, a, s, false);
      } else {
        const f16x2_t a = __builtin_bit_cast(f16x2_t, raw[2 * i + h]);
        c = h ? __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, a, s, true) : __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, a, s, false);
      }
    }
    codes[i] = __builtin_bit_cast(unsigned, c);
  }
  return byte;
}

typedef float f32x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void decode4(unsigned c, float s, float* v) {
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  v[0] = lo[0] * s;
  v[1] = lo[1] * s;
  v[2] = hi[0] * s;
  v[3] = hi[1] * s;
}

// blocks along a row of K elements, and the row of scale bytes up to whole dwords
__host__ __device__ __forceinline__ int row_blocks(int K) { return (K + kBlock - 1) / kBlock; }
__host__ __device__ __forceinline__ int scale_stride(int K) { return (row_blocks(K) + 3) & ~3; }

}  // namespace hecka
