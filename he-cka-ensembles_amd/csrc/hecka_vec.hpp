// Row elements as fp32 in registers: 16-byte pieces of fp32 / bf16 / fp16 rows, and sums over lanes, waves and workgroups.
#pragma once
#include <hip/hip_runtime.h>

namespace hecka {

struct Bf16 { unsigned short v; };
struct F16 { _Float16 v; };

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(Bf16 x) { return __uint_as_float((unsigned)x.v << 16); }
__device__ __forceinline__ float widen(F16 x) { return (float)x.v; }
// nearest, ties to even
__device__ __forceinline__ void narrow(float f, float& y) { y = f; }
__device__ __forceinline__ void narrow(float f, Bf16& y) { y.v = __builtin_bit_cast(unsigned short, (__bf16)f); }
__device__ __forceinline__ void narrow(float f, F16& y) { y.v = (_Float16)f; }

// Sixteen bytes of a row.  Rows of any length start at any element, so a piece is only aligned to its element: the hardware
// takes such loads and stores whole (global memory, unaligned access is on), at the price of one more line per wave.
template <class T>
struct Piece {
  static constexpr int N = 16 / sizeof(T);
  T e[N];
};

// elements [col, col + N) of a row of D (zeros behind its end); `row` points at the row
template <class T>
__device__ __forceinline__ Piece<T> load_piece(const T* row, int col, int D) {
  Piece<T> p;
  if (col + Piece<T>::N <= D) {
    __builtin_memcpy(&p, row + col, 16);
  } else {
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i) {
      if (col + i < D) p.e[i] = row[col + i];
      else narrow(0.f, p.e[i]);
    }
  }
  return p;
}
template <class T>
__device__ __forceinline__ void store_piece(T* row, int col, int D, const Piece<T>& p) {
  if (col + Piece<T>::N <= D) {
    __builtin_memcpy(row + col, &p, 16);
  } else {
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i)
      if (col + i < D) row[col + i] = p.e[i];
  }
}

// v of another lane of the same sixteen: ctrl 0xB1 / 0x4E exchange neighbours / pairs in a quad, 0x141 / 0x140 mirror eight /
// sixteen lanes.  Applied in this order every lane ends up with the sum (maximum) of its sixteen, in vector instructions alone.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float sum16(float v) {
  v += dpp<0xB1>(v);
  v += dpp<0x4E>(v);
  v += dpp<0x141>(v);
  return v + dpp<0x140>(v);
}
__device__ __forceinline__ unsigned max16(unsigned v) {
  auto with = [&](int o) { v = (unsigned)o > v ? (unsigned)o : v; };
  with(__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));
  with(__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));
  with(__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));
  with(__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true));
  return v;
}
__device__ __forceinline__ float lane_value(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
// sum over the LANES (8, 16, 32, 64) lanes that a row has of this wave
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (LANES == 8) {
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    return v + dpp<0x141>(v);
  }
  v = sum16(v);
  if constexpr (LANES == 16) return v;
  const float a = lane_value(v, 0) + lane_value(v, 16), b = lane_value(v, 32) + lane_value(v, 48);
  if constexpr (LANES == 32) return (threadIdx.x & 32) ? b : a;
  return a + b;
}

}  // namespace hecka
