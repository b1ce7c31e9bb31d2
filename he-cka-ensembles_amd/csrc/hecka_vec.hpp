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

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

}  // namespace hecka
