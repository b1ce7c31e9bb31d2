// 8-bit blocks (block8.hpp): rows and weights to codes, codes back, and activations that keep their input in codes
// (hecka_block8_*; contract in include/hecka.h).  All HBM bound: one read of the input, one write of each output.
// Sixteen lanes own a block, eight elements each, so a wave covers four blocks with 16-byte loads (two per lane for fp32),
// the maximum is four lane shuffles and the codes leave as 8 bytes per lane, 128 per block, contiguous.
#include "block8.hpp"
#include "hecka_host.hpp"

namespace hecka {

// eight elements [col, col + 8) of a row of K
template <class T>
__device__ __forceinline__ void load8(const T* row, int col, int K, float* v) {
#pragma unroll
  for (int j = 0; j < 8 / Piece<T>::N; ++j) {
    const Piece<T> p = load_piece(row, col + j * Piece<T>::N, K);
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i) v[j * Piece<T>::N + i] = widen(p.e[i]);
  }
}
template <class T>
__device__ __forceinline__ void store8(T* row, int col, int K, const float* v) {
#pragma unroll
  for (int j = 0; j < 8 / Piece<T>::N; ++j) {
    Piece<T> p;
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i) narrow(v[j * Piece<T>::N + i], p.e[i]);
    if (col + j * Piece<T>::N < K) store_piece(row, col + j * Piece<T>::N, K, p);
  }
}
__device__ __forceinline__ float max8(const float* v) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = fmaxf(a, finite_abs(v[i]));
  return a;
}

// codes and scale byte of the block that the sixteen lanes hold
__device__ __forceinline__ void write_block(float* v, unsigned char* codes, unsigned char* scales, long long row, int blk,
                                            int nblk, int lane16) {
  const int byte = scale_byte(max16(max8(v)));
  const float inv = inverse_scale(byte);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = encodable(v[i]);
  uint2 c;
  c.x = encode4(v[0], v[1], v[2], v[3], inv);
  c.y = encode4(v[4], v[5], v[6], v[7], inv);
  *reinterpret_cast<uint2*>(codes + (row * nblk + blk) * kBlock + lane16 * 8) = c;
  if (lane16 == 0) {
    unsigned char* s = scales + row * ((nblk + 3) & ~3);
    s[blk] = (unsigned char)byte;
    if (blk == nblk - 1)
      for (int i = nblk; i < ((nblk + 3) & ~3); ++i) s[i] = 127;
  }
}

enum { kActNone = 0, kActGelu = 1, kActSilu = 2, kActTanh = 3, kActSigmoid = 4, kActCrater = 5 };
static constexpr float kHalfRoot = 0.70710678118654752f, kCrater = 0.70710678118654752f + 0.008274364699f;

template <int ACT>
__device__ __forceinline__ float act_value(float x) {
  if (ACT == kActGelu) return 0.5f * x * erfcf(-kHalfRoot * x);      // erfc: no cancellation where gelu is close to zero
  if (ACT == kActSilu) return x / (1.0f + expf(-x));
  if (ACT == kActTanh) return tanhf(x);
  if (ACT == kActSigmoid) return 1.0f / (1.0f + expf(-x));
  return kCrater * x * (1.0f + tanhf(kHalfRoot * (x + 1.0f)));
}
template <int ACT>
__device__ __forceinline__ float act_slope(float x) {
  if (ACT == kActGelu) return fmaf(x * 0.39894228040143268f, expf(-0.5f * x * x), 0.5f * erfcf(-kHalfRoot * x));
  if (ACT == kActTanh) { const float t = tanhf(x); return 1.0f - t * t; }
  if (ACT == kActSilu || ACT == kActSigmoid) {
    const float p = 1.0f / (1.0f + expf(-x));
    return ACT == kActSilu ? p * (1.0f + x * (1.0f - p)) : p * (1.0f - p);
  }
  const float t = tanhf(kHalfRoot * (x + 1.0f));
  return kCrater * (1.0f + t + kHalfRoot * x * (1.0f - t * t));
}

// rows of K elements, `ld` apart; ACT != 0: y (rows of K, contiguous) = act(x) beside the codes of x
template <class T, int ACT>
__global__ __launch_bounds__(256) void block8_rows_kernel(const T* __restrict__ x, long long R, int K, long long ld,
                                                          unsigned char* __restrict__ codes, unsigned char* __restrict__ scales,
                                                          T* __restrict__ y) {
  const int nblk = row_blocks(K), lane16 = threadIdx.x & 15;
  const long long total = R * nblk;
  for (long long b = (long long)blockIdx.x * 16 + (threadIdx.x >> 4); b < total; b += (long long)gridDim.x * 16) {
    const long long row = total <= 0xffffffffLL ? (long long)((unsigned)b / (unsigned)nblk) : b / nblk;
    const int blk = (int)(b - row * nblk), col = blk * kBlock + lane16 * 8;
    float v[8];
    load8(x + row * ld, col, K, v);
    if (ACT != kActNone) {
      float a[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = act_value<ACT>(v[i]);
      store8(y + row * K, col, K, a);
    }
    write_block(v, codes, scales, row, blk, nblk, lane16);
  }
}

// ACT = 0: out = the values of the codes; else out = dy * act'(values)
template <class T, int ACT>
__global__ __launch_bounds__(256) void block8_values_kernel(const unsigned char* __restrict__ codes,
                                                            const unsigned char* __restrict__ scales, const T* __restrict__ dy,
                                                            long long R, int K, T* __restrict__ out) {
  const int nblk = row_blocks(K), lane16 = threadIdx.x & 15;
  const long long total = R * nblk;
  for (long long b = (long long)blockIdx.x * 16 + (threadIdx.x >> 4); b < total; b += (long long)gridDim.x * 16) {
    const long long row = total <= 0xffffffffLL ? (long long)((unsigned)b / (unsigned)nblk) : b / nblk;
    const int blk = (int)(b - row * nblk), col = blk * kBlock + lane16 * 8;
    const uint2 c = *reinterpret_cast<const uint2*>(codes + b * kBlock + lane16 * 8);
    const float s = scale_of(scales[row * ((nblk + 3) & ~3) + blk]);
    float v[8];
    decode4(c.x, s, v);
    decode4(c.y, s, v + 4);
    if (ACT != kActNone) {
      float d[8];
      load8(dy + row * K, col, K, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = d[i] * act_slope<ACT>(v[i]);
    } else if constexpr (__is_same(T, F16)) {      // fp16's largest, 65504, is kept as 65536: back to what fp16 holds
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = fabsf(v[i]) == 65536.f ? copysignf(65504.f, v[i]) : v[i];
    }
    store8(out + row * K, col, K, v);
  }
}

// Weights [M, O, I] in 128 x 128 blocks: one workgroup per block holds it in registers (64 elements per thread), takes the
// maximum, and writes the codes along the rows and - through LDS - along the columns, so that the same codes serve the
// product with W and the one with its transpose.  LDS rows of 132 bytes: the byte-wise column writes spread over the banks.
template <class T>
__global__ __launch_bounds__(256) void block8_weight_kernel(const T* __restrict__ W, int O, int I, long long mstride, unsigned char* __restrict__ codes,
                                                            unsigned char* __restrict__ scales, unsigned char* __restrict__ codes_t,
                                                            unsigned char* __restrict__ scales_t) {
  __shared__ float red[4];
  __shared__ unsigned tile[kBlock][kBlock / 4 + 1];
  const int nI = row_blocks(I), nO = row_blocks(O), bi = blockIdx.x, bo = blockIdx.y;
  const long long m = blockIdx.z;
  const int lane16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;      // 16 rows at a time, eight columns per lane
  const T* Wm = W + m * mstride;
  float v[8][8], a = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int o = bo * kBlock + j * 16 + r0;
    if (o < O) load8(Wm + (long long)o * I, bi * kBlock + lane16 * 8, I, v[j]);
    else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = 0.f;
    }
    a = fmaxf(a, max8(v[j]));
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor(a, o));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  const int byte = scale_byte(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
  const float inv = inverse_scale(byte);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int o = bo * kBlock + j * 16 + r0;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] = encodable(v[j][i]);
    uint2 c;
    c.x = encode4(v[j][0], v[j][1], v[j][2], v[j][3], inv);
    c.y = encode4(v[j][4], v[j][5], v[j][6], v[j][7], inv);
    if (o < O) *reinterpret_cast<uint2*>(codes + ((m * O + o) * nI + bi) * kBlock + lane16 * 8) = c;
    if (codes_t) {
      tile[j * 16 + r0][lane16 * 2] = c.x;
      tile[j * 16 + r0][lane16 * 2 + 1] = c.y;
    }
  }
  const int sI = scale_stride(I), sO = scale_stride(O);
  if (threadIdx.x == 0) {
    unsigned char* s = scales + (m * nO + bo) * sI;
    s[bi] = (unsigned char)byte;
    if (bi == nI - 1)
      for (int i = nI; i < sI; ++i) s[i] = 127;
    if (codes_t) {
      unsigned char* t = scales_t + (m * nI + bi) * sO;
      t[bo] = (unsigned char)byte;
      if (bo == nO - 1)
        for (int i = nO; i < sO; ++i) t[i] = 127;
    }
  }
  if (!codes_t) return;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int ic = j * 16 + r0, i = bi * kBlock + ic;      // a row of the transpose: eight codes of this lane
    unsigned c[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      unsigned u = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        u |= ((tile[lane16 * 8 + h * 4 + k][ic >> 2] >> (8 * (ic & 3))) & 255u) << (8 * k);
      c[h] = u;
    }
    if (i < I) *reinterpret_cast<uint2*>(codes_t + ((m * I + i) * nO + bo) * kBlock + lane16 * 8) = make_uint2(c[0], c[1]);
  }
}

// workgroups of a streaming launch: 16 blocks each, at most eight per CU
static unsigned stream_grid(long long blocks) {
  const long long want = (blocks + 15) / 16;
  return (unsigned)(want < 2048 ? want : 2048);
}

template <class T>
static int rows_run(const void* x, long long R, int K, long long ld, void* codes, void* scales, int act, void* y, hipStream_t st) {
  const unsigned grid = stream_grid(R * row_blocks(K));
#define HECKA_ROWS(A) \
  case A: block8_rows_kernel<T, A><<<grid, 256, 0, st>>>((const T*)x, R, K, ld, (unsigned char*)codes, (unsigned char*)scales, (T*)y); break;
  switch (act) { HECKA_ROWS(kActNone) HECKA_ROWS(kActGelu) HECKA_ROWS(kActSilu) HECKA_ROWS(kActTanh) HECKA_ROWS(kActSigmoid) HECKA_ROWS(kActCrater) }
#undef HECKA_ROWS
  return check_launch("block8_rows");
}
template <class T>
static int values_run(const void* codes, const void* scales, const void* dy, long long R, int K, int act, void* out, hipStream_t st) {
  const unsigned grid = stream_grid(R * row_blocks(K));
#define HECKA_VALUES(A) \
  case A: block8_values_kernel<T, A><<<grid, 256, 0, st>>>((const unsigned char*)codes, (const unsigned char*)scales, (const T*)dy, R, K, (T*)out); break;
  switch (act) { HECKA_VALUES(kActNone) HECKA_VALUES(kActGelu) HECKA_VALUES(kActSilu) HECKA_VALUES(kActTanh) HECKA_VALUES(kActSigmoid) HECKA_VALUES(kActCrater) }
#undef HECKA_VALUES
  return check_launch("block8_values");
}
template <class T>
static int weight_run(const void* W, int M, int O, int I, long long mstride, void* codes, void* scales, void* codes_t, void* scales_t, hipStream_t st) {
  block8_weight_kernel<T><<<dim3(row_blocks(I), row_blocks(O), M), 256, 0, st>>>(
      (const T*)W, O, I, mstride, (unsigned char*)codes, (unsigned char*)scales, (unsigned char*)codes_t, (unsigned char*)scales_t);
  return check_launch("block8_weight");
}

static bool bad_type(int dtype) { return dtype != HECKA_DT_F32 && dtype != HECKA_DT_BF16 && dtype != HECKA_DT_F16; }
// R * K below 2^46: every offset fits 64 bits with room, R * blocks as well
static bool bad_rows(long long R, int K) { return R <= 0 || K <= 0 || K > (1 << 30) || R > (1LL << 46) / K; }

}  // namespace hecka

using namespace hecka;

extern "C" {

int hecka_block8_quantize(const void* x, int dtype, long long R, int K, long long ld, int act, void* codes, void* scales,
                          void* y, void* stream) {
  if (bad_type(dtype)) return fail(HECKA_EINVAL, "block8_quantize: unknown dtype%s");
  if (bad_rows(R, K) || ld < K) return fail(HECKA_EINVAL, "%sblock8_quantize: bad size (%lld rows of %lld)", "", R, K);
  if (act < kActNone || act > kActCrater) return fail(HECKA_EINVAL, "%sblock8_quantize: unknown activation (%lld)", "", act);
  if (!x || !codes || !scales || (act != kActNone && !y)) return fail(HECKA_EINVAL, "block8_quantize: null pointer%s");
  if (!aligned16(codes)) return fail(HECKA_EINVAL, "block8_quantize: codes need 16-byte alignment%s");
  clear_error();
  hipStream_t st = (hipStream_t)stream;
  return dtype == HECKA_DT_F32 ? rows_run<float>(x, R, K, ld, codes, scales, act, y, st)
         : dtype == HECKA_DT_BF16 ? rows_run<Bf16>(x, R, K, ld, codes, scales, act, y, st)
                                  : rows_run<F16>(x, R, K, ld, codes, scales, act, y, st);
}

int hecka_block8_values(const void* codes, const void* scales, const void* dy, int dtype, long long R, int K, int act,
                        void* out, void* stream) {
  if (bad_type(dtype)) return fail(HECKA_EINVAL, "block8_values: unknown dtype%s");
  if (bad_rows(R, K)) return fail(HECKA_EINVAL, "%sblock8_values: bad size (%lld rows of %lld)", "", R, K);
  if (act < kActNone || act > kActCrater) return fail(HECKA_EINVAL, "%sblock8_values: unknown activation (%lld)", "", act);
  if (!codes || !scales || !out || (act != kActNone && !dy)) return fail(HECKA_EINVAL, "block8_values: null pointer%s");
  if (!aligned16(codes)) return fail(HECKA_EINVAL, "block8_values: codes need 16-byte alignment%s");
  clear_error();
  hipStream_t st = (hipStream_t)stream;
  return dtype == HECKA_DT_F32 ? values_run<float>(codes, scales, dy, R, K, act, out, st)
         : dtype == HECKA_DT_BF16 ? values_run<Bf16>(codes, scales, dy, R, K, act, out, st)
                                  : values_run<F16>(codes, scales, dy, R, K, act, out, st);
}

int hecka_block8_weight(const void* W, int dtype, int M, int O, int I, long long mstride, void* codes, void* scales, void* codes_t,
                        void* scales_t, void* stream) {
  if (bad_type(dtype)) return fail(HECKA_EINVAL, "block8_weight: unknown dtype%s");
  if (M <= 0 || M > 65535 || O <= 0 || I <= 0 || O > (65535 << 7) || I > (1 << 30))
    return fail(HECKA_EINVAL, "%sblock8_weight: bad size (O = %lld, I = %lld)", "", O, I);
  if (M > 1 && mstride < (long long)O * I) return fail(HECKA_EINVAL, "%sblock8_weight: members %lld elements apart", "", mstride);
  if (!W || !codes || !scales || !codes_t != !scales_t) return fail(HECKA_EINVAL, "block8_weight: null pointer%s");
  if (!aligned16(codes) || !aligned16(codes_t)) return fail(HECKA_EINVAL, "block8_weight: codes need 16-byte alignment%s");
  clear_error();
  hipStream_t st = (hipStream_t)stream;
  return dtype == HECKA_DT_F32 ? weight_run<float>(W, M, O, I, mstride, codes, scales, codes_t, scales_t, st)
         : dtype == HECKA_DT_BF16 ? weight_run<Bf16>(W, M, O, I, mstride, codes, scales, codes_t, scales_t, st)
                                  : weight_run<F16>(W, M, O, I, mstride, codes, scales, codes_t, scales_t, st);
}

}  // extern "C"
