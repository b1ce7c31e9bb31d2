// 8-bit blocks (block8.hpp): rows and weights to codes, codes back, and activations that keep their input in codes
// (hecka_block8_*; contract in include/hecka.h).  All HBM bound: one read of the input, one write of each output.
// Sixteen lanes own a block, eight elements each, so a wave covers four blocks with 16-byte loads (two per lane for fp32),
// the maximum is four lane permutes and the codes leave as 8 bytes per lane, 128 per block, contiguous.
// Measured at 10 x 4096 x 4096 (a copy reaches 5.3 TB/s): quantise 95 us bf16, 162 us fp32 (5.2 TB/s); decode 92 / 163 us (5.4 / 5.1); silu, tanh
// and sigmoid 167 / 286 us forward, 167 / 288 us backward (5.0 / 5.2), crater 168 / 180 in 16 bits; gelu fp32 287 / 288, fp16 178 / 178, bf16 217 / 200: the one that is
// near the vector units' rate (about fifty instructions an element).  With an exponential that is good for 16 bits only (its rounded exponent not
// put back) silu took 161, bf16 gelu 200 / 184 us.
#include "block8.hpp"
#include "hecka_host.hpp"

namespace hecka {

// A lane's eight elements of a block that begins at column col of a row of K: eight neighbours (one 16-byte piece), or of fp32 two
// pieces of four, 64 apart, so that every load and store instruction covers whole lines (decoding fp32, 10 x 4096 x 4096: 163 us, and
// 227 us with eight neighbours, whose stores are half lines each).
template <class T>
__device__ __forceinline__ void load_lane(const T* row, int col, int lane16, int K, Piece<T> (&p)[8 / Piece<T>::N]) {
#pragma unroll
  for (int j = 0; j < 8 / Piece<T>::N; ++j) p[j] = load_piece(row, col + j * 64 + lane16 * Piece<T>::N, K);
}
template <class T>
__device__ __forceinline__ void store_lane(T* row, int col, int lane16, int K, const Piece<T> (&p)[8 / Piece<T>::N]) {
#pragma unroll
  for (int j = 0; j < 8 / Piece<T>::N; ++j) {
    const int c = col + j * 64 + lane16 * Piece<T>::N;
    if (c < K) store_piece(row, c, K, p[j]);
  }
}
template <class T>
__device__ __forceinline__ void load_codes(const unsigned char* block, int lane16, unsigned (&c)[2]) {
  if constexpr (sizeof(T) == 4) {
    const unsigned* from = reinterpret_cast<const unsigned*>(block) + lane16;
    c[0] = from[0];
    c[1] = from[16];
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(block + lane16 * 8);
    c[0] = v.x;
    c[1] = v.y;
  }
}
template <class T>
__device__ __forceinline__ void store_codes(unsigned char* block, int lane16, const unsigned (&c)[2]) {
  if constexpr (sizeof(T) == 4) {
    unsigned* to = reinterpret_cast<unsigned*>(block) + lane16;
    to[0] = c[0];
    to[16] = c[1];
  } else {
    *reinterpret_cast<uint2*>(block + lane16 * 8) = make_uint2(c[0], c[1]);
  }
}
// eight neighbours [col, col + 8) of a weight's row of K
template <class T>
__device__ __forceinline__ void load8(const T* row, int col, int K, float* v) {
#pragma unroll
  for (int j = 0; j < 8 / Piece<T>::N; ++j) {
    const Piece<T> p = load_piece(row, col + j * Piece<T>::N, K);
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i) v[j * Piece<T>::N + i] = widen(p.e[i]);
  }
}
__device__ __forceinline__ float max8(const float* v) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = fmaxf(a, finite_abs(v[i]));
  return a;
}

enum { kActNone = 0, kActGelu = 1, kActSilu = 2, kActTanh = 3, kActSigmoid = 4, kActCrater = 5 };
static constexpr float kHalfRoot = 0.70710678118654752f, kCrater = 0.70710678118654752f + 0.008274364699f;

// e^(x + low), -1e4 <= x <= 0 and |low| far below 1, from the hardware's 2^x: the exponent's rounding error, |x| 2^-25, is worked out and put back,
// so the result is good to 3 u, u = 2^-24 (the hardware's own 2 u included); 0 where it is below 2^-126.
__device__ __forceinline__ float exp_near(float x, float low) {
  const float t = x * 1.44269504f;
  const float r = fmaf(x, 1.44269504f, -t) + x * 1.92596299e-8f;      // 1.44269504f + 1.92596299e-8f = log2 e
  const float p = __builtin_amdgcn_exp2f(t);
  return fmaf(p, fmaf(r, 0.69314718f, low), p);
}
// sigmoid(x) and 1 - sigmoid(x), both without cancellation: q = e^-|x| <= 1.  The hardware's 1 / (1 + q), a unit in the last place off, and the
// rounding of 1 + q are put right by one Newton step: the larger of the two is within u + 1.5 u (of q), the smaller within 5 u, u = 2^-24.
// Three instructions: no time in fp32, 1 - 2 % in 16 bits.
__device__ __forceinline__ void sigmoid_pair(float x, float& p, float& n) {
  const float q = exp_near(fmaxf(-fabsf(x), -104.f), 0.f), d = 1.0f + q, r = __builtin_amdgcn_rcpf(d);
  const float s = fmaf(r, fmaf(d - 1.0f - q, r, fmaf(-d, r, 1.0f)), r), qs = q * s;
  p = x >= 0.f ? s : qs;
  n = x >= 0.f ? qs : s;
  if (x != x) p = n = x;
}
// normal distribution below x, for x < 0 good relative to itself: with a = |x|, 0.5 erfc(a / sqrt 2) = e^(-a^2 / 2) t P(t), t = 1 / (1 + 0.265 a).
// P: degree 8, least relative error on 0 <= a <= 14.6 (1.4e-8; fitted with reweighted least squares, 0.265 is the best of a search); the
// evaluation in fp32 is within 6e-7 (10 u).  a^2 is rounded, and what that takes from the exponent put back: at a = 13 it is 42 u of the result.
// Beyond 20 both factors are zero as fp32 numbers.
__device__ __forceinline__ float normal_below(float x, float& bell) {
  const float a = fminf(fabsf(x), 20.f), t = __builtin_amdgcn_rcpf(fmaf(0.265f, a, 1.0f)), h = a * a;
  bell = exp_near(-0.5f * h, -0.5f * fmaf(a, a, -h));
  float c = fmaf(0.0305863377f, t, -0.143120438f);
  c = fmaf(c, t, 0.215588495f);
  c = fmaf(c, t, -0.113883875f);
  c = fmaf(c, t, 0.136284307f);
  c = fmaf(c, t, 0.0610073693f);
  c = fmaf(c, t, 0.102527015f);
  c = fmaf(c, t, 0.105270624f);
  c = fmaf(c, t, 0.105740167f);
  const float half = c * t * bell;
  return x >= 0.f ? 1.0f - half : half;
}

template <int ACT>
__device__ __forceinline__ float act_value(float x) {
  float p, n;
  if (ACT == kActGelu) return x * normal_below(x, n);
  if (ACT == kActTanh) return tanhf(x);
  sigmoid_pair(ACT == kActCrater ? 2.0f * kHalfRoot * (x + 1.0f) : x, p, n);      // 1 + tanh z = 2 sigmoid(2 z)
  return ACT == kActSilu ? x * p : ACT == kActSigmoid ? p : 2.0f * kCrater * (x * p);
}
template <int ACT>
__device__ __forceinline__ float act_slope(float x) {
  float p, n;
  if (ACT == kActGelu) {
    p = normal_below(x, n);
    return fmaf(x * 0.39894228f, n, p);
  }
  sigmoid_pair(ACT == kActTanh ? 2.0f * x : ACT == kActCrater ? 2.0f * kHalfRoot * (x + 1.0f) : x, p, n);
  if (ACT == kActTanh) return 4.0f * p * n;
  if (ACT == kActSigmoid) return p * n;
  if (ACT == kActSilu) return fmaf(x * p, n, p);
  return 2.0f * kCrater * fmaf(2.0f * kHalfRoot, x * (p * n), p);
}

// Which blocks a group of sixteen lanes works on, and where they lie.  FLAT (whole blocks, rows without gaps, their number a
// multiple of four so that the scale bytes have none either): everything is one long row.  UNROLL blocks at a time are loaded before
// the first is worked on: one block per lane group in flight (128 bytes of codes) leaves the memory idle - decoding bf16 reached
// 2.75 TB/s that way.
template <bool FLAT>
struct Place { long long row; int blk; };
template <bool FLAT>
__device__ __forceinline__ Place<FLAT> place_block(long long b, long long total, int nblk) {
  if constexpr (FLAT) return {0, 0};
  const long long row = total <= 0xffffffffLL ? (long long)((unsigned)b / (unsigned)nblk) : b / nblk;
  return {row, (int)(b - row * nblk)};
}

// rows of K elements, `ld` apart; ACT != 0: y (rows of K, contiguous) = act(x) beside the codes of x, or alone where codes is null
template <class T, int ACT, bool FLAT>
__global__ __launch_bounds__(256) void block8_rows_kernel(const T* __restrict__ x, long long R, int K, long long ld,
                                                          unsigned char* __restrict__ codes, unsigned char* __restrict__ scales,
                                                          T* __restrict__ y) {
  constexpr int UNROLL = 16 / sizeof(T) / 2;      // 4 (16-bit) or 2 blocks: 64 bytes per lane
  const int nblk = row_blocks(K), lane16 = threadIdx.x & 15, group = threadIdx.x >> 4;
  const long long total = R * nblk;
  for (long long b0 = (long long)blockIdx.x * (16 * UNROLL) + group; b0 < total; b0 += (long long)gridDim.x * (16 * UNROLL)) {
    Piece<T> p[UNROLL][8 / Piece<T>::N];
    Place<FLAT> at[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const long long b = b0 + u * 16 < total ? b0 + u * 16 : total - 1;
      at[u] = place_block<FLAT>(b, total, nblk);
      if constexpr (FLAT) load_lane(x + b * kBlock, 0, lane16, kBlock, p[u]);
      else load_lane(x + at[u].row * ld, at[u].blk * kBlock, lane16, K, p[u]);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const long long b = b0 + u * 16;
      if (b >= total) break;
      if (ACT != kActNone) {
        Piece<T> a[8 / Piece<T>::N];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          narrow(act_value<ACT>(widen(p[u][i / Piece<T>::N].e[i % Piece<T>::N])), a[i / Piece<T>::N].e[i % Piece<T>::N]);
        if constexpr (FLAT) store_lane(y + b * kBlock, 0, lane16, kBlock, a);
        else store_lane(y + at[u].row * K, at[u].blk * kBlock, lane16, K, a);
      }
      if (ACT != kActNone && !codes) continue;
      unsigned c[2];
      const int byte = encode<T, 8>(p[u], c, [](unsigned v) { return max16(v); });
      store_codes<T>(codes + b * kBlock, lane16, c);
      if (lane16 == 0) {
        if constexpr (FLAT) {
          scales[b] = (unsigned char)byte;
        } else {
          unsigned char* s = scales + at[u].row * ((nblk + 3) & ~3);
          s[at[u].blk] = (unsigned char)byte;
          if (at[u].blk == nblk - 1)
            for (int i = nblk; i < ((nblk + 3) & ~3); ++i) s[i] = 127;
        }
      }
    }
  }
}

// ACT = 0: out = the values of the codes; else out = dy * act'(values)
template <class T, int ACT, bool FLAT>
__global__ __launch_bounds__(256) void block8_values_kernel(const unsigned char* __restrict__ codes,
                                                            const unsigned char* __restrict__ scales, const T* __restrict__ dy,
                                                            long long R, int K, T* __restrict__ out) {
  constexpr int UNROLL = ACT == kActNone ? 4 : 16 / sizeof(T) / 2;
  const int nblk = row_blocks(K), lane16 = threadIdx.x & 15, group = threadIdx.x >> 4;
  const long long total = R * nblk;
  for (long long b0 = (long long)blockIdx.x * (16 * UNROLL) + group; b0 < total; b0 += (long long)gridDim.x * (16 * UNROLL)) {
    unsigned c[UNROLL][2];
    int byte[UNROLL];
    Piece<T> d[UNROLL][8 / Piece<T>::N];
    Place<FLAT> at[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const long long b = b0 + u * 16 < total ? b0 + u * 16 : total - 1;
      at[u] = place_block<FLAT>(b, total, nblk);
      load_codes<T>(codes + b * kBlock, lane16, c[u]);
      byte[u] = FLAT ? scales[b] : scales[at[u].row * ((nblk + 3) & ~3) + at[u].blk];
      if (ACT != kActNone) {
        if constexpr (FLAT) load_lane(dy + b * kBlock, 0, lane16, kBlock, d[u]);
        else load_lane(dy + at[u].row * K, at[u].blk * kBlock, lane16, K, d[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const long long b = b0 + u * 16;
      if (b >= total) break;
      float v[8];
      decode4(c[u][0], scale_of(byte[u]), v);
      decode4(c[u][1], scale_of(byte[u]), v + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        T& e = d[u][i / Piece<T>::N].e[i % Piece<T>::N];
        if (ACT != kActNone) v[i] = widen(e) * act_slope<ACT>(v[i]);
        else if (__is_same(T, F16) && fabsf(v[i]) == 65536.f) v[i] = copysignf(65504.f, v[i]);      // fp16's largest, 65504, is kept as 65536: back to what fp16 holds
        narrow(v[i], e);
      }
      if constexpr (FLAT) store_lane(out + b * kBlock, 0, lane16, kBlock, d[u]);
      else store_lane(out + at[u].row * K, at[u].blk * kBlock, lane16, K, d[u]);
    }
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

// workgroups of a streaming launch: 16 `unroll` blocks each a turn, at most eight per CU
static unsigned stream_grid(long long blocks, int unroll) {
  const long long want = (blocks + 16 * unroll - 1) / (16 * unroll);
  return (unsigned)(want < 2048 ? want : 2048);
}

template <class T>
static int rows_run(const void* x, long long R, int K, long long ld, void* codes, void* scales, int act, void* y, hipStream_t st) {
  const unsigned grid = stream_grid(R * row_blocks(K), 8 / sizeof(T));
  const bool flat = K % (4 * kBlock) == 0 && ld == K;
#define HECKA_ROWS(A) \
  case A: \
    if (flat) block8_rows_kernel<T, A, true><<<grid, 256, 0, st>>>((const T*)x, R, K, ld, (unsigned char*)codes, (unsigned char*)scales, (T*)y); \
    else block8_rows_kernel<T, A, false><<<grid, 256, 0, st>>>((const T*)x, R, K, ld, (unsigned char*)codes, (unsigned char*)scales, (T*)y); \
    break;
  switch (act) { HECKA_ROWS(kActNone) HECKA_ROWS(kActGelu) HECKA_ROWS(kActSilu) HECKA_ROWS(kActTanh) HECKA_ROWS(kActSigmoid) HECKA_ROWS(kActCrater) }
#undef HECKA_ROWS
  return check_launch("block8_rows");
}
template <class T>
static int values_run(const void* codes, const void* scales, const void* dy, long long R, int K, int act, void* out, hipStream_t st) {
  const unsigned grid = stream_grid(R * row_blocks(K), act == kActNone ? 4 : 8 / sizeof(T));
  const bool flat = K % (4 * kBlock) == 0;
#define HECKA_VALUES(A) \
  case A: \
    if (flat) block8_values_kernel<T, A, true><<<grid, 256, 0, st>>>((const unsigned char*)codes, (const unsigned char*)scales, (const T*)dy, R, K, (T*)out); \
    else block8_values_kernel<T, A, false><<<grid, 256, 0, st>>>((const unsigned char*)codes, (const unsigned char*)scales, (const T*)dy, R, K, (T*)out); \
    break;
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
  if (!x || !codes != !scales || (act == kActNone && !codes) || (act != kActNone && !y)) return fail(HECKA_EINVAL, "block8_quantize: null pointer%s");
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
