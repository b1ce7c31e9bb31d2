// Layer norm over the last axis, forward and backward (hecka_layernorm_fwd / _bwd; contract in include/hecka.h).
//
//   mu = mean x, r = 1 / sqrt(mean (x - mu)^2 + eps), xh = (x - mu) r, y = xh w + b
//   g = dy w, dx = r (g - mean g - xh mean(g xh)), dw = sum_rows dy xh, db = sum_rows dy
//
// HBM bound: the forward reads x and writes y once, the backward reads x and dy and writes dx once.  A row therefore stays in
// the registers of TPR threads (16 elements each at most) between its loads and its stores, so that the variance is the
// two-pass one (mean first, then squared distances) at no extra traffic; all statistics are fp32.  A row of up to 1024
// elements belongs to 8, 16, 32 or 64 lanes of a wave (its sums need no barrier), a longer one to 128 (forward only), 256, 512 or 1024
// threads; the next row's loads are under way while a row is summed.
// Measured (a copy reaches 5.3 TB/s): 2 x 16384 x 8192 bf16 209 us forward (5.1 TB/s), 335 us backward (4.8); 10 x 2048 x 2048 fp32 65 us
// (5.2) and 112 us (4.5, the partial sums included); rows of 1001 fp16, 5 x 300: 6 and 18 us, latency.
// The backward keeps every thread's columns of dw and db in registers over all rows of its workgroup and writes them once:
// [workgroups per member, 2, D] partial sums, added up in a fixed order by a second kernel - no atomics, the same bits on
// every run.
#include "hecka_host.hpp"
#include "hecka_vec.hpp"

namespace hecka {

// Sum of a value over the TPR threads of a row.  `red` is one of two LDS buffers used in turn: a wave that is past the
// barrier of one sum writes the other buffer next, so one barrier per sum suffices.
template <int TPR>
__device__ __forceinline__ float row_sum(float a, float* red) {
  constexpr int NW = TPR / 64;
  a = lanes_sum<TPR < 64 ? TPR : 64>(a);
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    a = red[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) a += red[i];
  }
  return a;
}
// of two values at once
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* red) {
  constexpr int NW = TPR / 64;
  a = lanes_sum<TPR < 64 ? TPR : 64>(a);
  b = lanes_sum<TPR < 64 ? TPR : 64>(b);
  if constexpr (NW > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) { red[wave] = a; red[NW + wave] = b; }
    __syncthreads();
    a = red[0];
    b = red[NW];
#pragma unroll
    for (int i = 1; i < NW; ++i) { a += red[i]; b += red[NW + i]; }
  }
}

// a thread's pieces of row r of a member's rows (those of the last row again where r is behind it)
template <class T, int TPR, int NV>
__device__ __forceinline__ void load_row(Piece<T> (&p)[NV], const T* x, long long r, long long R, int D, int lane) {
  const T* row = x + (r < R ? r : R - 1) * D;
#pragma unroll
  for (int j = 0; j < NV; ++j) p[j] = load_piece(row, (j * TPR + lane) * Piece<T>::N, D);
}
template <class T, int TPR, int NV>
__device__ __forceinline__ void load_params(float (&v)[NV * Piece<T>::N], const float* w, int D, int lane, float none) {
  constexpr int N = Piece<T>::N;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int h = 0; h < N / 4; ++h) {
      const int c = (j * TPR + lane) * N + 4 * h;
      const Piece<float> p = w ? load_piece(w, c, D) : Piece<float>{none, none, none, none};
#pragma unroll
      for (int i = 0; i < 4; ++i) v[j * N + 4 * h + i] = p.e[i];
    }
  }
}

template <class T, int TPR, int NV>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void layernorm_fwd_kernel(
    const T* __restrict__ x, long long R, int D, int chunks, const float* __restrict__ w, const float* __restrict__ b,
    long long wstride, float eps, T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int N = Piece<T>::N, RPB = TPR <= 64 ? 256 / TPR : 1;
  __shared__ float red[2][TPR < 64 ? 1 : TPR / 64];
  const long long m = blockIdx.x / chunks, step = (long long)chunks * RPB;
  const int chunk = blockIdx.x % chunks, sub = threadIdx.x / TPR, lane = threadIdx.x % TPR;
  float wr[NV * N], br[NV * N];
  Piece<T> p[NV];
  long long r = (long long)chunk * RPB + sub;
  x += m * R * D;
  y += m * R * D;
  load_row<T, TPR, NV>(p, x, r, R, D, lane);
  load_params<T, TPR, NV>(wr, w ? w + m * wstride : nullptr, D, lane, 1.f);
  load_params<T, TPR, NV>(br, b ? b + m * wstride : nullptr, D, lane, 0.f);
  for (; r < R; r += step) {
    float v[NV * N], s = 0.f;
#pragma unroll
    for (int k = 0; k < NV * N; ++k) { v[k] = widen(p[k / N].e[k % N]); s += v[k]; }
    load_row<T, TPR, NV>(p, x, r + step, R, D, lane);
    const float mu = row_sum<TPR>(s, red[0]) / (float)D;      // a division: a constant row of exact sum has this mean
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < NV * N; ++k) {
      v[k] -= mu;
      if ((k / N * TPR + lane) * N + k % N < D) q = fmaf(v[k], v[k], q);
    }
    const float rs = 1.0f / sqrtf(row_sum<TPR>(q, red[1]) / (float)D + eps);
    if (mean && lane == 0) { mean[m * R + r] = mu; rstd[m * R + r] = rs; }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Piece<T> o;
#pragma unroll
      for (int i = 0; i < N; ++i) narrow(fmaf(v[j * N + i] * rs, wr[j * N + i], br[j * N + i]), o.e[i]);
      store_piece(y + r * D, (j * TPR + lane) * N, D, o);
    }
  }
}

// AHEAD: the next row's pieces are loaded while a row is summed (up to 8 elements per thread).  Otherwise (16 elements) the
// registers hold one row, and what a row's sums took from its pieces is worked out again for dx.
template <class T, int TPR, int NV, bool AHEAD>
__global__ __launch_bounds__(TPR <= 64 ? 256 : TPR) void layernorm_bwd_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean, const float* __restrict__ rstd,
    long long R, int D, int chunks, const float* __restrict__ w, long long wstride, T* __restrict__ dx,
    float* __restrict__ dw, float* __restrict__ db, long long gstride, long long pstride) {
  constexpr int N = Piece<T>::N, E = NV * N, RPB = TPR <= 64 ? 256 / TPR : 1;
  __shared__ float red[2][TPR < 64 ? 1 : TPR / 32];
  __shared__ float fold[RPB > 1 ? RPB - 1 : 1][RPB > 1 ? TPR : 1][RPB > 1 ? 2 * E + 1 : 1];
  const long long m = blockIdx.x / chunks, step = (long long)chunks * RPB;
  const int chunk = blockIdx.x % chunks, sub = threadIdx.x / TPR, lane = threadIdx.x % TPR;
  float wr[E], aw[E], ab[E];
  Piece<T> px[NV], pd[NV];
  long long r = (long long)chunk * RPB + sub;
  x += m * R * D;
  dy += m * R * D;
  mean += m * R;
  rstd += m * R;
  if (AHEAD) {
    load_row<T, TPR, NV>(px, x, r, R, D, lane);
    load_row<T, TPR, NV>(pd, dy, r, R, D, lane);
  }
  load_params<T, TPR, NV>(wr, w ? w + m * wstride : nullptr, D, lane, 1.f);
#pragma unroll
  for (int k = 0; k < E; ++k) aw[k] = ab[k] = 0.f;
  const float inv = 1.0f / (float)D;
  int turn = 0;
  for (; r < R; r += step, turn ^= 1) {
    const float mu = mean[r], rs = rstd[r];
    if (!AHEAD) {
      load_row<T, TPR, NV>(px, x, r, R, D, lane);
      load_row<T, TPR, NV>(pd, dy, r, R, D, lane);
    }
    float g[AHEAD ? E : 1], h[AHEAD ? E : 1], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const float d = widen(pd[k / N].e[k % N]);      // zero behind the row's end, as d w then is: nothing of it enters the sums
      const float xh = (widen(px[k / N].e[k % N]) - mu) * rs, dw_ = d * wr[k];
      aw[k] = fmaf(d, xh, aw[k]);
      ab[k] += d;
      s1 += dw_;
      s2 = fmaf(dw_, xh, s2);
      if (AHEAD) { g[k] = dw_; h[k] = xh; }
    }
    if (AHEAD) {
      load_row<T, TPR, NV>(px, x, r + step, R, D, lane);
      load_row<T, TPR, NV>(pd, dy, r + step, R, D, lane);
    }
    if (dx) {
      row_sum2<TPR>(s1, s2, red[turn]);
      s1 *= inv;
      s2 *= inv;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        Piece<T> o;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int k = j * N + i;
          const float gk = AHEAD ? g[AHEAD ? k : 0] : widen(pd[j].e[i]) * wr[k];
          const float hk = AHEAD ? h[AHEAD ? k : 0] : (widen(px[j].e[i]) - mu) * rs;
          narrow(rs * (gk - s1 - hk * s2), o.e[i]);
        }
        store_piece(dx + (m * R + r) * D, (j * TPR + lane) * N, D, o);
      }
    }
  }
  if (!dw && !db) return;
  if constexpr (RPB > 1) {     // the sums of the same columns of different rows, added in order
    if (sub > 0) {
#pragma unroll
      for (int k = 0; k < NV * N; ++k) { fold[sub - 1][lane][2 * k] = aw[k]; fold[sub - 1][lane][2 * k + 1] = ab[k]; }
    }
    __syncthreads();
    if (sub > 0) return;
#pragma unroll 1
    for (int o = 0; o < RPB - 1; ++o) {
#pragma unroll
      for (int k = 0; k < NV * N; ++k) { aw[k] += fold[o][lane][2 * k]; ab[k] += fold[o][lane][2 * k + 1]; }
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int h = 0; h < N / 4; ++h) {
      const int c = (j * TPR + lane) * N + 4 * h, k = j * N + 4 * h;
      if (c < D) {
        if (dw) store_piece(dw + m * gstride + chunk * pstride, c, D, Piece<float>{aw[k], aw[k + 1], aw[k + 2], aw[k + 3]});
        if (db) store_piece(db + m * gstride + chunk * pstride, c, D, Piece<float>{ab[k], ab[k + 1], ab[k + 2], ab[k + 3]});
      }
    }
  }
}

// out[m][c] = sum over the P partial rows part[m][p][c], in a fixed order: 16 slices of p per column (a wave reads 64
// neighbouring columns), then the slices in order.  Columns [0, D) go to dw, [D, 2 D) to db.
__global__ __launch_bounds__(1024) void layernorm_fold_kernel(const float* __restrict__ part, int P, int D,
                                                              float* __restrict__ dw, float* __restrict__ db, long long gstride) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
  const long long m = blockIdx.y;
  const int c = blockIdx.x * 64 + lane;
  const float* p0 = part + m * P * 2 * D;
  float s = 0.f;
  if (c < 2 * D) {
#pragma unroll 8
    for (int p = slice; p < P; p += 16) s += p0[(long long)p * 2 * D + c];
  }
  red[slice][lane] = s;
  __syncthreads();
  if (slice == 0 && c < 2 * D) {
#pragma unroll
    for (int i = 1; i < 16; ++i) s += red[i][lane];
    float* o = c < D ? dw : db;
    if (o) o[m * gstride + (c < D ? c : c - D)] = s;
  }
}

static const int kMaxNormWidth = 16384;

// Threads of a row: few enough that most have work (a piece is 4 or 8 elements), enough that none has more than 16 elements
// (forward) or 8 (backward, which holds five values for each and would leave too few waves: bf16 rows of 8192 350 us with 8
// elements in 1024 threads, 475 us with 16 in 512).  Beyond 8192 the backward has 16 as well and loads nothing ahead.  Up to 1024
// elements a wave at most, whose sums need no barrier (2^25 elements of bf16, rows of 1024: 23 / 40 us forward / backward, 28 / 47 with two waves; of
// 128: 23 / 40 us with 16 lanes, 80 / 107 with 64; of 64: 23 / 41 us with 8 lanes, 43 / 62 with 16).
static int norm_threads(int D, int piece, bool forward) {
  if (D <= 8 * piece) return 8;
  if (D <= 16 * piece) return 16;
  if (D <= 32 * piece) return 32;
  if (D <= 1024) return 64;
  const int share = forward || D > 8192 ? 16 : 8;
  return D <= 128 * share ? 128 : D <= 256 * share ? 256 : D <= 512 * share ? 512 : 1024;
}

// Workgroups per member: every row its own share, up to `most` in all.  Forward: eight per CU, but for long rows (whose weight
// and bias, 8 bytes an element, a workgroup reads once) two.  Backward: enough to fill the chip once with sixteen waves per CU,
// so that the partial sums stay a few per cent of the traffic.
// 2^25 elements of bf16, rows of 2048, forward / backward: 24 / 42 us, with half as many 31 / 49, with twice as many 25 / 50; rows of
// 8192: 27 / 44, 26 / 45 and 29 / 54.
static int norm_chunks(long long G, long long R, int threads, bool forward) {
  const int rpb = threads <= 64 ? 256 / threads : 1;
  const long long most = forward ? (threads >= 1024 ? 512 : threads == 512 ? 1024 : 2048) : threads <= 256 ? 1024 : threads == 512 ? 512 : 256;
  const long long want = (R + rpb - 1) / rpb, share = most / G < 1 ? 1 : most / G;
  return (int)(want < share ? want : share);
}

template <class T, class F>
static int norm_dispatch(int D, const F& f) {
  constexpr int N = Piece<T>::N;
  const int t = norm_threads(D, N, F::kForward), need = (D + t * N - 1) / (t * N);      // pieces per thread
  switch (t) {
    case 8: return f.template run<T, 8, 1>();
    case 16: return f.template run<T, 16, 1>();
    case 32: return f.template run<T, 32, 1>();
    case 64: return need <= 1 ? f.template run<T, 64, 1>() : need <= 2 ? f.template run<T, 64, 2>() : f.template run<T, 64, 16 / N>();
  }
  if constexpr (F::kForward) {      // more than half of 16 elements a thread
    switch (t) {
      case 128: return f.template run<T, 128, 16 / N>();
      case 256: return f.template run<T, 256, 16 / N>();
      case 512: return f.template run<T, 512, 16 / N>();
      case 1024: return f.template run<T, 1024, 16 / N>();
    }
  } else {                          // more than half of 8, or of 16 beyond 8192
    switch (t) {
      case 256: return f.template run<T, 256, 8 / N>();
      case 512: return f.template run<T, 512, 8 / N>();
      case 1024: return D <= 8192 ? f.template run<T, 1024, 8 / N>() : f.template run<T, 1024, 16 / N>();
    }
  }
  return HECKA_EINVAL;
}

struct NormFwd {
  static constexpr bool kForward = true;
  const void* x; long long G, R; int D; const float *w, *b; long long wstride; float eps; void* y; float *mean, *rstd; hipStream_t st;
  template <class T, int TPR, int NV> int run() const {
    const int chunks = norm_chunks(G, R, TPR, true);
    layernorm_fwd_kernel<T, TPR, NV><<<dim3((unsigned)(G * chunks)), TPR <= 64 ? 256 : TPR, 0, st>>>(
        (const T*)x, R, D, chunks, w, b, wstride, eps, (T*)y, mean, rstd);
    return check_launch("layernorm_fwd");
  }
};
struct NormBwd {
  static constexpr bool kForward = false;
  const void *dy, *x; const float *mean, *rstd; long long G, R; int D; const float* w; long long wstride; void* dx; float *dw, *db; long long gstride; float* ws; hipStream_t st;
  template <class T, int TPR, int NV> int run() const {
    constexpr bool AHEAD = NV * Piece<T>::N <= 8;
    const int chunks = norm_chunks(G, R, TPR, false);
    const bool part = chunks > 1 && (dw || db);
    layernorm_bwd_kernel<T, TPR, NV, AHEAD><<<dim3((unsigned)(G * chunks)), TPR <= 64 ? 256 : TPR, 0, st>>>(
        (const T*)dy, (const T*)x, mean, rstd, R, D, chunks, w, wstride, (T*)dx, part ? ws : dw, part ? ws + D : db,
        part ? (long long)chunks * 2 * D : gstride, part ? 2LL * D : 0);
    if (part)
      layernorm_fold_kernel<<<dim3((2 * D + 63) / 64, (unsigned)G), 1024, 0, st>>>(ws, chunks, D, dw, db, gstride);
    return check_launch("layernorm_bwd");
  }
};

template <class F>
static int norm_type(int dtype, int D, const F& f) {
  return dtype == HECKA_DT_F32 ? norm_dispatch<float>(D, f) : dtype == HECKA_DT_BF16 ? norm_dispatch<Bf16>(D, f) : norm_dispatch<F16>(D, f);
}

static int norm_check(const char* what, int dtype, int G, long long R, int D) {
  if (dtype != HECKA_DT_F32 && dtype != HECKA_DT_BF16 && dtype != HECKA_DT_F16) return fail(HECKA_EINVAL, "%s: unknown dtype", what);
  if (G <= 0 || R <= 0 || D <= 0 || G > 65535) return fail(HECKA_EINVAL, "%s: bad size (G = %lld, rows = %lld)", what, G, R);
  if (D > kMaxNormWidth) return fail(HECKA_EINVAL, "%s: rows longer than 16384 elements (%lld)", what, D);
  return HECKA_OK;
}

}  // namespace hecka

using namespace hecka;

extern "C" {

int hecka_layernorm_fwd(const void* x, int dtype, int G, long long R, int D, const float* weight, const float* bias,
                        long long wstride, float eps, void* y, float* mean, float* rstd, void* stream) {
  if (int rc = norm_check("layernorm_fwd", dtype, G, R, D)) return rc;
  if (!x || !y || !mean != !rstd) return fail(HECKA_EINVAL, "layernorm_fwd: null pointer%s");
  clear_error();
  return norm_type(dtype, D, NormFwd{x, G, R, D, weight, bias, wstride, eps, y, mean, rstd, (hipStream_t)stream});
}

size_t hecka_layernorm_bwd_workspace_bytes(int G, long long R, int D) {
  if (G <= 0 || R <= 0 || D <= 0 || G > 65535 || D > kMaxNormWidth) return 0;
  const int fp32 = norm_chunks(G, R, norm_threads(D, 4, false), false), other = norm_chunks(G, R, norm_threads(D, 8, false), false);
  const int chunks = fp32 > other ? fp32 : other;
  return chunks > 1 ? (size_t)G * chunks * 2 * D * sizeof(float) : 0;
}

int hecka_layernorm_bwd(const void* dy, const void* x, int dtype, const float* mean, const float* rstd, int G, long long R,
                        int D, const float* weight, long long wstride, void* dx, float* dweight, float* dbias,
                        long long gstride, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = norm_check("layernorm_bwd", dtype, G, R, D)) return rc;
  if (!dy || !x || !mean || !rstd) return fail(HECKA_EINVAL, "layernorm_bwd: null pointer%s");
  if (!dx && !dweight && !dbias) return HECKA_OK;
  if ((dweight || dbias) && (ws ? ws_bytes : 0) < hecka_layernorm_bwd_workspace_bytes(G, R, D))
    return fail(HECKA_EWORKSPACE, "%slayernorm_bwd: workspace too small (%lld bytes given)", "", (long long)ws_bytes);
  clear_error();
  return norm_type(dtype, D, NormBwd{dy, x, mean, rstd, G, R, D, weight, wstride, dx, dweight, dbias, gstride, (float*)ws,
                                     (hipStream_t)stream});
}

}  // extern "C"
