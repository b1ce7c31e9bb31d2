// Layer norm over the last axis, forward and backward (hecka_layernorm_fwd / _bwd; contract in include/hecka.h).
//
//   mu = mean x, r = 1 / sqrt(mean (x - mu)^2 + eps), xh = (x - mu) r, y = xh w + b
//   g = dy w, dx = r (g - mean g - xh mean(g xh)), dw = sum_rows dy xh, db = sum_rows dy
//
// HBM bound: the forward reads x and writes y once, the backward reads x and dy and writes dx once.  A row therefore stays in
// the registers of TPR threads (16 elements each at most) between its loads and its stores, so that the variance is the
// two-pass one (mean first, then squared distances) at no extra traffic; all statistics are fp32.  A row of up to 1024
// elements belongs to one wave (its sums are shuffles, no barrier), a longer one to 256 / 512 / 1024 threads.
// The backward keeps every thread's columns of dw and db in registers over all rows of its workgroup and writes them once:
// [workgroups per member, 2, D] partial sums, added up in a fixed order by a second kernel - no atomics, the same bits on
// every run.  About 512 workgroups (two per CU) hold the partial sums to a few per cent of the traffic.
#include "hecka_host.hpp"
#include "hecka_vec.hpp"

namespace hecka {

// Sums of two values over the TPR threads of a row.  `red` is one of two LDS buffers used in turn: a wave that is past the
// barrier of one sum writes the other buffer next, so one barrier per sum suffices.
template <int TPR, int NW>
__device__ __forceinline__ void row_sum(float& a, float& b, float (*red)[2]) {
  a = wave_sum(a);
  b = wave_sum(b);
  if constexpr (NW > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) { red[wave][0] = a; red[wave][1] = b; }
    __syncthreads();
    a = red[0][0];
    b = red[0][1];
#pragma unroll
    for (int i = 1; i < NW; ++i) { a += red[i][0]; b += red[i][1]; }
  }
}
template <int TPR, int NW>
__device__ __forceinline__ float row_sum(float a, float (*red)[2]) {
  a = wave_sum(a);
  if constexpr (NW > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[wave][0] = a;
    __syncthreads();
    a = red[0][0];
#pragma unroll
    for (int i = 1; i < NW; ++i) a += red[i][0];
  }
  return a;
}

template <class T, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void layernorm_fwd_kernel(
    const T* __restrict__ x, long long R, int D, int chunks, const float* __restrict__ w, const float* __restrict__ b,
    long long wstride, float eps, T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int N = Piece<T>::N, NW = TPR / 64, RPB = TPR < 256 ? 256 / TPR : 1;
  __shared__ float red[2][NW][2];
  const long long m = blockIdx.x / chunks;
  const int chunk = blockIdx.x % chunks, sub = threadIdx.x / TPR, lane = threadIdx.x % TPR;
  float wr[NV * N], br[NV * N];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (j * TPR + lane) * N + i;
      wr[j * N + i] = w && c < D ? w[m * wstride + c] : 1.f;
      br[j * N + i] = b && c < D ? b[m * wstride + c] : 0.f;
    }
  }
  const float inv = 1.0f / (float)D;
  for (long long r = (long long)chunk * RPB + sub; r < R; r += (long long)chunks * RPB) {
    const T* xr = x + (m * R + r) * D;
    float v[NV * N], s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TPR + lane) * N;
      const Piece<T> p = load_piece(xr, c, D);
#pragma unroll
      for (int i = 0; i < N; ++i) { v[j * N + i] = widen(p.e[i]); s += v[j * N + i]; }
    }
    const float mu = row_sum<TPR, NW>(s, red[0]) / (float)D;      // a division: a constant row of exact sum has this mean
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[j * N + i] -= mu;
        if ((j * TPR + lane) * N + i < D) q = fmaf(v[j * N + i], v[j * N + i], q);
      }
    }
    const float rs = 1.0f / sqrtf(row_sum<TPR, NW>(q, red[1]) * inv + eps);
    if (mean && lane == 0) { mean[m * R + r] = mu; rstd[m * R + r] = rs; }
    T* yr = y + (m * R + r) * D;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Piece<T> p;
#pragma unroll
      for (int i = 0; i < N; ++i) narrow(fmaf(v[j * N + i] * rs, wr[j * N + i], br[j * N + i]), p.e[i]);
      store_piece(yr, (j * TPR + lane) * N, D, p);
    }
  }
}

template <class T, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void layernorm_bwd_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean, const float* __restrict__ rstd,
    long long R, int D, int chunks, const float* __restrict__ w, long long wstride, T* __restrict__ dx,
    float* __restrict__ dw, float* __restrict__ db, long long gstride, long long pstride) {
  constexpr int N = Piece<T>::N, NW = TPR / 64, RPB = TPR < 256 ? 256 / TPR : 1;
  __shared__ float red[2][NW][2];
  __shared__ float fold[RPB > 1 ? RPB - 1 : 1][RPB > 1 ? TPR : 1][RPB > 1 ? 2 * NV * N + 1 : 1];
  const long long m = blockIdx.x / chunks;
  const int chunk = blockIdx.x % chunks, sub = threadIdx.x / TPR, lane = threadIdx.x % TPR;
  float wr[NV * N], aw[NV * N], ab[NV * N];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (j * TPR + lane) * N + i;
      wr[j * N + i] = w && c < D ? w[m * wstride + c] : 1.f;
      aw[j * N + i] = ab[j * N + i] = 0.f;
    }
  }
  const float inv = 1.0f / (float)D;
  int turn = 0;
  for (long long r = (long long)chunk * RPB + sub; r < R; r += (long long)chunks * RPB, turn ^= 1) {
    const long long row = m * R + r;
    const float mu = mean[row], rs = rstd[row];
    float g[NV * N], h[NV * N], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TPR + lane) * N;
      const Piece<T> p = load_piece(x + row * D, c, D), q = load_piece(dy + row * D, c, D);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int k = j * N + i;
        const float d = widen(q.e[i]);      // zero behind the row's end, as g then is: nothing of it enters the sums
        h[k] = (widen(p.e[i]) - mu) * rs;
        aw[k] = fmaf(d, h[k], aw[k]);
        ab[k] += d;
        g[k] = d * wr[k];
        s1 += g[k];
        s2 = fmaf(g[k], h[k], s2);
      }
    }
    if (dx) {
      row_sum<TPR, NW>(s1, s2, red[turn]);
      s1 *= inv;
      s2 *= inv;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        Piece<T> p;
#pragma unroll
        for (int i = 0; i < N; ++i) narrow(rs * (g[j * N + i] - s1 - h[j * N + i] * s2), p.e[i]);
        store_piece(dx + row * D, (j * TPR + lane) * N, D, p);
      }
    }
  }
  if (!dw && !db) return;
  if constexpr (RPB > 1) {     // the waves' sums of the same columns, added in the order of the waves
    if (sub > 0) {
#pragma unroll
      for (int k = 0; k < NV * N; ++k) { fold[sub - 1][lane][2 * k] = aw[k]; fold[sub - 1][lane][2 * k + 1] = ab[k]; }
    }
    __syncthreads();
    if (sub > 0) return;
#pragma unroll
    for (int o = 0; o < RPB - 1; ++o) {
#pragma unroll
      for (int k = 0; k < NV * N; ++k) { aw[k] += fold[o][lane][2 * k]; ab[k] += fold[o][lane][2 * k + 1]; }
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (j * TPR + lane) * N + i;
      if (c < D) {
        if (dw) dw[m * gstride + chunk * pstride + c] = aw[j * N + i];
        if (db) db[m * gstride + chunk * pstride + c] = ab[j * N + i];
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

static int norm_threads(int D) { return D <= 1024 ? 64 : D <= 4096 ? 256 : D <= 8192 ? 512 : 1024; }

// workgroups per member: every row its own share up to `most` workgroups in all
static int norm_chunks(long long G, long long R, int D, long long most) {
  const int rpb = norm_threads(D) == 64 ? 4 : 1;
  const long long want = (R + rpb - 1) / rpb, share = most / G < 1 ? 1 : most / G;
  return (int)(want < share ? want : share);
}
static const long long kFwdBlocks = 2048, kBwdBlocks = 512;

template <class T, class F>
static int norm_dispatch(int D, const F& f) {
  constexpr int N = Piece<T>::N;
  const int t = norm_threads(D), need = (D + t * N - 1) / (t * N);      // pieces per thread: 1, 2 or (fp32) 4
#define HECKA_NORM(TPR) \
  case TPR: return need <= 1 ? f.template run<T, TPR, 1>() : need <= 2 ? f.template run<T, TPR, 2>() : f.template run<T, TPR, 16 / N>();
  switch (t) {
    HECKA_NORM(64)
    HECKA_NORM(256)
    HECKA_NORM(512)
    default: return need <= 1 ? f.template run<T, 1024, 1>() : need <= 2 ? f.template run<T, 1024, 2>() : f.template run<T, 1024, 16 / N>();
  }
#undef HECKA_NORM
}

struct NormFwd {
  const void* x; long long G, R; int D; const float *w, *b; long long wstride; float eps; void* y; float *mean, *rstd; hipStream_t st;
  template <class T, int TPR, int NV> int run() const {
    const int chunks = norm_chunks(G, R, D, kFwdBlocks);
    layernorm_fwd_kernel<T, TPR, NV><<<dim3((unsigned)(G * chunks)), TPR < 256 ? 256 : TPR, 0, st>>>(
        (const T*)x, R, D, chunks, w, b, wstride, eps, (T*)y, mean, rstd);
    return check_launch("layernorm_fwd");
  }
};
struct NormBwd {
  const void *dy, *x; const float *mean, *rstd; long long G, R; int D; const float* w; long long wstride; void* dx; float *dw, *db; long long gstride; float* ws; int chunks; hipStream_t st;
  template <class T, int TPR, int NV> int run() const {
    const bool part = chunks > 1 && (dw || db);
    layernorm_bwd_kernel<T, TPR, NV><<<dim3((unsigned)(G * chunks)), TPR < 256 ? 256 : TPR, 0, st>>>(
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
  const int chunks = norm_chunks(G, R, D, kBwdBlocks);
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
                                     norm_chunks(G, R, D, kBwdBlocks), (hipStream_t)stream});
}

}  // extern "C"
