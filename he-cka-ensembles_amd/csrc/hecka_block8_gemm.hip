// Products of 8-bit blocks (block8.hpp) on the matrix cores (hecka_block8_linear / _linear_token / _wgrad; include/hecka.h).
#include "block8.hpp"
#include "hecka_host.hpp"

namespace hecka {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef __attribute__((address_space(3))) i16x4* lds_i16x4;

// eight codes as bf16 times their scale: exact, a code has four significant bits (and 2^-133, the smallest bf16, is below 2^-9 2^-124)
__device__ __forceinline__ bf16x8 widen8(unsigned lo, unsigned hi, float s) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, s, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, s, true);
  bf16x8 r = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  return r;
}

// Loads that go straight to LDS: lane l's 16 (4) bytes land at base + 16 l (4 l).  As asm, because the compiler, which cannot tell
// the buffer that is being filled from the one that is being read, would wait for them before every LDS read; they write no
// register, and whoever issues them waits for them (wait_loads) before the barrier behind which they are read.
__device__ __forceinline__ unsigned lds_offset(const void* p) { return (unsigned)(uintptr_t)(lds_ptr)(const_cast<void*>(p)); }
__device__ __forceinline__ void load_lds16(i32x4 rsrc, int voffset, int soffset, unsigned base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :: "s"(__builtin_amdgcn_readfirstlane(base)), "v"(voffset), "s"(rsrc), "s"(soffset) : "memory", "m0");
}
__device__ __forceinline__ void load_lds4(const void* p, unsigned base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
               :: "s"(__builtin_amdgcn_readfirstlane(base)), "v"(p) : "memory", "m0");
}
// until LEFT of the loads are under way at most (they end in their order)
template <int LEFT>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(LEFT) : "memory"); }
__device__ __forceinline__ i32x4 buffer_of(const void* p) {      // raw buffer over the 2 GiB from p on
  const unsigned long long a = (unsigned long long)p;
  return i32x4{__builtin_amdgcn_readfirstlane((int)(unsigned)a), __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xffff)), 0x7fffffff, 0x00020000};
}

// Workgroup id -> tile.  Ids go round the eight XCDs; each XCD gets a contiguous run of tiles, walked in bands of up to four
// row tiles (eight or sixteen: 4 to 9 % slower), so that the operands which the tiles in flight on one XCD share stay in that XCD's L2.
__device__ __forceinline__ void place(int id, int total, int tn, int to, int& m, int& in, int& io) {
  const int q = total >> 3, r = total & 7, xcd = id & 7, at = id >> 3;
  int t = xcd < r ? xcd * (q + 1) + at : r * (q + 1) + (xcd - r) * q + at;
  const int per = tn * to;
  m = t / per;
  t -= m * per;
  const int band = t / (4 * to), first = band * 4, rows = tn - first < 4 ? tn - first : 4;
  t -= band * 4 * to;
  in = first + t % rows;
  io = t / rows;
}

// The results of a wave's 16 S x 16 S outputs, by way of LDS: a lane holds four neighbouring columns (row tile i of the first
// operand) of one row (column tile j), a store of a wave should cover whole lines.  `mine`: BYTES of LDS of this wave's own, for RP
// rows of RB bytes whose 16-byte piece c lies at c ^ (row & MASK).  out[row][col] = alpha acc + beta bias[col], `rows` x `cols` of
// them exist.
template <class T, int S, int BYTES>
__device__ __forceinline__ void store_tile(const f32x4v (&acc)[S][S], const Piece<float> (&bias)[S], float alpha, float beta,
                                           unsigned char* mine, T* out, long long ld, int rows, int cols) {
  constexpr int RB = 16 * S * (int)sizeof(T), CH = RB / 16, MASK = CH < 16 ? CH - 1 : 15, FIT = BYTES / RB;
  constexpr int RP = FIT >= 16 * S ? 16 * S : FIT >= 64 ? 64 : 32;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
#pragma unroll
  for (int pass = 0; pass < 16 * S / RP; ++pass) {
#pragma unroll
    for (int j = 0; j < RP / 16; ++j) {
#pragma unroll
      for (int i = 0; i < S; ++i) {
        struct { T e[4]; } v;
#pragma unroll
        for (int e = 0; e < 4; ++e) narrow(fmaf(alpha, acc[i][pass * (RP / 16) + j][e], beta * bias[i].e[e]), v.e[e]);
        const int row = j * 16 + l16, col = (i * 16 + 4 * g) * (int)sizeof(T);
        __builtin_memcpy(__builtin_assume_aligned(mine + row * RB + (((col >> 4) ^ (row & MASK)) << 4) + (col & 15), sizeof(v)), &v, sizeof(v));
      }
    }
#pragma unroll
    for (int t = 0; t < RP * CH / 64; ++t) {
      const int row = t * (64 / CH) + lane / CH, c = lane % CH, r = pass * RP + row, o = c * Piece<T>::N;
      const Piece<T> v = *reinterpret_cast<const Piece<T>*>(mine + row * RB + ((c ^ (row & MASK)) << 4));
      if (r < rows && o < cols) store_piece(out + r * ld, o, cols, v);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------
// y[m][n][o] = alpha sum_k x8[m][n][k] w8[m][o][k] + beta bias[m][o]
//
// A workgroup of four waves owns B x B outputs; per step, 128 codes (one block) of each of its rows come straight from memory into LDS
// (no registers), STAGES - 1 steps ahead of the products: one, or three (linear_run).  LDS rows are 128 bytes; the 16-byte piece c of row r sits
// at piece c ^ (r & 7), so that the sixteen rows which a fragment read touches fall on different banks.
// The weights are the first operand, so that a lane ends up with four neighbouring outputs of one row.
// EXACT = true: the codes are widened to bf16 on their way out of LDS - exact - and the bf16 instruction adds their products in fp32
//   (1.4e-7 at K = 8192).
// EXACT = false (HECKA_BLOCK8_FP8, 16-bit results only): the scaled fp8 instruction takes both scales as bytes, at nearly twice the
//   rate.  It adds groups of eight products aligned to the largest, keeping 13 bits below its leading one (measured; 1.5e-5 of the
//   result for normal values, whatever K), against a half step of 2^-8 of a bf16 result and 2^-11 of an fp16 one: a choice of the caller's.
// Bound by the matrix instructions at the clock that the power leaves them (zeros run a fifth faster than random values), and by LDS
// beside them: a step's 64 KB written and 128 KB read take three quarters of the time of its products.  256 x 256 tiles reach
// 2.42 - 2.64 PF (fp8) and 1.31 - 1.40 PF (widened) at 8192^3, where a library's plain products reach 2.70 - 3.16 and 1.41 - 1.58; 2048 x
// 8192 x 8192 2.25 / 1.39 PF (256 workgroups, one round: the first loads and the last stores hide behind nothing).  Four waves of 128 x 128 outputs each: 256 sums a lane leave every fragment read from LDS eight
// products, and one workgroup a CU.  128 x 128 tiles (1.47 PF at best) where those are too few for the chip (linear_plan).
// ------------------------------------------------------------------------------------------------------------------
template <bool EXACT> struct Raw { typedef i32x8 type; };
template <> struct Raw<true> { typedef i32x4 type; };
__device__ __forceinline__ i32x4 half4(i32x8 v, int h) {
  return h ? __builtin_shufflevector(v, v, 4, 5, 6, 7) : __builtin_shufflevector(v, v, 0, 1, 2, 3);
}
// The products of the 256 x 256 tiles as asm: all 256 accumulation registers of a lane are sums here, and the compiler, left to itself, moves sums
// about to place a result elsewhere than its addend, and the instructions to where they hide nothing.  What an instruction
// needs then is up to this code: two idle issue slots behind a vector instruction that wrote an operand (mfma_ready, once before a
// group of products whose operands are all there - most come from LDS and need none; an idle pair before every product cost 8 % of
// the bf16 rate), and 18 behind the last product before a sum is read (mfma_settle).
__device__ __forceinline__ void mfma_fp8(f32x4v& c, i32x8 a, i32x8 b, unsigned sa, unsigned sb) {
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]" : "+a"(c) : "v"(a), "v"(b), "v"(sa), "v"(sb));
}
__device__ __forceinline__ void mfma_bf16(f32x4v& c, i32x4 a, i32x4 b) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
// Sums in ordinary registers, from zero and further: settled before anything else can touch them.
__device__ __forceinline__ void first_columns(f32x4v& c, i32x4 a, i32x4 b) {
  asm volatile("s_nop 3\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void add_columns(f32x4v& c, i32x4 a, i32x4 b) {
  asm volatile("s_nop 3\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void settle_columns(f32x4v& c) { asm volatile("s_nop 15\n\ts_nop 3" : "+v"(c)); }

// A sum of any number of terms as accurate as one of a few: hi + lo, lo what the additions to hi have rounded off (exactly worked out: Knuth's
// two-sum).  Once hi is not finite lo is NaN and hi the answer.
struct Long { float hi, lo; };
__device__ __forceinline__ void add(Long& s, float t) {
  const float sum = s.hi + t, part = sum - s.hi;
  s.lo += (s.hi - (sum - part)) + (t - part);
  s.hi = sum;
}
__device__ __forceinline__ float value(const Long& s) { return s.lo == s.lo ? s.hi + s.lo : s.hi; }
// The same by the compiler's own means, which waits for what needs it: for the smaller tiles, whose sums leave it registers.
template <bool OWN>
__device__ __forceinline__ void mul_fp8(f32x4v& c, i32x8 a, i32x8 b, unsigned sa, unsigned sb) {
  if constexpr (OWN) mfma_fp8(c, a, b, sa, sb);
  else c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, (int)sa, 0, (int)sb);
}
template <bool OWN>
__device__ __forceinline__ void mul_bf16(f32x4v& c, i32x4 a, i32x4 b) {
  if constexpr (OWN) mfma_bf16(c, a, b);
  else c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ void mfma_ready() { asm volatile("s_nop 1"); }
__device__ __forceinline__ void mfma_settle() { asm volatile("s_nop 15\n\ts_nop 15"); }

template <class T, bool EXACT, int B, int STAGES>
__global__ __launch_bounds__(256) void block8_linear_kernel(
    const unsigned char* __restrict__ x, const unsigned char* __restrict__ xs, long long xstride, long long xsstride,
    const unsigned char* __restrict__ w, const unsigned char* __restrict__ ws, int N, int O, int allblk, int share,
    const float* __restrict__ bias, long long bstride, float alpha, float beta, T* __restrict__ y, int tiles_n, int tiles_o) {
  constexpr int TO = B / 32, TN = B / 32, U = EXACT ? 2 : 1, SYNC = TO / 2, L = B / 32, STAGE = 2 * B * kBlock;
  __shared__ __attribute__((aligned(1024))) unsigned char sm[STAGES][STAGE];
  __shared__ unsigned sc[2][2 * B];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wo = wave & 1, wn = wave >> 1, l16 = lane & 15, g = lane >> 4;
  int m, tn, to;
  place(blockIdx.x, gridDim.x, tiles_n, tiles_o, m, tn, to);
  const int n0 = tn * B, o0 = to * B, sstride = (allblk + 3) & ~3;
  const long long K = (long long)allblk * kBlock;
  // the blocks of K of this workgroup: share of them (a multiple of four: whole dwords of scales) from blockIdx.y * share on, its sums
  // to slab blockIdx.y
  const int first = blockIdx.y * share, nblk = allblk - first < share ? allblk - first : share;
  x += m * xstride + (long long)first * kBlock;
  xs += m * xsstride + first;
  w += (long long)m * O * K + (long long)first * kBlock;
  ws += (long long)m * ((O + kBlock - 1) / kBlock) * sstride + first;

  // what this lane loads: row (4 i + wave) 8 + lane / 8 of each operand's tile, rows behind the end repeat the last one;
  // offsets from the tile's first row stay below 2^30 (256 rows of at most 2^22), the step is the loads' scalar offset
  const i32x4 rw = buffer_of(w + (long long)o0 * K), rx = buffer_of(x + (long long)n0 * K);
  int vw[L], vx[L];
  const int piece = ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int r = (i * 4 + wave) * 8 + (lane >> 3);
    vw[i] = (o0 + r < O ? r : O - 1 - o0) * (int)K + piece;
    vx[i] = (n0 + r < N ? r : N - 1 - n0) * (int)K + piece;
  }
  // scale bytes: a dword holds four steps of a row, fetched with the first of them (a line per row: as dear as a row's codes)
  constexpr bool SPLIT = B < 256;      // 256 threads, 2 B rows: waves 0, 1 the weights' and 2, 3 those of x, or each thread both
  const unsigned char *psw, *psx;
  {
    const int r = threadIdx.x & (B - 1);
    const int o = o0 + r < O ? o0 + r : O - 1, n = n0 + r < N ? n0 + r : N - 1;
    psw = ws + (long long)(o / kBlock) * sstride;
    psx = xs + (long long)n * sstride;
    if (SPLIT && wave >= 2) psw = psx;
  }
  const unsigned base = lds_offset(sm), sbase = lds_offset(sc);
  // load `part` of the LOADS with which a wave brings in its share of step kb
  constexpr int LOADS = 2 * L + (SPLIT ? 1 : 2);
  auto fetch = [&](int part, int kb, int into) {
    const unsigned to_w = base + into * STAGE + wave * 1024, to_s = sbase + ((kb >> 2) & 1) * 2 * B * 4 + wave * 256;
    if (part < L) load_lds16(rw, vw[part < L ? part : 0], kb * kBlock, to_w + part * 4096);
    else if (part < 2 * L) load_lds16(rx, vx[part < 2 * L ? part - L : 0], kb * kBlock, to_w + B * kBlock + (part - L) * 4096);
    else if (kb & 3) return;
    else if (part == 2 * L) load_lds4(psw + kb, to_s);
    else load_lds4(psx + kb, to_s + B * 4);
  };

  // a lane's share of a fragment: pieces g and g + 4 of its row - 32 codes, one instruction's K (fp8), or 16 of them (EXACT: half
  // a step, two instructions' K once widened)
  typedef typename Raw<EXACT>::type raw_t;
  const int swz = (g ^ (l16 & 7)) * 16, flip = (swz & 64) ? -64 : 64;
  auto raw = [&](int kb, int u, int row) {
    const unsigned char* at = sm[kb & (STAGES - 1)] + (row + l16) * kBlock + swz;
    if constexpr (EXACT) return *reinterpret_cast<const i32x4*>(at + u * flip);
    else return __builtin_shufflevector(*reinterpret_cast<const i32x4*>(at), *reinterpret_cast<const i32x4*>(at + flip), 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto ready = [&](raw_t r, unsigned s) {      // what the instruction takes; s: the row's scale byte (EXACT)
    if constexpr (EXACT) {
      const float f = scale_of(s & 255);
      return __builtin_shufflevector(__builtin_bit_cast(i32x4, widen8(r[0], r[1], f)), __builtin_bit_cast(i32x4, widen8(r[2], r[3], f)), 0, 1, 2, 3, 4, 5, 6, 7);
    } else return r;
  };
  auto scale_w = [&](int kb) { return sc[(kb >> 2) & 1][wo * TO * 16] >> ((kb & 3) * 8); };
  auto scale_x = [&](int kb, int j) { return sc[(kb >> 2) & 1][B + (wn * TN + j) * 16 + l16] >> ((kb & 3) * 8); };

  f32x4v acc[TO][TN];
#pragma unroll
  for (int i = 0; i < TO; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4v{0.f, 0.f, 0.f, 0.f};

  // What a unit (a step; EXACT: half a step) holds when it begins: the fragments of all its x rows and of the first row tile of w.
  struct Unit { i32x8 fx[TN]; raw_t aw; unsigned sw, sx[TN]; };
  const int rw0 = wo * TO * 16, rx0 = B + wn * TN * 16;
  // One unit's products, and the next unit's fragments read meanwhile (the last steps' loads repeat what is there).
  auto unit = [&](int kb, int u, const Unit& c, Unit& n) {
    const bool turn = u == U - 1;      // the last reads of this step's codes
    const int nkb = turn ? kb + 1 : kb, nu = turn ? 0 : u + 1;
    const int far = kb + STAGES < nblk ? kb + STAGES : nblk - 1;
    raw_t aw[TO], nx[TN];
    aw[0] = c.aw;
#pragma unroll
    for (int i = 0; i < TO; ++i) {
      // row tiles ahead of their use: one, and before the turn all that are left
      if (i < SYNC - 1) aw[i + 1] = raw(kb, u, rw0 + (i + 1) * 16);
      if (i == SYNC - 1) {
#pragma unroll
        for (int k = SYNC; k < TO; ++k) aw[k] = raw(kb, u, rw0 + k * 16);
      }
      if (i == SYNC && turn) {
        wait_loads<(STAGES - 2) * 2 * L>();      // step kb + 1: behind it STAGES - 2 steps are under way, of 2 L loads at least
        __syncthreads();   // and nobody reads step kb any more
      }
      if (i >= SYNC) {
        constexpr int PER = TN / (TO - SYNC);
#pragma unroll
        for (int k = (i - SYNC) * PER; k < (i - SYNC + 1) * PER; ++k) {
          nx[k] = raw(nkb, nu, rx0 + k * 16);
          n.sx[k] = turn ? scale_x(nkb, k) : c.sx[k];
        }
        if (i == TO - 1) {
          n.aw = raw(nkb, nu, rw0);
          n.sw = turn ? scale_w(nkb) : c.sw;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      const i32x8 fw = ready(aw[i], c.sw);
      __builtin_amdgcn_sched_barrier(0);
      if (B == 256) mfma_ready();
#pragma unroll
      for (int e = 0; e < U * TN; ++e) {
        const int j = e % TN;
        if constexpr (EXACT) mul_bf16<B == 256>(acc[i][j], half4(fw, e / TN), half4(c.fx[j], e / TN));
        else mul_fp8<B == 256>(acc[i][j], fw, c.fx[j], c.sw, c.sx[j]);
        // step kb + STAGES into the freed buffer: the loads one by one between the products, because a load that finds the queue full
        // holds up its wave
        if (turn && i >= SYNC) {
          constexpr int SLOTS = (TO - SYNC) * U * TN;
          const int slot = (i - SYNC) * U * TN + e;
#pragma unroll
          for (int part = slot * LOADS / SLOTS; part < (slot + 1) * LOADS / SLOTS; ++part) fetch(part, far, kb & (STAGES - 1));
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) n.fx[j] = ready(nx[j], n.sx[j]);
  };

#pragma unroll
  for (int step = 0; step < STAGES; ++step) {
#pragma unroll
    for (int part = 0; part < LOADS; ++part) fetch(part, step < nblk ? step : nblk - 1, step);
  }
  wait_loads<(STAGES - 1) * 2 * L>();
  __syncthreads();
  Unit p, q;
  p.sw = scale_w(0);
  p.aw = raw(0, 0, rw0);
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    p.sx[j] = scale_x(0, j);
    p.fx[j] = ready(raw(0, 0, rx0 + j * 16), p.sx[j]);
  }
  // two units a turn of the loop, so that what one leaves the other finds in place
  int kb = 0;
  for (; kb + 2 <= nblk * U; kb += 2) {
    unit(EXACT ? kb >> 1 : kb, 0, p, q);
    unit(EXACT ? kb >> 1 : kb + 1, U - 1, q, p);
  }
  if (kb < nblk * U) unit(kb, 0, p, q);
  wait_loads<0>();      // the last steps' repeated loads write LDS: not past the end of the workgroup
  if constexpr (B == 256) {
    mfma_settle();
#pragma unroll
    for (int i = 0; i < TO; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) asm volatile("" : "+a"(acc[i][j]));
  }

  Piece<float> bv[TO];
#pragma unroll
  for (int i = 0; i < TO; ++i) {
    if (bias) bv[i] = load_piece(bias + m * bstride, o0 + (wo * TO + i) * 16 + 4 * g, O);
    else bv[i] = Piece<float>{};
  }
  __syncthreads();
  const int n1 = n0 + wn * (B / 2), o1 = o0 + wo * (B / 2);
  store_tile<T, TO, STAGE / 2>(acc, bv, alpha, beta, &sm[0][0] + wave * (STAGE / 2), y + (((long long)blockIdx.y * (gridDim.x / (tiles_n * tiles_o)) + m) * N + n1) * O + o1, O, N - n1, O - o1);
}

// y[m][e] = sum over S slabs part[s][m][e], in order, + beta bias[m][e mod O]; e < n = N O.  sum: one m whose slabs are all the members'.
template <class T>
__global__ __launch_bounds__(256) void block8_join_kernel(const float* __restrict__ part, int S, long long n, int O,
                                                          const float* __restrict__ bias, long long bstride, float beta, T* __restrict__ y) {
  const long long m = blockIdx.y, step = n * gridDim.y;
  part += m * n;
  y += m * n;
  for (long long e = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; e < n; e += (long long)gridDim.x * 1024) {
    const int left = (int)(n - e < 4 ? n - e : 4);
    Piece<float> s = load_piece(part + e, 0, left);
    for (int i = 1; i < S; ++i) {
      const Piece<float> v = load_piece(part + i * step + e, 0, left);
#pragma unroll
      for (int k = 0; k < 4; ++k) s.e[k] += v.e[k];
    }
    int o = bias ? (int)(e % O) : 0;
    struct { T e[4]; } out;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      narrow(bias ? fmaf(beta, bias[m * bstride + o], s.e[k]) : s.e[k], out.e[k]);
      if (++o == O) o = 0;
    }
    if (left == 4) {
      __builtin_memcpy(y + e, &out, sizeof(out));
    } else {
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (k < left) y[e + k] = out.e[k];
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------
// The same product for up to sixteen rows x (fp32 / bf16 / fp16) that are not in codes yet: one launch.  It reads every weight
// code once, which is what bounds it, so nothing is staged: a wave takes 16 NT weight rows, its W-th share of the blocks of K,
// reads 32 codes per lane and row, a block ahead, and makes the codes of x for its blocks by itself (the same codes as
// hecka_block8_quantize: 32 elements per lane, the maximum over the four lanes of a row).  All products in bf16, exact.
// The W waves' sums are added in order.
// 8 x 4096 x 4096, weights from HBM: 33 us, 4.0 TB/s of codes; 1 x 4096 x 4096 8.4 us; sixteen rows, 1 x 8192 x 8192, 23 us.  A kernel that
// only reads the codes, in this order, takes 26 us of the 33 (24 in any order); the rest is work on them that the loads do not
// cover.  A start elsewhere in K for every workgroup changes nothing, nor do two blocks ahead (34 us).
// ------------------------------------------------------------------------------------------------------------------
template <class T, int NT, int W>
__global__ __launch_bounds__(64 * W) void block8_token_kernel(const T* __restrict__ x, long long xstride, int N, int K,
                                                              const unsigned char* __restrict__ w, const unsigned char* __restrict__ ws,
                                                              int O, const float* __restrict__ bias, long long bstride, float alpha, float beta,
                                                              T* __restrict__ y) {
  __shared__ f32x4v red[W][NT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
  const int nblk = row_blocks(K), sstride = scale_stride(K), o0 = blockIdx.x * 16 * NT;
  const long long m = blockIdx.y, Kp = (long long)nblk * kBlock;
  x += m * xstride + (long long)(l16 < N ? l16 : N - 1) * K;
  w += m * O * Kp;
  const unsigned char* pw[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int o = o0 + i * 16 + l16;
    pw[i] = w + (long long)(o < O ? o : O - 1) * Kp + g * 32;
  }
  ws += (m * ((O + kBlock - 1) / kBlock) + o0 / kBlock) * sstride;      // 16 NT <= 128 rows of one block
  constexpr int PX = 32 / Piece<T>::N;
  i32x4 c[NT][2];
  Piece<T> px[PX];
  int sb = 127;
  auto load = [&](int kb) {
    kb = kb < nblk ? kb : nblk - 1;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      c[i][0] = *reinterpret_cast<const i32x4*>(pw[i] + (long long)kb * kBlock);
      c[i][1] = *reinterpret_cast<const i32x4*>(pw[i] + (long long)kb * kBlock + 16);
    }
    if ((kb + 1) * kBlock <= K) {      // a whole block: no guards, whose branches for every piece cost a sixth of the time
#pragma unroll
      for (int j = 0; j < PX; ++j) __builtin_memcpy(&px[j], x + kb * kBlock + g * 32 + j * Piece<T>::N, 16);
    } else {
#pragma unroll
      for (int j = 0; j < PX; ++j) px[j] = load_piece(x, kb * kBlock + g * 32 + j * Piece<T>::N, K);
    }
    sb = ws[kb];
  };
  f32x4v acc[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i] = f32x4v{0.f, 0.f, 0.f, 0.f};
  if (wave < nblk) load(wave);
  for (int kb = wave; kb < nblk; kb += W) {
    i32x4 d[NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i) { d[i][0] = c[i][0]; d[i][1] = c[i][1]; }
    unsigned cx[8];
    const float sx = scale_of(encode<T, 32>(px, cx, [](unsigned v) {      // a block's lanes are 16 apart
      unsigned o = (unsigned)__shfl_xor((int)v, 16);
      v = o > v ? o : v;
      o = (unsigned)__shfl_xor((int)v, 32);
      return o > v ? o : v;
    })), sw = scale_of(sb);
    load(kb + W);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bf16x8 bx = widen8(cx[2 * q], cx[2 * q + 1], sx);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const bf16x8 bw = widen8(d[i][q >> 1][(q & 1) * 2], d[i][q >> 1][(q & 1) * 2 + 1], sw);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bw, bx, acc[i], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) red[wave][i][lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < NT; i += W) {
    f32x4v s = red[0][i][lane];
#pragma unroll
    for (int k = 1; k < W; ++k) s += red[k][i][lane];
    const int o = o0 + i * 16 + 4 * g;
    if (l16 < N) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (o + e < O) narrow(fmaf(alpha, s[e], bias ? beta * bias[m * bstride + o + e] : 0.f), y[(m * N + l16) * O + o + e]);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------
// dW[m][o][i] = alpha sum_n dy[m][n][o] x8[m][n][i],  db[m][o] = beta sum_n dy[m][n][o]
//
// The sum runs down the rows of both operands.  A step stages 32 rows n of each in LDS as bf16, row major, and the
// transposing LDS read hands every lane four rows of its column at a time.  x8's codes are widened times their scale (exact);
// dy is split exactly into TERMS bf16 terms by cutting (bf16 1, fp16 2, fp32 3 terms of eight significant bits), every term
// multiplies x: the products are exact and added in fp32.  db: a step's sums of dy are one more product with a column of ones, made
// by the waves that hold the first columns i; the steps' sums are added with what the additions round off (Long), so that db is as good over a
// million rows as over 64: within 1e-7 of the 2-norm at 20000 rows, 2.2e-7 in one chain, at the same time.
// LDS rows hold units of 16 columns (32 bytes); unit u of row n sits at u ^ (n & 7): a transposing read takes one unit of
// sixteen rows, eight of which lie on different banks.
// Few tiles (small O x I): the rows are cut into pieces by blockIdx.y, whose sums a second kernel adds up in order.
// 8192^3: fp32 1.34 PF (three products each), fp16 1.37, bf16 1.16 (a library's a^T b 1.06 - 1.17); 8 x 4096 rows, 2048 x 2048: fp32 607 -
// 700 us, fp16 431 us, bf16 284 us.  fp32 and fp16 are bound by the matrix instructions at the clock that the power leaves them (fp32 values
// that fit one term: 585 us); bf16 by LDS beside them: a step's 64 KB written and 128 KB read are three quarters of the time of its
// products, and the staging's vector instructions share the issue slots.
// ------------------------------------------------------------------------------------------------------------------
template <class T, int TERMS, int B, bool WHOLE>
__global__ __launch_bounds__(256) void block8_wgrad_kernel(
    const T* __restrict__ dy, const unsigned char* __restrict__ x, const unsigned char* __restrict__ xs, long long xstride,
    long long xsstride, int N, int O, int I, float alpha, float beta, float* __restrict__ dW, float* __restrict__ db,
    int tiles_o, int tiles_i, int rows_per, long long slab, long long bslab) {
  constexpr int KS = TERMS == 1 ? 64 : 32, S = KS / 32, TT = B / 32;      // rows a step, 32-row parts of it, tiles a wave and side
  constexpr int TILE = KS * B * 2, STAGE = (TERMS + 1) * TILE;
  // both buffers of dy, then both of x: whichever buffer, an LDS instruction's 16-bit offset reaches it from one address register
  __shared__ __attribute__((aligned(1024))) unsigned char sm[2 * STAGE];
  auto dy_tile = [&](int buf, int q) { return sm + (buf * TERMS + q) * TILE; };
  auto x_tile = [&](int buf) { return sm + (2 * TERMS + buf) * TILE; };
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = wave & 1, wo = wave >> 1, l16 = lane & 15, g = lane >> 4;
  int m, to, ti;
  place(blockIdx.x, gridDim.x, tiles_o, tiles_i, m, to, ti);
  const int o0 = to * B, i0 = ti * B, nblk = row_blocks(I), sstride = scale_stride(I);
  const int first = blockIdx.y * rows_per, last = first + rows_per < N ? first + rows_per : N, steps = (last - first + KS - 1) / KS;
  const long long Kp = (long long)nblk * kBlock;
  dy += ((long long)m * N + first) * O;
  x += m * xstride + first * Kp;
  xs += m * xsstride + (long long)first * sstride;

  // Staging: a thread's share of a step are DL items of dy (16-byte pieces) and XL items of x (sixteen codes).  The registers hold
  // two steps: while one is written to LDS the next is in, and the one after it takes the place of what was written.  WHOLE (dy's rows are whole aligned pieces): buffer loads, zero behind
  // the last row; columns behind the end are the next row's - they only reach outputs that do not exist.
  constexpr int P = Piece<T>::N, DPR = B / P, DL = KS * DPR / 256, XPR = B / 16, XL = KS * XPR / 256;
  constexpr int DROWS = 256 / DPR, XROWS = 256 / XPR;      // rows from one item to the next
  Piece<T> rd[2][DL];
  i32x4 rx[2][XL];
  int rs[2][XL];
  float r[4];
  const int dn = tid / DPR, dc = (tid % DPR) * P, xn = tid / XPR, xc = (tid % XPR) * 16;
  const int dv = (dn * O + dc) * (int)sizeof(T), xv = xn * (int)Kp + xc, sv = xn * sstride + ((i0 + xc) >> 7);
  // Where the loads' step begins, and the bytes that each operand has from there on (what of them a buffer descriptor can say).
  // Worked out once a step and by halves of 32 bits, for which there are scalar instructions: 64-bit comparisons go through the
  // vector unit, and a descriptor made at every load cost a fifth of the time.
  struct Source { const T* dy; const unsigned char *x, *xs; long long dy_left, x_left; int left, dy_bytes, x_bytes, xs_bytes; };
  const long long dy_step = (long long)KS * O * (int)sizeof(T), x_step = KS * Kp;
  Source at;
  auto said = [](long long bytes) {
    const int hi = (int)(bytes >> 32), lo = (int)bytes;
    return __builtin_amdgcn_readfirstlane(hi < 0 ? 0 : hi > 0 || lo < 0 ? 0x7fffffff : lo);
  };
  auto say = [&]() {
    at.dy_bytes = said(at.dy_left);
    at.x_bytes = said(at.x_left);
    at.xs_bytes = said(at.left * (long long)sstride);
  };
  auto advance = [&]() {
    at.dy += KS * (long long)O;
    at.x += x_step;
    at.xs += KS * sstride;
    at.dy_left -= dy_step;
    at.x_left -= x_step;
    at.left -= KS;
    say();
  };
  at.dy = dy + o0;
  at.x = x + i0;
  at.xs = xs;
  at.left = last - first;
  at.dy_left = ((long long)at.left * O - o0) * (long long)sizeof(T);
  at.x_left = at.left * Kp - i0;
  say();
  auto buffer = [](const void* p, int bytes) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000); };
  auto load_dy = [&](int set, int item) {
    if constexpr (WHOLE) {
      rd[set][item] = __builtin_bit_cast(Piece<T>, __builtin_amdgcn_raw_buffer_load_b128(buffer(at.dy, at.dy_bytes), dv + item * DROWS * O * (int)sizeof(T), 0, 0));
    } else {
      const int n = dn + item * DROWS;
      rd[set][item] = load_piece(n < at.left ? at.dy - o0 + (long long)n * O : dy, n < at.left ? o0 + dc : O, O);
    }
  };
  auto load_x = [&](int set, int item) {
    rx[set][item] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(buffer(at.x, at.x_bytes), xv + item * XROWS * (int)Kp, 0, 0));
    rs[set][item] = __builtin_amdgcn_raw_buffer_load_b8(buffer(at.xs, at.xs_bytes), sv + item * XROWS * sstride, 0, 0);
  };
  // the work on one item in parts of three to six instructions, few enough to pass in the shadow of a product
  constexpr int QUADS = P / 4, PERQ = TERMS == 1 ? 1 : (sizeof(T) == 2 ? 1 : 0) + 3 * (TERMS - 1) + 1;
  constexpr int PERD = TERMS == 1 ? 1 : QUADS * PERQ, PARTS = DL * PERD + 2 * XL;
  auto part = [&](int id, int buf) {
    if (id < DL * PERD) {
      const int item = id / PERD, n = dn + item * DROWS;
      unsigned char* to = dy_tile(buf, 0) + n * B * 2 + (((dc >> 4) ^ (n & 7)) * 32) + (dc & 15) * 2;
      if constexpr (TERMS == 1) {
        *reinterpret_cast<Piece<T>*>(to) = rd[buf][item];
      } else {
        const int quad = id % PERD / PERQ;
        int what = id % PERQ;
        if constexpr (sizeof(T) == 2) --what;
        if (what == -1 || (sizeof(T) == 4 && what == 0)) {
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] = widen(rd[buf][item].e[quad * 4 + e]);
        }
        if (what >= 0 && what % 3 == 0) {      // the next term of all four
          const uint2 c = make_uint2(__builtin_amdgcn_perm(__float_as_uint(r[1]), __float_as_uint(r[0]), 0x07060302),
                                     __builtin_amdgcn_perm(__float_as_uint(r[3]), __float_as_uint(r[2]), 0x07060302));
          *reinterpret_cast<uint2*>(to + what / 3 * TILE + quad * 8) = c;
        } else if (what > 0) {                 // what is left of two of them
#pragma unroll
          for (int e = what % 3 * 2 - 2; e < what % 3 * 2; ++e) r[e] -= __uint_as_float(__float_as_uint(r[e]) & 0xffff0000u);
        }
      }
      if (id % PERD == PERD - 1) load_dy(buf, item);
    } else {
      const int j = (id - DL * PERD) / 2, h = (id - DL * PERD) % 2, n = xn + j * XROWS;
      bf16x8* to = reinterpret_cast<bf16x8*>(x_tile(buf) + n * B * 2 + (((xc >> 4) ^ (n & 7)) * 32));
      to[h] = widen8(rx[buf][j][2 * h], rx[buf][j][2 * h + 1], scale_of(rs[buf][j]));
      if (h == 1) load_x(buf, j);
    }
  };

  f32x4v acc[TT][TT];
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int j = 0; j < TT; ++j) acc[i][j] = f32x4v{0.f, 0.f, 0.f, 0.f};
  // The column sums: the TT tiles of a half of this workgroup's columns o are shared out to the 2 tiles_i waves that hold them; this
  // wave has tiles mine, mine + 2 tiles_i, ... - with many tiles_i one at most.
  constexpr int OWN = TT / 2;
  const int mine = db ? ti * 2 + wi : TT;
  Long sums[OWN];      // a step's rows are added by the matrix instruction, the steps by add(): the rows may be millions
#pragma unroll
  for (int n = 0; n < OWN; ++n) sums[n] = Long{0.f, 0.f};
  const i32x4 ones = {0x3f803f80, 0x3f803f80, 0x3f803f80, 0x3f803f80};

  // fragment of 16 columns (unit u) of a tile: rows 4 g .. 4 g + 3 and 16 more down
  const int fr = (g * 4 + (l16 >> 2)) * B * 2 + (l16 & 3) * 8, sw = (g & 1) * 4 + (l16 >> 2);
  auto frag = [&](const unsigned char* tile, int u) {
    const unsigned char* from = tile + fr + ((u ^ sw) * 32);
    const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(from));
    const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(from + 16 * B * 2));
    return __builtin_bit_cast(i32x4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  // A step is GROUPS groups of TT products: part sub of its rows, tile j of columns o, term q.  At group TURN every fragment that
  // is left of the step is in registers, the next step is in the other buffer, and the barrier there is the step's only one:
  // behind it the next step's first fragments are read, and this step's buffer takes the step after that.
  constexpr int GROUPS = S * TT * TERMS, TURN = GROUPS * 3 / 4, TAIL = GROUPS - TURN, SLOTS = GROUPS * TT;
  constexpr int LEAD = 1;      // groups between a fragment's read and its use
  i32x4 fx[2][TT], fd0[LEAD];
  auto frag_d = [&](int e, int buf) {
    const int sub = e / (TT * TERMS), j = e / TERMS % TT, q = e % TERMS;
    return frag(dy_tile(buf, q) + sub * 32 * B * 2, wo * TT + j);
  };
  auto frag_s = [&](int j, int f, int buf) { return frag(dy_tile(buf, f % TERMS) + f / TERMS * 32 * B * 2, wo * TT + j); };
  auto frag_x = [&](int i, int sub, int buf) { return frag(x_tile(buf) + sub * 32 * B * 2, wi * TT + i); };
  auto step = [&](int buf, int set) {      // set: which half of fx holds the step's first part
    i32x4 fd[GROUPS], fs[S * TERMS];
#pragma unroll
    for (int e = 0; e < LEAD; ++e) fd[e] = fd0[e];
#pragma unroll
    for (int e = 0; e < GROUPS; ++e) {
      const int sub = e / (TT * TERMS), j = e / TERMS % TT, hold = S == 2 ? sub : set;
      if (e == TURN - 2) {
#pragma unroll
        for (int f = 0; f < S * TERMS; ++f) fs[f] = frag_s(mine < TT ? mine : 0, f, buf);
      }
      if (e + LEAD < TURN) fd[e + LEAD] = frag_d(e + LEAD, buf);
      if (e == TURN - LEAD) {
#pragma unroll
        for (int f = TURN; f < GROUPS; ++f) fd[f] = frag_d(f, buf);
      }
      if (S == 2 && e < TT) fx[1][e] = frag_x(e, 1, buf);
      if (e == TURN) {
        if (mine < TT) {      // before the step's buffer is given up
          f32x4v c;
          first_columns(c, ones, fs[0]);
#pragma unroll
          for (int f = 1; f < S * TERMS; ++f) add_columns(c, ones, fs[f]);
          settle_columns(c);
          add(sums[0], c[0]);
#pragma unroll
          for (int n = 1; n < OWN; ++n) {
            if (mine + n * 2 * tiles_i < TT) {
              first_columns(c, ones, frag_s(mine + n * 2 * tiles_i, 0, buf));
#pragma unroll
              for (int f = 1; f < S * TERMS; ++f) add_columns(c, ones, frag_s(mine + n * 2 * tiles_i, f, buf));
              settle_columns(c);
              add(sums[n], c[0]);
            }
          }
        }
        __syncthreads();
      }
      if (e >= TURN) {
#pragma unroll
        for (int i = (e - TURN) * TT / TAIL; i < (e - TURN + 1) * TT / TAIL; ++i) fx[S == 2 ? 0 : set ^ 1][i] = frag_x(i, 0, buf ^ 1);
        if (e >= GROUPS - LEAD) fd0[e - (GROUPS - LEAD)] = frag_d(e - (GROUPS - LEAD), buf ^ 1);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (B == 256) mfma_ready();
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        mul_bf16<B == 256>(acc[i][j], fx[hold][i], fd[e]);
        // from turn to turn: the parts of the next step but one, evenly
        const int slot = (e < TURN ? e + TAIL : e - TURN) * TT + i;
#pragma unroll
        for (int id = slot * PARTS / SLOTS; id < (slot + 1) * PARTS / SLOTS; ++id) {
          if (id == 0) advance();
          part(id, e < TURN ? buf ^ 1 : buf);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

#pragma unroll
  for (int set = 0; set < 2; ++set) {
#pragma unroll
    for (int i = 0; i < DL; ++i) load_dy(set, i);
#pragma unroll
    for (int i = 0; i < XL; ++i) load_x(set, i);
    advance();
  }
#pragma unroll
  for (int id = 0; id < PARTS; ++id) part(id, 0);
  advance();
#pragma unroll
  for (int id = 0; id < TAIL * TT * PARTS / SLOTS; ++id) part(id, 1);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < TT; ++i) fx[0][i] = frag_x(i, 0, 0);
#pragma unroll
  for (int e = 0; e < LEAD; ++e) fd0[e] = frag_d(e, 0);
  // two steps a turn of the loop, so that buffers and fragments have fixed places (a step behind the last one adds zeros)
  for (int k = 0; k < steps; k += 2) {
    step(0, 0);
    step(1, 1);
  }
  __syncthreads();
  if constexpr (B == 256) {
    mfma_settle();
#pragma unroll
    for (int i = 0; i < TT; ++i)
#pragma unroll
      for (int j = 0; j < TT; ++j) asm volatile("" : "+a"(acc[i][j]));
  }

  if (g == 0) {
    float* to_db = db + blockIdx.y * bslab + (long long)m * O;
#pragma unroll
    for (int n = 0; n < OWN; ++n) {
      const int t = mine + n * 2 * tiles_i, o = o0 + (wo * TT + t) * 16 + l16;
      if (t < TT && o < O) to_db[o] = beta * value(sums[n]);
    }
  }
  const Piece<float> none[TT] = {};
  const int o1 = o0 + wo * (B / 2), i1 = i0 + wi * (B / 2);
  store_tile<float, TT, STAGE / 2>(acc, none, alpha, 0.f, sm + wave * (STAGE / 2), dW + blockIdx.y * slab + ((long long)m * O + o1) * I + i1,
                                   I, O - o1, I - i1);
}

// out[e] = sum over S slabs, in order, what its additions round off included; two arrays in one launch: n of out, then n2 of out2, whose slabs stand behind out's
__global__ __launch_bounds__(256) void block8_slabs_kernel(const float* __restrict__ part, int S, long long n, float* __restrict__ out,
                                                           long long n2, float* __restrict__ out2) {
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < n + n2; e += (long long)gridDim.x * 256) {
    const bool second = e >= n;
    const float* p = second ? part + S * n + (e - n) : part + e;
    const long long step = second ? n2 : n;
    Long s{p[0], 0.f};
    for (int i = 1; i < S; ++i) add(s, p[i * step]);
    (second ? out2[e - n] : out[e]) = value(s);
  }
}

static int cdiv(int a, int b) { return (a + b - 1) / b; }
static constexpr int kLinearFill = 256, kLinearLeast = 8;
// rounds of the chip's 256 CUs that M matrices of R x C take in tiles of 256 x 256
static long long large_rounds(int M, int R, int C) { return ((long long)M * cdiv(R, 256) * cdiv(C, 256) + 255) / 256; }

// 256 x 256 outputs a workgroup, one a CU, or 128 x 128, two a CU: a round of 256 large ones takes as long as about 512 small ones of fp8
// products and 900 of widened codes.  Where small ones leave half of the chip idle the blocks of K are shared out, eight at least to
// each, their sums joined by a second launch.  Measured (fp8 / widened codes), large tiles against small: 1 x 2048 x 8192 x 4096, 256
// large or 1024 small ones, 65 / 111 against 111 / 126 us; 1 x 1024 x 8192 x 4096, 128 or 512, 56 / 104 against 63 / 68; 5 x 1000 x 1000 x
// 1000, 80 or 320, 24 / 38 against 21 / 23; 8 x 300 x 4096 x 4096, 256 or 768, 60 / 115 against 80 / 103; 10 x 300 x 4096 x 784, 320 or 960,
// 44 / 68 against 38 / 36.  Shares: 1 x 64 x 8192 x 8192 48 / 73 us whole, 24 / 30 us in four shares, 31 / 30 us in eight; 1 x 64 x 1024 x 8192 41 / 73 us whole, 15 /
// 19 us in eight; 1 x 512 x 4096 x 4096 28 / 45 us whole, 27 / 35 us in two, 38 / 35 us in four; shares of four blocks: 1 x 256 x 4096 x
// 4096 32 us against 22.
struct LinearPlan { int tile, splits, share; };
static LinearPlan linear_plan(int M, int N, int O, int nblk, bool exact) {
  LinearPlan p{256, 1, (nblk + 3) & ~3};
  const long long tiles = (long long)M * cdiv(N, 128) * cdiv(O, 128), s = kLinearFill / tiles;
  if (large_rounds(M, N, O) * (exact ? 900 : 512) <= tiles) return p;
  p.tile = 128;
  if (s > 1) {
    const int most = nblk / kLinearLeast > 1 ? nblk / kLinearLeast : 1;
    p.splits = (int)(s < most ? s : most);
    p.share = (cdiv(nblk, p.splits) + 3) & ~3;
    p.splits = cdiv(nblk, p.share);
  }
  return p;
}
static size_t linear_workspace(const LinearPlan& p, int M, int N, int O, int y_members) {
  return p.splits > 1 || y_members < M ? (size_t)p.splits * M * N * O * sizeof(float) : 0;
}

template <class T, bool EXACT>
static int linear_run(const LinearPlan& p, const void* x, const void* xs, long long xstride, long long xsstride, const void* w,
                      const void* ws, int M, int N, int O, int nblk, const float* bias, long long bstride, float alpha, float beta,
                      void* y, int y_members, float* slabs, hipStream_t st) {
#define HECKA_LINEAR(TO, B, STAGES, BIAS, OUT) \
  block8_linear_kernel<TO, EXACT, B, STAGES><<<dim3((unsigned)(M * cdiv(N, B) * cdiv(O, B)), p.splits), 256, 0, st>>>( \
      (const unsigned char*)x, (const unsigned char*)xs, xstride, xsstride, (const unsigned char*)w, (const unsigned char*)ws, N, O, \
      nblk, p.share, BIAS, bstride, alpha, beta, OUT, cdiv(N, B), cdiv(O, B))
  // Long sums of fp8 products in 128 x 128 tiles that have a CU to themselves: three steps ahead (1 x 1024 x 4096 x 4096 28 us, one ahead 32;
  // 1 x 64 x 8192 x 8192 22 us, 24); with widened codes and in short sums the start costs what that saves (5 x 300 x 1200 x 784 fp8 10.2 us, 10.0;
  // widened 14.9, 14.2).
  constexpr int FAR = EXACT ? 2 : 4;
  const bool far = FAR > 2 && p.share >= 16 && (long long)M * cdiv(N, 128) * cdiv(O, 128) * p.splits <= 256;
  if (p.splits > 1 || y_members < M) {
    if (p.tile == 256) HECKA_LINEAR(float, 256, 2, nullptr, slabs);
    else if (far) HECKA_LINEAR(float, 128, FAR, nullptr, slabs);
    else HECKA_LINEAR(float, 128, 2, nullptr, slabs);
    const long long n = (long long)N * O, blocks = (n + 1023) / 1024;
    block8_join_kernel<T><<<dim3((unsigned)(blocks < 2048 ? blocks : 2048), y_members), 256, 0, st>>>(
        slabs, y_members < M ? p.splits * M : p.splits, n, O, bias, bstride, beta, (T*)y);
  } else if (p.tile == 256) HECKA_LINEAR(T, 256, 2, bias, (T*)y);
  else if (far) HECKA_LINEAR(T, 128, FAR, bias, (T*)y);
  else HECKA_LINEAR(T, 128, 2, bias, (T*)y);
#undef HECKA_LINEAR
  return check_launch("block8_linear");
}

template <class T>
static int token_run(const void* x, long long xstride, int M, int N, int K, const void* w, const void* ws, int O,
                     const float* bias, long long bstride, float alpha, float beta, void* y, hipStream_t st) {
#define HECKA_TOKEN(NT, W) \
  block8_token_kernel<T, NT, W><<<dim3(cdiv(O, 16 * NT), M), 64 * W, 0, st>>>((const T*)x, xstride, N, K, (const unsigned char*)w, \
                                                                           (const unsigned char*)ws, O, bias, bstride, alpha, beta, (T*)y)
  // Sixteen weight rows a wave where that makes few waves, 32 otherwise (a workgroup reads all of x, and makes its codes); K is
  // shared out to as many waves as fill the chip, two blocks each at least where there are many.  Measured (bf16, weights from HBM):
  // 8 x 4096 x 4096, one row, 33 us with 32 rows x 4 waves, 34 us with 32 x 8, 37 us with 16 x 4; sixteen rows 43, 45 and 56 us; 1 x 8192 x
  // 8192, sixteen rows, 23 us with 32 x 8, 30 us with 16 x 8.  With guarded loads: 1 x 4096 x 4096 11 us with 16 x 8, 17 us with 32 x 4;
  // 1 x 1000 x 8192 12 us with 16 x 16, 23 us with 16 x 4.
  const long long rows16 = (long long)M * cdiv(O, 16);
  const int nblk = row_blocks(K);
  if (rows16 >= 512) {
    if (rows16 >= 1024 || nblk < 16) HECKA_TOKEN(2, 4);
    else HECKA_TOKEN(2, 8);
  } else if (rows16 >= 128) {
    if (nblk < 16) HECKA_TOKEN(1, 4);
    else HECKA_TOKEN(1, 8);
  } else if (nblk <= 4) {
    HECKA_TOKEN(1, 4);
  } else if (nblk < 32) {
    HECKA_TOKEN(1, 8);
  } else {
    HECKA_TOKEN(1, 16);
  }
#undef HECKA_TOKEN
  return check_launch("block8_token");
}

struct WgradPlan { int tile, to, ti, splits, rows; };
static WgradPlan wgrad_plan(int M, int N, int O, int I, bool whole) {
  // 256 x 256 tiles, one workgroup per CU, where dy's rows are whole 16-byte pieces (guarded loads, for which 256 x 256 leaves no
  // registers, otherwise) and a round of them does the work of 700 of 128 x 128, two per CU; where small ones are too few the rows in pieces
  // of 256 at least.  Measured (bf16 / fp32): 4 x 2000 x 2000 x 2000, 256 large or 1024 small tiles, 82 / 177 against 107 / 208 us; 3 x 4096 x 2048
  // x 2048, 192 or 768, 132 / 302 against 153 / 312; ragged rows of dy, 4 x 2000 x 2001 x 2000, 324 / 259; large ones cut into pieces, 2 x 1024 x 2048 x 2048, 53 / 75 against 32 / 55 us, 1 x
  // 65536 x 256 x 512, 72 / 92 against 56 / 79.
  WgradPlan p{256, cdiv(O, 256), cdiv(I, 256), 1, cdiv(N, 64) * 64};
  const long long tiles = (long long)M * cdiv(O, 128) * cdiv(I, 128), s = tiles >= 512 ? 1 : 512 / tiles;
  if (whole && large_rounds(M, O, I) * 700 <= tiles) return p;
  p.tile = 128;
  p.to = cdiv(O, 128);
  p.ti = cdiv(I, 128);
  const int most = cdiv(N, 256);
  p.splits = (int)(s < most ? s : most);
  p.rows = cdiv(cdiv(N, p.splits), 64) * 64;
  p.splits = cdiv(N, p.rows);
  return p;
}

template <class T, int TERMS>
static int wgrad_run(const void* dy, const void* x, const void* xs, long long xstride, long long xsstride, int M, int N, int O,
                     int I, float alpha, float beta, float* dW, float* db, float* ws, hipStream_t st) {
  const bool whole = O % Piece<T>::N == 0 && aligned16(dy);
  const WgradPlan p = wgrad_plan(M, N, O, I, whole);
  const long long nw = (long long)M * O * I, nb = (long long)M * O;
  const bool cut = p.splits > 1;
#define HECKA_WGRAD(B, WHOLE) \
  block8_wgrad_kernel<T, TERMS, B, WHOLE><<<dim3((unsigned)(M * p.to * p.ti), p.splits), 256, 0, st>>>( \
      (const T*)dy, (const unsigned char*)x, (const unsigned char*)xs, xstride, xsstride, N, O, I, alpha, beta, cut ? ws : dW, \
      db ? (cut ? ws + p.splits * nw : db) : nullptr, p.to, p.ti, p.rows, nw, nb)
  if (p.tile == 256) HECKA_WGRAD(256, true);
  else if (whole) HECKA_WGRAD(128, true);
  else HECKA_WGRAD(128, false);
#undef HECKA_WGRAD
  if (cut) {
    const long long n2 = db ? nb : 0, blocks = (nw + n2 + 255) / 256;
    block8_slabs_kernel<<<dim3((unsigned)(blocks < 2048 ? blocks : 2048)), 256, 0, st>>>(ws, p.splits, nw, dW, n2, db);
  }
  return check_launch("block8_wgrad");
}

// whether `dtype` asks for the fp8 instruction, and that taken off it (left there, and so no known type, with fp32, whose products are exact)
static bool take_fp8(int& dtype) {
  if (dtype != (HECKA_DT_BF16 | HECKA_BLOCK8_FP8) && dtype != (HECKA_DT_F16 | HECKA_BLOCK8_FP8)) return false;
  dtype &= ~HECKA_BLOCK8_FP8;
  return true;
}
static bool bad_type(int dtype) { return dtype != HECKA_DT_F32 && dtype != HECKA_DT_BF16 && dtype != HECKA_DT_F16; }
// sizes for which every index that the kernels keep in 32 bits fits: sizes below 2^22, tiles below 2^31
static bool bad_sizes(int M, int N, int O, int I) {
  const int most = 1 << 22;
  return M <= 0 || N <= 0 || O <= 0 || I <= 0 || M > 65535 || N > most || O > most || I > most ||
         (long long)M * cdiv(N, 128) * cdiv(O, 128) > 0x7fffffffLL || (long long)M * cdiv(O, 128) * cdiv(I, 128) > 0x7fffffffLL;
}

}  // namespace hecka

using namespace hecka;

extern "C" {

size_t hecka_block8_linear_workspace_bytes(int M, int N, int O, int I, int y_members, int dtype) {
  const bool fp8 = take_fp8(dtype);
  if (bad_type(dtype) || bad_sizes(M, N, O, I) || (y_members != M && y_members != 1)) return 0;
  return linear_workspace(linear_plan(M, N, O, row_blocks(I), !fp8), M, N, O, y_members);
}

int hecka_block8_linear(const void* x, const void* xscales, int x_members, const void* w, const void* wscales, int M, int N, int O,
                        int I, const float* bias, long long bstride, float alpha, float beta, void* y, int dtype, int y_members,
                        void* ws, size_t ws_bytes, void* stream) {
  const bool fp8 = take_fp8(dtype);
  if (bad_type(dtype)) return fail(HECKA_EINVAL, "block8_linear: unknown dtype%s");
  if (bad_sizes(M, N, O, I)) return fail(HECKA_EINVAL, "%sblock8_linear: bad size (N = %lld, O = %lld)", "", N, O);
  if (x_members != M && x_members != 1) return fail(HECKA_EINVAL, "%sblock8_linear: codes of %lld members for %lld", "", x_members, M);
  if (y_members != M && (y_members != 1 || bias)) return fail(HECKA_EINVAL, "%sblock8_linear: %lld result members for %lld (their sum takes no bias)", "", y_members, M);
  if (!x || !xscales || !w || !wscales || !y) return fail(HECKA_EINVAL, "block8_linear: null pointer%s");
  if (!aligned16(x) || !aligned16(w) || (reinterpret_cast<uintptr_t>(xscales) & 3) || (reinterpret_cast<uintptr_t>(wscales) & 3))
    return fail(HECKA_EINVAL, "block8_linear: codes need 16-byte alignment, scales 4-byte%s");
  const int nblk = row_blocks(I);
  const LinearPlan p = linear_plan(M, N, O, nblk, !fp8);
  if ((ws ? ws_bytes : 0) < linear_workspace(p, M, N, O, y_members))
    return fail(HECKA_EWORKSPACE, "%sblock8_linear: workspace too small (%lld bytes given)", "", (long long)ws_bytes);
  clear_error();
  const long long xst = x_members == 1 ? 0 : (long long)N * nblk * kBlock, sst = x_members == 1 ? 0 : (long long)N * scale_stride(I);
  hipStream_t st = (hipStream_t)stream;
#define HECKA_RUN(T, EXACT) \
  linear_run<T, EXACT>(p, x, xscales, xst, sst, w, wscales, M, N, O, nblk, bias, bstride, alpha, beta, y, y_members, (float*)ws, st)
  if (fp8) return dtype == HECKA_DT_BF16 ? HECKA_RUN(Bf16, false) : HECKA_RUN(F16, false);
  return dtype == HECKA_DT_F32 ? HECKA_RUN(float, true) : dtype == HECKA_DT_BF16 ? HECKA_RUN(Bf16, true) : HECKA_RUN(F16, true);
#undef HECKA_RUN
}

int hecka_block8_linear_token(const void* x, int dtype, int x_members, const void* w, const void* wscales, int M, int N, int O, int I,
                              const float* bias, long long bstride, float alpha, float beta, void* y, void* stream) {
  if (bad_type(dtype)) return fail(HECKA_EINVAL, "block8_linear_token: unknown dtype%s");
  if (bad_sizes(M, N, O, I) || N > 16) return fail(HECKA_EINVAL, "%sblock8_linear_token: bad size (N = %lld, O = %lld)", "", N, O);
  if (x_members != M && x_members != 1) return fail(HECKA_EINVAL, "%sblock8_linear_token: rows of %lld members for %lld", "", x_members, M);
  if (!x || !w || !wscales || !y) return fail(HECKA_EINVAL, "block8_linear_token: null pointer%s");
  if (!aligned16(w)) return fail(HECKA_EINVAL, "block8_linear_token: codes need 16-byte alignment%s");
  clear_error();
  const long long xst = x_members == 1 ? 0 : (long long)N * I;
  hipStream_t st = (hipStream_t)stream;
  return dtype == HECKA_DT_F32 ? token_run<float>(x, xst, M, N, I, w, wscales, O, bias, bstride, alpha, beta, y, st)
         : dtype == HECKA_DT_BF16 ? token_run<Bf16>(x, xst, M, N, I, w, wscales, O, bias, bstride, alpha, beta, y, st)
                                  : token_run<F16>(x, xst, M, N, I, w, wscales, O, bias, bstride, alpha, beta, y, st);
}

size_t hecka_block8_wgrad_workspace_bytes(int M, int N, int O, int I) {
  if (bad_sizes(M, N, O, I)) return 0;
  size_t most = 0;
  for (bool whole : {false, true}) {
    const WgradPlan p = wgrad_plan(M, N, O, I, whole);
    const size_t need = p.splits > 1 ? (size_t)p.splits * M * O * ((size_t)I + 1) * sizeof(float) : 0;
    most = need > most ? need : most;
  }
  return most;
}

int hecka_block8_wgrad(const void* dy, int dtype, const void* x, const void* xscales, int x_members, int M, int N, int O, int I,
                       float alpha, float beta, float* dW, float* db, void* ws, size_t ws_bytes, void* stream) {
  if (bad_type(dtype)) return fail(HECKA_EINVAL, "block8_wgrad: unknown dtype%s");
  if (bad_sizes(M, N, O, I)) return fail(HECKA_EINVAL, "%sblock8_wgrad: bad size (N = %lld, O = %lld)", "", N, O);
  if (x_members != M && x_members != 1) return fail(HECKA_EINVAL, "%sblock8_wgrad: codes of %lld members for %lld", "", x_members, M);
  if (!dy || !x || !xscales || !dW) return fail(HECKA_EINVAL, "block8_wgrad: null pointer%s");
  if (!aligned16(x)) return fail(HECKA_EINVAL, "block8_wgrad: codes need 16-byte alignment%s");
  if ((ws ? ws_bytes : 0) < hecka_block8_wgrad_workspace_bytes(M, N, O, I))
    return fail(HECKA_EWORKSPACE, "%sblock8_wgrad: workspace too small (%lld bytes given)", "", (long long)ws_bytes);
  clear_error();
  const long long xst = x_members == 1 ? 0 : (long long)N * row_blocks(I) * kBlock, sst = x_members == 1 ? 0 : (long long)N * scale_stride(I);
  hipStream_t st = (hipStream_t)stream;
  return dtype == HECKA_DT_F32 ? wgrad_run<float, 3>(dy, x, xscales, xst, sst, M, N, O, I, alpha, beta, dW, db, (float*)ws, st)
         : dtype == HECKA_DT_BF16 ? wgrad_run<Bf16, 1>(dy, x, xscales, xst, sst, M, N, O, I, alpha, beta, dW, db, (float*)ws, st)
                                  : wgrad_run<F16, 2>(dy, x, xscales, xst, sst, M, N, O, I, alpha, beta, dW, db, (float*)ws, st);
}

// A layer's training step in two calls, each the launches above in their order: a small layer's time is its caller's.
namespace {
// the parts of a buffer, each at a multiple of 256 bytes
struct Parts {
  char* base;
  size_t used;
  void* take(size_t bytes, bool wanted = true) {
    if (!wanted) return nullptr;
    void* p = base + used;
    used += (bytes + 255) & ~(size_t)255;
    return p;
  }
};
struct Kept { void *xc, *xs, *tc, *ts; };      // rows x; weights transposed
struct Sizes {
  size_t xc, xs, wc, ws, tc, ts, dc, ds;
  Sizes(int M, int xm, int N, int O, int I) {
    xc = (size_t)xm * N * row_blocks(I) * kBlock;
    xs = (size_t)xm * N * scale_stride(I);
    wc = (size_t)M * O * row_blocks(I) * kBlock;
    ws = (size_t)M * row_blocks(O) * scale_stride(I);
    tc = (size_t)M * I * row_blocks(O) * kBlock;
    ts = (size_t)M * row_blocks(I) * scale_stride(O);
    dc = (size_t)M * N * row_blocks(O) * kBlock;
    ds = (size_t)M * N * scale_stride(O);
  }
};
Kept kept_parts(const Sizes& z, Parts& p, bool need_dx, bool need_dw) {
  Kept k;
  k.xc = p.take(z.xc, need_dw);
  k.xs = p.take(z.xs, need_dw);
  k.tc = p.take(z.tc, need_dx);
  k.ts = p.take(z.ts, need_dx);
  return k;
}
}  // namespace

size_t hecka_block8_train_bytes(int what, int M, int x_members, int N, int O, int I, int dtype, int need_dx, int need_dw) {
  const int products = dtype;      // with the choice of the instruction
  take_fp8(dtype);
  if (bad_type(dtype) || bad_sizes(M, N, O, I) || (x_members != M && x_members != 1)) return 0;
  const Sizes z(M, x_members, N, O, I);
  Parts p{nullptr, 0};
  if (what == 0) {
    kept_parts(z, p, need_dx, need_dw);
  } else if (what == 1) {
    p.take(z.xc, !need_dw);
    p.take(z.xs, !need_dw);
    p.take(z.wc);
    p.take(z.ws);
    p.take(hecka_block8_linear_workspace_bytes(M, N, O, I, M, products));
  } else {
    p.take(z.dc, need_dx);
    p.take(z.ds, need_dx);
    p.take(hecka_block8_linear_workspace_bytes(M, N, I, O, x_members, products), need_dx);
    p.take(hecka_block8_wgrad_workspace_bytes(M, N, O, I), need_dw);
  }
  return p.used;
}

int hecka_block8_train_fwd(const void* x, int dtype, int x_members, long long ld, const void* W, int wdtype, long long mstride, int M, int N,
                           int O, int I, const float* bias, long long bstride, float alpha, float beta, int need_dx, int need_dw, void* y,
                           void* kept, size_t kept_bytes, void* ws, size_t ws_bytes, void* stream) {
  const int products = dtype;
  take_fp8(dtype);
  if (bad_type(dtype) || bad_type(wdtype)) return fail(HECKA_EINVAL, "block8_train_fwd: unknown dtype%s");
  if (bad_sizes(M, N, O, I)) return fail(HECKA_EINVAL, "%sblock8_train_fwd: bad size (N = %lld, O = %lld)", "", N, O);
  if (x_members != M && x_members != 1) return fail(HECKA_EINVAL, "%sblock8_train_fwd: rows of %lld members for %lld", "", x_members, M);
  const size_t most = hecka_block8_train_bytes(0, M, x_members, N, O, I, dtype, need_dx, need_dw);
  if ((kept ? kept_bytes : 0) < most || (ws ? ws_bytes : 0) < hecka_block8_train_bytes(1, M, x_members, N, O, I, products, need_dx, need_dw))
    return fail(HECKA_EWORKSPACE, "%sblock8_train_fwd: workspace too small (%lld bytes given)", "", (long long)ws_bytes);
  const Sizes z(M, x_members, N, O, I);
  Parts pk{(char*)kept, 0}, pw{(char*)ws, 0};
  Kept k = kept_parts(z, pk, need_dx, need_dw);
  if (!need_dw) {
    k.xc = pw.take(z.xc);
    k.xs = pw.take(z.xs);
  }
  void *wc = pw.take(z.wc), *wsc = pw.take(z.ws);
  const size_t need = hecka_block8_linear_workspace_bytes(M, N, O, I, M, products);
  int rc = hecka_block8_quantize(x, dtype, (long long)x_members * N, I, ld, HECKA_ACT_NONE, k.xc, k.xs, nullptr, stream);
  if (!rc) rc = hecka_block8_weight(W, wdtype, M, O, I, mstride, wc, wsc, k.tc, k.ts, stream);
  if (!rc)
    rc = hecka_block8_linear(k.xc, k.xs, x_members, wc, wsc, M, N, O, I, bias, bstride, alpha, beta, y, products, M, need ? pw.take(need) : nullptr, need, stream);
  return rc;
}

int hecka_block8_train_bwd(const void* dy, int dtype, int x_members, int M, int N, int O, int I, float alpha, float beta, int need_dx,
                           int need_dw, const void* kept, size_t kept_bytes, void* dx, float* dW, float* db, void* ws, size_t ws_bytes,
                           void* stream) {
  const int products = dtype;
  take_fp8(dtype);
  if (bad_type(dtype)) return fail(HECKA_EINVAL, "block8_train_bwd: unknown dtype%s");
  if (bad_sizes(M, N, O, I)) return fail(HECKA_EINVAL, "%sblock8_train_bwd: bad size (N = %lld, O = %lld)", "", N, O);
  if (x_members != M && x_members != 1) return fail(HECKA_EINVAL, "%sblock8_train_bwd: rows of %lld members for %lld", "", x_members, M);
  if (!dy || (dx && !need_dx) || (dW && !need_dw) || (db && !dW)) return fail(HECKA_EINVAL, "block8_train_bwd: null pointer, or a gradient whose codes were not kept%s");
  if ((kept ? kept_bytes : 0) < hecka_block8_train_bytes(0, M, x_members, N, O, I, dtype, need_dx, need_dw) ||
      (ws ? ws_bytes : 0) < hecka_block8_train_bytes(2, M, x_members, N, O, I, products, dx != nullptr, dW != nullptr))
    return fail(HECKA_EWORKSPACE, "%sblock8_train_bwd: workspace too small (%lld bytes given)", "", (long long)ws_bytes);
  const Sizes z(M, x_members, N, O, I);
  Parts pk{(char*)const_cast<void*>(kept), 0}, pw{(char*)ws, 0};
  const Kept k = kept_parts(z, pk, need_dx, need_dw);
  int rc = 0;
  if (dx) {
    void *dc = pw.take(z.dc), *ds = pw.take(z.ds);
    const size_t need = hecka_block8_linear_workspace_bytes(M, N, I, O, x_members, products);
    void* slabs = need ? pw.take(need) : nullptr;
    rc = hecka_block8_quantize(dy, dtype, (long long)M * N, O, O, HECKA_ACT_NONE, dc, ds, nullptr, stream);
    if (!rc) rc = hecka_block8_linear(dc, ds, M, k.tc, k.ts, M, N, I, O, nullptr, 0, alpha, 0.f, dx, products, x_members, slabs, need, stream);
  }
  if (dW && !rc) {
    const size_t need = hecka_block8_wgrad_workspace_bytes(M, N, O, I);
    rc = hecka_block8_wgrad(dy, dtype, k.xc, k.xs, x_members, M, N, O, I, alpha, beta, dW, db, need ? pw.take(need) : nullptr, need, stream);
  }
  return rc;
}

}  // extern "C"
