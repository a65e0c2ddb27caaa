// orthogonalize.hip — the nearest semi-orthogonal matrix to an update, by Newton-Schulz products.
//
//   X = G / (|G|_F + eps), turned so that its m rows are the shorter side;
//   steps times:  A = X X^T,  X <- (a I + b A + c A A) X     (an odd polynomial of the singular values)
//
// All factors are polynomials of one symmetric matrix, so they commute, and a stage of a few steps needs X
// only at its ends:
//   A = X X^T;  each step:  Q = a I + b A + c A A,  P <- Q P,  A <- (Q A) Q;   X <- P X
// The m x m products are symmetric: only the tiles on and above the diagonal are computed (the epilogue
// writes both halves) where they fill the chip. A stage of r steps costs 3 m^2 n + (4 r - 3) m^3 operations
// instead of r (3 m^2 n + m^3): five steps as 3 + 2 6 m^2 n + 14 m^3 instead of 15 m^2 n + 5 m^3. X is kept both
// ways round, as [m, n] (operand of A) and as [n, m] (operand of P X): all operands of gemm_nt.h are
// contiguous along k.
//
// Rounding. Between products a matrix is held as two fp16 planes (23 bits) at a power-of-two scale that
// keeps it in range (the host bounds the singular values step by step). One plane would be off by 0.15 %
// on Gaussian matrices and by 1-4 % where a few strong directions hide the rest. A stage squares the
// ratio of the singular values once more for each step behind its first: five steps of nine float32 matrices
// (48 x 80 to 1024 x 1536, ratios 4 to 1000) measured 0.7 - 1.4e-6 off as single steps, 3.2e-6 at ratio 1000;
// 1.3 - 2.7e-6 as 2 + 2 + 1, 1.7 - 3.8e-6 as 3 + 2; plain float32 products 1.0 - 3.3e-6. float32 takes single
// steps; the 16-bit types, whose results round to 2^-11 and 2^-8, stages of 3. 16-bit inputs are exact in one
// plane, so the first stage reads one plane of them. (One plane of each operand in the last P X of bf16 results
// would save 80 us of 1150 at 6 x 1024 x 4096 and be 0.03 - 0.3 % off, against the 0.17 % of the result's own
// rounding.)
#include <limits.h>
#include <math.h>

#include "gemm_nt.h"

namespace smq {
namespace ortho {
using namespace gemm;

constexpr int kParts = 256;

__host__ __device__ constexpr int round32(int v) { return (v + 31) & ~31; }

// ---- the norm -----------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void square_sum_kernel(const T* x, int64_t ld, int64_t batch_stride,
                                                         int rows, int cols, double* part) {
  constexpr int V = 16 / sizeof(T);
  typedef typename Loose<T, V>::type vec;
  const T* p = x + blockIdx.y * batch_stride;
  const int whole = cols / V * V;
  double s = 0.0;
  for (int r = blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += gridDim.x * 4) {
    const T* q = p + (int64_t)r * ld;
    for (int k = (threadIdx.x & 63) * V; k < whole; k += 64 * V) {
      const vec v = *reinterpret_cast<const vec*>(q + k);
#pragma unroll
      for (int i = 0; i < V; i++) s += (double)v[i] * (double)v[i];
    }
    for (int k = whole + (threadIdx.x & 63); k < cols; k += 64) s += (double)q[k] * (double)q[k];
  }
  s = wave_sum(s);
  __shared__ double w[4];
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.y * gridDim.x + blockIdx.x] = (w[0] + w[1]) + (w[2] + w[3]);
}
// Per matrix: pow2 = 2^e that brings the norm to [2^13, 2^14) (so the fp16 planes hold it: an element of
// size norm / 2^27 still has full precision), rest = 1 / ((norm + eps) 2^e) and its square, which
// the products with X take as a factor.
__global__ __launch_bounds__(64) void norm_kernel(const double* part, int n, double eps, float* pow2,
                                                  float* rest, float* rest2) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 64) s += part[blockIdx.x * n + i];
  s = wave_sum(s);
  if (threadIdx.x == 0) {
    const double norm = sqrt(s);
    int e = 0;
    if (norm > 0.0 && norm < 1e300) {
      frexp(norm, &e);
      e = 14 - e;
      e = e > 120 ? 120 : e < -120 ? -120 : e;
    }
    // a matrix of zeros stays one, however small eps (rest2 would leave fp32's range below 1e-19)
    const double r = norm == 0.0 && eps > 0.0 ? 0.0 : 1.0 / ((norm + eps) * ldexp(1.0, e));
    pow2[blockIdx.x] = ldexpf(1.0f, e);
    rest[blockIdx.x] = (float)r;
    rest2[blockIdx.x] = (float)(r * r);
  }
}

// ---- one workgroup a matrix -----------------------------------------------------------------------
// m <= 64: the products of a stage are too small to fill the chip and each launch costs more than it
// computes, so one workgroup keeps A, Q and P of a matrix in LDS (as operands: two planes in the
// tiles of gemm_nt.h) and registers (as fp32). With `whole`, where n is short or the stack deep, it also
// forms A from X, applies P and goes through all stages; else it takes A from, and leaves P in, global
// memory. 64 x 64 float32, 5 steps: 52 us a call (110 as 18 launches of gemm_nt.h). For m up to 128, on 16
// waves, the same kernel was no faster than those launches.
//
// The workgroups of a stack do not wait for one another, and the buffers of X change their format between the
// stages: a matrix keeps to its own part of them, at one stride (x[k].batch, xt[k].batch) whatever the format.
struct SmallStep {
  float qa, qb, qc;  // coefficients a, b, c
  float sa, sq, sw, sp;  // 2^e of A, Q, W = Q A and P as operands
};
struct SmallArgs {
  SmallStep step[8];
  int steps;         // of this launch (a stage, or all)
  int stage;         // steps of a stage
  int m, n, batch;
  Mat x[2], xt[2];   // whole: X and X^T; the stages alternate (batch: room for a matrix in every format)
  Mat y;             // whole: the result
  int turned;
  int fmt_x0, fmt_xt0;
  const float* rest;
  const float* rest2;
  float ex[8];       // 2^-ex of X at each stage's start
  float ey[8];       // 2^ey of X at each stage's end
  Mat gram, p;       // not whole
  float gram_scale, p_scale;  // 2^-ea, 2^ep
};

#if defined(__HIP_DEVICE_COMPILE__)
struct Small {
  static constexpr int DIM = 64;
  // one 32 x 32 block a wave
  static constexpr int kWn = DIM / 32, kWaves = kWn * kWn;
  static constexpr int TM = 1, TN = 1;
  static constexpr int kTiles = DIM / 32;  // k tiles a region holds
  static constexpr int kTileHalves = DIM * 64;
  static constexpr int kLoads = DIM / 8 / kWaves;  // loads a wave issues per k tile
  typedef f32x16 Block[TM][TN];
  int lane, wave, wm, wn;

  __device__ __forceinline__ void clear(Block& v) const {
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) v[i][j][r] = 0.0f;
  }
  // k tile t of `rows` rows from row0 of a matrix -> region + slot (rows past the end: the last one)
  __device__ __forceinline__ void fetch(const Mat& a, int64_t batch, int row0, int rows, int t,
                                        _Float16* region, int slot) const {
    const int have = rows - row0 < DIM ? rows - row0 : DIM;
    const char* p = reinterpret_cast<const char*>(a.p) + 2 * (batch * a.batch + (int64_t)row0 * a.ld);
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)((have - 1) * a.ld * 2 + (t + 1) * 128), 0x00027000);
    const int chunk = ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
      const int r = (i * kWaves + wave) * 8 + (lane >> 3);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (lds_void*)(region + slot * kTileHalves + (i * kWaves + wave) * 512), 16,
          (int)((r < have ? r : have - 1) * a.ld * 2) + chunk, t * 128, 0, 0);
    }
  }
  template <int T>
  __device__ __forceinline__ void read(const _Float16* tile, int base, int s, f16x8 (&f)[T]) const {
    const int at = ((s * 2 + (lane >> 5)) ^ (lane & 7)) * 8;
#pragma unroll
    for (int i = 0; i < T; i++)
      f[i] = *reinterpret_cast<const f16x8*>(tile + (base * T * 32 + i * 32 + (lane & 31)) * 64 + at);
  }
  // acc[i][j] += rows of `u` (runs of a lane) x rows of `v` (one a lane)
  __device__ __forceinline__ void mma(const f16x8 (&u)[TN], const f16x8 (&v)[TM], Block& acc) const {
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++) acc[i][j] = Frag<_Float16>::mma(u[j], v[i], acc[i][j]);
  }
  // acc += (rows of a: one a lane) x (rows of b: runs of 4) over `tiles` k tiles. A wave's block is
  // (ba, bb).
  __device__ __forceinline__ void product(const _Float16* a, const _Float16* b, int tiles, bool two, int ba,
                                          int bb, Block& acc, Block& low) const {
#pragma unroll 1
    for (int t = 0; t < tiles; t++) {
      const _Float16 *ta = a + t * kTileHalves, *tb = b + t * kTileHalves;
      if (two) {
#pragma unroll
        for (int s = 0; s < 2; s++) {
          f16x8 ah[TM], al[TM], bh[TN], bl[TN];
          read(ta, ba, s, ah);
          read(tb, bb, s, bh);
          read(ta, ba, s + 2, al);
          read(tb, bb, s + 2, bl);
          mma(bh, ah, acc);
          mma(bl, ah, low);
          mma(bh, al, low);
        }
      } else {
#pragma unroll
        for (int s = 0; s < 4; s++) {
          f16x8 fa[TM], fb[TN];
          read(ta, ba, s, fa);
          read(tb, bb, s, fb);
          mma(fb, fa, acc);
        }
      }
    }
  }
  __device__ __forceinline__ void sum(Block& acc, const Block& low, float scale) const {
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[i][j][r] = (acc[i][j][r] + low[i][j][r]) * scale;
  }
  // f(i, j, r, row, col): the four values from register r on are columns col..col+3 of a row
  template <typename F>
  __device__ __forceinline__ void each(int br, int bc, F f) const {
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
          f(i, j, r, br * TM * 32 + i * 32 + (lane & 31), bc * TN * 32 + j * 32 + 2 * r + 4 * (lane >> 5));
  }
  // A symmetric matrix as an operand of two planes: v * scale, columns from m on are zeros.
  __device__ __forceinline__ void put(_Float16* region, const Block& v, float scale, int m) const {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    each(wm, wn, [&](int i, int j, int r, int row, int col) {
      h4 hi, lo;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float x = col + k < m ? v[i][j][r + k] * scale : 0.0f;
        hi[k] = (_Float16)x;
        lo[k] = (_Float16)(x - (float)hi[k]);
      }
      const int x7 = row & 7, c = (col & 31) >> 3;
      _Float16* t = region + (col >> 5) * kTileHalves + row * 64 + (col & 7);
      *reinterpret_cast<h4*>(t + (c ^ x7) * 8) = hi;
      *reinterpret_cast<h4*>(t + ((c + 4) ^ x7) * 8) = lo;
    });
  }
};
#endif

template <bool WHOLE>
__global__ __launch_bounds__(256, 2) void small_kernel(SmallArgs A) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef Small S;
  constexpr int DIM = S::DIM;
  typedef typename S::Block Block;
  __shared__ __attribute__((aligned(1024))) _Float16 r0[DIM * DIM * 2];
  __shared__ __attribute__((aligned(1024))) _Float16 r1[DIM * DIM * 2];
  S s;
  s.lane = threadIdx.x & 63;
  s.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  s.wm = s.wave / S::kWn, s.wn = s.wave % S::kWn;
  const int64_t batch = blockIdx.x;
  const int m = A.m, n = A.n, km = (m + 31) / 32;
  constexpr int kAll = S::kTiles * S::kLoads;  // loads of a whole region
  Block a, p, acc, low;
  for (int done = 0, stage = 0; done < A.steps; stage++) {
    const int r = A.steps - done < A.stage ? A.steps - done : A.stage;
    const bool end = done + r == A.steps;
    // ---- A = X X^T
    if constexpr (WHOLE) {
      Mat X = A.x[stage & 1];
      if (stage == 0) X.fmt = A.fmt_x0;
      else X.fmt = kSplit, X.ld = (int64_t)round32(n) * 2;
      const bool two = X.fmt == kSplit;
      const int kt = two ? (n + 31) / 32 : (n + 63) / 64;
      auto load = [&](int first, _Float16* region) {
#pragma unroll
        for (int t = 0; t < S::kTiles; t++)
          s.fetch(X, batch, 0, m, first + t < kt ? first + t : kt - 1, region, t);
      };
      s.clear(acc);
      s.clear(low);
      load(0, r0);
#pragma unroll 1
      for (int t = 0; t < kt; t += 2 * S::kTiles) {
        auto half = [&](int first, _Float16* here, _Float16* there) {
          load(first + S::kTiles, there);
          asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(kAll) : "memory");
          if (first < kt)
            s.product(here, here, kt - first < S::kTiles ? kt - first : S::kTiles, two, s.wm, s.wn, acc, low);
          asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        };
        half(t, r0, r1);
        half(t + S::kTiles, r1, r0);
      }
      asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
      const float f = A.ex[stage] * A.ex[stage] * (stage == 0 ? A.rest2[batch] : 1.0f);
#pragma unroll
      for (int i = 0; i < S::TM; i++)
#pragma unroll
        for (int j = 0; j < S::TN; j++)
#pragma unroll
          for (int q = 0; q < 16; q++) a[i][j][q] = (acc[i][j][q] + low[i][j][q]) * f;
    } else {
      s.each(s.wm, s.wn, [&](int i, int j, int q, int row, int col) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (row < m && col < A.gram.pad) v = load4(A.gram, batch, row, col);
        a[i][j][q] = v.x * A.gram_scale, a[i][j][q + 1] = v.y * A.gram_scale;
        a[i][j][q + 2] = v.z * A.gram_scale, a[i][j][q + 3] = v.w * A.gram_scale;
      });
    }
    s.put(r0, a, A.step[done].sa, m);
    __syncthreads();
    // ---- P of the stage
#pragma unroll 1
    for (int i = 0; i < r; i++) {
      const SmallStep& k = A.step[done + i];
      const float ia = 1.0f / k.sa, iq = 1.0f / k.sq;
      s.clear(acc);
      s.clear(low);
      s.product(r0, r0, km, true, s.wm, s.wn, acc, low);
      s.sum(acc, low, ia * ia);
      s.each(s.wm, s.wn, [&](int x, int y, int q, int row, int col) {
#pragma unroll
        for (int e = 0; e < 4; e++)
          acc[x][y][q + e] = (row == col + e ? k.qa : 0.0f) + k.qb * a[x][y][q + e] + k.qc * acc[x][y][q + e];
      });
      s.put(r1, acc, k.sq, m);
      if (i == 0) {
#pragma unroll
        for (int x = 0; x < S::TM; x++)
#pragma unroll
          for (int y = 0; y < S::TN; y++) p[x][y] = acc[x][y];
      }
      __syncthreads();
      if (i + 1 < r) {
        s.clear(acc);
        s.clear(low);
        s.product(r1, r0, km, true, s.wm, s.wn, acc, low);  // W = Q A
        s.sum(acc, low, iq * ia);
        __syncthreads();
        s.put(r0, acc, k.sw, m);
        __syncthreads();
        s.clear(a);
        s.clear(low);
        s.product(r0, r1, km, true, s.wm, s.wn, a, low);  // A <- W Q
        s.sum(a, low, iq / k.sw);
        __syncthreads();
      }
      if (i > 0) {  // P <- Q P
        if (i + 1 == r) __syncthreads();
        s.put(r0, p, A.step[done + i - 1].sp, m);
        __syncthreads();
        s.clear(p);
        s.clear(low);
        s.product(r1, r0, km, true, s.wm, s.wn, p, low);
        s.sum(p, low, iq / A.step[done + i - 1].sp);
        __syncthreads();
      }
      if (i + 1 < r) {
        s.put(r0, a, A.step[done + i + 1].sa, m);
        __syncthreads();
      }
    }
    // ---- X <- P X
    if constexpr (!WHOLE) {
      s.each(s.wm, s.wn, [&](int i, int j, int q, int row, int col) {
        if (row < m) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; e++) w[e] = p[i][j][q + e] * A.p_scale;
          store_n<4>(A.p, batch, row, col, m, w);
        }
      });
    } else {
      Mat XT = A.xt[stage & 1];
      XT.fmt = stage == 0 ? A.fmt_xt0 : kSplit;
      const bool two = XT.fmt == kSplit;
      if (stage > 0) XT.ld = (int64_t)round32(m) * 2;
      const float sp = A.step[done + r - 1].sp;
      const float f = A.ex[stage] * (stage == 0 ? A.rest[batch] : 1.0f) * A.ey[stage] / sp;
      __syncthreads();
      s.put(r0, p, sp, m);
      // the next stage's matrices
      Mat X2 = A.x[(stage + 1) & 1], XT2 = A.xt[(stage + 1) & 1];
      X2.fmt = kSplit, X2.ld = (int64_t)round32(n) * 2, X2.pad = round32(n);
      XT2.fmt = kSplit, XT2.ld = (int64_t)round32(m) * 2, XT2.pad = round32(m);
#pragma unroll 1
      for (int c0 = 0; c0 < n; c0 += DIM) {
        for (int t = 0; t < km; t++) s.fetch(XT, batch, c0, n, t, r1, t);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (!end || !A.turned) {
          s.clear(acc);
          s.clear(low);
          s.product(r0, r1, km, two, s.wm, s.wn, acc, low);
          s.sum(acc, low, f);
          s.each(s.wm, s.wn, [&](int i, int j, int q, int row, int col) {
            const float w[4] = {acc[i][j][q], acc[i][j][q + 1], acc[i][j][q + 2], acc[i][j][q + 3]};
            if (row < m) store_n<4>(end ? A.y : X2, batch, row, c0 + col, n, w);
          });
        }
        if (!end || A.turned) {  // the same product the other way round: runs along m
          s.clear(acc);
          s.clear(low);
          s.product(r1, r0, km, two, s.wm, s.wn, acc, low);
          s.sum(acc, low, f);
          s.each(s.wm, s.wn, [&](int i, int j, int q, int row, int col) {
            const float w[4] = {acc[i][j][q], acc[i][j][q + 1], acc[i][j][q + 2], acc[i][j][q + 3]};
            if (c0 + row < n) store_n<4>(end ? A.y : XT2, batch, c0 + row, col, m, w);
          });
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      }
      // this workgroup reads what it wrote
      asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    }
    done += r;
  }
#endif
}

// ---- host ---------------------------------------------------------------------------------------
struct Plan {
  int64_t batch, m, n;
  bool turned;
  int dtype, steps;
  double a, b, c;
};

// Steps of a stage: one for float32 (rounding, above) and for calls bound by their launches (under 2^20
// elements, not much longer than wide): a single step is three launches, three in a stage are eleven.
int stage_of(const Plan& p) {
  const bool launches = p.m > 64 && p.batch * p.m * p.n < (1 << 20) && p.n <= 4 * p.m;
  return p.dtype == SMQ_DTYPE_F32 || launches ? 1 : 3;
}

// Largest |a s + b s^3 + c s^5| over 0 <= s <= top.
double grown(const Plan& p, double top) {
  auto at = [&](double s) { return fabs(s * (p.a + s * s * (p.b + s * s * p.c))); };
  double best = at(top);
  auto look = [&](double q) {  // q: the square of a stationary point
    if (q > 0.0 && q < top * top) best = fmax(best, at(sqrt(q)));
  };
  if (p.c != 0.0) {
    const double d = 9.0 * p.b * p.b - 20.0 * p.a * p.c;
    if (d >= 0.0) {
      look((-3.0 * p.b + sqrt(d)) / (10.0 * p.c));
      look((-3.0 * p.b - sqrt(d)) / (10.0 * p.c));
    }
  } else if (p.b != 0.0) {
    look(-p.a / (3.0 * p.b));
  }
  return best;
}
// Exponent e with bound * 2^e <= 2^15, with some room for rounding.
int exponent_for(double bound) {
  int e;
  frexp(fmax(bound, 1e-30) * 1.02, &e);
  const int k = 15 - e;
  return k > 60 ? 60 : k;
}

struct Arena {
  char* base;
  size_t used = 0;
  explicit Arena(void* p) : base(reinterpret_cast<char*>(p)) {}
  template <typename T>
  T* take(size_t count) {
    used = (used + 255) & ~size_t(255);
    T* p = reinterpret_cast<T*>(base + used);
    used += count * sizeof(T);
    return p;
  }
};

struct Buffers {  // (those a call does not use are NULL)
  _Float16 *x[2], *xt[2], *gram[2], *q[2], *p[2], *w;
  float* part;  // shares of a product split over k
};

// One product, split over k or not.
void product(bool split, const Operand& A, const Operand& B, int kt, int batch, StoreEpi e,
             const Buffers& w, bool run, size_t* need, hipStream_t st) {
  // A symmetric product whose whole grid of small tiles fits the chip at once is not halved: the mirrored
  // store costs 2 us, the other half nothing. (Two planes in 256 x 256 tiles round more, gemm_nt.h, and
  // are no faster at these lengths.)
  if (e.tri && batch * tile_count(A.rows, B.rows, kT64, 0) <= 256) e.tri = 0, e.ot.fmt = kNone;
  const Shared plan = plan_product(A.rows, B.rows, kt, batch, e.tri, true, !split);
  const int tile = plan.tile, shares = plan.shares;
  const int64_t ld = round_up(B.rows, 4), per = (int64_t)A.rows * ld;
  if (shares > 1 && need) {
    const size_t floats = (size_t)shares * batch * per;
    if (floats > *need) *need = floats;
  }
  if (!run) return;
  StoreEpi d = e;
  if (shares > 1) {
    d = {1.0f, 0.0f, nullptr, {}, {w.part, ld, per, kF32, 0}, {}, 0, batch * per, 0.0f};
  }
  if (split) launch<_Float16, true>(tile, A, B, kt, batch, e.tri, shares, d, st);
  else launch<_Float16, false>(tile, A, B, kt, batch, e.tri, shares, d, st);
  if (shares > 1)
    launch_split_sum(w.part, ld, batch * per, shares, per, A.rows, B.rows, batch,
                     e.ot.fmt != kNone ? 1 : 0, e, st);
}

template <typename T>
void first_layout(const Plan& p, const T* g, int64_t ld, int64_t stride, double eps, double* part,
                  float* pow2, float* rest, float* rest2, const Mat& x, const Mat& xt, hipStream_t st) {
  const int rows = (int)(p.turned ? p.n : p.m), cols = (int)(p.turned ? p.m : p.n);
  const int grid = rows < 4 * kParts ? (rows + 3) / 4 : kParts;
  hipLaunchKernelGGL(square_sum_kernel<T>, dim3(grid, (unsigned)p.batch), dim3(256), 0, st, g, ld, stride,
                     rows, cols, part);
  hipLaunchKernelGGL(norm_kernel, dim3((unsigned)p.batch), dim3(64), 0, st, part, grid, eps, pow2, rest,
                     rest2);
  launch_layout(g, ld, stride, rows, cols, (int)p.batch, {}, {}, pow2, nullptr, 0, p.turned ? xt : x,
                p.turned ? x : xt, st);
}

// The products of a call of either format, walked without a launch: the floats their shares need.
size_t share_floats(const Plan& p) {
  size_t need = 0;
  const Operand X = {nullptr, 0, 0, (int)p.m}, XT = {nullptr, 0, 0, (int)p.n};
  const int km = operand_kt(p.m, true), batch = (int)p.batch;
  StoreEpi e = {};
  e.tri = 1;
  product(true, X, X, km, batch, e, {}, false, &need, nullptr);
  for (int s = 0; s < 2; s++) product(s == 0, X, X, operand_kt(p.n, s == 0), batch, e, {}, false, &need, nullptr);
  e.tri = 0;
  for (int s = 0; s < 2; s++) product(s == 0, X, XT, km, batch, e, {}, false, &need, nullptr);
  return need;
}

// The small kernel's steps first .. first + count of a call; *top is the bound of X's singular values
// before and after them. `stage`: where P starts anew.
void fill_steps(const Plan& p, int count, int stage, double* top, SmallArgs* a) {
  double most = 1.0;
  for (int i = 0; i < count; i++) {
    if (i % stage == 0) most = 1.0;
    const double t = *top * *top, lift = fabs(p.a) + fabs(p.b) * t + fabs(p.c) * t * t;
    most *= lift;
    a->step[i] = {(float)p.a, (float)p.b, (float)p.c, (float)ldexp(1.0, exponent_for(t)),
                  (float)ldexp(1.0, exponent_for(lift)), (float)ldexp(1.0, exponent_for(lift * t)),
                  (float)ldexp(1.0, exponent_for(most))};
    *top = grown(p, *top);
  }
}
template <bool WHOLE>
void launch_small(const SmallArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(small_kernel<WHOLE>, dim3(a.batch), dim3(256), 0, st, a);
}

// Lays the workspace out and, when `run`, enqueues the call. Returns the bytes used.
size_t enqueue(const Plan& p, const void* g, int64_t ld, int64_t stride, void* y, double eps, void* ws,
               bool run, hipStream_t st) {
  Arena a(ws);
  const int64_t bt = p.batch, m = p.m, n = p.n;
  const int batch = (int)bt;
  // room for the largest format; two of each X (a stage reads one and writes the other)
  const int64_t ldn = 2 * round_up(n, 64) + 64, ldm = 2 * round_up(m, 64) + 64;
  double* part = a.take<double>((size_t)(bt * kParts));
  float* pow2 = a.take<float>((size_t)bt);
  float* rest = a.take<float>((size_t)bt);
  float* rest2 = a.take<float>((size_t)bt);
  Buffers w = {};
  const bool small = m <= 64;
  const int longest = stage_of(p);
  auto square = [&]() { return a.take<_Float16>((size_t)(bt * m * ldm)); };
  for (int k = 0; k < 2; k++) {
    w.x[k] = a.take<_Float16>((size_t)(bt * m * ldn));
    w.xt[k] = a.take<_Float16>((size_t)(bt * n * ldm));
  }
  w.gram[0] = square();
  if (small) {
    w.p[0] = square();
  } else {
    w.q[0] = square();
    if (longest > 1) w.gram[1] = square(), w.q[1] = square(), w.p[0] = square(), w.p[1] = square(), w.w = square();
  }
  w.part = a.take<float>(share_floats(p));
  if (!run) return a.used;

  // (a matrix's place in its buffer is the same in every format, small_kernel)
  auto mat = [&](_Float16* q, int64_t cols, int64_t rows, int fmt) {
    const bool two = fmt != kF16;
    return Mat{q, operand_ld(cols, two), rows * (cols == n ? ldn : ldm), fmt, operand_pad(cols, two)};
  };
  auto op = [](const Mat& q, int64_t rows) { return Operand{q.p, q.ld, q.batch, (int)rows}; };
  const Mat none = {nullptr, 0, 0, kNone, 0};
  const int out = p.dtype == SMQ_DTYPE_F32 ? kF32 : p.dtype == SMQ_DTYPE_F16 ? kF16 : kBF16;
  Mat X = mat(w.x[0], n, m, p.dtype == SMQ_DTYPE_F32 ? kSplit : kF16);
  Mat XT = mat(w.xt[0], m, n, p.dtype == SMQ_DTYPE_F32 ? kSplit : kDup);
  if (p.dtype == SMQ_DTYPE_F32)
    first_layout(p, (const float*)g, ld, stride, eps, part, pow2, rest, rest2, X, XT, st);
  else if (p.dtype == SMQ_DTYPE_F16)
    first_layout(p, (const _Float16*)g, ld, stride, eps, part, pow2, rest, rest2, X, XT, st);
  else
    first_layout(p, (const __bf16*)g, ld, stride, eps, part, pow2, rest, rest2, X, XT, st);

  double top = 1.0;  // bound of X's singular values
  // One workgroup a matrix also for the products with X: where they are short, or the stack fills the chip.
  if (small && p.steps <= 8 && (n <= 256 || batch >= 128)) {
    SmallArgs sa = {};
    sa.steps = p.steps, sa.stage = longest, sa.m = (int)m, sa.n = (int)n, sa.batch = batch;
    sa.x[0] = X, sa.xt[0] = XT, sa.x[1].p = w.x[1], sa.xt[1].p = w.xt[1];
    sa.x[1].batch = X.batch, sa.xt[1].batch = XT.batch;
    sa.fmt_x0 = X.fmt, sa.fmt_xt0 = XT.fmt, sa.turned = p.turned ? 1 : 0;
    sa.y = {y, p.turned ? m : n, m * n, out, 0};
    sa.rest = rest, sa.rest2 = rest2;
    fill_steps(p, p.steps, longest, &top, &sa);
    double bound = 1.0;
    for (int s = 0, done = 0; done < p.steps; s++) {
      sa.ex[s] = s == 0 ? 1.0f : 1.0f / sa.ey[s - 1];
      for (int i = 0; i < longest && done < p.steps; i++, done++) bound = grown(p, bound);
      sa.ey[s] = done == p.steps ? 1.0f : (float)ldexp(1.0, exponent_for(bound));
    }
    launch_small<true>(sa, st);
    return a.used;
  }
  int ex = 0;  // X is held times 2^ex (in the first stage the factors `rest` say it)
  const int km = operand_kt(m, true);
  for (int done = 0, stage = 0; done < p.steps; stage++) {
    const int r = p.steps - done < longest ? p.steps - done : longest;
    done += r;
    const bool end = done == p.steps;
    // A = X X^T
    int ea = exponent_for(top * top);
    Mat A = mat(w.gram[0], m, m, kSplit);
    StoreEpi e = {(float)ldexp(1.0, ea - 2 * ex), 0.0f, stage ? nullptr : rest2, none, A, A, 1, 0, 0.0f};
    product(X.fmt == kSplit, op(X, m), op(X, m), operand_kt(n, X.fmt == kSplit), batch, e, w, true, nullptr, st);
    Mat P = none;
    int ep = 0;
    if (small) {
      SmallArgs sa = {};
      sa.steps = sa.stage = r, sa.m = (int)m, sa.batch = batch;
      sa.gram = A, sa.gram_scale = (float)ldexp(1.0, -ea);
      fill_steps(p, r, r, &top, &sa);
      P = mat(w.p[0], m, m, kSplit);
      sa.p = P, sa.p_scale = sa.step[r - 1].sp;
      frexpf(sa.p_scale, &ep);
      ep -= 1;
      launch_small<false>(sa, st);
    }
    double most = 1.0;  // bound of P
    for (int i = 0; i < r && !small; i++) {
      const double t = top * top, lift = fabs(p.a) + fabs(p.b) * t + fabs(p.c) * t * t;
      const int eq = exponent_for(lift);
      // Q = a I + b A + c A A
      const Mat Q = mat(w.q[i & 1], m, m, kSplit);
      e = {(float)ldexp(p.c, eq - 2 * ea), (float)ldexp(p.b, eq - ea), nullptr, A, Q, Q, 1, 0,
           (float)ldexp(p.a, eq)};
      product(true, op(A, m), op(A, m), km, batch, e, w, true, nullptr, st);
      most *= lift;
      if (i == 0) {
        P = Q, ep = eq;
      } else {
        // P <- Q P
        const int en = exponent_for(most);
        const Mat P2 = mat(w.p[i & 1], m, m, kSplit);
        e = {(float)ldexp(1.0, en - eq - ep), 0.0f, nullptr, none, P2, P2, 1, 0, 0.0f};
        product(true, op(Q, m), op(P, m), km, batch, e, w, true, nullptr, st);
        P = P2, ep = en;
      }
      const double next = grown(p, top);
      if (i + 1 < r) {
        // A <- (Q A) Q
        const int ew = exponent_for(lift * t), en = exponent_for(next * next);
        const Mat W = mat(w.w, m, m, kSplit), A2 = mat(w.gram[(i + 1) & 1], m, m, kSplit);
        e = {(float)ldexp(1.0, ew - eq - ea), 0.0f, nullptr, none, W, W, 1, 0, 0.0f};
        product(true, op(Q, m), op(A, m), km, batch, e, w, true, nullptr, st);
        e = {(float)ldexp(1.0, en - ew - eq), 0.0f, nullptr, none, A2, A2, 1, 0, 0.0f};
        product(true, op(W, m), op(Q, m), km, batch, e, w, true, nullptr, st);
        A = A2, ea = en;
      }
      top = next;
    }
    // X <- P X
    const int ey = end ? 0 : exponent_for(top);
    Mat X2, XT2;
    if (!end) {
      X2 = mat(w.x[(stage + 1) & 1], n, m, kSplit);
      XT2 = mat(w.xt[(stage + 1) & 1], m, n, kSplit);
    } else {
      const Mat Y = {y, p.turned ? m : n, m * n, out, 0};
      X2 = p.turned ? none : Y, XT2 = p.turned ? Y : none;
    }
    e = {(float)ldexp(1.0, ey - ep - ex), 0.0f, stage ? nullptr : rest, none, X2, XT2, 0, 0, 0.0f};
    product(XT.fmt == kSplit, op(P, m), op(XT, n), km, batch, e, w, true, nullptr, st);
    X = X2, XT = XT2, ex = ey;
  }
  return a.used;
}

constexpr double kMostGrowth = 256.0;
constexpr int64_t kStack = 65535;  // matrices of one walk through the launches (a grid's limit)
// f(plan of a part of the stack, its first matrix): deeper stacks go part by part through one workspace.
template <typename F>
void by_stacks(const Plan& all, F f) {
  for (int64_t b = 0; b < all.batch; b += kStack) {
    Plan p = all;
    p.batch = all.batch - b < kStack ? all.batch - b : kStack;
    f(p, b);
  }
}

int plan(const char* who, int dtype, int64_t batch, int64_t rows, int64_t cols, int steps,
         const double* coefficients, Plan* p) {
  if (dtype != SMQ_DTYPE_F32 && dtype != SMQ_DTYPE_F16 && dtype != SMQ_DTYPE_BF16) {
    set_error("%s: dtype %d is not one of SMQ_DTYPE_F32/F16/BF16", who, dtype);
    return SMQ_ERR_INVALID;
  }
  if (batch < 1 || batch > INT_MAX || rows < 1 || cols < 1 || rows > (1 << 20) || cols > (1 << 20)) {
    set_error("%s: needs 1 <= batch < 2^31 and 1 <= rows, cols <= 2^20, got %lld, %lld, %lld", who,
              (long long)batch, (long long)rows, (long long)cols);
    return SMQ_ERR_INVALID;
  }
  if (steps < 1 || steps > 64 || !coefficients) {
    set_error("%s: needs 1 <= steps <= 64 and three coefficients", who);
    return SMQ_ERR_INVALID;
  }
  *p = {batch, rows < cols ? rows : cols, rows < cols ? cols : rows, rows > cols, dtype, steps,
        coefficients[0], coefficients[1], coefficients[2]};
  double top = 1.0;
  for (int i = 0; i < steps; i++) {
    top = grown(*p, top);
    if (!(top <= kMostGrowth)) {
      set_error("%s: coefficients %g, %g, %g let a singular value of at most 1 grow past %g in %d steps",
                who, p->a, p->b, p->c, kMostGrowth, i + 1);
      return SMQ_ERR_INVALID;
    }
  }
  return SMQ_OK;
}
}  // namespace ortho
}  // namespace smq

using namespace smq;
using namespace smq::ortho;

extern "C" {

size_t smq_orthogonalize_workspace_bytes(int dtype, int64_t batch, int64_t rows, int64_t cols) {
  const double c[3] = {1.0, 0.0, 0.0};
  Plan p;
  if (plan("orthogonalize_workspace_bytes", dtype, batch, rows, cols, 1, c, &p) != SMQ_OK) return 0;
  size_t most = 0;
  by_stacks(p, [&](const Plan& part, int64_t) {
    if (part.batch < kStack || most == 0) {  // (full parts are alike)
      const size_t need = enqueue(part, nullptr, 0, 0, nullptr, 0.0, nullptr, false, nullptr);
      most = need > most ? need : most;
    }
  });
  return most + 256;
}

int smq_orthogonalize(const void* x, int64_t ld, int64_t batch_stride, int dtype, void* y,
                      int64_t batch, int64_t rows, int64_t cols, int steps,
                      const double* coefficients, double eps, void* workspace,
                      size_t workspace_bytes, void* stream) {
  Plan p;
  const int rc = plan("orthogonalize", dtype, batch, rows, cols, steps, coefficients, &p);
  if (rc != SMQ_OK) return rc;
  if (!x || !y || ld < cols || !(eps >= 0.0)) {
    set_error("orthogonalize: x and y must be non-NULL, the row pitch at least cols, eps >= 0");
    return SMQ_ERR_INVALID;
  }
  const size_t need = smq_orthogonalize_workspace_bytes(dtype, batch, rows, cols);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)) {
    set_error("orthogonalize: workspace: need %zu bytes on a 16-byte boundary, got %zu", need, workspace_bytes);
    return SMQ_ERR_WORKSPACE;
  }
  const int64_t size = dtype == SMQ_DTYPE_F32 ? 4 : 2;
  by_stacks(p, [&](const Plan& part, int64_t b) {
    enqueue(part, reinterpret_cast<const char*>(x) + b * batch_stride * size, ld, batch_stride,
            reinterpret_cast<char*>(y) + b * rows * cols * size, eps, workspace, true,
            reinterpret_cast<hipStream_t>(stream));
  });
  return check_launch("orthogonalize");
}

}  // extern "C"
