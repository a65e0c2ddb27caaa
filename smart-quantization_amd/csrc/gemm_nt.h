// gemm_nt.h — the matrix product the training-step operators share: C[m, n] = sum_k A[m, k] B[n, k]
// with both operands contiguous along k, fp16 or bf16 MFMA, fp32 accumulation.
//
// Operand formats (16-bit elements, row pitch ld, rows 16-byte aligned, k padded with zeros):
//   one plane   k padded to 64: a k tile is 64 consecutive elements of a row;
//   two planes  an fp32 value x is held as hi = fp16(x), lo = fp16(x - hi) (23 significant bits, the
//               caller scales by a power of two so that nothing overflows), k padded to 32, and each
//               32 columns stored as [32 hi | 32 lo]: a k tile is again 64 consecutive elements.
//               Three products hi*hi + hi*lo + lo*hi per k step; the dropped lo*lo is below 2^-24 of
//               the largest product. An fp32-class product at a third of the fp16 rate, where the
//               fp32 MFMA runs at a sixteenth.
//   float32     as it is (Raw32), k padded to 32: the fp32 instructions, a sixteenth of the fp16 rate but no
//               pass that makes planes; ld counts 16-bit units here too.
//   twice       one plane in the layout of two, [32 x | 32 x] (kDup): against an operand of two planes
//               the one-plane product gives (hi + lo) x.
//
// Kernel: a workgroup of WM x WN waves computes a BM x BN tile; a k tile of both operands (128 bytes
// a row) goes from global memory straight into one of two LDS buffers (buffer_load ... lds, 16 bytes
// a lane), while the other is read. Rows are 128 bytes apart, so the 16-byte chunk c of row r is kept
// at chunk c ^ (r & 7): the 8 rows a quarter wave reads with one ds_read_b128 lie in 8 different bank
// groups. The waves hold their fragments of the next 16 columns in registers while the MFMAs of the
// current ones run, across the barrier between k tiles too. The four LDS buffers are separate
// variables: the compiler then knows that a read of one does not wait for the loads into another.
//
// What bounds it: a wave's 128 x 64 part reads (128 + 64) * 16 * 2 bytes of LDS per 128 x 64 x 16
// product, 75 % of the LDS rate at the full MFMA rate; 64 x 64 parts need 100 %. Measured (fp16,
// random data): 8192 x 8192 x 4096 at 1100 TFLOP/s with 256 x 256 tiles and 950 with 128 x 128 (1040
// and 900 before the reads were spread between the MFMAs); two planes, which read LDS half as often
// per MFMA, 4096^3 at 430 (1290 of single products). A large library product reaches 1250-1300 here.
// Four waves of 128 x 128 parts measured 930, bands of 8 and 16 tile rows 1-3 % less than 4.
#pragma once

#include "smq_common.h"

namespace smq {
void set_error(const char* fmt, ...);
int check_launch(const char* what);

namespace gemm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;

template <typename H> struct Frag;
template <> struct Frag<__bf16> {
  typedef bf16x8 type;
  static __device__ __forceinline__ f32x16 mma(type a, type b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Frag<_Float16> {
  typedef f16x8 type;
  static __device__ __forceinline__ f32x16 mma(type a, type b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// float32 as it is, on the fp32 matrix instructions: a row's k tile is 32 floats, the same 128 bytes. A
// lane's 16 bytes are 4 columns, of which the four instructions take one each: which columns meet in
// one instruction does not matter as long as both operands agree.
struct Raw32 {
  uint16_t half;
};
typedef float f32x4v __attribute__((ext_vector_type(4)));
template <> struct Frag<Raw32> {
  typedef f32x4v type;
  static __device__ __forceinline__ f32x16 mma(type a, type b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

struct Operand {
  const void* p;
  int64_t ld;     // elements between rows
  int64_t batch;  // elements between matrices of a batch
  int rows;
  // of A, where the host knows only the most there can be (device memory, NULL: what the host says):
  const int* live = nullptr;   // rows
  const int* depth = nullptr;  // columns
};

// Output / source formats of a matrix an epilogue reads or writes.
enum Fmt : int { kNone = 0, kF32 = 1, kF16 = 2, kBF16 = 3, kSplit = 4, kDup = 5 };
struct Mat {
  void* p;
  int64_t ld;
  int64_t batch;
  int fmt;
  int pad;  // columns in [columns, pad) are written as zeros
};

__device__ __forceinline__ int64_t split_at(int64_t c) { return ((c >> 5) << 6) + (c & 31); }

// Four consecutive columns c..c+3 (c a multiple of 4) of row r.
__device__ __forceinline__ float4 load4(const Mat& s, int64_t b, int64_t r, int64_t c) {
  typedef _Float16 h4 __attribute__((ext_vector_type(4)));
  typedef __bf16 b4 __attribute__((ext_vector_type(4)));
  const int64_t row = b * s.batch + r * s.ld;
  if (s.fmt == kSplit) {
    const _Float16* p = reinterpret_cast<const _Float16*>(s.p) + row + split_at(c);
    const h4 hi = *reinterpret_cast<const h4*>(p), lo = *reinterpret_cast<const h4*>(p + 32);
    return make_float4((float)hi.x + (float)lo.x, (float)hi.y + (float)lo.y,
                       (float)hi.z + (float)lo.z, (float)hi.w + (float)lo.w);
  }
  if (s.fmt == kDup) {
    const h4 v = *reinterpret_cast<const h4*>(reinterpret_cast<const _Float16*>(s.p) + row + split_at(c));
    return make_float4((float)v.x, (float)v.y, (float)v.z, (float)v.w);
  }
  if (s.fmt == kF16) {
    const h4 v = *reinterpret_cast<const h4*>(reinterpret_cast<const _Float16*>(s.p) + row + c);
    return make_float4((float)v.x, (float)v.y, (float)v.z, (float)v.w);
  }
  if (s.fmt == kBF16) {
    const b4 v = *reinterpret_cast<const b4*>(reinterpret_cast<const __bf16*>(s.p) + row + c);
    return make_float4((float)v.x, (float)v.y, (float)v.z, (float)v.w);
  }
  return *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(s.p) + row + c);
}

__device__ __forceinline__ void store1(const Mat& d, int64_t row, int64_t c, float v) {
  if (d.fmt == kSplit) {
    _Float16* p = reinterpret_cast<_Float16*>(d.p) + row + split_at(c);
    const _Float16 hi = (_Float16)v;
    p[0] = hi;
    p[32] = (_Float16)(v - (float)hi);
  } else if (d.fmt == kDup) {
    _Float16* p = reinterpret_cast<_Float16*>(d.p) + row + split_at(c);
    p[0] = p[32] = (_Float16)v;
  } else if (d.fmt == kF16) {
    reinterpret_cast<_Float16*>(d.p)[row + c] = (_Float16)v;
  } else if (d.fmt == kBF16) {
    reinterpret_cast<__bf16*>(d.p)[row + c] = (__bf16)v;
  } else {
    reinterpret_cast<float*>(d.p)[row + c] = v;
  }
}

// N elements of T at any element's address, in one access where the hardware has one for the size: rows of
// an odd pitch cost little more than aligned ones that way.
template <typename T, int N> struct Loose {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
// N consecutive columns (N = 4 or 8, c a multiple of N) of row r; columns from `cols` on are padding
// (zeros up to d.pad, nothing behind it).
template <int N>
__device__ __forceinline__ void store_n(const Mat& d, int64_t b, int64_t r, int64_t c, int cols,
                                        const float (&v)[N]) {
  typedef _Float16 hN __attribute__((ext_vector_type(N)));
  typedef __bf16 bN __attribute__((ext_vector_type(N)));
  const int64_t row = b * d.batch + r * d.ld;
  const int end = d.pad > cols ? d.pad : cols;
  if (c >= end) return;
  float w[N];
#pragma unroll
  for (int i = 0; i < N; i++) w[i] = c + i < cols ? v[i] : 0.0f;
  if (c + N > end) {
    for (int i = 0; i < N; i++)
      if (c + i < end) store1(d, row, c + i, w[i]);
    return;
  }
  if (d.fmt == kSplit) {
    hN hi, lo;
#pragma unroll
    for (int i = 0; i < N; i++) {
      hi[i] = (_Float16)w[i];
      lo[i] = (_Float16)(w[i] - (float)hi[i]);
    }
    _Float16* p = reinterpret_cast<_Float16*>(d.p) + row + split_at(c);
    *reinterpret_cast<hN*>(p) = hi;
    *reinterpret_cast<hN*>(p + 32) = lo;
  } else if (d.fmt == kDup) {
    hN h;
#pragma unroll
    for (int i = 0; i < N; i++) h[i] = (_Float16)w[i];
    _Float16* p = reinterpret_cast<_Float16*>(d.p) + row + split_at(c);
    *reinterpret_cast<hN*>(p) = h;
    *reinterpret_cast<hN*>(p + 32) = h;
  } else if (d.fmt == kF16) {
    hN h;
#pragma unroll
    for (int i = 0; i < N; i++) h[i] = (_Float16)w[i];
    *reinterpret_cast<typename Loose<_Float16, N>::type*>(reinterpret_cast<_Float16*>(d.p) + row + c) = h;
  } else if (d.fmt == kBF16) {
    bN h;
#pragma unroll
    for (int i = 0; i < N; i++) h[i] = (__bf16)w[i];
    *reinterpret_cast<typename Loose<__bf16, N>::type*>(reinterpret_cast<__bf16*>(d.p) + row + c) = h;
  } else {
    float* p = reinterpret_cast<float*>(d.p) + row + c;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const typename Loose<float, 4>::type f = {w[i], w[i + 1], w[i + 2], w[i + 3]};
      *reinterpret_cast<typename Loose<float, 4>::type*>(p + i) = f;
    }
  }
}

// The tile a workgroup computes. Workgroup ids go round the 8 XCDs, each with its own L2: ids of one
// XCD get consecutive tiles, in bands of kBand tile rows, so the tiles an XCD has in flight share
// their rows of A and B. `tri`: only the tiles on and above the diagonal of a square tile grid (a
// symmetric product; the epilogue writes the mirrored part).
constexpr int kBand = 4;
__device__ __forceinline__ void pick_tile(int tm, int tn, int tri, int& im, int& in) {
  const int total = tri ? tm * (tm + 1) / 2 : tm * tn;
  const int id = blockIdx.x, x = id & 7, q = total >> 3, rem = total & 7;
  const int t = x * q + (x < rem ? x : rem) + (id >> 3);
  if (tri) {
    int r = (int)((2.0f * tm + 1.0f - sqrtf((2.0f * tm + 1.0f) * (2.0f * tm + 1.0f) - 8.0f * t)) * 0.5f);
    while (r > 0 && r * tm - r * (r - 1) / 2 > t) r--;
    while ((r + 1) * tm - (r + 1) * r / 2 <= t) r++;
    im = r;
    in = r + t - (r * tm - r * (r - 1) / 2);
    return;
  }
  const int band = t / (kBand * tn), first = band * kBand;
  const int high = tm - first < kBand ? tm - first : kBand;
  const int u = t - band * kBand * tn;
  im = first + u % high;
  in = u / high;
}

#if defined(__HIP_DEVICE_COMPILE__)  // the buffer builtins' types do not exist in the host pass
template <typename H, int BM, int BN, int WM, int WN, int STAGES, bool SPLIT, typename Epi>
__device__ __forceinline__ void gemm_nt_body(const Operand& A, const Operand& B, int kt, int tm, int tn,
                                             int tri, const Epi& epi, H* a0, H* b0, H* a1, H* b1, H* a2,
                                             H* b2, H* a3, H* b3) {
  typedef typename Frag<H>::type frag;
  constexpr int kWaves = WM * WN;
  constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
  constexpr int LA = BM / 8 / kWaves, LB = BN / 8 / kWaves;  // loads a wave issues per k tile
  static_assert(TM * WM * 32 == BM && TN * WN * 32 == BN, "tile");
  static_assert(LA * 8 * kWaves == BM && LB * 8 * kWaves == BN, "loads");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  int im, in;
  int m_rows = A.rows;
  if (A.live) {
    m_rows = *A.live < m_rows ? *A.live : m_rows;
    tm = (m_rows + BM - 1) / BM;
    if ((int)blockIdx.x >= tm * tn) return;
  }
  if (A.depth) {
    const int most = (*A.depth + (SPLIT ? 31 : 63)) / (SPLIT ? 32 : 64);
    kt = most < kt ? most : kt;
  }
  pick_tile(tm, tn, tri, im, in);
  const int row_a = im * BM, row_b = in * BN;
  const int64_t batch = blockIdx.z;
  // split k: this workgroup's share of the k tiles (gridDim.y = 1: all of them)
  const int k0 = (int)((int64_t)kt * blockIdx.y / gridDim.y);
  const int k1 = (int)((int64_t)kt * (blockIdx.y + 1) / gridDim.y);
  const int nk = k1 - k0;

  const int rows_a = m_rows - row_a < BM ? m_rows - row_a : BM;
  const int rows_b = B.rows - row_b < BN ? B.rows - row_b : BN;
  const char* pa = reinterpret_cast<const char*>(A.p) + 2 * (batch * A.batch + (int64_t)row_a * A.ld) + (int64_t)k0 * 128;
  const char* pb = reinterpret_cast<const char*>(B.p) + 2 * (batch * B.batch + (int64_t)row_b * B.ld) + (int64_t)k0 * 128;
  const int lda = (int)A.ld * 2, ldb = (int)B.ld * 2;
  const __amdgpu_buffer_rsrc_t ra =
      __builtin_amdgcn_make_buffer_rsrc((void*)pa, 0, (rows_a - 1) * lda + nk * 128, 0x00027000);
  const __amdgpu_buffer_rsrc_t rb =
      __builtin_amdgcn_make_buffer_rsrc((void*)pb, 0, (rows_b - 1) * ldb + nk * 128, 0x00027000);
  int va[LA], vb[LB];
  const int chunk = ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
  for (int i = 0; i < LA; i++) {
    const int r = (i * kWaves + wave) * 8 + (lane >> 3);
    va[i] = (r < rows_a ? r : rows_a - 1) * lda + chunk;
  }
#pragma unroll
  for (int i = 0; i < LB; i++) {
    const int r = (i * kWaves + wave) * 8 + (lane >> 3);
    vb[i] = (r < rows_b ? r : rows_b - 1) * ldb + chunk;
  }
  auto fetch = [&](H* la, H* lb, int t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < LA; i++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_void*)(la + (i * kWaves + wave) * 512), 16,
                                               va[i], t * 128, 0, 0);
#pragma unroll
    for (int i = 0; i < LB; i++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_void*)(lb + (i * kWaves + wave) * 512), 16,
                                               vb[i], t * 128, 0, 0);
  };
  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;

  const int fr = lane & 31, fk = lane >> 5, fx = lane & 7;
  auto read = [&](const H* la, const H* lb, int s, frag(&fa)[TM], frag(&fb)[TN])
      __attribute__((always_inline)) {
    const int at = ((s * 2 + fk) ^ fx) * 8;
#pragma unroll
    for (int i = 0; i < TM; i++)
      fa[i] = *reinterpret_cast<const frag*>(la + (wm * TM * 32 + i * 32 + fr) * 64 + at);
#pragma unroll
    for (int j = 0; j < TN; j++)
      fb[j] = *reinterpret_cast<const frag*>(lb + (wn * TN * 32 + j * 32 + fr) * 64 + at);
  };
  // hi*lo and lo*hi in sums of their own: hi*hi then rounds a third as often (8e-8 instead of 1.4e-7 of
  // a sum of 640 positive products). 256 x 256 tiles have no registers for them.
  constexpr bool kApart = SPLIT && BM < 256;
  f32x16 low[kApart ? TM : 1][kApart ? TN : 1];
  if constexpr (kApart) {
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) low[i][j][r] = 0.0f;
  }
  // operands swapped: a lane then holds runs of 4 consecutive n of one m
  auto mma = [&](const frag(&fa)[TM], const frag(&fb)[TN]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++) acc[i][j] = Frag<H>::mma(fb[j], fa[i], acc[i][j]);
  };
  auto cross = [&](const frag(&fa)[TM], const frag(&fb)[TN]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++) {
        if constexpr (kApart) low[i][j] = Frag<H>::mma(fb[j], fa[i], low[i][j]);
        else acc[i][j] = Frag<H>::mma(fb[j], fa[i], acc[i][j]);
      }
  };
  frag fa0[TM], fb0[TN], fa1[TM], fb1[TN], fa2[TM], fb2[TN];
  // One LDS read behind each MFMA: left to itself the compiler sinks a read to just before its use
  // and waits there.
  auto mix = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM + TN; i++) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto landed = [&]() __attribute__((always_inline)) {
    if constexpr (STAGES == 2)
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * (LA + LB)) : "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // One k tile in (la, lb), whose first fragments are in f0; (ma, mb) is the next tile's buffer.
  auto tile = [&](H* la, H* lb, H* ma, H* mb, int t) __attribute__((always_inline)) {
    if constexpr (!SPLIT) {
      read(la, lb, 1, fa1, fb1);
      mma(fa0, fb0);
      mix();
      read(la, lb, 2, fa0, fb0);
      mma(fa1, fb1);
      mix();
      read(la, lb, 3, fa1, fb1);
      mma(fa0, fb0);
      mix();
    } else {
      // chunks 0-3 are hi, 4-7 are lo
      read(la, lb, 2, fa1, fb1);
      mma(fa0, fb0);
      mix();
      cross(fa0, fb1);
      read(la, lb, 1, fa2, fb2);
      cross(fa1, fb0);
      mix();
      read(la, lb, 3, fa1, fb1);
      mma(fa2, fb2);
      mix();
    }
    // every wave has its fragments of this tile, and the next tile has landed (the ones behind it
    // may still be on their way)
    __builtin_amdgcn_s_setprio(0);
    landed();
    if constexpr (STAGES == 2) {
      if (t + 2 < nk) fetch(la, lb, t + 2);
    } else {  // always: `landed` counts the loads behind the next tile's
      fetch(la, lb, t + STAGES < nk ? t + STAGES : nk - 1);
    }
    __builtin_amdgcn_s_setprio(1);
    read(ma, mb, 0, fa0, fb0);
    if constexpr (!SPLIT) {
      mma(fa1, fb1);
      mix();
    } else {
      cross(fa2, fb1);
      cross(fa1, fb2);
      mix();
    }
  };
  if (nk > 0) {
    // (a tile past the end is the last one again: the counts of loads in flight stay the same)
    fetch(a0, b0, 0);
    fetch(a1, b1, nk > 1 ? 1 : 0);
    if constexpr (STAGES == 4) {
      fetch(a2, b2, nk > 2 ? 2 : 0);
      fetch(a3, b3, nk > 3 ? 3 : 0);
    }
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((STAGES - 1) * (LA + LB)) : "memory");
    read(a0, b0, 0, fa0, fb0);
    for (int t = 0;;) {
      if constexpr (STAGES == 2) {
        tile(a0, b0, a1, b1, t);
        if (++t >= nk) break;
        tile(a1, b1, a0, b0, t);
        if (++t >= nk) break;
      } else {
        tile(a0, b0, a1, b1, t);
        if (++t >= nk) break;
        tile(a1, b1, a2, b2, t);
        if (++t >= nk) break;
        tile(a2, b2, a3, b3, t);
        if (++t >= nk) break;
        tile(a3, b3, a0, b0, t);
        if (++t >= nk) break;
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // loads still in flight write the LDS
  }
  if constexpr (kApart) {
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int j = 0; j < TN; j++) acc[i][j] += low[i][j];
  }
  __syncthreads();  // the LDS buffers are free for the epilogue

  // 32 rows of the wave's part as fp32, in one of the four buffers
  constexpr int kPitch = TN * 32 + 4;
  constexpr int kNeed = 32 * kPitch * 4;
  constexpr int kInA = BM * 128 / kNeed, kInB = BN * 128 / kNeed;
  static_assert(2 * (kInA + kInB) >= kWaves, "staging");
  float* stage;
  {
    int w = wave;
    if (w < kInA) stage = reinterpret_cast<float*>(a0) + w * 32 * kPitch;
    else if ((w -= kInA) < kInB) stage = reinterpret_cast<float*>(b0) + w * 32 * kPitch;
    else if ((w -= kInB) < kInA) stage = reinterpret_cast<float*>(a1) + w * 32 * kPitch;
    else stage = reinterpret_cast<float*>(b1) + (w - kInA) * 32 * kPitch;
  }
  epi.template finish<BM, BN, WM, WN, TM, TN>(acc, stage, row_a + wm * TM * 32,
                                              row_b + wn * TN * 32, m_rows, B.rows, im, in, wm, wn,
                                              lane, batch);
}
#endif

// The LDS buffers of each depth are variables of their own kernel: that is what the compiler tells
// them apart by.
#define SMQ_TILE_LDS(name, rows) __shared__ __attribute__((aligned(1024))) H name[(rows) * 64]
template <typename H, int BM, int BN, int WM, int WN, bool SPLIT, typename Epi>
__global__ __launch_bounds__(WM* WN * 64, 2) void gemm_nt_kernel(Operand A, Operand B, int kt, int tm,
                                                                 int tn, int tri, Epi epi) {
#if defined(__HIP_DEVICE_COMPILE__)
  SMQ_TILE_LDS(a0, BM);
  SMQ_TILE_LDS(b0, BN);
  SMQ_TILE_LDS(a1, BM);
  SMQ_TILE_LDS(b1, BN);
  gemm_nt_body<H, BM, BN, WM, WN, 2, SPLIT>(A, B, kt, tm, tn, tri, epi, a0, b0, a1, b1, a0, b0, a1, b1);
#endif
}
template <typename H, int BM, int BN, int WM, int WN, bool SPLIT, typename Epi>
__global__ __launch_bounds__(WM* WN * 64, 1) void gemm_nt_deep_kernel(Operand A, Operand B, int kt,
                                                                      int tm, int tn, int tri, Epi epi) {
#if defined(__HIP_DEVICE_COMPILE__)
  SMQ_TILE_LDS(a0, BM);
  SMQ_TILE_LDS(b0, BN);
  SMQ_TILE_LDS(a1, BM);
  SMQ_TILE_LDS(b1, BN);
  SMQ_TILE_LDS(a2, BM);
  SMQ_TILE_LDS(b2, BN);
  SMQ_TILE_LDS(a3, BM);
  SMQ_TILE_LDS(b3, BN);
  gemm_nt_body<H, BM, BN, WM, WN, 4, SPLIT>(A, B, kt, tm, tn, tri, epi, a0, b0, a1, b1, a2, b2, a3, b3);
#endif
}
#undef SMQ_TILE_LDS

__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Walks a wave's part of C through its LDS stage, 32 rows at a time: `f(m, n, v)` turns four
// consecutive accumulators of row m into the values to be written, which go to `o` row by row and,
// where `ot` is set, to `ot` transposed. `colsum(n, v)`, where given, gets the sum over the part's
// rows of column n. Lanes past the edges call neither. `prep(m)` (ROWS): what f needs of a row, four words, read
// once per row into the stage's spare columns (f's fourth argument): the first is a factor of the row in the
// transposed copy, `weigh(v, last)` makes the term of a column's sum of the copy's value and the row's last word,
// `out(v)` what goes to `o`.
template <int TM, int TN, bool ROWS, typename P, typename F, typename O, typename W, typename S>
__device__ __forceinline__ void stage_out(const f32x16 (&acc)[TM][TN], float* stage, int m0, int n0,
                                          int M, int N, int lane, int64_t batch, const Mat& o,
                                          const Mat& ot, bool mirror, bool sums, P prep, F f, O out, W weigh,
                                          S colsum) {
  constexpr int kCols = TN * 32, kPitch = kCols + 4;
  constexpr int kPer = kCols / 4, kRows = 64 / kPer;  // row phase: lanes a row, rows a pass
  float total = 0.0f;
#pragma unroll
  for (int i = 0; i < TM; i++) {
    const int mb = m0 + i * 32;
    if (mb < M || (mirror && mb < ot.pad)) {  // rows from M on are the transposed matrix's padding
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
          *reinterpret_cast<float4*>(stage + (lane & 31) * kPitch + j * 32 + 2 * r + 4 * (lane >> 5)) =
              make_float4(acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]);
      if constexpr (ROWS) {
        if (lane < 32 && mb + lane < M)
          *reinterpret_cast<float4*>(stage + lane * kPitch + kCols) = prep(mb + lane);
      }
      wave_sync();
#pragma unroll 4
      for (int p = 0; p < 32; p += kRows) {
        const int r = p + lane / kPer, c = (lane % kPer) * 4;
        float* at = stage + r * kPitch + c;
        float4 v = *reinterpret_cast<const float4*>(at);
        if (mb + r < M) {
          float factor = 1.0f;
          if (n0 + c < N) {
            if constexpr (ROWS) {
              const float4 row = *reinterpret_cast<const float4*>(stage + r * kPitch + kCols);
              v = f(mb + r, n0 + c, v, row);
              factor = row.x;
            } else {
              v = f(mb + r, n0 + c, v);
            }
          }
          if (o.fmt != kNone) {
            float4 u = v;
            if constexpr (ROWS) u = out(v);
            const float w[4] = {u.x, u.y, u.z, u.w};
            store_n<4>(o, batch, mb + r, n0 + c, N, w);
          }
          if constexpr (ROWS) v.x *= factor, v.y *= factor, v.z *= factor, v.w *= factor;
          if (mirror || sums) *reinterpret_cast<float4*>(at) = v;
        }
      }
      if (mirror || sums) {
        wave_sync();
        if (lane < kCols) {
          const int n = n0 + (lane % kCols);
          if (n < N) {
#pragma unroll
            for (int r = 0; r < 32; r += 8) {
              float w[8];
#pragma unroll
              for (int k = 0; k < 8; k++) w[k] = mb + r + k < M ? stage[(r + k) * kPitch + lane % kCols] : 0.0f;
              if constexpr (ROWS) {
                if (sums) {
#pragma unroll
                  for (int k = 0; k < 8; k++)
                    if (mb + r + k < M) total += weigh(w[k], stage[(r + k) * kPitch + kCols + 3]);
                }
              }
              if (mirror) store_n<8>(ot, batch, n, mb + r, M, w);
            }
          }
        }
      }
      wave_sync();
    }
  }
  if (mirror && m0 < M && m0 + TM * 32 >= M && lane < kCols && n0 + lane < N) {
    // padding behind the tile's own rows (a 32-row tile under a 64-column pad)
    const float zero[8] = {};
    for (int m = m0 + TM * 32; m < ot.pad; m += 8) store_n<8>(ot, batch, n0 + lane, m, M, zero);
  }
  if (sums && (lane < kCols) && n0 + lane < N) colsum(n0 + lane, total);
}

// C = (alpha * acc + beta * src + diag * I) * rows[m], to `o` and / or transposed to `ot` (a symmetric product
// writes the same matrix twice; its diagonal tiles once). `scale`: a factor of alpha in device memory,
// one per matrix of the batch, or NULL.
// A launch split over k (gridDim.y shares) writes share y to o + y * share.
__device__ __forceinline__ void add_diag(float4& v, int m, int n, float d) {
  const int k = m - n;
  v.x += k == 0 ? d : 0.0f, v.y += k == 1 ? d : 0.0f, v.z += k == 2 ? d : 0.0f, v.w += k == 3 ? d : 0.0f;
}
struct StoreEpi {
  float alpha, beta;
  const float* scale;
  Mat src, o, ot;
  int tri;
  int64_t share;
  float diag;
  // split_sum_kernel only: row m goes to row map[m] of `o`, those from *live on as zeros (NULL: as they are)
  const int* map = nullptr;
  const int* live = nullptr;
  const float* rows = nullptr;  // a factor per row, `row_step` apart (NULL: none)
  int row_step = 1;
  template <int BM, int BN, int WM, int WN, int TM, int TN>
  __device__ __forceinline__ void finish(f32x16 (&acc)[TM][TN], float* stage, int m0, int n0, int M,
                                         int N, int im, int in, int, int, int lane,
                                         int64_t batch) const {
    const float al = scale ? alpha * scale[batch] : alpha;
    Mat s = src, d = o;
    if (gridDim.y > 1) {
      d.p = reinterpret_cast<float*>(d.p) + blockIdx.y * share;
      if (s.fmt != kNone) s.p = reinterpret_cast<float*>(s.p) + blockIdx.y * share;
    }
    const float be = beta, dg = diag;
    stage_out<TM, TN, false>(
        acc, stage, m0, n0, M, N, lane, batch, d, ot, ot.fmt != kNone && !(tri && im == in), false, 0,
        [&](int m, int n, float4 v) {
          v.x *= al, v.y *= al, v.z *= al, v.w *= al;
          if (s.fmt != kNone) {
            const float4 c = load4(s, batch, m, n);
            v.x += be * c.x, v.y += be * c.y, v.z += be * c.z, v.w += be * c.w;
          }
          add_diag(v, m, n, dg);
          if (rows) {
            const float f = rows[(int64_t)m * row_step];
            v.x *= f, v.y *= f, v.z *= f, v.w *= f;
          }
          return v;
        },
        0, 0, [](int, float) {});
  }
};

// The second half of a product split over k: C = (alpha * sum over the shares + beta * src + diag * I) * rows[m],
// 32 x 32 a workgroup (the same walk as the product's own epilogue, with the tile in LDS).
static __global__ __launch_bounds__(256) void split_sum_kernel(const float* part, int64_t ld,
                                                               int64_t share, int shares,
                                                               int64_t batch_stride, int M, int N,
                                                               int mirror, StoreEpi e) {
  __shared__ float tile[32][36];
  const int im = blockIdx.y, in = blockIdx.x;
  if (e.tri && in / 2 < im / 2) return;  // (the shares hold whole tiles of 64, so the diagonal's both halves)
  const int64_t batch = blockIdx.z;
  const float al = e.scale ? e.alpha * e.scale[batch] : e.alpha;
  const int c = (threadIdx.x & 7) * 4, r = threadIdx.x >> 3;
  const bool turn = mirror && !(e.tri && im / 2 == in / 2);
  const int m = im * 32 + r, n = in * 32 + c;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (m < M) {
    if (n < N && !(e.live && m >= *e.live)) {
      const float* q = part + batch * batch_stride + (int64_t)m * ld + n;
#pragma unroll 4
      for (int k = 0; k < shares; k++) {
        const float4 w = *reinterpret_cast<const float4*>(q + k * share);
        v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
      }
      v.x *= al, v.y *= al, v.z *= al, v.w *= al;
      if (e.src.fmt != kNone) {
        const float4 s = load4(e.src, batch, m, n);
        v.x += e.beta * s.x, v.y += e.beta * s.y, v.z += e.beta * s.z, v.w += e.beta * s.w;
      }
      add_diag(v, m, n, e.diag);
      if (e.rows) {
        const float f = e.rows[(int64_t)m * e.row_step];
        v.x *= f, v.y *= f, v.z *= f, v.w *= f;
      }
    }
    const float w[4] = {v.x, v.y, v.z, v.w};
    if (e.o.fmt != kNone) store_n<4>(e.o, batch, e.map ? e.map[m] : m, n, N, w);
  }
  if (!turn) return;
  *reinterpret_cast<float4*>(&tile[r][c]) = v;
  __syncthreads();
  const int nt = in * 32 + (threadIdx.x & 31), m0 = im * 32 + (threadIdx.x >> 5) * 4;
  if (nt < N) {
    float w[4];
#pragma unroll
    for (int k = 0; k < 4; k++) w[k] = m0 + k < M ? tile[(threadIdx.x >> 5) * 4 + k][threadIdx.x & 31] : 0.0f;
    store_n<4>(e.ot, batch, nt, m0, M, w);
  }
}
static inline void launch_split_sum(const float* part, int64_t ld, int64_t share, int shares,
                                    int64_t batch_stride, int M, int N, int batch, int mirror,
                                    const StoreEpi& e, hipStream_t st) {
  // (whole 64-column pads of an operand: its padding is written here too)
  hipLaunchKernelGGL(split_sum_kernel, dim3((N + 63) / 64 * 2, (M + 63) / 64 * 2, batch), dim3(256), 0, st,
                     part, ld, share, shares, batch_stride, M, N, mirror, e);
}

// Tile shapes. 256 x 256 runs fastest per tile, but a grid below the CU count leaves CUs idle; smaller
// tiles fill them. kT128 has two k tiles in LDS and leaves room for a second workgroup on the CU;
// kDeep, kT64 and kSkinny have four on the way, for grids that give a CU only one workgroup to hide
// the loads behind. kSkinny: up to 32 rows of A, the product bounded by the read of B.
enum Tile : int { kT256 = 0, kT128 = 1, kT64 = 2, kSkinny = 3, kDeep = 4 };
struct TileShape {
  int bm, bn, wm;
};
static inline TileShape shape_of(int t) {
  switch (t) {
    case kT256: return {256, 256, 2};
    case kT128: return {128, 128, 2};
    case kDeep: return {128, 128, 2};
    case kT64: return {64, 64, 2};
    default: return {32, 128, 1};
  }
}
static inline int64_t tile_count(int64_t m, int64_t n, int t, int tri) {
  const TileShape s = shape_of(t);
  const int64_t a = (m + s.bm - 1) / s.bm, b = (n + s.bn - 1) / s.bn;
  return tri ? a * (a + 1) / 2 : a * b;
}
// Tile and shares of the k range for C [m, n] x batch over kt k tiles, by a cost in units of 28 ps: what a
// CU needs for one element of C and one k tile at the rate of 256 x 256 tiles. A round of workgroups
// costs its tile's area over the tile's relative rate (measured: 128 x 128 0.87 with two workgroups a CU,
// 0.75 with one, 64 x 64 0.6 and 0.4, and so 32 x 128 by its area); rows and columns past the edge cost as
// much as others, so a short m takes short tiles. Sharing k costs a pass over the partial sums (0.07 an
// element and share) and a launch. 2048 x 768 over 938: 10 shares of 256 x 256 (24 tiles without);
// 6 x 1024 x 4096 over 32: 128 x 128 in three full rounds (74 us) instead of 256 x 256 in two (81 us).
struct Shared {
  int tile, shares;
};
static inline Shared plan_product(int64_t m, int64_t n, int64_t kt, int64_t batch, int tri, bool share,
                                  bool big = true) {
  Shared best = {kT64, 1};
  double least = -1.0;
  const int most = !share || kt < 16 ? 1 : (int)(kt / 8 > 64 ? 64 : kt / 8);
  auto look = [&](int tile, int64_t slots, double one, double both) {
    const int64_t count = batch * tile_count(m, n, tile, tri);
    for (int s = 1; s <= most; s++) {
      const int64_t wgs = count * s;
      const double rounds = wgs <= 256 ? one : both * (double)((wgs + slots - 1) / slots);
      double cost = rounds * (double)((kt + s - 1) / s);
      if (s > 1) cost += 0.07 * (double)s * (double)(batch * m * n) + 175e3;
      if (least < 0.0 || cost < least) least = cost, best = {tile, s};
      if (wgs >= 2 * slots) break;
    }
  };
  if (big) look(kT256, 256, 65536.0, 65536.0);
  look(kT128, 512, 21845.0, 37664.0);
  if (best.tile == kT128 && batch * tile_count(m, n, kT128, tri) * best.shares <= 256) best.tile = kDeep;
  const Shared before = best;
  look(kT64, 512, 10240.0, 13650.0);
  if (best.tile != kT64) best = before;
  if (m <= 32 && !tri) look(kSkinny, 256, 10240.0, 10240.0);
  return best;
}

template <typename H, int BM, int BN, int WM, int WN, bool DEEP, bool SPLIT, typename Epi>
static inline void launch_tile(const Operand& A, const Operand& B, int kt, int batch, int tri,
                               int shares, const Epi& epi, hipStream_t st) {
  const int tm = (A.rows + BM - 1) / BM, tn = (B.rows + BN - 1) / BN;
  const dim3 grid(tri ? tm * (tm + 1) / 2 : tm * tn, shares, batch), block(WM * WN * 64);
  if constexpr (DEEP)
    hipLaunchKernelGGL((gemm_nt_deep_kernel<H, BM, BN, WM, WN, SPLIT, Epi>), grid, block, 0, st, A, B, kt,
                       tm, tn, tri, epi);
  else
    hipLaunchKernelGGL((gemm_nt_kernel<H, BM, BN, WM, WN, SPLIT, Epi>), grid, block, 0, st, A, B, kt, tm,
                       tn, tri, epi);
}
template <typename H, bool SPLIT, typename Epi>
static inline void launch(int tile, const Operand& A, const Operand& B, int kt, int batch, int tri,
                          int shares, const Epi& epi, hipStream_t st) {
  switch (tile) {
    case kT256: return launch_tile<H, 256, 256, 2, 4, false, SPLIT>(A, B, kt, batch, tri, shares, epi, st);
    case kT128: return launch_tile<H, 128, 128, 2, 2, false, SPLIT>(A, B, kt, batch, tri, shares, epi, st);
    case kDeep: return launch_tile<H, 128, 128, 2, 2, true, SPLIT>(A, B, kt, batch, tri, shares, epi, st);
    case kT64: return launch_tile<H, 64, 64, 2, 2, true, SPLIT>(A, B, kt, batch, tri, shares, epi, st);
    default: return launch_tile<H, 32, 128, 1, 4, true, SPLIT>(A, B, kt, batch, tri, shares, epi, st);
  }
}

// In a sum whose largest terms have scale 2^0 a term of 2^-k is the product of a factor (of the tensor's row, whose
// largest element is at 2^14) and a probability (at 2^14 and far below): this part of k comes off the factor's
// fp16 planes, the rest off the probability's, so that both stay in fp16's range. The factor keeps 2^-24 of its
// row's largest for the first 15, and only then the probability loses from its end, 2^-39; past 30 they share.
// (Past 100 both are 0 in fp16; the probability's part stays a normal float.)
__device__ __forceinline__ int share_of(int k) {
  return k > 100 ? k - 50 : k > 30 ? k >> 1 : k > 15 ? 15 : k;
}
// Power-of-two exponents of a matrix' rows: e[step * r] (step 0: *e for all of them); e NULL: 0. With `least`, the
// smallest of them, their share of the difference comes off.
struct Exponents {
  const int* e = nullptr;
  int step = 0;
  const int* least = nullptr;
  __device__ __forceinline__ int all() const { return e && step == 0 ? *e : 0; }
  __device__ __forceinline__ int at(int r) const {
    if (!step) return all();
    const int v = e[step * r];
    return least ? v - share_of(v - *least) : v;
  }
};
// Layout pass: src [rows, cols] of type T, row pitch ld, times *factor (NULL: 1), to `d` row by row, times
// 2^exponent of the row, and / or to `dt` transposed, times 2^turned (either may be absent), zero padded.
// Rows whose keep[row] equals `skip` are written as zeros (keep NULL: none). With `map`, row r is src's row
// map[r], and rows from *live on are zeros. 64 x 64 a workgroup; bound by its reads and writes of memory.
template <typename T>
static __global__ __launch_bounds__(256) void layout_kernel(const T* src, int64_t ld,
                                                            int64_t batch_stride, int rows, int cols,
                                                            Exponents exponent, Exponents turned,
                                                            const float* factor,
                                                            const int64_t* keep, int64_t skip,
                                                            const int* map, const int* live, Mat d,
                                                            Mat dt) {
  __shared__ float tile[64][65];
  const int64_t batch = blockIdx.z;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  const float fa = factor ? factor[batch] : 1.0f;
  const T* p = src + batch * batch_stride;
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
  int er[4], et[4];
#pragma unroll
  for (int i = 0; i < 4; i++) er[i] = exponent.all(), et[i] = turned.all();
  if (exponent.step | turned.step) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int r = r0 + y + i * 16 < rows ? r0 + y + i * 16 : 0;
      er[i] = exponent.at(r), et[i] = turned.at(r);
    }
  }
#pragma unroll
  for (int i = 0; i < 64; i += 16) {
    const int r = r0 + y + i, c = c0 + x * 4;
    float w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (r < rows && !(keep && keep[r] == skip) && !(map && r >= *live)) {
      const T* q = p + (int64_t)(map ? map[r] : r) * ld;
      typedef typename Loose<T, 4>::type t4;
      if (c + 4 <= cols) {
        const t4 v = *reinterpret_cast<const t4*>(q + c);
#pragma unroll
        for (int k = 0; k < 4; k++) w[k] = (float)v[k];
      } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (c + k < cols) w[k] = (float)q[c + k];
      }
#pragma unroll
      for (int k = 0; k < 4; k++) w[k] *= fa;
    }
    if (dt.fmt != kNone) {
#pragma unroll
      for (int k = 0; k < 4; k++) tile[y + i][x * 4 + k] = ldexpf(w[k], et[i / 16]);
    }
    if (d.fmt != kNone && r < rows) {
#pragma unroll
      for (int k = 0; k < 4; k++) w[k] = ldexpf(w[k], er[i / 16]);
      store_n<4>(d, batch, r, c, cols, w);
    }
  }
  if (dt.fmt == kNone) return;
  __syncthreads();
  // lanes: 8 runs of 8 rows, 8 columns a wave and pass
  const int run = (threadIdx.x & 7) * 8, cc = threadIdx.x >> 3;
#pragma unroll
  for (int i = 0; i < 64; i += 32) {
    const int c = c0 + cc + i;
    if (c < cols) {
      float w[8];
#pragma unroll
      for (int k = 0; k < 8; k++) w[k] = tile[run + k][cc + i];
      store_n<8>(dt, batch, c, r0 + run, rows, w);
    }
  }
}
template <typename T>
static inline void launch_layout(const T* src, int64_t ld, int64_t batch_stride, int rows, int cols,
                                 int batch, const Exponents& exponent, const Exponents& turned,
                                 const float* factor, const int64_t* keep, int64_t skip, const Mat& d, const Mat& dt,
                                 hipStream_t st, const int* map = nullptr, const int* live = nullptr) {
  hipLaunchKernelGGL(layout_kernel<T>, dim3((cols + 63) / 64, (rows + 63) / 64, batch), dim3(256), 0,
                     st, src, ld, batch_stride, rows, cols, exponent, turned, factor, keep, skip, map, live, d,
                     dt);
}

static inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
// Row pitch (elements) and padded columns of a k-contiguous operand of k columns. A pitch of whole 2 KiB
// gets 128 bytes more: rows that far apart would meet in few memory channels (8192 x 8192 x 8192 runs
// at 1033 TFLOP/s with rows 16 KiB apart, x 21504 at 1166).
static inline int64_t operand_ld(int64_t k, bool split) {
  const int64_t l = split ? 2 * round_up(k, 32) : round_up(k, 64);
  return l % 1024 == 0 ? l + 64 : l;
}
static inline int operand_pad(int64_t k, bool split) { return (int)round_up(k, split ? 32 : 64); }
static inline int operand_kt(int64_t k, bool split) {
  return (int)(split ? round_up(k, 32) / 32 : round_up(k, 64) / 64);
}

}  // namespace gemm
}  // namespace smq
