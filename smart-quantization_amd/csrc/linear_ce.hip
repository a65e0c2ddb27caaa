// linear_ce.hip — softmax cross entropy of a linear head, without keeping the logits, and its gradient.
//
//   l[m, v] = h[m] . w[v] + b[v],   lse[m] = log sum_v exp l[m, v],   loss[m] = lse[m] - l[m, t[m]]
//   dl[m, v] = g[m] (exp(l[m, v] - lse[m]) - [v = t[m]]),   dh = dl w,   dw = dl^T h,   db = sum_m dl
//
// Forward: one matrix product whose epilogue keeps, per row and per block of columns, the maximum and
// the sum of exponentials (and the target's logit); a second small launch joins them. The logits
// exist in registers only. Backward: the vocabulary in pieces. Per piece the logits are computed
// again, dl is written once as the 16-bit operand of the two gradient products, row by row and
// transposed, and used up. Only lse is kept between the two passes.
//
// By size and type:
//   up to 16 tokens        no matrix cores: the weight is read as it is, once in the forward and twice in the
//                          backward (1 x 768 x 30000 float32 forward: 23 us, 18 at the rate of a copy)
//   float32, to 128        the logits on the fp32 matrix instructions from the inputs in place, where their rows
//                          allow (64 x 1024 x 30000: forward 47 us, both directions 275)
//   the rest               16-bit matrix products; long ones over the rows that take part only (Kept).
// Measured, forward and backward: 8192 x 4096 x 131072 bf16 33.5 ms (8 N V D operations with the logits'
// second computation: 1050 TFLOP/s), 2048 x 768 x 30000 float32 1.32 ms, 777 x 1001 x 50001 fp16 with a third
// of the rows ignored 0.63 ms. What bounds the large ones is the product itself, then dl's two copies.
//
// float32 inputs run as two fp16 planes (gemm_nt.h), in the logits each row scaled by a power of two of its
// own, taken off in the epilogue: every row is as exact as if it were alone, whatever the others' size. bf16 and
// fp16 inputs run as they are. In the gradient products every 16-bit operand is fp16: dl rounded to 11 bits
// (8 bits of bf16 were off by up to 2e-3 in the gradient of a target's row), and bf16 inputs, exact in
// fp16 once scaled (what lies 2^-28 below a row's largest magnitude loses bits), in the transposed copies
// that these products need anyway. dl is kept times 2^14, so that fp16 holds probabilities from 4e-9 up in
// full precision, and the powers of two come off in the fp32 epilogues. A row's gradient g stays out of dl's
// copy for dh, whose epilogue takes it: a row of dh is as exact as if it were alone. The sum over the rows in dw
// has one scale, that of the largest |g| |h| of a row; a row 2^-k of it (float32, bf16) has k taken off h's
// transposed copy and dl's, shared so that both stay in fp16's range (share_of, Row); dh's sum over float32 entries
// the same of the largest |w|. float32: h and w to 2^-24 of their row's largest and p to 2^-38 up to k = 15, p to
// 2^(k - 53) up to k = 30, both to 2^(k / 2 - 38) beyond. The row exponents cost one read more of the weight in
// each direction than one for all.
#include <limits.h>

#include <type_traits>

#include "gemm_nt.h"

namespace smq {
namespace ce {  // named: a kernel template's arguments need linkage
using namespace gemm;

constexpr float kDlScale = 16384.0f;
constexpr size_t kPieceBytes = size_t(1) << 30;  // default limit of a backward piece's buffers

// What a pass keeps on the device; the count is what the forward leaves for the backward.
struct Head {
  int exp_w;     // backward: exponent of the transposed weight
  int rows;      // rows that take part, where they are gathered (Kept)
  double count;  // rows that take part
  int exp_dw;    // backward: the largest exponent of a row's g times its h
  float scale_dh, scale_dw;  // the factors of the gradients
};
// What the backward keeps of a row. Where its |g| |h| is 2^-k of the largest row's, h's transposed copy has
// share_of(k) of k taken off, dl's the rest: t is below 2^(share - k) in magnitude.
struct Row {
  float g;     // its gradient (ignored: 0, a bad target: NaN)
  float t;     // the factor of dl's transposed copy, g 2^(-exp_dw - turned)
  int exp;     // exponent of its h, whose largest magnitude it brings to [2^13, 2^14) (fp16: 0)
  int turned;  // exponent of h's transposed copy, exp - share
};


// ---- largest magnitudes -> exponents -------------------------------------------------------------
__device__ __forceinline__ float finite_max(float top, float x) {
  const float a = fabsf(x);
  return a < __builtin_inff() ? fmaxf(top, a) : top;
}
// Exponent e with max * 2^e in [2^13, 2^14): room for the fp16 planes and for sums of their products.
__device__ int plane_exponent(float top) {
  if (!(top > 0.0f)) return 120;  // zeros: like the smallest
  int e;
  frexpf(top, &e);
  const int k = 14 - e;
  return k > 120 ? 120 : k;
}
// Workgroups below gh take h [tokens, dim], the others w [vocab, dim]: the largest magnitude of what each
// reads, to part, and the exponents of the rows, to eh and ew (NULL: not wanted). 2^k lanes read a row, as many
// as its vectors keep busy. A weight without gaps whose rows' exponents are not wanted is read as one row, in
// whole vectors whatever the columns. What is not finite, and rows that are ignored, set no scale.
template <typename T>
__global__ __launch_bounds__(256) void absmax_kernel(const T* h, int64_t ldh, int64_t tokens, const T* w,
                                                     int64_t ldw, int64_t vocab, int cols,
                                                     const int64_t* target, int64_t ignore, int gh, float* part,
                                                     int* eh, int* ew) {
  constexpr int V = 16 / sizeof(T);
  typedef typename Loose<T, V>::type vec;
  const bool first = (int)blockIdx.x < gh;
  const T* x = first ? h : w;
  int* e = first ? eh : ew;
  const int64_t ld = first ? ldh : ldw, rows = first ? tokens : vocab;
  const int block = first ? blockIdx.x : blockIdx.x - gh, blocks = first ? gh : gridDim.x - gh;
  float top = 0.0f;
  if (!first && ld == cols && !e) {
    const int64_t total = rows * cols, vecs = total / V, step = (int64_t)blocks * 256;
    const vec* p = reinterpret_cast<const vec*>(x);
#pragma unroll 4
    for (int64_t k = block * 256 + threadIdx.x; k < vecs; k += step) {
      const vec v = p[k];
#pragma unroll
      for (int i = 0; i < V; i++) top = finite_max(top, (float)v[i]);
    }
    if (block == 0 && (int)threadIdx.x < total - vecs * V)
      top = finite_max(top, (float)x[vecs * V + threadIdx.x]);
  } else {
    const int whole = cols / V * V;
    int shift = 6;
    while (shift > 2 && V << (shift - 1) >= cols) shift--;
    const int lanes = 1 << shift, at = threadIdx.x & (lanes - 1);
    for (int64_t r = ((int64_t)block * 256 + threadIdx.x) >> shift; r < rows; r += ((int64_t)blocks * 256) >> shift) {
      float m = 0.0f;
      if (!(first && target[r] == ignore)) {
        const T* p = x + r * ld;
#pragma unroll 4
        for (int k = at * V; k < whole; k += lanes * V) {
          const vec v = *reinterpret_cast<const vec*>(p + k);
#pragma unroll
          for (int i = 0; i < V; i++) m = finite_max(m, (float)v[i]);
        }
        for (int k = whole + at; k < cols; k += lanes) m = finite_max(m, (float)p[k]);
      }
      if (e) {  // (a row's lanes are here together)
        for (int o = lanes >> 1; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        if (at == 0) e[r] = plane_exponent(m);
      }
      top = fmaxf(top, m);
    }
  }
  top = wave_max_dpp(top);
  __shared__ float m[4];
  if ((threadIdx.x & 63) == 0) m[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// The largest of one value a thread, in all threads of a workgroup of 16 waves.
__device__ float largest_of(float v, float* sh) {
  v = wave_max_dpp(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  for (int k = 0; k < 16; k++) v = fmaxf(v, sh[k]);
  return v;
}

// ---- rows that take part, gathered --------------------------------------------------------------------
// Padding and masked tokens are ignored rows. Where the products are long, the others are gathered and
// only they are multiplied: their count stays on the device (gemm_nt.h's `live` and `depth`). map holds
// the rows taking part in order, then the ignored ones; the other arrays are in the gathered order.
struct Kept {
  int* map;
  int64_t* target;
  int* exp;    // forward, float32: the rows' exponents, else NULL
  float* lse;  // backward
};
// put(row, place, whether it takes part) for all rows, and their count; one workgroup of 16 waves.
template <typename F>
__device__ __forceinline__ void partition_rows(const int64_t* target, int64_t ignore, int rows, int* live,
                                               F put) {
  __shared__ int counts[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int total = 0;
  for (int m = threadIdx.x; m < rows; m += 1024) total += target[m] != ignore ? 1 : 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
  if (lane == 0) counts[wave] = total;
  __syncthreads();
  total = 0;
  for (int k = 0; k < 16; k++) total += counts[k];
  int done = 0;
  for (int base = 0; base < rows; base += 1024) {
    const int m = base + threadIdx.x;
    const bool keep = m < rows && target[m] != ignore;
    const uint64_t mask = __ballot(keep);
    __syncthreads();
    if (lane == 0) counts[wave] = __popcll(mask);
    __syncthreads();
    int at = done + __popcll(mask & ((1ull << lane) - 1));
    for (int k = 0; k < 16; k++) {
      at += k < wave ? counts[k] : 0;
      done += counts[k];
    }
    if (m < rows) put(m, keep ? at : total + (m - at), keep);
  }
  if (threadIdx.x == 0) *live = total;
}
// eh: the exponents of all rows (kept.exp NULL: none).
__global__ __launch_bounds__(1024) void gather_kernel(const int64_t* target, int64_t ignore, int rows,
                                                      const int* eh, Head* head, Kept kept) {
  partition_rows(target, ignore, rows, &head->rows, [&](int m, int at, bool keep) {
    kept.map[at] = m;
    if (keep) kept.target[at] = target[m];
    if (keep && kept.exp) kept.exp[at] = eh[m];
  });
}

// exp(x) for x <= about 0, within 2 ulp: the product with log2(e) is carried in two parts (a single
// one is off by up to |x| 2^-24, 1e-6 of the result at x = -11). NaN stays NaN.
__device__ __forceinline__ float exp_near(float x) {
  x = x < -200.0f ? -200.0f : x;
  const float t = x * 1.44269504f;
  const float e = fmaf(x, 1.44269504f, -t) + x * 1.92596303e-8f;
  const float p = __builtin_amdgcn_exp2f(t);
  return fmaf(p, e * 0.693147181f, p);
}

// ---- forward epilogue ---------------------------------------------------------------------------
// Per row and per tile's columns: the maximum and the sum of exp(l - maximum), joined over the tile's
// waves in LDS; the target's logit goes straight out (one lane of the grid owns it).
template <bool PLANES>
struct SoftmaxEpi {
  const int *eh, *ew;  // PLANES: exponents that come off a row and a column
  const float* bias;
  const int64_t* target;
  float2* part;  // [tiles][rows]
  float* picked;
  template <int BM, int BN, int WM, int WN, int TM, int TN>
  __device__ __forceinline__ void finish(f32x16 (&acc)[TM][TN], float*, int m0, int n0, int M, int N,
                                         int im, int in, int wm, int wn, int lane, int64_t) const {
    __shared__ float2 joint[WN][BM];
    int em[TM];
#pragma unroll
    for (int i = 0; i < TM; i++) {
      const int m = m0 + i * 32 + (lane & 31);
      em[i] = PLANES && m < M ? eh[m] : 0;
    }
    const float ninf = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int n = n0 + j * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
        const float b = bias && n < N ? bias[n] : 0.0f;
        const int en = PLANES ? ew[n] : 0;  // (past N: its padding)
#pragma unroll
        for (int i = 0; i < TM; i++) {
          const float l = PLANES ? ldexpf(acc[i][j][r], -(em[i] + en)) : acc[i][j][r];
          acc[i][j][r] = n < N ? l + b : ninf;
        }
      }
#pragma unroll
    for (int i = 0; i < TM; i++) {
      const int m = m0 + i * 32 + (lane & 31);
      float top = ninf;
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) top = fmaxf(top, acc[i][j][r]);
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float at = top == ninf ? 0.0f : top;
      float sum = 0.0f;
      const int64_t t = m < M ? target[m] : -1;
      const int off = t >= n0 && t < n0 + TN * 32 ? (int)(t - n0) : -1;
#pragma unroll
      for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          sum += exp_near(acc[i][j][r] - at);
          if (off == j * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3) && t < N)
            picked[m] = acc[i][j][r];
        }
      sum += __shfl_xor(sum, 32, 64);
      if (lane < 32) joint[wn][wm * TM * 32 + i * 32 + lane] = make_float2(top, sum);
    }
    __syncthreads();
    const int row = threadIdx.x;
    if (row < BM && im * BM + row < M) {
      float2 a = joint[0][row];
#pragma unroll
      for (int k = 1; k < WN; k++) {
        const float2 b = joint[k][row];
        const float t = fmaxf(a.x, b.x), at = t == ninf ? 0.0f : t;
        a.y = a.y * exp_near(a.x - at) + b.y * exp_near(b.x - at);
        a.x = t;
      }
      part[(int64_t)in * M + im * BM + row] = a;
    }
  }
};

// ---- few tokens -----------------------------------------------------------------------------------
// Bound by reading the weight (and writing its gradient): each wave takes kRows vocabulary entries at a
// time straight from memory in their own type (no fp16 planes, no transposed copies), V elements a lane,
// against up to NT rows of hidden kept in LDS as fp32. Ignored rows are zeros there. Where there are fewer
// rows than NT the last one stands for the missing, whose results go nowhere and whose factors are 0.
constexpr int kRows = 4;
template <typename T, int V> struct FewVec {
  typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T> struct FewVec<T, 1> {
  typedef T type;
};
template <typename T, int V>
__device__ __forceinline__ void few_load(const T* p, float (&x)[V]) {
  const typename FewVec<T, V>::type v = *reinterpret_cast<const typename FewVec<T, V>::type*>(p);
  if constexpr (V == 1) x[0] = (float)v;
  else {
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = (float)v[i];
  }
}
template <int V>
__device__ __forceinline__ void few_hidden(const float* p, float (&y)[V]) {
  if constexpr (V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 q = *reinterpret_cast<const float4*>(p + i);
      y[i] = q.x, y[i + 1] = q.y, y[i + 2] = q.z, y[i + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) y[i] = p[i];
  }
}
template <typename T>
__device__ __forceinline__ void few_stage(const T* h, int64_t ldh, int tokens, int dim,
                                          const int64_t* target, int64_t ignore, float* hs) {
  for (int i = threadIdx.x; i < tokens * dim; i += blockDim.x) {
    const int t = i / dim;
    hs[i] = target[t] != ignore ? (float)h[(int64_t)t * ldh + (i - t * dim)] : 0.0f;
  }
  __syncthreads();
}
// Which of a step's kRows x NT logits a lane ends with: number (r, t) = (n / NT, n % NT), n = lane >> kSame; its
// 2^kSame neighbours hold the same one.
template <int NT> struct FewLane {
  static constexpr int kCount = kRows * NT;
  static constexpr int kSame = kCount == 64 ? 0 : kCount == 32 ? 1 : kCount == 16 ? 2 : kCount == 8 ? 3 : 4;
};
template <int N, int D>
__device__ __forceinline__ void fold_lanes(float* acc, int lane) {
  if constexpr (N > 1) {
    const bool up = (lane & D) != 0;
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
      const float mine = up ? acc[i + N / 2] : acc[i], theirs = up ? acc[i] : acc[i + N / 2];
      acc[i] = mine + __shfl_xor(theirs, D, 64);
    }
  } else {
    acc[0] += __shfl_xor(acc[0], D, 64);
  }
  if constexpr (D > 1) fold_lanes<(N > 1 ? N / 2 : 1), D / 2>(acc, lane);
}
// The logits of entries v0 .. v0 + kRows - 1, one a lane (FewLane), without the bias. The sums over the
// wave's lanes halve the values held at each exchange: 63 exchanges for 64 values, where a sum apiece in
// all lanes takes 384, and what follows (exponentials) is done once instead of by all lanes.
template <typename T, int V, int NT>
__device__ __forceinline__ float few_logits(const T* w, int64_t ldw, int tokens, int dim, int vocab,
                                            const float* hs, int v0, int lane) {
  constexpr int N = kRows * NT;
  const T* p[kRows];
#pragma unroll
  for (int r = 0; r < kRows; r++) p[r] = w + (int64_t)(v0 + r < vocab ? v0 + r : vocab - 1) * ldw;
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; i++) acc[i] = 0.0f;
#pragma unroll 2
  for (int k = lane * V; k < dim; k += 64 * V) {
    float x[kRows][V];
#pragma unroll
    for (int r = 0; r < kRows; r++) few_load<T, V>(p[r] + k, x[r]);
#pragma unroll
    for (int t = 0; t < NT; t++) {
      float y[V];
      few_hidden<V>(hs + (t < tokens ? t : tokens - 1) * dim + k, y);
#pragma unroll
      for (int r = 0; r < kRows; r++)
#pragma unroll
        for (int i = 0; i < V; i++) acc[r * NT + t] = fmaf(x[r][i], y[i], acc[r * NT + t]);
    }
  }
  fold_lanes<N, 32>(acc, lane);
  return acc[0];
}

// Forward: each lane keeps the (maximum, sum of exponentials) of its token over its rows.
template <typename T, int V, int NT>
__global__ __launch_bounds__(1024) void few_kernel(const T* h, int64_t ldh, const T* w, int64_t ldw,
                                                   int tokens, int dim, int vocab, const float* bias,
                                                   const int64_t* target, int64_t ignore, float2* part,
                                                   float* picked) {
  extern __shared__ float hs[];  // [tokens][dim]
  __shared__ float2 joint[16][kRows * NT];
  few_stage<T>(h, ldh, tokens, dim, target, ignore, hs);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int n = lane >> FewLane<NT>::kSame, r = n / NT, t = n % NT;
  const float ninf = -__builtin_inff();
  const int64_t y = t < tokens ? target[t] : -1;
  float top = ninf, sum = 0.0f;
  for (int v0 = (blockIdx.x * waves + wave) * kRows; v0 < vocab; v0 += gridDim.x * waves * kRows) {
    float l = few_logits<T, V, NT>(w, ldw, tokens, dim, vocab, hs, v0, lane);
    const int v = v0 + r;
    if (v < vocab) {
      if (bias) l += bias[v];
      if (y == v) picked[t] = l;
      const float m = fmaxf(top, l), at = m == ninf ? 0.0f : m;
      sum = sum * exp_near(top - at) + exp_near(l - at);
      top = m;
    }
  }
  joint[wave][n] = make_float2(top, sum);
  __syncthreads();
  if ((int)threadIdx.x < tokens) {
    float m = ninf, s = 0.0f;
    for (int k = 0; k < waves; k++)
      for (int q = 0; q < kRows; q++) m = fmaxf(m, joint[k][q * NT + threadIdx.x].x);
    const float at = m == ninf ? 0.0f : m;
    for (int k = 0; k < waves; k++)
      for (int q = 0; q < kRows; q++) {
        const float2 b = joint[k][q * NT + threadIdx.x];
        s += b.y * exp_near(b.x - at);
      }
    part[(int64_t)blockIdx.x * tokens + threadIdx.x] = make_float2(m, s);
  }
}

// Backward, one read of the weight: dl [vocab, NT] in fp32 (for dh, NULL: not kept), the rows of dw, db.
template <typename T, int V, int NT>
__global__ __launch_bounds__(1024) void few_backward_kernel(const T* h, int64_t ldh, const T* w, int64_t ldw,
                                                            int tokens, int dim, int vocab,
                                                            const float* bias, const int64_t* target,
                                                            int64_t ignore, int reduction, const float* lse,
                                                            const float* grad, const Head* head, float* dl,
                                                            T* dw, float* db) {
  typedef typename FewVec<T, V>::type vec;
  constexpr int kSame = FewLane<NT>::kSame;
  extern __shared__ float hs[];  // [tokens][dim]
  few_stage<T>(h, ldh, tokens, dim, target, ignore, hs);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int n = lane >> kSame, r = n / NT, t = n % NT;
  // the lane's token: its factor (a bad target makes it NaN), lse and target
  float g = 0.0f, ls = 0.0f;
  int at = -1;
  if (t < tokens && target[t] != ignore) {
    g = reduction == SMQ_REDUCE_NONE ? grad[t]
        : reduction == SMQ_REDUCE_SUM ? *grad : (float)((double)*grad / head->count);
    ls = lse[t];
    const int64_t y = target[t];
    if (y >= 0 && y < vocab) at = (int)y;
    else g = __builtin_nanf("");
  }
  for (int v0 = (blockIdx.x * waves + wave) * kRows; v0 < vocab; v0 += gridDim.x * waves * kRows) {
    float l = few_logits<T, V, NT>(w, ldw, tokens, dim, vocab, hs, v0, lane);
    const int v = v0 + r;
    if (bias && v < vocab) l += bias[v];
    const float p = exp_near(l - ls) - (at == v ? 1.0f : 0.0f);
    const float d = g == 0.0f ? 0.0f : p * g;
    if (dl && v < vocab && (lane & ((1 << kSame) - 1)) == 0) dl[(int64_t)v0 * NT + n] = d;
    if (db) {
      float total = d;
#pragma unroll
      for (int q = NT / 2; q >= 1; q >>= 1) total += __shfl_xor(total, q << kSame, 64);
      if (t == 0 && v < vocab) db[v] = total;
    }
    if (!dw) continue;
    float u[kRows][NT];  // wave-uniform
#pragma unroll
    for (int i = 0; i < kRows; i++)
#pragma unroll
      for (int q = 0; q < NT; q++)
        u[i][q] = __builtin_bit_cast(
            float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, d), (i * NT + q) << kSame));
    for (int k = lane * V; k < dim; k += 64 * V) {
      float o[kRows][V];
#pragma unroll
      for (int i = 0; i < kRows; i++)
#pragma unroll
        for (int e = 0; e < V; e++) o[i][e] = 0.0f;
#pragma unroll
      for (int q = 0; q < NT; q++) {
        float y[V];
        few_hidden<V>(hs + (q < tokens ? q : tokens - 1) * dim + k, y);
#pragma unroll
        for (int i = 0; i < kRows; i++)
#pragma unroll
          for (int e = 0; e < V; e++) o[i][e] = fmaf(u[i][q], y[e], o[i][e]);
      }
#pragma unroll
      for (int i = 0; i < kRows; i++)
        if (v0 + i < vocab) {
          vec x;
          if constexpr (V == 1) x = (T)o[i][0];
          else {
#pragma unroll
            for (int e = 0; e < V; e++) x[e] = (T)o[i][e];
          }
          *reinterpret_cast<vec*>(dw + (int64_t)(v0 + i) * dim + k) = x;
        }
    }
  }
}

// dh of a chunk of the vocabulary: 64 V columns a workgroup, whose waves take turns at the chunk's
// entries and are summed in LDS -> part [chunk][tokens][ld].
template <typename T, int V, int NT>
__global__ __launch_bounds__(256) void few_dh_kernel(const float* dl, const T* w, int64_t ldw, int tokens,
                                                     int dim, int vocab, int64_t ld, float* part) {
  __shared__ float sh[3][64 * V];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int k = (blockIdx.x * 64 + lane) * V;
  const int first = (int)((int64_t)vocab * blockIdx.y / gridDim.y);
  const int last = (int)((int64_t)vocab * (blockIdx.y + 1) / gridDim.y);
  float acc[NT][V];
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int i = 0; i < V; i++) acc[t][i] = 0.0f;
  if (k < dim) {
#pragma unroll 4
    for (int v = first + wave; v < last; v += 4) {
      float x[V];
      few_load<T, V>(w + (int64_t)v * ldw + k, x);
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const float d = dl[(int64_t)v * NT + t];
#pragma unroll
        for (int i = 0; i < V; i++) acc[t][i] = fmaf(d, x[i], acc[t][i]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; t++) {
    __syncthreads();
    if (wave) {
#pragma unroll
      for (int i = 0; i < V; i++) sh[wave - 1][lane * V + i] = acc[t][i];
    }
    __syncthreads();
    if (wave == 0 && k < dim && t < tokens) {
      float* o = part + ((int64_t)blockIdx.y * tokens + t) * ld + k;
#pragma unroll
      for (int i = 0; i < V; i++)
        o[i] = (acc[t][i] + sh[0][lane * V + i]) + (sh[1][lane * V + i] + sh[2][lane * V + i]);
    }
  }
}

// ---- joining the blocks -------------------------------------------------------------------------
// A row's joined statistics: R rows a workgroup (a power of two), blockDim / R threads share a row's
// blocks. Returns in the first R threads. A target that is neither ignored nor in [0, vocab) gives NaN
// (nothing is read for it).
__device__ __forceinline__ void join_row(const float2* part, int blocks, int rows, int R, int m,
                                         const int64_t* target, int64_t ignore, int64_t vocab,
                                         const float* picked, float2* sh, float* lse, float* loss) {
  const float ninf = -__builtin_inff();
  const int share = blockDim.x / R;
  float top = ninf, sum = 0.0f;
  if (m < rows) {
#pragma unroll 4
    for (int k = threadIdx.x / R; k < blocks; k += share) {
      const float2 p = part[(int64_t)k * rows + m];
      const float t = fmaxf(top, p.x), at = t == ninf ? 0.0f : t;
      sum = sum * exp_near(top - at) + p.y * exp_near(p.x - at);
      top = t;
    }
  }
  sh[threadIdx.x] = make_float2(top, sum);
  for (int h = blockDim.x / 2; h >= R; h >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < h) {
      const float2 a = sh[threadIdx.x], b = sh[threadIdx.x + h];
      const float t = fmaxf(a.x, b.x), at = t == ninf ? 0.0f : t;
      sh[threadIdx.x] = make_float2(t, a.y * exp_near(a.x - at) + b.y * exp_near(b.x - at));
    }
  }
  if ((int)threadIdx.x >= R || m >= rows) return;
  const float2 a = sh[threadIdx.x];
  const float l = (a.x == ninf ? 0.0f : a.x) + logf(a.y);
  *lse = l;
  const int64_t y = target[m];
  *loss = y == ignore ? 0.0f : y >= 0 && y < vocab ? l - picked[m] : __builtin_nanf("");
}
// (live: the gathered rows' count, map their rows; the ignored ones get 0)
__global__ __launch_bounds__(256) void join_kernel(const float2* part, int blocks, int rows, int R,
                                                   const int64_t* target, int64_t ignore,
                                                   int64_t vocab, const float* picked, const int* map,
                                                   const int* live, float* lse, float* row_loss) {
  __shared__ float2 sh[256];
  const int m = blockIdx.x * R + (threadIdx.x & (R - 1)), n = map ? *live : rows;
  const int to = map && m < rows ? map[m] : m;
  join_row(part, blocks, n, R, m, target, ignore, vocab, picked, sh, lse + to, row_loss + to);
  if ((int)threadIdx.x < R && m >= n && m < rows) lse[to] = row_loss[to] = 0.0f;
}

// The loss over rows (fp64 sums in a fixed order) and the count of rows taking part, from each thread's
// sums; one workgroup of 16 waves.
__device__ __forceinline__ void finish_loss(double s, double c, int reduction, float* loss, Head* head) {
  s = wave_sum(s), c = wave_sum(c);
  __shared__ double a[16], b[16];
  if ((threadIdx.x & 63) == 0) a[threadIdx.x >> 6] = s, b[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = c = 0.0;
    for (int k = 0; k < 16; k++) s += a[k], c += b[k];
    head->count = c;
    if (reduction == SMQ_REDUCE_MEAN) *loss = (float)(s / c);
    if (reduction == SMQ_REDUCE_SUM) *loss = (float)s;
  }
}
__global__ __launch_bounds__(1024) void loss_kernel(const float* row_loss, const int64_t* target,
                                                    int64_t ignore, int rows, int reduction, float* loss,
                                                    Head* head) {
  double s = 0.0, c = 0.0;
  for (int m = threadIdx.x; m < rows; m += 1024) {
    s += (double)row_loss[m];
    c += target[m] != ignore ? 1.0 : 0.0;
    if (reduction == SMQ_REDUCE_NONE) loss[m] = row_loss[m];
  }
  finish_loss(s, c, reduction, loss, head);
}
// Both in one workgroup, where the partial statistics are few.
__global__ __launch_bounds__(1024) void join_loss_kernel(const float2* part, int blocks, int rows, int R,
                                                         const int64_t* target, int64_t ignore,
                                                         int64_t vocab, const float* picked, float* lse,
                                                         int reduction, float* loss, Head* head) {
  __shared__ float2 sh[1024];
  const int m = threadIdx.x & (R - 1);
  float l, value;
  join_row(part, blocks, rows, R, m, target, ignore, vocab, picked, sh, &l, &value);
  double s = 0.0, c = 0.0;
  if ((int)threadIdx.x < R && m < rows) {
    lse[m] = l;
    if (reduction == SMQ_REDUCE_NONE) loss[m] = value;
    s = (double)value;
    c = target[m] != ignore ? 1.0 : 0.0;
  }
  finish_loss(s, c, reduction, loss, head);
}

// ---- backward -----------------------------------------------------------------------------------
// One workgroup: the transposed weight's exponent (part: gw partial maxima, NULL: none), the rows' factors, and
// what comes off again in the epilogues. Ignored rows get 0 or are left out (Kept), rows whose gradient is not
// finite that gradient itself, rows whose target is no entry NaN. eh: the exponents of all rows of h (NULL: as
// they are).
__global__ __launch_bounds__(1024) void factor_kernel(const float* grad, const int64_t* target,
                                                      int64_t ignore, int rows, int64_t vocab, int reduction,
                                                      const Head* head, const float* part, int gw,
                                                      const float* lse, const int* eh, Kept kept, Row* out,
                                                      Head* fac) {
  __shared__ float sh[16];
  int exp_w = 0;
  if (part) {
    float top = 0.0f;
    for (int i = threadIdx.x; i < gw; i += 1024) top = fmaxf(top, part[i]);
    exp_w = plane_exponent(largest_of(top, sh));
  }
  // (no row takes part: no gradient)
  const float one = reduction == SMQ_REDUCE_NONE  ? 0.0f
                    : reduction == SMQ_REDUCE_SUM ? *grad
                    : head->count > 0.0           ? (float)((double)*grad / head->count) : 0.0f;
  auto size = [&](int m, float g) {  // the exponent of |g| |h|; g is finite and not 0
    int e;
    frexpf(g, &e);
    return e - (eh ? eh[m] : 0);
  };
  auto counts = [&](float g) { return g != 0.0f && fabsf(g) < __builtin_inff(); };
  const float none = (float)INT_MIN;
  float top = none;
  for (int m = threadIdx.x; m < rows; m += 1024) {
    const float g = reduction == SMQ_REDUCE_NONE ? grad[m] : one;
    if (target[m] != ignore && counts(g)) top = fmaxf(top, (float)size(m, g));
  }
  top = largest_of(top, sh);
  const int most = top == none ? 0 : (int)top;
  if (threadIdx.x == 0) {
    fac->exp_w = exp_w, fac->exp_dw = most;
    fac->scale_dh = ldexpf(1.0f / kDlScale, -exp_w);
    fac->scale_dw = ldexpf(1.0f / kDlScale, most < 141 ? most : 141);  // (finite: its products with 0 are 0)
  }
  auto row = [&](int m, bool keep) {
    const float g = !keep                                ? 0.0f
                    : target[m] < 0 || target[m] >= vocab ? __builtin_nanf("")
                    : reduction == SMQ_REDUCE_NONE        ? grad[m] : one;
    const int e = eh ? eh[m] : 0;
    int turned = e;
    if (!counts(g)) return Row{g, g, e, turned};
    const int k = most - size(m, g);
    if (eh) turned -= share_of(k);
    return Row{g, ldexpf(g, -most - turned), e, turned};
  };
  if (kept.map) {
    partition_rows(target, ignore, rows, &fac->rows, [&](int m, int at, bool keep) {
      kept.map[at] = m;
      if (keep) kept.target[at] = target[m], kept.lse[at] = lse[m], out[at] = row(m, true);
    });
    return;
  }
  for (int m = threadIdx.x; m < rows; m += 1024) out[m] = row(m, target[m] != ignore);
}

// dl of a piece from its logits, to `o` [rows, piece], without the rows' gradients, and transposed, with them
// (Row::t), to `ot` [piece, rows]; column sums (the bias' gradient) per block of rows.
template <bool PLANES, bool F32>
struct DlEpi {
  const int* ew;  // F32: the exponents of w's rows; PLANES: they come off the logits, as the rows' do
  const float* bias;
  const int64_t* target;
  const float* lse;
  const Row* row;
  const Head* fac;
  int64_t first;  // the piece's first vocabulary entry
  Mat o, ot;
  float* sums;  // [blocks][piece] or NULL
  template <int BM, int BN, int WM, int WN, int TM, int TN>
  __device__ __forceinline__ void finish(f32x16 (&acc)[TM][TN], float* stage, int m0, int n0, int M,
                                         int N, int im, int, int wm, int, int lane,
                                         int64_t batch) const {
    // a lane's four columns are the same in all of stage_out's rows
    int en[4] = {};
    float part[4] = {};  // of an entry 2^-k of the largest what stays with dl
    if constexpr (F32) {
      const int least = fac->exp_w;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        en[k] = ew[n0 + lane % (TN * 8) * 4 + k];  // (past N: its padding)
        const int d = en[k] - least;
        part[k] = ldexpf(1.0f, share_of(d) - d);
      }
    }
    Mat ot = this->ot;  // padded to whole k tiles of the rows there are
    const int tile = ot.fmt == kSplit ? 32 : 64;
    ot.pad = (M + tile - 1) / tile * tile;
    float* sum = sums ? sums + (int64_t)(im * WM + wm) * N : nullptr;
    const int back = fac->exp_dw - 14;
    stage_out<TM, TN, true>(
        acc, stage, m0, n0, M, N, lane, batch, o, ot, true, sum != nullptr,
        // the factor of the transposed copy, lse, the target's place in the piece (-1: elsewhere, -2: the row
        // has no gradient), its two exponents
        [&](int m) {
          const Row q = row[m];
          const int64_t at = target[m] - first;
          const int k = q.g == 0.0f ? -2 : at >= 0 && at < N ? (int)at : -1;
          return make_float4(q.t, lse[m], __builtin_bit_cast(float, k),
                             __builtin_bit_cast(float, (int)((unsigned)q.turned << 16 | (q.exp & 0xffff))));
        },
        [&](int, int n, float4 v, float4 row) {
          const int k0 = __builtin_bit_cast(int, row.z), at = k0 - n;
          const int er = (int16_t)__builtin_bit_cast(int, row.w);
          float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; k++) {
            float l = PLANES ? ldexpf(w[k], -(er + en[k])) : w[k];
            if (bias && n + k < N) l += bias[first + n + k];
            const float p = fmaf(exp_near(l - row.y), kDlScale, at == k ? -kDlScale : 0.0f);
            w[k] = k0 == -2 ? 0.0f : p;
          }
          return make_float4(w[0], w[1], w[2], w[3]);
        },
        [&](float4 v) {
          return F32 ? make_float4(v.x * part[0], v.y * part[1], v.z * part[2], v.w * part[3]) : v;
        },
        // p g from kDlScale p g 2^(-exp_dw - turned)
        [&](float v, float w) { return ldexpf(v, back + (__builtin_bit_cast(int, w) >> 16)); },
        [&](int n, float s) { sum[n] = s; });
  }
};

// (live: `per` blocks for each `high` of the rows there are)
__global__ __launch_bounds__(256) void bias_sum_kernel(const float* part, int blocks, int n, const int* live,
                                                       int high, int per, float* db) {
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v >= n) return;
  double s = 0.0;
  if (live) blocks = (*live + high - 1) / high * per;
  for (int k = 0; k < blocks; k++) s += (double)part[(int64_t)k * n + v];
  db[v] = (float)s;
}

// ---- host ---------------------------------------------------------------------------------------
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

struct Shape {
  int64_t tokens, dim, vocab, piece;
  int dtype;
  bool split() const { return dtype == SMQ_DTYPE_F32; }
  size_t size() const { return dtype == SMQ_DTYPE_F32 ? 4 : 2; }
};

constexpr int kMaxParts = 1024;
inline int absmax_grid(int64_t rows) { return (int)(rows < 4 * kMaxParts ? (rows + 3) / 4 : kMaxParts); }
// Entries of the array of a weight's exponents: the epilogues read whole tiles of columns.
inline size_t exponent_room(int64_t vocab) { return (size_t)vocab + 256; }

// A 16-bit tensor is an operand as it is when its rows are whole k tiles on 16-byte boundaries.
inline bool direct(const void* p, int64_t ld, int64_t cols, int dtype) {
  return dtype != SMQ_DTYPE_F32 && cols % 64 == 0 && ld % 8 == 0 && ld <= (1 << 21) &&
         (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}
inline int plane_fmt(int dtype) {
  return dtype == SMQ_DTYPE_F32 ? kSplit : dtype == SMQ_DTYPE_F16 ? kF16 : kBF16;
}
inline int out_fmt(int dtype) {
  return dtype == SMQ_DTYPE_F32 ? kF32 : dtype == SMQ_DTYPE_F16 ? kF16 : kBF16;
}
const Mat kNoMat = {nullptr, 0, 0, kNone, 0};

void layout(const void* src, int dtype, int64_t ld, int64_t rows, int64_t cols, const Exponents& exponent,
            const Exponents& turned, const int64_t* keep, int64_t skip, const Mat& d, const Mat& dt, hipStream_t st,
            const int* map = nullptr, const int* live = nullptr) {
  if (dtype == SMQ_DTYPE_F32)
    launch_layout((const float*)src, ld, 0, (int)rows, (int)cols, 1, exponent, turned, nullptr, keep, skip, d, dt,
                  st, map, live);
  else if (dtype == SMQ_DTYPE_F16)
    launch_layout((const _Float16*)src, ld, 0, (int)rows, (int)cols, 1, exponent, turned, nullptr, keep, skip, d, dt,
                  st, map, live);
  else
    launch_layout((const __bf16*)src, ld, 0, (int)rows, (int)cols, 1, exponent, turned, nullptr, keep, skip, d, dt,
                  st, map, live);
}

// The partial maxima of both inputs, absmax_grid of the tokens and of the vocabulary, and their rows' exponents.
template <typename T>
void maxima(const T* h, int64_t ldh, const T* w, int64_t ldw, const Shape& s, const int64_t* target,
            int64_t ignore, float* part, int* eh, int* ew, hipStream_t st) {
  const int gh = absmax_grid(s.tokens), gw = absmax_grid(s.vocab);
  hipLaunchKernelGGL(absmax_kernel<T>, dim3(gh + gw), dim3(256), 0, st, h, ldh, s.tokens, w, ldw, s.vocab,
                     (int)s.dim, target, ignore, gh, part, eh, ew);
}

// A gradient's product, of two planes or one of fp16.
void product(bool split, int tile, const Operand& A, const Operand& B, int kt, int shares, const StoreEpi& e,
             hipStream_t st) {
  if (split) launch<_Float16, true>(tile, A, B, kt, 1, 0, shares, e, st);
  else launch<_Float16, false>(tile, A, B, kt, 1, 0, shares, e, st);
}

// Which rows of h an operand is made of: those with keep[row] != skip (the others zeros; keep NULL: all), or
// with `map` the first *live that it names, gathered.
struct Pick {
  const int64_t* keep = nullptr;
  int64_t skip = 0;
  const int* map = nullptr;
  const int* live = nullptr;
};
// [rows, cols] in operand form: in place where it can be, else laid out in the workspace. `turned` (absent:
// fmt kNone) is written transposed along the way.
Operand operand(Arena& ws, const void* p, int64_t ld, int64_t rows, int64_t cols, const Shape& s,
                const Exponents& exponent, const Exponents& turned_exponent, const Pick& pick, const Mat& turned,
                bool run, hipStream_t st) {
  if (direct(p, ld, cols, s.dtype) && !pick.map) {
    if (run && turned.fmt != kNone)
      layout(p, s.dtype, ld, rows, cols, {}, turned_exponent, pick.keep, pick.skip, kNoMat, turned, st);
    return {p, ld, 0, (int)rows};
  }
  const int64_t to = operand_ld(cols, s.split());
  _Float16* q = ws.take<_Float16>((size_t)(rows * to));
  if (run)
    layout(p, s.dtype, ld, rows, cols, exponent, turned_exponent, pick.keep, pick.skip,
           {q, to, 0, plane_fmt(s.dtype), operand_pad(cols, s.split())}, turned, st, pick.map, pick.live);
  return {q, to, 0, (int)rows, pick.live};
}

int validate(const char* who, const void* h, int64_t ldh, const void* w, int64_t ldw, int dtype,
             const int64_t* target, int64_t tokens, int64_t dim, int64_t vocab, int reduction) {
  if (dtype != SMQ_DTYPE_F32 && dtype != SMQ_DTYPE_F16 && dtype != SMQ_DTYPE_BF16) {
    set_error("%s: dtype %d is not one of SMQ_DTYPE_F32/F16/BF16", who, dtype);
    return SMQ_ERR_INVALID;
  }
  if (tokens < 1 || dim < 1 || vocab < 1 || tokens > (1 << 20) || dim > (1 << 20) || vocab > (1 << 21)) {
    set_error("%s: needs 1 <= tokens, dim <= 2^20 and 1 <= vocab <= 2^21, got %lld, %lld, %lld", who,
              (long long)tokens, (long long)dim, (long long)vocab);
    return SMQ_ERR_INVALID;
  }
  if (tokens * vocab > ((int64_t)1 << 38)) {  // a launch has fewer than 2^32 threads
    set_error("%s: tokens * vocab is limited to 2^38, got %lld * %lld", who, (long long)tokens,
              (long long)vocab);
    return SMQ_ERR_INVALID;
  }
  if (!h || !w || !target || ldh < dim || ldw < dim) {
    set_error("%s: hidden, weight and target must be non-NULL, row pitches at least dim", who);
    return SMQ_ERR_INVALID;
  }
  if (reduction != SMQ_REDUCE_NONE && reduction != SMQ_REDUCE_MEAN && reduction != SMQ_REDUCE_SUM) {
    set_error("%s: reduction %d invalid", who, reduction);
    return SMQ_ERR_INVALID;
  }
  return SMQ_OK;
}

// float32 logits of up to 128 tokens, where both tensors are operands as they are: on the fp32 matrix
// instructions straight from them. Making planes of the weight moves it three times more; with more tokens
// the planes' fivefold rate pays for that (64 x 1024 x 30000: 275 us a step against 370 with planes, 128 tokens 363
// against 417, 256 tokens 520 against 488; 130 x 484 x 48351, whose rows would have to be copied, was 573 with
// the copies, 404 with planes).
bool in_place32(const void* p, int64_t ld, int64_t cols) {
  return cols % 32 == 0 && ld % 4 == 0 && ld <= (1 << 20) && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}
bool raw32(const void* h, int64_t ldh, const void* w, int64_t ldw, const Shape& s) {
  return s.split() && s.tokens <= 128 && in_place32(h, ldh, s.dim) && in_place32(w, ldw, s.dim);
}
// Whether the rows that take part are gathered: where a product is long against the copy of h (which float32
// makes anyway) and the launch that finds them. Training, none / 15 % / 40 % ignored, gathered against not:
// float32 512 x 768 x 30000 526 / 507 / 466 us against 518 / 513 / 504 (256 tokens 396 / 386 / 366, 387 /
// 390 / 388), fp16 1024 x 1024 x 32000 492 / 455 / 403 against 476 / 474 / 472 (768 x 30000 390 / 366 / 327,
// 376 / 373 / 372), fp16 2048 x 1024 x 50000 1323 / 1156 / 907 against 1310 / 1306 / 1298.
bool gathered(const Shape& s) {
  return s.tokens > 128 && s.tokens * s.vocab >= ((int64_t)1 << (s.split() ? 33 : 35)) / s.dim;
}
// The logits' product: by planes, one plane or raw float32, with the epilogue make(planes, float32).
template <typename F>
void logits(const Shape& s, bool raw, int tile, const Operand& A, const Operand& B, F make, hipStream_t st) {
  const int kt = operand_kt(s.dim, s.split());
  const std::true_type yes;
  const std::false_type no;
  if (raw) launch<Raw32, false>(tile, A, B, (int)(round_up(s.dim, 32) / 32), 1, 0, 1, make(no, yes), st);
  else if (s.dtype == SMQ_DTYPE_BF16) launch<__bf16, false>(tile, A, B, kt, 1, 0, 1, make(no, no), st);
  else if (s.dtype == SMQ_DTYPE_F16) launch<_Float16, false>(tile, A, B, kt, 1, 0, 1, make(no, no), st);
  else launch<_Float16, true>(tile, A, B, kt, 1, 0, 1, make(yes, yes), st);
}

// Few tokens: up to 16, hidden within 148 KiB of LDS; 0: not few.
constexpr size_t kFewLds = 148 * 1024;
struct Few {
  int nt, v;
  size_t lds;
  int threads, grid;
};
Few few_tokens(const void* w, int64_t ldw, const Shape& s) {
  if (s.tokens > 16) return {};
  const int nt = s.tokens <= 1 ? 1 : s.tokens <= 2 ? 2 : s.tokens <= 4 ? 4 : s.tokens <= 8 ? 8 : 16;
  const size_t lds = (size_t)s.tokens * s.dim * 4;
  if (lds > kFewLds) return {};
  const int size = (int)s.size();
  int v = 8 / size < 4 ? 4 : 8 / size;  // 4 elements a lane
  while (v > 1 && (s.dim % v || ldw % v || (reinterpret_cast<uintptr_t>(w) & (v * size - 1)))) v /= 2;
  // The more LDS a workgroup needs, the more waves share it; no more workgroups than are there at once
  // (each stages hidden anew), but small ones.
  const int threads = lds <= 16 * 1024 ? 256 : lds <= 40 * 1024 ? 512 : 1024;
  const int64_t rows = threads / 64 * kRows, all = (s.vocab + rows - 1) / rows;
  const int64_t fit = 160 * 1024 / (lds + 4096), room = 2048 / threads;
  const int64_t most = lds <= 16 * 1024 ? 2048 : 256 * (fit < room ? fit : room);
  return {nt, v, lds, threads, (int)(all < most ? all : most)};
}
int few_chunks(const Shape& s, const Few& f) {
  const int64_t cols = (s.dim + 64 * f.v - 1) / (64 * f.v);
  int64_t c = (1024 + cols - 1) / cols;
  if (c > s.vocab / 32) c = s.vocab / 32;
  return (int)(c < 1 ? 1 : c > 128 ? 128 : c);
}
// kernel<T, V, NT> for a plan's v and nt
template <typename T, int V, typename F>
void few_tokens_case(int nt, F f) {
  if (nt == 1) f(std::integral_constant<int, V>(), std::integral_constant<int, 1>());
  else if (nt == 2) f(std::integral_constant<int, V>(), std::integral_constant<int, 2>());
  else if (nt == 4) f(std::integral_constant<int, V>(), std::integral_constant<int, 4>());
  else if (nt == 8) f(std::integral_constant<int, V>(), std::integral_constant<int, 8>());
  else f(std::integral_constant<int, V>(), std::integral_constant<int, 16>());
}
template <typename T, typename F>
void few_case(const Few& p, F f) {
  if (p.v == 4) few_tokens_case<T, 4>(p.nt, f);
  else if (p.v == 2) few_tokens_case<T, 2>(p.nt, f);
  else few_tokens_case<T, 1>(p.nt, f);
}
// More than 64 KiB of dynamic LDS has to be asked for.
template <typename K>
void allow_lds(K kernel, size_t bytes) {
  if (bytes > 48 * 1024)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)kFewLds);
}
template <typename T>
void launch_few(const Few& p, const void* h, int64_t ldh, const void* w, int64_t ldw, const Shape& s,
                const float* bias, const int64_t* target, int64_t ignore, float2* part, float* picked,
                hipStream_t st) {
  few_case<T>(p, [&](auto v, auto nt) {
    auto kernel = few_kernel<T, v.value, nt.value>;
    allow_lds(kernel, p.lds);
    hipLaunchKernelGGL(kernel, dim3(p.grid), dim3(p.threads), p.lds, st, reinterpret_cast<const T*>(h), ldh,
                       reinterpret_cast<const T*>(w), ldw, (int)s.tokens, (int)s.dim, (int)s.vocab, bias,
                       target, ignore, part, picked);
  });
}
template <typename T>
void launch_few_backward(const Few& p, const void* h, int64_t ldh, const void* w, int64_t ldw, const Shape& s,
                         const float* bias, const int64_t* target, int64_t ignore, int reduction,
                         const float* lse, const float* grad, const Head* head, float* dl, float* part,
                         int64_t ld, int chunks, void* dh, void* dw, float* db, hipStream_t st) {
  few_case<T>(p, [&](auto v, auto nt) {
    auto kernel = few_backward_kernel<T, v.value, nt.value>;
    allow_lds(kernel, p.lds);
    hipLaunchKernelGGL(kernel, dim3(p.grid), dim3(p.threads), p.lds, st, reinterpret_cast<const T*>(h), ldh,
                       reinterpret_cast<const T*>(w), ldw, (int)s.tokens, (int)s.dim, (int)s.vocab, bias,
                       target, ignore, reduction, lse, grad, head, dl, reinterpret_cast<T*>(dw), db);
    if (dh)
      hipLaunchKernelGGL((few_dh_kernel<T, v.value, nt.value>),
                         dim3((unsigned)((s.dim + 64 * p.v - 1) / (64 * p.v)), chunks), dim3(256), 0, st, dl,
                         reinterpret_cast<const T*>(w), ldw, (int)s.tokens, (int)s.dim, (int)s.vocab, ld, part);
  });
  if (dh) {
    const StoreEpi se = {1.0f, 0.0f, nullptr, kNoMat, {dh, s.dim, 0, out_fmt(s.dtype), 0}, kNoMat, 0, 0, 0.0f};
    launch_split_sum(part, ld, s.tokens * ld, chunks, 0, (int)s.tokens, (int)s.dim, 1, 0, se, st);
  }
}

// Lays the workspace out; enqueues when `run`. Returns the bytes used.
size_t forward(const void* h, int64_t ldh, const void* w, int64_t ldw, const Shape& s,
                    const int64_t* target, const float* bias, int64_t ignore, int reduction,
                    float* loss, float* lse, Head* head, void* ws, bool run, hipStream_t st) {
  Arena a(ws);
  const int tile = plan_product(s.tokens, s.vocab, operand_kt(s.dim, s.split()), 1, 0, false).tile;
  const TileShape ts = shape_of(tile);
  const int64_t tn = (s.vocab + ts.bn - 1) / ts.bn;
  const Few few = few_tokens(w, ldw, s);
  const int blocks = few.nt ? few.grid : (int)tn;
  float2* part = a.take<float2>((size_t)blocks * s.tokens);
  float* picked = a.take<float>(s.tokens);
  float* rows = a.take<float>(s.tokens);
  int *eh = nullptr, *ew = nullptr;
  const bool raw = raw32(h, ldh, w, ldw, s), gather = !few.nt && gathered(s);
  if (s.split() && !few.nt && !raw) {
    float* top = a.take<float>(2 * kMaxParts);
    eh = a.take<int>(s.tokens), ew = a.take<int>(exponent_room(s.vocab));
    if (run) maxima((const float*)h, ldh, (const float*)w, ldw, s, target, ignore, top, eh, ew, st);
  }
  Kept kept = {};
  Pick pick;
  if (gather) {
    kept = {a.take<int>(s.tokens), a.take<int64_t>(s.tokens), eh ? a.take<int>(s.tokens) : nullptr, nullptr};
    pick.map = kept.map, pick.live = &head->rows;
    if (run)
      hipLaunchKernelGGL(gather_kernel, dim3(1), dim3(1024), 0, st, target, ignore, (int)s.tokens, eh, head, kept);
    eh = kept.exp;
  }
  const int64_t* at = gather ? kept.target : target;
  if (few.nt) {
    if (run) {
      if (s.dtype == SMQ_DTYPE_F32) launch_few<float>(few, h, ldh, w, ldw, s, bias, target, ignore, part, picked, st);
      else if (s.dtype == SMQ_DTYPE_F16) launch_few<_Float16>(few, h, ldh, w, ldw, s, bias, target, ignore, part, picked, st);
      else launch_few<__bf16>(few, h, ldh, w, ldw, s, bias, target, ignore, part, picked, st);
    }
  } else {
    const Operand A = raw ? Operand{h, 2 * ldh, 0, (int)s.tokens}
                          : operand(a, h, ldh, s.tokens, s.dim, s, eh ? Exponents{eh, 1} : Exponents(), {}, pick, kNoMat, run, st);
    const Operand B = raw ? Operand{w, 2 * ldw, 0, (int)s.vocab}
                          : operand(a, w, ldw, s.vocab, s.dim, s, ew ? Exponents{ew, 1} : Exponents(), {}, {}, kNoMat, run, st);
    if (run)
      logits(s, raw, tile, A, B,
             [&](auto planes, auto) { return SoftmaxEpi<planes.value>{eh, ew, bias, at, part, picked}; }, st);
  }
  if (run) {
    int per = 1;
    if (!gather && s.tokens <= 1024 && s.tokens * blocks <= 16384) {
      while (per < s.tokens) per *= 2;
      hipLaunchKernelGGL(join_loss_kernel, dim3(1), dim3(1024), 0, st, part, blocks, (int)s.tokens, per,
                         target, ignore, s.vocab, picked, lse, reduction, loss, head);
    } else {
      per = s.tokens >= 2048 ? 16 : s.tokens >= 256 ? 4 : 1;
      hipLaunchKernelGGL(join_kernel, dim3((unsigned)((s.tokens + per - 1) / per)), dim3(256), 0, st, part,
                         blocks, (int)s.tokens, per, at, ignore, s.vocab, picked, pick.map, pick.live, lse, rows);
      hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(1024), 0, st, rows, target, ignore, (int)s.tokens,
                         reduction, loss, head);
    }
  }
  return a.used;
}

int64_t default_piece(const Shape& s) {
  const int64_t planes = s.split() ? 2 : 1;
  const int64_t per = 2 * planes * (2 * round_up(s.tokens, 64) + round_up(s.dim, 64));
  int64_t p = (int64_t)(kPieceBytes / per);
  p = p / 256 * 256;
  return p < 256 ? 256 : p > (1 << 20) ? 1 << 20 : p;
}

size_t backward(const void* h, int64_t ldh, const void* w, int64_t ldw, Shape s, const int64_t* target,
                const float* bias, int64_t ignore, int reduction, const float* lse, const Head* head,
                const float* grad, void* dh, void* dw, float* db, void* ws, bool run, hipStream_t st) {
  Arena a(ws);
  if (const Few few = few_tokens(w, ldw, s); few.nt) {
    const int chunks = few_chunks(s, few);
    const int64_t ld = round_up(s.dim, 4);
    float* dl = dh ? a.take<float>((size_t)(s.vocab * few.nt)) : nullptr;
    float* part = dh ? a.take<float>((size_t)(chunks * s.tokens * ld)) : nullptr;
    if (run) {
      auto go = [&](auto type) {
        launch_few_backward<decltype(type)>(few, h, ldh, w, ldw, s, bias, target, ignore, reduction, lse, grad,
                                            head, dl, part, ld, chunks, dh, dw, db, st);
      };
      if (s.dtype == SMQ_DTYPE_F32) go(0.0f);
      else if (s.dtype == SMQ_DTYPE_F16) go((_Float16)0);
      else go((__bf16)0.0f);
    }
    return a.used;
  }
  const bool sp = s.split();
  const int fmt = sp ? kSplit : kF16;  // the gradient products' operands
  if (s.piece <= 0) s.piece = default_piece(s);
  if (s.piece > s.vocab) s.piece = s.vocab;
  const int64_t pieces = (s.vocab + s.piece - 1) / s.piece;
  Row* row = a.take<Row>(s.tokens);
  Head* fac = a.take<Head>(1);
  const bool gather = gathered(s);
  Kept kept = {};
  Pick pick;
  pick.keep = target, pick.skip = ignore;
  if (gather) {
    kept = {a.take<int>(s.tokens), a.take<int64_t>(s.tokens), nullptr, a.take<float>(s.tokens)};
    pick = Pick();
    pick.map = kept.map, pick.live = &fac->rows;
  }
  const bool raw = raw32(h, ldh, w, ldw, s), scaled = s.dtype != SMQ_DTYPE_F16;
  // exponents of h's rows, and of float32 w's
  int* eh = scaled ? a.take<int>(s.tokens) : nullptr;
  int* ew = sp ? a.take<int>(exponent_room(s.vocab)) : nullptr;
  float* top = nullptr;
  if (scaled) {
    top = a.take<float>(2 * kMaxParts);
    if (run && sp) maxima((const float*)h, ldh, (const float*)w, ldw, s, target, ignore, top, eh, ew, st);
    else if (run)
      maxima((const __bf16*)h, ldh, (const __bf16*)w, ldw, s, target, ignore, top, eh, nullptr, st);
  }
  const Exponents turned_eh = scaled ? Exponents{&row->turned, 4} : Exponents();
  if (run)
    hipLaunchKernelGGL(factor_kernel, dim3(1), dim3(1024), 0, st, grad, target, ignore,
                       (int)s.tokens, s.vocab, reduction, head, top ? top + absmax_grid(s.tokens) : nullptr,
                       absmax_grid(s.vocab), lse, eh, kept, row, fac);
  // h, and transposed the operand of dw. Ignored rows are left out or zeros, whatever they hold (where h is
  // read in place its ignored rows' logits are not used).
  const int64_t ldt = operand_ld(s.tokens, sp);
  const int padt = operand_pad(s.tokens, sp);
  _Float16* ht = dw ? a.take<_Float16>((size_t)(s.dim * ldt)) : nullptr;
  const Mat turned_h = dw ? Mat{ht, ldt, 0, fmt, padt} : kNoMat;
  if (run && raw && dw)  // (not gathered)
    layout(h, s.dtype, ldh, s.tokens, s.dim, {}, turned_eh, target, ignore, kNoMat, turned_h, st);
  const Operand A =
      raw ? Operand{h, 2 * ldh, 0, (int)s.tokens}
          : operand(a, h, ldh, s.tokens, s.dim, s, sp ? Exponents{&row->exp, 4} : Exponents(), turned_eh, pick,
                    turned_h, run, st);
  const int64_t ldp = operand_ld(s.piece, sp);
  _Float16* dl = a.take<_Float16>((size_t)(s.tokens * ldp));
  _Float16* dlt = a.take<_Float16>((size_t)(s.piece * ldt));
  _Float16* wt = dh ? a.take<_Float16>((size_t)(s.dim * ldp)) : nullptr;
  const int tile_l = plan_product(s.tokens, s.piece, operand_kt(s.dim, sp), 1, 0, false).tile;
  const int row_blocks = (int)((s.tokens + shape_of(tile_l).bm - 1) / shape_of(tile_l).bm) * shape_of(tile_l).wm;
  float* sums = db ? a.take<float>((size_t)row_blocks * s.piece) : nullptr;
  const Shared dp = plan_product(s.tokens, s.dim, operand_kt(s.piece, sp), 1, 0, true);
  const int tile_dh = dp.tile, shares = dp.shares;
  const int64_t ldacc = round_up(s.dim, 4);
  const bool whole = pieces == 1 && shares == 1 && !gather;
  float* accum = dh && !whole ? a.take<float>((size_t)(shares * s.tokens * ldacc)) : nullptr;
  const size_t wsize = s.size();
  const size_t mark = a.used;
  size_t most = mark;
  for (int64_t i = 0; i < pieces; i++) {
    a.used = mark;
    const int64_t v0 = i * s.piece, n = s.vocab - v0 < s.piece ? s.vocab - v0 : s.piece;
    const char* wp = reinterpret_cast<const char*>(w) + (size_t)(v0 * ldw) * wsize;
    const int padn = operand_pad(n, sp);
    const Mat turned_w = dh ? Mat{wt, ldp, 0, fmt, padn} : kNoMat;
    const Exponents of_w = ew ? Exponents{ew + v0, 1} : Exponents();
    const Exponents turned_ew = ew ? Exponents{ew + v0, 1, &fac->exp_w} : Exponents{scaled ? &fac->exp_w : nullptr, 0};
    if (run && raw && dh) layout(wp, s.dtype, ldw, n, s.dim, {}, turned_ew, nullptr, 0, kNoMat, turned_w, st);
    const Operand B = raw ? Operand{wp, 2 * ldw, 0, (int)n}
                          : operand(a, wp, ldw, n, s.dim, s, of_w, turned_ew, {}, turned_w, run, st);
    if (a.used > most) most = a.used;
    if (!run) continue;
    logits(s, raw, tile_l, A, B, [&](auto planes, auto f32) {
      return DlEpi<planes.value, f32.value>{ew ? ew + v0 : nullptr, bias, gather ? kept.target : target,
                                            gather ? kept.lse : lse, row, fac, v0,
                                            {dl, ldp, 0, fmt, padn}, {dlt, ldt, 0, fmt, padt}, sums};
    }, st);
    if (db)
      hipLaunchKernelGGL(bias_sum_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, sums,
                         row_blocks, (int)n, pick.live, shape_of(tile_l).bm, shape_of(tile_l).wm, db + v0);
    if (dh) {
      const Operand L = {dl, ldp, 0, (int)s.tokens, pick.live}, W = {wt, ldp, 0, (int)s.dim};
      StoreEpi se = {1.0f, 1.0f, whole ? &fac->scale_dh : nullptr, kNoMat, kNoMat, kNoMat, 0, s.tokens * ldacc, 0.0f};
      se.o = whole ? Mat{dh, s.dim, 0, out_fmt(s.dtype), 0} : Mat{accum, ldacc, 0, kF32, 0};
      if (i > 0) se.src = se.o;
      if (whole) se.rows = &row->g, se.row_step = 4;
      product(sp, tile_dh, L, W, operand_kt(n, sp), shares, se, st);
    }
    if (dw) {
      const Operand L = {dlt, ldt, 0, (int)n, nullptr, pick.live}, H = {ht, ldt, 0, (int)s.dim};
      StoreEpi se = {1.0f, 0.0f, &fac->scale_dw, kNoMat, kNoMat, kNoMat, 0, 0, 0.0f};
      se.o = {reinterpret_cast<char*>(dw) + (size_t)(v0 * s.dim) * wsize, s.dim, 0, out_fmt(s.dtype), 0};
      const int kt = operand_kt(s.tokens, sp);
      product(sp, plan_product(n, s.dim, kt, 1, 0, false).tile, L, H, kt, 1, se, st);
    }
  }
  if (run && dh && !whole) {
    StoreEpi se = {1.0f, 0.0f, &fac->scale_dh, kNoMat, {dh, s.dim, 0, out_fmt(s.dtype), 0}, kNoMat, 0, 0, 0.0f};
    se.map = pick.map, se.live = pick.live, se.rows = &row->g, se.row_step = 4;
    launch_split_sum(accum, ldacc, s.tokens * ldacc, shares, 0, (int)s.tokens, (int)s.dim, 1, 0, se, st);
  }
  return most;
}

}  // namespace ce
}  // namespace smq

using namespace smq;
using namespace smq::ce;

extern "C" {

size_t smq_linear_ce_workspace_bytes(const void* hidden, int64_t hidden_ld, const void* weight,
                                     int64_t weight_ld, int dtype, int64_t tokens, int64_t dim,
                                     int64_t vocab, int64_t piece, int grad_flags) {
  const int64_t none = 0;
  if (validate("linear_ce_workspace_bytes", hidden, hidden_ld, weight, weight_ld, dtype, &none, tokens,
               dim, vocab, SMQ_REDUCE_SUM) != SMQ_OK)
    return 0;
  const int all = SMQ_CE_GRAD_HIDDEN | SMQ_CE_GRAD_WEIGHT | SMQ_CE_GRAD_BIAS;
  if (piece < 0 || piece > (1 << 20) || (grad_flags & ~all)) {
    set_error("linear_ce_workspace_bytes: needs 0 <= piece <= 2^20 and flags of SMQ_CE_GRAD_*, got %lld, %d",
              (long long)piece, grad_flags);
    return 0;
  }
  const Shape s = {tokens, dim, vocab, piece, dtype};
  Head* head = nullptr;
  if (!grad_flags)
    return forward(hidden, hidden_ld, weight, weight_ld, s, nullptr, nullptr, 0, 0, nullptr, nullptr,
                   head, nullptr, false, nullptr) + 256;
  char mark[1];
  return backward(hidden, hidden_ld, weight, weight_ld, s, nullptr, nullptr, 0, 0, nullptr, head,
                  nullptr, grad_flags & SMQ_CE_GRAD_HIDDEN ? mark : nullptr,
                  grad_flags & SMQ_CE_GRAD_WEIGHT ? mark : nullptr,
                  grad_flags & SMQ_CE_GRAD_BIAS ? reinterpret_cast<float*>(mark) : nullptr, nullptr,
                  false, nullptr) + 256;
}

int smq_linear_ce_forward(const void* hidden, int64_t hidden_ld, const void* weight, int64_t weight_ld,
                          int dtype, const int64_t* target, const float* bias, int64_t tokens,
                          int64_t dim, int64_t vocab, int64_t ignore_index, int reduction, float* loss,
                          float* lse, void* head, void* workspace, size_t workspace_bytes,
                          void* stream) {
  const int rc = validate("linear_ce_forward", hidden, hidden_ld, weight, weight_ld, dtype, target,
                          tokens, dim, vocab, reduction);
  if (rc != SMQ_OK) return rc;
  if (!loss || !lse || !head) {
    set_error("linear_ce_forward: loss, lse and head must be non-NULL");
    return SMQ_ERR_INVALID;
  }
  const size_t need = smq_linear_ce_workspace_bytes(hidden, hidden_ld, weight, weight_ld, dtype,
                                                    tokens, dim, vocab, 0, 0);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)) {
    set_error("linear_ce_forward: workspace: need %zu bytes on a 16-byte boundary, got %zu", need, workspace_bytes);
    return SMQ_ERR_WORKSPACE;
  }
  const Shape s = {tokens, dim, vocab, 0, dtype};
  forward(hidden, hidden_ld, weight, weight_ld, s, target, bias, ignore_index, reduction, loss, lse,
          reinterpret_cast<Head*>(head), workspace, true, reinterpret_cast<hipStream_t>(stream));
  return check_launch("linear_ce_forward");
}

int smq_linear_ce_backward(const void* hidden, int64_t hidden_ld, const void* weight,
                           int64_t weight_ld, int dtype, const int64_t* target, const float* bias,
                           int64_t tokens, int64_t dim, int64_t vocab, int64_t ignore_index,
                           int reduction, const float* lse, const void* head, const float* grad_loss,
                           void* grad_hidden, void* grad_weight, float* grad_bias, int64_t piece,
                           void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = validate("linear_ce_backward", hidden, hidden_ld, weight, weight_ld, dtype, target,
                          tokens, dim, vocab, reduction);
  if (rc != SMQ_OK) return rc;
  if (!lse || !head || !grad_loss || (!grad_hidden && !grad_weight && !grad_bias) || piece < 0 ||
      piece > (1 << 20)) {
    set_error("linear_ce_backward: lse, head, grad_loss and one gradient must be non-NULL, "
              "0 <= piece <= 2^20");
    return SMQ_ERR_INVALID;
  }
  const int flags = (grad_hidden ? SMQ_CE_GRAD_HIDDEN : 0) | (grad_weight ? SMQ_CE_GRAD_WEIGHT : 0) |
                    (grad_bias ? SMQ_CE_GRAD_BIAS : 0);
  const size_t need = smq_linear_ce_workspace_bytes(hidden, hidden_ld, weight, weight_ld, dtype,
                                                    tokens, dim, vocab, piece, flags);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)) {
    set_error("linear_ce_backward: workspace: need %zu bytes on a 16-byte boundary, got %zu", need, workspace_bytes);
    return SMQ_ERR_WORKSPACE;
  }
  if ((reinterpret_cast<uintptr_t>(grad_hidden) | reinterpret_cast<uintptr_t>(grad_weight)) & 15) {
    set_error("linear_ce_backward: gradients have to start on 16-byte boundaries");
    return SMQ_ERR_INVALID;
  }
  const Shape s = {tokens, dim, vocab, piece, dtype};
  backward(hidden, hidden_ld, weight, weight_ld, s, target, bias, ignore_index, reduction, lse,
           reinterpret_cast<const Head*>(head), grad_loss, grad_hidden, grad_weight, grad_bias,
           workspace, true, reinterpret_cast<hipStream_t>(stream));
  return check_launch("linear_ce_backward");
}

}  // extern "C"
