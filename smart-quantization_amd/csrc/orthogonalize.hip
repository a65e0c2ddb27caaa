// orthogonalize.hip — the nearest semi-orthogonal matrix to an update, by Newton-Schulz products.
//
//   X = G / (|G|_F + eps), turned so that its m rows are the shorter side;
//   steps times:  A = X X^T,  B = b A + c A A,  X <- a X + B X     (an odd polynomial of the singular values)
//
// Every product runs on gemm_nt.h with both operands contiguous along k: A and B are symmetric, so
// only their tiles on and above the diagonal are computed (the epilogue writes both), and X is kept
// both ways round, as [m, n] (operand of A) and as [n, m] (operand of B X); the last product's
// epilogue writes both again. 3 m^2 n + m^3 operations a step instead of 4 m^2 n + 2 m^3.
//
// Rounding. What is stored between products is fp16 at a power-of-two scale that keeps it in range
// (the host bounds the singular values step by step), as two planes (hi + lo, 23 bits, three products
// a multiply-add): float32-class. One plane would be off by 0.15 % on Gaussian matrices and by 1-4 %
// where a few strong directions hide the rest (the polynomial raises the small singular values 3.4-fold
// a step, and with them the error the large ones leave there); one bf16 plane by 1-11 %. The last two
// steps no longer raise anything: for bf16 results, themselves off by 0.17 %, steps from the fourth on
// keep one plane (0.05-0.2 % off), at a third of the operations.
#include <math.h>

#include "gemm_nt.h"

namespace smq {
namespace ortho {
using namespace gemm;

constexpr int kParts = 256;
constexpr int kPlaneSteps = 3;  // bf16 results: steps that keep two planes

// ---- the norm -----------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void square_sum_kernel(const T* x, int64_t ld, int64_t batch_stride,
                                                         int rows, int cols, double* part) {
  constexpr int V = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(V)));
  const T* p = x + blockIdx.y * batch_stride;
  const bool wide = (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % V == 0;
  const int whole = wide ? cols / V * V : 0;
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
// factor[batch] = scale / (norm + eps)
__global__ __launch_bounds__(64) void norm_kernel(const double* part, int n, double eps, double scale,
                                                  float* factor) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 64) s += part[blockIdx.x * n + i];
  s = wave_sum(s);
  if (threadIdx.x == 0) factor[blockIdx.x] = (float)(scale / (sqrt(s) + eps));
}

// ---- host ---------------------------------------------------------------------------------------
struct Plan {
  int64_t batch, m, n;
  bool turned;
  int dtype, steps;
  double a, b, c;
};

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

// Shares of the k range where the tiles alone leave CUs idle: at least 8 k tiles a share, at most 8
// shares (their sum costs a pass over all of them).
int shares_for(int64_t wgs, int kt) {
  int64_t k = 256 / (wgs < 1 ? 1 : wgs);
  if (k > kt / 8) k = kt / 8;
  return (int)(k < 1 ? 1 : k > 8 ? 8 : k);
}

struct Buffers {
  _Float16 *x[2], *xt[2], *gram, *poly;
  float* part;  // shares of a product split over k
};

// One product, split over k or not.
void product(bool split, const Operand& A, const Operand& B, int kt, int batch, const StoreEpi& e,
             const Buffers& w, bool run, size_t* need, hipStream_t st) {
  const int tile = choose_tile(A.rows, B.rows, batch, e.tri);
  const int shares = tile == kT256 ? 1 : shares_for(batch * tile_count(A.rows, B.rows, tile, e.tri), kt);
  const int64_t ld = round_up(B.rows, 4), per = (int64_t)A.rows * ld;
  if (shares > 1 && need) {
    const size_t floats = (size_t)shares * batch * per;
    if (floats > *need) *need = floats;
  }
  if (!run) return;
  StoreEpi d = e;
  if (shares > 1) {
    d = {1.0f, 0.0f, nullptr, {}, {w.part, ld, per, kF32, 0}, {}, 0, batch * per};
  }
  if (split) launch<_Float16, true>(tile, A, B, kt, batch, e.tri, shares, d, st);
  else launch<_Float16, false>(tile, A, B, kt, batch, e.tri, shares, d, st);
  if (shares > 1)
    hipLaunchKernelGGL(split_sum_kernel,
                       dim3((unsigned)((B.rows + 63) / 64), (unsigned)((A.rows + 63) / 64), batch),
                       dim3(256), 0, st, w.part, ld, batch * per, shares, per, A.rows, B.rows,
                       e.ot.fmt != kNone ? 1 : 0, e);
}

// Small stacks, bound by their launches, keep two planes throughout: it costs them nothing.
bool planes_at(const Plan& p, int step) {
  return p.dtype != SMQ_DTYPE_BF16 || step < kPlaneSteps ||
         (double)p.batch * p.m * p.m * p.n < (double)(1 << 28);
}

template <typename T>
void first_layout(const Plan& p, const T* g, int64_t ld, int64_t stride, double eps, double scale,
                  double* part, float* factor, const Mat& x, const Mat& xt, hipStream_t st) {
  const int rows = (int)(p.turned ? p.n : p.m), cols = (int)(p.turned ? p.m : p.n);
  const int grid = rows < 4 * kParts ? (rows + 3) / 4 : kParts;
  hipLaunchKernelGGL(square_sum_kernel<T>, dim3(grid, (unsigned)p.batch), dim3(256), 0, st, g, ld, stride,
                     rows, cols, part);
  hipLaunchKernelGGL(norm_kernel, dim3((unsigned)p.batch), dim3(64), 0, st, part, grid, eps, scale, factor);
  launch_layout(g, ld, stride, rows, cols, (int)p.batch, nullptr, factor, nullptr, 0, p.turned ? xt : x,
                p.turned ? x : xt, st);
}

// The products of one step of either format, walked without a launch: the floats their shares need.
size_t share_floats(const Plan& p) {
  size_t need = 0;
  for (int s = 0; s < 2; s++) {
    const bool sp = s == 0;
    const Operand X = {nullptr, 0, 0, (int)p.m}, XT = {nullptr, 0, 0, (int)p.n};
    StoreEpi e = {};
    e.tri = 1;
    product(sp, X, X, operand_kt(p.n, sp), (int)p.batch, e, {}, false, &need, nullptr);
    product(sp, X, X, operand_kt(p.m, sp), (int)p.batch, e, {}, false, &need, nullptr);
    e.tri = 0;
    product(sp, X, XT, operand_kt(p.m, sp), (int)p.batch, e, {}, false, &need, nullptr);
  }
  return need;
}

// Lays the workspace out and, when `run`, enqueues the call. Returns the bytes used.
size_t enqueue(const Plan& p, const void* g, int64_t ld, int64_t stride, void* y, double eps, void* ws,
               bool run, hipStream_t st) {
  Arena a(ws);
  const int64_t bt = p.batch, m = p.m, n = p.n;
  const int batch = (int)bt;
  // room for the larger of the two formats; two of each X (a step reads one and writes the other)
  const int64_t ldn = 2 * round_up(n, 64), ldm = 2 * round_up(m, 64);
  double* part = a.take<double>((size_t)(bt * kParts));
  float* factor = a.take<float>((size_t)bt);
  Buffers w;
  for (int k = 0; k < 2; k++) {
    w.x[k] = a.take<_Float16>((size_t)(bt * m * ldn));
    w.xt[k] = a.take<_Float16>((size_t)(bt * n * ldm));
  }
  w.gram = a.take<_Float16>((size_t)(bt * m * ldm));
  w.poly = a.take<_Float16>((size_t)(bt * m * ldm));
  w.part = a.take<float>(share_floats(p));
  if (!run) return a.used;

  auto mat = [&](_Float16* q, int64_t cols, int64_t rows, bool planes) {
    const int64_t l = operand_ld(cols, planes);
    return Mat{q, l, rows * l, planes ? kSplit : kF16, operand_pad(cols, planes)};
  };
  auto op = [](const Mat& q, int64_t rows) { return Operand{q.p, q.ld, q.batch, (int)rows}; };
  const Mat none = {nullptr, 0, 0, kNone, 0};
  const int out = p.dtype == SMQ_DTYPE_F32 ? kF32 : p.dtype == SMQ_DTYPE_F16 ? kF16 : kBF16;
  double top = 1.0;  // bound of X's singular values
  int ex = exponent_for(top);
  Mat X = mat(w.x[0], n, m, planes_at(p, 0)), XT = mat(w.xt[0], m, n, planes_at(p, 0));
  const double scale = ldexp(1.0, ex);
  if (p.dtype == SMQ_DTYPE_F32)
    first_layout(p, (const float*)g, ld, stride, eps, scale, part, factor, X, XT, st);
  else if (p.dtype == SMQ_DTYPE_F16)
    first_layout(p, (const _Float16*)g, ld, stride, eps, scale, part, factor, X, XT, st);
  else
    first_layout(p, (const __bf16*)g, ld, stride, eps, scale, part, factor, X, XT, st);
  for (int i = 0; i < p.steps; i++) {
    const bool last = i + 1 == p.steps, sp = planes_at(p, i);
    const double q = top * top;
    const int ea = exponent_for(q), eb = exponent_for(fabs(p.b) * q + fabs(p.c) * q * q);
    const Mat A = mat(w.gram, m, m, sp), P = mat(w.poly, m, m, sp);
    // A = X X^T
    StoreEpi e = {(float)ldexp(1.0, ea - 2 * ex), 0.0f, nullptr, none, A, A, 1, 0};
    product(sp, op(X, m), op(X, m), operand_kt(n, sp), batch, e, w, true, nullptr, st);
    // B = b A + c A A
    e = {(float)ldexp(p.c, eb - 2 * ea), (float)ldexp(p.b, eb - ea), nullptr, A, P, P, 1, 0};
    product(sp, op(A, m), op(A, m), operand_kt(m, sp), batch, e, w, true, nullptr, st);
    // X <- a X + B X
    top = grown(p, top);
    const int ey = last ? 0 : exponent_for(top);
    Mat X2, XT2;
    if (!last) {
      const bool np = planes_at(p, i + 1);
      X2 = mat(w.x[(i + 1) & 1], n, m, np), XT2 = mat(w.xt[(i + 1) & 1], m, n, np);
    } else {
      const Mat Y = {y, p.turned ? m : n, m * n, out, 0};
      X2 = p.turned ? none : Y, XT2 = p.turned ? Y : none;
    }
    e = {(float)ldexp(1.0, ey - eb - ex), (float)ldexp(p.a, ey - ex), nullptr, X, X2, XT2, 0, 0};
    product(sp, op(P, m), op(XT, n), operand_kt(m, sp), batch, e, w, true, nullptr, st);
    X = X2, XT = XT2, ex = ey;
  }
  return a.used;
}

constexpr double kMostGrowth = 256.0;

int plan(const char* who, int dtype, int64_t batch, int64_t rows, int64_t cols, int steps,
         const double* coefficients, Plan* p) {
  if (dtype != SMQ_DTYPE_F32 && dtype != SMQ_DTYPE_F16 && dtype != SMQ_DTYPE_BF16) {
    set_error("%s: dtype %d is not one of SMQ_DTYPE_F32/F16/BF16", who, dtype);
    return SMQ_ERR_INVALID;
  }
  if (batch < 1 || batch > 65535 || rows < 1 || cols < 1 || rows > (1 << 20) || cols > (1 << 20)) {
    set_error("%s: needs 1 <= batch <= 65535 and 1 <= rows, cols <= 2^20, got %lld, %lld, %lld", who,
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
  return enqueue(p, nullptr, 0, 0, nullptr, 0.0, nullptr, false, nullptr) + 256;
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
  if (!workspace || workspace_bytes < need) {
    set_error("orthogonalize: workspace too small: need %zu bytes, got %zu", need, workspace_bytes);
    return SMQ_ERR_WORKSPACE;
  }
  enqueue(p, x, ld, batch_stride, y, eps, workspace, true, reinterpret_cast<hipStream_t>(stream));
  return check_launch("orthogonalize");
}

}  // extern "C"
