// group_norm.hip — group norm with an activation on channels-last tensors, forward and backward.
//
//   x [n, s, c] (s positions, c channels, c contiguous), group g = c / (channels / groups):
//   xhat = (x - mean) rstd,  z = weight xhat + bias,  y = act(z)
//   dz = dy act'(z),  dweight = sum dz xhat,  dbias = sum dz,
//   dx = rstd (weight dz - c1 - xhat c2),  c1, c2 = means over the group of weight dz, weight dz xhat
// The backward computes z again from x, mean and rstd: only x and 2 n groups floats are kept.
//
// Memory bound. Two forms, by the size of what a workgroup would have to hold:
//   resident   one workgroup takes a block of whole groups of one sample into registers, reduces and
//              transforms it: x is read once (forward 2 passes over memory, backward 3). Statistics by
//              two passes over the registers (mean, then squared deviations).
//   streaming  a launch for per-channel partial sums of row chunks, a small one that joins them, one
//              that transforms: x is read twice. Statistics of the forward are means and squared
//              deviations from them (no cancellation against a large mean), joined in fp64.
// A thread owns V adjacent channels (16 bytes where the channel count allows) and walks rows, so its
// parameters stay in registers. No atomics: the sums have a fixed order.
#include <limits.h>

#include "smq_common.h"

namespace smq {
void set_error(const char* fmt, ...);
int check_launch(const char* what);

namespace gn {

template <typename T, int V> struct Pack {
  typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T> struct Pack<T, 1> {
  typedef T type;
};
template <typename T, int V>
__device__ __forceinline__ float at(const typename Pack<T, V>::type& v, int i) {
  if constexpr (V == 1) return (float)v;
  else return (float)v[i];
}
template <typename T, int V>
__device__ __forceinline__ void put(typename Pack<T, V>::type& v, int i, float f) {
  if constexpr (V == 1) v = (T)f;
  else v[i] = (T)f;
}

// 1 / (1 + exp(-z)) from the hardware's exp2 and reciprocal: off by (1 - s) |z| 2^-23 + 2 ulp relative, so
// exact to float32's size wherever z s counts; 0 and 1 at the ends. A library expf and an IEEE division
// cost three times the rest of the kernel (it is bound by these instructions, not by memory, otherwise).
__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f));
}
// The activation of V values, one branch for all of them.
template <int V>
__device__ __forceinline__ void act_of(int act, float (&z)[V]) {
  if (act == SMQ_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < V; i++) z[i] = z[i] < 0.0f ? 0.0f : z[i];
  } else if (act == SMQ_ACT_SILU) {
    // -inf stays 0 x -inf = NaN as z times its sigmoid is
#pragma unroll
    for (int i = 0; i < V; i++) z[i] *= sigmoid(z[i]);
  } else if (act == SMQ_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < V; i++) z[i] = 0.5f * z[i] * (1.0f + erff(z[i] * 0.707106781f));
  }
}
// dy times the activation's slope at z.
template <int V>
__device__ __forceinline__ void slope_of(int act, const float (&z)[V], float (&dy)[V]) {
  if (act == SMQ_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < V; i++) dy[i] = z[i] > 0.0f ? dy[i] : z[i] == z[i] ? 0.0f : z[i];
  } else if (act == SMQ_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < V; i++) {
      const float s = sigmoid(z[i]);
      dy[i] *= fmaf(z[i] * s, 1.0f - s, s);
    }
  } else if (act == SMQ_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < V; i++) {
      const float p = __builtin_amdgcn_exp2f(z[i] * z[i] * -0.721347520f);
      dy[i] *= fmaf(z[i] * p, 0.398942280f, 0.5f + 0.5f * erff(z[i] * 0.707106781f));
    }
  }
}

struct Args {
  const void* x;
  const void* dy;
  void* y;  // forward: y, backward: dx
  const float* weight;
  const float* bias;
  float* mean;  // [n, groups], written by the forward
  float* rstd;
  float2* part;  // streaming: [n, chunks, channels]
  float2* coef;  // streaming backward: [n, groups] (c1, c2)
  float2* chan;  // [n, channels]: streaming forward (mul, add) of z = x mul + add, backward sums of dz, dz xhat
  int64_t s;     // positions
  int n, c, groups, cg;
  int block;   // channels a workgroup covers
  int chunks;  // streaming: row chunks
  int act;
  float eps;
};

// Sums of per-thread channel values over the rows of threads: `v` [V] of thread (row, col) -> the
// workgroup's channels. `sh` holds blockDim * V floats. Returns the number of parts P; the caller finds
// P partial sums per channel at sh[p * block + c].
template <int V>
__device__ __forceinline__ int fold(const float (&v)[V], float* sh, int row, int col, int rows, int block,
                                    bool active) {
  __syncthreads();
  if (active) {
#pragma unroll
    for (int i = 0; i < V; i++) sh[row * block + col * V + i] = v[i];
  }
  __syncthreads();
  int parts = blockDim.x / block;
  parts = parts < 1 ? 1 : parts > rows ? rows : parts;
  for (int id = threadIdx.x; id < block * parts; id += blockDim.x) {
    const int c = id % block, p = id / block;
    float s = 0.0f;
    for (int r = p; r < rows; r += parts) s += sh[r * block + c];
    sh[p * block + c] = s;  // only this thread reads or writes rows p, p + parts, ... of channel c
  }
  __syncthreads();
  return parts;
}
// The sum over a group's channels (and parts), in the lanes of one wave.
__device__ __forceinline__ float group_sum(const float* sh, const float* scale, int first, int cg,
                                           int block, int parts) {
  float s = 0.0f;
  for (int k = threadIdx.x & 63; k < cg * parts; k += 64) {
    const int c = first + k % cg;
    const float v = sh[(k / cg) * block + c];
    s += scale ? v * scale[c] : v;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  return s;
}

// Groups of adjacent channels, one division for all of them.
struct Groups {
  int g, left, cg;
  __device__ __forceinline__ Groups(int channel, int cg_) : g(channel / cg_), cg(cg_) {
    left = cg - (channel - g * cg);
  }
  __device__ __forceinline__ int next() {
    const int at = g;
    if (--left == 0) left = cg, g++;
    return at;
  }
};

// ---- resident -----------------------------------------------------------------------------------
// Dynamic LDS: blockDim * V floats, then 2 floats per group of the block.
template <typename T, int V, int R>
__global__ __launch_bounds__(1024) void resident_forward(Args A) {
  typedef typename Pack<T, V>::type vec;
  extern __shared__ float sh[];
  float* stat = sh + blockDim.x * V;
  const int cols = A.block / V, rows = blockDim.x / cols;
  const int col = threadIdx.x % cols, row = threadIdx.x / cols;
  const bool active = row < rows;
  const int c0 = blockIdx.x * A.block, groups = A.block / A.cg, g0 = c0 / A.cg;
  const int64_t base = (int64_t)blockIdx.y * A.s * A.c + c0 + col * V;
  const T* x = reinterpret_cast<const T*>(A.x) + base;
  T* y = reinterpret_cast<T*>(A.y) + base;
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6, lane = threadIdx.x & 63;
  const float inv = 1.0f / ((float)A.s * (float)A.cg);
  vec v[R];
#pragma unroll
  for (int k = 0; k < R; k++) {
    const int64_t r = row + (int64_t)k * rows;
    if (active && r < A.s) v[k] = *reinterpret_cast<const vec*>(x + r * A.c);
  }
  float sum[V], mean[V], rstd[V];
#pragma unroll
  for (int i = 0; i < V; i++) sum[i] = 0.0f;
#pragma unroll
  for (int k = 0; k < R; k++)
    if (active && row + (int64_t)k * rows < A.s) {
#pragma unroll
      for (int i = 0; i < V; i++) sum[i] += at<T, V>(v[k], i);
    }
  int parts = fold<V>(sum, sh, row, col, rows, A.block, active);
  for (int g = wave; g < groups; g += waves) {
    const float s = group_sum(sh, nullptr, g * A.cg, A.cg, A.block, parts);
    if (lane == 0) stat[g] = s * inv;
  }
  __syncthreads();
  const Groups own(col * V, A.cg);
  {
    Groups at_group = own;
#pragma unroll
    for (int i = 0; i < V; i++) {
      mean[i] = stat[at_group.next()];
      sum[i] = 0.0f;
    }
  }
#pragma unroll
  for (int k = 0; k < R; k++)
    if (active && row + (int64_t)k * rows < A.s) {
#pragma unroll
      for (int i = 0; i < V; i++) {
        const float d = at<T, V>(v[k], i) - mean[i];
        sum[i] += d * d;
      }
    }
  parts = fold<V>(sum, sh, row, col, rows, A.block, active);
  for (int g = wave; g < groups; g += waves) {
    const float s = group_sum(sh, nullptr, g * A.cg, A.cg, A.block, parts);
    if (lane == 0) {
      const float r = 1.0f / sqrtf(s * inv + A.eps);
      A.mean[(int64_t)blockIdx.y * A.groups + g0 + g] = stat[g];
      A.rstd[(int64_t)blockIdx.y * A.groups + g0 + g] = r;
      stat[groups + g] = r;
    }
  }
  __syncthreads();
  float mul[V], add[V];
  Groups at_group = own;
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int c = c0 + col * V + i;
    rstd[i] = stat[groups + at_group.next()];
    mul[i] = (A.weight ? A.weight[active ? c : 0] : 1.0f) * rstd[i];
    add[i] = A.bias ? A.bias[active ? c : 0] : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < R; k++) {
    const int64_t r = row + (int64_t)k * rows;
    if (active && r < A.s) {
      vec o;
      float z[V];
#pragma unroll
      for (int i = 0; i < V; i++) z[i] = fmaf(at<T, V>(v[k], i) - mean[i], mul[i], add[i]);
      act_of<V>(A.act, z);
#pragma unroll
      for (int i = 0; i < V; i++) put<T, V>(o, i, z[i]);
      *reinterpret_cast<vec*>(y + r * A.c) = o;
    }
  }
}

template <typename T, int V, int R>
__global__ __launch_bounds__(1024) void resident_backward(Args A) {
  typedef typename Pack<T, V>::type vec;
  extern __shared__ float sh[];
  float* stat = sh + blockDim.x * V;
  const int cols = A.block / V, rows = blockDim.x / cols;
  const int col = threadIdx.x % cols, row = threadIdx.x / cols;
  const bool active = row < rows;
  const int c0 = blockIdx.x * A.block, groups = A.block / A.cg;
  const int64_t base = (int64_t)blockIdx.y * A.s * A.c + c0 + col * V;
  const T* x = reinterpret_cast<const T*>(A.x) + base;
  const T* dy = reinterpret_cast<const T*>(A.dy) + base;
  T* dx = reinterpret_cast<T*>(A.y) + base;
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6, lane = threadIdx.x & 63;
  vec v[R], d[R];
#pragma unroll
  for (int k = 0; k < R; k++) {
    const int64_t r = row + (int64_t)k * rows;
    if (active && r < A.s) {
      v[k] = *reinterpret_cast<const vec*>(x + r * A.c);
      d[k] = *reinterpret_cast<const vec*>(dy + r * A.c);
    }
  }
  // d = x - mean; z = d mul + b; sums of dz and dz d (times rstd: dz xhat)
  float mean[V], rstd[V], mul[V], b[V], p1[V], p2[V];
  const Groups own(col * V, A.cg);
  Groups at_group = own;
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int c = active ? c0 + col * V + i : 0;
    const int64_t g = (int64_t)blockIdx.y * A.groups + c0 / A.cg + at_group.next();
    mean[i] = A.mean[g], rstd[i] = A.rstd[g];
    mul[i] = (A.weight ? A.weight[c] : 1.0f) * rstd[i];
    b[i] = A.bias ? A.bias[c] : 0.0f;
    p1[i] = p2[i] = 0.0f;
  }
  auto slopes = [&](int k, float (&x0)[V], float (&dz)[V]) __attribute__((always_inline)) {
    float z[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
      x0[i] = at<T, V>(v[k], i) - mean[i];
      z[i] = fmaf(x0[i], mul[i], b[i]);
      dz[i] = at<T, V>(d[k], i);
    }
    slope_of<V>(A.act, z, dz);
  };
#pragma unroll
  for (int k = 0; k < R; k++)
    if (active && row + (int64_t)k * rows < A.s) {
      float x0[V], dz[V];
      slopes(k, x0, dz);
#pragma unroll
      for (int i = 0; i < V; i++) {
        p1[i] += dz[i];
        p2[i] = fmaf(dz[i], x0[i], p2[i]);
      }
    }
#pragma unroll
  for (int i = 0; i < V; i++) p2[i] *= rstd[i];
  const float inv = 1.0f / ((float)A.s * (float)A.cg);
  const float* scale = A.weight ? A.weight + c0 : nullptr;
  float* chan = reinterpret_cast<float*>(A.chan + (int64_t)blockIdx.y * A.c + c0);
#pragma unroll
  for (int h = 0; h < 2; h++) {  // the two sums, through the same LDS
    const int parts = fold<V>(h ? p2 : p1, sh, row, col, rows, A.block, active);
    for (int c = threadIdx.x; c < A.block; c += blockDim.x) {
      float s = 0.0f;
      for (int p = 0; p < parts; p++) s += sh[p * A.block + c];
      chan[2 * c + h] = s;
    }
    for (int g = wave; g < groups; g += waves) {
      const float s = group_sum(sh, scale, g * A.cg, A.cg, A.block, parts);
      if (lane == 0) stat[h * groups + g] = s * inv;
    }
  }
  __syncthreads();
  // dx = rstd (dz w - c1 - xhat c2) = dz mul - rstd c1 - d rstd^2 c2
  at_group = own;
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int g = at_group.next();
    p1[i] = -rstd[i] * stat[g], p2[i] = -rstd[i] * rstd[i] * stat[groups + g];
  }
#pragma unroll
  for (int k = 0; k < R; k++) {
    const int64_t r = row + (int64_t)k * rows;
    if (active && r < A.s) {
      vec o;
      float x0[V], dz[V];
      slopes(k, x0, dz);
#pragma unroll
      for (int i = 0; i < V; i++) put<T, V>(o, i, fmaf(dz[i], mul[i], fmaf(x0[i], p2[i], p1[i])));
      *reinterpret_cast<vec*>(dx + r * A.c) = o;
    }
  }
}

// ---- streaming ----------------------------------------------------------------------------------
// 256 threads: `cols` vectors of V channels, 256 / cols rows a step; grid (chunks, channel blocks, n).
struct Walk {
  int col, row, rows, c;
  int64_t first, last;
  bool active;
};
template <int V>
__device__ __forceinline__ Walk walk_of(const Args& A) {
  Walk w;
  const int cols = A.block / V;
  w.rows = 256 / cols;
  w.col = threadIdx.x % cols, w.row = threadIdx.x / cols;
  w.c = blockIdx.y * A.block + w.col * V;
  w.active = w.row < w.rows && w.c < A.c;
  w.first = A.s * blockIdx.x / A.chunks, w.last = A.s * (blockIdx.x + 1) / A.chunks;
  return w;
}
// Two per-channel sums of a chunk -> part[n, chunk, channel].
template <int V>
__device__ __forceinline__ void chunk_sums(const Args& A, const Walk& w, const float (&a)[V],
                                           const float (&b)[V], float2* sh) {
  if (w.active) {
#pragma unroll
    for (int i = 0; i < V; i++) sh[w.row * A.block + w.col * V + i] = make_float2(a[i], b[i]);
  }
  __syncthreads();
  const int c0 = blockIdx.y * A.block;
  for (int c = threadIdx.x; c < A.block && c0 + c < A.c; c += 256) {
    float s1 = 0.0f, s2 = 0.0f;
    for (int r = 0; r < w.rows; r++) s1 += sh[r * A.block + c].x, s2 += sh[r * A.block + c].y;
    A.part[((int64_t)blockIdx.z * A.chunks + blockIdx.x) * A.c + c0 + c] = make_float2(s1, s2);
  }
}

// A chunk's mean and squared deviations from it. A thread sums about its own first value, which is one of
// those it sums: an outlier there costs no more than its own share of the variance (sums about the
// channel's first value lost 10 % of it where that was the outlier). Threads are joined by their means.
template <typename T, int V>
__global__ __launch_bounds__(256) void stream_stats(Args A) {
  typedef typename Pack<T, V>::type vec;
  __shared__ float2 sh[256 * V];
  const Walk w = walk_of<V>(A);
  auto count = [&](int row) {
    const int64_t left = w.last - w.first - row;
    return left > 0 ? (int)((left + w.rows - 1) / w.rows) : 0;
  };
  if (w.active) {
    float s1[V], s2[V], k[V];
#pragma unroll
    for (int i = 0; i < V; i++) s1[i] = s2[i] = k[i] = 0.0f;
    const T* x = reinterpret_cast<const T*>(A.x) + (int64_t)blockIdx.z * A.s * A.c + w.c;
    const int n = count(w.row);
    const vec f = *reinterpret_cast<const vec*>(x + (n ? w.first + w.row : 0) * A.c);
#pragma unroll
    for (int i = 0; i < V; i++) k[i] = at<T, V>(f, i);
#pragma unroll 4
    for (int64_t r = w.first + w.row; r < w.last; r += w.rows) {
      const vec v = *reinterpret_cast<const vec*>(x + r * A.c);
#pragma unroll
      for (int i = 0; i < V; i++) {
        const float d = at<T, V>(v, i) - k[i];
        s1[i] += d;
        s2[i] = fmaf(d, d, s2[i]);
      }
    }
    const float inv = n ? 1.0f / (float)n : 0.0f;
#pragma unroll
    for (int i = 0; i < V; i++) {
      const float m = s1[i] * inv, q = s2[i] - s1[i] * m;
      sh[w.row * A.block + w.col * V + i] = make_float2(k[i] + m, q < 0.0f ? 0.0f : q);
    }
  }
  __syncthreads();
  const int c0 = blockIdx.y * A.block;
  for (int c = threadIdx.x; c < A.block && c0 + c < A.c; c += 256) {
    float mean = 0.0f, q = 0.0f;
    for (int r = 0; r < w.rows; r++) mean = fmaf((float)count(r), sh[r * A.block + c].x, mean);
    mean /= (float)(w.last - w.first);
    for (int r = 0; r < w.rows; r++) {
      const float2 p = sh[r * A.block + c];
      const float d = p.x - mean;
      q += fmaf((float)count(r) * d, d, p.y);
    }
    A.part[((int64_t)blockIdx.z * A.chunks + blockIdx.x) * A.c + c0 + c] = make_float2(mean, q);
  }
}

// One workgroup per (group, n): the chunks of its channels -> mean, rstd.
template <typename T>
__global__ __launch_bounds__(256) void join_stats(Args A) {
  const int g = blockIdx.x, n = blockIdx.y, c0 = g * A.cg;
  const T* x = reinterpret_cast<const T*>(A.x) + (int64_t)n * A.s * A.c;
  double s = 0.0, q = 0.0;  // about k, the group's first value
  const double k = (double)(float)x[c0];
  // a thread keeps to one channel where the group has at most 256
  const int per = A.cg < 256 ? A.cg : 256, lanes = 256 / per;
  const int first = threadIdx.x % per, at0 = threadIdx.x / per;
  if (at0 < lanes)
    for (int i = first; i < A.cg; i += per) {
      const float2* part = A.part + (int64_t)n * A.chunks * A.c + c0 + i;
#pragma unroll 4
      for (int ch = at0; ch < A.chunks; ch += lanes) {
        const float2 p = part[(int64_t)ch * A.c];
        const double rows = (double)(A.s * (ch + 1) / A.chunks - A.s * ch / A.chunks);
        const double d = (double)p.x - k;
        s += rows * d, q += (double)p.y + rows * d * d;
      }
    }
  s = wave_sum(s), q = wave_sum(q);
  __shared__ double a[4], b[4];
  if ((threadIdx.x & 63) == 0) a[threadIdx.x >> 6] = s, b[threadIdx.x >> 6] = q;
  __syncthreads();
  // every thread: the group's statistics, then its channels' mul = w rstd, add = b - mean mul (its rounding,
  // 2^-24 |mean mul|, is that of the mean itself)
  const double m = (double)A.s * A.cg;
  s = ((a[0] + a[1]) + (a[2] + a[3])) / m;
  q = ((b[0] + b[1]) + (b[2] + b[3])) / m - s * s;
  s += k;
  const double rstd = 1.0 / sqrt((q < 0.0 ? 0.0 : q) + (double)A.eps);
  if (threadIdx.x == 0) {
    A.mean[(int64_t)n * A.groups + g] = (float)s;
    A.rstd[(int64_t)n * A.groups + g] = (float)rstd;
  }
  for (int i = threadIdx.x; i < A.cg; i += 256) {
    const float mul = (float)((A.weight ? (double)A.weight[c0 + i] : 1.0) * rstd);
    A.chan[(int64_t)n * A.c + c0 + i] =
        make_float2(mul, (float)((A.bias ? (double)A.bias[c0 + i] : 0.0) - s * (double)mul));
  }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void stream_forward(Args A) {
  typedef typename Pack<T, V>::type vec;
  const Walk w = walk_of<V>(A);
  if (!w.active) return;
  const int64_t base = (int64_t)blockIdx.z * A.s * A.c + w.c;
  const T* x = reinterpret_cast<const T*>(A.x) + base;
  T* y = reinterpret_cast<T*>(A.y) + base;
  float mul[V], add[V];
  const float2* coef = A.chan + (int64_t)blockIdx.z * A.c + w.c;
  if constexpr (V == 1) {
    mul[0] = coef->x, add[0] = coef->y;
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float4 q = *reinterpret_cast<const float4*>(coef + i);
      mul[i] = q.x, add[i] = q.y, mul[i + 1] = q.z, add[i + 1] = q.w;
    }
  }
#pragma unroll 4
  for (int64_t r = w.first + w.row; r < w.last; r += w.rows) {
    const vec v = *reinterpret_cast<const vec*>(x + r * A.c);
    vec o;
    float z[V];
#pragma unroll
    for (int i = 0; i < V; i++) z[i] = fmaf(at<T, V>(v, i), mul[i], add[i]);
    act_of<V>(A.act, z);
#pragma unroll
    for (int i = 0; i < V; i++) put<T, V>(o, i, z[i]);
    *reinterpret_cast<vec*>(y + r * A.c) = o;
  }
}

// One row at a time: with four in flight the eight channels' coefficients and sums took 165 registers, 3
// waves a SIMD (4 x 256 x 256 x 256 bf16 silu: 72 us, 62 now; its 268 MB take 52 at the rate of a copy).
template <typename T, int V>
__global__ __launch_bounds__(256) void stream_sums(Args A) {
  typedef typename Pack<T, V>::type vec;
  __shared__ float2 sh[256 * V];
  const Walk w = walk_of<V>(A);
  float p1[V], p2[V];
#pragma unroll
  for (int i = 0; i < V; i++) p1[i] = p2[i] = 0.0f;
  if (w.active) {
    const int64_t base = (int64_t)blockIdx.z * A.s * A.c + w.c;
    const T* x = reinterpret_cast<const T*>(A.x) + base;
    const T* dy = reinterpret_cast<const T*>(A.dy) + base;
    float mean[V], rstd[V], mul[V], b[V];
    Groups at_group(w.c, A.cg);
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int64_t g = (int64_t)blockIdx.z * A.groups + at_group.next();
      mean[i] = A.mean[g], rstd[i] = A.rstd[g];
      mul[i] = (A.weight ? A.weight[w.c + i] : 1.0f) * rstd[i];
      b[i] = A.bias ? A.bias[w.c + i] : 0.0f;
    }
#pragma unroll 1
    for (int64_t r = w.first + w.row; r < w.last; r += w.rows) {
      const vec v = *reinterpret_cast<const vec*>(x + r * A.c);
      const vec d = *reinterpret_cast<const vec*>(dy + r * A.c);
      float x0[V], z[V], dz[V];
#pragma unroll
      for (int i = 0; i < V; i++) {
        x0[i] = at<T, V>(v, i) - mean[i];
        z[i] = fmaf(x0[i], mul[i], b[i]);
        dz[i] = at<T, V>(d, i);
      }
      slope_of<V>(A.act, z, dz);
#pragma unroll
      for (int i = 0; i < V; i++) {
        p1[i] += dz[i];
        p2[i] = fmaf(dz[i], x0[i], p2[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < V; i++) p2[i] *= rstd[i];
  }
  chunk_sums<V>(A, w, p1, p2, sh);
}

// One workgroup per (group, n): the chunks' sums per channel -> chan, and the group's c1, c2. A wave
// takes a channel, its lanes the chunks.
static __global__ __launch_bounds__(256) void join_sums(Args A) {
  const int g = blockIdx.x, n = blockIdx.y, c0 = g * A.cg, wave = threadIdx.x >> 6;
  double c1 = 0.0, c2 = 0.0;
  for (int i = wave; i < A.cg; i += 4) {
    double s1 = 0.0, s2 = 0.0;
    for (int ch = threadIdx.x & 63; ch < A.chunks; ch += 64) {
      const float2 p = A.part[((int64_t)n * A.chunks + ch) * A.c + c0 + i];
      s1 += (double)p.x, s2 += (double)p.y;
    }
    s1 = wave_sum(s1), s2 = wave_sum(s2);
    if ((threadIdx.x & 63) == 0)
      A.chan[(int64_t)n * A.c + c0 + i] = make_float2((float)s1, (float)s2);
    const double w = A.weight ? (double)A.weight[c0 + i] : 1.0;
    c1 += s1 * w, c2 += s2 * w;
  }
  __shared__ double a[4], b[4];
  if ((threadIdx.x & 63) == 0) a[wave] = c1, b[wave] = c2;
  __syncthreads();
  if (threadIdx.x == 0) {
    const double m = (double)A.s * A.cg;
    A.coef[(int64_t)n * A.groups + g] = make_float2((float)(((a[0] + a[1]) + (a[2] + a[3])) / m),
                                                    (float)(((b[0] + b[1]) + (b[2] + b[3])) / m));
  }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void stream_backward(Args A) {
  typedef typename Pack<T, V>::type vec;
  const Walk w = walk_of<V>(A);
  if (!w.active) return;
  const int64_t base = (int64_t)blockIdx.z * A.s * A.c + w.c;
  const T* x = reinterpret_cast<const T*>(A.x) + base;
  const T* dy = reinterpret_cast<const T*>(A.dy) + base;
  T* dx = reinterpret_cast<T*>(A.y) + base;
  float mean[V], mul[V], b[V], c1[V], c2[V];
  Groups at_group(w.c, A.cg);
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int64_t g = (int64_t)blockIdx.z * A.groups + at_group.next();
    const float rstd = A.rstd[g];
    const float2 k = A.coef[g];
    mean[i] = A.mean[g];
    mul[i] = (A.weight ? A.weight[w.c + i] : 1.0f) * rstd;
    b[i] = A.bias ? A.bias[w.c + i] : 0.0f;
    c1[i] = -rstd * k.x, c2[i] = -rstd * rstd * k.y;
  }
#pragma unroll 2
  for (int64_t r = w.first + w.row; r < w.last; r += w.rows) {
    const vec v = *reinterpret_cast<const vec*>(x + r * A.c);
    const vec d = *reinterpret_cast<const vec*>(dy + r * A.c);
    vec o;
    float x0[V], z[V], dz[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
      x0[i] = at<T, V>(v, i) - mean[i];
      z[i] = fmaf(x0[i], mul[i], b[i]);
      dz[i] = at<T, V>(d, i);
    }
    slope_of<V>(A.act, z, dz);
#pragma unroll
    for (int i = 0; i < V; i++) put<T, V>(o, i, fmaf(dz[i], mul[i], fmaf(x0[i], c2[i], c1[i])));
    *reinterpret_cast<vec*>(dx + r * A.c) = o;
  }
}

// dweight, dbias: chan summed over n. 64 channels a workgroup, 16 waves share the samples.
static __global__ __launch_bounds__(1024) void param_sums(const float2* chan, int n, int c, float* dweight,
                                                          float* dbias) {
  const int t = threadIdx.x & 63, ch = blockIdx.x * 64 + t, w = threadIdx.x >> 6;
  double s1 = 0.0, s2 = 0.0;
  if (ch < c) {
#pragma unroll 4
    for (int i = w; i < n; i += 16) {
      const float2 p = chan[(int64_t)i * c + ch];
      s1 += (double)p.x, s2 += (double)p.y;
    }
  }
  __shared__ double a[16][64], b[16][64];
  a[w][t] = s1, b[w][t] = s2;
  __syncthreads();
  if (w == 0 && ch < c) {
    for (int i = 1; i < 16; i++) s1 += a[i][t], s2 += b[i][t];
    if (dbias) dbias[ch] = (float)s1;
    if (dweight) dweight[ch] = (float)s2;
  }
}

// ---- host ---------------------------------------------------------------------------------------
struct Plan {
  int v;       // channels a thread owns
  int block;   // channels a workgroup covers
  int r;       // resident: vectors a thread holds (0: streaming)
  int threads; // resident
  int chunks;  // streaming
};

int lcm_of(int a, int b) {
  int x = a, y = b;
  while (y) { const int t = x % y; x = y, y = t; }
  return a / x * b;
}

// Vector width: 16 bytes where the channel count is a multiple and the tensors are aligned, else less.
int width_of(int dtype, int c, const void* const* ptrs, int count) {
  const int size = dtype == SMQ_DTYPE_F32 ? 4 : 2;
  for (int v = 16 / size; v > 1; v /= 2) {
    bool ok = c % v == 0;
    for (int i = 0; i < count; i++) ok = ok && (reinterpret_cast<uintptr_t>(ptrs[i]) & (v * size - 1)) == 0;
    if (ok) return v;
  }
  return 1;
}

Plan plan_of(int dtype, int v, int64_t n, int64_t s, int c, int cg, bool backward) {
  const int size = dtype == SMQ_DTYPE_F32 ? 4 : 2;
  Plan p = {v, 0, 0, 0, 0};
  // Resident: whole groups, whole vectors, at least a 64-byte run of channels a row where there are so
  // many, in at most 1024 threads of 16 vectors (8 + 8 in the backward: x and dy).
  const int unit = lcm_of(cg, v), most = backward ? 8 : 16;
  if (c % unit == 0 && unit / v <= 1024) {
    int block = unit;
    while (block * size < 64 && c % (block * 2) == 0 && block * 2 / v <= 1024) block *= 2;
    const int cols = block / v;
    // Small workgroups of full threads first: several on a CU overlap their loads and their sums. A grid
    // that leaves CUs idle takes large ones of short threads instead.
    const bool few = n * (c / block) < 256;
    for (int t = 256; t <= 1024 && !p.r; t *= 2) {
      const int rows = t / cols;
      if (rows < 1) continue;
      const int64_t need = (s + rows - 1) / rows;
      for (int r = 1; r <= most; r *= 2)
        if (need <= r && (!few || r <= 2 || t == 1024)) {
          p.r = r, p.threads = t, p.block = block;
          break;
        }
    }
  }
  if (p.r) return p;
  const int cols = c / v, blocks = (cols + 255) / 256, per = (cols + blocks - 1) / blocks;
  p.block = per * v;
  const int rows = 256 / per;
  // about 2048 workgroups, each at least four steps long
  int64_t chunks = 2048 / (n * blocks);
  if (chunks > s / (4 * rows)) chunks = s / (4 * rows);
  p.chunks = (int)(chunks < 1 ? 1 : chunks);
  return p;
}

size_t align_up(size_t b) { return (b + 255) & ~size_t(255); }

#define SMQ_GN_V(T, K, ...)                                          \
  do {                                                               \
    if (p.v == 8) { if constexpr (sizeof(T) == 2) { K(T, 8, __VA_ARGS__); } } \
    else if (p.v == 4) { K(T, 4, __VA_ARGS__); }                     \
    else if (p.v == 2) { K(T, 2, __VA_ARGS__); }                     \
    else { K(T, 1, __VA_ARGS__); }                                   \
  } while (0)
#define SMQ_GN_RES(T, V, KERNEL, LDS)                                                              \
  do {                                                                                             \
    const dim3 grid(A.c / A.block, (unsigned)A.n);                                                 \
    if (p.r <= 1) hipLaunchKernelGGL((KERNEL<T, V, 1>), grid, dim3(p.threads), LDS, st, A);        \
    else if (p.r == 2) hipLaunchKernelGGL((KERNEL<T, V, 2>), grid, dim3(p.threads), LDS, st, A);   \
    else if (p.r == 4) hipLaunchKernelGGL((KERNEL<T, V, 4>), grid, dim3(p.threads), LDS, st, A);   \
    else if (p.r == 8) hipLaunchKernelGGL((KERNEL<T, V, 8>), grid, dim3(p.threads), LDS, st, A);   \
    else hipLaunchKernelGGL((KERNEL<T, V, 16>), grid, dim3(p.threads), LDS, st, A);                \
  } while (0)
#define SMQ_GN_STREAM(T, V, KERNEL, UNUSED) \
  hipLaunchKernelGGL((KERNEL<T, V>), grid, dim3(256), 0, st, A)

// f(part of the samples): a launch takes at most kSamples of them (its grid's limit).
constexpr int kSamples = 65535;
template <typename T, typename F>
void by_samples(const Args& all, F f) {
  for (int n0 = 0; n0 < all.n; n0 += kSamples) {
    Args A = all;
    const int64_t at = (int64_t)n0 * A.s * A.c, g = (int64_t)n0 * A.groups;
    A.n = all.n - n0 < kSamples ? all.n - n0 : kSamples;
    A.x = reinterpret_cast<const T*>(A.x) + at;
    if (A.dy) A.dy = reinterpret_cast<const T*>(A.dy) + at;
    A.y = reinterpret_cast<T*>(A.y) + at;
    A.mean += g, A.rstd += g;
    A.part += (int64_t)n0 * A.chunks * A.c, A.coef += g, A.chan += (int64_t)n0 * A.c;
    f(A);
    if (all.n - n0 <= kSamples) return;
  }
}

template <typename T>
void forward(const Args& A, const Plan& p, hipStream_t st) {
  if (p.r) {
    const size_t lds = (size_t)(p.threads * p.v + 2 * (p.block / A.cg)) * 4;
    SMQ_GN_V(T, SMQ_GN_RES, resident_forward, lds);
    return;
  }
  const dim3 grid(p.chunks, (A.c + p.block - 1) / p.block, (unsigned)A.n);
  SMQ_GN_V(T, SMQ_GN_STREAM, stream_stats, 0);
  hipLaunchKernelGGL(join_stats<T>, dim3(A.groups, (unsigned)A.n), dim3(256), 0, st, A);
  SMQ_GN_V(T, SMQ_GN_STREAM, stream_forward, 0);
}

template <typename T>
void backward(const Args& A, const Plan& p, hipStream_t st) {
  if (p.r) {
    const size_t lds = (size_t)(p.threads * p.v + 2 * (p.block / A.cg)) * 4;
    SMQ_GN_V(T, SMQ_GN_RES, resident_backward, lds);
  } else {
    const dim3 grid(p.chunks, (A.c + p.block - 1) / p.block, (unsigned)A.n);
    SMQ_GN_V(T, SMQ_GN_STREAM, stream_sums, 0);
    hipLaunchKernelGGL(join_sums, dim3(A.groups, (unsigned)A.n), dim3(256), 0, st, A);
    SMQ_GN_V(T, SMQ_GN_STREAM, stream_backward, 0);
  }
}

int validate(const char* who, int dtype, int64_t n, int64_t s, int64_t c, int64_t groups, int act) {
  if (dtype != SMQ_DTYPE_F32 && dtype != SMQ_DTYPE_F16 && dtype != SMQ_DTYPE_BF16) {
    set_error("%s: dtype %d is not one of SMQ_DTYPE_F32/F16/BF16", who, dtype);
    return SMQ_ERR_INVALID;
  }
  if (n < 1 || s < 1 || c < 1 || n > INT_MAX || c > (1 << 20) || s > ((int64_t)1 << 40) / c) {
    set_error("%s: needs 1 <= n < 2^31, 1 <= channels <= 2^20, 1 <= positions * channels <= 2^40, got "
              "%lld, %lld, %lld", who, (long long)n, (long long)c, (long long)s);
    return SMQ_ERR_INVALID;
  }
  if (groups < 1 || c % groups) {
    set_error("%s: %lld groups do not divide %lld channels", who, (long long)groups, (long long)c);
    return SMQ_ERR_INVALID;
  }
  if (act < SMQ_ACT_NONE || act > SMQ_ACT_GELU) {
    set_error("%s: activation %d invalid", who, act);
    return SMQ_ERR_INVALID;
  }
  return SMQ_OK;
}

// Workspace: part, coef, chan. Sized for any vector width (alignment is not known to the query).
size_t workspace(int dtype, int64_t n, int64_t s, int c, int cg, bool backward, Args* A,
                 void* ws) {
  size_t parts = 0;
  for (int v = 16 / (dtype == SMQ_DTYPE_F32 ? 4 : 2); v >= 1; v /= 2) {
    if (c % v) continue;
    const Plan p = plan_of(dtype, v, n, s, c, cg, backward);
    const size_t b = (size_t)n * p.chunks * c * sizeof(float2);
    if (b > parts) parts = b;
  }
  parts = align_up(parts);
  const size_t coef = backward ? align_up((size_t)n * (c / cg) * sizeof(float2)) : 0;
  const size_t chan = backward || parts ? align_up((size_t)n * c * sizeof(float2)) : 0;
  if (A) {
    char* p = reinterpret_cast<char*>(ws);
    A->part = reinterpret_cast<float2*>(p);
    A->coef = reinterpret_cast<float2*>(p + parts);
    A->chan = reinterpret_cast<float2*>(p + parts + coef);
  }
  return parts + coef + chan + 256;
}
}  // namespace gn
}  // namespace smq

using namespace smq;
using namespace smq::gn;

extern "C" {

size_t smq_group_norm_workspace_bytes(int dtype, int64_t n, int64_t positions, int64_t channels,
                                      int64_t groups, int backward) {
  if (gn::validate("group_norm_workspace_bytes", dtype, n, positions, channels, groups, 0) != SMQ_OK) return 0;
  return gn::workspace(dtype, n, positions, (int)channels, (int)(channels / groups), backward != 0,
                       nullptr, nullptr);
}

int smq_group_norm_act(const void* x, int dtype, void* y, int64_t n, int64_t positions, int64_t channels,
                       int64_t groups, const float* weight, const float* bias, double eps, int activation,
                       float* mean, float* rstd, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = gn::validate("group_norm_act", dtype, n, positions, channels, groups, activation);
  if (rc != SMQ_OK) return rc;
  if (!x || !y || !mean || !rstd || !(eps >= 0.0)) {
    set_error("group_norm_act: x, y, mean and rstd must be non-NULL, eps >= 0");
    return SMQ_ERR_INVALID;
  }
  const int c = (int)channels, cg = (int)(channels / groups);
  const void* ptrs[2] = {x, y};
  const int v = width_of(dtype, c, ptrs, 2);
  Args A = {};
  const size_t need = gn::workspace(dtype, n, positions, c, cg, false, &A, workspace);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)) {
    set_error("group_norm_act: workspace: need %zu bytes on a 16-byte boundary, got %zu", need, workspace_bytes);
    return SMQ_ERR_WORKSPACE;
  }
  const Plan p = plan_of(dtype, v, n, positions, c, cg, false);
  A.x = x, A.y = y, A.weight = weight, A.bias = bias, A.mean = mean, A.rstd = rstd;
  A.s = positions, A.n = (int)n, A.c = c, A.groups = (int)groups, A.cg = cg;
  A.block = p.block, A.chunks = p.chunks, A.act = activation, A.eps = (float)eps;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto go = [&](auto t) {
    by_samples<decltype(t)>(A, [&](const Args& part) { gn::forward<decltype(t)>(part, p, st); });
  };
  if (dtype == SMQ_DTYPE_F32) go(0.0f);
  else if (dtype == SMQ_DTYPE_F16) go((_Float16)0);
  else go((__bf16)0.0f);
  return check_launch("group_norm_act");
}

int smq_group_norm_act_backward(const void* x, const void* dy, int dtype, void* dx, int64_t n,
                                int64_t positions, int64_t channels, int64_t groups,
                                const float* weight, const float* bias, int activation,
                                const float* mean, const float* rstd, float* dweight, float* dbias,
                                void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = gn::validate("group_norm_act_backward", dtype, n, positions, channels, groups, activation);
  if (rc != SMQ_OK) return rc;
  if (!x || !dy || !dx || !mean || !rstd) {
    set_error("group_norm_act_backward: x, dy, dx, mean and rstd must be non-NULL");
    return SMQ_ERR_INVALID;
  }
  const int c = (int)channels, cg = (int)(channels / groups);
  const void* ptrs[3] = {x, dy, dx};
  const int v = width_of(dtype, c, ptrs, 3);
  Args A = {};
  const size_t need = gn::workspace(dtype, n, positions, c, cg, true, &A, workspace);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)) {
    set_error("group_norm_act_backward: workspace: need %zu bytes on a 16-byte boundary, got %zu", need, workspace_bytes);
    return SMQ_ERR_WORKSPACE;
  }
  const Plan p = plan_of(dtype, v, n, positions, c, cg, true);
  A.x = x, A.dy = dy, A.y = dx, A.weight = weight, A.bias = bias;
  A.mean = const_cast<float*>(mean), A.rstd = const_cast<float*>(rstd);
  A.s = positions, A.n = (int)n, A.c = c, A.groups = (int)groups, A.cg = cg;
  A.block = p.block, A.chunks = p.chunks, A.act = activation;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto go = [&](auto t) {
    by_samples<decltype(t)>(A, [&](const Args& part) { gn::backward<decltype(t)>(part, p, st); });
  };
  if (dtype == SMQ_DTYPE_F32) go(0.0f);
  else if (dtype == SMQ_DTYPE_F16) go((_Float16)0);
  else go((__bf16)0.0f);
  if (dweight || dbias)
    hipLaunchKernelGGL(param_sums, dim3((c + 63) / 64), dim3(1024), 0, st, A.chan, A.n, c, dweight, dbias);
  return check_launch("group_norm_act_backward");
}

}  // extern "C"
