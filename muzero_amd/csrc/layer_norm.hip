// Layer norm over the last dimension, forward and backward (the training-block counterpart of bn_train.hip for batches
// that batch statistics do not suit: single states, unequal games):
//     y = (x - m) r w + b,   m = mean(x),  r = 1 / sqrt(mean((x - m)^2) + eps)          per row
//     dx = r (w dy - mean(w dy) - xh mean(w dy xh)),  dw = sum_rows dy xh,  db = sum_rows dy,   xh = (x - m) r
// All sums in float32 (rows too wide for registers: float64).  A float32 mean m0 is off by its own rounding and its sum's, which
// under a large common offset is no small part of the deviations: a constant row of 12345.6 would come out as 0.3.  So
// the second pass over the registers sums the deviations d = x - m0 too: t = mean(d) is what m0 is off by (x - m0 is exact
// where it matters, x and m0 being close), m = m0 + t and var = mean(d^2) - t^2, the error of which is that of d's sums times
// t^2, far below d's own.  The backward pass gets m rounded to float32 and finds t the same way, from the row it reads
// anyway, in the same exchange as its other two sums:
//     mean(w dy xh) = mean(w dy d r) - t r mean(w dy),   xh = (d - t) r
//
// HBM-bound: forward reads x and writes y, backward reads x and dy and writes dx, each once.  A row lives in the
// registers of a group of TPR threads (16, 32 or 64 lanes, or a workgroup), NV 16-byte vectors a thread; groups walk
// down the rows with the parameters of their columns - and, backward, the columns' running dw and db - in registers.
// Every workgroup leaves its dw and db in a float32 partial row and a second launch adds those up: no atomics, the
// same bits on every run.
//
// Measured on an MI355X, forward / backward with both launches: 65536 x 4096 bf16 204 / 330 us (5.3 and 4.9 TB/s; a copy
// of 2 GiB runs at 5.0), 4000 x 16384 float32 98 / 167 us, 18432 x 256 bf16 5.7 / 11.7 us, 4097 x 1001 float32 9.4 / 18.3 us,
// 1000 x 256 bf16 2.6 / 5.5 us: the smaller ones live in the Infinity Cache and are bound by the launches' own time - a third of
// the backward's is the second launch, a few workgroups that add up what up to 768 have left.  Rows wider than registers: 2000 x
// 32768 bf16 256 / 324 us.  What t costs: nothing at 65536 x 4096, 0.8 us of 8.6 in the forward pass of 4097 x 1001, and where
// wide rows' parameters alone want gradients a pass over x (2000 x 32768: 53 us without, 92).
#include "block_common.h"

#include <algorithm>

namespace {

constexpr int kMaxRegisterCols = 16384;     // 1024 threads x 16 columns; wider rows take the looping kernels
constexpr int kMaxWorkgroupCols = 4096;     // wider rows have 512 threads or more
// Most workgroups that leave partial sums of C columns, of whichever type: of up to 256 threads, of more (one a compute unit), and
// down the rows of the column sums of wide rows (256 threads of eight columns, four workgroups a compute unit in all).  An MI355X's
// compute units, so that a workspace's size is the same everywhere.
constexpr int kCus = 256;
constexpr int max_partials(int C) {
  if (C <= kMaxWorkgroupCols) return 4 * kCus;
  if (C <= kMaxRegisterCols) return kCus;
  const int across = (C + 2047) / 2048;
  return (4 * kCus + across - 1) / across;
}

struct LnArgs {
  const void* x;
  const void* dy;
  const void* weight;
  const void* bias;
  void* out;               // y or dx
  float* mean;
  float* rstd;
  float* partial;          // [blocks][2][C]
  float* shift;            // wide rows: [rows] t of the backward pass
  long ldx, lddy, rows;
  int C, affine_f32;
  float eps;
};

// sums of v[0], v[1] .. over the TPR threads of a row; `red` holds K floats per wavefront of the workgroup.  Rows wider
// than a wavefront have the workgroup to themselves, and every thread of it gets here.
template <int TPR, int K> __device__ __forceinline__ void row_sums(float (&v)[K], float* red) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = lanes_sum<TPR <= 64 ? TPR : 64>(v[k]);
  if constexpr (TPR > 64) {
    __syncthreads();                        // the previous sums have been read
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) red[(threadIdx.x >> 6) * K + k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int i = 0; i < TPR / 64; ++i) v[k] += red[i * K + k];
    }
  }
}

// a b, rounded: a mean whose product the compiler fused into some of the differences x - m0 and not into others would be two means
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// What was computed from `v` before is computed again after, not kept
template <typename T> __device__ __forceinline__ void forget(Vec16<T>& v) {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  u32x4 t = __builtin_bit_cast(u32x4, v.v);
  asm volatile("" : "+v"(t));
  v.v = __builtin_bit_cast(typename Vec16<T>::type, t);
}

// the variance from the mean square q of the deviations and their mean t
__device__ __forceinline__ float variance(float q, float t) {
  return q < __FLT_MAX__ ? q - fminf(t * t, q) : q;            // t^2 <= q but for rounding; an overflowed q stays
}

// sums over the 1024 threads of a wide row in float64; `red` holds K doubles per wavefront
template <int K> __device__ __forceinline__ void wide_sums(double (&v)[K], double* red) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v[k] += __shfl_xor(v[k], m);
  __syncthreads();                          // the previous sums have been read
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) red[(threadIdx.x >> 6) * K + k] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = 0.;
#pragma unroll
    for (int i = 0; i < 16; ++i) v[k] += red[i * K + k];
  }
}

template <int TPR> constexpr int block_threads() { return TPR < 256 ? 256 : TPR; }

// ------------------------------------------------------------------------------------------------------------ forward
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(block_threads<TPR>()) void ln_fwd_kernel(LnArgs a) {
  constexpr int N = Vec16<T>::N, RPB = block_threads<TPR>() / TPR;
  __shared__ float red[TPR > 64 ? TPR / 32 : 1];
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.out);
  const float inv_c = 1.f / (float)a.C;
  float w[NV][N], b[NV][N];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    load_params<T, N>(a.weight, a.affine_f32, (k * TPR + lane) * N, a.C, 1.f, w[k]);
    load_params<T, N>(a.bias, a.affine_f32, (k * TPR + lane) * N, a.C, 0.f, b[k]);
  }
  for (long r0 = (long)blockIdx.x * RPB; r0 < a.rows; r0 += (long)gridDim.x * RPB) {
    const long r = r0 + sub;
    const bool live = r < a.rows;           // TPR > 64: one row a workgroup, always live
    Vec16<T> v[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + lane) * N;
      v[k].load_upto(x + r * a.ldx + c, live ? a.C - c : 0);
    }
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < N; ++j) s[0] += (float)v[k].v[j];
    row_sums<TPR>(s, red);
    const float m0 = product(s[0], inv_c);
    float q[2] = {0.f, 0.f};                // sums of d^2 and d
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float d = (k * TPR + lane) * N + j < a.C ? (float)v[k].v[j] - m0 : 0.f;
        q[0] += d * d;
        q[1] += d;
      }
    row_sums<TPR>(q, red);
    const float t = q[1] * inv_c, rstd = 1.f / sqrtf(variance(q[0] * inv_c, t) + a.eps);
    if (!live) continue;
    if (a.mean && lane == 0) {
      a.mean[r] = m0 + t;
      a.rstd[r] = rstd;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + lane) * N;
      Vec16<T> o;
#pragma unroll
      for (int j = 0; j < N; ++j) o.v[j] = (T)(((float)v[k].v[j] - m0 - t) * rstd * w[k][j] + b[k][j]);
      o.store_upto(y + r * (long)a.C + c, a.C - c);
    }
  }
}

// rows wider than the registers of a workgroup: three passes over the row, the later two out of the caches.  A thread's sum
// has up to 2^14 terms, which float32 would not hold to the digits that the deviations need: float64, and the mean is used as
// two floats.
template <typename T> __global__ __launch_bounds__(1024) void ln_fwd_wide_kernel(LnArgs a) {
  constexpr int N = Vec16<T>::N;
  __shared__ double red[16];
  for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.ldx;
    T* y = static_cast<T*>(a.out) + r * (long)a.C;
    double s[1] = {0.};
    for (int c = threadIdx.x * N; c < a.C; c += 1024 * N) {
      Vec16<T> v;
      v.load_upto(x + c, a.C - c);
#pragma unroll
      for (int j = 0; j < N; ++j) s[0] += (double)(float)v.v[j];
    }
    wide_sums(s, red);
    const double mean = s[0] / a.C;
    const float m0 = (float)mean, t = (float)(mean - (double)m0);
    double q[1] = {0.};
    for (int c = threadIdx.x * N; c < a.C; c += 1024 * N) {
      Vec16<T> v;
      v.load_upto(x + c, a.C - c);
      float part = 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float d = (float)v.v[j] - m0 - t;
        part += c + j < a.C ? d * d : 0.f;
      }
      q[0] += (double)part;
    }
    wide_sums(q, red);
    const float rstd = 1.f / sqrtf((float)(q[0] / a.C) + a.eps);
    if (a.mean && threadIdx.x == 0) {
      a.mean[r] = m0;
      a.rstd[r] = rstd;
    }
    for (int c = threadIdx.x * N; c < a.C; c += 1024 * N) {
      Vec16<T> v;
      v.load_upto(x + c, a.C - c);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (c + j < a.C) {
          const float w = a.weight ? load_param<T>(a.weight, a.affine_f32, c + j) : 1.f;
          const float b = a.bias ? load_param<T>(a.bias, a.affine_f32, c + j) : 0.f;
          v.v[j] = (T)(((float)v.v[j] - m0 - t) * rstd * w + b);
        }
      v.store_upto(y + c, a.C - c);
    }
  }
}

// ----------------------------------------------------------------------------------------------------------- backward
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(block_threads<TPR>()) void ln_bwd_kernel(LnArgs a) {
  constexpr int N = Vec16<T>::N, RPB = block_threads<TPR>() / TPR;
  constexpr int kCols = TPR * NV * N;
  // Across a row's sums a thread of many columns keeps x and dy in the elements' type, not their float32 derivatives, and compares
  // its columns with C anew for every row, not in two scalar registers each: all that kept takes 147 registers instead of 112 at
  // 4096 columns of 16 bits, and 1024 threads spill (4000 x 16384 float32: 211 us).  With few columns there is room (18432 x 256
  // bf16: 12.1 us, 12.6 the other way).
  constexpr bool kTight = NV * N > 8;
  __shared__ float red[TPR > 64 ? 3 * TPR / 64 : 1];
  __shared__ float cols[RPB > 1 ? RPB * 2 * kCols : 1];
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  T* dx = static_cast<T*>(a.out);
  const float inv_c = 1.f / (float)a.C;
  float w[NV][N], dw[NV][N], db[NV][N];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    load_params<T, N>(a.weight, a.affine_f32, (k * TPR + lane) * N, a.C, 1.f, w[k]);
#pragma unroll
    for (int j = 0; j < N; ++j) dw[k][j] = db[k][j] = 0.f;
  }
  for (long r0 = (long)blockIdx.x * RPB; r0 < a.rows; r0 += (long)gridDim.x * RPB) {
    const long r = r0 + sub;
    const bool live = r < a.rows;
    Vec16<T> xv[NV], gv[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + lane) * N;
      xv[k].load_upto(x + r * a.ldx + c, live ? a.C - c : 0);
      gv[k].load_upto(dy + r * a.lddy + c, live ? a.C - c : 0);
    }
    const float mean = live ? a.mean[r] : 0.f, rstd = live ? a.rstd[r] : 0.f;
    float s[3] = {0.f, 0.f, 0.f};           // sums of w dy, w dy d r and d; columns past the end have dy = 0
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      int left = a.C - (k * TPR + lane) * N;
      if constexpr (kTight) asm volatile("" : "+v"(left));
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float g = (float)gv[k].v[j] * w[k][j], d = (float)xv[k].v[j] - mean;
        s[0] += g;
        s[1] += g * (d * rstd);
        s[2] += j < left ? d : 0.f;
      }
      if constexpr (kTight) {
        forget(xv[k]);
        forget(gv[k]);
      }
    }
    row_sums<TPR>(s, red);
    const float t = s[2] * inv_c, m1 = s[0] * inv_c, m2 = s[1] * inv_c - t * rstd * m1;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + lane) * N;
      Vec16<T> o;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float g = (float)gv[k].v[j], xh = ((float)xv[k].v[j] - mean - t) * rstd;
        dw[k][j] += g * xh;
        db[k][j] += g;
        o.v[j] = (T)(rstd * (g * w[k][j] - m1 - xh * m2));
      }
      if (a.out && live) o.store_upto(dx + r * (long)a.C + c, a.C - c);
    }
  }
  if (!a.partial) return;
  float* mine = a.partial + (long)blockIdx.x * 2 * a.C;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = (k * TPR + lane) * N + j;
        if (c < a.C) {
          mine[c] = dw[k][j];
          mine[a.C + c] = db[k][j];
        }
      }
  } else {                                  // several rows a workgroup: add its row groups' sums up first
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = (k * TPR + lane) * N + j;
        cols[(sub * 2 + 0) * kCols + c] = dw[k][j];
        cols[(sub * 2 + 1) * kCols + c] = db[k][j];
      }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * kCols; i += block_threads<TPR>()) {
      const int which = i / kCols, c = i - which * kCols;
      if (c >= a.C) continue;
      float s = 0.f;
#pragma unroll
      for (int g = 0; g < RPB; ++g) s += cols[(g * 2 + which) * kCols + c];
      mine[which * (long)a.C + c] = s;
    }
  }
}

// wide rows: dx, and each row's t for the column sums; without dx only the latter
template <typename T> __global__ __launch_bounds__(1024) void ln_bwd_wide_kernel(LnArgs a) {
  constexpr int N = Vec16<T>::N;
  __shared__ double red[3 * 16];
  for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + r * a.lddy;
    T* dx = static_cast<T*>(a.out) + r * (long)a.C;
    const float mean = a.mean[r], rstd = a.rstd[r];
    double s[3] = {0., 0., 0.};             // sums of w dy, w dy d r and d
    for (int c = threadIdx.x * N; c < a.C; c += 1024 * N) {
      Vec16<T> xv, gv;
      float part[3] = {0.f, 0.f, 0.f};
      xv.load_upto(x + c, a.C - c);
#pragma unroll
      for (int j = 0; j < N; ++j) part[2] += c + j < a.C ? (float)xv.v[j] - mean : 0.f;
      if (a.out) {
        gv.load_upto(dy + c, a.C - c);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float w = a.weight && c + j < a.C ? load_param<T>(a.weight, a.affine_f32, c + j) : 1.f;
          const float g = (float)gv.v[j] * w;
          part[0] += g;
          part[1] += g * (((float)xv.v[j] - mean) * rstd);
        }
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) s[k] += (double)part[k];
    }
    wide_sums(s, red);
    const float t = (float)(s[2] / a.C);
    if (a.shift && threadIdx.x == 0) a.shift[r] = t;
    if (!a.out) continue;
    const float m1 = (float)(s[0] / a.C), m2 = (float)(s[1] / a.C - s[2] / a.C * rstd * (s[0] / a.C));
    for (int c = threadIdx.x * N; c < a.C; c += 1024 * N) {
      Vec16<T> xv, gv;
      xv.load_upto(x + c, a.C - c);
      gv.load_upto(dy + c, a.C - c);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float w = a.weight && c + j < a.C ? load_param<T>(a.weight, a.affine_f32, c + j) : 1.f;
        const float xh = ((float)xv.v[j] - mean - t) * rstd;
        gv.v[j] = (T)(rstd * ((float)gv.v[j] * w - m1 - xh * m2));
      }
      gv.store_upto(dx + c, a.C - c);
    }
  }
}

// column sums for the wide rows: workgroup (bx, by) owns 256 vectors of columns and every gridDim.y-th row
template <typename T> __global__ __launch_bounds__(256) void ln_bwd_wide_cols_kernel(LnArgs a) {
  constexpr int N = Vec16<T>::N;
  const int c = (blockIdx.x * 256 + threadIdx.x) * N;
  if (c >= a.C) return;
  float dw[N], db[N];
#pragma unroll
  for (int j = 0; j < N; ++j) dw[j] = db[j] = 0.f;
  for (long r = blockIdx.y; r < a.rows; r += gridDim.y) {
    Vec16<T> xv, gv;
    xv.load_upto(static_cast<const T*>(a.x) + r * a.ldx + c, a.C - c);
    gv.load_upto(static_cast<const T*>(a.dy) + r * a.lddy + c, a.C - c);
    const float mean = a.mean[r], t = a.shift[r], rstd = a.rstd[r];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float g = (float)gv.v[j];
      dw[j] += g * (((float)xv.v[j] - mean - t) * rstd);
      db[j] += g;
    }
  }
  float* mine = a.partial + (long)blockIdx.y * 2 * a.C;
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (c + j < a.C) {
      mine[c + j] = dw[j];
      mine[a.C + c + j] = db[j];
    }
}

// dw and db from the workgroups' partial rows: 32 columns x 32 row lanes a workgroup
template <typename T>
__global__ __launch_bounds__(1024) void ln_bwd_finish_kernel(const float* __restrict__ partial, int blocks, int C,
                                                             void* dweight, void* dbias, int affine_f32) {
  __shared__ float red[2][32][33];
  const int col = threadIdx.x & 31, lane = threadIdx.x >> 5, c = blockIdx.x * 32 + col;
  float s = 0.f, q = 0.f;
  if (c < C)
    for (int k0 = lane; k0 < blocks; k0 += 32 * 4) {      // eight loads in flight
      float t[2][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = k0 + 32 * i;
        t[0][i] = k < blocks ? partial[(long)k * 2 * C + c] : 0.f;
        t[1][i] = k < blocks ? partial[(long)k * 2 * C + C + c] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s += t[0][i];
        q += t[1][i];
      }
    }
  red[0][lane][col] = s;
  red[1][lane][col] = q;
  __syncthreads();
  if (lane >= 2 || c >= C) return;
  float t = 0.f;
#pragma unroll
  for (int k = 0; k < 32; ++k) t += red[lane][k][col];
  void* out = lane == 0 ? dweight : dbias;
  if (out) store_param<T>(out, affine_f32, c, t);
}

// ------------------------------------------------------------------------------------------------------------- launch
// How a row is laid over threads: the fewest threads that hold it at up to two vectors each (up to 16 columns a thread
// for workgroup rows).
template <typename T, typename Fwd> int with_shape(int C, Fwd&& f) {
  constexpr int N = Vec16<T>::N;
  const int units = (C + N - 1) / N;
#define MZ_SHAPE(tpr, nv) if (units <= (tpr) * (nv)) return f(std::integral_constant<int, tpr>{}, std::integral_constant<int, nv>{})
  MZ_SHAPE(16, 1);
  MZ_SHAPE(32, 1);
  MZ_SHAPE(64, 1);
  MZ_SHAPE(64, 2);
  MZ_SHAPE(256, 1);
  MZ_SHAPE(256, 2);
  if constexpr (N == 4) MZ_SHAPE(256, 4);
  MZ_SHAPE(512, 16 / N);
  MZ_SHAPE(1024, 16 / N);
#undef MZ_SHAPE
  return -1;
}

// workgroups for `rows`: as many as `cap`, fewer where that gives all of them the same number of rounds
int row_blocks(long rows, int rows_per_block, int cap) {
  const long groups = (rows + rows_per_block - 1) / rows_per_block, rounds = (groups + cap - 1) / cap;
  return (int)((groups + rounds - 1) / rounds);
}

// Workgroups of the backward pass.  Each leaves 8 C bytes of partial sums that are written and read once more, so it
// should walk at least eight rows (at 2000 x 8192 bf16: 34 us, with four rows 45 us), as long as every compute unit
// has one (500 x 2048: 10.5 us with one each, 12.4 with one in four).
int bwd_blocks(long rows, int rows_per_block, int threads, int C) {
  const int cus = mz::compute_units();
  long cap = threads >= 512 ? cus : 3 * cus;
  const long few = rows / 8 > cus ? rows / 8 : cus;
  if (cap > few) cap = few;
  if (cap > max_partials(C)) cap = max_partials(C);
  return row_blocks(rows, rows_per_block, (int)cap);
}

template <typename T> int ln_fwd(const LnArgs& a, hipStream_t s) {
  if (a.C > kMaxRegisterCols) {
    hipLaunchKernelGGL((ln_fwd_wide_kernel<T>), dim3(row_blocks(a.rows, 1, 4 * mz::compute_units())), dim3(1024), 0, s, a);
    return MZ_OK;
  }
  return with_shape<T>(a.C, [&](auto tpr, auto nv) {
    constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, NT = block_threads<TPR>();
    const int blocks = row_blocks(a.rows, NT / TPR, mz::compute_units() * 1024 / NT);
    hipLaunchKernelGGL((ln_fwd_kernel<T, TPR, NV>), dim3(blocks), dim3(NT), 0, s, a);
    return MZ_OK;
  });
}

template <typename T> int ln_bwd(const LnArgs& a, void* dweight, void* dbias, hipStream_t s) {
  int blocks = 0;
  if (a.C > kMaxRegisterCols) {
    if (a.out || a.partial)
      hipLaunchKernelGGL((ln_bwd_wide_kernel<T>), dim3(row_blocks(a.rows, 1, 2 * mz::compute_units())), dim3(1024), 0, s, a);
    if (a.partial) {
      constexpr int kCols = 256 * Vec16<T>::N;
      const int bx = (a.C + kCols - 1) / kCols;
      int by = (4 * mz::compute_units() + bx - 1) / bx;
      by = row_blocks(a.rows, 1, by < max_partials(a.C) ? by : max_partials(a.C));
      blocks = by;
      hipLaunchKernelGGL((ln_bwd_wide_cols_kernel<T>), dim3(bx, by), dim3(256), 0, s, a);
    }
  } else {
    with_shape<T>(a.C, [&](auto tpr, auto nv) {
      // the widest float32 rows on half the threads with twice the registers: 1024 threads spill (4000 x 16384: 230 us)
      constexpr bool kHalve = decltype(tpr)::value == 1024 && sizeof(T) == 4;
      constexpr int TPR = kHalve ? 512 : decltype(tpr)::value, NV = kHalve ? 8 : decltype(nv)::value, NT = block_threads<TPR>();
      blocks = bwd_blocks(a.rows, NT / TPR, NT, a.C);
      hipLaunchKernelGGL((ln_bwd_kernel<T, TPR, NV>), dim3(blocks), dim3(NT), 0, s, a);
      return MZ_OK;
    });
  }
  if (a.partial)
    hipLaunchKernelGGL((ln_bwd_finish_kernel<T>), dim3((a.C + 31) / 32), dim3(1024), 0, s, a.partial, blocks, a.C, dweight,
                       dbias, a.affine_f32);
  return MZ_OK;
}

int64_t partial_floats(int64_t rows, int32_t C) { return std::min<int64_t>(rows, max_partials(C)) * 2 * C; }

int check_rows(const char* who, int64_t rows, int32_t C, int64_t ld) {
  MZ_REQUIRE(ld >= C || rows == 1, "%s: rows overlap (stride %lld < C = %d)", who, (long long)ld, C);
  MZ_REQUIRE(rows == 1 || ld <= (1ll << 48) / rows, "%s: %lld rows %lld elements apart lie past any memory", who, (long long)rows,
             (long long)ld);
  return MZ_OK;
}

int check(const char* who, int64_t rows, int32_t C, int64_t ld, int32_t dtype, int32_t affine_dtype) {
  MZ_REQUIRE(rows > 0 && C > 0 && C <= (1 << 24), "%s: rows > 0 and 0 < C <= 2^24 expected (rows = %lld, C = %d)", who,
             (long long)rows, C);
  if (int rc = check_rows(who, rows, C, ld)) return rc;
  MZ_REQUIRE(dtype == MZ_F32 || dtype == MZ_BF16 || dtype == MZ_F16, "%s: unknown element type %d", who, dtype);
  MZ_REQUIRE(affine_dtype == MZ_F32 || affine_dtype == dtype, "%s: parameters are float32 or of the activations' type", who);
  return MZ_OK;
}

}  // namespace

extern "C" {

int mz_layer_norm_fwd(const void* x, int64_t ldx, const void* weight, const void* bias, int32_t affine_dtype, double eps,
                      int64_t rows, int32_t C, int32_t dtype, void* y, float* mean, float* rstd, mz_stream_t stream) {
  MZ_REQUIRE(x && y, "mz_layer_norm_fwd: null tensor");
  MZ_REQUIRE((mean == nullptr) == (rstd == nullptr), "mz_layer_norm_fwd: mean and rstd go together");
  if (int rc = check("mz_layer_norm_fwd", rows, C, ldx, dtype, affine_dtype)) return rc;
  MZ_REQUIRE(eps >= 0.0, "mz_layer_norm_fwd: eps must not be negative");
  const LnArgs a = {x, nullptr, weight, bias, y, mean, rstd, nullptr, nullptr, ldx, 0, rows, C, affine_dtype == MZ_F32, (float)eps};
  hipStream_t s = mz::as_stream(stream);
  if (dtype == MZ_F32) ln_fwd<float>(a, s);
  else if (dtype == MZ_BF16) ln_fwd<__bf16>(a, s);
  else ln_fwd<_Float16>(a, s);
  return mz::check_launch("mz_layer_norm_fwd");
}

int64_t mz_layer_norm_workspace_bytes(int64_t rows, int32_t C) {
  if (rows <= 0 || C <= 0) return 0;
  return partial_floats(rows, C) * 4 + (C > kMaxRegisterCols ? rows * 4 : 0);
}

int mz_layer_norm_bwd(const void* x, int64_t ldx, const void* dy, int64_t lddy, const void* weight, int32_t affine_dtype,
                      const float* mean, const float* rstd, int64_t rows, int32_t C, int32_t dtype, void* dx, void* dweight,
                      void* dbias, void* workspace, int64_t workspace_bytes, mz_stream_t stream) {
  MZ_REQUIRE(x && dy && mean && rstd, "mz_layer_norm_bwd: null tensor");
  MZ_REQUIRE(dx || dweight || dbias, "mz_layer_norm_bwd: no gradient asked for");
  if (int rc = check("mz_layer_norm_bwd", rows, C, ldx, dtype, affine_dtype)) return rc;
  if (int rc = check_rows("mz_layer_norm_bwd: dy", rows, C, lddy)) return rc;
  const bool params = dweight || dbias;
  MZ_REQUIRE(!params || (workspace && workspace_bytes >= mz_layer_norm_workspace_bytes(rows, C) && (size_t)workspace % 4 == 0),
             "mz_layer_norm_bwd: workspace too small or not aligned to float");
  float* partial = params ? static_cast<float*>(workspace) : nullptr;
  float* shift = params && C > kMaxRegisterCols ? partial + partial_floats(rows, C) : nullptr;
  const LnArgs a = {x, dy, weight, nullptr, dx, const_cast<float*>(mean), const_cast<float*>(rstd), partial, shift, ldx, lddy, rows, C, affine_dtype == MZ_F32, 0.f};
  hipStream_t s = mz::as_stream(stream);
  if (dtype == MZ_F32) ln_bwd<float>(a, dweight, dbias, s);
  else if (dtype == MZ_BF16) ln_bwd<__bf16>(a, dweight, dbias, s);
  else ln_bwd<_Float16>(a, dweight, dbias, s);
  return mz::check_launch("mz_layer_norm_bwd");
}

}  // extern "C"
