// Dropout whose mask is a function of (seed, offset, call, element) and is never stored:
//     y = [residual +] (keep ? x * scale : 0),   scale = 65536 / (65536 - t),   t = round(65536 p)
// keep: 16 bits of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011)
// compared with t.  One evaluation under key = seed at counter = (block, call, offset low, offset high) serves the
// eight elements 8 block .. 8 block + 7, element j taking bits 16 (j % 2) .. of word j / 2: a generator round costs two
// 32 x 32 -> 64 bit products, which the vector units do at a quarter of their rate, so 32 bits an element would make
// the kernel bound by them instead of by memory; 16 round p to a multiple of 2^-16, and the scale is that p's own.
// The backward pass is the same kernel on the gradient.  A dropped element is zero whatever it held (NaN, infinity).
// HBM-bound: reads x (+ residual), writes y.  Measured on an MI355X: 16385 x 8191 bf16 with a residual, forward and
// backward 259 us (1.34 GB: 5.2 TB/s, a copy of 2 GiB runs at 5.0); 18432 x 256 bf16 6.4 us, 128 x 256 float32 2.8 us (a
// launch).
#include "block_common.h"

namespace {

struct Philox {
  unsigned k0, k1;
  __device__ __forceinline__ uint4 operator()(unsigned c0, unsigned c1, unsigned c2, unsigned c3) const {
    unsigned a = k0, b = k1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      const unsigned long long p = 0xD2511F53ull * c0, q = 0xCD9E8D57ull * c2;
      c0 = (unsigned)(q >> 32) ^ c1 ^ a;
      c1 = (unsigned)q;
      c2 = (unsigned)(p >> 32) ^ c3 ^ b;
      c3 = (unsigned)p;
      a += 0x9E3779B9u;
      b += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
  }
};

template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, const T* residual,
                                                      T* y, long n, unsigned threshold, float scale,
                                                      const long long* __restrict__ rng, unsigned call) {
  constexpr int N = Vec16<T>::N;
  const unsigned long long seed = (unsigned long long)rng[0], offset = (unsigned long long)rng[1];
  const Philox philox = {(unsigned)seed, (unsigned)(seed >> 32)};
  const long blocks = (n + 7) / 8;
  for (long u = (long)blockIdx.x * 256 + threadIdx.x; u < blocks; u += (long)gridDim.x * 256) {
    Vec16<T> v[8 / N], r[8 / N];
#pragma unroll
    for (int k = 0; k < 8 / N; ++k) v[k].load_upto(x + u * 8 + k * N, n - (u * 8 + k * N));
    if (residual) {
#pragma unroll
      for (int k = 0; k < 8 / N; ++k) r[k].load_upto(residual + u * 8 + k * N, n - (u * 8 + k * N));
    }
    const uint4 word = philox((unsigned)u, call, (unsigned)offset, (unsigned)(offset >> 32));
    const unsigned bits[4] = {word.x, word.y, word.z, word.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned b = (j & 1) ? bits[j / 2] >> 16 : bits[j / 2] & 0xffffu;
      float o = b >= threshold ? (float)v[j / N].v[j % N] * scale : 0.f;
      if (residual) o += (float)r[j / N].v[j % N];
      v[j / N].v[j % N] = (T)o;
    }
#pragma unroll
    for (int k = 0; k < 8 / N; ++k) v[k].store_upto(y + u * 8 + k * N, n - (u * 8 + k * N));
  }
}

template <typename T>
void launch(const void* x, const void* residual, void* y, long n, unsigned threshold, float scale, const int64_t* rng,
            unsigned call, hipStream_t s) {
  const long want = ((n + 7) / 8 + 255) / 256, cap = 16L * mz::compute_units();
  hipLaunchKernelGGL((dropout_kernel<T>), dim3((unsigned)(want < cap ? want : cap)), dim3(256), 0, s,
                     static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<T*>(y), n, threshold, scale,
                     reinterpret_cast<const long long*>(rng), call);
}

}  // namespace

extern "C" int mz_dropout(const void* x, const void* residual, void* y, int64_t n, double p, const int64_t* rng,
                          uint32_t call, int32_t dtype, mz_stream_t stream) {
  MZ_REQUIRE(x && y && rng, "mz_dropout: null tensor");
  MZ_REQUIRE(n > 0 && n <= (1ll << 35), "mz_dropout: 0 < n <= 2^35 elements expected (n = %lld)", (long long)n);
  MZ_REQUIRE(p >= 0.0 && p <= 1.0, "mz_dropout: p in [0, 1] expected");
  MZ_REQUIRE(dtype == MZ_F32 || dtype == MZ_BF16 || dtype == MZ_F16, "mz_dropout: unknown element type %d", dtype);
  const unsigned t = (unsigned)nearbyint(p * 65536.0);
  const float scale = t < 65536 ? (float)(65536.0 / (double)(65536 - t)) : 0.f;
  hipStream_t s = mz::as_stream(stream);
  if (dtype == MZ_F32) launch<float>(x, residual, y, n, t, scale, rng, call, s);
  else if (dtype == MZ_BF16) launch<__bf16>(x, residual, y, n, t, scale, rng, call, s);
  else launch<_Float16>(x, residual, y, n, t, scale, rng, call, s);
  return mz::check_launch("mz_dropout");
}
