// Shared by the training-block operators (layer_norm.hip, gated_ff*, dropout.hip): element types, 16-byte vectors that
// need only their element's alignment, sums over groups of lanes.
#pragma once
#include "common.h"

namespace {

// ---- element types of activations and parameters, as the C ABI numbers them (MZ_F32, MZ_BF16, MZ_F16)
template <typename T> struct ElemTraits;
template <> struct ElemTraits<float> { static constexpr int kVec = 4; };
template <> struct ElemTraits<__bf16> { static constexpr int kVec = 8; };
template <> struct ElemTraits<_Float16> { static constexpr int kVec = 8; };

// 16 bytes of elements.  Rows of odd widths start at any element, so the vector type claims no more than the element's
// alignment; global memory takes such accesses as one instruction.
template <typename T> struct Vec16 {
  static constexpr int N = ElemTraits<T>::kVec;
  typedef T type __attribute__((ext_vector_type(ElemTraits<T>::kVec)));
  typedef type unaligned __attribute__((aligned(sizeof(T))));
  type v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const unaligned*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<unaligned*>(p) = v; }
  // elements [0, n) of the unit, the rest zero; n >= N loads the whole vector
  __device__ __forceinline__ void load_upto(const T* p, long n) {
    if (n >= N) {
      load(p);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = j < n ? p[j] : (T)0.f;
    }
  }
  __device__ __forceinline__ void store_upto(T* p, long n) const {
    if (n >= N) {
      store(p);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < n) p[j] = v[j];
    }
  }
};

// a parameter of either type the operators take (float32, or the activations' type)
template <typename T> __device__ __forceinline__ float load_param(const void* p, int is_f32, long i) {
  return is_f32 ? static_cast<const float*>(p)[i] : (float)static_cast<const T*>(p)[i];
}
template <typename T> __device__ __forceinline__ void store_param(void* p, int is_f32, long i, float v) {
  if (is_f32) static_cast<float*>(p)[i] = v;
  else static_cast<T*>(p)[i] = (T)v;
}

// Sum over aligned groups of `W` lanes (a power of two, at most 64), returned in each of them.
template <int W> __device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int d = 1; d < W; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

}  // namespace
