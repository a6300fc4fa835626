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

// parameters c .. c + N - 1 of [0, C) as float32, `missing` where there is none
template <typename T, int N>
__device__ __forceinline__ void load_params(const void* p, int is_f32, long c, long C, float missing, float (&v)[N]) {
  if (p && c + N <= C) {
    if (is_f32) {
#pragma unroll
      for (int k = 0; k < N; k += 4) {
        Vec16<float> t;
        t.load(static_cast<const float*>(p) + c + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[k + j] = t.v[j];
      }
    } else {
      Vec16<T> t;
      t.load(static_cast<const T*>(p) + c);
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = (float)t.v[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = p && c + j < C ? load_param<T>(p, is_f32, c + j) : missing;
  }
}

// Sum over aligned groups of W lanes (16, 32 or 64), the same bits in each of them.  All in the vector units: quad
// permutes and row mirrors within 16 lanes, then gfx950's row and half swaps - a value swapped with itself leaves the
// two partners' values side by side.
template <int W> __device__ __forceinline__ float lanes_sum(float v) {
  static_assert(W == 16 || W == 32 || W == 64, "group of lanes");
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, false));   // quad_perm [1,0,3,2]
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, false));   // quad_perm [2,3,0,1]
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, false));  // row_half_mirror
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, false));  // row_mirror
  if constexpr (W >= 32) {
    const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(t[0]) + __uint_as_float(t[1]);
  }
  if constexpr (W == 64) {
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(t[0]) + __uint_as_float(t[1]);
  }
  return v;
}

}  // namespace
