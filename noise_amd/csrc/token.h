// Element types, vector loads and lane reductions shared by the token operators (layernorm.hip, decay_attn.hip,
// adamw_multi.hip).  Arithmetic is fp32 whatever the element type; a store rounds once, to nearest even.
#pragma once
#include "common.h"

// dtype codes of the C ABI
enum { NOISE_F32 = 0, NOISE_BF16 = 1, NOISE_F16 = 2 };

#ifdef __HIPCC__
using bf16_t = __bf16;
using f16_t = _Float16;

template <typename T, int V>
struct VecOf {
  using type = T __attribute__((ext_vector_type(V)));
};
template <typename T>
struct VecOf<T, 1> {
  using type = T;
};

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&out)[V]) {
  if constexpr (V == 1) {
    out[0] = (float)*p;
  } else if constexpr (sizeof(T) * V <= 16) {
    const auto v = *reinterpret_cast<const typename VecOf<T, V>::type*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (float)v[i];
  } else {   // fp32 parameters beside 16-bit activations: V floats in 16-byte pieces
#pragma unroll
    for (int k = 0; k < V / 4; ++k) {
      const auto v = *reinterpret_cast<const typename VecOf<T, 4>::type*>(p + 4 * k);
#pragma unroll
      for (int i = 0; i < 4; ++i) out[4 * k + i] = (float)v[i];
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[V]) {
  if constexpr (V == 1) {
    *p = (T)in[0];
  } else {
    typename VecOf<T, V>::type v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)in[i];
    *reinterpret_cast<typename VecOf<T, V>::type*>(p) = v;
  }
}

// The same store past the caches (NT): for results larger than the last-level cache could keep for their reader.
template <bool NT, typename T, int V>
__device__ __forceinline__ void store_vec_nt(T* p, const float (&in)[V]) {
  if constexpr (!NT || V == 1) {
    store_vec<T, V>(p, in);
  } else {
    typename VecOf<T, V>::type v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)in[i];
    __builtin_nontemporal_store(v, reinterpret_cast<typename VecOf<T, V>::type*>(p));
  }
}

template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// Sum over aligned groups of LANES lanes, the result in every lane.  Within 16 lanes the exchange is a DPP operand of the
// addition (lane ^ 1, lane ^ 2, mirrored halves, mirrored rows); the two wider steps go through the LDS crossbar.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  static_assert(LANES <= 64 && (LANES & (LANES - 1)) == 0, "a group is a power of two within a wave");
  if constexpr (LANES >= 2) v += dpp_move<0xB1>(v);
  if constexpr (LANES >= 4) v += dpp_move<0x4E>(v);
  if constexpr (LANES >= 8) v += dpp_move<0x141>(v);
  if constexpr (LANES >= 16) v += dpp_move<0x140>(v);
  if constexpr (LANES >= 32) v += __shfl_xor(v, 16, 64);
  if constexpr (LANES >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}
#endif
