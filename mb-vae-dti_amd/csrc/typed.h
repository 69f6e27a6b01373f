// Element types of the operators that take fp32, bf16 and fp16 tensors: 16-byte accesses at element alignment, arithmetic in fp32.
#pragma once
#include "common.h"

#define MBVAE_F32 0
#define MBVAE_BF16 1
#define MBVAE_F16 2
// integer types of class ids
#define MBVAE_ID_I8 1
#define MBVAE_ID_I16 2
#define MBVAE_ID_U8 3
#define MBVAE_ID_I32 4
#define MBVAE_ID_I64 8

typedef __bf16 mbvae_bf16;
typedef _Float16 mbvae_f16;

static inline int mbvae_dtype_size(int dtype) { return dtype == MBVAE_F32 ? 4 : (dtype == MBVAE_BF16 || dtype == MBVAE_F16) ? 2 : 0; }

// Elements of one 16-byte access.  Rows of odd width start at any element, so the vector types carry the element's
// alignment only: gfx950 runs global accesses of every width at any address, and an aligned one costs the same.
template <typename T>
struct MbvaeVec {
  static constexpr int N = 16 / (int)sizeof(T);
  typedef T Aligned __attribute__((ext_vector_type(16 / sizeof(T))));
  typedef Aligned Any __attribute__((aligned(sizeof(T))));
};

// v[0..N) = the N elements at p as fp32; those from `left` on are not read and become 0.
template <typename T>
__device__ __forceinline__ void mbvae_load_vec(const T* p, int left, float* v) {
  constexpr int N = MbvaeVec<T>::N;
  if (left >= N) {
    const typename MbvaeVec<T>::Aligned t = *reinterpret_cast<const typename MbvaeVec<T>::Any*>(p);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = (float)t[e];
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = e < left ? (float)p[e] : 0.f;
  }
}

// The same as one vector of the type itself.
template <typename T>
__device__ __forceinline__ typename MbvaeVec<T>::Aligned mbvae_load_raw(const T* p, int left) {
  constexpr int N = MbvaeVec<T>::N;
  typename MbvaeVec<T>::Aligned t;
  if (left >= N) {
    t = *reinterpret_cast<const typename MbvaeVec<T>::Any*>(p);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) t[e] = e < left ? p[e] : (T)0.f;
  }
  return t;
}

// The first min(N, left) elements at p = v, each rounded once to nearest even.
template <typename T>
__device__ __forceinline__ void mbvae_store_vec(T* p, int left, const float* v) {
  constexpr int N = MbvaeVec<T>::N;
  if (left >= N) {
    typename MbvaeVec<T>::Aligned t;
#pragma unroll
    for (int e = 0; e < N; ++e) t[e] = (T)v[e];
    *reinterpret_cast<typename MbvaeVec<T>::Any*>(p) = t;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < left) p[e] = (T)v[e];
  }
}

// Parameter vectors (gamma, beta, scale) may have another type than the activations: the type is a run-time, wave-uniform choice.
__device__ __forceinline__ void mbvae_store_param(void* p, int dtype, int64_t i, float v) {
  if (dtype == MBVAE_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dtype == MBVAE_BF16) reinterpret_cast<mbvae_bf16*>(p)[i] = (mbvae_bf16)v;
  else reinterpret_cast<mbvae_f16*>(p)[i] = (mbvae_f16)v;
}

// Sum over aligned groups of TPR lanes of a wave (a power of two from 2 to 64), left in every lane.  Steps inside 16 lanes are
// lane permutations of the vector ALU; after a step all lanes of the smaller group agree, so a mirror serves as the exchange.
template <int CTRL>
__device__ __forceinline__ float mbvae_dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int TPR>
__device__ __forceinline__ float mbvae_team_sum(float v) {
  static_assert(TPR >= 2 && TPR <= 64 && (TPR & (TPR - 1)) == 0, "a team is a power of two of lanes of one wave");
  v = mbvae_dpp_add<0xB1>(v);                       // quad_perm [1,0,3,2]
  if (TPR >= 4) v = mbvae_dpp_add<0x4E>(v);         // quad_perm [2,3,0,1]
  if (TPR >= 8) v = mbvae_dpp_add<0x141>(v);        // row_half_mirror
  if (TPR >= 16) v = mbvae_dpp_add<0x140>(v);       // row_mirror
  if (TPR >= 32) v += __shfl_xor(v, 16, 64);
  if (TPR >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}
