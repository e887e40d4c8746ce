// Element types of the layer kernels (trl_norm.hip, trl_decay.hip): float32, bfloat16 and float16 in memory, float32 in
// registers.  A conversion to a narrower type rounds to nearest even, once, where a result is stored.
#pragma once
#include "trl_common.h"

typedef __bf16 trl_bf16;
typedef _Float16 trl_f16;

template <typename T>
struct TrlIo {
  static constexpr int V = 16 / (int)sizeof(T);      // elements of one 16 B access
};

// 16 B of elements from / to an address that is aligned to the element only: gfx950 takes dword accesses of four at any
// address, so rows of odd widths need no scalar path (an access that crosses a cache line costs a second line)
template <typename T>
__device__ __forceinline__ void trl_load16(const T *__restrict__ p, float (&f)[TrlIo<T>::V]) {
  T t[TrlIo<T>::V];
  __builtin_memcpy(t, p, 16);
#pragma unroll
  for (int i = 0; i < TrlIo<T>::V; ++i) f[i] = (float)t[i];
}

template <typename T>
__device__ __forceinline__ void trl_store16(T *__restrict__ p, const float (&f)[TrlIo<T>::V]) {
  T t[TrlIo<T>::V];
#pragma unroll
  for (int i = 0; i < TrlIo<T>::V; ++i) t[i] = (T)f[i];
  __builtin_memcpy(p, t, 16);
}

// `n` elements (1 .. V - 1) of the last, partial access of a row; the others read as `fill`
template <typename T>
__device__ __forceinline__ void trl_load_part(const T *__restrict__ p, int n, float fill, float (&f)[TrlIo<T>::V]) {
#pragma unroll
  for (int i = 0; i < TrlIo<T>::V; ++i) f[i] = i < n ? (float)p[i] : fill;
}

template <typename T>
__device__ __forceinline__ void trl_store_part(T *__restrict__ p, int n, const float (&f)[TrlIo<T>::V]) {
#pragma unroll
  for (int i = 0; i < TrlIo<T>::V; ++i)
    if (i < n) p[i] = (T)f[i];
}

// Sum over W consecutive lanes (a power of two), the same bits in every one of them.  Up to 16 lanes the exchange is a DPP
// operand of the addition itself; 32 and 64 go through the LDS crossbar.
template <int CTRL>
__device__ __forceinline__ float trl_dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}

template <int W>
__device__ __forceinline__ float trl_lanes_sum(float v) {
  if (W >= 2) v += trl_dpp<0xB1>(v);        // quad_perm 1,0,3,2
  if (W >= 4) v += trl_dpp<0x4E>(v);        // quad_perm 2,3,0,1
  if (W >= 8) v += trl_dpp<0x141>(v);       // row_half_mirror
  if (W >= 16) v += trl_dpp<0x140>(v);      // row_mirror
  if (W >= 32) v += __shfl_xor(v, 16, 64);
  if (W >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}

// Instantiates `CALL` with `T` bound to the element type of `dtype` (checked by the caller)
#define TRL_FOR_DTYPE(dtype, ...)                       \
  do {                                                  \
    if ((dtype) == TRL_F32) {                           \
      using T = float;                                  \
      __VA_ARGS__;                                      \
    } else if ((dtype) == TRL_BF16) {                   \
      using T = trl_bf16;                               \
      __VA_ARGS__;                                      \
    } else {                                            \
      using T = trl_f16;                                \
      __VA_ARGS__;                                      \
    }                                                   \
  } while (0)

static inline bool trl_float_dtype(int32_t dtype) { return dtype == TRL_F32 || dtype == TRL_BF16 || dtype == TRL_F16; }
