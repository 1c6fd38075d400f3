// Shared pieces of the token operators (layernorm.hip, dropout.hip, mha_fwd.hip, mha_bwd.hip): element types and loads that need no alignment
// beyond the element's own.
#pragma once
#include "common.h"

#define PDAE_DT_F32 0
#define PDAE_DT_BF16 1

typedef __bf16 tk_bf16;
typedef float tk_f32x2 __attribute__((ext_vector_type(2)));
typedef float tk_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned tk_u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 tk_bf16x2 __attribute__((ext_vector_type(2)));

static inline bool tk_dtype_ok(int dt) { return dt == PDAE_DT_F32 || dt == PDAE_DT_BF16; }
static inline size_t tk_size(int dt) { return dt == PDAE_DT_F32 ? 4 : 2; }
static inline bool tk_aligned(const void* p, int dt) { return (((uintptr_t)p) & (tk_size(dt) - 1)) == 0; }

// Two fp32 values rounded to nearest-even bf16, the first one in the low half (v_cvt_pk_bf16_f32).
__device__ __forceinline__ unsigned tk_pack2(float a, float b) {
  const tk_f32x2 v = {a, b};
  return __builtin_bit_cast(unsigned, __builtin_convertvector(v, tk_bf16x2));
}

// Eight consecutive elements of type T as fp32.  Loads and stores are 16-byte instructions at whatever address the element's alignment allows
// (global memory takes them unaligned): rows of an odd length and views at odd offsets run on the same path as aligned ones.
template <typename T> struct TkVec;
template <> struct TkVec<float> {
  __device__ static __forceinline__ void load8(const float* p, float (&v)[8]) { __builtin_memcpy(v, p, 32); }
  __device__ static __forceinline__ void store8(float* p, const float (&v)[8]) { __builtin_memcpy(p, v, 32); }
  __device__ static __forceinline__ float load(const float* p) { return *p; }
  __device__ static __forceinline__ void store(float* p, float v) { *p = v; }
};
template <> struct TkVec<tk_bf16> {
  __device__ static __forceinline__ void load8(const tk_bf16* p, float (&v)[8]) {
    unsigned w[4];
    __builtin_memcpy(w, p, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[2 * j] = __uint_as_float(w[j] << 16); v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u); }
  }
  __device__ static __forceinline__ void store8(tk_bf16* p, const float (&v)[8]) {
    unsigned w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = tk_pack2(v[2 * j], v[2 * j + 1]);
    __builtin_memcpy(p, w, 16);
  }
  __device__ static __forceinline__ float load(const tk_bf16* p) { return (float)*p; }
  __device__ static __forceinline__ void store(tk_bf16* p, float v) { *p = (tk_bf16)v; }
};
