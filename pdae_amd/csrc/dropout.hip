// Dropout from a counter: y = res + x * keep / (1 - p) and its backward dx (+)= dy * keep / (1 - p), the keep mask a pure function of
// (seed, offset, element index) that both directions compute and neither stores.
//
// Generator: Philox2x32, ten rounds (norm.hip uses the same counters for the dropout behind a GroupNorm: one mask definition in the library).
// Element e of the tensor is lane e & 3 of counter e >> 2; a lane is 16 bits, dropped when below round(p * 65536).
//
// Bound: HBM.  One call of ten rounds serves four elements and costs ten 32 x 32 -> 64-bit multiplies (v_mad_u64_u32, quarter rate) and twenty xors,
// ~280 issue cycles per 256 elements and SIMD = 2.2e12 elements/s on the chip: above the rate at which HBM delivers bf16 pairs (4 bytes an element,
// 1.5e12 /s).  Eight elements a thread and pass (16-byte accesses in bf16, 2 x 16 in fp32).  41 M bf16 elements: with a residual 47 us (5.2 TB/s), without 27 us
// (6.1); a large copy moves 5.2.  128 x 2048 fp32: 2.5 us, a launch.
#include "token.h"
#include "kernels.h"

__device__ __forceinline__ void dp_philox(unsigned& a, unsigned& b, unsigned key) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const unsigned long long prod = (unsigned long long)a * 0xD256D193u;
    a = (unsigned)(prod >> 32) ^ key ^ b;
    b = (unsigned)prod;
    key += 0x9E3779B9u;
  }
}
// factors of the four elements of `quad`: 0 or scale
__device__ __forceinline__ void dp_factors(unsigned long long quad, unsigned step, unsigned key, unsigned thr, float scale, float* f) {
  unsigned a = (unsigned)quad, b = step ^ ((unsigned)(quad >> 32) * 0x85EBCA6Bu);
  dp_philox(a, b, key);
  f[0] = (a & 0xffffu) >= thr ? scale : 0.f; f[1] = (a >> 16) >= thr ? scale : 0.f;
  f[2] = (b & 0xffffu) >= thr ? scale : 0.f; f[3] = (b >> 16) >= thr ? scale : 0.f;
}

// RES: add `add` (forward: the residual; backward with accumulation: dx itself).  A dropped element contributes an exact zero, whatever x holds there
// (0 * inf would be NaN): masks select, they do not multiply.
template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_kernel(const T* x, const T* add, T* y, long long n, unsigned step, unsigned key, unsigned thr,
                                                      float scale) {
  const long long n8 = n >> 3, stride = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n8; i += stride) {
    float v[8], r[8], f[8];
    TkVec<T>::load8(x + i * 8, v);
    if (RES) TkVec<T>::load8(add + i * 8, r);
    dp_factors((unsigned long long)i * 2, step, key, thr, scale, f);
    dp_factors((unsigned long long)i * 2 + 1, step, key, thr, scale, f + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) { const float d = f[j] != 0.f ? v[j] * f[j] : 0.f; v[j] = RES ? r[j] + d : d; }
    TkVec<T>::store8(y + i * 8, v);
  }
  const long long e = n8 * 8 + threadIdx.x;                 // the last 0..7 elements
  if (blockIdx.x == 0 && e < n) {
    float f[4];
    dp_factors((unsigned long long)e >> 2, step, key, thr, scale, f);
    const float fe = (e & 3) == 0 ? f[0] : (e & 3) == 1 ? f[1] : (e & 3) == 2 ? f[2] : f[3];
    float d = fe != 0.f ? TkVec<T>::load(x + e) * fe : 0.f;
    if (RES) d += TkVec<T>::load(add + e);
    TkVec<T>::store(y + e, d);
  }
}

template <typename T> static void dropout_launch(const void* x, const void* add, void* y, long long n, unsigned step, unsigned key, unsigned thr, float scale,
                                                 hipStream_t st) {
  const long long want = ((n >> 3) + 255) / 256;
  const int grid = (int)(want < 1 ? 1 : want > 256 * 32 ? 256 * 32 : want);
  if (add) hipLaunchKernelGGL((dropout_kernel<T, true>), dim3(grid), dim3(256), 0, st, (const T*)x, (const T*)add, (T*)y, n, step, key, thr, scale);
  else hipLaunchKernelGGL((dropout_kernel<T, false>), dim3(grid), dim3(256), 0, st, (const T*)x, (const T*)add, (T*)y, n, step, key, thr, scale);
}

int k_dropout(const void* x, const void* add, long long n, float p, unsigned long long seed, unsigned long long offset, void* y, int dtype, hipStream_t st) {
  PDAE_CHECK_ARG(tk_dtype_ok(dtype), "dropout: dtype must be 0 (fp32) or 1 (bf16), got %d", dtype);
  PDAE_CHECK_ARG(n >= 0, "dropout: negative element count");
  PDAE_CHECK_ARG(p >= 0.f && p < 1.f, "dropout: p must lie in [0, 1), got %g", (double)p);
  if (n == 0) return PDAE_OK;
  PDAE_CHECK_ARG(x && y, "dropout: null pointer");
  PDAE_CHECK_ARG(tk_aligned(x, dtype) && tk_aligned(y, dtype) && tk_aligned(add, dtype), "dropout: tensors must be aligned to their element size");
  const unsigned thr = (unsigned)(p * 65536.0f + 0.5f);
  const unsigned key = (unsigned)seed ^ ((unsigned)(seed >> 32) * 0xC2B2AE35u) ^ ((unsigned)(offset >> 32) * 0x27D4EB2Fu);
  const float scale = 1.0f / (1.0f - p);
  if (dtype == PDAE_DT_F32) dropout_launch<float>(x, add, y, n, (unsigned)offset, key, thr, scale, st);
  else dropout_launch<tk_bf16>(x, add, y, n, (unsigned)offset, key, thr, scale, st);
  return pdae_launch_status("dropout");
}
