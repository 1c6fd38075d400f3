// Layer norm over rows: y = (x - mu) rstd gamma + beta, mu / rstd over the C channels of a row (biased variance), and its backward
//     g = dy gamma;  dx = rstd (g - mean(g) - xh mean(g xh)) (+ add);  dgamma = sum_rows dy xh;  dbeta = sum_rows dy,   xh = (x - mu) rstd.
//
// Bound: HBM (forward one read and one write of the tensor, backward two reads and one write).  A row is read ONCE and lives in registers between its
// reductions: a wave owns a row (WPR = 1: short rows, four rows a block, no barrier) or the block's four waves share it (WPR = 4).  NV vectors of eight
// elements a lane; rows longer than 4 * 64 * 8 * 8 = 16384 channels are streamed from L2 a second and third time (NV = 0).
// The variance is taken from the deviations (two passes over registers), not from E[x^2] - E[x]^2, which loses what a large mean leaves.
//
// Weight gradients: every block walks a fixed set of rows and keeps sum dy xh / sum dy of its lanes' own channels in registers; it leaves ONE partial row per
// block, and a second launch adds the partial rows in a fixed order (no atomics: bit-identical from run to run).
#include "token.h"
#include "kernels.h"

#define LN_T 256
#define LN_MAXB 1024           // partial rows of the weight gradients (blocks of the backward launch)

template <int WPR> __device__ __forceinline__ float ln_sum(float v, float* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  if constexpr (WPR == 4) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

// Elements of a row: nv = C / 8 whole vectors (vector i of lane `lane` is number lane + i * lanes) and C % 8 single elements on the first lanes.
template <typename T, int WPR, int NV>
__global__ void __launch_bounds__(LN_T) layernorm_fwd_kernel(const T* __restrict__ x, long long ldx, const float* __restrict__ gamma,
                                                             const float* __restrict__ beta, int R, int C, float eps, T* __restrict__ y, long long ldy,
                                                             float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float red[4];
  constexpr int LANES = 64 * WPR, RPB = 4 / WPR;
  const int lane = threadIdx.x % LANES, row = blockIdx.x * RPB + threadIdx.x / LANES;
  if (row >= R) return;                                    // WPR == 4: never (one row a block)
  const int nv = C >> 3, tail = C & 7, te = nv * 8 + lane;
  const T* xr = x + (long long)row * ldx;
  T* yr = y + (long long)row * ldy;
  const float n = (float)C;                                // (divided by, not multiplied with its reciprocal: the mean of a constant row is exact)
  const bool has = lane < tail;
  const float xt = has ? TkVec<T>::load(xr + te) : 0.f;
  float v[NV > 0 ? NV : 1][8];
  float s = xt;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane + i * LANES;
      if (c < nv) TkVec<T>::load8(xr + c * 8, v[i]);
      else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[i][j];
    }
  } else {
    for (int c = lane; c < nv; c += LANES) {
      TkVec<T>::load8(xr + c * 8, v[0]);
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[0][j];
    }
  }
  const float mu = ln_sum<WPR>(s, red) / n;
  float q = has ? (xt - mu) * (xt - mu) : 0.f;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + i * LANES < nv) {
#pragma unroll
        for (int j = 0; j < 8; ++j) { const float d = v[i][j] - mu; q += d * d; }
      }
  } else {
    for (int c = lane; c < nv; c += LANES) {
      TkVec<T>::load8(xr + c * 8, v[0]);
#pragma unroll
      for (int j = 0; j < 8; ++j) { const float d = v[0][j] - mu; q += d * d; }
    }
  }
  const float rs = 1.0f / sqrtf(ln_sum<WPR>(q, red) / n + eps);
  if (lane == 0) {
    if (mean) mean[row] = mu;
    if (rstd) rstd[row] = rs;
  }
  auto emit = [&](int c, const float (&e)[8]) {
    float g[8], b[8], o[8];
    if (gamma) TkVec<float>::load8(gamma + c * 8, g);
    if (beta) TkVec<float>::load8(beta + c * 8, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) { o[j] = (e[j] - mu) * rs; if (gamma) o[j] *= g[j]; if (beta) o[j] += b[j]; }
    TkVec<T>::store8(yr + c * 8, o);
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + i * LANES < nv) emit(lane + i * LANES, v[i]);
  } else {
    for (int c = lane; c < nv; c += LANES) { TkVec<T>::load8(xr + c * 8, v[0]); emit(c, v[0]); }
  }
  if (has) TkVec<T>::store(yr + te, (xt - mu) * rs * (gamma ? gamma[te] : 1.f) + (beta ? beta[te] : 0.f));
}

// part: [gridDim.x][2][C] partial sums of dy xh and dy (written only when WG).  With NV == 0 (streamed rows) the block adds its rows into its own
// partial row in memory: every channel of it belongs to one lane, so no other thread touches it.
template <typename T, int WPR, int NV, bool WG>
__global__ void __launch_bounds__(LN_T) layernorm_bwd_kernel(const T* __restrict__ x, long long ldx, const float* __restrict__ gamma,
                                                             const float* __restrict__ mean, const float* __restrict__ rstd, const T* __restrict__ dy,
                                                             long long lddy, const T* add, long long ldadd, int R, int C, T* dx, long long lddx,
                                                             float* __restrict__ part) {
  __shared__ float red[8];
  __shared__ float comb[WPR == 1 && WG && NV > 0 ? 2 * 64 * 9 : 1];
  constexpr int LANES = 64 * WPR, RPB = 4 / WPR, NR = NV > 0 ? NV : 1;
  const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
  const int nv = C >> 3, tail = C & 7, te = nv * 8 + lane;
  const float n = (float)C;                                // (divided by, not multiplied with its reciprocal: the mean of a constant row is exact)
  const bool has = lane < tail;
  float ag[NR][8], ab[NR][8], agt = 0.f, abt = 0.f;
  float* pg = part + (size_t)blockIdx.x * 2 * C;
  float* pb = pg + C;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) ag[i][j] = ab[i][j] = 0.f;
  } else if constexpr (WG) {
    const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int c = lane; c < nv; c += LANES) { TkVec<float>::store8(pg + c * 8, z); TkVec<float>::store8(pb + c * 8, z); }
  }
  for (long long row0 = (long long)blockIdx.x * RPB; row0 < R; row0 += (long long)gridDim.x * RPB) {
    const long long row = row0 + sub;
    if (row >= R) break;                                   // WPR == 4: never (whole blocks)
    const T* xr = x + row * ldx;
    const T* dr = dy + row * lddy;
    const T* ar = add ? add + row * ldadd : nullptr;
    T* or_ = dx + row * lddx;
    const float mu = mean[row], rs = rstd[row];
    float xh[NR][8], g[NR][8];
    float s1 = 0.f, s2 = 0.f, xt = 0.f, gt = 0.f;
    if (has) {
      const float d = TkVec<T>::load(dr + te);
      xt = (TkVec<T>::load(xr + te) - mu) * rs;
      gt = gamma ? d * gamma[te] : d;
      s1 = gt; s2 = gt * xt;
      agt += d * xt; abt += d;
    }
    auto take = [&](int c, float (&xv)[8], float (&gv)[8]) {          // xv: xh, gv: dy gamma; returns with the row sums updated
      TkVec<T>::load8(xr + c * 8, xv);
      TkVec<T>::load8(dr + c * 8, gv);
    };
    auto weigh = [&](int c, float (&xv)[8], float (&gv)[8], float* accg, float* accb) {
      float gm[8];
      if (gamma) TkVec<float>::load8(gamma + c * 8, gm);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xv[j] = (xv[j] - mu) * rs;
        if (WG) { accg[j] += gv[j] * xv[j]; accb[j] += gv[j]; }
        if (gamma) gv[j] *= gm[j];
        s1 += gv[j]; s2 += gv[j] * xv[j];
      }
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (lane + i * LANES < nv) take(lane + i * LANES, xh[i], g[i]);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (lane + i * LANES < nv) weigh(lane + i * LANES, xh[i], g[i], ag[i], ab[i]);
    } else {
      for (int c = lane; c < nv; c += LANES) {
        float pgv[8], pbv[8];
        take(c, xh[0], g[0]);
        if (WG) { TkVec<float>::load8(pg + c * 8, pgv); TkVec<float>::load8(pb + c * 8, pbv); }
        weigh(c, xh[0], g[0], pgv, pbv);
        if (WG) { TkVec<float>::store8(pg + c * 8, pgv); TkVec<float>::store8(pb + c * 8, pbv); }
      }
    }
    const float m1 = ln_sum<WPR>(s1, red) / n, m2 = ln_sum<WPR>(s2, red + 4) / n;
    auto emit = [&](int c, const float (&xv)[8], const float (&gv)[8]) {
      float o[8], a[8];
      if (ar) TkVec<T>::load8(ar + c * 8, a);
#pragma unroll
      for (int j = 0; j < 8; ++j) { o[j] = rs * (gv[j] - m1 - xv[j] * m2); if (ar) o[j] += a[j]; }
      TkVec<T>::store8(or_ + c * 8, o);
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (lane + i * LANES < nv) emit(lane + i * LANES, xh[i], g[i]);
    } else {
      for (int c = lane; c < nv; c += LANES) {
        float gm[8];
        take(c, xh[0], g[0]);
        if (gamma) TkVec<float>::load8(gamma + c * 8, gm);
#pragma unroll
        for (int j = 0; j < 8; ++j) { xh[0][j] = (xh[0][j] - mu) * rs; if (gamma) g[0][j] *= gm[j]; }
        emit(c, xh[0], g[0]);
      }
    }
    if (has) TkVec<T>::store(or_ + te, rs * (gt - m1 - xt * m2) + (ar ? TkVec<T>::load(ar + te) : 0.f));
  }
  if constexpr (WG) {
    if constexpr (WPR == 4) {
      if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (lane + i * LANES < nv) { TkVec<float>::store8(pg + (lane + i * LANES) * 8, ag[i]); TkVec<float>::store8(pb + (lane + i * LANES) * 8, ab[i]); }
      }
      if (has) { pg[te] = agt; pb[te] = abt; }
    } else {                                               // four waves, one partial row: added in wave order through LDS, a vector at a time
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        for (int w = 0; w < 4; ++w) {
          if (sub == w) {
            float* c0 = comb + lane * 9;
            float* c1 = comb + (64 + lane) * 9;
#pragma unroll
            for (int j = 0; j < 8; ++j) { c0[j] = w ? c0[j] + ag[i][j] : ag[i][j]; c1[j] = w ? c1[j] + ab[i][j] : ab[i][j]; }
            if (w == 3 && lane + i * 64 < nv) {
#pragma unroll
              for (int j = 0; j < 8; ++j) { pg[(lane + i * 64) * 8 + j] = c0[j]; pb[(lane + i * 64) * 8 + j] = c1[j]; }
            }
          }
          __syncthreads();
        }
      }
      for (int w = 0; w < 4; ++w) {
        if (sub == w) {
          comb[lane * 9] = w ? comb[lane * 9] + agt : agt;
          comb[(64 + lane) * 9] = w ? comb[(64 + lane) * 9] + abt : abt;
          if (w == 3 && has) { pg[te] = comb[lane * 9]; pb[te] = comb[(64 + lane) * 9]; }
        }
        __syncthreads();
      }
    }
  }
}

// dgamma / dbeta (+)= sums of the nb partial rows: 32 columns x 32 slices a block, the slices added in order through LDS.
__global__ void __launch_bounds__(1024) layernorm_wsum_kernel(const float* __restrict__ part, int nb, int C, float* dgamma, float* dbeta, int acc) {
  __shared__ float sm[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), sl = threadIdx.x >> 5;
  float s = 0.f;
  if (col < 2 * C) {
#pragma unroll 8
    for (int b = sl; b < nb; b += 32) s += part[(size_t)b * 2 * C + col];
  }
  sm[sl][threadIdx.x & 31] = s;
  __syncthreads();
  if (sl == 0 && col < 2 * C) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += sm[k][threadIdx.x];
    float* d = col < C ? dgamma : dbeta;
    const int c = col < C ? col : col - C;
    if (d) d[c] = acc ? d[c] + t : t;
  }
}

// Row form by length: one wave a row while it fits 4 vectors a lane (2048 channels), else four waves a row up to 8 vectors, else streamed.
struct LnForm { int wpr, nv; };
static LnForm ln_form(int C) {
  const int nv = C / 8;
  if (nv <= 64 * 4) return {1, nv <= 64 ? 1 : nv <= 128 ? 2 : nv <= 192 ? 3 : 4};
  if (nv <= 256 * 8) return {4, nv <= 512 ? 2 : nv <= 1024 ? 4 : 8};
  return {4, 0};
}
static int ln_blocks(int R, int C) {
  const LnForm f = ln_form(C);
  const int want = f.wpr == 1 ? cdiv(R, 4) : R;
  return want < LN_MAXB ? want : LN_MAXB;
}
size_t k_layernorm_workspace_bytes(int R, int C) { return R > 0 && C > 0 ? (size_t)ln_blocks(R, C) * 2 * C * sizeof(float) : 0; }

#define LN_FORMS(X)                                                                                           \
  switch (f.wpr * 16 + f.nv) {                                                                                \
    case 17: X(1, 1); break;                                                                                  \
    case 18: X(1, 2); break;                                                                                  \
    case 19: X(1, 3); break;                                                                                  \
    case 20: X(1, 4); break;                                                                                  \
    case 66: X(4, 2); break;                                                                                  \
    case 68: X(4, 4); break;                                                                                  \
    case 72: X(4, 8); break;                                                                                  \
    default: X(4, 0); break;                                                                                  \
  }

template <typename T> static void ln_fwd(const void* x, long long ldx, const float* gamma, const float* beta, int R, int C, float eps, void* y, long long ldy,
                                         float* mean, float* rstd, hipStream_t st) {
  const LnForm f = ln_form(C);
  const int grid = f.wpr == 1 ? cdiv(R, 4) : R;
#define LN_X(W, V) hipLaunchKernelGGL((layernorm_fwd_kernel<T, W, V>), dim3(grid), dim3(LN_T), 0, st, (const T*)x, ldx, gamma, beta, R, C, eps, (T*)y, ldy, mean, rstd)
  LN_FORMS(LN_X)
#undef LN_X
}
template <typename T, bool WG> static void ln_bwd(const void* x, long long ldx, const float* gamma, const float* mean, const float* rstd, const void* dy, long long lddy,
                                                  const void* add, long long ldadd, int R, int C, void* dx, long long lddx, float* ws, hipStream_t st) {
  const LnForm f = ln_form(C);
  const int grid = ln_blocks(R, C);
#define LN_X(W, V)                                                                                                                                       \
  hipLaunchKernelGGL((layernorm_bwd_kernel<T, W, V, WG>), dim3(grid), dim3(LN_T), 0, st, (const T*)x, ldx, gamma, mean, rstd, (const T*)dy, lddy, (const T*)add, \
                     ldadd, R, C, (T*)dx, lddx, ws)
  LN_FORMS(LN_X)
#undef LN_X
}

int k_layernorm_fwd(const void* x, long long ldx, const float* gamma, const float* beta, int R, int C, float eps, void* y, long long ldy, float* mean, float* rstd,
                    int dtype, hipStream_t st) {
  PDAE_CHECK_ARG(tk_dtype_ok(dtype), "layernorm: dtype must be 0 (fp32) or 1 (bf16), got %d", dtype);
  PDAE_CHECK_ARG(R >= 0 && C > 0, "layernorm: need R >= 0 and C > 0 (got %d, %d)", R, C);
  PDAE_CHECK_ARG(eps >= 0.f, "layernorm: eps must not be negative");
  PDAE_CHECK_ARG(ldx >= C && ldy >= C, "layernorm: a row stride is shorter than the row (%lld, %lld < %d)", ldx, ldy, C);
  if (R == 0) return PDAE_OK;
  PDAE_CHECK_ARG(x && y, "layernorm_fwd: null pointer");
  PDAE_CHECK_ARG(tk_aligned(x, dtype) && tk_aligned(y, dtype), "layernorm: tensors must be aligned to their element size");
  if (dtype == PDAE_DT_F32) ln_fwd<float>(x, ldx, gamma, beta, R, C, eps, y, ldy, mean, rstd, st);
  else ln_fwd<tk_bf16>(x, ldx, gamma, beta, R, C, eps, y, ldy, mean, rstd, st);
  return pdae_launch_status("layernorm_fwd");
}

int k_layernorm_bwd(const void* x, long long ldx, const float* gamma, const float* mean, const float* rstd, const void* dy, long long lddy, const void* add,
                    long long ldadd, int R, int C, void* dx, long long lddx, float* dgamma, float* dbeta, int acc_param, void* ws, size_t ws_bytes, int dtype,
                    hipStream_t st) {
  PDAE_CHECK_ARG(tk_dtype_ok(dtype), "layernorm: dtype must be 0 (fp32) or 1 (bf16), got %d", dtype);
  PDAE_CHECK_ARG(R >= 0 && C > 0, "layernorm: need R >= 0 and C > 0 (got %d, %d)", R, C);
  PDAE_CHECK_ARG(ldx >= C && lddy >= C && lddx >= C && (!add || ldadd >= C), "layernorm: a row stride is shorter than the row");
  const bool wg = dgamma || dbeta;
  if (R > 0) {
    PDAE_CHECK_ARG(x && mean && rstd && dy && dx, "layernorm_bwd: null pointer");
    PDAE_CHECK_ARG(tk_aligned(x, dtype) && tk_aligned(dy, dtype) && tk_aligned(dx, dtype) && tk_aligned(add, dtype),
                   "layernorm: tensors must be aligned to their element size");
    PDAE_CHECK_ARG(!wg || (ws && ws_bytes >= k_layernorm_workspace_bytes(R, C)), "layernorm_bwd: weight gradients need %zu bytes of workspace (got %zu)",
                   k_layernorm_workspace_bytes(R, C), ws ? ws_bytes : (size_t)0);
    if (dtype == PDAE_DT_F32) {
      if (wg) ln_bwd<float, true>(x, ldx, gamma, mean, rstd, dy, lddy, add, ldadd, R, C, dx, lddx, (float*)ws, st);
      else ln_bwd<float, false>(x, ldx, gamma, mean, rstd, dy, lddy, add, ldadd, R, C, dx, lddx, (float*)ws, st);
    } else {
      if (wg) ln_bwd<tk_bf16, true>(x, ldx, gamma, mean, rstd, dy, lddy, add, ldadd, R, C, dx, lddx, (float*)ws, st);
      else ln_bwd<tk_bf16, false>(x, ldx, gamma, mean, rstd, dy, lddy, add, ldadd, R, C, dx, lddx, (float*)ws, st);
    }
    if (int e = pdae_launch_status("layernorm_bwd")) return e;
  }
  if (!wg || (R == 0 && acc_param)) return PDAE_OK;
  hipLaunchKernelGGL(layernorm_wsum_kernel, dim3(cdiv(2 * (long long)C, 32)), dim3(1024), 0, st, (const float*)ws, R > 0 ? ln_blocks(R, C) : 0, C, dgamma, dbeta, acc_param);
  return pdae_launch_status("layernorm_wsum");
}
