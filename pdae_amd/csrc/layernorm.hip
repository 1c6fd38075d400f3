// Layer norm over rows: y = (x - mu) rstd gamma + beta, mu / rstd over the C channels of a row (biased variance), and its backward
//     g = dy gamma;  dx = rstd (g - mean(g) - xh mean(g xh)) (+ add);  dgamma = sum_rows dy xh;  dbeta = sum_rows dy,   xh = (x - mu) rstd.
//
// Bound: HBM (forward one read and one write of the tensor, backward two reads and one write).  A row is read ONCE and lives in registers between its
// reductions: L lanes share it (8 .. 64 of a wave, or a block of 256 / 512), NV vectors of eight elements a lane; only rows beyond 16384 channels are
// streamed again from L2 (NV = 0).  65536 x 1536 bf16: forward 75 us, backward 133 us + 5 for the partial rows
// (5.3 / 4.6 TB/s; a large copy on this chip moves 5.2; first ten passes 77 and 135 .. 141).  128 x 2048 fp32: 3.6 + 3.8 us, two launches.  9001 x 1027 bf16 forward: 11 .. 12 us
// (3.3 TB/s): 8192 rows are resident, one a wave, and the last 809 run alone.
// The variance is taken from the deviations (two passes over registers), not from E[x^2] - E[x]^2, which loses what a large mean leaves.
//
// Weight gradients: every block walks a fixed set of rows and keeps sum dy xh / sum dy of its lanes' own channels in registers; it leaves ONE partial row per
// block, and a second launch adds the partial rows in a fixed order (no atomics: bit-identical from run to run).  Few rows are latency, not bytes: one launch,
// in which blocks of their own add up the columns.
#include "token.h"
#include "kernels.h"

// sum over the L lanes that share a row (L <= 64: neighbouring lanes of a wave; else the whole block of L threads)
template <int L> __device__ __forceinline__ float ln_sum(float v, float* red) {
#pragma unroll
  for (int off = (L < 64 ? L : 64) / 2; off > 0; off >>= 1) v += __shfl_xor(v, off);
  if constexpr (L > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
    if constexpr (L == 512) v += (red[4] + red[5]) + (red[6] + red[7]);
  }
  return v;
}
#define LN_THREADS(L) ((L) > 256 ? (L) : 256)

// Elements of a row: nv = C / 8 whole vectors (vector i of lane `lane` is number lane + i * lanes) and C % 8 single elements on the first lanes.
// y may be x: a lane writes the elements that it has read, after the row's sums (x and y are not declared apart).
template <typename T, int L, int NV>
__global__ void __launch_bounds__(LN_THREADS(L)) layernorm_fwd_kernel(const T* x, long long ldx, const float* __restrict__ gamma,
                                                             const float* __restrict__ beta, int R, int C, float eps, T* y, long long ldy,
                                                             float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float red[8];
  constexpr int RPB = LN_THREADS(L) / L;
  const int lane = threadIdx.x % L, row = blockIdx.x * RPB + threadIdx.x / L;
  if (row >= R) return;                                    // (whole lane groups; L > 64: never, one row a block)
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
      const int c = lane + i * L;
      if (c < nv) TkVec<T>::load8(xr + c * 8, v[i]);
      else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[i][j];
    }
  } else {
    for (int c = lane; c < nv; c += L) {
      TkVec<T>::load8(xr + c * 8, v[0]);
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[0][j];
    }
  }
  const float mu = ln_sum<L>(s, red) / n;
  float q = has ? (xt - mu) * (xt - mu) : 0.f;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + i * L < nv) {
#pragma unroll
        for (int j = 0; j < 8; ++j) { const float d = v[i][j] - mu; q += d * d; }
      }
  } else {
    for (int c = lane; c < nv; c += L) {
      TkVec<T>::load8(xr + c * 8, v[0]);
#pragma unroll
      for (int j = 0; j < 8; ++j) { const float d = v[0][j] - mu; q += d * d; }
    }
  }
  const float rs = 1.0f / sqrtf(ln_sum<L>(q, red) / n + eps);
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
      if (lane + i * L < nv) emit(lane + i * L, v[i]);
  } else {
    for (int c = lane; c < nv; c += L) { TkVec<T>::load8(xr + c * 8, v[0]); emit(c, v[0]); }
  }
  if (has) TkVec<T>::store(yr + te, (xt - mu) * rs * (gamma ? gamma[te] : 1.f) + (beta ? beta[te] : 0.f));
}

// Eight elements as they lie in memory (four or eight dwords), and as fp32.
template <typename T> struct LnRaw { unsigned w[sizeof(T) * 2]; };
template <typename T> __device__ __forceinline__ void ln_read(const T* p, LnRaw<T>& r) { __builtin_memcpy(r.w, p, 8 * sizeof(T)); }
template <typename T> __device__ __forceinline__ float ln_elem(const LnRaw<T>& r, int j) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[j]);
  else return __uint_as_float(j & 1 ? r.w[j / 2] & 0xffff0000u : r.w[j / 2] << 16);
}

// part: [gridDim.x][2][C] partial sums of dy xh and dy (written only when WG).  A row is held as it was read and converted twice (row sums, then dx): its fp32
// forms would take four times the registers, and the row AFTER it could not be in flight meanwhile -- with one row at a time a wave waited for HBM
// on every row (65536 x 1536 bf16: 239 us, 2.5 TB/s).
template <typename T, int L, int NV, bool WG>
__device__ __forceinline__ void ln_bwd_rows(const T* __restrict__ x, long long ldx, const float* __restrict__ gamma, const float* __restrict__ mean,
                                            const float* __restrict__ rstd, const T* __restrict__ dy, long long lddy, const T* add, long long ldadd, int R, int C, T* dx,
                                            long long lddx, float* __restrict__ part, int blocks) {
  __shared__ float red[16];
  __shared__ float comb[L <= 64 && WG ? 2 * L * 9 : 1];
  constexpr int RPB = LN_THREADS(L) / L;
  const int lane = threadIdx.x % L, sub = L > 64 ? 0 : L == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : (int)threadIdx.x / L;
  const int nv = C >> 3, tail = C & 7, te = nv * 8 + lane;
  const float n = (float)C;
  const bool has = lane < tail;
  float ag[NV][8], ab[NV][8], gm[NV][8], agt = 0.f, abt = 0.f, gmt = 1.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) { ag[i][j] = ab[i][j] = 0.f; gm[i][j] = 1.f; }
    if (gamma && lane + i * L < nv) TkVec<float>::load8(gamma + (lane + i * L) * 8, gm[i]);
  }
  if (gamma && has) gmt = gamma[te];
  LnRaw<T> qx[2][NV], qd[2][NV];
  float tx[2], td[2], mu[2], rs[2];
  const long long step = (long long)blocks * RPB;
  auto fetch = [&](long long row, LnRaw<T> (&rx)[NV], LnRaw<T> (&rd)[NV], float& ex, float& ed, float& m, float& r) __attribute__((always_inline)) {
    const T* xr = x + row * ldx;
    const T* dr = dy + row * lddy;
    m = mean[row]; r = rstd[row];
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + i * L < nv) { ln_read(xr + (lane + i * L) * 8, rx[i]); ln_read(dr + (lane + i * L) * 8, rd[i]); }
      else {
#pragma unroll
        for (int j = 0; j < (int)(sizeof(T) * 2); ++j) rx[i].w[j] = rd[i].w[j] = 0;
      }
    ex = has ? TkVec<T>::load(xr + te) : 0.f;
    ed = has ? TkVec<T>::load(dr + te) : 0.f;
  };
  auto work = [&](long long row, LnRaw<T> (&rx)[NV], LnRaw<T> (&rd)[NV], float ex, float ed, float m, float r) __attribute__((always_inline)) {
    float s1 = 0.f, s2 = 0.f;
    float xt = 0.f, gt = 0.f;
    if (has) {
      xt = (ex - m) * r; gt = ed * gmt;
      s1 = gt; s2 = gt * xt;
      agt += ed * xt; abt += ed;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + i * L < nv) {                          // (lanes past the row's end hold zeros, but (0 - mu) rstd is none)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float xh = (ln_elem(rx[i], j) - m) * r, d = ln_elem(rd[i], j), g = d * gm[i][j];
          if (WG) { ag[i][j] += d * xh; ab[i][j] += d; }
          s1 += g; s2 += g * xh;
        }
      }
    const float m1 = ln_sum<L>(s1, red) / n, m2 = ln_sum<L>(s2, red + 8) / n;
    const T* ar = add ? add + row * ldadd : nullptr;
    T* orow = dx + row * lddx;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + i * L < nv) {
#pragma unroll
        for (int j = 0; j < (int)(sizeof(T) * 2); ++j) { asm volatile("" : "+v"(rx[i].w[j])); asm volatile("" : "+v"(rd[i].w[j])); }      // convert anew, do not keep
        const int c = (lane + i * L) * 8;
        float o[8], e[8];
        if (ar) TkVec<T>::load8(ar + c, e);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float xh = (ln_elem(rx[i], j) - m) * r, g = ln_elem(rd[i], j) * gm[i][j];
          o[j] = r * (g - m1 - xh * m2);
          if (ar) o[j] += e[j];
        }
        TkVec<T>::store8(orow + c, o);
      }
    if (has) TkVec<T>::store(orow + te, r * (gt - m1 - xt * m2) + (ar ? TkVec<T>::load(ar + te) : 0.f));
  };
  const long long row0 = (long long)blockIdx.x * RPB + sub;
  if constexpr (sizeof(T) == 4 && L == 512 && WG) {        // a second row of 16384 fp32 channels finds no registers (2000 rows: 126 us spilled, 96 one by one)
    for (long long row = row0; row < R; row += step) {
      fetch(row, qx[0], qd[0], tx[0], td[0], mu[0], rs[0]);
      work(row, qx[0], qd[0], tx[0], td[0], mu[0], rs[0]);
    }
  } else {
    // two rows in turn, the next one in flight while this one is worked on (L > 64: all waves of the block walk the same rows)
    if (row0 < R) fetch(row0, qx[0], qd[0], tx[0], td[0], mu[0], rs[0]);
    for (long long row = row0; row < R; row += 2 * step) {
      if (row + step < R) fetch(row + step, qx[1], qd[1], tx[1], td[1], mu[1], rs[1]);
      work(row, qx[0], qd[0], tx[0], td[0], mu[0], rs[0]);
      if (row + 2 * step < R) fetch(row + 2 * step, qx[0], qd[0], tx[0], td[0], mu[0], rs[0]);
      if (row + step < R) work(row + step, qx[1], qd[1], tx[1], td[1], mu[1], rs[1]);
    }
  }
  if constexpr (WG) {
    float* pg = part + (size_t)blockIdx.x * 2 * C;
    float* pb = pg + C;
    if constexpr (L > 64) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (lane + i * L < nv) { TkVec<float>::store8(pg + (lane + i * L) * 8, ag[i]); TkVec<float>::store8(pb + (lane + i * L) * 8, ab[i]); }
      if (has) { pg[te] = agt; pb[te] = abt; }
    } else {
      // first the lane groups of a wave, then the four waves in wave order through LDS, a vector at a time
      const int w = threadIdx.x >> 6;
#pragma unroll
      for (int off = L; off < 64; off <<= 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) { ag[i][j] += __shfl_xor(ag[i][j], off); ab[i][j] += __shfl_xor(ab[i][j], off); }
        agt += __shfl_xor(agt, off); abt += __shfl_xor(abt, off);
      }
      const bool mine = (threadIdx.x & 63) < L;
#pragma unroll
      for (int i = 0; i <= NV; ++i) {                       // i == NV: the C % 8 single channels
        for (int k = 0; k < 4; ++k) {
          if (w == k && mine) {
            float* c0 = comb + lane * 9;
            float* c1 = comb + (L + lane) * 9;
#pragma unroll
            for (int j = 0; j < (i < NV ? 8 : 1); ++j) {
              const float g = i < NV ? ag[i < NV ? i : 0][j] : agt, b = i < NV ? ab[i < NV ? i : 0][j] : abt;
              c0[j] = k ? c0[j] + g : g; c1[j] = k ? c1[j] + b : b;
            }
            if (k == 3 && i < NV && lane + i * L < nv) {
#pragma unroll
              for (int j = 0; j < 8; ++j) { pg[(lane + i * L) * 8 + j] = c0[j]; pb[(lane + i * L) * 8 + j] = c1[j]; }
            }
            if (k == 3 && i == NV && has) { pg[te] = c0[0]; pb[te] = c1[0]; }
          }
          __syncthreads();
        }
      }
    }
  }
}

template <typename T, int L, int NV, bool WG>
__global__ void __launch_bounds__(LN_THREADS(L)) layernorm_bwd_kernel(const T* __restrict__ x, long long ldx, const float* __restrict__ gamma,
                                                             const float* __restrict__ mean, const float* __restrict__ rstd, const T* __restrict__ dy,
                                                             long long lddy, const T* add, long long ldadd, int R, int C, T* dx, long long lddx,
                                                             float* __restrict__ part) {
  ln_bwd_rows<T, L, NV, WG>(x, ldx, gamma, mean, rstd, dy, lddy, add, ldadd, R, C, dx, lddx, part, gridDim.x);
}
// Few rows: one launch.  The first `blocks` blocks take rows as above, the others 32 columns each (8 slices of the rows, added in order) and read x and dy
// of their columns once more.
template <typename T, int L, int NV>
__global__ void __launch_bounds__(256) layernorm_bwd_few_kernel(const T* __restrict__ x, long long ldx, const float* __restrict__ gamma, const float* __restrict__ mean,
                                                                const float* __restrict__ rstd, const T* __restrict__ dy, long long lddy, const T* add,
                                                                long long ldadd, int R, int C, T* dx, long long lddx, int blocks, float* dgamma, float* dbeta,
                                                                int acc) {
  if ((int)blockIdx.x < blocks) {
    ln_bwd_rows<T, L, NV, false>(x, ldx, gamma, mean, rstd, dy, lddy, add, ldadd, R, C, dx, lddx, nullptr, blocks);
    return;
  }
  __shared__ float sg[8][32], sb[8][32];
  const int c = ((int)blockIdx.x - blocks) * 32 + (threadIdx.x & 31), sl = threadIdx.x >> 5;
  float g = 0.f, b = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int row = sl; row < R; row += 8) {
      const float d = TkVec<T>::load(dy + row * lddy + c);
      g += d * ((TkVec<T>::load(x + row * ldx + c) - mean[row]) * rstd[row]);
      b += d;
    }
  }
  sg[sl][threadIdx.x & 31] = g; sb[sl][threadIdx.x & 31] = b;
  __syncthreads();
  if (sl < 2 && c < C) {
    float* to = sl ? dbeta : dgamma;
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += sl ? sb[k][threadIdx.x & 31] : sg[k][threadIdx.x & 31];
    if (to) to[c] = acc ? to[c] + t : t;
  }
}

// Rows too long for registers: the block reads its row twice (the second time from L2) and adds into its own partial row in memory; every channel of
// it belongs to one lane, so no other thread touches it.
template <typename T, bool WG>
__global__ void __launch_bounds__(512) layernorm_bwd_long_kernel(const T* __restrict__ x, long long ldx, const float* __restrict__ gamma,
                                                                 const float* __restrict__ mean, const float* __restrict__ rstd, const T* __restrict__ dy,
                                                                 long long lddy, const T* add, long long ldadd, int R, int C, T* dx, long long lddx,
                                                                 float* __restrict__ part) {
  __shared__ float red[16];
  const float n = (float)C;
  const int t = threadIdx.x, nv = C >> 3, te = nv * 8 + t;
  const bool has = t < (C & 7);
  float* pg = part + (size_t)blockIdx.x * 2 * C;
  float* pb = pg + C;
  for (long long row = blockIdx.x; row < R; row += gridDim.x) {
    const T* xr = x + row * ldx;
    const T* dr = dy + row * lddy;
    const T* ar = add ? add + row * ldadd : nullptr;
    T* orow = dx + row * lddx;
    const float mu = mean[row], rs = rstd[row];
    const bool one = row == blockIdx.x;                    // the partial row starts with the block's first row
    float s1 = 0.f, s2 = 0.f, xt = 0.f, gt = 0.f;
    if (has) {
      const float d = TkVec<T>::load(dr + te);
      xt = (TkVec<T>::load(xr + te) - mu) * rs;
      gt = gamma ? d * gamma[te] : d;
      s1 = gt; s2 = gt * xt;
      if (WG) { pg[te] = one ? d * xt : pg[te] + d * xt; pb[te] = one ? d : pb[te] + d; }
    }
    for (int c = t; c < nv; c += 512) {
      float xh[8], d[8], gm[8], p[8], q[8];
      TkVec<T>::load8(xr + c * 8, xh);
      TkVec<T>::load8(dr + c * 8, d);
      if (gamma) TkVec<float>::load8(gamma + c * 8, gm);
      if (WG && !one) { TkVec<float>::load8(pg + c * 8, p); TkVec<float>::load8(pb + c * 8, q); }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xh[j] = (xh[j] - mu) * rs;
        p[j] = (one ? 0.f : p[j]) + d[j] * xh[j]; q[j] = (one ? 0.f : q[j]) + d[j];
        const float g = gamma ? d[j] * gm[j] : d[j];
        s1 += g; s2 += g * xh[j];
      }
      if (WG) { TkVec<float>::store8(pg + c * 8, p); TkVec<float>::store8(pb + c * 8, q); }
    }
    const float m1 = ln_sum<512>(s1, red) / n, m2 = ln_sum<512>(s2, red + 8) / n;
    for (int c = t; c < nv; c += 512) {
      float xh[8], d[8], gm[8], e[8], o[8];
      TkVec<T>::load8(xr + c * 8, xh);
      TkVec<T>::load8(dr + c * 8, d);
      if (gamma) TkVec<float>::load8(gamma + c * 8, gm);
      if (ar) TkVec<T>::load8(ar + c * 8, e);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        o[j] = rs * ((gamma ? d[j] * gm[j] : d[j]) - m1 - (xh[j] - mu) * rs * m2);
        if (ar) o[j] += e[j];
      }
      TkVec<T>::store8(orow + c * 8, o);
    }
    if (has) TkVec<T>::store(orow + te, rs * (gt - m1 - xt * m2) + (ar ? TkVec<T>::load(ar + te) : 0.f));
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

// Row form: the smallest group of lanes that holds a row in one vector each (8, 16, 32 or a whole wave up to 512 channels: 64-channel rows on whole
// waves ran at 0.75 TB/s, seven lanes of eight idle), a wave up to 4 vectors a lane (2048 channels; backward, which keeps more state: 3), then four
// waves, eight waves (16384 channels), streamed beyond.  Few rows (fewer blocks than CUs at four rows a block) go to four waves each: 128 rows of
// 2048 fp32, one layer of a latent batch, took 5.0 us forward with one wave a row, 4.0 with four.
struct LnForm { int lanes, nv; };
static LnForm ln_form(int R, int C, bool bwd) {
  const int nv = C / 8;
  if (nv <= 8) return {8, 1};
  if (nv <= 16) return {16, 1};
  if (nv <= 32) return {32, 1};
  if (nv <= 64) return {64, 1};
  if (nv <= 64 * (bwd ? 3 : 4) && (R + 3) / 4 >= 256) return {64, nv <= 128 ? 2 : nv <= 192 ? 3 : 4};
  if (nv <= 256) return {256, 1};
  if (nv <= 512) return {256, 2};
  if (nv <= 1024) return {256, 4};
  if (nv <= 2048) return {512, 4};
  return {512, 0};
}
static int ln_rows_per_block(const LnForm& f) { return f.lanes <= 256 ? 256 / f.lanes : 1; }
// blocks of the backward launch = partial rows of the weight gradients: as many as are resident at once.  More start when the first ones end and run
// their whole share alone: 65536 x 1536 bf16 took 173 us with 768 blocks, 135 with 512
static int ln_blocks(int R, int C) {
  const LnForm f = ln_form(R, C, true);
  const int want = cdiv(R, ln_rows_per_block(f)), most = f.lanes == 512 ? 256 : f.nv == 1 ? 1024 : 512;
  return want < most ? want : most;
}
// One launch up to 1024 rows: reading x and dy of 32 columns in 8 slices takes no longer than the row blocks beside it, and a launch less counts (2048 channels bf16,
// 512 rows 11.6 -> 7.0 us, 1024 rows 16.1 -> 10.4; 2048 rows 18.4 -> 23.4).  The workspace is asked for all the same: what a caller has to hold does not change with this rule.
static bool ln_few(int R, int C) { return R <= 1024 && ln_form(R, C, true).lanes <= 256; }
size_t k_layernorm_workspace_bytes(int R, int C) { return R > 0 && C > 0 ? (size_t)ln_blocks(R, C) * 2 * C * sizeof(float) : 0; }

#define LN_FORMS(X, X4, X0)                                                                                       \
  switch (f.lanes * 8 + f.nv) {                                                                               \
    case 8 * 8 + 1: X(8, 1); break;                                                                           \
    case 16 * 8 + 1: X(16, 1); break;                                                                         \
    case 32 * 8 + 1: X(32, 1); break;                                                                         \
    case 64 * 8 + 1: X(64, 1); break;                                                                         \
    case 64 * 8 + 2: X(64, 2); break;                                                                         \
    case 64 * 8 + 3: X(64, 3); break;                                                                         \
    case 64 * 8 + 4: X4; break;                                                                               \
    case 256 * 8 + 1: X(256, 1); break;                                                                       \
    case 256 * 8 + 2: X(256, 2); break;                                                                       \
    case 256 * 8 + 4: X(256, 4); break;                                                                       \
    case 512 * 8 + 4: X(512, 4); break;                                                                       \
    default: X0; break;                                                                                       \
  }

template <typename T> static void ln_fwd(const void* x, long long ldx, const float* gamma, const float* beta, int R, int C, float eps, void* y, long long ldy,
                                         float* mean, float* rstd, hipStream_t st) {
  const LnForm f = ln_form(R, C, false);
  const int per = ln_rows_per_block(f);
  for (long long r0 = 0; r0 < R; r0 += (long long)per << 22) {                 // (a launch holds fewer than 2^32 threads)
    const int n = (int)(R - r0 < (long long)per << 22 ? R - r0 : (long long)per << 22);
#define LN_X(W, V)                                                                                                                                                  \
  hipLaunchKernelGGL((layernorm_fwd_kernel<T, W, V>), dim3(cdiv(n, per)), dim3(LN_THREADS(W)), 0, st, (const T*)x + r0 * ldx, ldx, gamma, beta, n, C, eps, (T*)y + r0 * ldy, \
                     ldy, mean ? mean + r0 : nullptr, rstd ? rstd + r0 : nullptr)
    LN_FORMS(LN_X, LN_X(64, 4), LN_X(512, 0))
#undef LN_X
  }
}
template <typename T, bool WG> static void ln_bwd(const void* x, long long ldx, const float* gamma, const float* mean, const float* rstd, const void* dy, long long lddy,
                                                  const void* add, long long ldadd, int R, int C, void* dx, long long lddx, float* ws, hipStream_t st) {
  const LnForm f = ln_form(R, C, true);
  const int grid = ln_blocks(R, C);
#define LN_ARGS(TH) dim3(grid), dim3(TH), 0, st, (const T*)x, ldx, gamma, mean, rstd, (const T*)dy, lddy, (const T*)add, ldadd, R, C, (T*)dx, lddx, ws
#define LN_X(W, V) hipLaunchKernelGGL((layernorm_bwd_kernel<T, W, V, WG>), LN_ARGS(LN_THREADS(W)))
#define LN_LONG hipLaunchKernelGGL((layernorm_bwd_long_kernel<T, WG>), LN_ARGS(512))
  LN_FORMS(LN_X, break, LN_LONG)          // (64, 4) is a forward form only
#undef LN_X
#undef LN_LONG
#undef LN_ARGS
}

template <typename T> static void ln_bwd_few(const void* x, long long ldx, const float* gamma, const float* mean, const float* rstd, const void* dy, long long lddy,
                                             const void* add, long long ldadd, int R, int C, void* dx, long long lddx, float* dgamma, float* dbeta, int acc, hipStream_t st) {
  const LnForm f = ln_form(R, C, true);
  const int blocks = ln_blocks(R, C);
#define LN_X(W, V)                                                                                                                                             \
  if constexpr (W <= 256)                                                                                                                                      \
    hipLaunchKernelGGL((layernorm_bwd_few_kernel<T, W, V>), dim3(blocks + cdiv(C, 32)), dim3(256), 0, st, (const T*)x, ldx, gamma, mean, rstd, (const T*)dy, lddy, \
                       (const T*)add, ldadd, R, C, (T*)dx, lddx, blocks, dgamma, dbeta, acc)
  LN_FORMS(LN_X, break, break)
#undef LN_X
}

int k_layernorm_fwd(const void* x, long long ldx, const float* gamma, const float* beta, int R, int C, float eps, void* y, long long ldy, float* mean, float* rstd,
                    int dtype, hipStream_t st) {
  PDAE_CHECK_ARG(tk_dtype_ok(dtype), "layernorm: dtype must be 0 (fp32) or 1 (bf16), got %d", dtype);
  PDAE_CHECK_ARG(R >= 0 && C > 0 && C <= 1 << 24, "layernorm: need R >= 0 and C > 0, C at most 2^24 (got %d, %d)", R, C);
  PDAE_CHECK_ARG(eps >= 0.f, "layernorm: eps must not be negative");
  PDAE_CHECK_ARG(ldx >= C && ldy >= C, "layernorm: a row stride is shorter than the row (%lld, %lld < %d)", ldx, ldy, C);
  if (R == 0) return PDAE_OK;
  PDAE_CHECK_ARG(x && y, "layernorm_fwd: null pointer");
  PDAE_CHECK_ARG(tk_aligned(x, dtype) && tk_aligned(y, dtype), "layernorm: tensors must be aligned to their element size");
  PDAE_CHECK_ARG(y != x || ldy == ldx, "layernorm_fwd: y in the place of x with another row stride");
  if (dtype == PDAE_DT_F32) ln_fwd<float>(x, ldx, gamma, beta, R, C, eps, y, ldy, mean, rstd, st);
  else ln_fwd<tk_bf16>(x, ldx, gamma, beta, R, C, eps, y, ldy, mean, rstd, st);
  return pdae_launch_status("layernorm_fwd");
}

int k_layernorm_bwd(const void* x, long long ldx, const float* gamma, const float* mean, const float* rstd, const void* dy, long long lddy, const void* add,
                    long long ldadd, int R, int C, void* dx, long long lddx, float* dgamma, float* dbeta, int acc_param, void* ws, size_t ws_bytes, int dtype,
                    hipStream_t st) {
  PDAE_CHECK_ARG(tk_dtype_ok(dtype), "layernorm: dtype must be 0 (fp32) or 1 (bf16), got %d", dtype);
  PDAE_CHECK_ARG(R >= 0 && C > 0 && C <= 1 << 24, "layernorm: need R >= 0 and C > 0, C at most 2^24 (got %d, %d)", R, C);
  PDAE_CHECK_ARG(ldx >= C && lddy >= C && lddx >= C && (!add || ldadd >= C), "layernorm: a row stride is shorter than the row");
  const bool wg = dgamma || dbeta;
  if (R > 0) {
    PDAE_CHECK_ARG(x && mean && rstd && dy && dx, "layernorm_bwd: null pointer");
    PDAE_CHECK_ARG(tk_aligned(x, dtype) && tk_aligned(dy, dtype) && tk_aligned(dx, dtype) && tk_aligned(add, dtype) && tk_aligned(ws, PDAE_DT_F32),
                   "layernorm: tensors must be aligned to their element size");
    PDAE_CHECK_ARG(!wg || (ws && ws_bytes >= k_layernorm_workspace_bytes(R, C)), "layernorm_bwd: weight gradients need %zu bytes of workspace (got %zu)",
                   k_layernorm_workspace_bytes(R, C), ws ? ws_bytes : (size_t)0);
    PDAE_CHECK_ARG(dx != x && dx != dy, "layernorm_bwd: dx in the place of x or dy (blocks of columns may still read them)");
    PDAE_CHECK_ARG(dx != add || lddx == ldadd, "layernorm_bwd: dx in the place of add with another row stride");
    if (wg && ln_few(R, C)) {
      if (dtype == PDAE_DT_F32) ln_bwd_few<float>(x, ldx, gamma, mean, rstd, dy, lddy, add, ldadd, R, C, dx, lddx, dgamma, dbeta, acc_param, st);
      else ln_bwd_few<tk_bf16>(x, ldx, gamma, mean, rstd, dy, lddy, add, ldadd, R, C, dx, lddx, dgamma, dbeta, acc_param, st);
      return pdae_launch_status("layernorm_bwd");
    }
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
