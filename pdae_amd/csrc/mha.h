// Attention over any number of tokens (mha_fwd.hip, mha_bwd.hip): shared parameters, tile staging and matrix-core fragments.
//
//   o[q] = sum_j p[q][j] v[j],   p[q][j] = exp(scale q.k[j] - lse[q]),   lse[q] = log sum_j exp(scale q.k[j])      over the keys j that row q sees
//   key j is seen by query i of sample b iff  j < k_len[b]  and (causal)  j <= i + k_len[b] - q_len[b];   queries i >= q_len[b] do not exist.
//
// Element formats: bf16 tensors are ONE bf16 plane (NP = 1); fp32 tensors are split exactly into THREE (8 + 8 + 8 mantissa bits) whose six leading products
// are accumulated (NP = 3, ~2^-23 a product: fp32 grade, free of range limits).  Everything that is summed is fp32.
//
// Fragments of v_mfma_f32_32x32x16_bf16: lane l gives A[row l%32][k (l/32)*8 ..+7] and B[k (l/32)*8 ..+7][col l%32]; accumulator register r is
// D[(r&3) + 8*(r>>2) + 4*(l/32)][l%32].  The kernels always put the side whose statistics matter on the COLUMNS (queries in the forward and dQ
// kernels, keys in the dK / dV kernel), so a column's scores lie in one lane and its partner 32 lanes away, and registers 8s .. 8s+7 of a
// 32 x 32 block, packed, ARE the B fragment of the next product for the k order {4h..4h+3, 8+4h..8+4h+3} (+16s): probabilities never pass through LDS.
// The A side of that next product needs the same k order with the channels on its rows: ds_read_b64_tr_b16 reads it out of the token-major tile
// (16 lanes get 16 channels of 4 consecutive tokens).
#pragma once
#include "token.h"

typedef float mh_f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 mh_bf16x8 __attribute__((ext_vector_type(8)));
typedef short mh_s16x4 __attribute__((ext_vector_type(4)));
typedef short mh_s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) mh_s16x4* mh_lds4;

#define MH_LOG2E 1.4426950408889634f
#define MH_LN2 0.6931471805599453f
#define MH_INF __builtin_inff()

struct MhaParams {
  const void *q, *k, *v, *o, *d_o;
  void *out, *dq, *dk, *dv;
  float *lse, *delta;
  float *part;                               // partial results of a split axis
  const int *q_len, *k_len;                  // device, or NULL
  int B, Hq, Hkv, G, Tq, Tk, D, causal;
  int GP, HP, R;                             // forward: GP query heads share a tile row block (1 or G); HP = Hq / GP head groups of R = Tq * GP rows
  float scale, sc2;                          // sc2 = scale * log2(e)
  long long qb, qt, qh, kb, kt, kh, vb, vt, vh, ob, ot, oh;      // element strides (batch, token, head)
  int tiles, splits, units;                  // row tiles, ranges of the summed axis, (batch, head) pairs
};

// blockIdx.x -> (unit, tile, split).  Workgroups go round-robin over the 8 XCDs: with a multiple of 8 units (or many) all tiles of a unit get the
// same residue mod 8, so its keys and values are fetched into ONE XCD's L2.  Otherwise plain order: an uneven share would leave XCDs idle.
__host__ __device__ inline bool mh_by_xcd(int units) { return units % 8 == 0 || units >= 64; }
__device__ __forceinline__ bool mh_where(const MhaParams& P, int& unit, int& tile, int& split) {
  const int per = P.tiles * P.splits;
  int rem;
  if (mh_by_xcd(P.units)) {
    const int j = blockIdx.x >> 3;
    unit = (j / per) * 8 + (blockIdx.x & 7);
    rem = j % per;
  } else {
    unit = blockIdx.x / per;
    rem = blockIdx.x % per;
  }
  tile = rem / P.splits;
  split = rem % P.splits;
  return unit < P.units;
}
static inline long long mh_grid(const MhaParams& P) {
  return (long long)(mh_by_xcd(P.units) ? (P.units + 7) / 8 * 8 : P.units) * P.tiles * P.splits;
}

__device__ __forceinline__ int mh_len(const int* len, int b, int T) {
  if (!len) return T;
  const int n = len[b];
  return n < 0 ? 0 : n > T ? T : n;          // a length outside the tensor is cut to it: no read or write leaves the buffers
}

// ---- formats
template <typename T> struct MhNP;
template <> struct MhNP<float> { static constexpr int NP = 3; };
template <> struct MhNP<tk_bf16> { static constexpr int NP = 1; };

__device__ __forceinline__ float mh_trunc(float a) { return __uint_as_float(__float_as_uint(a) & 0xffff0000u); }
__device__ __forceinline__ unsigned mh_top2(float a, float b) { return (__float_as_uint(a) >> 16) | (__float_as_uint(b) & 0xffff0000u); }
// eight fp32 values -> fragment planes: rounded to nearest bf16 (NP = 1) or split exactly into three bf16 planes
template <int NP> __device__ __forceinline__ void mh_planes(const float (&e)[8], mh_bf16x8 (&f)[NP]) {
  if constexpr (NP == 1) {
    const tk_u32x4 w = {tk_pack2(e[0], e[1]), tk_pack2(e[2], e[3]), tk_pack2(e[4], e[5]), tk_pack2(e[6], e[7])};
    f[0] = __builtin_bit_cast(mh_bf16x8, w);
  } else {
    unsigned w[3][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = e[2 * j], b = e[2 * j + 1];
      const float ra = a - mh_trunc(a), rb = b - mh_trunc(b);
      w[0][j] = mh_top2(a, b);
      w[1][j] = mh_top2(ra, rb);
      w[2][j] = mh_top2(ra - mh_trunc(ra), rb - mh_trunc(rb));
    }
#pragma unroll
    for (int p = 0; p < 3; ++p) { const tk_u32x4 v = {w[p][0], w[p][1], w[p][2], w[p][3]}; f[p] = __builtin_bit_cast(mh_bf16x8, v); }
  }
}
template <int NP> __device__ __forceinline__ void mh_mma(const mh_bf16x8 (&A)[NP], const mh_bf16x8 (&B)[NP], mh_f32x16& acc) {
  if constexpr (NP == 3) {                   // small terms first
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[1], B[1], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[0], B[2], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[2], B[0], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[0], B[1], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[1], B[0], acc, 0, 0, 0);
  }
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[0], B[0], acc, 0, 0, 0);
}
__device__ __forceinline__ void mh_zero(mh_f32x16& a) {
#pragma unroll
  for (int r = 0; r < 16; ++r) a[r] = 0.f;
}

// Eight channels [c, c + 8) of one token as fp32; channels >= D read as zero and are not touched.
template <typename T> __device__ __forceinline__ void mh_load8(const T* p, int c, int D, float (&e)[8]) {
  if (c + 8 <= D) TkVec<T>::load8(p + c, e);
  else {
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = c + j < D ? TkVec<T>::load(p + c + j) : 0.f;
  }
}
// B (or A) fragments of this lane's token row, straight from global memory: channels ks * 16 + h * 8 ..+7 of every k-step.  valid = 0: zeros.
template <typename T, int NP, int DP> __device__ __forceinline__ void mh_row_frags(const T* row, bool valid, int D, int h, mh_bf16x8 (&f)[DP / 16][NP]) {
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    float e[8];
    if (valid) mh_load8(row, ks * 16 + h * 8, D, e);
    else {
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = 0.f;
    }
    mh_planes<NP>(e, f[ks]);
  }
}

// ---- token-major LDS tile [plane][ROWS][DP + 8] bf16: rows 16 bytes off a multiple of 128 keep ds_read_b128 of 32 rows at one channel free of conflicts
#define MH_PAD 8
template <int NP, int ROWS, int DP> struct MhTile {
  static constexpr int LD = DP + MH_PAD, PLANE = ROWS * LD, ELEMS = NP * PLANE;
};
// Global -> registers -> LDS of ROWS tokens by 256 threads: chunks of 8 channels.
template <typename T, int NP, int ROWS, int DP> struct MhStage {
  static constexpr int CPR = DP / 8, CH = ROWS * CPR, N = (CH + 255) / 256, LD = DP + MH_PAD, PLANE = ROWS * LD;
  static constexpr int W = sizeof(T) == 2 ? 4 : 8;         // dwords a chunk holds in registers
  unsigned r[N][W];
  // tokens [row0, row0 + ROWS) of base (token stride `st` elements); those outside [lo, hi) and channels >= D come as zero and are never read
  __device__ __forceinline__ void load(const T* base, long long st, int row0, int lo, int hi, int D) {
#pragma unroll
    for (int l = 0; l < N; ++l) {
      const int i = threadIdx.x + 256 * l, row = row0 + i / CPR, c = (i % CPR) * 8;
#pragma unroll
      for (int j = 0; j < W; ++j) r[l][j] = 0;
      if ((CH % 256 == 0 || i < CH) && row >= lo && row < hi && c < D) {
        const T* p = base + (long long)row * st + c;
        if (c + 8 <= D) __builtin_memcpy(r[l], p, 8 * sizeof(T));
        else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (c + j < D) {
              if constexpr (sizeof(T) == 4) r[l][j] = __float_as_uint(TkVec<T>::load(p + j));
              else r[l][j / 2] |= (unsigned)__builtin_bit_cast(unsigned short, p[j]) << (16 * (j & 1));
            }
        }
      }
    }
  }
  __device__ __forceinline__ void store(unsigned short* lds) const {
#pragma unroll
    for (int l = 0; l < N; ++l) {
      const int i = threadIdx.x + 256 * l;
      if (CH % 256 != 0 && i >= CH) continue;
      unsigned short* d = lds + (i / CPR) * LD + (i % CPR) * 8;
      if constexpr (NP == 1) *reinterpret_cast<tk_u32x4*>(d) = tk_u32x4{r[l][0], r[l][1], r[l][2], r[l][3]};
      else {
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = __uint_as_float(r[l][j % W]);
        mh_bf16x8 f[NP];
        mh_planes<NP>(e, f);
#pragma unroll
        for (int p = 0; p < NP; ++p) *reinterpret_cast<mh_bf16x8*>(d + p * PLANE) = f[p];
      }
    }
  }
};
// A fragment, tokens on rows: token row0 + l%32, channels ks * 16 + h * 8 ..+7
template <int NP, int ROWS, int DP> __device__ __forceinline__ void mh_frag_rows(const unsigned short* lds, int row0, int ks, int li, int h, mh_bf16x8 (&f)[NP]) {
#pragma unroll
  for (int p = 0; p < NP; ++p)
    f[p] = *reinterpret_cast<const mh_bf16x8*>(lds + p * MhTile<NP, ROWS, DP>::PLANE + (row0 + li) * MhTile<NP, ROWS, DP>::LD + ks * 16 + h * 8);
}
// A fragment, channels db * 32 + l%32 on rows, k = the sixteen tokens from row0 in the order of packed accumulator registers
template <int NP, int ROWS, int DP> __device__ __forceinline__ void mh_frag_cols(const unsigned short* lds, int row0, int db, int lane, mh_bf16x8 (&f)[NP]) {
  constexpr int LD = MhTile<NP, ROWS, DP>::LD;
  const int i = lane & 15, g = (lane >> 4) & 1, h = lane >> 5;
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const unsigned short* a = lds + p * MhTile<NP, ROWS, DP>::PLANE + (row0 + 4 * h + (i >> 2)) * LD + db * 32 + g * 16 + (i & 3) * 4;
    const mh_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mh_lds4)(a));
    const mh_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mh_lds4)(a + 8 * LD));
    const mh_s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    f[p] = __builtin_bit_cast(mh_bf16x8, v);
  }
}
// Stores the four channels [c, c + 4) of one token row.
template <typename T> __device__ __forceinline__ void mh_store4(T* row, int c, int D, float a, float b, float e, float d) {
  if (c + 4 <= D) {
    if constexpr (sizeof(T) == 2) { const unsigned w[2] = {tk_pack2(a, b), tk_pack2(e, d)}; __builtin_memcpy(row + c, w, 8); }
    else { const float w[4] = {a, b, e, d}; __builtin_memcpy(row + c, w, 16); }
  } else {
    if (c < D) TkVec<T>::store(row + c, a);
    if (c + 1 < D) TkVec<T>::store(row + c + 1, b);
    if (c + 2 < D) TkVec<T>::store(row + c + 2, e);
  }
}
// mask of a 32 x 32 score block whose rows are keys base + 4h + (r & 3) + 8 (r >> 2): columns see keys below `limit`
__device__ __forceinline__ void mh_mask_keys(mh_f32x16& s, int base, int limit) {
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = base + (r & 3) + 8 * (r >> 2) < limit ? s[r] : -MH_INF;
}
