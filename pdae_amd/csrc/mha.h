// Attention over any number of tokens (mha_fwd.hip, mha_bwd.hip): shared parameters, tile staging and matrix-core fragments.
//
//   o[q] = sum_j p[q][j] v[j],   p[q][j] = exp(scale q.k[j] - lse[q]),   lse[q] = log sum_j exp(scale q.k[j])      over the keys j that row q sees
//   key j is seen by query i of sample b iff  j < k_len[b]  and (causal)  j <= i + k_len[b] - q_len[b];   queries i >= q_len[b] do not exist.
//
// Element formats: bf16 tensors are ONE bf16 plane (NP = 1); fp32 tensors are split exactly into THREE (8 + 8 + 8 mantissa bits, by truncation) whose six
// leading products are accumulated (NP = 3).  What is dropped of a product is below 2^-20 |a||b| (2 x 2^-7 x 2^-14), 2^-24.5 in the mean over normally
// distributed values: the bound is sixteen times a rounding to fp32, the mean is one.  Below 2^-110 the lower planes leave fp32's range.  Everything that is
// summed is fp32.
// Roundings to fewer bits in bf16 tensors: the weights p (before p v and p^T dO) and dS (before dS^T Q; two planes before dS K) become bf16, because the matrix
// cores take bf16: up to 2^-8 of each value, 1.7e-3 of the norm.  A caller who needs more has fp32 tensors.
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
// Range of the unnormalised output.  Weights are kept 2^-32 of what the running maximum would give them, and the reference moves when a lane's weights of
// one tile (32 keys of 64, or 16 of 32) sum to more than MH_GROW: all weights of a row sum to less than keys x 2^-20, so sum p v stays below max |v| for up
// to 2^20 keys, whatever finite v is; weights below 2^-94 of the row's largest are zero (fp32 and bf16 share their exponent range).  bf16: the
// reference itself lies MH_LIFT above the maximum, which costs nothing in the loop; an exponent of -32 is exact to 2^-19, far below a bf16 weight's rounding.
// fp32 keeps its exponents small and multiplies the weights.
#define MH_LIFT 32.f
#define MH_DOWN 2.3283064365386963e-10f      // 2^-32
#define MH_GROW 1.52587890625e-5f      // 2^-16
template <int NP> __device__ __forceinline__ float mh_lift() { return NP == 1 ? MH_LIFT : 0.f; }
// the reference that a row maximum asks for.  (Not contracted: the fused form keeps MH_LIFT in a vector register, one too many where a wave has 64 rows.)
template <int NP> __device__ __forceinline__ float mh_reference(float mx, float sc2) {
#pragma clang fp contract(off)
  const float t = mx * sc2;
  return NP == 1 ? t + MH_LIFT : t;
}
// natural log-sum-exp of a row from its reference and its sum of weights
template <int NP> __device__ __forceinline__ float mh_lse(float m, float l) { return ((m - mh_lift<NP>()) + __builtin_amdgcn_logf(l * (1.f / MH_DOWN))) * MH_LN2; }
template <int I> struct MhInt { static constexpr int value = I; };

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
// Causal tiles differ in length: the longest tiles of ALL units come first, so the launch ends with short ones (unit after unit, the last unit's long
// tiles ran alone at the end: 19 % of the CU time of 64 units x 32 tiles).  Full tiles: unit after unit, so few keys and values are live in an L2 at once.
__device__ __forceinline__ bool mh_where(const MhaParams& P, int& unit, int& tile, int& split) {
  const bool x = mh_by_xcd(P.units);
  const int nu = x ? (P.units + 7) >> 3 : P.units, j = x ? blockIdx.x >> 3 : blockIdx.x;
  split = j % P.splits;
  const int k = j / P.splits;
  int u;
  if (P.causal) { u = k % nu; tile = k / nu; }
  else { u = k / P.tiles; tile = k % P.tiles; }
  unit = x ? u * 8 + (blockIdx.x & 7) : u;
  return unit < P.units;
}
// Ranges of the summed axis of `tokens`.  256 workgroups give every CU one, and a split costs an fp32 partial written, read and joined, and a prologue: full batches
// are split only below that, into ~512 (one fp32 sample of 4 heads, 1568 tokens, forward and backward: 167 us at 208 workgroups, 143 at 312, 146 at 468).  With lengths
// the work per workgroup varies by as much as they do, and the longest decides: ~1024.  A range is at least two tiles; with lengths (they are cut unevenly) and for
// single tokens (a wave takes 32 keys a step) twice that: one sample, 8 key heads, 8192 keys: 11.3 us with ranges of 256, 16.1 with 128.  Up to five bf16 tiles are
// not worth a join (training, one sample, 8 heads of 128, 256 tokens: 53 us in ranges, 49 without; 323 tokens the same; 383 tokens, 4 heads of 64: 42 and 44).
static inline int mh_splits(long long wgs, long long tokens, int dtype, bool lengths, bool token = false) {
  if (wgs <= 0 || (!lengths && wgs >= 256) || (dtype == PDAE_DT_BF16 && tokens <= 320)) return 1;
  const long long s = (lengths ? 1024 : 512) / wgs, most = tokens / ((dtype == PDAE_DT_BF16 ? 128 : 64) * (lengths || token ? 2 : 1));
  return (int)(s > most ? most < 1 ? 1 : most : s < 1 ? 1 : s);
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
// the same with a second bf16 plane for what the first rounding left (2^-17 of the value remains)
__device__ __forceinline__ void mh_planes2(const float (&e)[8], mh_bf16x8 (&f)[2]) {
  unsigned w[2][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = e[2 * j], b = e[2 * j + 1];
    w[0][j] = tk_pack2(a, b);
    w[1][j] = tk_pack2(a - __uint_as_float(w[0][j] << 16), b - __uint_as_float(w[0][j] & 0xffff0000u));
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) { const tk_u32x4 v = {w[p][0], w[p][1], w[p][2], w[p][3]}; f[p] = __builtin_bit_cast(mh_bf16x8, v); }
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

// ---- global loads.  Everything goes through buffer instructions: a lane whose row or channel does not exist passes an offset beyond num_records and
// gets zeros without touching memory, so the loops have no divergent branch (those cost the kernels a wait per load).  The resource starts at the
// tile's own first row (a 64-bit scalar address): only the distance inside a tile has to fit 31 bits, which the host checks.
// WH (whole): D is a multiple of 8, a chunk of 8 channels is one or two 16-byte loads.  !WH: single elements, any D.
#define MH_OOB 0xffffffffu
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mh_rsrc(const void* p) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, 0x7fffffff, 0x00020000); }
template <typename T, bool WH> __device__ __forceinline__ void mh_raw8(__amdgpu_buffer_rsrc_t s, unsigned off, int left, unsigned (&r)[sizeof(T) * 2]) {
  if constexpr (WH) {
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k) {
      const tk_u32x4 v = __builtin_bit_cast(tk_u32x4, __builtin_amdgcn_raw_buffer_load_b128(s, (int)(off == MH_OOB ? MH_OOB : off + 16 * k), 0, 0));
#pragma unroll
      for (int j = 0; j < 4; ++j) r[4 * k + j] = v[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) * 2; ++j) r[j] = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {                          // `left`: channels of this chunk that exist
      const int o = (int)(off == MH_OOB || j >= left ? MH_OOB : off + j * (unsigned)sizeof(T));
      if constexpr (sizeof(T) == 4) r[j] = (unsigned)__builtin_amdgcn_raw_buffer_load_b32(s, o, 0, 0);
      else r[j / 2] |= (unsigned)(unsigned short)__builtin_amdgcn_raw_buffer_load_b16(s, o, 0, 0) << (16 * (j & 1));
    }
  }
}
template <typename T> __device__ __forceinline__ void mh_raw_floats(const unsigned (&r)[sizeof(T) * 2], float (&e)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (sizeof(T) == 4) e[j] = __uint_as_float(r[j]);
    else e[j] = __uint_as_float(j & 1 ? r[j / 2] & 0xffff0000u : r[j / 2] << 16);
  }
}
template <typename T, int NP> __device__ __forceinline__ void mh_raw_planes(const unsigned (&r)[sizeof(T) * 2], mh_bf16x8 (&f)[NP]) {
  if constexpr (NP == 1) { const tk_u32x4 v = {r[0], r[1], r[2], r[3]}; f[0] = __builtin_bit_cast(mh_bf16x8, v); }
  else {
    float e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = __uint_as_float(r[j % (sizeof(T) * 2)]);
    mh_planes<NP>(e, f);
  }
}
// B fragments of this lane's token row, straight from global memory: channels ks * 16 + h * 8 ..+7 of every k-step.  off: the row's byte offset from
// `base` (MH_OOB: the row does not exist, zeros).
template <typename T, int NP, int DP, bool WH> __device__ __forceinline__ void mh_row_frags(const T* base, unsigned off, int D, int h, mh_bf16x8 (&f)[DP / 16][NP]) {
  const __amdgpu_buffer_rsrc_t s = mh_rsrc(base);
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    const int c = ks * 16 + h * 8;
    unsigned r[sizeof(T) * 2];
    mh_raw8<T, WH>(s, off == MH_OOB || c >= D ? MH_OOB : off + c * (unsigned)sizeof(T), D - c, r);
    mh_raw_planes<T, NP>(r, f[ks]);
  }
}

// Every global load issued so far has arrived.  Placed between the fragment loads of a kernel's prologue and its loop: without it the loop's own waits have to
// assume that those loads may still be pending, and the first product of EVERY iteration waits for the tile that was only just requested.
__device__ __forceinline__ void mh_loads_done() { __builtin_amdgcn_s_waitcnt(0x0F70); }      // vmcnt(0), other counters free

// ---- token-major LDS tile [plane][ROWS][LD] bf16 in 16-byte chunks, chunk c of row r at position c ^ mh_swz(r).  64 banks of 4 bytes: a row read (16 lanes =
// 16 consecutive rows, one chunk each) and a transposing read (32 lanes = 4 rows x 4 chunks) both touch every bank once.  With rows padded by 16 bytes
// instead, the four rows of a transposing read overlapped in up to four ways: half of all LDS cycles of the kernels were conflicts.
template <int DP> struct MhLd { static constexpr int NC = DP <= 32 ? 4 : DP <= 64 ? 8 : 16, LD = NC * 8; };      // chunks of a row (a power of two), elements
template <int DP> __device__ __forceinline__ int mh_swz(int row) {
  constexpr int NC = MhLd<DP>::NC, RPL = 16 / NC, NB = NC / 4;          // rows that share a 256-byte line; 64-byte blocks of a row
  return ((row / RPL) % NB) * 4 + ((row / RPL / NB) & 3);
}
template <int NP, int ROWS, int DP> struct MhTile {
  static constexpr int LD = MhLd<DP>::LD, PLANE = ROWS * LD, ELEMS = NP * PLANE;
};
// Global -> LDS of ROWS tokens in 16-byte chunks by the block's 256 threads (NT = 64: by one wave for itself); load() may run while the other buffer is read, the tile is complete after store() + mh_arrive() and a
// barrier.  bf16 with D % 8 == 0 goes straight into LDS (buffer_load .. lds: a wave's 64 chunks land at consecutive addresses, so the LANE picks the
// channels that belong at its place): no registers hold the tile in flight.  The other formats pass through registers (split, single elements).
template <typename T, int NP, int ROWS, int DP, bool WH, int NT = 256> struct MhStage {
  static constexpr bool DMA = NP == 1 && WH;
  static constexpr int LD = MhLd<DP>::LD, PLANE = ROWS * LD, CPR = DMA ? LD / 8 : DP / 8, CH = ROWS * CPR, N = (CH + NT - 1) / NT, W = sizeof(T) * 2;
  unsigned r[DMA ? 1 : N][DMA ? 1 : W], off[N];            // chunk in flight; its byte offset from the tile's first row
  int D;
  __device__ __forceinline__ static int tid() { return NT == 256 ? (int)threadIdx.x : (int)threadIdx.x & (NT - 1); }
  __device__ __forceinline__ static int row_of(int l) { return (tid() + NT * l) / CPR; }
  __device__ __forceinline__ static int chunk_of(int l) {
    const int c = (tid() + NT * l) % CPR;
    return DMA ? c ^ mh_swz<DP>(row_of(l)) : c;
  }
  __device__ __forceinline__ void init(long long stride, int D_) {
    D = D_;
#pragma unroll
    for (int l = 0; l < N; ++l) {
      const int c = chunk_of(l) * 8;
      off[l] = (CH % NT == 0 || tid() + NT * l < CH) && c < D ? (unsigned)(row_of(l) * stride + c) * (unsigned)sizeof(T) : MH_OOB;
    }
  }
  // tokens [row0, row0 + ROWS) of base (token stride `stride` elements); those outside [lo, hi) come as zero and are never read
  __device__ __forceinline__ void load(const T* base, long long stride, int row0, int lo, int hi, unsigned short* lds) {
    const T* p = base + (long long)row0 * stride;
    if constexpr (DMA) {
      static_assert(CH % NT == 0 || CH < NT, "whole waves");
      const unsigned long long a = (unsigned long long)p;
      const tk_u32x4 s = {(unsigned)a, (unsigned)(a >> 32) & 0xffffu, 0x7fffffffu, 0x00020000u};
      const unsigned dst = (unsigned)(size_t)(mh_lds4)(lds) + (NT == 256 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024 : 0);
#pragma unroll
      for (int l = 0; l < N; ++l) {
        const int row = row0 + row_of(l);
        const unsigned o = row >= lo && row < hi ? off[l] : MH_OOB;
        if (CH % NT == 0 || __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 64 < CH)
          asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(o), "s"(s), "s"(dst + l * (NT * 16)) : "memory", "m0");
      }
    } else {
      const __amdgpu_buffer_rsrc_t s = mh_rsrc(p);
#pragma unroll
      for (int l = 0; l < N; ++l) {
        const int row = row0 + row_of(l);
        mh_raw8<T, WH>(s, row >= lo && row < hi ? off[l] : MH_OOB, D - chunk_of(l) * 8, r[l]);
      }
    }
  }
  __device__ __forceinline__ void store(unsigned short* lds) const {
    if constexpr (!DMA) {
#pragma unroll
      for (int l = 0; l < N; ++l) {
        if (CH % NT != 0 && tid() + NT * l >= CH) continue;
        unsigned short* d = lds + row_of(l) * LD + (chunk_of(l) ^ mh_swz<DP>(row_of(l))) * 8;
        mh_bf16x8 f[NP];
        mh_raw_planes<T, NP>(r[l], f);
#pragma unroll
        for (int p = 0; p < NP; ++p) *reinterpret_cast<mh_bf16x8*>(d + p * PLANE) = f[p];
      }
    }
  }
};
// This wave's direct loads have landed (the compiler does not count them).
template <bool DMA> __device__ __forceinline__ void mh_arrive() {
  if constexpr (DMA) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}
template <int LEFT> __device__ __forceinline__ void mh_arrive_but() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory"); }      // all but the newest LEFT
// A fragment, tokens on rows: token row0 + l%32 (row0 a multiple of 32), channels ks * 16 + h * 8 ..+7
template <int NP, int ROWS, int DP> __device__ __forceinline__ void mh_frag_rows(const unsigned short* lds, int row0, int ks, int li, int h, mh_bf16x8 (&f)[NP]) {
  constexpr int LD = MhLd<DP>::LD;
#pragma unroll
  for (int p = 0; p < NP; ++p)
    f[p] = *reinterpret_cast<const mh_bf16x8*>(lds + p * MhTile<NP, ROWS, DP>::PLANE + row0 * LD + li * LD + ((ks * 2 + h) ^ mh_swz<DP>(li)) * 8);
}
// A fragment, channels db * 32 + l%32 on rows, k = the sixteen tokens from row0 (a multiple of 16) in the order of packed accumulator registers
template <int NP, int ROWS, int DP> __device__ __forceinline__ void mh_frag_cols(const unsigned short* lds, int row0, int db, int lane, mh_bf16x8 (&f)[NP]) {
  constexpr int LD = MhLd<DP>::LD;
  const int i = lane & 15, g = (lane >> 4) & 1, h = lane >> 5, r = 4 * h + (i >> 2), c = db * 4 + g * 2 + ((i & 3) >> 1);
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const unsigned short* a = lds + p * MhTile<NP, ROWS, DP>::PLANE + row0 * LD + (i & 1) * 4;
    const mh_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mh_lds4)(a + r * LD + (c ^ mh_swz<DP>(r)) * 8));
    const mh_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mh_lds4)(a + (r + 8) * LD + (c ^ mh_swz<DP>(r + 8)) * 8));
    const mh_s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    f[p] = __builtin_bit_cast(mh_bf16x8, v);
  }
}
// Order of a product phase of STEPS steps, each with DS LDS reads and MM matrix instructions: the reads run PD steps ahead.  Left to itself the compiler keeps
// few fragments in flight (read, wait, multiply, read, ...), and every read's ~120 cycles of latency stand between two matrix instructions.
template <int STEPS, int PD, int DS, int MM, int FIRST = 0> __device__ __forceinline__ void mh_order() {
  __builtin_amdgcn_sched_group_barrier(0x100, FIRST + DS * (PD < STEPS ? PD : STEPS), 0);      // FIRST: reads of the phase that belong to no step
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, MM, 0);
    if (i + PD < STEPS) __builtin_amdgcn_sched_group_barrier(0x100, DS, 0);
  }
}
// Stores the four channels [c, c + 4) of one token row.
template <typename T, bool WH> __device__ __forceinline__ void mh_store4(T* row, int c, int D, float a, float b, float e, float d) {
  if (WH ? c < D : c + 4 <= D) {
    if constexpr (sizeof(T) == 2) { const unsigned w[2] = {tk_pack2(a, b), tk_pack2(e, d)}; __builtin_memcpy(row + c, w, 8); }
    else { const float w[4] = {a, b, e, d}; __builtin_memcpy(row + c, w, 16); }
  } else if constexpr (!WH) {
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
