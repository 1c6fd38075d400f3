// Attention backward (mha.h): the probabilities are recomputed from q, k and the saved row log-sum-exp, nothing of size tokens x tokens exists.
//
//   P = exp(scale q.k - lse),  dP = dO.v,  dS = P (dP - delta),  delta[q] = sum_d dO[q][d] O[q][d] = sum_j P dP
//   dQ = scale dS K                   mha_dq_kernel:  a wave owns 32 queries (columns), the keys stream through LDS; it also leaves delta for
//   dV = P^T dO,  dK = scale dS^T Q   mha_dkv_kernel: a wave owns 32 keys (columns), the queries stream through LDS
//
// Two kernels recompute S and dP twice (7 products of 2 Tq Tk D instead of 5): dK / dV and dQ then each have ONE writer, so there are no atomics and the
// results are the same bits every run.  dK / dV of a key head sum over the query heads that share it inside the kernel.
// Bound: products and exponentials, which hardly overlap, and the clock.  4 x 16 heads of 128, 4096 tokens, causal, bf16, after a hundred passes: dQ 492 us (1120
// TFLOP/s of its four products), dK / dV 515 us (1070); in the first ten 530 .. 557 and 570 .. 608 (the clock rises from 1.6 to 1.8 GHz of 2.4); matrix pipes busy
// 61 / 57 % of the CUs' time, vector instructions 54 / 35 %, LDS 23 / 43 %, no bank conflicts.  fp32, 8 x 4 heads of 64, 1024 tokens: 75 + 94 us, first ten passes 88 + 111.
// Roundings of bf16 tensors: dQ takes dS in TWO bf16 planes (a matrix instruction more on the same fragment): it is off by 1.65e-3 .. 1.85e-3 of its norm, of which its
// own rounding is 1.65e-3 and delta from the rounded o up to 0.9e-3, in squares.  With one plane it was 2.5e-3, one and a half times what rounding the result
// costs; the second plane is 4 .. 7 % of a training pass (4 x 16 heads of 128, 4096 tokens, causal: 1256 -> 1305 us; 7 padded samples 184 -> 195).  dK and dV round dS
// and P once (2.3e-3 .. 2.4e-3): a second plane finds no registers beside K, V and both accumulators.
// Few tiles: the summed axis is split into ranges (grid `splits`), every range leaves an fp32 partial, mha_bwd_join_kernel adds them in order.
// Row validity is decided where rows are staged: queries that do not exist or (causal) see no key come as zeros with lse = +inf, so P = 0 exactly and
// non-finite values in them reach nothing.
#include "kernels.h"
#include "mha.h"

#define MH_SHORT 256

// accumulators (channels on rows, this lane's token on the column) -> row of a tensor, or fp32 partial row
template <typename T, int DB, bool WH> __device__ __forceinline__ void mh_put(const mh_f32x16 (&a)[DB], float f, bool keep, T* row, int D, int h) {
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = d * 32 + g * 8 + h * 4;
      mh_store4<T, WH>(row, c, D, keep ? a[d][g * 4] * f : 0.f, keep ? a[d][g * 4 + 1] * f : 0.f, keep ? a[d][g * 4 + 2] * f : 0.f, keep ? a[d][g * 4 + 3] * f : 0.f);
    }
}

template <typename T, int DP, int KT, int OCC, bool WH>
__global__ void __launch_bounds__(256, OCC) mha_dq_kernel(const MhaParams P) {
  constexpr int NP = MhNP<T>::NP, KS = DP / 16, DB = DP / 32, KB = KT / 32;
  constexpr int TE = MhTile<NP, KT, DP>::ELEMS, MM = NP == 3 ? 6 : 1, PD = NP == 3 ? 2 : 4, SP = NP == 3 ? 3 : 2;      // SP: planes of dS
  extern __shared__ __attribute__((aligned(16))) unsigned short mh_sm[];       // [2 buffers][K tile | V tile]
  int unit, tile, split;
  if (!mh_where(P, unit, tile, split)) return;
  if (P.causal) tile = P.tiles - 1 - tile;
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), li = lane & 31, h = lane >> 5;
  const int b = unit / P.Hq, hq = unit % P.Hq, hk = hq / P.G;
  const int lq = mh_len(P.q_len, b, P.Tq), lk = mh_len(P.k_len, b, P.Tk), off = lk - lq;
  const int row0 = tile * 128, tq = row0 + wv * 32 + li;
  const T* kbase = (const T*)P.k + b * P.kb + hk * P.kh;
  const T* vbase = (const T*)P.v + b * P.vb + hk * P.vh;
  int nk = row0 >= lq ? 0 : P.causal ? min(lk, min(row0 + 127, lq - 1) + off + 1) : lk;
  nk = max(nk, 0);
  const int ntiles = (nk + KT - 1) / KT;
  const int tb = (int)((long long)ntiles * split / P.splits), te = (int)((long long)ntiles * (split + 1) / P.splits);
  const bool ok = tq < lq && lk > 0 && (!P.causal || tq + off >= 0);           // the query exists and sees a key
  const int kmax = ok ? (P.causal ? min(lk, tq + off + 1) : lk) : lk;
  const bool wlive = __any(ok);

  mh_bf16x8 Q[KS][NP], G[KS][NP];
  mh_row_frags<T, NP, DP, WH>((const T*)P.q + b * P.qb + (long long)row0 * P.qt + (long long)hq * P.qh,
                              ok ? (unsigned)((tq - row0) * P.qt) * (unsigned)sizeof(T) : MH_OOB, P.D, h, Q);
  mh_row_frags<T, NP, DP, WH>((const T*)P.d_o + b * P.ob + (long long)row0 * P.ot + (long long)hq * P.oh,
                              ok ? (unsigned)((tq - row0) * P.ot) * (unsigned)sizeof(T) : MH_OOB, P.D, h, G);
  const long long row = ((long long)b * P.Hq + hq) * P.Tq + tq;
  float lse2 = MH_INF;
  // delta of this lane's query from dO and O: half of the channels here, half 32 lanes away.  (A launch of its own for it read both once more: 35 us of 4 x 16
  // heads of 128, 4096 tokens.)
  float del = 0.f;
  {
    const __amdgpu_buffer_rsrc_t so = mh_rsrc((const T*)P.o + b * P.ob + (long long)row0 * P.ot + (long long)hq * P.oh);
    const __amdgpu_buffer_rsrc_t sg = mh_rsrc((const T*)P.d_o + b * P.ob + (long long)row0 * P.ot + (long long)hq * P.oh);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int c = ks * 16 + h * 8;
      const unsigned at = ok && c < P.D ? (unsigned)((tq - row0) * P.ot + c) * (unsigned)sizeof(T) : MH_OOB;
      unsigned x[sizeof(T) * 2], y[sizeof(T) * 2];
      mh_raw8<T, WH>(so, at, P.D - c, x);
      mh_raw8<T, WH>(sg, at, P.D - c, y);
      float e[8], f[8];
      mh_raw_floats<T>(x, e);
      mh_raw_floats<T>(y, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) del += e[j] * f[j];
    }
    del += __shfl_xor(del, 32);
  }
  if (ok) {
    const float e = P.lse[row];
    lse2 = e == -MH_INF ? MH_INF : e * MH_LOG2E;
  }
  mh_f32x16 dQ[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) mh_zero(dQ[d]);

  MhStage<T, NP, KT, DP, WH> sk, sv;
  sk.init(P.kt, P.D); sv.init(P.vt, P.D);
  // bf16: delta from the ROUNDED o is off by 2^-9 sum |dO||O|, which rows over few keys (large |O|) feel as much as all other roundings together.  Tiles that see
  // at most MH_SHORT keys take it exactly, delta = sum_j p dP, in a sweep of its own over those keys, too.
  const bool sweep = NP == 1 && nk > 0 && nk <= MH_SHORT;
  // tile `it` of the sweep lies in buffer (ntiles - it) & 1, so the loop's first tile, in flight behind the last one, lies in buffer 0
  const int t0 = sweep ? 0 : tb;
  if (sweep || tb < te) {
    unsigned short* to = mh_sm + (sweep ? ntiles & 1 : 0) * 2 * TE;
    sk.load(kbase, P.kt, t0 * KT, 0, lk, to); sv.load(vbase, P.vt, t0 * KT, 0, lk, to + TE);
    sk.store(to); sv.store(to + TE);
  }
  mh_loads_done();
  __syncthreads();
  if (sweep) {
    float acc = 0.f;
    for (int it = 0; it < ntiles; ++it) {
      const unsigned short* cur = mh_sm + ((ntiles - it) & 1) * 2 * TE;
      unsigned short* nxt = mh_sm + ((ntiles - it - 1) & 1) * 2 * TE;
      const int tn = it + 1 < ntiles ? it + 1 : tb;
      const bool more = it + 1 < ntiles || tb < te;
      if (more) { sk.load(kbase, P.kt, tn * KT, 0, lk, nxt); sv.load(vbase, P.vt, tn * KT, 0, lk, nxt + TE); }
#pragma unroll 1
      for (int kb = 0; kb < KB; ++kb) {
        mh_f32x16 S, E;
        mh_zero(S); mh_zero(E);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          mh_bf16x8 A[NP];
          mh_frag_rows<NP, KT, DP>(cur, kb * 32, ks, li, h, A);
          mh_mma<NP>(A, Q[ks], S);
          mh_frag_rows<NP, KT, DP>(cur + TE, kb * 32, ks, li, h, A);
          mh_mma<NP>(A, G[ks], E);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(S[r], P.sc2, -lse2)) * E[r];
          acc += it * KT + kb * 32 + 4 * h + (r & 3) + 8 * (r >> 2) < kmax ? x : 0.f;
        }
      }
      if (more) { sk.store(nxt); sv.store(nxt + TE); }
      mh_arrive<decltype(sk)::DMA>();
      __syncthreads();
    }
    acc += __shfl_xor(acc, 32);
    if (ok) del = acc;
  }
  if (ok && split == 0 && h == 0) P.delta[row] = del;
  for (int it = tb; it < te; ++it) {
    const unsigned short* cur = mh_sm + ((it - tb) & 1) * 2 * TE;
    unsigned short* nxt = mh_sm + (((it - tb) & 1) ^ 1) * 2 * TE;
    const bool more = it + 1 < te;
    if (more) { sk.load(kbase, P.kt, (it + 1) * KT, 0, lk, nxt); sv.load(vbase, P.vt, (it + 1) * KT, 0, lk, nxt + TE); }
    const int k0 = it * KT;
    if (wlive && __any(kmax > k0)) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        mh_f32x16 S, E;
        mh_zero(S); mh_zero(E);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          mh_bf16x8 A[NP];
          mh_frag_rows<NP, KT, DP>(cur, kb * 32, ks, li, h, A);
          mh_mma<NP>(A, Q[ks], S);
          mh_frag_rows<NP, KT, DP>(cur + TE, kb * 32, ks, li, h, A);
          mh_mma<NP>(A, G[ks], E);
        }
        mh_order<2 * KS, PD, NP, MM>();
        __builtin_amdgcn_sched_barrier(0);
        const int base = k0 + kb * 32 + 4 * h;
        const bool cut = __any(k0 + kb * 32 + 32 > kmax);
        mh_bf16x8 F[2][SP];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          float e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int r = s * 8 + j;
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(S[r], P.sc2, -lse2));
            e[j] = p * (E[r] - del);
            if (cut && base + (r & 3) + 8 * (r >> 2) >= kmax) e[j] = 0.f;
          }
          if constexpr (NP == 1) mh_planes2(e, F[s]);
          else mh_planes<NP>(e, F[s]);
        }
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            mh_bf16x8 A[NP];
            mh_frag_cols<NP, KT, DP>(cur, kb * 32 + s * 16, d, lane, A);
            if constexpr (NP == 1) {                                           // small terms first
              dQ[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[0], F[s][1], dQ[d], 0, 0, 0);
              dQ[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[0], F[s][0], dQ[d], 0, 0, 0);
            } else {
              mh_mma<NP>(A, F[s], dQ[d]);
            }
          }
        mh_order<2 * DB, PD, 2 * NP, NP == 1 ? 2 : MM>();
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (more) { sk.store(nxt); sv.store(nxt + TE); }
    mh_arrive<decltype(sk)::DMA>();
    __syncthreads();
  }
  if (tq >= P.Tq) return;
  if (P.splits > 1) {
    if (tq < lq) mh_put<float, DB, WH>(dQ, P.scale, ok, P.part + ((long long)split * P.B * P.Hq * P.Tq + row) * P.D, P.D, h);
  } else {
    mh_put<T, DB, WH>(dQ, P.scale, ok, (T*)P.dq + b * P.qb + (long long)tq * P.qt + (long long)hq * P.qh, P.D, h);
  }
}

template <typename T, int DP, int QT, int OCC, bool WH, bool KL>
__global__ void __launch_bounds__(256, OCC) mha_dkv_kernel(const MhaParams P) {
  constexpr int NP = MhNP<T>::NP, KS = DP / 16, DB = DP / 32, QB = QT / 32;
  constexpr int MM = NP == 3 ? 6 : 1, PD = NP == 3 ? 2 : 4;
  constexpr int TE = MhTile<NP, QT, DP>::ELEMS, BUF = 2 * TE + 4 * QT;         // Q tile | dO tile | -lse2[QT], -delta[QT] (floats)
  extern __shared__ __attribute__((aligned(16))) unsigned short mh_sm[];
  int unit, tile, split;
  if (!mh_where(P, unit, tile, split)) return;
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), li = lane & 31, h = lane >> 5;
  const int b = unit / P.Hkv, hk = unit % P.Hkv;
  const int lq = mh_len(P.q_len, b, P.Tq), lk = mh_len(P.k_len, b, P.Tk), off = lk - lq;
  const int key0 = tile * 128, kw = key0 + wv * 32, key = kw + li;
  const bool ok = key < lk;
  const int qlo = P.causal ? max(0, -off) : 0;                                 // first query that sees a key
  const int first = P.causal ? max(qlo, key0 - off) : 0;                       // first query that sees key0
  const int q0t = first / QT, nq = key0 < lk && first < lq ? (lq + QT - 1) / QT - q0t : 0;
  const int items = nq * P.G;                                                  // (query head, query tile) pairs in order (the host checks G * tiles < 2^31)
  const int ib = (int)((long long)items * split / P.splits), ie = (int)((long long)items * (split + 1) / P.splits);
  int lh = nq > 0 ? ib / nq : 0, lt = nq > 0 ? ib - lh * nq : 0;               // the pair that is loaded next

  mh_bf16x8 K[KS][NP], V[KS][NP];
  mh_row_frags<T, NP, DP, WH>((const T*)P.k + b * P.kb + (long long)key0 * P.kt + (long long)hk * P.kh,
                              ok ? (unsigned)((key - key0) * P.kt) * (unsigned)sizeof(T) : MH_OOB, P.D, h, K);
  mh_row_frags<T, NP, DP, WH>((const T*)P.v + b * P.vb + (long long)key0 * P.vt + (long long)hk * P.vh,
                              ok ? (unsigned)((key - key0) * P.vt) * (unsigned)sizeof(T) : MH_OOB, P.D, h, V);
  // KL: this wave's K fragments live in LDS (a lane reads back its own 16 bytes) instead of 4 KS NP registers
  unsigned short* kl = mh_sm + 2 * BUF + wv * (KS * NP * 512) + lane * 8;
  if constexpr (KL) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int p = 0; p < NP; ++p) *reinterpret_cast<mh_bf16x8*>(kl + (ks * NP + p) * 512) = K[ks][p];
  }
  mh_f32x16 dK[DB], dV[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) { mh_zero(dK[d]); mh_zero(dV[d]); }

  MhStage<T, NP, QT, DP, WH> sq, sg;
  sq.init(P.qt, P.D); sg.init(P.ot, P.D);
  float rl = 0.f, rd = 0.f;
  bool rin = false;
  auto load = [&](unsigned short* buf) {
    const int hq = hk * P.G + lh, q0 = (q0t + lt) * QT;
    sq.load((const T*)P.q + b * P.qb + (long long)hq * P.qh, P.qt, q0, qlo, lq, buf);
    sg.load((const T*)P.d_o + b * P.ob + (long long)hq * P.oh, P.ot, q0, qlo, lq, buf + TE);
    const int tq = q0 + (t & (QT - 1));
    rin = tq >= qlo && tq < lq;
    const long long i = ((long long)b * P.Hq + hq) * P.Tq + (rin ? tq : 0);
    rl = P.lse[i]; rd = P.delta[i];                                            // (looked at in store(): here it would wait for the loads)
    if (++lt == nq) { lt = 0; ++lh; }
  };
  auto store = [&](unsigned short* buf) {
    sq.store(buf); sg.store(buf + TE);
    float* st = reinterpret_cast<float*>(buf + 2 * TE);
    // rows that do not count come as -lse = -inf: their probabilities are exact zeros
    if (t < QT) { st[t] = !rin || rl == -MH_INF ? -MH_INF : rl * -MH_LOG2E; st[QT + t] = rin ? -rd : 0.f; }
  };
  int ct = lt;                                                                 // query tile of the pair being multiplied
  if (ib < ie) { load(mh_sm); store(mh_sm); }
  mh_loads_done();
  __syncthreads();
  // the statistics of a lane's 16 rows: 8 g + 4 h ..+3 for g = 0..3
  auto stat = [&](const float* st, mh_f32x16& v) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const tk_f32x4 x = *reinterpret_cast<const tk_f32x4*>(st + 8 * g + 4 * h);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[g * 4 + j] = x[j];
    }
  };
  for (int it = ib; it < ie; ++it) {
    const unsigned short* cur = mh_sm + ((it - ib) & 1) * BUF;
    unsigned short* nxt = mh_sm + (((it - ib) & 1) ^ 1) * BUF;
    const bool more = it + 1 < ie;
    if (more) load(nxt);
    const int q0 = (q0t + ct) * QT;
    if (++ct == nq) ct = 0;
    const float* st = reinterpret_cast<const float*>(cur + 2 * TE);
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int qa = q0 + qb * 32;
      mh_f32x16 S, E;
      mh_zero(S);
      stat(st + QT + qb * 32, E);                                              // dP - delta: the accumulator starts at -delta
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        mh_bf16x8 A[NP];
        mh_frag_rows<NP, QT, DP>(cur, qb * 32, ks, li, h, A);
        if constexpr (KL) {
          mh_bf16x8 Kf[NP];
#pragma unroll
          for (int p = 0; p < NP; ++p) Kf[p] = *reinterpret_cast<const mh_bf16x8*>(kl + (ks * NP + p) * 512);
          mh_mma<NP>(A, Kf, S);
        } else {
          mh_mma<NP>(A, K[ks], S);
        }
        mh_frag_rows<NP, QT, DP>(cur + TE, qb * 32, ks, li, h, A);
        mh_mma<NP>(A, V[ks], E);
      }
      if constexpr (KL) {                                                      // two reads (fragment and K) for every first, one for every second product
        __builtin_amdgcn_sched_group_barrier(0x100, 4 + 3 * NP * 2, 0);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 2 * MM, 0);
          if (i + 2 < KS) __builtin_amdgcn_sched_group_barrier(0x100, 3 * NP, 0);
        }
      } else {
        mh_order<2 * KS, PD, NP, MM, 4>();
      }
      __builtin_amdgcn_sched_barrier(0);
      if (P.causal && qa + off < kw + 31) {                                    // a pair above the diagonal is in the block (uniform)
        asm volatile("");                                                      // (a branch, not selects in every block)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool see = qa + 4 * h + (r & 3) + 8 * (r >> 2) + off >= key;
          S[r] = see ? S[r] : -MH_INF; E[r] = see ? E[r] : 0.f;
        }
      }
      mh_f32x16 L;
      mh_bf16x8 FP[2][NP], FS[2][NP];
      stat(st + qb * 32, L);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float p[8], e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int r = s * 8 + j;
          p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[r], P.sc2, L[r]));
          e[j] = p[j] * E[r];
        }
        mh_planes<NP>(p, FP[s]);
        mh_planes<NP>(e, FS[s]);
      }
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          mh_bf16x8 A[NP];
          mh_frag_cols<NP, QT, DP>(cur + TE, qb * 32 + s * 16, d, lane, A);
          mh_mma<NP>(A, FP[s], dV[d]);
          mh_frag_cols<NP, QT, DP>(cur, qb * 32 + s * 16, d, lane, A);
          mh_mma<NP>(A, FS[s], dK[d]);
        }
      mh_order<4 * DB, PD, 2 * NP, MM, 4>();
      __builtin_amdgcn_sched_barrier(0);
    }
    if (more) store(nxt);
    mh_arrive<decltype(sq)::DMA>();
    __syncthreads();
  }
  const int ln = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)), he = ln >> 5, ke = kw + (ln & 31);      // (anew: no register has to hold them in the loop)
  const bool in = ke < lk;
  if (P.splits > 1) {
    if (!in) return;                                                           // (the join writes the zeros behind the length)
    const long long n = (long long)P.B * P.Hkv * P.Tk;
    float* row = P.part + ((long long)split * 2 * n + (long long)unit * P.Tk + ke) * P.D;
    mh_put<float, DB, WH>(dK, P.scale, true, row, P.D, he);
    mh_put<float, DB, WH>(dV, 1.f, true, row + n * P.D, P.D, he);
  } else if (ke < P.Tk) {
    mh_put<T, DB, WH>(dK, P.scale, in, (T*)P.dk + b * P.kb + (long long)ke * P.kt + (long long)hk * P.kh, P.D, he);
    mh_put<T, DB, WH>(dV, 1.f, in, (T*)P.dv + b * P.vb + (long long)ke * P.vt + (long long)hk * P.vh, P.D, he);
  }
}

// out[b][t][h][d ..] = sum over splits of part[s][(b, h, t)][d ..], in order; `step`: floats between two ranges.  V channels a thread.  blockIdx.y: which
// of two tensors (their partials lie behind one another).  Rows behind their length have no partials: zeros.
struct MhaJoinTo { void* p; long long sb, st, sh; };
template <typename T, int V>
__global__ void __launch_bounds__(256) mha_bwd_join_kernel(const float* __restrict__ part, long long step, int splits, MhaJoinTo to0, MhaJoinTo to1, const int* len,
                                                           int H, int Tn, int D, long long rows) {
  const MhaJoinTo to = blockIdx.y ? to1 : to0;
  const int dv = D / V;
  const long long e = (long long)blockIdx.x * 256 + threadIdx.x, row = e / dv;
  if (row >= rows) return;
  const int c = (int)(e - row * dv) * V, tok = (int)(row % Tn), hh = (int)(row / Tn % H), b = (int)(row / Tn / H);
  const float* p = part + ((long long)blockIdx.y * rows + row) * D + c;
  float s[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s[j] = 0.f;
  const int ranges = tok < mh_len(len, b, Tn) ? splits : 0;
#pragma unroll 8
  for (int k = 0; k < ranges; ++k) {
    float v[V];
    __builtin_memcpy(v, p + k * step, 4 * V);
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] += v[j];
  }
  T* o = (T*)to.p + b * to.sb + (long long)tok * to.st + (long long)hh * to.sh;
  if constexpr (V == 4) mh_store4<T, true>(o, c, D, s[0], s[1], s[2], s[3]);
  else TkVec<T>::store(o + c, s[0]);
}

// ---- host
struct MhaBwdPlan { int dq_tiles, dq_splits, dkv_tiles, dkv_splits; size_t delta_floats, dq_floats, dkv_floats; };
static MhaBwdPlan mh_bwd_plan(const MhaParams& P, int dtype, bool lengths) {
  MhaBwdPlan L = {};
  L.delta_floats = ((size_t)P.B * P.Hq * P.Tq + 3) / 4 * 4;
  if (P.Tq > 0) {
    L.dq_tiles = cdiv(P.Tq, 128);
    L.dq_splits = mh_splits((long long)L.dq_tiles * P.B * P.Hq, P.Tk, dtype, lengths);
    if (L.dq_splits > 1) L.dq_floats = (size_t)L.dq_splits * P.B * P.Hq * P.Tq * P.D;
  }
  if (P.Tk > 0) {
    L.dkv_tiles = cdiv(P.Tk, 128);
    L.dkv_splits = mh_splits((long long)L.dkv_tiles * P.B * P.Hkv, (long long)P.Tq * P.G, dtype, lengths);
    if (L.dkv_splits > 1) L.dkv_floats = (size_t)L.dkv_splits * 2 * P.B * P.Hkv * P.Tk * P.D;
  }
  return L;
}
// dQ and dK / dV partials share their space: the kernels run one after the other
static size_t mh_bwd_bytes(const MhaBwdPlan& L) {
  return (L.delta_floats + (L.dq_floats > L.dkv_floats ? L.dq_floats : L.dkv_floats)) * sizeof(float);
}
size_t k_mha_bwd_workspace_bytes(const MhaParams& P, int dtype) {               // for calls with and without lengths
  const size_t n = mh_bwd_bytes(mh_bwd_plan(P, dtype, true)), m = mh_bwd_bytes(mh_bwd_plan(P, dtype, false));
  return n > m ? n : m;
}

template <typename T, int DP, int KT, int OCC, bool WH = true> static void mh_dq_go(const MhaParams& P, hipStream_t st) {
  constexpr int lds = 4 * MhTile<MhNP<T>::NP, KT, DP>::ELEMS * 2;
  static_assert(lds <= 163840, "LDS");
  hipFuncSetAttribute(reinterpret_cast<const void*>(&mha_dq_kernel<T, DP, KT, OCC, WH>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  hipLaunchKernelGGL((mha_dq_kernel<T, DP, KT, OCC, WH>), dim3((unsigned)mh_grid(P)), dim3(256), lds, st, P);
}
template <typename T, int DP, int QT, int OCC, bool WH = true, bool KL = false> static void mh_dkv_go(const MhaParams& P, hipStream_t st) {
  constexpr int lds = (2 * (2 * MhTile<MhNP<T>::NP, QT, DP>::ELEMS + 4 * QT) + (KL ? 4 * DP / 16 * MhNP<T>::NP * 512 : 0)) * 2;
  static_assert(lds <= 163840, "LDS");
  hipFuncSetAttribute(reinterpret_cast<const void*>(&mha_dkv_kernel<T, DP, QT, OCC, WH, KL>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  hipLaunchKernelGGL((mha_dkv_kernel<T, DP, QT, OCC, WH, KL>), dim3((unsigned)mh_grid(P)), dim3(256), lds, st, P);
}
static void mh_bwd_join(bool bf, const MhaParams& P, long long step, MhaJoinTo to0, MhaJoinTo to1, int n, const int* len, int H, int Tn, long long rows, hipStream_t st) {
  const dim3 grid((unsigned)((rows * P.D / (P.D % 4 ? 1 : 4) + 255) / 256), n);
  if (P.D % 4 == 0) {
    if (bf) hipLaunchKernelGGL((mha_bwd_join_kernel<tk_bf16, 4>), grid, dim3(256), 0, st, P.part, step, P.splits, to0, to1, len, H, Tn, P.D, rows);
    else hipLaunchKernelGGL((mha_bwd_join_kernel<float, 4>), grid, dim3(256), 0, st, P.part, step, P.splits, to0, to1, len, H, Tn, P.D, rows);
  } else {
    if (bf) hipLaunchKernelGGL((mha_bwd_join_kernel<tk_bf16, 1>), grid, dim3(256), 0, st, P.part, step, P.splits, to0, to1, len, H, Tn, P.D, rows);
    else hipLaunchKernelGGL((mha_bwd_join_kernel<float, 1>), grid, dim3(256), 0, st, P.part, step, P.splits, to0, to1, len, H, Tn, P.D, rows);
  }
}

int k_mha_bwd(const MhaParams& P0, int dtype, void* ws, size_t ws_bytes, hipStream_t st) {
  MhaParams P = P0;
  const bool bf = dtype == PDAE_DT_BF16;
  const MhaBwdPlan L = mh_bwd_plan(P, dtype, P.q_len || P.k_len);
  const size_t need = mh_bwd_bytes(L);
  if (P.B == 0 || (P.Tq == 0 && P.Tk == 0)) return PDAE_OK;
  PDAE_CHECK_ARG(need == 0 || (ws && ws_bytes >= need), "mha_bwd: needs %zu bytes of workspace (got %zu)", need, ws ? ws_bytes : (size_t)0);
  P.delta = (float*)ws;
  P.part = (float*)ws + L.delta_floats;
  const long long nq = (long long)P.B * P.Hq * P.Tq, nk = (long long)P.B * P.Hkv * P.Tk;
  PDAE_CHECK_ARG(nq * P.D / 256 < (1ll << 31) && nk * P.D / 256 < (1ll << 31), "mha_bwd: too many rows for one launch");
  const auto query_side = [&] { P.units = P.B * P.Hq; P.tiles = L.dq_tiles; P.splits = L.dq_splits; };
  const auto key_side = [&] { P.units = P.B * P.Hkv; P.tiles = L.dkv_tiles; P.splits = L.dkv_splits; };
  // every check stands before the first launch: a refused call has written nothing
  if (P.Tq > 0) {
    query_side();
    PDAE_CHECK_ARG(mh_grid(P) < (1 << 24), "mha_bwd: too many query tiles for one launch");
  }
  if (P.Tk > 0) {
    key_side();
    PDAE_CHECK_ARG(mh_grid(P) < (1 << 24) && (long long)cdiv(P.Tq, 32) * P.G < (1ll << 31), "mha_bwd: too many tiles for one launch");
  }
  const void* in[5] = {P.Tq ? P.q : nullptr, P.Tk ? P.k : nullptr, P.Tk ? P.v : nullptr, P.Tq ? P.o : nullptr, P.Tq ? P.d_o : nullptr};
  const void* out[3] = {P.Tq ? P.dq : nullptr, P.Tk ? P.dk : nullptr, P.Tk ? P.dv : nullptr};
  for (int i = 0; i < 3; ++i) {
    bool own = true;
    for (const void* x : in) own = own && (!out[i] || out[i] != x);
    for (int j = 0; j < i; ++j) own = own && (!out[i] || out[i] != out[j]);
    PDAE_CHECK_ARG(own, "mha_bwd: a gradient in the place of an input or of another gradient");
  }
  if (P.Tq > 0) {
    query_side();
    if (bf) {
      if (P.D & 7) mh_dq_go<tk_bf16, 128, 64, 1, false>(P, st);
      else if (P.D <= 32) mh_dq_go<tk_bf16, 32, 64, 2>(P, st);
      else if (P.D <= 64) mh_dq_go<tk_bf16, 64, 64, 2>(P, st);
      else if (P.D <= 96) mh_dq_go<tk_bf16, 96, 64, 2>(P, st);
      else mh_dq_go<tk_bf16, 128, 64, 2>(P, st);
    } else {
      if (P.D & 7) mh_dq_go<float, 128, 32, 1, false>(P, st);
      else if (P.D <= 32) mh_dq_go<float, 32, 32, 2>(P, st);
      else if (P.D <= 64) mh_dq_go<float, 64, 32, 2>(P, st);
      else if (P.D <= 96) mh_dq_go<float, 96, 32, 1>(P, st);
      else mh_dq_go<float, 128, 32, 1>(P, st);
    }
    if (int e = pdae_launch_status("mha_dq")) return e;
    if (P.splits > 1) {
      const MhaJoinTo to = {P.dq, P.qb, P.qt, P.qh};
      mh_bwd_join(bf, P, nq * P.D, to, to, 1, P.q_len, P.Hq, P.Tq, nq, st);
    }
  }
  if (P.Tk > 0) {
    key_side();
    if (bf) {
      if (P.D & 7) mh_dkv_go<tk_bf16, 128, 32, 1, false>(P, st);
      else if (P.D <= 32) mh_dkv_go<tk_bf16, 32, 32, 2>(P, st);
      else if (P.D <= 64) mh_dkv_go<tk_bf16, 64, 32, 2>(P, st);
      else if (P.D <= 96) mh_dkv_go<tk_bf16, 96, 32, 2>(P, st);
      else mh_dkv_go<tk_bf16, 128, 32, 2, true, true>(P, st);
    } else {
      if (P.D & 7) mh_dkv_go<float, 128, 32, 1, false>(P, st);
      else if (P.D <= 32) mh_dkv_go<float, 32, 32, 2>(P, st);
      else if (P.D <= 64) mh_dkv_go<float, 64, 32, 1>(P, st);
      else if (P.D <= 96) mh_dkv_go<float, 96, 32, 1>(P, st);
      else mh_dkv_go<float, 128, 32, 1>(P, st);
    }
    if (int e = pdae_launch_status("mha_dkv")) return e;
    if (P.splits > 1) mh_bwd_join(bf, P, 2 * nk * P.D, MhaJoinTo{P.dk, P.kb, P.kt, P.kh}, MhaJoinTo{P.dv, P.vb, P.vt, P.vh}, 2, P.k_len, P.Hkv, P.Tk, nk, st);
  }
  return pdae_launch_status("mha_bwd");
}
