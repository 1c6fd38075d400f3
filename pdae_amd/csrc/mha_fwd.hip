// Attention forward for any number of tokens (mha.h): one pass over the keys with a running reference and sum per query.
//
// Workgroup = 4 waves; wave w owns QB * 32 query rows (its Q fragments stay in registers), the four share key / value tiles of KT tokens in LDS, double
// buffered: the next tile is on its way while this one is multiplied (bf16 with D a multiple of 8: straight into LDS, else through registers), one barrier a
// tile.  Per 32 keys x 32 queries: S^T = K Q^T (DP / 16 MFMAs), p = 2^(sc2 s - reference), O^T += V^T P (DP / 16 MFMAs).
// Every lane holds 16 of a column's 32 scores: the row maximum is a register tree and one exchange with lane ^ 32, the sum stays per lane until the end.
// The reference is the maximum (bf16: MH_LIFT above it) when it is set, and only moves when a tile's weights outgrow MH_GROW: then the accumulators are scaled.
//
// Bound: products and exponentials, which hardly overlap, and the clock.  4 x 16 heads of 128, 4096 tokens, causal, bf16: 272 us after a hundred passes (1010 TFLOP/s;
// the library's 8192^3 product runs at 1320), 302 .. 313 us in the first ten (the clock rises from 1.6 to 1.8 GHz of 2.4); matrix pipes busy 54 % of the CUs' time,
// vector instructions 45 %, LDS 27 %, no bank conflicts.  4 x 8 heads of 64, 4096 tokens: 144 us (957; first ten passes 159).  QB = 2 (64 rows a wave) halves the LDS
// reads a product and pays at D <= 64, where registers allow it (both in their first passes: 162 us, with QB = 1 173).
// fp32, 8 x 4 heads of 64, 1024 tokens: 57 us, first ten passes 67 (six products each: 904 TFLOP/s of bf16 work).  A head width that is no multiple of 8 loads single
// elements and multiplies 128 channels: 4 x 8 heads, 1024 tokens, bf16 59 us at 20 channels, 16 at 24.
//
// Few rows (a token or a few per sample against a long cache): query heads that share a key head are rows of ONE tile (GP = G), and the keys are split into
// ranges (grid `splits`), each leaving an unnormalised partial (O, m, l); the join kernels add them in a fixed order.
#include "kernels.h"
#include "mha.h"

template <typename T, int DP, int QB, int KT, int OCC, bool WH>
__global__ void __launch_bounds__(256, OCC) mha_fwd_kernel(const MhaParams P) {
  constexpr int NP = MhNP<T>::NP, KS = DP / 16, DB = DP / 32, KB = KT / 32;
  constexpr int TE = MhTile<NP, KT, DP>::ELEMS, MM = NP == 3 ? 6 : 1, PD = NP == 3 ? 2 : 4;
  extern __shared__ __attribute__((aligned(16))) unsigned short mh_sm[];       // [2 buffers][K tile | V tile]
  int unit, tile, split;
  if (!mh_where(P, unit, tile, split)) return;
  if (P.causal) tile = P.tiles - 1 - tile;                                     // long rows first
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), li = lane & 31, h = lane >> 5;
  const int b = unit / P.HP, hp = unit % P.HP, hk = hp * P.GP / P.G;
  const int lq = mh_len(P.q_len, b, P.Tq), lk = mh_len(P.k_len, b, P.Tk), off = lk - lq;
  const int row0 = tile * (128 * QB);
  const T* kbase = (const T*)P.k + b * P.kb + hk * P.kh;
  const T* vbase = (const T*)P.v + b * P.vb + hk * P.vh;

  // keys the tile's last existing query sees
  int tlast = (min(row0 + 128 * QB, P.R) - 1) / P.GP;
  tlast = min(tlast, lq - 1);
  int nk = row0 / P.GP >= lq ? 0 : P.causal ? min(lk, tlast + off + 1) : lk;
  nk = max(nk, 0);
  const int ntiles = (nk + KT - 1) / KT;
  const int tb = (int)((long long)ntiles * split / P.splits), te = (int)((long long)ntiles * (split + 1) / P.splits);

  // this lane's query columns
  mh_bf16x8 Q[QB][KS][NP];
  int kmax[QB];
  bool live = false;
#pragma unroll
  for (int a = 0; a < QB; ++a) {
    const int r = row0 + wv * (32 * QB) + a * 32 + li, tq = r / P.GP;
    const bool ok = r < P.R && tq < lq;
    kmax[a] = ok ? (P.causal ? min(lk, tq + off + 1) : lk) : lk;               // rows that do not exist never force the masked path; they are zeroed at the end
    live = live || ok;
    const int t0 = row0 / P.GP;                                                // (the tile's first token: offsets inside a tile fit 32 bits)
    mh_row_frags<T, NP, DP, WH>((const T*)P.q + b * P.qb + (long long)t0 * P.qt + (long long)hp * P.GP * P.qh,
                                ok ? (unsigned)((tq - t0) * P.qt + (r % P.GP) * P.qh) * (unsigned)sizeof(T) : MH_OOB, P.D, h, Q[a]);
  }
  const bool wlive = __any(live);
  int kwave = 0;                                                               // last key any of the wave's rows sees
#pragma unroll
  for (int a = 0; a < QB; ++a) kwave = max(kwave, kmax[a]);

  mh_f32x16 O[QB][DB];
  float m[QB], ms[QB], l[QB];                                                 // reference (log2) so far, the same with 0 for -inf, sum of 2^(t - ms)
#pragma unroll
  for (int a = 0; a < QB; ++a) {
    m[a] = -MH_INF; ms[a] = 0.f; l[a] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) mh_zero(O[a][d]);
  }

  auto weights = [&](const mh_f32x16 (&S)[KB], float ref, mh_bf16x8 (&F)[KB][2][NP]) __attribute__((always_inline)) {
    float sum = 0.f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[kb][s * 8 + j], P.sc2, -ref));
          if (NP == 3) e[j] *= MH_DOWN;
          sum += e[j];
        }
        mh_planes<NP>(e, F[kb][s]);
      }
    return sum;
  };
  MhStage<T, NP, KT, DP, WH> sk, sv;
  sk.init(P.kt, P.D); sv.init(P.vt, P.D);
  if (tb < te) {
    sk.load(kbase, P.kt, tb * KT, 0, lk, mh_sm);
    sv.load(vbase, P.vt, tb * KT, 0, lk, mh_sm + TE);
    sk.store(mh_sm); sv.store(mh_sm + TE);
  }
  mh_loads_done();
  __syncthreads();
  // One key tile: BUF (which buffer it lies in) is a constant, so every LDS address below is one register and an immediate.
  auto step = [&](auto buf_, int it) __attribute__((always_inline)) {
    constexpr int BUF = decltype(buf_)::value;
    const unsigned short* cur = mh_sm + BUF * 2 * TE;
    unsigned short* nxt = mh_sm + (BUF ^ 1) * 2 * TE;
    const bool more = it + 1 < te;
    if (more) { sk.load(kbase, P.kt, (it + 1) * KT, 0, lk, nxt); sv.load(vbase, P.vt, (it + 1) * KT, 0, lk, nxt + TE); }
    const int k0 = it * KT;
    if (wlive && __any(kwave > k0)) {
      mh_f32x16 S[QB][KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int a = 0; a < QB; ++a) mh_zero(S[a][kb]);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          mh_bf16x8 A[NP];
          mh_frag_rows<NP, KT, DP>(cur, kb * 32, ks, li, h, A);
#pragma unroll
          for (int a = 0; a < QB; ++a) mh_mma<NP>(A, Q[a][ks], S[a][kb]);
        }
      }
      mh_order<KB * KS, PD, NP, MM * QB>();
      __builtin_amdgcn_sched_barrier(0);
      mh_bf16x8 F[QB][KB][2][NP];
#pragma unroll
      for (int a = 0; a < QB; ++a) {
        if (__any(k0 + KT > kmax[a])) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) mh_mask_keys(S[a][kb], k0 + kb * 32 + 4 * h, kmax[a]);
        }
        // p = 2^(t - ms) with the reference ms of the tiles before, which only has to be NEAR the maximum (MH_LIFT, MH_GROW: neither the weights nor their
        // products with v leave the range).  It moves (below) when a column has seen no key yet or a tile outgrows it, which leaves three instructions a score here.
        float sum = weights(S[a], ms[a], F[a]);
        if (__any(m[a] == -MH_INF || !(sum <= MH_GROW))) {
          float mx = S[a][0][0];
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, S[a][kb][r]);
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          const float mn = fmaxf(m[a], mh_reference<NP>(mx, P.sc2));
          ms[a] = mn == -MH_INF ? 0.f : mn;                                    // a column that has seen no key yet keeps p = 2^-inf = 0
          const float al = __builtin_amdgcn_exp2f(m[a] - ms[a]);
          m[a] = mn;
          sum = weights(S[a], ms[a], F[a]);
          l[a] *= al;
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) O[a][d][r] *= al;
        }
        l[a] += sum;
      }
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            mh_bf16x8 A[NP];
            mh_frag_cols<NP, KT, DP>(cur + TE, kb * 32 + s * 16, d, lane, A);
#pragma unroll
            for (int a = 0; a < QB; ++a) mh_mma<NP>(A, F[a][kb][s], O[a][d]);
          }
      mh_order<DB * KB * 2, PD, 2 * NP, MM * QB>();
    }
    if (more) { sk.store(nxt); sv.store(nxt + TE); }
    mh_arrive<decltype(sk)::DMA>();
    __syncthreads();
  };
  for (int it = tb; it < te; it += 2) {
    step(MhInt<0>(), it);
    if (it + 1 < te) step(MhInt<1>(), it + 1);
  }

  const int ln = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)), he = ln >> 5;      // rows anew: kept from above, they are spilled around the loop (QB = 2)
#pragma unroll
  for (int a = 0; a < QB; ++a) {
    const int r = row0 + wv * (32 * QB) + a * 32 + (ln & 31);
    if (r >= P.R) continue;
    const int tq = r / P.GP, hq = hp * P.GP + r % P.GP;
    const float ls = l[a] + __shfl_xor(l[a], 32);
    if (P.splits > 1) {
      const long long idx = ((long long)split * P.units + unit) * P.R + r;
      float* po = P.part + idx * P.D;
      float* ml = P.part + (long long)P.splits * P.units * P.R * P.D + idx * 2;
      const bool any = tq < lq && ls != 0.f;                                   // (NaN counts: it has to reach the output)
      if (he == 0) { ml[0] = any ? m[a] : -MH_INF; ml[1] = any ? ls : 0.f; }
      if (any) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g) mh_store4<float, WH>(po, d * 32 + g * 8 + he * 4, P.D, O[a][d][g * 4], O[a][d][g * 4 + 1], O[a][d][g * 4 + 2], O[a][d][g * 4 + 3]);
      }
      continue;
    }
    const bool any = tq < lq && ls != 0.f;                                     // padded rows and rows whose masks leave nothing: zero
    const float inv = any ? 1.0f / ls : 0.f;
    T* orow = (T*)P.out + b * P.ob + (long long)tq * P.ot + (long long)hq * P.oh;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float x0 = any ? O[a][d][g * 4] * inv : 0.f, x1 = any ? O[a][d][g * 4 + 1] * inv : 0.f;
        const float x2 = any ? O[a][d][g * 4 + 2] * inv : 0.f, x3 = any ? O[a][d][g * 4 + 3] * inv : 0.f;
        mh_store4<T, WH>(orow, d * 32 + g * 8 + he * 4, P.D, x0, x1, x2, x3);
      }
    if (P.lse && he == 0) P.lse[((long long)b * P.Hq + hq) * P.Tq + tq] = any ? mh_lse<NP>(m[a], ls) : -MH_INF;      // (v_log_f32: log2)
  }
}

// At most 32 rows (a token, or a few, of the heads that share a key head), bf16: every wave works for itself on 32 keys at a time, loaded straight into its own LDS,
// double buffered, without a barrier; the waves of a block take turns through its key range and are joined in LDS at the end.  In the kernel above the
// 128-row tile would leave three waves without rows, and the fourth's latency per tile would be the block's (24 samples, 32 heads on 8 of 128, ragged caches of up to
// 8191, with the join: 112 us there, 89 here).  Bound: HBM; full caches of 8192 keys run at 5.1 .. 5.6 TB/s, 2048 keys of 32 key heads at 5.7 .. 6.0.
template <int DP, int OCC>
__global__ void __launch_bounds__(256, OCC) mha_token_kernel(const MhaParams P) {
  constexpr int KS = DP / 16, DB = DP / 32, TE = MhTile<1, 32, DP>::ELEMS, OL = DP + 4;
  using Stage = MhStage<tk_bf16, 1, 32, DP, true, 64>;
  static_assert(Stage::DMA && 32 * OL * 4 + 256 <= 8 * TE, "a wave's result fits its own tiles");
  extern __shared__ __attribute__((aligned(16))) unsigned short mh_sm[];       // per wave: [2 buffers][K tile | V tile], then its O [32][OL], m[32], l[32] (floats)
  int unit, tile, split;
  if (!mh_where(P, unit, tile, split)) return;
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), li = lane & 31, h = lane >> 5;
  const int b = unit / P.HP, hp = unit % P.HP, hk = hp * P.GP / P.G;
  const int lq = mh_len(P.q_len, b, P.Tq), lk = mh_len(P.k_len, b, P.Tk), off = lk - lq;
  const tk_bf16* kbase = (const tk_bf16*)P.k + b * P.kb + hk * P.kh;
  const tk_bf16* vbase = (const tk_bf16*)P.v + b * P.vb + hk * P.vh;
  const int nk = max(0, lq <= 0 ? 0 : P.causal ? min(lk, min((P.R - 1) / P.GP, lq - 1) + off + 1) : lk), ntiles = (nk + 31) / 32;
  const int tb = (int)((long long)ntiles * split / P.splits), te = (int)((long long)ntiles * (split + 1) / P.splits);
  const int tq = li / P.GP;
  const bool ok = li < P.R && tq < lq;
  const int kmax = ok ? (P.causal ? min(lk, tq + off + 1) : lk) : lk;
  mh_bf16x8 Q[KS][1];
  mh_row_frags<tk_bf16, 1, DP, true>((const tk_bf16*)P.q + b * P.qb + (long long)hp * P.GP * P.qh,
                                     ok ? (unsigned)(tq * P.qt + (li % P.GP) * P.qh) * 2u : MH_OOB, P.D, h, Q);
  unsigned short* mine = mh_sm + wv * 4 * TE;
  mh_f32x16 O[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) mh_zero(O[d]);
  float m = -MH_INF, ms = 0.f, l = 0.f;
  Stage sk, sv;
  sk.init(P.kt, P.D); sv.init(P.vt, P.D);
  mh_loads_done();
  int it = tb + wv, buf = 0;
  if (it < te) { sk.load(kbase, P.kt, it * 32, 0, lk, mine); sv.load(vbase, P.vt, it * 32, 0, lk, mine + TE); }
  for (; it < te; it += 4, buf ^= 1) {
    const unsigned short* cur = mine + buf * 2 * TE;
    if (it + 4 < te) {
      unsigned short* nxt = mine + (buf ^ 1) * 2 * TE;
      sk.load(kbase, P.kt, (it + 4) * 32, 0, lk, nxt); sv.load(vbase, P.vt, (it + 4) * 32, 0, lk, nxt + TE);
      mh_arrive_but<2 * Stage::N>();
    } else {
      mh_arrive_but<0>();
    }
    mh_f32x16 S;
    mh_zero(S);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      mh_bf16x8 A[1];
      mh_frag_rows<1, 32, DP>(cur, 0, ks, li, h, A);
      mh_mma<1>(A, Q[ks], S);
    }
    mh_order<KS, 4, 1, 1>();
    __builtin_amdgcn_sched_barrier(0);
    if (__any(it * 32 + 32 > kmax)) mh_mask_keys(S, it * 32 + 4 * h, kmax);
    float mx = S[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, S[r]);
    mx = mh_reference<1>(fmaxf(mx, __shfl_xor(mx, 32)), P.sc2);
    if (__any(m == -MH_INF || !(mx - m <= 12.f))) {                             // weights up to 2^(12 - MH_LIFT) = 2^-20: the bound of MH_GROW
      const float mn = fmaxf(m, mx), msn = mn == -MH_INF ? 0.f : mn, al = __builtin_amdgcn_exp2f(m - msn);
      m = mn; ms = msn; l *= al;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[d][r] *= al;
    }
    mh_bf16x8 F[2][1];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) { e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[s * 8 + j], P.sc2, -ms)); l += e[j]; }
      mh_planes<1>(e, F[s]);
    }
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        mh_bf16x8 A[1];
        mh_frag_cols<1, 32, DP>(cur + TE, s * 16, d, lane, A);
        mh_mma<1>(A, F[s], O[d]);
      }
    mh_order<DB * 2, 4, 2, 1>();
    __builtin_amdgcn_sched_barrier(0);
  }
  // join of the four waves, in wave order
  l += __shfl_xor(l, 32);
  float* po = reinterpret_cast<float*>(mine);
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<tk_f32x4*>(po + li * OL + d * 32 + g * 8 + h * 4) = tk_f32x4{O[d][g * 4], O[d][g * 4 + 1], O[d][g * 4 + 2], O[d][g * 4 + 3]};
  if (h == 0) { po[32 * OL + li] = ok && l != 0.f ? m : -MH_INF; po[32 * OL + 32 + li] = ok ? l : 0.f; }
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(mh_sm);
  for (int i = t; i < P.R * (DP / 4); i += 256) {
    const int r = i / (DP / 4), c = i % (DP / 4) * 4;
    if (c >= P.D) continue;
    float M = -MH_INF, L = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, all[w * 2 * TE + 32 * OL + r]);
    const float Ms = M == -MH_INF ? 0.f : M;
    tk_f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float lw = all[w * 2 * TE + 32 * OL + 32 + r];
      if (lw == 0.f) continue;                                                  // a wave without keys
      const float x = __builtin_amdgcn_exp2f(all[w * 2 * TE + 32 * OL + r] - Ms);
      const tk_f32x4 v = *reinterpret_cast<const tk_f32x4*>(all + w * 2 * TE + r * OL + c);
      L += x * lw;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += x * v[j];
    }
    if (P.splits > 1) {
      const long long idx = ((long long)split * P.units + unit) * P.R + r;
      if (L != 0.f) __builtin_memcpy(P.part + idx * P.D + c, &o, 16);
      if (c == 0) {
        float* ml = P.part + (long long)P.splits * P.units * P.R * P.D + idx * 2;
        ml[0] = M; ml[1] = L;
      }
      continue;
    }
    const float inv = L != 0.f ? 1.0f / L : 0.f;
    const int tr = r / P.GP, hr = hp * P.GP + r % P.GP;
    tk_bf16* orow = (tk_bf16*)P.out + b * P.ob + (long long)tr * P.ot + (long long)hr * P.oh;
    mh_store4<tk_bf16, true>(orow, c, P.D, L != 0.f ? o[0] * inv : 0.f, L != 0.f ? o[1] * inv : 0.f, L != 0.f ? o[2] * inv : 0.f, L != 0.f ? o[3] * inv : 0.f);
    if (P.lse && c == 0) P.lse[((long long)b * P.Hq + hr) * P.Tq + tr] = L != 0.f ? mh_lse<1>(M, L) : -MH_INF;
  }
}

// Adds the key ranges of a split forward: o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s.  One thread per four channels of a row (V = 1: one channel, D % 4).
template <typename T, int V>
__global__ void __launch_bounds__(256) mha_join_kernel(const MhaParams P) {
  const int dv = P.D / V;
  const long long n = (long long)P.units * P.R, e = (long long)blockIdx.x * 256 + threadIdx.x, i = e / dv;
  if (i >= n) return;
  const int c = (int)(e - i * dv) * V, unit = (int)(i / P.R), r = (int)(i % P.R), b = unit / P.HP, hq = unit % P.HP * P.GP + r % P.GP, tq = r / P.GP;
  const float* ml = P.part + (long long)P.splits * n * P.D;
  // loads of eight ranges in flight: one by one, 32 ranges of a single token were 30 us of latency
  float M = -MH_INF;
#pragma unroll 8
  for (int s = 0; s < P.splits; ++s) {
    const tk_f32x2 x = *reinterpret_cast<const tk_f32x2*>(ml + (s * n + i) * 2);
    M = fmaxf(M, x[1] != 0.f ? x[0] : -MH_INF);
  }
  const float Ms = M == -MH_INF ? 0.f : M;
  float L = 0.f, o[V];
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = 0.f;
#pragma unroll 8
  for (int s = 0; s < P.splits; ++s) {
    const tk_f32x2 x = *reinterpret_cast<const tk_f32x2*>(ml + (s * n + i) * 2);
    const bool any = x[1] != 0.f;                                              // an empty range wrote no O: what lies there is not used
    const float w = any ? __builtin_amdgcn_exp2f(x[0] - Ms) : 0.f;
    float v[V];
    __builtin_memcpy(v, P.part + (s * n + i) * P.D + c, 4 * V);
    L += w * x[1];
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] += any ? w * v[j] : 0.f;
  }
  const float inv = L != 0.f ? 1.0f / L : 0.f;
  T* orow = (T*)P.out + b * P.ob + (long long)tq * P.ot + (long long)hq * P.oh;
  if constexpr (V == 4) mh_store4<T, true>(orow, c, P.D, L != 0.f ? o[0] * inv : 0.f, L != 0.f ? o[1] * inv : 0.f, L != 0.f ? o[2] * inv : 0.f, L != 0.f ? o[3] * inv : 0.f);
  else TkVec<T>::store(orow + c, L != 0.f ? o[0] * inv : 0.f);
  if (P.lse && c == 0) P.lse[((long long)b * P.Hq + hq) * P.Tq + tq] = L != 0.f ? mh_lse<MhNP<T>::NP>(M, L) : -MH_INF;
}
// The same for few rows in many ranges: a block per row, its G = 256 / lanes groups take every G-th range and are added in group order through LDS (one
// thread after another through 32 ranges of a single token was 19 us of latency beside 7 us of attention).
template <typename T>
__global__ void __launch_bounds__(256) mha_join_row_kernel(const MhaParams P) {
  __shared__ float wsum[8][129];
  __shared__ float mls[2][256];
  const long long n = (long long)P.units * P.R, i = blockIdx.x;
  const int t = threadIdx.x, lane = t & 31, g = t >> 5, c = lane * 4;                       // D <= 128: 32 lanes of four channels, eight groups
  const float* ml = P.part + (long long)P.splits * n * P.D;
  const int S = P.splits;                                                                   // (the host: at most 256)
  if (t < S) {
    const tk_f32x2 x = *reinterpret_cast<const tk_f32x2*>(ml + (t * n + i) * 2);
    mls[0][t] = x[1] != 0.f ? x[0] : -MH_INF; mls[1][t] = x[1];
  }
  __syncthreads();
  float M = -MH_INF;
  for (int s = 0; s < S; ++s) M = fmaxf(M, mls[0][s]);
  const float Ms = M == -MH_INF ? 0.f : M;
  float L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = g; s < S; s += 8) {
    const float l = mls[1][s], w = l != 0.f ? __builtin_amdgcn_exp2f(mls[0][s] - Ms) : 0.f;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = c + j < P.D ? P.part[(s * n + i) * P.D + c + j] : 0.f;
    L += w * l;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] += l != 0.f ? w * v[j] : 0.f;                          // an empty range wrote no O
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) wsum[g][c + j] = o[j];
  if (lane == 0) wsum[g][128] = L;
  __syncthreads();
  if (t >= P.D) return;
  float x = 0.f, l = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) { x += wsum[k][t]; l += wsum[k][128]; }
  const int unit = (int)(i / P.R), r = (int)(i % P.R), b = unit / P.HP, hq = unit % P.HP * P.GP + r % P.GP, tq = r / P.GP;
  TkVec<T>::store((T*)P.out + b * P.ob + (long long)tq * P.ot + (long long)hq * P.oh + t, l != 0.f ? x / l : 0.f);
  if (P.lse && t == 0) P.lse[((long long)b * P.Hq + hq) * P.Tq + tq] = l != 0.f ? mh_lse<MhNP<T>::NP>(M, l) : -MH_INF;
}
template <typename T> static void mh_join(const MhaParams& P, hipStream_t st) {
  if (P.splits >= 4 && P.splits <= 256 && (long long)P.units * P.R <= 4096) {
    hipLaunchKernelGGL((mha_join_row_kernel<T>), dim3((unsigned)((long long)P.units * P.R)), dim3(256), 0, st, P);
    return;
  }
  const long long n = (long long)P.units * P.R * P.D;
  if (P.D % 4 == 0) hipLaunchKernelGGL((mha_join_kernel<T, 4>), dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, st, P);
  else hipLaunchKernelGGL((mha_join_kernel<T, 1>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, P);
}

// ---- host: row packing, key ranges
static bool mh_token(const MhaParams& P, int dtype) { return dtype == PDAE_DT_BF16 && P.R <= 32 && P.D % 8 == 0; }
// 64 rows a wave where the chip stays full with half the workgroups (4 heads of 64, 256 tokens: 11.8 us that way, 8.2 with 32 rows; 16 x 8 heads of 40, 1024 x 77 tokens: 15.7
// and 16.5)
static int mh_qb(const MhaParams& P, int dtype) {
  return dtype == PDAE_DT_BF16 && P.R > 128 && P.D <= 64 && P.D % 8 == 0 && (long long)P.units * cdiv(P.R, 256) >= 256 ? 2 : 1;
}
// Rows of a tile: with few query tokens the G heads that share a key head become rows of one tile, so its keys are read once for all of them.
// Then, where the tiles do not fill the chip, the keys are split into ranges.
static void mh_fwd_plan(MhaParams& P, int dtype, bool lengths) {
  P.GP = (long long)P.Tq * P.G <= 128 ? P.G : 1;
  P.HP = P.Hq / P.GP;
  P.R = P.Tq * P.GP;
  P.units = P.B * P.HP;
  P.tiles = cdiv(P.R, 128 * mh_qb(P, dtype));
  P.splits = mh_splits((long long)P.units * P.tiles, P.Tk, dtype, lengths, mh_token(P, dtype));
}
template <int DP, int OCC> static void mh_token_go(const MhaParams& P, hipStream_t st) {
  constexpr int lds = 16 * MhTile<1, 32, DP>::ELEMS * 2;
  hipFuncSetAttribute(reinterpret_cast<const void*>(&mha_token_kernel<DP, OCC>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  hipLaunchKernelGGL((mha_token_kernel<DP, OCC>), dim3((unsigned)mh_grid(P)), dim3(256), lds, st, P);
}
static size_t mh_fwd_part_floats(const MhaParams& P) { return P.splits > 1 ? (size_t)P.splits * P.units * P.R * (P.D + 2) : 0; }

// for calls with and without lengths
size_t k_mha_fwd_workspace_bytes(const MhaParams& P0, int dtype) {
  MhaParams P = P0;
  if (P.B <= 0 || P.Tq <= 0) return 0;
  mh_fwd_plan(P, dtype, true);
  const size_t n = mh_fwd_part_floats(P);
  mh_fwd_plan(P, dtype, false);
  const size_t m = mh_fwd_part_floats(P);
  return (n > m ? n : m) * sizeof(float);
}

template <typename T, int DP, int QB, int KT, int OCC, bool WH = true> static void mh_fwd_go(const MhaParams& P, hipStream_t st) {
  constexpr int NP = MhNP<T>::NP;
  const size_t lds = (size_t)4 * MhTile<NP, KT, DP>::ELEMS * 2;
  static_assert(4 * MhTile<NP, KT, DP>::ELEMS * 2 <= 163840, "LDS");
  hipFuncSetAttribute(reinterpret_cast<const void*>(&mha_fwd_kernel<T, DP, QB, KT, OCC, WH>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  hipLaunchKernelGGL((mha_fwd_kernel<T, DP, QB, KT, OCC, WH>), dim3((unsigned)mh_grid(P)), dim3(256), lds, st, P);
}

int k_mha_fwd(const MhaParams& P0, int dtype, void* ws, size_t ws_bytes, hipStream_t st) {
  MhaParams P = P0;
  if (P.B == 0 || P.Tq == 0) return PDAE_OK;
  mh_fwd_plan(P, dtype, P.q_len || P.k_len);
  const size_t need = mh_fwd_part_floats(P) * sizeof(float);
  PDAE_CHECK_ARG(need == 0 || (ws && ws_bytes >= need), "mha_fwd: needs %zu bytes of workspace (got %zu)", need, ws ? ws_bytes : (size_t)0);
  PDAE_CHECK_ARG(mh_grid(P) < (1 << 24) && (long long)P.units * P.R < (1ll << 31), "mha_fwd: too many query rows for one launch");
  PDAE_CHECK_ARG(P.splits == 1 || (long long)P.units * P.R * P.D / 256 < (1ll << 31), "mha_fwd: too many query rows for one launch");      // (the join)
  PDAE_CHECK_ARG(P.out != P.q && (P.Tk == 0 || (P.out != P.k && P.out != P.v)), "mha_fwd: o in the place of q, k or v");
  P.part = (float*)ws;
  const int qb = mh_qb(P, dtype);
  if (mh_token(P, dtype)) {
    if (P.D <= 32) mh_token_go<32, 4>(P, st);
    else if (P.D <= 64) mh_token_go<64, 2>(P, st);
    else if (P.D <= 96) mh_token_go<96, 1>(P, st);
    else mh_token_go<128, 1>(P, st);
  } else if (dtype == PDAE_DT_BF16) {
    if (P.D & 7) mh_fwd_go<tk_bf16, 128, 1, 64, 2, false>(P, st);
    else if (P.D <= 32) { if (qb == 2) mh_fwd_go<tk_bf16, 32, 2, 64, 2>(P, st); else mh_fwd_go<tk_bf16, 32, 1, 64, 2>(P, st); }
    else if (P.D <= 64) { if (qb == 2) mh_fwd_go<tk_bf16, 64, 2, 64, 2>(P, st); else mh_fwd_go<tk_bf16, 64, 1, 64, 2>(P, st); }
    else if (P.D <= 96) mh_fwd_go<tk_bf16, 96, 1, 64, 2>(P, st);
    else mh_fwd_go<tk_bf16, 128, 1, 64, 2>(P, st);
  } else {
    if (P.D & 7) mh_fwd_go<float, 128, 1, 32, 1, false>(P, st);
    else if (P.D <= 32) mh_fwd_go<float, 32, 1, 32, 2>(P, st);
    else if (P.D <= 64) mh_fwd_go<float, 64, 1, 32, 2>(P, st);
    else if (P.D <= 96) mh_fwd_go<float, 96, 1, 32, 1>(P, st);
    else mh_fwd_go<float, 128, 1, 32, 1>(P, st);
  }
  if (int e = pdae_launch_status("mha_fwd")) return e;
  if (P.splits > 1) {
    if (dtype == PDAE_DT_BF16) mh_join<tk_bf16>(P, st);
    else mh_join<float>(P, st);
    return pdae_launch_status("mha_join");
  }
  return PDAE_OK;
}
