// Attention in a sliding window with sinks on gfx950, backward (definitions, operand layouts and LDS image: win_attn.h).
//
// With P from the forward pass's log-sum-exp and Delta = rowsum(dO o O):  dV = P^T dO,  dS = P o (dO V^T - Delta),  dQ = scale dS K,  dK = scale dS^T Q.
//   dq_kernel     query rows as in the forward kernel: S^T, dP^T with a query per lane, dQ^T += K^T dS^T.  Also writes Delta.
//   dkv_kernel, window_pass   128 keys of one (sequence, k|v head), 32 per wave: k, v (heads of 128: in LDS) and both gradients stay in registers while the query rows whose windows hold the keys pass
//                 through a double-buffered LDS ring, for every query head that shares the keys: their gradients are summed here, no atomics.
//   dkv_kernel, sink_pass     the sinks meet EVERY later row: one key block would walk the whole sequence while all others walk a window.  The pairs (sink, row beyond its
//                 window) are a pass of their own, split over the rows, a wave per 32-row tile; f32 partial sums.
//   dkv_reduce_kernel  adds the partial sums of split keys in a fixed order.  Every result is bit-reproducible.
// Seven products per visible block (five are needed at least; the other two are S and dP again, because dQ across key tiles would need float atomics).
//
// Bounds, MI355X.  32768 tokens, 12 heads of 64, window 512 + 512: dQ 219, dK / dV 311, reduction 7 us (0.70 and 0.66 PFLOP/s of the seven products; a large one reaches 1.2): dQ has
// the matrix cores busy 0.36 of the time, the vector units 0.49, the LDS 0.19, dK / dV 0.33, 0.41, 0.27: no unit is at its limit, but the shares add up to the whole, for a wave's step
// goes from one to the next and the two waves of a SIMD overlap little of it.  2 x 8191 tokens, 32 heads of
// 128 on 8, causal window 1023: dQ 452-484, dK / dV 640-750 us (cards differ), 0.83 and 0.75 PFLOP/s.
#include "win_attn.h"

namespace win {

template <typename T, int D, bool DROP, bool FINE>
__global__ __launch_bounds__(256, 2) void dq_kernel(Params p, int nunits, int nqt) {
  typedef Geo<T, D> G;
  constexpr int KT = G::KT, TILE = KT * G::ROWB;
  extern __shared__ __attribute__((aligned(16))) char lds[];       // [2][K | V], additive mask [2][KT]
  float* kb = reinterpret_cast<float*>(lds + 4 * TILE);
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, c = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Unit u = unit_of(p, blockIdx.x, nunits, nqt, p.G);
  if (!u.real) return;
  const Rows rw = rows_of(p, u.b);
  const int q0 = u.tile * QB;
  if (q0 >= rw.lq) return;
  const int h = u.hk * p.G + u.g, nq = rw.lq - q0 < QB ? rw.lq - q0 : QB;
  const int lo = p.q_start + q0, hi = lo + nq - 1;
  const TileList tl = tile_list<KT>(lo, hi, p.left, p.right, p.sinks, rw.lk);

  int row = q0 + 32 * wave + c;
  const bool real = row < rw.lq;
  row = real ? row : rw.lq - 1;
  const int wlo = lo + 32 * wave, whi = wlo + 31 < hi ? wlo + 31 : hi;
  const int pos = p.q_start + row;
  RowFrag<T, D> qf, df;
  row_frag_global<T, D>(qf, reinterpret_cast<const T*>(p.q) + (rw.q0 + row) * p.ldq + (int64_t)h * D, half);
  row_frag_global<T, D>(df, reinterpret_cast<const T*>(p.dout) + (rw.q0 + row) * p.lddo + (int64_t)h * D, half);
  float delta;
  {
    RowFrag<T, D> of;
    row_frag_global<T, D>(of, reinterpret_cast<const T*>(p.o) + (rw.q0 + row) * p.ldo + (int64_t)h * D, half);
    delta = row_dot<D>(of, df);
    if (sizeof(T) == 2 && p.out_lo) {      // the O that the probabilities give, to 2^-17: with the rounded one alone its error is half of dS's (kernel-uniform)
      row_frag_global<T, D>(of, reinterpret_cast<const T*>(p.out_lo) + (rw.q0 + row) * p.ldo + (int64_t)h * D, half);
      delta += row_dot<D>(of, df);
    }
    delta = half_sum(delta);
  }
  float top = p.lse[(int64_t)h * p.Mq + rw.q0 + row], lsum = p.lse[(int64_t)(p.H + h) * p.Mq + rw.q0 + row];
  row_frag_arrive<T, D>(qf);
  row_frag_arrive<T, D>(df);
  asm volatile("" : "+v"(top), "+v"(lsum));
  const float lse = top + lsum;
  if (real && half == 0) p.delta[(int64_t)h * p.Mq + rw.q0 + row] = delta;
  const Sight sight(wlo, whi, p.left, p.right, p.sinks, rw.lk);
  const LaneAt<T, D> at(lane);
  KeyPipe<T, D, KT, 256> kp(p, rw.k0, u.hk, rw.lk, lo - p.left, hi + p.right, tid);
  f32x16 acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  const int64_t sh = (int64_t)u.b * p.H + h;
  int state = 0;
  if (tl.n > 0) {
    kp.issue(lds, lds + TILE, tile_at(tl, 0) * KT, tid);
    state = kp.settle(lds, lds + TILE, kb, tid);
  }
  __syncthreads();
  for (int it = 0; it < tl.n; ++it) {
    const int buf = it & 1, j0 = tile_at(tl, it) * KT;
    const bool more = it + 1 < tl.n;
    char* next = lds + (buf ^ 1) * 2 * TILE;               // (its readers are behind the last barrier)
    if (more) kp.issue(next, next + TILE, tile_at(tl, it + 1) * KT, tid);
    if (state != 2) {
#pragma unroll
      for (int b = 0; b < KT / 32; ++b) {
        const int jb = j0 + 32 * b;
        const char *kt = lds + buf * 2 * TILE + 32 * b * G::ROWB, *vt = kt + TILE;
        const int see = sight.of(jb);
        if (!see) continue;
        RowFrag<T, D> kf;
        row_frag_lds<T, D>(kf, kt, at);
        f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
        s = mma_rows<D>(kf, qf, s);
        row_frag_lds<T, D>(kf, vt, at);
        dp = mma_rows<D>(kf, df, dp);
        float pr[16];
        if (state) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(kb + buf * KT + 32 * b + 8 * g + 4 * half);
#pragma unroll
            for (int e = 0; e < 4; ++e) pr[4 * g + e] = __builtin_amdgcn_exp2f(fmaf(s[4 * g + e], p.scale2, a[e]) - top - lsum);
          }
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) pr[r] = __builtin_amdgcn_exp2f(fmaf(s[r], p.scale2, -lse));
        }
        if (see == 1) {
          const int bb = jb + 4 * half;
          const int jh = (pos + p.right < rw.lk - 1 ? pos + p.right : rw.lk - 1) - bb, jl = pos - p.left - bb, sk_ = p.sinks - bb;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int j = 8 * (r >> 2) + (r & 3);
            pr[r] = (j <= jh && (j >= jl || j < sk_)) ? pr[r] : 0.f;
          }
        }
        if (DROP) {
          float dm[16];
          drop_of_query<true>(dm, p, sh, row, jb, half);
#pragma unroll
          for (int r = 0; r < 16; ++r) dp[r] *= dm[r];
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) pr[r] *= dp[r] - delta;
        PFrag<T> pf;
        p_frag(pf, pr);
        mma_cols<T, D>(acc, kt, at, pf, lane);
        if constexpr (FINE) {
          p_rest(pr);
          p_frag(pf, pr);
          mma_cols<T, D>(acc, kt, at, pf, lane);
        }
      }
    }
    if (more) state = kp.settle(next, next + TILE, kb + (buf ^ 1) * KT, tid);
    __syncthreads();
  }
  const int wr = q0 + 32 * wave;           // (everybody is behind the last barrier: the tiles' space is free)
  store_rows<T, D, false>(lds + wave * 32 * G::ROWB, acc, p.scale, reinterpret_cast<T*>(p.dq) + (rw.q0 + wr) * p.lddq + (int64_t)h * D, p.lddq, rw.lq - wr, lane);
}

// The shape of the dK / dV kernel.  Four waves with k, v and both gradients of 32 keys each in registers, or (bf16 heads of 128, where that is 192 registers and would leave
// a SIMD one wave) k and v in LDS and eight waves, two to a 32-key block: 1105 against 1150 us for the backward pass of 2 x 8191 tokens, 32 heads on 8; k in registers
// beside v in LDS spills (1558).  Heads of 64 that way: 549 instead of 467 us for 32768 tokens of 12 heads, with four waves per SIMD (spills) 1057.
// Not everything that is shipped fits its registers either: of heads of 128 the bf16 form keeps 21 of them in scratch with dropout and 7 with remainders (65 with both), and in
// dQ with remainders 18 (24 with dropout too); f32 dQ of heads of 128 keeps 115 (150 with dropout), f32 dK / dV of heads of 64 32 (39).  2 x 4095 tokens, 16 heads of 128, window 511, causal: backward 211 us,
// 315 with dropout; 4 x 8192 tokens, 12 heads of 64: 301 and 496, most of it the generator's vector work.
template <typename T, int D> struct Dkv {
  static constexpr bool IN_LDS = sizeof(T) == 2 && D == 128;
  static constexpr int PAIR = IN_LDS ? 2 : 1, WAVES = 4 * PAIR, NT = 64 * WAVES;
  static constexpr int QT = sizeof(T) == 2 ? 64 : 32;      // query rows of a step
  static constexpr int TILE = QT * Geo<T, D>::ROWB, KEYS = IN_LDS ? 2 * QB * Geo<T, D>::ROWB : 0;      // bytes: a tile of rows, k and v
  static constexpr int WINDOW = KEYS + 4 * TILE + 6 * QT * 4;                                          // [k | v], [2][Q | dO], [2][statistics]
  static constexpr int OWN = 64 * Geo<T, D>::ROWB + 384;                                               // a wave's [Q | dO | statistics] of 32 rows
  static constexpr int SINK = (IN_LDS ? 64 * Geo<T, D>::ROWB : 0) + WAVES * OWN, FOLD = WAVES * 32 * (D + 4) * 4;
  static constexpr int LDS = WINDOW > SINK ? (WINDOW > FOLD ? WINDOW : FOLD) : (SINK > FOLD ? SINK : FOLD);
};
// 32 staged queries against the 32 keys of a wave
template <typename T, int D, bool IN_LDS = Dkv<T, D>::IN_LDS> struct KeyState {
  RowFrag<T, D> kf, vf;
  f32x16 dk[D / 32], dv[D / 32];
};
template <typename T, int D> struct KeyState<T, D, true> {
  const char *kb, *vb;                     // the keys' 32 rows in LDS
  f32x16 dk[D / 32], dv[D / 32];
};
// dropout multipliers of a lane's key and the 16 queries row + 8 (r >> 2) + 4 h + (r & 3).  The four lanes of a key quad need the same eight blocks (2 rows x 4 keys
// each): every lane draws two and the words travel by DPP quad broadcasts.
template <int LANE> __device__ __forceinline__ uint32_t quad_bcast(uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, LANE * 0x55, 0xF, 0xF, true); }
__device__ __forceinline__ void drop_of_key(float (&m)[16], const Params& p, int64_t sh, int row, int j, int half) {
  const uint64_t seed = p.seed + (p.seed_state ? p.seed_state[0] : 0ull);
  const uint32_t thr = attn_drop_threshold(p.drop_p);
  const int ln = (int)(threadIdx.x & 3);
  u32x4 own[2];                            // blocks 2 ln, 2 ln + 1: rows row + 8 ln + 4 h + {0, 1}, {2, 3}
#pragma unroll
  for (int s = 0; s < 2; ++s) own[s] = attn_drop_block(seed, sh, p.Lk, row + 8 * ln + 4 * half + 2 * s, j);
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    u32x4 w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[0][e] = quad_bcast<0>(own[s][e]); w[1][e] = quad_bcast<1>(own[s][e]); w[2][e] = quad_bcast<2>(own[s][e]); w[3][e] = quad_bcast<3>(own[s][e]);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int e = 0; e < 2; ++e) m[4 * g + 2 * s + e] = attn_drop_pick(w[g], e, j, thr, p.inv_keep);
  }
}
// FAR: the sink pass (keys seen because they are sinks, j < i - left); otherwise the window (i - left <= j <= i + right).
template <typename T, int D, bool DROP, bool FAR, bool FINE>
__device__ __forceinline__ void query_block(KeyState<T, D>& st, const char* qt, const char* dt, const float* stat, int rows, const LaneAt<T, D>& at, const Params& p,
                                            int row, int j, float kbias, bool partial, int lane, int64_t sh) {
  const int half = lane >> 5;
  constexpr bool IN_LDS = Dkv<T, D>::IN_LDS;
  RowFrag<T, D> f, f2;
  row_frag_lds<T, D>(f, qt, at);
  f32x16 s, dp;
#pragma unroll
  for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
  if constexpr (IN_LDS) {
    row_frag_lds<T, D>(f2, st.kb, at);
    s = mma_rows<D>(f, f2, s);
  } else {
    row_frag_lds<T, D>(f2, dt, at);
    s = mma_rows<D>(f, st.kf, s);
  }
  if (partial) {                           // row >= j - right, row <= j + left (positions), or beyond: row > j + left and j a sink
    const int o = p.q_start + row + 4 * half;
    const int rl = j - p.right - o, rh = j + p.left - o;
    const bool sink = j < p.sinks;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int i = 8 * (r >> 2) + (r & 3);
      s[r] = (FAR ? (sink && i > rh) : (i >= rl && i <= rh)) ? s[r] : -INFINITY;
    }
  }
  float pr[16], dm[16], ls[16], de[16];    // (stat: RowSource::put_stat)
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(stat + 8 * g + 4 * half), b = *reinterpret_cast<const f32x4*>(stat + rows + 8 * g + 4 * half);
#pragma unroll
    for (int e = 0; e < 4; ++e) { ls[4 * g + e] = a[e]; de[4 * g + e] = b[e]; }
  }
  if (p.keymask) {                         // kernel-uniform; without a mask: 0, and keys past the end are zeros whose gradients nobody stores
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(stat + 2 * rows + 8 * g + 4 * half);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[4 * g + e] = fmaf(s[4 * g + e], p.scale2, kbias) - a[e] - ls[4 * g + e];
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], p.scale2, -ls[r]);
  }
  if (DROP) drop_of_key(dm, p, sh, row, j, half);
  PFrag<T> pf, df;
  if constexpr (IN_LDS) {                  // one operand at a time
    row_frag_lds<T, D>(f, dt, at);
    row_frag_lds<T, D>(f2, st.vb, at);
    dp = mma_rows<D>(f, f2, dp);
  } else {
    dp = mma_rows<D>(f2, st.vf, dp);
  }
  ColFrag<T, D> dc, qc;
  if constexpr (!IN_LDS) col_frag_lds<D>(dc, dt, at);
  float pd[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) { pr[r] = __builtin_amdgcn_exp2f(s[r]); pd[r] = DROP ? pr[r] * dm[r] : pr[r]; }
  p_frag(pf, pd);
  if constexpr (IN_LDS) col_frag_lds<D>(dc, dt, at);
  else col_frag_lds<D>(qc, qt, at);
  mma_cols<D>(st.dv, dc, pf, lane);
  if constexpr (FINE) {
    p_rest(pd);
    p_frag(pf, pd);
    mma_cols<D>(st.dv, dc, pf, lane);
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) pr[r] *= (DROP ? dp[r] * dm[r] : dp[r]) - de[r];
  p_frag(df, pr);
  if constexpr (IN_LDS) col_frag_lds<D>(qc, qt, at);
  mma_cols<D>(st.dk, qc, df, lane);
  if constexpr (FINE) {
    p_rest(pr);
    p_frag(df, pr);
    mma_cols<D>(st.dk, qc, df, lane);
  }
}

// A wave's keys j, 32 of the ROWS that its workgroup has (the first is `first`): into its registers, or all of them into LDS, which every wave takes part in.  Hidden keys
// and keys past the end are zeros and carry a bias (returned) of -inf.
template <int ROWS, typename T, int D> __device__ __forceinline__ float load_keys(KeyState<T, D>& st, const Params& p, const Rows& rw, int hk, int first, int j, char* lds, const LaneAt<T, D>& at,
                                                                               int tid) {
  const int half = (tid & 63) >> 5, jr = j < rw.lk ? j : rw.lk - 1;
  const float km = p.keymask ? p.keymask[rw.k0 + jr] : 0.f;
  const bool on = j < rw.lk && km > HIDDEN;
  if constexpr (Dkv<T, D>::IN_LDS) {
    constexpr int NT = Dkv<T, D>::NT, ROWB = Geo<T, D>::ROWB, NCH = Geo<T, D>::NCH;
    char* v = lds + ROWS * ROWB;
    Dma<T, D, ROWS, NT> dma;
    dma.init((int)p.ldk * (int)sizeof(T), tid);
    dma.issue(lds, reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.k) + (rw.k0 + first) * p.ldk + (int64_t)hk * D), (int)p.ldk * (int)sizeof(T), rw.lk - first, tid);
    dma.init((int)p.ldv * (int)sizeof(T), tid);
    dma.issue(v, reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.v) + (rw.k0 + first) * p.ldv + (int64_t)hk * D), (int)p.ldv * (int)sizeof(T), rw.lk - first, tid);
    dma_arrive();
    st.kb = lds + (j - (tid & 31) - first) * ROWB;
    st.vb = st.kb + ROWS * ROWB;
    if (p.keymask) {
      __syncthreads();
      if (!on) {                           // (by every wave that has these keys)
        const u32x4 z = {0, 0, 0, 0};
        char* row = lds + (j - first) * ROWB + half * (ROWB / 2);
#pragma unroll
        for (int n = 0; n < NCH / 2; ++n) { *reinterpret_cast<u32x4*>(row + n * 16) = z; *reinterpret_cast<u32x4*>(row + ROWS * ROWB + n * 16) = z; }
      }
    }
    __syncthreads();
  } else {
    row_frag_global<T, D>(st.kf, reinterpret_cast<const T*>(p.k) + (rw.k0 + jr) * p.ldk + (int64_t)hk * D, half);
    row_frag_global<T, D>(st.vf, reinterpret_cast<const T*>(p.v) + (rw.k0 + jr) * p.ldv + (int64_t)hk * D, half);
    row_frag_arrive<T, D>(st.kf);
    row_frag_arrive<T, D>(st.vf);
    if (!on) { row_frag_zero<T, D>(st.kf); row_frag_zero<T, D>(st.vf); }
  }
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) { st.dk[i][r] = 0.f; st.dv[i][r] = 0.f; }
  return on ? km * LOG2E_ : -INFINITY;
}

// Query rows (q, dO and their statistics) on their way into LDS, ROWS at a time.
struct RowSource {
  const char *q, *d;
  const float *lse, *delta;
  int64_t sums;                            // from a row's maximum to the log of its sum
  int ldq, ldd, lq, r0;
  float st, sl, sdel;
  template <typename T, int D> __device__ __forceinline__ void init(const Params& p, const Rows& rw, int h0) {
    q = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.q) + rw.q0 * p.ldq + (int64_t)h0 * D);
    d = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.dout) + rw.q0 * p.lddo + (int64_t)h0 * D);
    lse = p.lse + (int64_t)h0 * p.Mq + rw.q0;
    delta = p.delta + (int64_t)h0 * p.Mq + rw.q0;
    ldq = (int)p.ldq * (int)sizeof(T); ldd = (int)p.lddo * (int)sizeof(T);
    sums = (int64_t)p.H * p.Mq;
    lq = rw.lq; r0 = 0; st = 0.f; sl = 0.f; sdel = 0.f;
  }
  template <int ROWS> __device__ __forceinline__ void get_stat(const Params& p, int g, int tid) {
    const int r = r0 + (tid & (ROWS - 1)) < lq ? r0 + (tid & (ROWS - 1)) : lq - 1;
    const int64_t at = (int64_t)g * p.Mq + r;
    st = lse[at];                          // (loaded whatever the row: a branch around a load is waited for at its end)
    sl = lse[at + sums];
    sdel = delta[at];
  }
  // what is taken off a score in the end, Deltas, what is taken off it first: without a mask the log-sum-exp at once; rows past the end: probability 0
  template <int ROWS> __device__ __forceinline__ void put_stat(float* stat, bool masked, int tid) const {
    const int r = r0 + (tid & (ROWS - 1));
    if (tid < ROWS) {
      stat[tid] = r < lq ? (masked ? sl : st + sl) : INFINITY;
      stat[ROWS + tid] = r < lq ? sdel : 0.f;
      if (masked) stat[2 * ROWS + tid] = r < lq ? st : 0.f;
    }
  }
};
template <typename T, int D, int ROWS, int NT> struct RowPipe {    // through LDS-DMA: issue() into a buffer that nobody reads, settle() before the barrier
  RowSource src;
  Dma<T, D, ROWS, NT> dq, dd;
  __device__ __forceinline__ RowPipe(const Params& p, const Rows& rw, int h0, int tid) {
    src.init<T, D>(p, rw, h0);
    dq.init(src.ldq, tid);
    dd.init(src.ldd, tid);
  }
  __device__ __forceinline__ void issue(const Params& p, char* qt, char* dt, int g, int first, int tid) {
    src.r0 = first;
    dq.issue(qt, src.q + (int64_t)first * src.ldq + g * (D * (int)sizeof(T)), src.ldq, src.lq - first, tid);
    dd.issue(dt, src.d + (int64_t)first * src.ldd + g * (D * (int)sizeof(T)), src.ldd, src.lq - first, tid);
    src.get_stat<ROWS>(p, g, tid);
  }
  __device__ __forceinline__ void settle(float* stat, bool masked, int tid) const {
    dma_arrive();
    src.put_stat<ROWS>(stat, masked, tid);
  }
};
// keys of a sequence's sink blocks: whole blocks of 32 that hold a sink with rows beyond its window (0: the sequence is too short for any)
__device__ __forceinline__ int sink_keys(const Params& p, const Rows& rw) {
  const int far = p.q_start + rw.lq - 1 - p.left, n = p.sinks < far ? p.sinks : far;
  return n > 0 ? (n + 31) & ~31 : 0;
}
// Where the partial sums of sink j of a sequence lie.  One behind the other (sequence b at b * s32) or, among packed sequences, of which most may be too short to have any, by
// the place of the sequence's rows, at floor(k0 * s32 / step).  A sequence of `len` rows has 32 ceil((len - 1 - left) / 32) of these keys, s32 at most; step (sink_steps) is such that
// floor(len * s32 / step) is never less, so no two sequences meet and the last one ends within floor(Mk * s32 / step).  (8192 tokens beside 999 reports of 30, 12 heads of
// 64, window 256: 58 MB with 4 sinks, 325 MB with 512; with s32 rows for every sequence it was 393 MB and 6.3 GB.)
__device__ __forceinline__ int64_t sink_row(const Params& p, const Rows& rw, int b, int hk, int j) {
  return hk * p.sink_rows + (p.sink_step ? rw.k0 * p.s32 / p.sink_step : (int64_t)b * p.s32) + j;
}
// len = left + 2 + 32 i rows are the fewest that have i + 1 blocks: step <= (s32 / 32) (left + 2 + 32 i) / (i + 1) for i = 0 ... s32 / 32 - 1, a monotone function of i
inline int64_t sink_steps(int s32, int left) {
  const int64_t last = (int64_t)s32 + left - 30, first = (int64_t)(s32 / 32) * (left + 2);
  return last < first ? last : first;
}
// where the partial sums of key j lie: split passes hold every key, unsplit ones the keys of the sink blocks
__device__ __forceinline__ int64_t part_row(const Params& p, const Rows& rw, int b, int hk, int j) {
  return p.nsplit > 1 ? (int64_t)hk * p.Mk + rw.k0 + j : sink_row(p, rw, b, hk, j);
}
__host__ __device__ inline int64_t part_rows(const Params& p) { return p.Hk * (p.nsplit > 1 ? p.Mk : p.sink_rows); }

template <typename T, int D, bool DROP, bool FINE>
__device__ __forceinline__ void window_pass(const Params& p, char* lds, int id, int split, int nunits, int nkt) {
  typedef Geo<T, D> G;
  typedef Dkv<T, D> X;
  constexpr int QT = X::QT, TILE = X::TILE;
  char* ring = lds + X::KEYS;
  float* stat = reinterpret_cast<float*>(ring + 4 * TILE);
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, c = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) & 3, par = __builtin_amdgcn_readfirstlane(tid >> 8);      // 32-key block; which of the waves that share it
  const Unit u = unit_of(p, id, nunits, nkt, 1);
  if (!u.real) return;
  const Rows rw = rows_of(p, u.b);
  const int k0 = u.tile * QB;
  if (k0 >= rw.lk) return;
  const int kend = k0 + QB - 1 < rw.lk - 1 ? k0 + QB - 1 : rw.lk - 1;
  // rows whose windows hold one of the keys
  int rlo = k0 - p.right - p.q_start, rhi = kend + p.left - p.q_start;
  rlo = rlo < 0 ? 0 : rlo;
  rhi = rhi < rw.lq - 1 ? rhi : rw.lq - 1;
  const int t0 = rlo / QT, nt = rhi >= rlo ? rhi / QT - t0 + 1 : 0, steps = nt * p.G;
  const int i0 = (int)((int64_t)steps * split / p.nsplit), i1 = (int)((int64_t)steps * (split + 1) / p.nsplit);

  const int jw = k0 + 32 * wave, j = jw + c;
  const LaneAt<T, D> at(lane);
  KeyState<T, D> st;
  const float kbias = load_keys<QB, T, D>(st, p, rw, u.hk, k0, j, lds, at, tid);
  const bool any = __builtin_amdgcn_ballot_w64(kbias > -INFINITY) != 0;      // wave-uniform
  RowPipe<T, D, QT, X::NT> rp(p, rw, u.hk * p.G, tid);
  if (i0 < i1) {
    rp.issue(p, ring, ring + TILE, i0 / nt, (t0 + i0 % nt) * QT, tid);
    rp.settle(stat, p.keymask != nullptr, tid);
  }
  __syncthreads();
  int g = i0 < i1 ? i0 / nt : 0, t = i0 < i1 ? i0 % nt : 0;        // the step's head of the group and tile
  for (int i = i0; i < i1; ++i) {
    const int buf = (i - i0) & 1, r0 = (t0 + t) * QT;
    const int64_t sh = (int64_t)u.b * p.H + u.hk * p.G + g;
    const bool more = i + 1 < i1;
    if (++t == nt) { t = 0; ++g; }
    char* next = ring + (buf ^ 1) * 2 * TILE;              // (its readers are behind the last barrier)
    if (more) rp.issue(p, next, next + TILE, g, (t0 + t) * QT, tid);
#pragma unroll
    for (int n = 0; n < QT / 32 / X::PAIR; ++n) {
      const int b = X::PAIR * n + par;
      const int lo = p.q_start + r0 + 32 * b, last = p.q_start + rw.lq - 1;
      const int see = any ? Sight(lo, lo + 31 < last ? lo + 31 : last, p.left, p.right, 0, rw.lk).of(jw) : 0;
      if (see) {
        const char* qt = ring + buf * 2 * TILE + 32 * b * G::ROWB;
        query_block<T, D, DROP, false, FINE>(st, qt, qt + TILE, stat + buf * 3 * QT + 32 * b, QT, at, p, r0 + 32 * b, j, kbias, see == 1, lane, sh);
      }
    }
    if (more) rp.settle(stat + (buf ^ 1) * 3 * QT, p.keymask != nullptr, tid);
    __syncthreads();
  }
  if constexpr (X::PAIR == 2) {            // the second wave of a pair hands its sums to the first, lane to lane: [block][register][lane], dK, then dV
    float* hand = reinterpret_cast<float*>(lds) + wave * (D / 2) * 64 + lane;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      f32x16(&a)[D / 32] = which ? st.dv : st.dk;
      if (which) __syncthreads();
      if (par) {
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
#pragma unroll
          for (int r = 0; r < 16; ++r) hand[(16 * x + r) * 64] = a[x][r];
      }
      __syncthreads();
      if (!par) {
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
#pragma unroll
          for (int r = 0; r < 16; ++r) a[x][r] += hand[(16 * x + r) * 64];
      }
    }
    if (par) return;
  }
  if (p.nsplit > 1 || jw < sink_keys(p, rw)) {
    if (j >= rw.lk) return;
    const int64_t N = part_rows(p), r = (int64_t)split * N + part_row(p, rw, u.b, u.hk, j);
    store_part<D>(p.part + r * D, st.dk, half);
    store_part<D>(p.part + ((int64_t)p.nsplit * N + r) * D, st.dv, half);
    return;
  }
  char* turn = ring + wave * 32 * G::ROWB;
  store_rows<T, D, false>(turn, st.dk, p.scale, reinterpret_cast<T*>(p.dk) + (rw.k0 + jw) * p.lddk + (int64_t)u.hk * D, p.lddk, rw.lk - jw, lane);
  store_rows<T, D, false>(turn, st.dv, 1.f, reinterpret_cast<T*>(p.dv) + (rw.k0 + jw) * p.lddv + (int64_t)u.hk * D, p.lddv, rw.lk - jw, lane);
}

template <typename T, int D, bool DROP, bool FINE>
__device__ __forceinline__ void sink_pass(const Params& p, char* lds, int id, int nblk) {
  typedef Geo<T, D> G;
  typedef Dkv<T, D> X;
  constexpr int TILE = 32 * G::ROWB;                               // lds: [k | v of 32 keys], a wave's own [Q | dO | lse, Delta] of 32 rows; reused to fold the waves
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, c = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int chunk = id % p.nchunk, blk = id / p.nchunk % nblk, hk = id / (p.nchunk * nblk) % p.Hk, b = id / (p.nchunk * nblk * p.Hk);
  const Rows rw = rows_of(p, b);
  const int jw = 32 * blk, j = jw + c;
  if (jw >= sink_keys(p, rw)) return;
  int rlo = jw + p.left + 1 - p.q_start;                           // first row that has a key of this block beyond its window
  rlo = rlo < 0 ? 0 : rlo;
  const int t0 = rlo / 32, nt = rw.lq > rlo ? (rw.lq - 1) / 32 - t0 + 1 : 0, steps = nt * p.G;
  const int i0 = (int)((int64_t)steps * chunk / p.nchunk), i1 = (int)((int64_t)steps * (chunk + 1) / p.nchunk);
  const LaneAt<T, D> at(lane);
  KeyState<T, D> st;
  const float kbias = load_keys<32, T, D>(st, p, rw, hk, jw, j, lds, at, tid);
  char* qtile = lds + X::SINK - (X::WAVES - wave) * X::OWN;
  char* dtile = qtile + TILE;
  float* stat = reinterpret_cast<float*>(dtile + TILE);
  RowPipe<T, D, 32, 64> rp(p, rw, hk * p.G, lane);
  for (int i = i0 + wave; i < i1; i += X::WAVES) {                 // (the other waves of the SIMD work while this one waits for its rows)
    const int g = i / nt, r0 = (t0 + i % nt) * 32;
    rp.issue(p, qtile, dtile, g, r0, lane);
    rp.settle(stat, p.keymask != nullptr, lane);
    wave_sync();
    query_block<T, D, DROP, true, FINE>(st, qtile, dtile, stat, 32, at, p, r0, j, kbias, true, lane, (int64_t)b * p.H + hk * p.G + g);
    wave_sync();
  }
  // fold the waves, dK then dV, in their order
  float* fa = reinterpret_cast<float*>(lds);                       // [WAVES][32][D + 4]
  const int64_t r = sink_row(p, rw, b, hk, jw), S = p.Hk * p.sink_rows;
  float* base = p.part + (int64_t)2 * p.nsplit * part_rows(p) * D;
  constexpr int TPR = X::NT / 32, PER = D / TPR;                   // threads of a row, columns of a thread
  const int fr = tid / TPR, fc = tid % TPR * PER;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x16& a = which ? st.dv[n] : st.dk[n];
        const f32x4 t = {a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
        *reinterpret_cast<f32x4*>(fa + (wave * 32 + c) * (D + 4) + 32 * n + 8 * q + 4 * half) = t;
      }
    __syncthreads();
    float* dst = base + (((int64_t)which * p.nchunk + chunk) * S + r + fr) * D + fc;
#pragma unroll
    for (int e = 0; e < PER; e += 4) {
      float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < X::WAVES; ++w)
#pragma unroll
        for (int x = 0; x < 4; ++x) t[x] += fa[(w * 32 + fr) * (D + 4) + fc + e + x];
      store4(dst + e, t);
    }
  }
}
// The first nsink workgroups take the sink pass, so that it runs beside the window pass instead of in front of it.
template <typename T, int D, bool DROP, bool FINE>
__global__ __launch_bounds__((Dkv<T, D>::NT), (D == 128 && sizeof(T) == 4 ? 1 : 2)) void dkv_kernel(Params p, int nunits, int nkt, int nsink) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int id = (int)blockIdx.x - nsink;
  if (id < 0) { sink_pass<T, D, DROP, FINE>(p, lds, blockIdx.x, p.s32 / 32); return; }
  const int per = (nunits + 7) / 8 * 8;
  window_pass<T, D, DROP, FINE>(p, lds, id % per, id / per, nunits, nkt);
}

// Keys whose sums came in parts, added in a fixed order: D / 4 threads across the columns of a key, the others across keys (a workgroup of the key range behind `deep`) or,
// where the parts are many, PG of them across the parts of one key (the sinks' chunks: one thread's chain of dependent additions over 43 took 40 us; PG threads for
// every key, most with two parts: 69 against 54 us for the whole backward pass of 2048 tokens, 12 heads of 64).
template <typename T, int D>
__global__ __launch_bounds__(256) void dkv_reduce_kernel(Params p, int keys, int deep) {
  constexpr int C = D / 4, PER = 256 / C, PG = PER < 16 ? PER : 16, DK = PER / PG;             // keys of a workgroup: PER, or DK
  __shared__ __attribute__((aligned(16))) float fold[2][PG][DK][D];
  const int hk = blockIdx.y, nd = (deep + DK - 1) / DK;
  const bool split = (int)blockIdx.x < nd;
  const int col = (threadIdx.x % C) * 4, sub = threadIdx.x / C;
  const int pg = split ? sub / DK : 0, step = split ? PG : 1;
  const int j = split ? blockIdx.x * DK + sub % DK : deep + (blockIdx.x - nd) * PER + sub;
  const int end = split ? deep : keys;
  for (int b = blockIdx.z; b < p.nseq; b += gridDim.z) {
    const Rows rw = rows_of(p, b);
    const int sk = sink_keys(p, rw);
    if (p.nsplit == 1 && !sk) continue;    // (its keys have been stored by the window's pass)
    const bool on = j < end && j < rw.lk && (p.nsplit > 1 || j < sk);
    const int64_t N = part_rows(p), S = p.Hk * p.sink_rows, r = part_row(p, rw, b, hk, j), rs = sink_row(p, rw, b, hk, j);
    const float* sink = p.part + 2 * p.nsplit * N * D;
    const int parts = p.nsplit + (j < sk ? p.nchunk : 0);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float o[4] = {0.f, 0.f, 0.f, 0.f};
      if (on)
        for (int s = pg; s < parts; s += step) {
          const float* src = s < p.nsplit ? p.part + (((int64_t)which * p.nsplit + s) * N + r) * D
                                          : sink + (((int64_t)which * p.nchunk + s - p.nsplit) * S + rs) * D;
          float a[4];
          load4(src + col, a);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] += a[e];
        }
      if (split) {
        store4(&fold[which][pg][sub % DK][col], o);
        __syncthreads();
        if (pg == 0) {
#pragma unroll
          for (int g = 1; g < PG; ++g) {
            float a[4];
            load4(&fold[which][g][sub][col], a);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += a[e];
          }
        }
      }
      if (on && pg == 0) {
        const float mul = which ? 1.f : p.scale;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= mul;
        store4((which ? reinterpret_cast<T*>(p.dv) + (rw.k0 + j) * p.lddv : reinterpret_cast<T*>(p.dk) + (rw.k0 + j) * p.lddk) + (int64_t)hk * D + col, o);
      }
    }
    if (split) __syncthreads();            // (the next sequence's parts go to the same place)
  }
}

struct BwdPlan { int nsplit, s32, nchunk; int64_t sink_rows, sink_step; };
inline BwdPlan bwd_plan(int nseq, int Lq, int Lk, int64_t Mk, int H, int Hk, int D, int left, int right, int sinks, int q_start, int ntiles, int dtype) {
  BwdPlan b{1, 0, 0, 0, 0};
  const int G = H / Hk;
  const int64_t units = ntiles ? (int64_t)ntiles * Hk : (int64_t)nseq * Hk * cdiv(Lk, QB);
  const int64_t span = (int64_t)QB + left + right < Lq ? (int64_t)QB + left + right : Lq;
  const int64_t steps = cdiv(span, dtype == DT_F32 ? 32 : 64) * G;         // of a workgroup that is not split
  // Too few key tiles for the workgroups that are resident at once (one per CU for heads of 128, two otherwise): split the rows and heads that they meet, but not below four
  // steps, for the parts are written and read again.  dQ, dK and dV of 1000 tokens, 8 heads on 2, no window: 48 us, unsplit 145; causal 2048, 4 heads of 128 on 1: 99 and 307;
  // 1024 tokens, 12 heads, window 128: 34, with parts of two steps 40.  Two workgroups per CU for heads of 128: 106 instead of 91 us (4096 tokens, 4 heads, window 1023).
  int64_t s = (D == 128 ? 256 : 512) / units;
  if (s > steps / 4) s = steps / 4;
  if (s > 1) b.nsplit = (int)s;
  const int64_t far = (int64_t)q_start + Lq - 1 - left;            // sinks 0 ... far - 1 have rows beyond their window
  if (sinks > 0 && far > 0) {
    const int64_t n = sinks < far ? sinks : far;
    b.s32 = (int)(cdiv(n, 32) * 32);
    b.sink_rows = (int64_t)nseq * b.s32;
    const int64_t step = sink_steps(b.s32, left), packed = Mk * b.s32 / step;
    if (ntiles && packed < b.sink_rows) { b.sink_rows = packed; b.sink_step = step; }
    const int64_t blocks = Hk * cdiv(b.sink_rows, 32), tiles = cdiv(far, 32) * G;
    int64_t ch = cdiv(512, blocks);
    if (ch > tiles / 8) ch = tiles / 8;    // two tiles per wave at least; unsplit, the backward pass of 32768 tokens, 12 heads, takes 549 instead of 490 us
    b.nchunk = (int)(ch < 1 ? 1 : ch);
  }
  return b;
}
inline int64_t bwd_floats(const BwdPlan& b, int64_t Mk, int Hk, int D) {
  const int64_t win = b.nsplit > 1 ? b.nsplit * Mk : b.sink_rows;
  return 2 * (win + b.nchunk * b.sink_rows) * Hk * D;
}

template <typename T, int D, bool DROP, bool FINE> int launch_bwd(Params& p, hipStream_t s) {
  typedef Geo<T, D> G;
  constexpr int lds_q = 4 * G::KT * G::ROWB + 2 * G::KT * 4, lds_kv = Dkv<T, D>::LDS;
  const int nqt = (int)cdiv(p.Lq, QB), nkt = (int)cdiv(p.Lk, QB);
  const int64_t nq = p.offsets ? (int64_t)p.ntiles * p.H : (int64_t)p.nseq * p.H * nqt, nk = p.offsets ? (int64_t)p.ntiles * p.Hk : (int64_t)p.nseq * p.Hk * nkt;
  const int64_t nsink = (int64_t)(p.s32 / 32) * p.Hk * p.nseq * p.nchunk, grid = nsink + 8 * cdiv(nk, 8) * p.nsplit;
  const int keys = p.nsplit > 1 ? p.Lk : p.s32;
  constexpr int PER = 256 / (D / 4), DK = PER < 16 ? 1 : PER / 16;           // (as in dkv_reduce_kernel)
  const int deep = p.nsplit > 8 ? keys : (p.nsplit + p.nchunk > 8 ? (p.s32 < keys ? p.s32 : keys) : 0);
  const int64_t nred = cdiv(deep, DK) + cdiv(keys - deep, PER);
  int rc;                                  // everything that can be refused, before the first launch writes
  if ((rc = check_grid(8 * cdiv(nq, 8), 256)) || (rc = check_grid(grid, Dkv<T, D>::NT)) || (rc = check_grid(nred, 256)) ||
      (rc = raise_lds<dq_kernel<T, D, DROP, FINE>>(lds_q)) || (rc = raise_lds<dkv_kernel<T, D, DROP, FINE>>(lds_kv))) return rc;
  if (nq) hipLaunchKernelGGL((dq_kernel<T, D, DROP, FINE>), dim3((unsigned)(8 * cdiv(nq, 8))), dim3(256), lds_q, s, p, (int)nq, nqt);
  if ((rc = ctclip_check_launch("win_attn_bwd dq"))) return rc;
  if (nk) hipLaunchKernelGGL((dkv_kernel<T, D, DROP, FINE>), dim3((unsigned)grid), dim3(Dkv<T, D>::NT), lds_kv, s, p, (int)nk, nkt, (int)nsink);
  if ((rc = ctclip_check_launch("win_attn_bwd dkv"))) return rc;
  if (!keys) return CTCLIP_OK;
  const unsigned nz = p.nseq < 32768 ? p.nseq : 32768;
  hipLaunchKernelGGL((dkv_reduce_kernel<T, D>), dim3((unsigned)nred, p.Hk, nz), dim3(256), 0, s, p, keys, deep);
  return ctclip_check_launch("win_attn_bwd reduce");
}
template <typename T, int D> int launch_bwd_d(Params& p, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (fine_pass(p, DT_BF16, true)) return p.drop_p > 0.f ? launch_bwd<T, D, true, true>(p, s) : launch_bwd<T, D, false, true>(p, s);
  }
  return p.drop_p > 0.f ? launch_bwd<T, D, true, false>(p, s) : launch_bwd<T, D, false, false>(p, s);
}
template <typename T> int launch_bwd_t(Params& p, int D, hipStream_t s) {
  return D == 32 ? launch_bwd_d<T, 32>(p, s) : (D == 64 ? launch_bwd_d<T, 64>(p, s) : launch_bwd_d<T, 128>(p, s));
}
}  // namespace win

// bytes of workspace of ctclip_win_attn_bwd (partial sums of the sinks' gradients and of split key tiles; 0: none).  ntiles: packed sequences, else 0
extern "C" int64_t ctclip_win_attn_bwd_workspace(int nseq, int Lq, int Lk, int64_t Mk, int H, int Hk, int D, int left, int right, int sinks, int q_start, int ntiles) {
  if (nseq < 1 || Lq < 1 || Lk < 1 || H < 1 || Hk < 1 || H % Hk) return 0;
  const int l = left < 0 || left > Lk ? Lk : left, r = right < 0 || right > Lk ? Lk : right, s = sinks < Lk ? sinks : Lk;
  int64_t need = 0;                        // (of either type: the larger)
  for (int dtype : {DT_F32, DT_BF16}) {
    const int64_t n = win::bwd_floats(win::bwd_plan(nseq, Lq, Lk, Mk, H, Hk, D, l, r, s, q_start, ntiles, dtype), Mk, Hk, D) * 4;
    need = n > need ? n : need;
  }
  return need;
}

// gradients of ctclip_win_attn_fwd: o, lse as it wrote them; delta: [H][Mq] f32 scratch; dq, dk, dv in the inputs' type, every row of a sequence written
extern "C" int ctclip_win_attn_bwd(const void* q, const void* k, const void* v, const float* keymask, const int32_t* offsets, const int32_t* tiles, int ntiles, const void* o,
                                   const void* o_lo, const void* dout, const float* lse, float* delta, void* dq, void* dk, void* dv, int nseq, int Lq, int Lk, int64_t Mq, int64_t Mk, int H,
                                   int Hk, int D, int left, int right, int sinks, int q_start, int64_t ldq, int64_t ldk, int64_t ldv, int64_t ldo, int64_t lddo,
                                   int64_t lddq, int64_t lddk, int64_t lddv, float scale, float dropout_p, uint64_t dropout_seed, int dtype, void* workspace,
                                   int64_t workspace_bytes, hipStream_t stream) {
  using namespace win;
  int rc = check_shape(nseq, Lq, Lk, Mq, Mk, H, Hk, D, left, right, sinks, q_start, offsets != nullptr, dtype);
  if (rc) return rc;
  if (!(scale > 0.f) || !(scale < 1e30f) || !(dropout_p >= 0.f) || !(dropout_p < 1.f)) { ctclip_set_error("win_attn_bwd: scale > 0, 0 <= dropout < 1"); return CTCLIP_EBADARG; }
  if (nseq == 0 || Lk == 0 || Lq == 0 || (offsets && ntiles == 0)) return CTCLIP_OK;
  if (offsets && (!tiles || ntiles < 0)) { ctclip_set_error("win_attn_bwd: packed sequences need their tiles"); return CTCLIP_EBADARG; }
  if (!lse || !delta) { ctclip_set_error("win_attn_bwd: needs lse and delta"); return CTCLIP_EBADARG; }
  if ((rc = check_rows(q, ldq, Lq, H, D, dtype, false, "win_attn_bwd: q rows 16-byte aligned")) || (rc = check_rows(k, ldk, Lk, Hk, D, dtype, false, "win_attn_bwd: k rows 16-byte aligned")) ||
      (rc = check_rows(v, ldv, Lk, Hk, D, dtype, false, "win_attn_bwd: v rows 16-byte aligned")) || (rc = check_rows(o, ldo, Lq, H, D, dtype, false, "win_attn_bwd: o rows 16-byte aligned")) ||
      (o_lo && (rc = check_rows(o_lo, ldo, Lq, H, D, dtype, false, "win_attn_bwd: o_lo rows 16-byte aligned"))) ||
      (rc = check_rows(dout, lddo, Lq, H, D, dtype, false, "win_attn_bwd: dout rows 16-byte aligned")) || (rc = check_rows(dq, lddq, Lq, H, D, dtype, true, "win_attn_bwd: dq rows 16-byte aligned, apart")) ||
      (rc = check_rows(dk, lddk, Lk, Hk, D, dtype, true, "win_attn_bwd: dk rows 16-byte aligned, apart")) || (rc = check_rows(dv, lddv, Lk, Hk, D, dtype, true, "win_attn_bwd: dv rows 16-byte aligned, apart"))) return rc;
  Params p{};
  fill(p, nseq, Lq, Lk, Mq, Mk, H, Hk, left, right, sinks, q_start, scale, dropout_p, dropout_seed, offsets, tiles, ntiles, keymask);
  p.q = q; p.k = k; p.v = v; p.o = o; p.out_lo = dtype == DT_BF16 ? const_cast<void*>(o_lo) : nullptr; p.dout = dout; p.lse = const_cast<float*>(lse); p.delta = delta; p.dq = dq; p.dk = dk; p.dv = dv;
  p.ldq = ldq; p.ldk = ldk; p.ldv = ldv; p.ldo = ldo; p.lddo = lddo; p.lddq = lddq; p.lddk = lddk; p.lddv = lddv;
  const BwdPlan b = bwd_plan(nseq, Lq, Lk, Mk, H, Hk, D, p.left, p.right, p.sinks, q_start, offsets ? ntiles : 0, dtype);
  p.nsplit = b.nsplit; p.s32 = b.s32; p.nchunk = b.nchunk; p.sink_rows = b.sink_rows; p.sink_step = b.sink_step;
  const int64_t need = bwd_floats(b, Mk, Hk, D) * 4;
  if (need) {
    if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16) { ctclip_set_error("win_attn_bwd: workspace"); return CTCLIP_EWORKSPACE; }
    p.part = (float*)workspace;
  }
  return dtype == DT_F32 ? launch_bwd_t<float>(p, D, stream) : launch_bwd_t<bf16_t>(p, D, stream);
}
