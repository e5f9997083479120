// Attention in a sliding window with sinks on gfx950, forward (definitions, operand layouts and LDS image: win_attn.h).
//
//   fwd_kernel   a workgroup owns 128 query rows of one (sequence, head), a wave 32 of them; the key tiles that the rows' windows and the sinks cover
//                pass through a double-buffered LDS ring (one barrier per tile, the next tile's loads in flight under the current one's products).
//   rows_kernel  few query rows against many keys (one token, the [CLS] row): the rows of all heads that share a k|v head are ONE 32-row block, the four
//                waves take different key tiles and the axis is split over workgroups until the chip is full.  Bound by reading k and v once.
//   join_kernel  folds the split passes of either.
// One pass over the keys with the running maximum and sum of the softmax in f32, log2 domain.  P is rounded to the operand type (bf16: half a step is 2^-8 of the value,
// one rounding per probability) because the matrix cores read it; sums are taken of the unrounded values.  FINE adds what that rounding left over (win_attn.h, fine_pass).
//
// Bounds, MI355X.  One token of 4 sequences over 32768 keys, 32 heads of 128 on 8: 113 + 4 us (rows + join), 537 MB at 4.7 TB/s; a large copy runs at 5.1.  4 x 8192 tokens,
// 12 heads of 64, window 256 + 256: 95 us, 0.54 PFLOP/s of 1.2 that a large product reaches: matrix instructions 0.26 of the time, vector instructions (exponentials, masks,
// maxima, conversions) 0.58, LDS 0.16, which add up: a wave's step is a chain through all three, and four waves per SIMD overlap little of it.
#include "win_attn.h"

namespace win {

// Workspace of split passes, `rows` = splits x heads x query rows: maxima and sums of the rows, then (16-byte aligned) their accumulators.
__host__ __device__ inline int64_t part_acc(int64_t rows) { return (2 * rows + 3) & ~(int64_t)3; }
inline int64_t part_bytes(int64_t rows, int D) { return (part_acc(rows) + rows * D) * 4; }

template <int D> struct SoftRow {          // the running softmax of a lane's query
  f32x16 acc[D / 32];
  float m, l;
  __device__ __forceinline__ void clear() {
    m = -INFINITY; l = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  }
};

// The running maximum is raised only when some row's scores outgrow it by more than 2^LAZY: accumulators and sums then hold probabilities up to 2^8 times the
// final ones, which f32 (and the operand type: bf16 has the range of f32) does not notice, and the rescale of the accumulators -- with 32 rows to a wave some row's
// maximum moves in nearly every block -- becomes rare.  LAZY = 0: 107 instead of 98 us for 4 x 8192 tokens of 12 heads of 64, 407 instead of 375 for 2 x 8191 of 32 of 128.
constexpr float LAZY = 8.f;

// A 32-key block: scores -> running softmax -> acc.  vt = the block's v rows in LDS; bias = its additive mask (or null); pos = the lane's position
template <typename T, int D, bool DROP, bool PAIRED, bool FINE>
__device__ __forceinline__ void key_block(SoftRow<D>& st, f32x16 s, const char* vt, const float* bias, const LaneAt<T, D>& at, const Params& p, int j0, int pos, int lk,
                                          bool partial, int lane, int64_t sh, int qi) {
  const int half = lane >> 5;
  float sc = p.scale2;                                     // (scale > 0: the maximum may be taken of the unscaled scores; one rounding in the fma below)
  if (bias) {
    sc = 1.f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(bias + 8 * g + 4 * half);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[4 * g + e] = fmaf(s[4 * g + e], p.scale2, a[e]);
    }
  }
  if (partial) {
    const int o = j0 + 4 * half;
    const int hi = (pos + p.right < lk - 1 ? pos + p.right : lk - 1) - o, lo = pos - p.left - o, sk = p.sinks - o;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int j = 8 * (r >> 2) + (r & 3);
      s[r] = (j <= hi && (j >= lo || j < sk)) ? s[r] : -INFINITY;
    }
  }
  float mx = s[0];
#pragma unroll
  for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
  mx = half_max(mx) * sc;
  if (__builtin_amdgcn_ballot_w64(mx > st.m + LAZY) != 0) {        // wave-uniform
    const float mn = fmaxf(st.m, mx);
    const float alpha = __builtin_amdgcn_exp2f(st.m - (mn == -INFINITY ? 0.f : mn));
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) st.acc[i][r] *= alpha;
    st.l *= alpha;
    st.m = mn;
  }
  const float ms = st.m == -INFINITY ? 0.f : st.m;         // nothing seen so far: every exp2 below is exp2(-inf) = 0
  float pr[16], ps[4];                                     // (four sums: one would be a chain of 16 dependent additions)
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    pr[r] = __builtin_amdgcn_exp2f(fmaf(s[r], sc, -ms));
    ps[r & 3] = r < 4 ? pr[r] : ps[r & 3] + pr[r];
  }
  st.l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
  if (DROP) {                                              // on the normalised probabilities: the sum above stays undropped
    float dm[16];
    drop_of_query<PAIRED>(dm, p, sh, qi, j0, half);
#pragma unroll
    for (int r = 0; r < 16; ++r) pr[r] *= dm[r];
  }
  PFrag<T> pf;
  p_frag(pf, pr);
  ColFrag<T, D> vf;
  col_frag_lds<D>(vf, vt, at);
  mma_cols<D>(st.acc, vf, pf, lane);
  if constexpr (FINE) {
    p_rest(pr);
    p_frag(pf, pr);
    mma_cols<D>(st.acc, vf, pf, lane);
  }
}
template <typename T, int D> __device__ __forceinline__ f32x16 scores(const RowFrag<T, D>& kf, const RowFrag<T, D>& qf) {
  f32x16 s;
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = 0.f;
  return mma_rows<D>(kf, qf, s);
}

// Four waves per SIMD (bf16, heads up to 64): 98 and 165 us for 4 x 8192 and 1 x 32768 tokens of 12 heads of 64, with two 103 and 172.  128 registers hold such a wave, but for the
// dropout form of heads of 64, which keeps 6 in scratch and is the faster for it all the same: 4 x 8192 tokens 177 us, with two waves and none in scratch 187.
template <typename T, int D, bool DROP, bool FINE>
__global__ __launch_bounds__(256, (sizeof(T) == 2 && D <= 64 && !FINE ? 4 : 2)) void fwd_kernel(Params p, int nunits, int nqt) {
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
  const int lo = p.q_start + q0, hi = lo + nq - 1;                 // positions of the workgroup's rows
  const TileList tl = tile_list<KT>(lo, hi, p.left, p.right, p.sinks, rw.lk);
  const int i0 = (int)((int64_t)tl.n * blockIdx.y / p.nsplit), i1 = (int)((int64_t)tl.n * (blockIdx.y + 1) / p.nsplit);

  int row = q0 + 32 * wave + c;
  const bool real = row < rw.lq;
  row = real ? row : rw.lq - 1;
  const int wlo = lo + 32 * wave, whi = wlo + 31 < hi ? wlo + 31 : hi;      // the wave's positions (whi < wlo: it has none)
  const Sight sight(wlo, whi, p.left, p.right, p.sinks, rw.lk);
  const int pos = p.q_start + row;
  RowFrag<T, D> qf;
  row_frag_global<T, D>(qf, reinterpret_cast<const T*>(p.q) + (rw.q0 + row) * p.ldq + (int64_t)h * D, half);
  const LaneAt<T, D> at(lane);
  KeyPipe<T, D, KT, 256> kp(p, rw.k0, u.hk, rw.lk, lo - p.left, hi + p.right, tid);
  SoftRow<D> st;
  st.clear();
  const int64_t sh = (int64_t)u.b * p.H + h;
  int state = 0;
  if (i0 < i1) {
    kp.issue(lds, lds + TILE, tile_at(tl, i0) * KT, tid);
    state = kp.settle(lds, lds + TILE, kb, tid);
  }
  row_frag_arrive<T, D>(qf);                               // (behind the first tile's loads)
  __syncthreads();
  for (int it = i0; it < i1; ++it) {
    const int buf = (it - i0) & 1, j0 = tile_at(tl, it) * KT;
    const bool more = it + 1 < i1;
    char* next = lds + (buf ^ 1) * 2 * TILE;               // (its readers are behind the last barrier)
    if (more) kp.issue(next, next + TILE, tile_at(tl, it + 1) * KT, tid);
    if (state != 2) {
      const char *kt = lds + buf * 2 * TILE, *vt = kt + TILE;
      const float* bias = state ? kb + buf * KT : nullptr;
#pragma unroll
      for (int b = 0; b < KT / 32; ++b) {
        const int a = sight.of(j0 + 32 * b), o = 32 * b * G::ROWB;
        if (!a) continue;
        RowFrag<T, D> kf;
        row_frag_lds<T, D>(kf, kt + o, at);
        key_block<T, D, DROP, true, FINE>(st, scores<T, D>(kf, qf), vt + o, bias ? bias + 32 * b : nullptr, at, p, j0 + 32 * b, pos, rw.lk, a != 2, lane, sh, row);
      }
    }
    if (more) state = kp.settle(next, next + TILE, kb + (buf ^ 1) * KT, tid);
    __syncthreads();
  }
  const float l = half_sum(st.l);
  if (p.nsplit > 1) {
    if (!real) return;
    const int64_t r = ((int64_t)blockIdx.y * p.H + h) * p.Mq + rw.q0 + row;
    const int64_t rows = (int64_t)p.nsplit * p.H * p.Mq;
    store_part<D>(p.part + part_acc(rows) + r * D, st.acc, half);
    if (half == 0) { p.part[r] = st.m; p.part[rows + r] = l; }
    return;
  }
  // (everybody is behind the last barrier: the tiles' space is free)
  const int wr = q0 + 32 * wave;
  const int64_t o = (rw.q0 + wr) * p.ldo + (int64_t)h * D;
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  store_rows<T, D, false>(lds + wave * 32 * G::ROWB, st.acc, inv, reinterpret_cast<T*>(p.out) + o, p.ldo, rw.lq - wr, lane);
  if (sizeof(T) == 2 && p.out_lo) store_rows<T, D, true>(lds + wave * 32 * G::ROWB, st.acc, inv, reinterpret_cast<T*>(p.out_lo) + o, p.ldo, rw.lq - wr, lane);
  if (!real) return;
  if (half == 0) store_lse(p, (int64_t)h * p.Mq + rw.q0 + row, st.m, l);
}

// ---- few query rows: R = Lq * G <= 32 rows (row c = head g = c / Lq of the group, query c % Lq).  A wave's keys meet no other wave's rows, so k goes straight from
// memory into the first product's operand registers (the next block's while this one is worked on), only v through LDS, two blocks per wave.
template <typename T, int D, bool DROP, bool FINE>
__global__ __launch_bounds__(256, (sizeof(T) == 4 && D == 128 ? 1 : 2)) void rows_kernel(Params p, int nunits) {
  typedef Geo<T, D> G;
  constexpr int TILE = 32 * G::ROWB;
  extern __shared__ __attribute__((aligned(16))) char lds[];       // four waves x ([2][V] of 32 keys, [2][32] additive mask); reused to fold the waves
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, c = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Unit u = unit_of(p, blockIdx.x, nunits, 1, 1);
  if (!u.real) return;
  const Rows rw = rows_of(p, u.b);
  const int R = rw.lq * p.G;
  const int lo = p.q_start, hi = p.q_start + rw.lq - 1;
  const TileList tl = tile_list<32>(lo, hi, p.left, p.right, p.sinks, rw.lk);
  const int i0 = (int)((int64_t)tl.n * blockIdx.y / p.nsplit), i1 = (int)((int64_t)tl.n * (blockIdx.y + 1) / p.nsplit);
  const int rc = c < R ? c : R - 1;
  const int g = rc / rw.lq, row = rc - g * rw.lq, h = u.hk * p.G + g, pos = p.q_start + row;
  RowFrag<T, D> qf;
  row_frag_global<T, D>(qf, reinterpret_cast<const T*>(p.q) + (rw.q0 + row) * p.ldq + (int64_t)h * D, half);
  char* vtile = lds + wave * (2 * TILE + 256);
  float* kb = reinterpret_cast<float*>(vtile + 2 * TILE);
  const Sight sight(lo, hi, p.left, p.right, p.sinks, rw.lk);
  const LaneAt<T, D> at(lane);
  KeySource src;
  src.init<T, D>(p, rw.k0, u.hk, rw.lk, lo - p.left, hi + p.right);
  Dma<T, D, 32, 64> dv;
  dv.init(src.ldv, lane);
  RowFrag<T, D> kf;
  float km = 0.f;
  auto fetch = [&](int j0, int buf) {                              // (rows past the end: k of the last row, v zeros)
    const int r = c < src.lk - 1 - j0 ? c : src.lk - 1 - j0;
    if (src.mask) km = src.mask[j0 + r];
    row_frag_global<T, D>(kf, reinterpret_cast<const T*>(src.k + (int64_t)(j0 + r) * src.ldk), half);
    dv.issue(vtile + buf * TILE, src.v + (int64_t)j0 * src.ldv, src.ldv, src.jhi + 1 - j0, lane);
  };
  SoftRow<D> st;
  st.clear();
  const int64_t sh = (int64_t)u.b * p.H + h;
  int it = i0 + wave, buf = 0;
  if (it < i1) fetch(tile_at(tl, it) * 32, 0);
  row_frag_arrive<T, D>(qf);
  for (; it < i1; it += 4, buf ^= 1) {                             // (no barrier: a wave's tiles are its own, and a refill waits for its reads)
    const int j0 = tile_at(tl, it) * 32;
    dma_arrive();
    int state = 0;
    if (src.mask || j0 < src.jlo || j0 + 31 > src.jhi) {
      uint64_t keep;
      state = src.look<32>(keep, km, kb + buf * 32, j0, lane);
      if (~keep) {
        dv.erase(vtile + buf * TILE, keep, lane);
        row_frag_arrive<T, D>(kf);
        if (!((keep >> c) & 1)) row_frag_zero<T, D>(kf);
      }
    }
    wave_sync();
    const f32x16 s = scores<T, D>(kf, qf);
    if (it + 4 < i1) fetch(tile_at(tl, it + 4) * 32, buf ^ 1);
    const int a = sight.of(j0);
    if (a && state != 2) key_block<T, D, DROP, false, FINE>(st, s, vtile + buf * TILE, state ? kb + buf * 32 : nullptr, at, p, j0, pos, rw.lk, a == 1, lane, sh, row);
    wave_sync();
  }
  // fold the four waves: row maxima first, then sums and accumulators under the common maximum
  float* fm = reinterpret_cast<float*>(lds);                       // [4][32] maxima, [4][32] sums, [4][32][D + 4] accumulators (+ 4: two lanes' rows a bank apart)
  float* fl = fm + 128;
  float* fa = fl + 128;
  const float l = half_sum(st.l);
  __syncthreads();
  if (half == 0) { fm[wave * 32 + c] = st.m; fl[wave * 32 + c] = l; }
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 a = {st.acc[i][4 * q], st.acc[i][4 * q + 1], st.acc[i][4 * q + 2], st.acc[i][4 * q + 3]};
      *reinterpret_cast<f32x4*>(fa + (wave * 32 + c) * (D + 4) + 32 * i + 8 * q + 4 * half) = a;
    }
  __syncthreads();
  constexpr int PER = D / 8;                                       // eight threads per row, D / 8 columns each
  const int fr = tid >> 3, fc = (tid & 7) * PER;
  if (fr >= R) return;
  float m = fm[fr];
#pragma unroll
  for (int w = 1; w < 4; ++w) m = fmaxf(m, fm[w * 32 + fr]);
  const float ms = m == -INFINITY ? 0.f : m;
  float lsum = 0.f, o[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) o[e] = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = __builtin_amdgcn_exp2f(fm[w * 32 + fr] - ms);
    lsum = fmaf(fl[w * 32 + fr], f, lsum);
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] = fmaf(fa[(w * 32 + fr) * (D + 4) + fc + e], f, o[e]);
  }
  const int og = fr / rw.lq, orow = fr - og * rw.lq, oh = u.hk * p.G + og;
  if (p.nsplit > 1) {
    const int64_t r = ((int64_t)blockIdx.y * p.H + oh) * p.Mq + rw.q0 + orow, rows = (int64_t)p.nsplit * p.H * p.Mq;
#pragma unroll
    for (int e = 0; e < PER; e += 4) { const float t[4] = {o[e], o[e + 1], o[e + 2], o[e + 3]}; store4(p.part + part_acc(rows) + r * D + fc + e, t); }
    if ((tid & 7) == 0) { p.part[r] = m; p.part[rows + r] = lsum; }
    return;
  }
  const float mul = lsum > 0.f ? 1.f / lsum : (lsum == 0.f ? 0.f : lsum);
#pragma unroll
  for (int e = 0; e < PER; e += 4) { float t[4] = {o[e] * mul, o[e + 1] * mul, o[e + 2] * mul, o[e + 3] * mul}; store_out<T>(p, rw.q0 + orow, (int64_t)oh * D + fc + e, t); }
  if ((tid & 7) == 0) store_lse(p, (int64_t)oh * p.Mq + rw.q0 + orow, m, lsum);
}

// out = sum_s exp2(m_s - M) acc_s / sum_s exp2(m_s - M) l_s over the split passes, in a fixed order.  D / 4 threads across the columns of a (head, row); the others across
// the splits (SG = 256 / (D / 4): one thread's chain over 16 splits took 11 us), or across rows (SG = 1) where there are many rows (f32, 3 x 577
// tokens of 8 heads, split in two: 20 us, with a workgroup for each row and head 45, unsplit 27).
template <typename T, int D, int SG>
__global__ __launch_bounds__(256) void join_kernel(Params p) {
  constexpr int C = D / 4, PER = 256 / C / SG;
  __shared__ __attribute__((aligned(16))) float fo[SG][D], fl[SG];
  const int64_t n = (int64_t)p.H * p.Mq, rows = (int64_t)p.nsplit * n, i = (int64_t)blockIdx.x * PER + (SG == 1 ? threadIdx.x / C : 0);
  if (i >= n) return;                      // (SG > 1: the whole workgroup or nobody)
  const int col = (threadIdx.x % C) * 4, sg = SG == 1 ? 0 : threadIdx.x / C;
  float m = -INFINITY;
  if constexpr (SG > 1) {
    for (int s = threadIdx.x & 63; s < p.nsplit; s += 64) m = fmaxf(m, p.part[s * n + i]);
    m = wave_max(m);
  } else {
    for (int s = 0; s < p.nsplit; ++s) m = fmaxf(m, p.part[s * n + i]);
  }
  const float ms = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = sg; s < p.nsplit; s += SG) {
    const float f = __builtin_amdgcn_exp2f(p.part[s * n + i] - ms);
    l = fmaf(p.part[rows + s * n + i], f, l);
    float a[4];
    load4(p.part + part_acc(rows) + (s * n + i) * D + col, a);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(a[e], f, o[e]);
  }
  if constexpr (SG > 1) {
    store4(&fo[sg][col], o);
    if (col == 0) fl[sg] = l;
    __syncthreads();
    if (sg) return;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = 0.f;
#pragma unroll
    for (int g = 0; g < SG; ++g) {
      float a[4];
      load4(&fo[g][col], a);
      l += fl[g];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += a[e];
    }
  }
  const int64_t h = i / p.Mq, row = i - h * p.Mq;
  const float mul = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] *= mul;
  store_out<T>(p, row, h * D + col, o);
  if (col == 0) store_lse(p, i, m, l);
}

// ---- host side
struct Plan { bool rows; int nsplit; };
// Which kernel, and over how many workgroups a key axis is split.
inline Plan plan(int nseq, int Lq, int Lk, int H, int Hk, int left, int right, int sinks, int q_start, bool packed, int dtype) {
  Plan pl{false, 1};
  const int G = H / Hk;
  if (packed) return pl;
  // rows_kernel where the rows of a group fit its 32: one token of 4 sequences of 32768 keys, 32 heads of 128 on 8, takes 115 us (fwd_kernel, where the heads that share k and v
  // are rows of different workgroups: 197), the [CLS] rows of 8 x 512 5.9 (6.9).  Split for two workgroups per CU, eight blocks (two per wave) each at least: unsplit 468 us.
  if ((int64_t)Lq * G <= 32) {
    pl.rows = true;
    const TileList tl = tile_list<32>(q_start, q_start + Lq - 1, left, right, sinks, Lk);
    const int64_t units = (int64_t)nseq * Hk;
    int64_t s = cdiv(512, units);
    if (s > tl.n / 8) s = tl.n / 8;
    pl.nsplit = (int)(s < 1 ? 1 : s);
    return pl;
  }
  const int64_t units = (int64_t)nseq * H * cdiv(Lq, QB);
  // fewer tiles than CUs: split, but not below four steps.  1 x 4096, 2 heads of 64, no window: 29 us, unsplit 70; 200 rows against 8192 keys, 12 heads: 27 and 140; 512 tokens
  // of 12 heads, window 128: 13.5, with parts of two steps 15.3
  if (units < 256) {
    const int last = (int)((Lq - 1) / QB) * QB, lo = q_start + last, hi = q_start + Lq - 1;
    const int tiles = dtype == DT_F32 ? tile_list<32>(lo, hi, left, right, sinks, Lk).n : tile_list<64>(lo, hi, left, right, sinks, Lk).n;
    int64_t s = 256 / units;
    if (s > tiles / 4) s = tiles / 4;
    if (s > 1) pl.nsplit = (int)s;
  }
  return pl;
}

template <typename T, int D, bool DROP, bool FINE> int launch_fwd(Params& p, const Plan& pl, hipStream_t s) {
  typedef Geo<T, D> G;
  if (pl.rows) {
    const int64_t nu = (int64_t)p.nseq * p.Hk;
    int lds = 4 * (2 * 32 * G::ROWB + 256);
    const int fold = 1024 + 4 * 32 * (D + 4) * 4;
    if (fold > lds) lds = fold;
    int rc = check_grid(8 * cdiv(nu, 8), 256);
    if (!rc) rc = raise_lds<rows_kernel<T, D, DROP, FINE>>(lds);
    if (rc) return rc;
    hipLaunchKernelGGL((rows_kernel<T, D, DROP, FINE>), dim3((unsigned)(8 * cdiv(nu, 8)), p.nsplit), dim3(256), lds, s, p, (int)nu);
  } else {
    const int nqt = (int)cdiv(p.Lq, QB);
    const int64_t nu = p.offsets ? (int64_t)p.ntiles * p.H : (int64_t)p.nseq * p.H * nqt;
    const int lds = 4 * G::KT * G::ROWB + 2 * G::KT * 4;
    int rc = check_grid(8 * cdiv(nu, 8), 256);
    if (!rc) rc = raise_lds<fwd_kernel<T, D, DROP, FINE>>(lds);
    if (rc) return rc;
    hipLaunchKernelGGL((fwd_kernel<T, D, DROP, FINE>), dim3((unsigned)(8 * cdiv(nu, 8)), p.nsplit), dim3(256), lds, s, p, (int)nu, nqt);
  }
  int rc = ctclip_check_launch("win_attn_fwd");
  if (rc || p.nsplit == 1) return rc;
  const int64_t n = (int64_t)p.H * p.Mq;
  constexpr int SG = 256 / (D / 4);
  if (n > 4096) hipLaunchKernelGGL((join_kernel<T, D, 1>), dim3((unsigned)cdiv(n, SG)), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((join_kernel<T, D, SG>), dim3((unsigned)n), dim3(256), 0, s, p);
  return ctclip_check_launch("win_attn_fwd join");
}
template <typename T, int D> int launch_fwd_d(Params& p, const Plan& pl, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (fine_pass(p, DT_BF16, false)) return p.drop_p > 0.f ? launch_fwd<T, D, true, true>(p, pl, s) : launch_fwd<T, D, false, true>(p, pl, s);
  }
  return p.drop_p > 0.f ? launch_fwd<T, D, true, false>(p, pl, s) : launch_fwd<T, D, false, false>(p, pl, s);
}
template <typename T> int launch_fwd_t(Params& p, const Plan& pl, int D, hipStream_t s) {
  return D == 32 ? launch_fwd_d<T, 32>(p, pl, s) : (D == 64 ? launch_fwd_d<T, 64>(p, pl, s) : launch_fwd_d<T, 128>(p, pl, s));
}
}  // namespace win

// bytes of workspace of ctclip_win_attn_fwd (split passes; 0: none)
extern "C" int64_t ctclip_win_attn_fwd_workspace(int nseq, int Lq, int Lk, int H, int Hk, int D, int left, int right, int sinks, int q_start, int packed) {
  if (nseq < 1 || Lq < 1 || Lk < 1 || H < 1 || Hk < 1 || H % Hk || packed) return 0;
  const int l = left < 0 || left > Lk ? Lk : left, r = right < 0 || right > Lk ? Lk : right, s = sinks < Lk ? sinks : Lk;
  const int a = win::plan(nseq, Lq, Lk, H, Hk, l, r, s, q_start, false, DT_F32).nsplit, b = win::plan(nseq, Lq, Lk, H, Hk, l, r, s, q_start, false, DT_BF16).nsplit;
  const int n = a > b ? a : b;             // (of either type: the larger)
  return n > 1 ? win::part_bytes((int64_t)n * H * nseq * Lq, D) : 0;
}

// q (Mq, H D), k | v (Mk, Hk D) -> out (Mq, H D), lse [2][H][Mq] f32 (row maximum and log2 of the row's sum, log2 domain; optional: backward needs it).  Sequence b = rows b Lq ... of q and b Lk ... of
// k | v; with offsets (nseq + 1, int32) the rows offsets[b] ... offsets[b + 1] - 1 of all three (Lq = Lk = the longest), tiles = (sequence, 128-row tile) pairs.
// keymask: additive f32 per key row; a value <= -1e30 or NaN hides the key, whatever k and v hold there.
extern "C" int ctclip_win_attn_fwd(const void* q, const void* k, const void* v, const float* keymask, const int32_t* offsets, const int32_t* tiles, int ntiles, void* out,
                                   void* out_lo, float* lse, int nseq, int Lq, int Lk, int64_t Mq, int64_t Mk, int H, int Hk, int D, int left, int right, int sinks, int q_start,
                                   int64_t ldq, int64_t ldk, int64_t ldv, int64_t ldo, float scale, float dropout_p, uint64_t dropout_seed, int dtype, void* workspace,
                                   int64_t workspace_bytes, hipStream_t stream) {
  using namespace win;
  int rc = check_shape(nseq, Lq, Lk, Mq, Mk, H, Hk, D, left, right, sinks, q_start, offsets != nullptr, dtype);
  if (rc) return rc;
  if (!(scale > 0.f) || !(scale < 1e30f) || !(dropout_p >= 0.f) || !(dropout_p < 1.f)) { ctclip_set_error("win_attn_fwd: scale > 0, 0 <= dropout < 1"); return CTCLIP_EBADARG; }
  if (nseq == 0 || Lq == 0 || (offsets && ntiles == 0)) return CTCLIP_OK;
  if (offsets && (!tiles || ntiles < 0)) { ctclip_set_error("win_attn_fwd: packed sequences need their tiles"); return CTCLIP_EBADARG; }
  if ((rc = check_rows(q, ldq, Lq, H, D, dtype, false, "win_attn_fwd: q rows 16-byte aligned")) || (rc = check_rows(k, ldk, Lk, Hk, D, dtype, false, "win_attn_fwd: k rows 16-byte aligned")) ||
      (rc = check_rows(v, ldv, Lk, Hk, D, dtype, false, "win_attn_fwd: v rows 16-byte aligned")) || (rc = check_rows(out, ldo, Lq, H, D, dtype, true, "win_attn_fwd: out rows 16-byte aligned, apart")) ||
      (out_lo && (rc = check_rows(out_lo, ldo, Lq, H, D, dtype, true, "win_attn_fwd: out_lo rows 16-byte aligned")))) return rc;
  Params p{};
  fill(p, nseq, Lq, Lk, Mq, Mk, H, Hk, left, right, sinks, q_start, scale, dropout_p, dropout_seed, offsets, tiles, ntiles, keymask);
  p.q = q; p.k = k; p.v = v; p.out = out; p.out_lo = dtype == DT_BF16 ? out_lo : nullptr; p.lse = lse; p.ldq = ldq; p.ldk = ldk; p.ldv = ldv; p.ldo = ldo;
  const Plan pl = plan(nseq, Lq, Lk, H, Hk, p.left, p.right, p.sinks, q_start, offsets != nullptr, dtype);
  p.nsplit = pl.nsplit;
  if (p.nsplit > 1) {
    if (!workspace || workspace_bytes < part_bytes((int64_t)p.nsplit * H * Mq, D) || reinterpret_cast<uintptr_t>(workspace) % 16) { ctclip_set_error("win_attn_fwd: workspace"); return CTCLIP_EWORKSPACE; }
    p.part = (float*)workspace;
  }
  return dtype == DT_F32 ? launch_fwd_t<float>(p, pl, D, stream) : launch_fwd_t<bf16_t>(p, pl, D, stream);
}
