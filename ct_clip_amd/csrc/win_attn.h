// Shared pieces of the windowed attention kernels (win_attn.hip: forward, win_attn_bwd.hip: backward).
//
// Position i of a query sees key j when j <= i + right, and j >= i - left or j < sinks, and the key mask does not hide j.  O = softmax(scale q k^T + mask) v.
// Both products of a pass run on mfma 32x32 (bf16: x16, f32: x2) in the orientation S^T = K Q^T: a lane owns ONE query (column lane & 31) and 16 keys of a
// 32 x 32 block in registers, register r of half h = lane >> 5 being key 8 (r >> 2) + 4 h + (r & 3).  Row maximum and sum are therefore in-lane plus one
// exchange between the halves, and P^T feeds the second product as it stands: slot e of half h of the k-step G is key 16 G + 8 (e >> 2) + 4 h + (e & 3), and the
// matching V^T operand is two transposing LDS reads (ds_read_b64_tr_b16: four keys of one column per lane) of the row-major tile.  No transposed copies exist.
//
// LDS tiles are row-major without padding; the 16-byte chunks of row r are XOR-permuted with swz(r) so that the 16 rows of a ds_read_b128 group and the four
// rows x 64 bytes of a transposing read fall into distinct 16-byte slots of the 256-byte bank row.
#pragma once
#include <atomic>

#include "common.h"

namespace win {

constexpr float LOG2E_ = 1.4426950408889634f, LN2_ = 0.6931471805599453f;
constexpr float HIDDEN = -1e30f;          // an additive key mask value at or below this (or NaN) hides the key: HF's finfo.min, -inf
constexpr int QB = 128;                   // rows (queries, or keys in the dK / dV kernel) of a workgroup: 4 waves x 32

struct Params {
  const void *q, *k, *v, *o, *dout;
  const float* keymask;                   // additive, (key rows) f32, or null
  const int32_t* offsets;                 // packed sequences: first row of each (nseq + 1), or null: sequence b = rows b * Lq / b * Lk
  const int32_t* tiles;                   // packed sequences: (sequence, 128-row tile) of every tile
  int ntiles;
  void *out, *dq, *dk, *dv;
  void* out_lo;                           // bf16: what the rounding of `out` left over (pitch ldo), for the backward pass's Delta; or null
  float *lse, *delta;                     // [2][H][query rows]: maximum and log2 of the sum (0 and +inf for a row that sees nothing), apart: where a mask shifts every key of a row by
                                          // -1e9 their sum has lost the second; [H][query rows]: rowsum(dO o O)
  float* part;                            // workspace of split passes
  int nseq, Lq, Lk, H, Hk, G;
  int left, right, sinks, q_start;
  int64_t Mq, Mk;
  int64_t ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
  float scale, scale2;                    // scale2 = scale * log2 e
  uint64_t seed; const unsigned long long* seed_state; float drop_p, inv_keep;
  int nsplit;
  int s32, nchunk;                        // backward: keys of sink blocks (multiple of 32; of the longest sequence), chunks of the rows beyond their window
  int64_t sink_rows, sink_step;           // backward: rows of a k|v head that the sinks' partial sums take, and how they are shared out (win_attn_bwd.hip: sink_row)
};

template <typename T, int D> struct Geo {
  static constexpr int ESZ = (int)sizeof(T);
  static constexpr int ROWB = D * ESZ;                     // bytes of a tile row
  static constexpr int NCH = ROWB / 16;                    // 16-byte chunks of a row
  static constexpr int KT = ESZ == 2 ? 64 : 32;            // keys of a forward / dQ step
  static constexpr int NB = D / 32;                        // 32-column blocks of a head
};
// chunk permutation of row r (see the header comment); NCH = 4, 8, 16 or 32 chunks per row
template <int NCH> __device__ __forceinline__ int swz(int r) {
  if (NCH == 4) return (r >> 2) & 3;
  if (NCH == 8) { const int m = (r >> 1) & 7; return ((m & 1) << 2) | (m >> 1); }
  return ((r & 3) << 2) | ((r >> 2) & 3);
}
template <typename T, int D> __device__ __forceinline__ int lds_at(int row, int chunk) { return row * Geo<T, D>::ROWB + ((chunk ^ swz<Geo<T, D>::NCH>(row)) << 4); }

// operand whose rows are the matrix product's rows / columns and whose contraction runs along D: bf16 slot (g, e) of half h = column 16 g + 8 h + e,
// f32 instruction 4 g + e = column 8 g + 4 h + e
template <typename T, int D> struct RowFrag;
template <int D> struct RowFrag<bf16_t, D> { bf16x8 v[D / 16]; };
template <int D> struct RowFrag<float, D> { f32x4 v[D / 8]; };
template <typename T, int D> __device__ __forceinline__ void row_frag_zero(RowFrag<T, D>& f) {
#pragma unroll
  for (int g = 0; g < Geo<T, D>::NCH / 2; ++g) { const u32x4 z = {0, 0, 0, 0}; f.v[g] = __builtin_bit_cast(decltype(f.v[0] + f.v[0]), z); }
}
template <typename T, int D> __device__ __forceinline__ void row_frag_global(RowFrag<T, D>& f, const T* row, int half) {
#pragma unroll
  for (int g = 0; g < Geo<T, D>::NCH / 2; ++g) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(row) + (2 * g + half) * 16);
    f.v[g] = __builtin_bit_cast(decltype(f.v[0] + f.v[0]), w);
  }
}
template <int D> __device__ __forceinline__ f32x16 mma_rows(const RowFrag<bf16_t, D>& a, const RowFrag<bf16_t, D>& b, f32x16 c) {
#pragma unroll
  for (int g = 0; g < D / 16; ++g) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v[g], b.v[g], c, 0, 0, 0);
  return c;
}
template <int D> __device__ __forceinline__ f32x16 mma_rows(const RowFrag<float, D>& a, const RowFrag<float, D>& b, f32x16 c) {
#pragma unroll
  for (int g = 0; g < D / 8; ++g)
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[g][e], b.v[g][e], c, 0, 0, 0);
  return c;
}
// Wait for a fragment HERE.  Left to itself the compiler waits in front of the first product of a loop, in every round of it (it cannot count the loads of the first
// round), and so for the loads of the next round too, which are to arrive under the products.
template <typename T, int D> __device__ __forceinline__ void row_frag_arrive(RowFrag<T, D>& f) {
#pragma unroll
  for (int g = 0; g < Geo<T, D>::NCH / 2; ++g) {
    u32x4 w = __builtin_bit_cast(u32x4, f.v[g]);
    asm volatile("" : "+v"(w));
    f.v[g] = __builtin_bit_cast(decltype(f.v[0] + f.v[0]), w);
  }
}
// a lane's half of a row's dot product
template <int D> __device__ __forceinline__ float row_dot(const RowFrag<bf16_t, D>& a, const RowFrag<bf16_t, D>& b) {
  float s = 0.f;
#pragma unroll
  for (int g = 0; g < D / 16; ++g) {
    const u32x4 x = __builtin_bit_cast(u32x4, a.v[g]), y = __builtin_bit_cast(u32x4, b.v[g]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s = fmaf(__uint_as_float(x[e] << 16), __uint_as_float(y[e] << 16), s);
      s = fmaf(__uint_as_float(x[e] & 0xffff0000u), __uint_as_float(y[e] & 0xffff0000u), s);
    }
  }
  return s;
}
template <int D> __device__ __forceinline__ float row_dot(const RowFrag<float, D>& a, const RowFrag<float, D>& b) {
  float s = 0.f;
#pragma unroll
  for (int g = 0; g < D / 8; ++g)
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fmaf(a.v[g][e], b.v[g][e], s);
  return s;
}
// 32 probabilities (or dS) of a lane's query / key, 16 registers, as the second product's operand
template <typename T> struct PFrag;
template <> struct PFrag<bf16_t> { bf16x8 v[2]; };
template <> struct PFrag<float> { float v[16]; };
__device__ __forceinline__ void p_frag(PFrag<bf16_t>& f, const float (&p)[16]) {
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pack2bf(p[8 * g + 2 * e], p[8 * g + 2 * e + 1]);
    f.v[g] = __builtin_bit_cast(bf16x8, w);
  }
}
__device__ __forceinline__ void p_frag(PFrag<float>& f, const float (&p)[16]) {
#pragma unroll
  for (int r = 0; r < 16; ++r) f.v[r] = p[r];
}
// what that rounding left over (bf16), for a second product with the same other operand
__device__ __forceinline__ void p_rest(float (&p)[16]) {
#pragma unroll
  for (int r = 0; r < 16; ++r) p[r] -= bf2f(f2bf(p[r]));
}
typedef __attribute__((ext_vector_type(4))) short s16x4;
// A lane's byte offsets inside a 32-row block, computed once: `row` for the products along D (row c = lane & 31), `col` for the transposing reads of the second
// product (32-column block i, rows + 8 u).  Blocks are multiples of 32 rows apart, which the chunk permutation does not see, so everything else is an immediate.
template <typename T, int D> struct LaneAt {
  int row[Geo<T, D>::NCH / 2];
  int col[D / 32][2];
  __device__ __forceinline__ explicit LaneAt(int lane) {
    const int half = lane >> 5, c = lane & 31, t = lane & 15, g1 = (lane >> 4) & 1;
#pragma unroll
    for (int g = 0; g < Geo<T, D>::NCH / 2; ++g) row[g] = lds_at<T, D>(c, 2 * g + half);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u) col[i][u] = sizeof(T) == 2 ? lds_at<T, D>(8 * u + 4 * half + (t >> 2), 4 * i + 2 * g1 + ((t & 3) >> 1)) + (t & 1) * 8 : 0;
  }
};
template <typename T, int D> __device__ __forceinline__ void row_frag_lds(RowFrag<T, D>& f, const char* block, const LaneAt<T, D>& at) {
#pragma unroll
  for (int g = 0; g < Geo<T, D>::NCH / 2; ++g) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(block + at.row[g]);
    f.v[g] = __builtin_bit_cast(decltype(f.v[0] + f.v[0]), w);
  }
}
// Operand of the second product: the block's 32 rows read transposed from the row-major tile.  Read apart from the product, so that it can be on its way while
// something else is computed (bf16; f32 reads element by element inside the product).
template <typename T, int D> struct ColFrag;
template <int D> struct ColFrag<bf16_t, D> { bf16x8 v[2][D / 32]; };
template <int D> struct ColFrag<float, D> { const char* block; };
template <int D> __device__ __forceinline__ void col_frag_lds(ColFrag<bf16_t, D>& f, const char* block, const LaneAt<bf16_t, D>& at) {
#pragma unroll
  for (int G = 0; G < 2; ++G)
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(block + 16 * G * Geo<bf16_t, D>::ROWB + at.col[i][0]));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(block + 16 * G * Geo<bf16_t, D>::ROWB + at.col[i][1]));
      f.v[G][i] = bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
}
template <int D> __device__ __forceinline__ void col_frag_lds(ColFrag<float, D>& f, const char* block, const LaneAt<float, D>&) { f.block = block; }
// acc[i] += (32-column block i)^T x P
template <int D> __device__ __forceinline__ void mma_cols(f32x16 (&acc)[D / 32], const ColFrag<bf16_t, D>& f, const PFrag<bf16_t>& p, int) {
#pragma unroll
  for (int G = 0; G < 2; ++G)
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.v[G][i], p.v[G], acc[i], 0, 0, 0);
}
template <int D> __device__ __forceinline__ void mma_cols(f32x16 (&acc)[D / 32], const ColFrag<float, D>& f, const PFrag<float>& p, int lane) {
  const int half = lane >> 5, c = lane & 31;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = 8 * (r >> 2) + 4 * half + (r & 3);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const float a = *reinterpret_cast<const float*>(f.block + lds_at<float, D>(row, 8 * i + (c >> 2)) + (c & 3) * 4);
      acc[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p.v[r], acc[i], 0, 0, 0);
    }
  }
}
template <typename T, int D> __device__ __forceinline__ void mma_cols(f32x16 (&acc)[D / 32], const char* block, const LaneAt<T, D>& at, const PFrag<T>& p, int lane) {
  ColFrag<T, D> f;
  col_frag_lds<D>(f, block, at);
  mma_cols<D>(acc, f, p, lane);
}

__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : (n <= 0 ? 0ull : (1ull << n) - 1ull); }

__device__ __forceinline__ float mask_value(float km) { return km > HIDDEN ? km * LOG2E_ : -INFINITY; }      // (NaN hides)
// ---- a tile's journey, 16 bytes per lane straight from memory into LDS (buffer_load ... lds).  Through registers (load, then write to LDS) the tile in flight cost 16 to 64
// of them (a wave per SIMD less); with the lazily raised maximum of the forward pass 139 -> 101 us for 4 x 8192 tokens, 12 heads of 64, window 256 + 256.  The LDS side is linear in the thread index, so the
// chunk permutation is applied to the address that a lane READS.  Rows past the valid ones are outside the buffer descriptor, and the load writes zeros for them.
// Inline asm on purpose: next to the builtin the compiler waits for all loads in front of every LDS read, since it cannot tell the buffer being filled from the one
// being read.  There is no output register; dma_arrive() waits for everything in flight.
// A load writes LDS when its data comes back, past the queue that a wave's own LDS instructions keep their order in: issue() first waits for the wave's reads (of
// wave-private tiles: what it still reads of the tile that is refilled; shared tiles have a barrier in between, and nothing is left to wait for).
template <typename T, int D, int ROWS, int NT> struct Dma {
  static constexpr int N = ROWS * Geo<T, D>::NCH / NT;
  static_assert(N >= 1 && ROWS * Geo<T, D>::NCH % NT == 0 && NT % 64 == 0, "whole chunks per thread");
  uint32_t off[N];                                         // a lane's byte offsets inside a tile
  __device__ static __forceinline__ int row(int tid, int i) { return (tid + i * NT) / Geo<T, D>::NCH; }
  __device__ __forceinline__ void init(int ldb, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = row(tid, i), c = (tid + i * NT) % Geo<T, D>::NCH;
      const uint64_t o = (uint64_t)(uint32_t)r * (uint32_t)ldb + (uint32_t)((c ^ swz<Geo<T, D>::NCH>(r)) << 4);
      off[i] = o < 0x7fffffffull ? (uint32_t)o : 0x7fffffffu;              // (a row that far is past the valid ones)
    }
  }
  // tile, ldb (bytes between rows), valid (rows from the tile's first on that may be read, >= 1) are uniform; valid rows lie within 2^31 bytes (check_rows)
  __device__ __forceinline__ void issue(char* lds_tile, const char* tile, int ldb, int valid, int tid) const {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const uint64_t base = reinterpret_cast<uint64_t>(tile);
    const uint32_t bytes = valid >= ROWS ? 0x7fffffffu : (uint32_t)((valid - 1) * ldb) + (uint32_t)Geo<T, D>::ROWB;
    const u32x4 rsrc = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)base), (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(base >> 32) & 0xffffu)),
                        (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00027000u};
    const uint32_t dst = (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds_tile + (uint32_t)(tid & ~63) * 16u));
#pragma unroll
    for (int i = 0; i < N; ++i)
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" :: "s"(dst + (uint32_t)(i * NT * 16)), "v"(off[i]), "s"(rsrc) : "memory", "m0");
  }
  // (behind dma_arrive()) zeros over the rows of this thread's chunks that `keep` leaves out
  __device__ __forceinline__ void erase(char* lds_tile, uint64_t keep, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (!((keep >> row(tid, i)) & 1)) { const u32x4 z = {0, 0, 0, 0}; *reinterpret_cast<u32x4*>(lds_tile + (tid + i * NT) * 16) = z; }
  }
};
__device__ __forceinline__ void dma_arrive() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// The key tiles (KT keys of k and v) of a (sequence, k|v head) on their way into LDS, with the key mask.  NT threads share a tile; every wave knows the whole tile's
// mask by a ballot (lane = key), so hidden rows and the state are wave-uniform masks.
struct KeySource {
  const char *k, *v;
  const float* mask;
  int ldk, ldv, lk, jlo, jhi, sinks;                       // keys outside [jlo, jhi] and the sinks are seen by nobody here
  template <typename T, int D> __device__ __forceinline__ void init(const Params& p, int64_t k0, int hk, int lk_, int jlo_, int jhi_) {
    k = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.k) + k0 * p.ldk + (int64_t)hk * D);
    v = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.v) + k0 * p.ldv + (int64_t)hk * D);
    mask = p.keymask ? p.keymask + k0 : nullptr;
    ldk = (int)p.ldk * (int)sizeof(T); ldv = (int)p.ldv * (int)sizeof(T);
    lk = lk_; jlo = jlo_; jhi = jhi_ < lk_ - 1 ? jhi_ : lk_ - 1; sinks = p.sinks;
  }
  // rows of the tile at j0 that may be seen, and (return) what its mask looks like: 0 nothing, 1 some additive values (written to `bias`), 2 no key is seen
  template <int KT> __device__ __forceinline__ int look(uint64_t& keep, float km, float* bias, int j0, int tid) const {
    keep = low_bits(jhi + 1 - j0);
    if (j0 < jlo) keep &= ~low_bits(jlo - j0) | low_bits(sinks - j0);
    int state = 0;
    if (mask) {
      const float b = mask_value(km);
      const uint64_t seen = __builtin_amdgcn_ballot_w64(b > -INFINITY);
      keep &= seen;
      state = (keep & low_bits(KT)) == 0 ? 2 : (__builtin_amdgcn_ballot_w64(b != 0.f) != 0 ? 1 : 0);
      if (tid < KT) bias[tid] = b;
    }
    keep |= ~low_bits(KT);
    return state;
  }
};
template <typename T, int D, int KT, int NT> struct KeyPipe {      // through LDS-DMA: issue() into a buffer that nobody reads, settle() before the barrier
  KeySource src;
  Dma<T, D, KT, NT> dk, dv;
  float km;
  int j0;
  __device__ __forceinline__ KeyPipe(const Params& p, int64_t k0, int hk, int lk, int jlo, int jhi, int tid) {
    src.init<T, D>(p, k0, hk, lk, jlo, jhi);
    dk.init(src.ldk, tid);
    dv.init(src.ldv, tid);
    km = 0.f; j0 = 0;
  }
  __device__ __forceinline__ void issue(char* kt, char* vt, int first, int tid) {
    j0 = first;
    dk.issue(kt, src.k + (int64_t)first * src.ldk, src.ldk, src.jhi + 1 - first, tid);
    dv.issue(vt, src.v + (int64_t)first * src.ldv, src.ldv, src.jhi + 1 - first, tid);
    if (src.mask) { const int j = first + (tid & (KT - 1)); km = src.mask[j < src.lk ? j : src.lk - 1]; }
  }
  __device__ __forceinline__ int settle(char* kt, char* vt, float* bias, int tid) const {
    dma_arrive();
    if (!src.mask && j0 >= src.jlo) return 0;              // (rows past jhi have been written as zeros)
    uint64_t keep;
    const int state = src.look<KT>(keep, km, bias, j0, tid);
    if (~keep) { dk.erase(kt, keep, tid); dv.erase(vt, keep, tid); }
    return state;
  }
};
// visibility by position of 32 x 32 blocks: rows lo ... hi (positions; hi < lo: none) against keys j0 ... j0 + 31: 0 nothing, 1 some, 2 everything
struct Sight {
  int none_above, full_above, full_below, none_below, sinks;
  __device__ __forceinline__ Sight(int lo, int hi, int left, int right, int sinks_, int lk) {
    const int top = lk - 1;
    none_above = hi < lo ? -1 : (hi + right < top ? hi + right : top);       // first key of the block past this: nothing
    full_above = lo + right < top ? lo + right : top;                        // last key of the block past this: not everything
    full_below = hi - left;
    none_below = lo - left;
    sinks = sinks_;
  }
  __device__ __forceinline__ int of(int j0) const {
    const int j1 = j0 + 31;
    if (j0 > none_above) return 0;
    if (j1 <= full_above && (j0 >= full_below || j1 < sinks)) return 2;
    return j1 < none_below && j0 >= sinks ? 0 : 1;
  }
};

// dropout multipliers of a lane's query row qi and the 16 keys j0 + 8 (r >> 2) + 4 h + (r & 3): common.h attn_drop_block (one Philox call per 2 rows x 4 keys).
// PAIRED: lanes c, c ^ 1 hold rows 2 n, 2 n + 1 of one sequence and head, so each draws two of the four blocks and they swap
template <bool PAIRED> __device__ __forceinline__ void drop_of_query(float (&m)[16], const Params& p, int64_t sh, int qi, int j0, int half) {
  const uint64_t seed = p.seed + (p.seed_state ? p.seed_state[0] : 0ull);
  const uint32_t thr = attn_drop_threshold(p.drop_p);
  u32x4 w[4];
  if (PAIRED) {
    const int par = (int)(threadIdx.x & 1);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const u32x4 own = attn_drop_block(seed, sh, p.Lk, qi, j0 + 8 * (2 * s + par) + 4 * half);
      u32x4 oth;
#pragma unroll
      for (int e = 0; e < 4; ++e) oth[e] = (uint32_t)__builtin_amdgcn_mov_dpp((int)own[e], 0xB1, 0xF, 0xF, true);
#pragma unroll
      for (int e = 0; e < 4; ++e) { w[2 * s][e] = par ? oth[e] : own[e]; w[2 * s + 1][e] = par ? own[e] : oth[e]; }
    }
  } else {
#pragma unroll
    for (int s = 0; s < 4; ++s) w[s] = attn_drop_block(seed, sh, p.Lk, qi, j0 + 8 * s + 4 * half);
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) m[r] = attn_drop_pick(w[r >> 2], qi, r & 3, thr, p.inv_keep);
}

// which unit of work a workgroup has.  Units of one (sequence, k|v head) are neighbours and one XCD (workgroup index mod 8) gets a contiguous run of them, so
// that a key tile read by the query tiles around it comes from that XCD's L2.  Packed sequences: heads outermost, so that a run holds every sequence.
struct Unit { int b, hk, g, tile; bool real; };
__device__ __forceinline__ Unit unit_of(const Params& p, int id, int n, int per_seq_tiles, int G) {
  const int per = (n + 7) >> 3;
  const int v = (id & 7) * per + (id >> 3);
  Unit u{0, 0, 0, 0, v < n};
  if (!u.real) return u;
  u.g = v % G;
  int w = v / G;
  if (p.offsets) {
    const int i = w % p.ntiles;
    u.hk = w / p.ntiles;
    u.b = p.tiles[2 * i];
    u.tile = p.tiles[2 * i + 1];
    u.real = u.b >= 0 && u.b < p.nseq && u.tile >= 0 && u.tile < (1 << 22);
  } else {
    u.tile = w % per_seq_tiles;
    w /= per_seq_tiles;
    u.hk = w % p.Hk;
    u.b = w / p.Hk;
  }
  return u;
}
// rows of sequence b; packed offsets are clamped to the tensors, whatever they hold
struct Rows { int64_t q0, k0; int lq, lk; };
__device__ __forceinline__ Rows rows_of(const Params& p, int b) {
  Rows r;
  if (p.offsets) {
    int64_t a = p.offsets[b], e = p.offsets[b + 1];
    a = a < 0 ? 0 : (a > p.Mq ? p.Mq : a);
    e = e < a ? a : (e > p.Mq ? p.Mq : e);
    r.q0 = r.k0 = a;
    r.lq = r.lk = (int)(e - a < p.Lk ? e - a : p.Lk);
  } else {
    r.q0 = (int64_t)b * p.Lq; r.k0 = (int64_t)b * p.Lk;
    r.lq = p.Lq; r.lk = p.Lk;
  }
  return r;
}
// key tiles (of KT keys) that positions lo ... hi can see: nsink tiles from 0, then first ... first + n - nsink - 1
struct TileList { int nsink, first, n; };
template <int KT> __device__ __host__ __forceinline__ TileList tile_list(int lo, int hi, int left, int right, int sinks, int Lk) {
  TileList t;
  const int jhi = hi + right < Lk - 1 ? hi + right : Lk - 1;
  int jlo = lo - left; if (jlo < 0) jlo = 0;
  const int s = sinks < jhi + 1 ? sinks : jhi + 1;
  t.nsink = s > 0 ? (s + KT - 1) / KT : 0;
  t.first = jlo / KT; if (t.first < t.nsink) t.first = t.nsink;
  const int last = jhi >= jlo ? jhi / KT : -1;
  t.n = t.nsink + (last >= t.first ? last - t.first + 1 : 0);
  return t;
}
__device__ __forceinline__ int tile_at(const TileList& t, int i) { return i < t.nsink ? i : t.first + i - t.nsink; }

// a lane's row: columns 32 i + 8 g + 4 h + e; four consecutive columns per store (partial sums)
template <int D> __device__ __forceinline__ void store_part(float* row, const f32x16 (&acc)[D / 32], int half) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) *reinterpret_cast<f32x4*>(row + 32 * i + 8 * g + 4 * half) = f32x4{acc[i][4 * g], acc[i][4 * g + 1], acc[i][4 * g + 2], acc[i][4 * g + 3]};
}
__device__ __forceinline__ void wave_sync();
// A wave's 32 rows to memory, by way of 32 * ROWB bytes of LDS that nobody else touches: a lane holds four columns of one row at a time, and stored from there an
// instruction would touch 32 lines for 16 bytes each; after the turn it writes whole lines.  lane c = lane & 31 is row c; rows from `n` on are not stored.
// REST: what the rounding of the values leaves over, instead of the values (bf16)
template <typename T, int D, bool REST> __device__ __forceinline__ void store_rows(char* lds, const f32x16 (&acc)[D / 32], float mul, T* first, int64_t ld, int n, int lane) {
  const int half = lane >> 5, c = lane & 31;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] = acc[i][4 * g + e] * mul;
        if (REST && sizeof(T) == 2) o[e] -= bf2f(f2bf(o[e]));
      }
      store4(reinterpret_cast<T*>(lds + lds_at<T, D>(c, sizeof(T) == 2 ? 4 * i + g : 8 * i + 2 * g + half) + (sizeof(T) == 2 ? 8 * half : 0)), o);
    }
  wave_sync();
#pragma unroll
  for (int k = 0; k < 32 * Geo<T, D>::NCH / 64; ++k) {
    const int r = (lane + 64 * k) / Geo<T, D>::NCH, ch = (lane + 64 * k) % Geo<T, D>::NCH;
    const u32x4 w = *reinterpret_cast<const u32x4*>(lds + lds_at<T, D>(r, ch));
    if (r < n) *reinterpret_cast<u32x4*>(reinterpret_cast<char*>(first + (int64_t)r * ld) + ch * 16) = w;
  }
  wave_sync();
}
// four columns of a finished row of O
template <typename T> __device__ __forceinline__ void store_out(const Params& p, int64_t row, int64_t col, float (&o)[4]) {
  store4(reinterpret_cast<T*>(p.out) + row * p.ldo + col, o);
  if constexpr (sizeof(T) == 2) {
    if (p.out_lo) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] -= bf2f(f2bf(o[e]));
      store4(reinterpret_cast<T*>(p.out_lo) + row * p.ldo + col, o);
    }
  }
}
// the statistics of a finished row: what the backward pass takes its probabilities from
__device__ __forceinline__ void store_lse(const Params& p, int64_t i, float m, float l) {
  if (!p.lse) return;
  p.lse[i] = l == 0.f ? 0.f : m;
  p.lse[(int64_t)p.H * p.Mq + i] = l == 0.f ? INFINITY : __builtin_amdgcn_logf(l);
}
// lanes of a wave exchange through LDS: its LDS instructions retire in order, so only the compiler has to keep them in place (loads into LDS are no such instructions: Dma::issue)
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}


// ---- host side
inline int check_shape(int nseq, int Lq, int Lk, int64_t Mq, int64_t Mk, int H, int Hk, int D, int left, int right, int sinks, int q_start, bool packed, int dtype) {
  if (nseq < 0 || Lq < 0 || Lk < 0 || H < 1 || Hk < 1 || H % Hk || sinks < 0 || q_start < 0 || left < -1 || right < -1) { ctclip_set_error("win_attn: bad sizes (H a multiple of the k|v heads, window >= -1, sinks, q_start >= 0)"); return CTCLIP_EBADARG; }
  if ((D != 32 && D != 64 && D != 128) || (dtype != DT_F32 && dtype != DT_BF16)) { ctclip_set_error("win_attn: heads of 32, 64 or 128, f32 or bf16"); return CTCLIP_EUNSUPPORTED; }
  if (Lk > (1 << 29) || H > 65535 || (int64_t)Mq > ((int64_t)1 << 31) - 256 || (int64_t)Mk > ((int64_t)1 << 31) - 256) { ctclip_set_error("win_attn: too many rows or heads"); return CTCLIP_EUNSUPPORTED; }
  if (packed ? (Lq != Lk || Mq != Mk || q_start) : ((int64_t)q_start + Lq > Lk || Mq != (int64_t)nseq * Lq || Mk != (int64_t)nseq * Lk)) { ctclip_set_error("win_attn: query rows must be positions of the key axis (q_start + Lq <= Lk); packed sequences: q and k|v share their rows"); return CTCLIP_EBADARG; }
  return CTCLIP_OK;
}
// rows: of a sequence; those of one tile (128 at most) must lie within 2^31 bytes
inline int check_rows(const void* x, int64_t ld, int rows, int heads, int D, int dtype, bool written, const char* what) {
  const int e = dtype == DT_F32 ? 4 : 2;
  if (!x) { ctclip_set_error("win_attn: null tensor"); return CTCLIP_EBADARG; }
  if ((reinterpret_cast<uintptr_t>(x) % 16) || (ld * e) % 16 || ld < 0 || ld > ((int64_t)1 << 31) / e - 256 || (written && ld < (int64_t)heads * D)) { ctclip_set_error(what); return CTCLIP_EBADARG; }
  if ((int64_t)((rows < QB ? rows : QB) - 1) * ld * e + (int64_t)D * e >= ((int64_t)1 << 31) - 1) { ctclip_set_error("win_attn: 128 rows within 2 GiB"); return CTCLIP_EUNSUPPORTED; }
  return CTCLIP_OK;
}
inline void fill(Params& p, int nseq, int Lq, int Lk, int64_t Mq, int64_t Mk, int H, int Hk, int left, int right, int sinks, int q_start, float scale, float dropout_p,
          uint64_t seed, const int32_t* offsets, const int32_t* tiles, int ntiles, const float* keymask) {
  p.nseq = nseq; p.Lq = Lq; p.Lk = Lk; p.Mq = Mq; p.Mk = Mk; p.H = H; p.Hk = Hk; p.G = H / Hk;
  p.left = left < 0 || left > Lk ? Lk : left; p.right = right < 0 || right > Lk ? Lk : right; p.sinks = sinks < Lk ? sinks : Lk; p.q_start = q_start;
  p.scale = scale; p.scale2 = scale * LOG2E_;
  p.seed = seed; p.seed_state = ctclip_step_state(); p.drop_p = dropout_p; p.inv_keep = dropout_p > 0.f ? 1.f / (1.f - dropout_p) : 1.f;
  p.offsets = offsets; p.tiles = tiles; p.ntiles = ntiles; p.keymask = keymask;
}

// FINE (bf16): P and dS are rounded to the operand type for the second products; FINE passes take what that left over as well, in a second instruction each.
//   Forward, up to 64 visible keys: Delta = rowsum(dO o O) has the probabilities' rounding over the root of the keys that count, which would be seen beside the one rounding that
//   dS = P o (dP - Delta) has of its own (300 tokens, window 8 + 2: dq 2.60e-3 from 64 bits, then 2.36e-3; at 81 keys 2.39e-3 without it).  8 x 512 tokens, 12 heads, window
//   16 + 16: 15.8 -> 17.2 us.
//   Both passes, up to 2^20 pairs of a query and a visible key: few probabilities leave no average of their roundings (4 tokens, 4 heads: 2.6e-3), and a call of that size is
//   launches and latency: forward and
//   backward of 8 x 4 tokens 4.8 + 13.1 -> 4.9 + 13.9 us, of 500 tokens, 12 heads, window 80 + 80 (0.97 * 2^20 pairs) 15.5 + 34.9 -> 16.7 + 37.5; errors 2.35e-3 -> 1.66e-3,
//   which is the results' own rounding.
//   A forward pass without a backward one takes them by the same rule, so that an output's bits do not depend on the mode of autograd: 8 x 512 tokens, 12 heads, window 16 + 16,
//   13.8 -> 15.4 us, 4 x 8192 tokens, window 30 + 30, 48.9 -> 59.2, the [CLS] rows of 8 x 512 5.7 -> 5.9 (error 2.1e-3 -> 1.7e-3).
inline bool fine_pass(const Params& p, int dtype, bool backward) {
  const int64_t window = (int64_t)p.left + p.right + 1 + p.sinks, keys = window < p.Lk ? window : p.Lk;
  return dtype == DT_BF16 && ((!backward && keys <= 64) || keys * p.Mq * p.H <= (1 << 20));
}
// a launch holds fewer than 2^32 threads along its grid's first axis
inline int check_grid(int64_t workgroups, int threads) {
  if (workgroups < ((int64_t)1 << 32) / threads) return CTCLIP_OK;
  ctclip_set_error("win_attn: too many sequences, heads or tiles for a launch (2^32 threads)");
  return CTCLIP_EUNSUPPORTED;
}
template <auto KERNEL> int raise_lds(int bytes) {       // more than 64 KB of LDS is opted into, once per kernel and device (or, by several threads at once, a few times)
  static std::atomic<bool> done[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) { ctclip_set_error("win_attn: no device"); return CTCLIP_EBADARG; }
  if (!done[dev].load(std::memory_order_acquire)) {
    const hipError_t e = hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) { ctclip_set_error("win_attn: LDS size refused"); return -(1000 + (int)e); }
    done[dev].store(true, std::memory_order_release);
  }
  return CTCLIP_OK;
}

}  // namespace win
