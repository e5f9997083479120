// Rotary positions on gfx950: q and k of a projection's output, rotated in one launch.
//
// A pair (a, b) of a head at position p with frequency f (radians per position) becomes magnitude * (a cos pf - b sin pf, b cos pf + a sin pf); the backward
// pass is the rotation by -pf with the same magnitude.  Pairs are x[i], x[i + rot/2] (half layout) or x[2i], x[2i+1] (interleaved), columns rot ... D - 1 of a
// head pass through.
//
// Angles.  f / 2 pi is given as a 64-bit binary FRACTION OF A TURN (mod 1): p * turns mod 2^64 is then the exact angle of an integer position in fixed
// point -- whole turns fall off the top by themselves, so that position 10^6 is as exact as position 1 (an f32 product p * f has lost 0.06 radians there)
// and there is no table with a last row.  The top 32 bits are split into the nearest quarter turn and a remainder in [-1/8, 1/8] turn, sin / cos of which
// are their Taylor polynomials (first terms left out: x^11 / 11! < 1.8e-9, x^12 / 12! < 1.2e-10 at pi / 4).
//
// Bound: HBM, every element is read and written once.  A workgroup takes a few tokens, computes their rot / 2 sines and cosines once into LDS (f32) and
// then streams the tokens' heads, 16 bytes per load; without the sharing the 24 heads of a BERT token would each pay the ~40 instructions of an angle.
// MI355X: 32002 tokens, 40 heads of 128 (bf16, interleaved) 131 us a direction, 655 MB at 5.0 TB/s (a large copy: 5.1); 8 x 512 tokens, 24 heads of 64 5.3 us, 25 MB at
// 4.7 TB/s; f32, 12297 tokens, 16 heads of 32 11.7 us, 50 MB at 4.3 TB/s; four tokens 2.6 us, which is a launch.
#include "common.h"

namespace {

struct RotaryParams {
  const void *q, *k;
  void *qo, *ko;
  const uint64_t* turns;      // rot / 2 fractions of a turn per position, times 2^64
  const void* pos;            // positions of the rows (int32 / int64), or null: start + row % L
  int pos64;
  int64_t M, L, start;
  int Hq, Hk, D, rot, inplace;
  int64_t ldq, ldk, ldqo, ldko;
  float mag, sgn;             // sgn = -1: the inverse rotation (backward)
  int tb;                     // tokens of a workgroup
  int nch, nitem;             // vector kernel: work items of a head / of a token
  uint32_t magic;             // item / nch = item * magic >> 20 (checked on the host)
};

__device__ __forceinline__ int64_t row_position(const RotaryParams& p, int64_t row) {
  if (p.pos) return p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[row] : (int64_t)reinterpret_cast<const int32_t*>(p.pos)[row];
  return p.start + row % p.L;
}
// cos and sin of a 64-bit fraction of a turn
__device__ __forceinline__ void turn_cos_sin(uint64_t u, float& c, float& s) {
  const int32_t hi = (int32_t)((u + 0x80000000ull) >> 32);                        // turns * 2^32, nearest
  const int32_t n = (int32_t)(((uint32_t)hi + (1u << 29)) >> 30);                 // nearest quarter turn (mod 4)
  const int32_t r = (int32_t)((uint32_t)hi - ((uint32_t)n << 30));                // what is left: [-2^29, 2^29)
  const float x = (float)r * 1.4629180792671596e-9f, x2 = x * x;                  // (pi / 2) / 2^30
  float sp = fmaf(x2, 2.7557319e-6f, -1.9841270e-4f);                             // sin: x - x^3/3! + x^5/5! - x^7/7! + x^9/9!
  sp = fmaf(sp, x2, 8.3333333e-3f); sp = fmaf(sp, x2, -0.16666667f);
  sp = fmaf(sp * x2, x, x);
  float cp = fmaf(x2, -2.7557319e-7f, 2.4801587e-5f);                             // cos: 1 - x^2/2! + x^4/4! - x^6/6! + x^8/8! - x^10/10!
  cp = fmaf(cp, x2, -1.3888889e-3f); cp = fmaf(cp, x2, 4.1666667e-2f); cp = fmaf(cp, x2, -0.5f);
  cp = fmaf(cp, x2, 1.f);
  const float a = (n & 1) ? sp : cp, b = (n & 1) ? cp : sp;
  c = ((n + 1) & 2) ? -a : a;
  s = (n & 2) ? -b : b;
}

// 16-byte kernel: D, rot / 2 (half) or rot (interleaved) and D - rot multiples of 8, rows 16-byte aligned.
// An item is 8 pairs (half: 8 columns of either half; interleaved: 16 columns would be two lines apart for no gain: 8 columns, 4 pairs) or 8 columns that
// pass through; those come after the rotated items of a head and are left out in place.
template <typename T, int LAYOUT>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p) {
  extern __shared__ __attribute__((aligned(16))) float cs[];                      // [token][cos: rot / 2 | sin: rot / 2]
  const int half = p.rot >> 1;
  const int64_t row0 = (int64_t)blockIdx.x * p.tb;
  const int nt = (int)(p.M - row0 < p.tb ? p.M - row0 : p.tb);
  for (int i = threadIdx.x; i < nt * half; i += 256) {
    const int t = i / half, f = i - t * half;
    float c, s;
    turn_cos_sin((uint64_t)row_position(p, row0 + t) * p.turns[f], c, s);
    cs[t * p.rot + f] = c * p.mag;
    cs[t * p.rot + half + f] = s * p.mag * p.sgn;
  }
  __syncthreads();
  const int nrot = LAYOUT == 0 ? half >> 3 : p.rot >> 3;
  int t = 0, item = threadIdx.x;
  for (;;) {
    while (item >= p.nitem) { item -= p.nitem; ++t; }
    if (t >= nt) break;
    const int head = (int)(((uint32_t)item * p.magic) >> 20), ch = item - head * p.nch;
    const bool isq = head < p.Hq;
    const int h = isq ? head : head - p.Hq;
    const int64_t row = row0 + t;
    const T* src = reinterpret_cast<const T*>(isq ? p.q : p.k) + row * (isq ? p.ldq : p.ldk) + h * p.D;
    T* dst = reinterpret_cast<T*>(isq ? p.qo : p.ko) + row * (isq ? p.ldqo : p.ldko) + h * p.D;
    const float* ct = cs + t * p.rot;
    if (ch >= nrot) {
      const int col = p.rot + (ch - nrot) * 8;
      float v[8];
      load8(src + col, v);
      store8(dst + col, v);
    } else if (LAYOUT == 0) {
      const int col = ch * 8;
      float a[8], b[8], c[8], s[8], x[8], y[8];
      load8(src + col, a);
      load8(src + half + col, b);
      load8(ct + col, c);
      load8(ct + half + col, s);
#pragma unroll
      for (int e = 0; e < 8; ++e) { x[e] = fmaf(a[e], c[e], -b[e] * s[e]); y[e] = fmaf(b[e], c[e], a[e] * s[e]); }
      store8(dst + col, x);
      store8(dst + half + col, y);
    } else {
      const int col = ch * 8;
      float a[8], c[4], s[4], x[8];
      load8(src + col, a);
      load4(ct + (col >> 1), c);
      load4(ct + half + (col >> 1), s);
#pragma unroll
      for (int e = 0; e < 4; ++e) { x[2 * e] = fmaf(a[2 * e], c[e], -a[2 * e + 1] * s[e]); x[2 * e + 1] = fmaf(a[2 * e + 1], c[e], a[2 * e] * s[e]); }
      store8(dst + col, x);
    }
    item += 256;
  }
}

// any even rot, any alignment: one thread per pair or passed-through element, an angle each (on the shapes above 481, 17.1 and 16.6 us)
template <typename T>
__global__ __launch_bounds__(256) void rotary_any_kernel(RotaryParams p, int interleaved) {
  const int half = p.rot >> 1, per = half + (p.inplace ? 0 : p.D - p.rot), heads = p.Hq + p.Hk;
  const int64_t n = p.M * heads * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int e = (int)(i % per);
    const int64_t th = i / per;
    const int head = (int)(th % heads);
    const int64_t row = th / heads;
    const bool isq = head < p.Hq;
    const int h = isq ? head : head - p.Hq;
    const T* src = reinterpret_cast<const T*>(isq ? p.q : p.k) + row * (isq ? p.ldq : p.ldk) + (int64_t)h * p.D;
    T* dst = reinterpret_cast<T*>(isq ? p.qo : p.ko) + row * (isq ? p.ldqo : p.ldko) + (int64_t)h * p.D;
    if (e >= half) { dst[half + e] = src[half + e]; continue; }                   // column rot + (e - half)
    float c, s;
    turn_cos_sin((uint64_t)row_position(p, row) * p.turns[e], c, s);
    c *= p.mag; s *= p.mag * p.sgn;
    const int ia = interleaved ? 2 * e : e, ib = interleaved ? 2 * e + 1 : e + half;
    const float a = Elem<T>::ld(src + ia), b = Elem<T>::ld(src + ib);
    Elem<T>::st(dst + ia, fmaf(a, c, -b * s));
    Elem<T>::st(dst + ib, fmaf(b, c, a * s));
  }
}

template <typename T> int rotary_launch(RotaryParams& p, int interleaved, hipStream_t s) {
  const int rowsz = (int)sizeof(T), half = p.rot / 2, heads = p.Hq + p.Hk;
  auto al = [&](const void* x, int64_t ld) { return !x || ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)(ld * rowsz)) % 16 == 0); };
  const bool vec = p.D % 8 == 0 && p.rot % 8 == 0 && (interleaved || half % 8 == 0) && al(p.q, p.ldq) && al(p.k, p.ldk) && al(p.qo, p.ldqo) && al(p.ko, p.ldko);
  const int nrot = interleaved ? p.rot / 8 : half / 8;
  p.nch = nrot + (p.inplace ? 0 : (p.D - p.rot) / 8);
  p.nitem = heads * p.nch;
  // (the second line keeps item * magic >> 20 = item / nch exact and below 2^32, and the angles of 16 tokens within 32 KB of LDS)
  if (vec && (int64_t)p.nitem * p.nch < (1 << 20) && heads < 2048 && p.rot <= 512) {
    p.magic = ((1u << 20) + p.nch - 1) / p.nch;
    // tokens of a workgroup: eight items per thread keep the angles' share of the time small, but not at the price of an empty chip (2 048 workgroups:
    // eight per CU).  One token per workgroup at least: a single token of BERT-base is 96 items.  8 x 512 tokens of 24 heads: 5.3 us; one token always 6.8, sixteen always 7.5;
    // f32, 12297 tokens of 16 heads of 32: 11.7, 14.0 and 12.0.
    int tb = 2048 / p.nitem;
    if (tb > 16) tb = 16;
    if (tb * (int64_t)2048 > p.M) tb = (int)(p.M / 2048);
    if (tb < 1) tb = 1;
    p.tb = tb;
    if (cdiv(p.M, tb) >= (1 << 24)) { ctclip_set_error("rotary: too many rows"); return CTCLIP_EUNSUPPORTED; }      // (2^32 threads of a launch)
    const dim3 grid((unsigned)cdiv(p.M, tb));
    const size_t lds = (size_t)tb * p.rot * 4;
    if (interleaved) hipLaunchKernelGGL((rotary_kernel<T, 1>), grid, dim3(256), lds, s, p);
    else hipLaunchKernelGGL((rotary_kernel<T, 0>), grid, dim3(256), lds, s, p);
  } else {
    int64_t nb = cdiv(p.M * heads * (half + (p.inplace ? 0 : p.D - p.rot)), 256);
    if (nb > 16384) nb = 16384;
    hipLaunchKernelGGL(rotary_any_kernel<T>, dim3((unsigned)nb), dim3(256), 0, s, p, interleaved);
  }
  return ctclip_check_launch("rotary");
}

}  // namespace

// q (M, Hq D) and k (M, Hk D; null with Hk = 0) -> qo, ko (the same pointers and pitches: in place).  turns: rot / 2 frequencies as 64-bit fractions of a
// turn per position.  positions: one integer per row (pos_bytes 4 or 8), or null: start + row % L.
extern "C" int ctclip_rotary(const void* q, const void* k, void* qo, void* ko, const uint64_t* turns, const void* positions, int pos_bytes, int64_t M,
                             int64_t L, int64_t start, int Hq, int Hk, int D, int rot, int64_t ldq, int64_t ldk, int64_t ldqo, int64_t ldko, int interleaved,
                             float magnitude, int inverse, int dtype, hipStream_t stream) {
  if (M < 0 || Hq < 1 || Hk < 0 || D < 2 || rot < 2 || rot > D || (rot & 1) || (!positions && L < 1)) { ctclip_set_error("rotary: bad sizes (rot even, 2 <= rot <= D)"); return CTCLIP_EBADARG; }
  if (M == 0) return CTCLIP_OK;
  if (!q || !qo || !turns || (Hk && (!k || !ko))) { ctclip_set_error("rotary: null argument"); return CTCLIP_EBADARG; }
  if (positions && pos_bytes != 4 && pos_bytes != 8) { ctclip_set_error("rotary: positions are 4- or 8-byte integers"); return CTCLIP_EBADARG; }
  if (dtype != DT_F32 && dtype != DT_BF16) { ctclip_set_error("rotary: f32 or bf16"); return CTCLIP_EUNSUPPORTED; }
  if (ldqo < (int64_t)Hq * D || (Hk && ldko < (int64_t)Hk * D) || ldq < 0 || ldk < 0) { ctclip_set_error("rotary: output rows overlap"); return CTCLIP_EBADARG; }
  const bool iq = q == qo, ik = !Hk || k == ko;
  if (iq != (Hk ? k == ko : iq) || (iq && (ldq != ldqo || (Hk && ldk != ldko)))) { ctclip_set_error("rotary: in place means both tensors with their own pitches"); return CTCLIP_EBADARG; }
  if (M > ((int64_t)1 << 31) || (int64_t)(Hq + Hk) * D > (1 << 24)) { ctclip_set_error("rotary: too large"); return CTCLIP_EUNSUPPORTED; }
  RotaryParams p{};
  p.q = q; p.k = k; p.qo = qo; p.ko = ko; p.turns = turns; p.pos = positions; p.pos64 = pos_bytes == 8;
  p.M = M; p.L = L < 1 ? 1 : L; p.start = start; p.Hq = Hq; p.Hk = Hk; p.D = D; p.rot = rot; p.inplace = iq && ik;
  p.ldq = ldq; p.ldk = ldk; p.ldqo = ldqo; p.ldko = ldko; p.mag = magnitude; p.sgn = inverse ? -1.f : 1.f;
  return dtype == DT_F32 ? rotary_launch<float>(p, interleaved, stream) : rotary_launch<bf16_t>(p, interleaved, stream);
}
