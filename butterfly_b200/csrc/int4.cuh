// int4.cuh — the 4-bit rows of a paged key/value cache.
// A row of dh columns is cut into groups of 64.  A group holds its minimum m and the scale
// s = (maximum - m) / 15, both rounded to the rows' 16-bit type, and codes c = rint((x - m) / s) in 0..15:
// x is read as s c + m, off by s / 2 (and by 15 times the scale's rounding at the upper end).
// Groups of 64 cost half a bit a column; of 32 they would cost a whole one, for a step 12% smaller on
// normal data.
//
// 16 tokens of a head lie together in a block of 18 dh bytes, so that a granule's keys and values are one
// contiguous read: key codes [16][dh / 2], key (s, m) pairs [16][dh / 64], and the same of the values.
// Code word (8 codes, the first in the lowest bits) g * groups + y of a row holds columns
// 64 y + 8 g .. + 7: the lanes g of a matrix fragment then find the same part of every group side by side.
#pragma once
#include "common.cuh"

namespace bna {

constexpr int kInt4Group = 64;   // columns that share a scale
constexpr int kInt4Tokens = 16;  // tokens of a block
__host__ __device__ constexpr int int4_half_bytes(int dh) { return 9 * dh; }  // keys or values of a block
__host__ __device__ constexpr int int4_block_bytes(int dh) { return 18 * dh; }
// Byte offsets in a half: the code word of columns 8 c .. 8 c + 7, and the (s, m) pair of their group.
__device__ __forceinline__ int int4_word_at(int dh, int token, int c) { return token * (dh / 2) + 4 * ((c & 7) * (dh / 64) + (c >> 3)); }
__device__ __forceinline__ int int4_pair_at(int dh, int token, int c) { return 8 * dh + 4 * (token * (dh / 64) + (c >> 3)); }

// Two columns in a register: the smaller and the larger of each half (NaN if either is), one half alone, and both negated.
template <typename T> struct Pair16;
template <> struct Pair16<__nv_bfloat16> {
  using V = __nv_bfloat162;
  static constexpr float kTiny = 0x1p-100f;  // scales below this are divided by
};
template <> struct Pair16<__half> {
  using V = __half2;
  static constexpr float kTiny = 0x1p-14f;  // (subnormal: rounding one may leave codes above 15)
};
template <typename T>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  using V = typename Pair16<T>::V;
  const V r = __hmin2_nan(*reinterpret_cast<V*>(&a), *reinterpret_cast<V*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  using V = typename Pair16<T>::V;
  const V r = __hmax2_nan(*reinterpret_cast<V*>(&a), *reinterpret_cast<V*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// (a, b) of lower halves as the two halves
__device__ __forceinline__ uint32_t lower2(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The smallest column and minus the largest, as the two halves, of N registers of columns in each of L lanes side by
// side (L a power of two; the lanes of the mask take part).  NaN where a column is.
template <typename T, int N, int L>
__device__ __forceinline__ uint32_t int4_extremes(const uint32_t (&u)[N]) {
  uint32_t lo = u[0], hi = u[0];
#pragma unroll
  for (int i = 1; i < N; ++i) {
    lo = min2<T>(lo, u[i]);
    hi = max2<T>(hi, u[i]);
  }
  // (lower halves, upper halves) of both, the largest negated
  uint32_t e = min2<T>(lower2(lo, hi ^ 0x80008000u), __byte_perm(lo, hi ^ 0x80008000u, 0x7632));
#pragma unroll
  for (int o = 1; o < L; o <<= 1) e = min2<T>(e, __shfl_xor_sync(0xffffffffu, e, o));
  return e;
}

// A group's (s, m) from its extremes.  With a NaN or an infinity s = m = NaN; where the range passes the type's s = inf.
template <typename T>
__device__ __forceinline__ uint32_t int4_pair(uint32_t extremes) {
  const float2 e = ElemTraits<T>::unpack2(extremes);
  const bool good = e.x > -INFINITY && e.y > -INFINITY;  // (neither NaN nor infinite: e.x <= -e.y)
  const float m = good ? e.x : __int_as_float(0x7fc00000);
  return ElemTraits<T>::pack2(good ? __fdiv_rn(-e.y - m, 15.f) : m, m);
}

// The code word of 8 columns (4 registers): rint(d / s) of each difference d = x - m, ties to even, 15 at most; 0 for
// all where s is not a positive number.
// c = rint(d r) with r a little below 1 / s (by more than its own error) is the code, or the one below it where d / s lies
// at a tie or 15 2^-21 above one.  The residual e = d - c s tells: it is exact (both terms are multiples of the
// smaller one's last place, and no more than 24 bits of it apart), so e = s / 2 means a tie, and rint(c + 1 / 2) is
// its even code; e > s / 2, the next code, needs a difference that was rounded.  Ties are common in bf16
// data (one value in 450 of a normal sample; in fp16 one in 3,600), so they take no branch.  Columns i and i + 4 go as a pair.
template <typename T>
__device__ __forceinline__ uint32_t int4_codes(const uint32_t* u, float2 sm) {
  const float s = sm.x, m = sm.y;
  if (!(s > 0.f && s < INFINITY)) return 0;
  Two d[4], c[4];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float2 a = halves_plus<T>(u[j], -m), b = halves_plus<T>(u[2 + j], -m);
    d[2 * j] = two(a.x, b.x);
    d[2 * j + 1] = two(a.y, b.y);
  }
  if (s < Pair16<T>::kTiny) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = apart(d[i]);
      c[i] = two(fminf(rintf(__fdiv_rn(x.x, s)), 15.f), fminf(rintf(__fdiv_rn(x.y, s)), 15.f));
    }
  } else {  // (the scale is off by 2^-9 of itself at most: no code passes 15)
    constexpr float kRint = 0x1.8p23f;  // adding it rounds to an integer
    const float r = rcp_approx(s) * (1.f - 0x1p-21f), h = 0.5f * s;
    const Two r2 = two(r, r), s2 = two(-s, -s), up = two(kRint, kRint), down = two(-kRint, -kRint), half = two(0.5f, 0.5f);
    float worst = -1.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const Two t = fma2(d[i], r2, up);
      const float2 e = apart(fma2(add2(t, down), s2, d[i]));
      worst = fmax3(worst, e.x, e.y);
      c[i] = add2(fma2(two(e.x >= h ? 1.f : 0.f, e.y >= h ? 1.f : 0.f), half, t), down);
    }
    if (worst > h) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Two t = add2(fma2(d[i], r2, up), down);
        const float2 k = apart(t), e = apart(fma2(t, s2, d[i])), even = apart(c[i]);
        c[i] = two(e.x > h ? k.x + 1.f : even.x, e.y > h ? k.y + 1.f : even.y);
      }
    }
  }
  const Two by = two(16.f, 16.f);  // the sums' last 16 bits are the codes
  const float2 w = apart(add2(fma2(fma2(fma2(c[3], by, c[2]), by, c[1]), by, c[0]), two(0x1p23f, 0x1p23f)));
  return lower2(__float_as_uint(w.x), __float_as_uint(w.y));
}

// The code word and the group's (s, m) of 8 columns in each lane; lanes 8 i .. 8 i + 7 hold a group, and all 32
// lanes of the warp take part.
template <typename T>
__device__ __forceinline__ void int4_pack(const uint4& raw, uint32_t& word, uint32_t& pair) {
  const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
  pair = int4_pair<T>(int4_extremes<T, 4, 8>(u));
  word = int4_codes<T>(u, ElemTraits<T>::unpack2(pair));
}

// Column i (0..7) of a code word, read with its group's (s, m).
__device__ __forceinline__ float int4_value(uint32_t word, int i, float2 pair) {
  return fmaf((float)((word >> (4 * i)) & 15u), pair.x, pair.y);
}

}  // namespace bna
