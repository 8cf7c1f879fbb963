// int4.cuh — the 4-bit rows of a paged key/value cache.
// A row of dh columns is cut into groups of 64.  A group holds its minimum m and the scale
// s = (maximum - m) / 15, both rounded to the rows' 16-bit type, and codes c = rint((x - m) / s) in 0..15:
// x is read as s c + m, off by s / 2 (and by 15 times the scale's rounding at the upper end).
// Groups of 64 cost half a bit a column; of 32 they would cost a whole one, for a step 17% smaller on
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

// The code word and the group's (s, m) of 8 columns in each lane; lanes 8 i .. 8 i + 7 hold a group, and all 32
// lanes of the warp take part.  A group with a NaN or an infinity gets s = m = NaN, one whose range passes the
// type's gets s = inf: both read as NaN.
template <typename T>
__device__ __forceinline__ void int4_pack(const uint4& raw, uint32_t& word, uint32_t& pair) {
  const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = ElemTraits<T>::unpack2(u[i]);
    x[2 * i] = p.x;
    x[2 * i + 1] = p.y;
  }
  float lo = x[0], hi = x[0];
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    finite &= fabsf(x[i]) < INFINITY;
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const int lane = threadIdx.x & 31;
  const bool good = ((__ballot_sync(0xffffffffu, finite) >> (lane & 24)) & 255u) == 255u;
  const float m = good ? lo : __int_as_float(0x7fc00000);
  pair = ElemTraits<T>::pack2(good ? __fdiv_rn(hi - lo, 15.f) : m, m);
  const float s = ElemTraits<T>::unpack2(pair).x;
  word = 0;
  if (s > 0.f && s < INFINITY) {
#pragma unroll
    for (int i = 0; i < 8; ++i) word |= (uint32_t)fminf(rintf(__fdiv_rn(x[i] - m, s)), 15.f) << (4 * i);
  }
}

// Column i (0..7) of a code word, read with its group's (s, m).
__device__ __forceinline__ float int4_value(uint32_t word, int i, float2 pair) {
  return fmaf((float)((word >> (4 * i)) & 15u), pair.x, pair.y);
}

}  // namespace bna
