// paged_decode_int4.cu — attention of one new token per request over a paged cache held in 4 bits (int4.cuh).
//   s_j = scale * q . k_j   for keys j in [max(0, len - window), len)
//   out = sum_j softmax(s)_j v_j,   lse = log sum_j exp(s_j);  no key: out = 0, lse = -inf
// With x = s c + m per group y of 64 columns both products are taken on the codes, which are exact in 16 bits:
//   q . k_j = sum_y  sk_jy (q_y . ck_jy) + mk_jy sum(q_y)
//   out     = sum_j  (p_j sv_jy) cv_jy + sum_j p_j mv_jy
// so nothing is rounded in undoing the quantisation; the scales work on fp32 scores and probabilities.
//
// Tensor-core form (m16n8k16, 16 keys x up to 8 query heads): S^T = C_k Q^T and O^T = C_v^T P^T.  A code
// c masked in place in a 16-bit half of a code word is the fp16 subnormal 2^-24 c, or 2^-20 c for the
// odd code beside it, so a code word becomes four operand registers with five integer instructions and
// no conversion.  q is scaled by a power of two into the fp16 range (by head; exact but for entries 2^-23 of
// the head's largest), and 2^-4 of that meets the odd codes.
//
// Bytes: 18 dh / 16 a token and head.  A read serves up to 8 query heads (16 at head_dim 64 and 128 with more than 8).
//
// Schedule: the keys of every pair (request, KV head) in granules of 16 form one line, which is cut evenly over
// the CTAs.  A cut that falls within kSlack granules of a pair's end moves there, so that short pairs stay whole;
// of a pair that is cut each CTA leaves a part in the workspace, and a second kernel joins the parts.  Every warp
// copies its granules into a ring of its own by cp.async and waits for nobody until a pair ends.
//
// Warp-level matrix instructions, as their operand is made in registers: the fifth-generation ones read it from shared
// or tensor memory, where the unpacked codes would be four times the bytes that came, written and read once more.
// p sv is held in fp16 in a unit of its head and column group, in which the largest product so far is 2^(kLeast - 1) or more: what
// falls below fp16's 2^-24 is lost against the group's own sum.
// Half of the keys enter P V as 15 - c with scale -s and minimum m + 15 s, so that what the tensor core cuts off its
// sums cancels.
//
// Measured at 1,965 MHz: 64 requests of 65,536 tokens, 8 / 2 heads of 128, bf16: 215 us for 1.21 GB, 5.6 TB/s (0.86 of a copy; the
// 16-bit kernel takes 610 us for its 4.3 GB; one unit for all groups and heads, which lost small ones, 211 us); call after call, under the
// power cap at 1,700 MHz, 236 to 252 us.  Bound by the instructions of a
// granule as much as by HBM.  One request of 131,072 tokens: 18.3 us, some 4 of them before the first keys and 4 in the join.  4 requests of 37 to 513 tokens: 10 us, latency.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "int4.cuh"
#include "mma.cuh"
#include "sm100.cuh"

namespace bna {
namespace {
using namespace sm100;

constexpr int kGran = kInt4Tokens;  // keys of a granule: a block
constexpr int kMaxCtas = 320;       // the workspace is sized for this many
constexpr int kWarps = 8, kThreads = 32 * kWarps;
// Granules within which a cut moves to the end of its pair, and of the longest pair up to which none is cut where there
// are pairs enough or the table has room for no longer one.  A cut costs its parts' way through memory and the
// join, some 4 us.  2 heads of 128, slack 10 / 20 / 40: one request of 2,500 tokens 10.1 / 10.0 / 12.2 us, 8 of
// 4,000 13.2 / 12.6 / 16.0.  Whole / cut: 64 requests of 1,200 tokens with a table for no more 10.5 / 15.8 us
// (with one for 4,000 17.7 / 15.9), 128 of 1,250 and 4 heads 33.0 / 36.0, one of 1,000 (table 2,000) 11.0 / 9.4.
constexpr int kSlack = 20, kWhole = 80;
// Granules a CTA gets at least of a cut line (fewer CTAs otherwise); 16 / 32: one request of 20,000 tokens 12.1 / 10.5 us,
// of 6,000 10.0 / 10.1.
constexpr int kMinShare = 32;
constexpr int kKeepLens = 1024;  // lengths kept in shared memory
constexpr int kShift = 11;  // probabilities are held times 2^kShift, and so are l and o; the divisions undo it
constexpr float kMove = 4.f;  // a reference moves when a score lies more than that above it
// A new unit of products is 2^kRoom times the largest scale or more, so that ones up to 2^(kRoom - 1) times as large need no other,
// but leaves the largest product at 2^kLeast or more, however large the scales of keys without weight are.
constexpr int kRoom = 3, kLeast = 3;
constexpr float kNone = 0x1.fffffep127f;  // `add` of a reference that has seen no key: any score moves it, however low

struct Int4Args {
  const uint8_t* q;
  int64_t q_b, q_h;
  uint8_t* pool;
  int64_t p_p, p_h, p_g;  // byte strides: page, head, block
  const uint8_t *kn, *vn;  // the new token's rows, or null
  int64_t kn_b, kn_h, vn_b, vn_h;
  const uint8_t* active;  // requests that have a new row (null: all)
  uint8_t* out;
  int64_t o_b, o_h;
  float* lse;
  int64_t ls_b, ls_h;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  int B, Hkv, G, width, num_pages, page_size, window;
  int page_grans, page_shift;  // blocks of a page, and their log2 (or -1)
  int whole;               // one pair a CTA
  int chunks, chunk_rows;  // the G heads in `chunks` groups of chunk_rows
  float scale_log2;
  uint8_t* ws;
};

// Workspace: (the first 4 KB belong to the 16-bit kernel and stay zero), a record of the cut pair that begins in each
// CTA, (m, l) of every part, their outputs.  CTA c has the slots 2 c and 2 c + 1: the pair that ends in it, and the one that begins.
constexpr int kPartRows = 16;
struct CutPair {
  int b, h, r0, rows_parts;  // rows and, from bit 8 on, parts (0: no cut pair begins in the CTA)
};
constexpr int64_t kWsCut = 4096;
constexpr int64_t kWsMl = kWsCut + kMaxCtas * (int64_t)sizeof(CutPair);
constexpr int64_t kWsO = kWsMl + (int64_t)2 * kMaxCtas * kPartRows * 8;
constexpr int kPartFloats = 2048;  // a part has 8 rows of 256 or 16 of 128 at most
constexpr int64_t kWsBytes = kWsO + (int64_t)2 * kMaxCtas * kPartFloats * 4;

__device__ __forceinline__ int first_key(const Int4Args& a, int len) { return a.window > 0 ? max(0, len - a.window) : 0; }
__device__ __forceinline__ int clamp_len(const Int4Args& a, int len) {
  return (int)min((int64_t)max(len, 0), (int64_t)a.width * a.page_size);
}
__device__ __forceinline__ int granules_of(const Int4Args& a, int len) {
  return len == 0 ? 0 : (len + kGran - 1) / kGran - first_key(a, len) / kGran;
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int AT, int N>  // N words of 32 bits at `AT` bytes past addr
__device__ __forceinline__ void lds(uint32_t addr, uint32_t (&r)[N]) {
  static_assert(N == 1 || N == 2 || N == 4 || N == 8, "");
  if constexpr (N == 1) {
    asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(r[0]) : "r"(addr), "n"(AT) : "memory");
  } else if constexpr (N == 2) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2+%3];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr), "n"(AT) : "memory");
  } else {
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4+%5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr), "n"(AT)
                 : "memory");
    if constexpr (N == 8)
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4+%5];"
                   : "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                   : "r"(addr), "n"(AT + 16)
                   : "memory");
  }
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
// D = A B for one m16n8k16 tile of fp16 (mma_16816 without a sum to start from)
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// 8x8 matrix of 16-bit entries, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
constexpr int kMaxExp = 126;
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ int exponent(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }  // of x >= 0 (0: -127)
__device__ __forceinline__ float lane_max(float x) {  // over the lanes with the same lane % 4
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
}
__device__ __forceinline__ float lane_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 4);
  x += __shfl_xor_sync(0xffffffffu, x, 8);
  return x + __shfl_xor_sync(0xffffffffu, x, 16);
}
// Both halves of a register as floats.  bf16: by the adder that takes 16-bit terms, as the integer pipe, which
// would shift and mask, is the busiest one here (64 x 65,536 tokens: 241 -> 233 us).
template <typename T>
__device__ __forceinline__ float2 halves(uint32_t w) {
  return std::is_same<T, __half>::value ? ElemTraits<T>::unpack2(w) : halves_plus<T>(w, 0.f);
}
// (m, l) with l times 2^kShift
__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.f ? -INFINITY : (m + log2f(l) - (float)kShift) * 0.6931471805599453f;
}

// A stretch of a (request, KV head, head group) inside a CTA: granules [g0, g0 + n), keys attended to [lo, hi).
struct Seg {
  int b, h, r0, rows, g0, n, lo, hi, slot;  // slot of the part (-1: the whole pair)
};

// ROWS: query heads served together at most: 4, 8 or 16
template <typename T_, int DH_, int ROWS>
struct Form {
  using T = T_;
  static constexpr int DH = DH_;
  static constexpr int kTiles = ROWS > 8 ? 2 : 1;  // of 8 columns
  static constexpr int kHeads = 8 * kTiles;
  // For fp16 results a probability times the scale is held as two fp16 parts: one would add as much error to the output
  // as its final rounding does (for bf16 ones an eighth of it).  With up to 4 heads the low parts ride in
  // columns 4-7, with more they take products of their own.
  static constexpr bool kTwoParts = std::is_same<T, __half>::value && ROWS > 4, kLowColumns = std::is_same<T, __half>::value && ROWS <= 4;
  // For bf16 results with up to 4 heads two granules share the columns: all 8 get the same queries, and of the scores
  // lanes t < 2 keep the first granule's, the others the second one's.  What follows on scores and probabilities is then done once
  // for both, and the two halves' sums meet as the warps join: 64 x 65,536 tokens 240 -> 209 us, 64 of 1,200 10.5 -> 9.5, one of
  // 131,072 18.8 -> 19.2.  (fp16, whose columns hold low parts, gains nothing by products for those instead: 84 us on 13
  // requests to 262,144 either way.)
  static constexpr bool kPaired = std::is_same<T, __nv_bfloat16>::value && ROWS <= 4;
  static constexpr int kStep = kPaired ? 2 : 1;  // granules at a time
  // two CTAs an SM where their registers fit, so that the end of one's pair overlaps the other's reads
  static constexpr int kCtas = ROWS > 8 || DH == 256 ? 1 : 2;
  static constexpr int GR = DH / kInt4Group;
  static constexpr int kBlock = int4_block_bytes(DH);
  // (paired with 4 / 5 / 6 slots: 64 x 65,536 tokens 211 / 216 / 217 us)
  static constexpr int kStages = kPaired ? 4 : DH == 256 ? 5 : ROWS > 8 ? 8 : 4;  // granules of a warp's ring
  static constexpr int kRing = kStages * kBlock;
  static_assert(kStages % kStep == 0, "a pair of granules lies side by side");
  static constexpr int kPitch = DH + 4;  // floats of a row, as the warps join
  static_assert(kHeads * kPitch * 4 <= kRing, "a warp's outputs take its ring's place");
  static constexpr int kMl = kWarps * kRing;                   // (m, l) [warp][head]
  static constexpr int kRuns = kMl + kWarps * kHeads * 8;      // granules up to the end of each thread's run of requests
  static constexpr int kLens = kRuns + kThreads * 4;
  static constexpr int kBytes = kLens + 4 * kKeepLens;
  static_assert(kCtas * (kBytes + 1024 + 256) <= 233472, "shared memory of an SM (1 KB a CTA is the system's, and some static)");
};

// What a warp holds of a segment.  Scores come as S^T: lane 4 g + t has two keys, row(g) and row(g) + 4, and heads 2 t,
// 2 t + 1 (of every tile).  Matrix row g is key row(g) = g / 2 + 8 (g % 2), so that lane t's keys in P V are t, t + 8 and t + 4,
// t + 12: one address and fixed offsets, two lanes to a bank.  Outputs o come as O^T: columns 64 y + 8 g .. + 7 of
// heads 2 t, 2 t + 1.
template <class F>
struct Acc {
  using T = typename F::T;
  static constexpr int GR = F::GR, NT = F::kTiles, DH = F::DH;
  uint32_t qb[NT][GR][2][2][2];  // Q^T fragments: tile, group, word of the lane, step, register
  float qs[NT][GR][2];           // sum(q_y), scaled as the products with codes are
  float f[NT][2];                // from those to scores in the exp2 domain
  float ref[NT][2], add[NT][2];  // running reference (no score lies kMove above it), and kShift less it
  float l[NT][2], wm[NT][GR][2];  // this lane's keys: sum p, sum p mv_y
  float o[NT][GR][4][4];          // sum p sv cv, in units of 2^-24 (odd columns 2^-20) 2^k
  // 2^-k of each head and group.  The unit follows the group's largest product p sv, also down as the reference moves, so that what is
  // lost below fp16's range is lost against the column's own sum, whatever scales other groups, keys without
  // weight or other heads have.
  float inv[NT][GR][2];

  // This lane's part of the queries.  q: the head group's first row; rows from `rows` on count as zeros
  struct Queries {
    uint4 raw[NT][GR][2];
    __device__ __forceinline__ void load(const uint8_t* q, int64_t q_h, int rows, int lane) {
      const int g = F::kLowColumns || F::kPaired ? (lane >> 2) & 3 : lane >> 2, t = lane & 3;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int y = 0; y < GR; ++y)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            raw[n][y][j] = g + 8 * n < rows ? ld_nc_128(q + 2 * ((g + 8 * n) * q_h + 64 * y + 16 * t + 8 * j)) : make_uint4(0, 0, 0, 0);
    }
  };
  __device__ __forceinline__ void begin(const Queries& from, float scale_log2, int lane) {
    const int t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint4(&raw)[GR][2] = from.raw[n];
      float top = 0.f;
#pragma unroll
      for (int y = 0; y < GR; ++y)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t u[4] = {raw[y][j].x, raw[y][j].y, raw[y][j].z, raw[y][j].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 p = ElemTraits<T>::unpack2(u[i]);
            top = fmaxf(top, fmaxf(fabsf(p.x), fabsf(p.y)));
          }
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = min(max(140 - (int)(__float_as_uint(top) >> 23), -100), 120);  // the largest in [2^13, 2^14)
      const float up = pow2(e);
      float sums[GR];
#pragma unroll
      for (int y = 0; y < GR; ++y) {
        sums[y] = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t u[4] = {raw[y][j].x, raw[y][j].y, raw[y][j].z, raw[y][j].w};
          float x[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 p = ElemTraits<T>::unpack2(u[i]);
            x[2 * i] = p.x * up;
            x[2 * i + 1] = p.y * up;
            sums[y] += x[2 * i] + x[2 * i + 1];
          }
          // the codes of a word meet as (0, 4), 2^4 (1, 5), (2, 6), 2^4 (3, 7)
#pragma unroll
          for (int st = 0; st < 2; ++st) {
            qb[n][y][j][st][0] = ElemTraits<__half>::pack2(x[2 * st], x[2 * st + 4]);
            qb[n][y][j][st][1] = ElemTraits<__half>::pack2(x[2 * st + 1] * 0.0625f, x[2 * st + 5] * 0.0625f);
          }
        }
        sums[y] += __shfl_xor_sync(0xffffffffu, sums[y], 1);
        sums[y] += __shfl_xor_sync(0xffffffffu, sums[y], 2);
        sums[y] *= 0x1p-24f;
      }
      // (never 0, which would make a masked score of -inf a NaN: small queries, or none, under a small scale)
      const float down = fmaxf(pow2(min(24 - e, 124)) * scale_log2, 0x1p-126f);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int src = 4 * (2 * t + x);
        f[n][x] = __shfl_sync(0xffffffffu, down, src);
#pragma unroll
        for (int y = 0; y < GR; ++y) {
          qs[n][y][x] = __shfl_sync(0xffffffffu, sums[y], src);
          wm[n][y][x] = 0.f;
          inv[n][y][x] = pow2(kMaxExp);
        }
        ref[n][x] = -INFINITY;
        add[n][x] = kNone;
        l[n][x] = 0.f;
      }
#pragma unroll
      for (int y = 0; y < GR; ++y)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[n][y][i][x] = 0.f;
    }
  }

  // A granule in shared memory, its first key at `pos`; with `edge` keys outside [lo, hi) are masked.  Paired: also the
  // one at `second`; `pos` is that of the lane's granule.
  __device__ __forceinline__ void granule(uint32_t tile, uint32_t second, int pos, bool edge, int lo, int hi, int lane) {
    constexpr uint32_t M0 = 0x000f000fu, M1 = 0x00f000f0u;
    const int g = lane >> 2, t = lane & 3;
    const int row = (g >> 1) + 8 * (g & 1);
    const uint32_t own = F::kPaired && t >= 2 ? second : tile;  // the granule of the lane's scores
    // scores
    float u[NT][4];
    {
      float acc[GR][NT][4];
      uint32_t p[2][GR];
#pragma unroll
      for (int x = 0; x < F::kStep; ++x) {
        const uint32_t from = x == 0 ? tile : second;
        uint32_t w[2][2 * GR];
        lds<0>(from + row * (DH / 2) + t * (8 * GR), w[0]);
        lds<4 * (DH / 2)>(from + row * (DH / 2) + t * (8 * GR), w[1]);
        if (x == 0) {
          lds<8 * DH>(own + row * (4 * GR), p[0]);
          lds<8 * DH + 16 * GR>(own + row * (4 * GR), p[1]);
        }
#pragma unroll
        for (int y = 0; y < GR; ++y) {
          float c[NT][4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t a0 = w[0][j * GR + y], a1 = w[1][j * GR + y];
            const uint32_t even[4] = {a0 & M0, a1 & M0, a0 & M1, a1 & M1};
            const uint32_t odd[4] = {(a0 >> 8) & M0, (a1 >> 8) & M0, (a0 >> 8) & M1, (a1 >> 8) & M1};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if (j == 0) mma_first(c[n], even, qb[n][y][j][0][0], qb[n][y][j][0][1]);
              else mma_16816<__half>(c[n], even, qb[n][y][j][0][0], qb[n][y][j][0][1]);
              mma_16816<__half>(c[n], odd, qb[n][y][j][1][0], qb[n][y][j][1][1]);
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[y][n][i] = x == 0 || t >= 2 ? c[n][i] : acc[y][n][i];
        }
      }
#pragma unroll
      for (int y = 0; y < GR; ++y)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float2 sm = halves<T>(p[r][y]);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float base = y == 0 ? sm.y * qs[n][y][x] : fmaf(sm.y, qs[n][y][x], u[n][2 * r + x]);
              u[n][2 * r + x] = fmaf(sm.x, acc[y][n][2 * r + x], base);
            }
        }
    }
    float sv[2][GR], mv[2][GR];
    {
      uint32_t p[2][GR];
      lds<17 * DH>(own + row * (4 * GR), p[0]);
      lds<17 * DH + 16 * GR>(own + row * (4 * GR), p[1]);
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int y = 0; y < GR; ++y) {
          const float2 sm = halves<T>(p[r][y]);
          sv[r][y] = sm.x;
          mv[r][y] = r == 0 ? sm.y : fmaf(15.f, sm.x, sm.y);
        }
    }
    if (edge) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int key = pos + row + 4 * r;
        if (key < lo || key >= hi) {
#pragma unroll
          for (int n = 0; n < NT; ++n) u[n][2 * r] = u[n][2 * r + 1] = -INFINITY;
#pragma unroll
          for (int y = 0; y < GR; ++y) sv[r][y] = mv[r][y] = 0.f;  // what the page holds there could be NaN
        }
      }
    }
    // probabilities times 2^kShift, and their products with the scales, in the units held
    float e[NT][4], w[NT][GR][4], most = -INFINITY, top = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int y = 0; y < GR; ++y) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float2 v = apart(mul2(two(sv[r][y], sv[r][y]), two(inv[n][y][0], inv[n][y][1])));
          w[n][y][2 * r] = v.x;
          w[n][y][2 * r + 1] = v.y;
        }
        top = fmax3(fmax3(top, w[n][y][0], w[n][y][1]), w[n][y][2], w[n][y][3]);
      }
      // The scores are rounded before the reference is taken off, here and in a move: from 2^27 on their roundings are above 2^kMove, and
      // equal ones must stay equal.  (A packed product and sum would be made one operation.)
#pragma unroll
      for (int x = 0; x < 4; ++x) e[n][x] = __fadd_rn(__fmul_rn(f[n][x & 1], u[n][x]), add[n][x & 1]);
      most = fmax3(most, fmaxf(e[n][0], e[n][1]), fmaxf(e[n][2], e[n][3]));
    }
    // without a move no product is above 2^(kShift + kMove) = 2^15
    const bool move = __any_sync(0xffffffffu, top > 1.f || most > kShift + kMove);
    if (move) {
      int high[GR];  // of the largest scale
#pragma unroll
      for (int y = 0; y < GR; ++y) high[y] = exponent(lane_max(fmaxf(sv[0][y], sv[1][y])));
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float s0 = __fmul_rn(f[n][x], u[n][x]), s1 = __fmul_rn(f[n][x], u[n][2 + x]), mx = fmaxf(ref[n][x], lane_max(fmaxf(s0, s1)));
          const float to = mx == -INFINITY ? kNone : (float)kShift - mx, by = to - add[n][x], al = ex2_approx(by);
          // (differences of whole parts: many small moves take the unit as far as one large one)
          const int less = (int)fmaxf(ceilf(to) - ceilf(add[n][x]), -4.f * kMaxExp);
          ref[n][x] = mx;
          add[n][x] = to;
          l[n][x] *= al;
          const float e0 = s0 + to, e1 = s1 + to;
          e[n][x] = ex2_approx(e0);
          e[n][2 + x] = ex2_approx(e1);
#pragma unroll
          for (int y = 0; y < GR; ++y) {
            wm[n][y][x] *= al;
            // the largest product's exponent, or one less
            const float largest = lane_max(fmaxf(e0 + (float)exponent(sv[0][y]), e1 + (float)exponent(sv[1][y])));
            const int old = -exponent(inv[n][y][x]);
            const int k = min(max(max(old + less, min(high[y] + kRoom, (int)floorf(fmaxf(largest, -4.f * kMaxExp)) - kLeast)), -kMaxExp), kMaxExp);
            const float scale = ex2_approx(by + (float)(old - k));
            inv[n][y][x] = pow2(-k);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              o[n][y][i][x] *= scale;
              o[n][y][i][2 + x] *= scale;
            }
            // (in this order: a scale by 2^-k might overflow under a probability of 0)
            w[n][y][x] = e[n][x] * sv[0][y] * inv[n][y][x];
            w[n][y][2 + x] = e[n][2 + x] * sv[1][y] * inv[n][y][x];
          }
        }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float(&p)[4] = e[n];
          p[2 * r] = ex2_approx(p[2 * r]);
          p[2 * r + 1] = ex2_approx(p[2 * r + 1]);
#pragma unroll
          for (int y = 0; y < GR; ++y) {
            const float2 v = apart(mul2(two(w[n][y][2 * r], w[n][y][2 * r + 1]), two(p[2 * r], p[2 * r + 1])));
            w[n][y][2 * r] = v.x;
            w[n][y][2 * r + 1] = v.y;
          }
        }
    }
    uint32_t pb[NT][GR][2], pl[NT][GR][2];  // P^T sv fragments: high parts, and low ones for fp16 results
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int x = 0; x < 2; ++x) l[n][x] += e[n][x] + e[n][2 + x];
#pragma unroll
      for (int y = 0; y < GR; ++y) {
#pragma unroll
        for (int x = 0; x < 2; ++x) wm[n][y][x] = fmaf(e[n][x], mv[0][y], fmaf(e[n][2 + x], mv[1][y], wm[n][y][x]));
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float w0 = r == 0 ? w[n][y][0] : -w[n][y][2], w1 = r == 0 ? w[n][y][1] : -w[n][y][3];
          uint32_t part = ElemTraits<__half>::pack2(w0, w1), low = 0;
          if (F::kTwoParts || F::kLowColumns) {
            const float2 h = ElemTraits<__half>::unpack2(part);
            low = ElemTraits<__half>::pack2(w0 - h.x, w1 - h.y);
          }
          if (F::kLowColumns && t >= 2) part = low;
          pb[n][y][r] = transposed(part);
          if (F::kTwoParts) pl[n][y][r] = transposed(low);
        }
      }
    }
    // outputs
#pragma unroll
    for (int z = 0; z < F::kStep; ++z) {
      uint32_t c[4][GR];
      const uint32_t at = (z == 0 ? tile : second) + t * (DH / 2) + g * (4 * GR);
      lds<9 * DH>(at, c[0]);
      lds<9 * DH + 8 * (DH / 2)>(at, c[1]);
      lds<9 * DH + 4 * (DH / 2)>(at, c[2]);
      lds<9 * DH + 12 * (DH / 2)>(at, c[3]);
      const bool here = !F::kPaired || (lane >= 16) == (z == 1);  // the granule's columns
#pragma unroll
      for (int y = 0; y < GR; ++y) {
        uint32_t b[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) b[n][r] = here ? pb[n][y][r] : 0u;
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // columns 0-3, then 4-7 of the word, of a pair of keys each
          uint32_t x0 = __byte_perm(c[0][y], c[1][y], half ? 0x7632 : 0x5410), x1 = __byte_perm(c[2][y], c[3][y], half ? 0x7632 : 0x5410);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t a[4] = {x0 & M0, x0 & M1, ~x1 & M0, ~x1 & M1};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_16816<__half>(o[n][y][2 * half + i], a, b[n][0], b[n][1]);
              if (F::kTwoParts) mma_16816<__half>(o[n][y][2 * half + i], a, pl[n][y][0], pl[n][y][1]);
            }
            x0 >>= 8;
            x1 >>= 8;
          }
        }
      }
    }
  }

  // Sums over the warp; o becomes the output over this warp's keys alone (0 without any).
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        l[n][x] = lane_sum(l[n][x]);
        const float d = l[n][x] == 0.f ? 0.f : 1.f / l[n][x];
#pragma unroll
        for (int y = 0; y < GR; ++y) {
          const float m = lane_sum(wm[n][y][x]) * d;
          const float unit = __uint_as_float((254u << 23) - __float_as_uint(inv[n][y][x]));  // 2^k
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (F::kLowColumns) {
              o[n][y][i][x] += __shfl_xor_sync(0xffffffffu, o[n][y][i][x], 2);
              o[n][y][i][2 + x] += __shfl_xor_sync(0xffffffffu, o[n][y][i][2 + x], 2);
            }
            o[n][y][i][x] = fmaf(o[n][y][i][x] * (d * 0x1p24f), unit, m);
            o[n][y][i][2 + x] = fmaf(o[n][y][i][2 + x] * (d * 0x1p20f), unit, m);
          }
        }
      }
  }
  // Columns 64 y + 8 g .. + 7 of head 8 n + 2 t + x
  __device__ __forceinline__ void columns(int n, int y, int x, float (&c)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[2 * i] = o[n][y][i][x];
      c[2 * i + 1] = o[n][y][i][2 + x];
    }
  }
};

// Granules up to the end of each thread's run of requests, cut evenly over C CTAs (the first U % C get one more).
struct Line {
  const int* runs;
  int per, per_b, U, C, q, r, slack;

  __device__ int raw(int c) const { return c * q + min(c, r); }
  __device__ int cta_of(int x) const {  // whose raw stretch holds x
    const int wide = r * (q + 1);
    return x < wide ? x / (q + 1) : r + (x - wide) / max(q, 1);
  }
};
// A request's place on the line, and the granules of each of its pairs.
struct At {
  int b, nt, begin;
};

template <class F>
__global__ void __launch_bounds__(kThreads, F::kCtas) int4_decode_kernel(const __grid_constant__ Int4Args a) {
  using T = typename F::T;
  constexpr int DH = F::DH, GR = F::GR;
  extern __shared__ __align__(128) uint8_t sm[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per_b = a.Hkv * a.chunks;
  int* lens = reinterpret_cast<int*>(sm + F::kLens);
  auto len_of = [&](int b) { return b < kKeepLens ? lens[b] : clamp_len(a, a.lens[b]); };
  Line line{reinterpret_cast<const int*>(sm + F::kRuns), (a.B + kThreads - 1) / kThreads, per_b, 0, 1, 0, 0, kSlack};
  At at{0, 0, 0};
  int cur = 0, end = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (!a.whole) {
    // ---- the line
    __shared__ int warp_sums[kWarps];
    int* runs = reinterpret_cast<int*>(sm + F::kRuns);
    int mine = 0, pairs = 0, longest = 0;
    for (int b = tid * line.per; b < min((tid + 1) * line.per, a.B); ++b) {
      const int len = clamp_len(a, a.lens[b]), nt = granules_of(a, len);
      if (b < kKeepLens) lens[b] = len;
      mine += nt;
      pairs += nt > 0;
      longest = max(longest, nt);
    }
    mine *= per_b;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    pairs = __reduce_add_sync(0xffffffffu, pairs) * per_b;
    longest = __reduce_max_sync(0xffffffffu, longest);
    __shared__ int warp_pairs[kWarps], warp_longest[kWarps];
    if (lane == 31) {
      warp_sums[warp] = incl;
      warp_pairs[warp] = pairs;
      warp_longest[warp] = longest;
    }
    __syncthreads();
    pairs = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) incl += warp_sums[w];
      pairs += warp_pairs[w];
      longest = max(longest, warp_longest[w]);
    }
    runs[tid] = incl;
    __syncthreads();
    line.U = runs[kThreads - 1];
    // A CTA for every kMinShare granules, or for every pair, where that is more.  Where all pairs are short, and enough
    // for every CTA, cuts move to the nearest end however far it is.
    const bool whole = longest <= kWhole && pairs >= (int)gridDim.x;
    line.C = min((int)gridDim.x, max(1, max(pairs, (line.U + kMinShare - 1) / kMinShare)));
    line.slack = whole ? kWhole : kSlack;
    line.q = line.U / line.C;
    line.r = line.U - line.q * line.C;
    auto locate = [&](int x) {  // of a place before U: the warp whose runs reach past it, the run, the request
      const int w = __popc(__ballot_sync(0xffffffffu, lane < kWarps && line.runs[32 * (lane & (kWarps - 1)) + 31] <= x));
      const int i = 32 * w + __popc(__ballot_sync(0xffffffffu, line.runs[32 * w + lane] <= x));
      At r{i * line.per, 0, i > 0 ? line.runs[i - 1] : 0};
      for (;; ++r.b) {
        r.nt = granules_of(a, r.b < a.B ? len_of(r.b) : 0);
        if (r.b >= a.B - 1 || r.begin + r.nt * per_b > x) return r;
        r.begin += r.nt * per_b;
      }
    };
    if ((int)blockIdx.x < line.C) {
      // both ends of the stretch, moved to the nearest end of their pair where that is close
#pragma unroll 1
      for (int i = 1; i >= 0; --i) {
        int x = line.raw((int)blockIdx.x + i);
        if (x < line.U) {
          at = locate(x);
          if (x > 0) {
            const int t = (x - at.begin) % max(at.nt, 1), rest = at.nt - t;
            x = t <= line.slack && t <= rest ? x - t : rest <= line.slack ? x + rest : x;
          }
        }
        if (i == 1) end = x;
        else cur = x;
      }
    }
  } else {
    // ---- one pair a CTA, none of them long enough to be cut: nothing to find out but its length
    at.b = (int)blockIdx.x / per_b;
    const int len = clamp_len(a, a.lens[at.b]);
    at.nt = granules_of(a, len);
    cur = ((int)blockIdx.x - at.b * per_b) * at.nt;
    end = cur + at.nt;
  }
  CutPair begun{};

  // ---- the pairs of this CTA's stretch
  const uint32_t ring = smem_u32(sm) + warp * F::kRing;
  float2* ml = reinterpret_cast<float2*>(sm + F::kMl);
  while (cur < end) {
    while (cur >= at.begin + at.nt * per_b && at.b + 1 < a.B) {  // (requests without keys are passed over)
      at.begin += at.nt * per_b;
      ++at.b;
      at.nt = granules_of(a, len_of(at.b));
    }
    const int local = cur - at.begin;
    if (at.nt == 0 || local >= at.nt * per_b) break;  // (only where lengths changed under the call)
    const int pair = local / at.nt, t0 = local - pair * at.nt;
    const int len = a.whole ? clamp_len(a, a.lens[at.b]) : len_of(at.b);
    Seg s;
    s.b = at.b;
    s.h = pair / a.chunks;
    s.r0 = (pair - s.h * a.chunks) * a.chunk_rows;
    s.rows = min(a.chunk_rows, a.G - s.r0);
    s.lo = first_key(a, len);
    s.hi = len;
    s.g0 = s.lo / kGran + t0;
    s.n = min(at.nt - t0, end - cur);
    s.slot = s.n == at.nt ? -1 : 2 * (int)blockIdx.x + (t0 == 0 ? 1 : 0);
    if (s.slot >= 0 && t0 == 0) {
      // A cut pair begins here: its parts are those of the CTAs up to the one that holds its end.  Cuts within it kept their
      // places (those near its end have moved there): the last of them lies at or before this place.
      const int last = min(max((int)blockIdx.x + 1, line.cta_of(cur + at.nt - line.slack - 1)), line.C - 1);
      begun = CutPair{s.b, s.h, s.r0, s.rows | (last - (int)blockIdx.x + 1) << 8};
    }
    cur += s.n;

    // this warp's granules: warp, warp + kWarps, ...
    const int mine = (s.n - warp + kWarps - 1) / kWarps;
    const int32_t* table = a.table + s.b * a.table_stride;
    auto block_at = [&](int gr) -> uint8_t* {  // where the request's granule gr lies (null: its page is outside the pool)
      const int pi = a.page_shift >= 0 ? gr >> a.page_shift : gr / a.page_grans, page = table[pi];
      return page >= 0 && page < a.num_pages ? a.pool + page * a.p_p + s.h * a.p_h + (gr - pi * a.page_grans) * a.p_g : nullptr;
    };
    auto look_up = [&](int k0) -> const uint8_t* {  // lane i: granule i of a batch of 32
      const int k = k0 + lane;
      return k < mine ? block_at(s.g0 + warp + k * kWarps) : nullptr;
    };
    const uint8_t *batch = look_up(0), *next = look_up(32);
    typename Acc<F>::Queries queries;
    queries.load(a.q + 2 * (s.b * a.q_b + (int64_t)(s.h * a.G + s.r0) * a.q_h), a.q_h, s.rows, lane);
    // The new token's row, if this warp gets its granule (the request's last): packed, for the granule and, once where
    // several head groups share it, for its page.
    constexpr int kNew = (2 * (DH / 8) + 31) / 32;
    uint32_t new_word[kNew], new_pair[kNew];
    const bool owns_new = a.kn && s.g0 + s.n == (s.hi + kGran - 1) / kGran && (s.n - 1) % kWarps == warp && (!a.active || a.active[s.b]);
    auto new_at = [&](int i, int& word, int& pair) {  // byte offsets in the block of what the lane has of it; false: none
      const int x = 32 * i + lane, c = x % (DH / 8), half = x >= DH / 8 ? int4_half_bytes(DH) : 0, token = (s.hi - 1) % kGran;
      word = half + int4_word_at(DH, token, c);
      pair = (c & 7) == 0 ? half + int4_pair_at(DH, token, c) : -1;
      return x < 2 * (DH / 8);
    };
    if (owns_new) {
      uint8_t* block = s.r0 == 0 ? block_at((s.hi - 1) / kGran) : nullptr;
#pragma unroll
      for (int i = 0; i < kNew; ++i) {
        const int x = 32 * i + lane, c = x % (DH / 8);
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (x < DH / 8) raw = ld_128(a.kn + 2 * (s.b * a.kn_b + s.h * a.kn_h) + 16 * c);
        else if (x < 2 * (DH / 8)) raw = ld_128(a.vn + 2 * (s.b * a.vn_b + s.h * a.vn_h) + 16 * c);
        int4_pack<T>(raw, new_word[i], new_pair[i]);
        int word, pair;
        if (new_at(i, word, pair) && block) {
          *reinterpret_cast<uint32_t*>(block + word) = new_word[i];
          if (pair >= 0) *reinterpret_cast<uint32_t*>(block + pair) = new_pair[i];
        }
      }
    }
    auto issue = [&](int k) {
      if ((k & 31) == 0 && k > 0) {
        batch = next;
        next = look_up(k + 32);
      }
      if (k < mine) {
        const uint8_t* src = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(batch), k & 31));
        const uint32_t dst = ring + (k % F::kStages) * F::kBlock + 16 * lane;
        if (src) {
          src += 16 * lane;
#pragma unroll
          for (int i = 0; i < F::kBlock / 512; ++i) cp_async_16(dst + 512 * i, src + 512 * i);
          if (F::kBlock % 512 && lane < F::kBlock % 512 / 16) cp_async_16(dst + F::kBlock / 512 * 512, src + F::kBlock / 512 * 512);
        } else {  // a page outside the pool reads as zeros
          for (int i = lane; i < F::kBlock / 16; i += 32) sts128(dst + 16 * (i - lane), make_uint4(0, 0, 0, 0));
        }
      }
      cp_async_commit();  // (a group for every granule, empty ones past the end)
    };
    constexpr int kAhead = F::kStages - F::kStep;  // granules in flight beside those at hand
#pragma unroll 1
    for (int k = 0; k < kAhead; ++k) issue(k);
    Acc<F> acc;
    acc.begin(queries, a.scale_log2, lane);
#pragma unroll 1
    for (int k = 0; k < mine; k += F::kStep) {
#pragma unroll
      for (int i = 0; i < F::kStep; ++i) issue(k + kAhead + i);
      cp_async_wait<kAhead>();
      __syncwarp();
      int pos = (s.g0 + warp + k * kWarps) * kGran;
      bool edge = pos < s.lo || pos + kGran > s.hi;
      const uint32_t tile = ring + (k % F::kStages) * F::kBlock, second = tile + F::kBlock;
      if (F::kPaired) {
        // without a second granule the slot's scores are those of keys behind the last one
        const bool two = k + 1 < mine;
        const int other = two ? pos + kWarps * kGran : s.hi;
        edge = edge || !two || other + kGran > s.hi;
        pos = lane & 2 ? other : pos;
      }
      if (owns_new && k + F::kStep >= mine) {
        const uint32_t slot = F::kPaired && k + 1 < mine ? second : tile;
#pragma unroll
        for (int i = 0; i < kNew; ++i) {
          int word, pair;
          if (new_at(i, word, pair)) {
            sts32(slot + word, new_word[i]);
            if (pair >= 0) sts32(slot + pair, new_pair[i]);
          }
        }
        __syncwarp();
      }
      acc.granule(tile, second, pos, edge, s.lo, s.hi, lane);
      __syncwarp();  // the slots have been read
    }
    acc.finish();

    // ---- the warps' results joined: each leaves (m, l) and its outputs in its ring's place
    const int g = lane >> 2, t = lane & 3;
    cp_async_wait<0>();
    __syncwarp();
#pragma unroll
    for (int n = 0; n < F::kTiles; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = 8 * n + 2 * t + x;
        if ((F::kPaired ? r & 3 : r) >= s.rows) continue;
        if (g == 0) ml[warp * F::kHeads + r] = make_float2(acc.ref[n][x], acc.l[n][x]);
        float* dst = reinterpret_cast<float*>(sm + warp * F::kRing) + r * F::kPitch;
#pragma unroll
        for (int y = 0; y < GR; ++y) {
          float c[8];
          acc.columns(n, y, x, c);
          *reinterpret_cast<float4*>(dst + 64 * y + 8 * g) = make_float4(c[0], c[1], c[2], c[3]);
          *reinterpret_cast<float4*>(dst + 64 * y + 8 * g + 4) = make_float4(c[4], c[5], c[6], c[7]);
        }
      }
    __syncthreads();
    for (int it = tid; it < s.rows * (DH / 4); it += kThreads) {
      const int r = it / (DH / 4), c = it % (DH / 4) * 4;
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < F::kStep * kWarps; ++w) M = fmaxf(M, ml[w / F::kStep * F::kHeads + r + w % F::kStep * 4].x);
      const float base = M == -INFINITY ? 0.f : M;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < F::kStep * kWarps; ++w) {  // (paired: rows r and r + 4 of each warp)
        const int at = w / F::kStep, row = r + w % F::kStep * 4;
        const float2 x = ml[at * F::kHeads + row];
        const float4 y = *reinterpret_cast<const float4*>(sm + at * F::kRing + 4 * (row * F::kPitch + c));
        const float p = x.y * ex2_approx(x.x - base);
        L += p;
        v.x = fmaf(y.x, p, v.x);
        v.y = fmaf(y.y, p, v.y);
        v.z = fmaf(y.z, p, v.z);
        v.w = fmaf(y.w, p, v.w);
      }
      const float d = L == 0.f ? 0.f : 1.f / L;
      v = make_float4(v.x * d, v.y * d, v.z * d, v.w * d);
      if (s.slot < 0) {
        const int64_t hq = s.h * a.G + s.r0 + r;
        *reinterpret_cast<uint2*>(a.out + 2 * (s.b * a.o_b + hq * a.o_h + c)) =
            make_uint2(ElemTraits<T>::pack2(v.x, v.y), ElemTraits<T>::pack2(v.z, v.w));
        if (a.lse && c == 0) a.lse[s.b * a.ls_b + hq * a.ls_h] = lse_of(M, L);
      } else {
        *reinterpret_cast<float4*>(a.ws + kWsO + 4 * ((int64_t)s.slot * kPartFloats + r * DH + c)) = v;
        if (c == 0) reinterpret_cast<float2*>(a.ws + kWsMl)[s.slot * kPartRows + r] = make_float2(M, L);
      }
    }
    if (cur < end) __syncthreads();  // the rings are free again
  }
  // for the join: the cut pair that begins in this CTA, if one does (else it has no parts)
  if (!a.whole && tid == 0) reinterpret_cast<CutPair*>(a.ws + kWsCut)[blockIdx.x] = begun;
  auto no_keys = [&](int b) {
    const int hq = a.Hkv * a.G;
    for (int i = tid; i < hq * (DH / 8); i += kThreads)
      st_128(a.out + 2 * (b * a.o_b + (int64_t)(i / (DH / 8)) * a.o_h) + 16 * (i % (DH / 8)), make_uint4(0, 0, 0, 0));
    if (a.lse)
      for (int i = tid; i < hq; i += kThreads) a.lse[b * a.ls_b + i * a.ls_h] = -INFINITY;
  };
  if (a.whole) {
    if (at.nt == 0 && (int)blockIdx.x == at.b * per_b) no_keys(at.b);
  } else {
    for (int b = blockIdx.x; b < a.B; b += gridDim.x)
      if (len_of(b) == 0) no_keys(b);
  }
}

// Head blockIdx.y of the blockIdx.x-th cut pair: its parts' outputs, weighted and summed in the order of the line.  A
// warp takes every kWarps-th part, BATCH at a time, and asks for the first ones before it knows their weights;
// the weights of part i are in lane i % 32 of every warp.
// A launch of its own, as a CTA that waited for the others' parts would hold its SM meanwhile.  Bound by latency: the launch and two
// reads that depend on one another (the records, then weights and outputs).
template <typename T, int DH, int BATCH>
__global__ void __launch_bounds__(kThreads) int4_join_kernel(const __grid_constant__ Int4Args a, int ctas) {
  constexpr int kPer = kMaxCtas / 32;      // parts a lane has the weights of
  constexpr int kMine = kMaxCtas / kWarps;  // parts of a warp
  constexpr int V = DH / 32;  // columns of a lane
  __shared__ float sums[kWarps][DH];
  __shared__ CutPair found;
  __shared__ int found_cta, before[2 * kWarps];
  static_assert(kMaxCtas <= 2 * kThreads && kMine % BATCH == 0, "");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = blockIdx.y;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // the pair's record among those of all CTAs
  CutPair mine[2];
  unsigned some[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int c = k * kThreads + tid;
    mine[k] = c < ctas ? reinterpret_cast<const CutPair*>(a.ws + kWsCut)[c] : CutPair{};
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    some[k] = __ballot_sync(0xffffffffu, mine[k].rows_parts != 0);
    if (lane == 0) before[k * kWarps + warp] = __popc(some[k]);
  }
  if (tid == 0) found_cta = -1;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    int at = __popc(some[k] & ((1u << lane) - 1));
    for (int w = 0; w < k * kWarps + warp; ++w) at += before[w];
    if (mine[k].rows_parts != 0 && at == (int)blockIdx.x) {
      found = mine[k];
      found_cta = k * kThreads + tid;
    }
  }
  __syncthreads();
  const int first = found_cta;
  const CutPair p = found;
  const int rows = p.rows_parts & 255, parts = p.rows_parts >> 8;
  if (first < 0 || r >= rows) return;
  auto slot = [&](int i) { return 2 * (first + i) + (i == 0 ? 1 : 0); };
  const float2* ml = reinterpret_cast<const float2*>(a.ws + kWsMl) + r;
  const float* o = reinterpret_cast<const float*>(a.ws + kWsO) + r * DH + V * lane;
  float2 x[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) x[k] = 32 * k + lane < parts ? ml[slot(32 * k + lane) * kPartRows] : make_float2(-INFINITY, 0.f);
  float u[BATCH][V], v[V];
  auto fetch = [&](int j0) {
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const int i = (j0 + j) * kWarps + warp;
      if (i >= parts) break;
      const float* src = o + (int64_t)slot(i) * kPartFloats;
      if constexpr (V == 2) *reinterpret_cast<float2*>(u[j]) = *reinterpret_cast<const float2*>(src);
      else
#pragma unroll
        for (int c = 0; c < V; c += 4) *reinterpret_cast<float4*>(u[j] + c) = *reinterpret_cast<const float4*>(src + c);
    }
  };
  fetch(0);
  float M = -INFINITY, L = 0.f;
#pragma unroll
  for (int k = 0; k < kPer; ++k) M = fmaxf(M, x[k].x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
  const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    x[k].x = x[k].y * ex2_approx(x[k].x - base);
    L += x[k].x;
  }
  L = warp_sum(L);
#pragma unroll
  for (int c = 0; c < V; ++c) v[c] = 0.f;
#pragma unroll
  for (int j0 = 0; j0 < kMine; j0 += BATCH) {
    if (j0 * kWarps >= parts) break;
    if (j0 > 0) fetch(j0);
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const int i = (j0 + j) * kWarps + warp;  // part i: lane i % 32, its weight i / 32
      const float w = __shfl_sync(0xffffffffu, x[(j0 + j) * kWarps / 32].x, (j0 + j) * kWarps % 32 + warp);
      if (i < parts)
#pragma unroll
        for (int c = 0; c < V; ++c) v[c] = fmaf(u[j][c], w, v[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < V; ++c) sums[warp][V * lane + c] = v[c];
  __syncthreads();
  const float d = L == 0.f ? 0.f : 1.f / L;
  const int64_t hq = p.h * a.G + p.r0 + r;
  if (tid < DH / 2) {
    float y[2] = {0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      y[0] += sums[w][2 * tid];
      y[1] += sums[w][2 * tid + 1];
    }
    *reinterpret_cast<uint32_t*>(a.out + 2 * (p.b * a.o_b + hq * a.o_h + 2 * tid)) = ElemTraits<T>::pack2(y[0] * d, y[1] * d);
  }
  if (a.lse && tid == 0) a.lse[p.b * a.ls_b + hq * a.ls_h] = lse_of(M, L);
}

template <class K, class... Args>
int launch_dependent(K kern, dim3 grid, int smem, cudaStream_t s, const char* what, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, args...), what);
}

template <class F>
int launch(const Int4Args& a, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};  // devices (bits) whose kernel has its shared memory allowed
  static std::atomic<int> sms[64];
  int dev = 0;
  cudaGetDevice(&dev);
  int n = dev < 64 ? sms[dev].load() : 0;
  if (n == 0 || !(ready.load() >> dev & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(int4_decode_kernel<F>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kBytes);
    if (e != cudaSuccess) return check_cuda(e, "paged_decode_int4 attributes");
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (dev < 64) {
      sms[dev].store(n);
      ready.fetch_or(1ull << dev);
    }
  }
  const int64_t keys = a.window > 0 ? std::min((int64_t)a.width * a.page_size, (int64_t)a.window + 2 * kGran) : (int64_t)a.width * a.page_size;
  const int64_t longest = (keys + kGran - 1) / kGran, pairs = (int64_t)a.B * a.Hkv * a.chunks;
  if (pairs > INT_MAX / longest) return fail(BNA_UNSUPPORTED, "paged_decode_int4: requests x heads x tokens of a table row beyond 2^35");
  Int4Args b = a;
  b.whole = longest <= kWhole;
  // No more CTAs than there could be pairs or shares.
  const int64_t most = std::max(pairs, (pairs * longest + kMinShare - 1) / kMinShare);
  const int grid = (int)(b.whole ? pairs : std::min<int64_t>(std::min(n * F::kCtas, kMaxCtas), most));
  if (int rc = launch_dependent(int4_decode_kernel<F>, dim3(grid), F::kBytes, s, "paged_decode_int4 launch", b)) return rc;
  if (b.whole || grid == 1) return BNA_OK;
  // A cut pair begins in each CTA at most, and there are no more of them than pairs.
  const dim3 joins((unsigned)std::min<int64_t>(grid, pairs), (unsigned)a.chunk_rows);
  // Few pairs have many parts each, and then fewer rounds are faster (one request of 131,072 tokens, 2 heads of 128: 18.8 us against
  // 20.3); else the longer code and its registers cost more than they give (64 of 1,200: 17.3 against 16.1).
  constexpr int kMany = F::DH == 256 ? 10 : 20;
  const auto join = grid >= 64 * pairs ? int4_join_kernel<typename F::T, F::DH, kMany> : int4_join_kernel<typename F::T, F::DH, 8>;
  return launch_dependent(join, joins, 0, s, "paged_decode_int4 join launch", b, grid);
}

}  // namespace

int64_t paged_decode_int4_workspace_bytes() { return kWsBytes; }

int launch_paged_decode_int4(const bna_tensor4* q, bna_tensor4* pool, const bna_tensor4* kn, const bna_tensor4* vn, const uint8_t* active,
                             bna_tensor4* out, float* lse, int64_t ls_b, int64_t ls_h, int dtype, const int32_t* table,
                             int64_t table_stride, int width, const int32_t* lens, int window, float scale, void* ws, cudaStream_t s) {
  Int4Args a{};
  a.q = static_cast<const uint8_t*>(q->data);
  a.q_b = q->stride[0], a.q_h = q->stride[1];
  a.pool = static_cast<uint8_t*>(pool->data);
  a.p_p = pool->stride[0], a.p_h = pool->stride[1], a.p_g = pool->stride[2];
  if (kn) {
    a.kn = static_cast<const uint8_t*>(kn->data), a.vn = static_cast<const uint8_t*>(vn->data);
    a.active = active;
    a.kn_b = kn->stride[0], a.kn_h = kn->stride[1], a.vn_b = vn->stride[0], a.vn_h = vn->stride[1];
  }
  a.out = static_cast<uint8_t*>(out->data);
  a.o_b = out->stride[0], a.o_h = out->stride[1];
  a.lse = lse, a.ls_b = ls_b, a.ls_h = ls_h;
  a.table = table, a.table_stride = table_stride, a.lens = lens;
  const int dh = (int)q->size[3];
  a.B = (int)q->size[0], a.Hkv = (int)pool->size[1], a.G = (int)(q->size[1] / pool->size[1]);
  a.width = width, a.num_pages = (int)pool->size[0], a.page_grans = (int)pool->size[2], a.page_size = a.page_grans * kGran, a.window = window;
  const int most_rows = dh == 256 ? 8 : 16;
  a.page_shift = (a.page_grans & (a.page_grans - 1)) == 0 ? __builtin_ctz((unsigned)a.page_grans) : -1;
  a.chunks = (a.G + most_rows - 1) / most_rows;
  a.chunk_rows = (a.G + a.chunks - 1) / a.chunks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.ws = static_cast<uint8_t*>(ws);
  const int rows = a.chunk_rows;
  auto pick = [&](auto form) {
    constexpr int DH = decltype(form)::DH;
    if (dtype == BNA_BF16) {
      if constexpr (DH < 256)
        if (rows > 8) return launch<Form<__nv_bfloat16, DH, 16>>(a, s);
      return rows > 4 ? launch<Form<__nv_bfloat16, DH, 8>>(a, s) : launch<Form<__nv_bfloat16, DH, 4>>(a, s);
    }
    if constexpr (DH < 256)
      if (rows > 8) return launch<Form<__half, DH, 16>>(a, s);
    return rows > 4 ? launch<Form<__half, DH, 8>>(a, s) : launch<Form<__half, DH, 4>>(a, s);
  };
  switch (dh) {
    case 64: return pick(Form<__half, 64, 8>());
    case 128: return pick(Form<__half, 128, 8>());
    case 256: return pick(Form<__half, 256, 8>());
    default: return fail(BNA_UNSUPPORTED, "paged_decode_attention_int4: head_dim must be 64, 128 or 256");
  }
}

}  // namespace bna
