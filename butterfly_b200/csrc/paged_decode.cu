// paged_decode.cu — attention of one new token per request over a paged key/value cache.
//   s_j = scale * q . k_j   for keys j in [max(0, len - window), len)
//   out = sum_j softmax(s)_j v_j,   lse = log sum_j exp(s_j);  no key: out = 0, lse = -inf
// One pass over the keys with a running maximum m, sum l and output o; a set of keys cut into
// parts is joined by  M = max m_i,  L = sum l_i 2^(m_i - M),  out = sum o_i 2^(m_i - M) / L
// (m in the exp2 domain).
//
// Each key and value is read once and serves the G = Hq / Hkv query heads of its KV head (more than 16
// in chunks of equal size, each of which reads them: 16 requests of 16,384 tokens, 2 KV heads of
// 128, take 56.5 us with 16 query heads per KV head and 93.3 us with 32): 2 G FLOP per byte,
// far below the tensor cores' balance, so the kernel is bound by HBM and is built to keep its
// reads in flight:
//   * The keys of a pair (request, KV head) come in granules of 16.  One persistent CTA per SM (two
//     at head_dim 64) takes either whole pairs, as they are claimed (in turn, if all are short), or, where single pairs
//     are long beside an even share, an equal stretch of the line of all granules: one long
//     request spreads over all SMs, and only its parts have to be joined.
//   * The producer warp looks the pages up and issues one TMA tile copy for a granule's keys and
//     one for its values into a ring of granule slots (128 KB an SM); it runs ahead into the
//     next pairs.
//   * Eight consumer warps (four at head_dim 64 and 256) take the granules in turn, each with its own m,
//     l and o in registers: no barrier between warps until a pair, or a CTA's part of it, ends.
//   * Of a pair cut by CTA boundaries each CTA leaves a part in the workspace, and the CTA that
//     arrives last joins the parts in their order on the line (of many, groups first).  Every sum has its order fixed by
//     the lengths and the grid, whichever CTA runs when: equal calls give equal bits.
// Measured (GPU time, bf16, 8 / 2 heads of 128): 64 x 65,536 tokens 610 us = 7.0 TB/s (a copy reaches
// 6.45 TB/s here), DRAM reads equal to the keys and values, tensor pipe 17% busy; one request of
// 131,072 tokens 34.4 us = 3.9 TB/s: 4 us until the first granule, 19 to 22 us of reads, 7 us from
// the last CTA's arrival through two rounds of joins; four requests of 37 to 513 tokens 9.1 us,
// a chain of dependent reads (lengths, pages, keys) and one pass of the code.
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <map>
#include <mutex>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "mma.cuh"
#include "ring.cuh"
#include "sm100.cuh"

namespace bna {
int* device_error_word();

namespace {
using namespace sm100;

constexpr int kGran = 16;       // keys of a granule
constexpr int kMaxSms = 160;    // the workspace is sized for this many, with two CTAs each
constexpr int kMaxCtas = 2 * kMaxSms;
constexpr int kRows = 16;       // query heads of one KV head served together
constexpr int kMinPart = 16;    // granules a CTA gets at least of an even cut (fewer CTAs otherwise)
constexpr int kFan = 16;        // parts of a pair joined at a time; up to kFan + 4 where that is all
constexpr int kKeepLens = 1024;  // lengths kept in shared memory, once read
constexpr int kLanes = 8;       // producer lanes that issue copies side by side
constexpr int kErrSite = 0x40;  // device error sites of this file

struct PagedArgs {
  const uint8_t* q;
  int64_t q_b, q_h;
  uint8_t *kp, *vp;
  int64_t kp_p, kp_h, kp_t, vp_p, vp_h, vp_t;
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
  int page_shift;          // log2(page_size), or -1
  int chunks, chunk_rows;  // the G heads in `chunks` groups of chunk_rows <= kRows
  float scale_log2;
  uint8_t* ws;
  int* err;
};

// Workspace: counters (zero between calls: pairs claimed, arrivals at a pair by its first CTA, at a
// group of its parts by the first one's slot),
// (m, l) of every part, then the outputs.
constexpr int64_t kWsMl = 4096;
constexpr int64_t kWsO = kWsMl + (int64_t)2 * kMaxCtas * kRows * 8;
constexpr int64_t kWsBytes = kWsO + (int64_t)2 * kMaxCtas * kRows * 256 * 4;
static_assert(4 * (3 * kMaxCtas + 1) <= kWsMl && kMaxCtas <= kFan * (kFan + 4), "counters, rounds");

// One stretch of a (request, KV head, head group) inside a CTA.
struct Seg {
  int b, h, r0, rows;  // request, KV head, first query head of the group (within G) and their count
  int g0, n;           // granules (16-key blocks of the request) [g0, g0 + n); n < 0: no more
  int lo, hi;          // keys attended to
  int first_cta, parts, slot;  // parts of a cut pair, the CTA of the first one, this part's slot (-1: uncut)
};

template <int DH>
struct Layout {
  // CTAs of an SM, and consumer warps of a CTA.  head_dim 64: two CTAs of four warps, so that the end
  // of one's pair overlaps the other's reads (96 x 3 pairs of up to 1,000 keys: 22 us with
  // one of eight).  head_dim 256: four warps, as the output and score registers of eight
  // would not fit beside each other.
  static constexpr int kCtas = DH == 64 ? 2 : 1;
  static constexpr int kCons = DH == 128 ? 8 : 4;
  static constexpr int kThreads = 32 * (kCons + 1);      // and the producer
  static constexpr int kSlotBytes = 2 * kGran * DH * 2;  // keys, then values
  // 128 KB of ring an SM keeps the memory busy; with 192 KB requests queue and the SMs that a loaded
  // GPU serves last fall further behind (640 against 615 us at 64 x 65,536 tokens).
  static constexpr int kSlots = 128 * 1024 / kCtas / kSlotBytes;
  // Every consumer warp has slots of its own (ring.cuh).  Granule i of a segment goes to warp
  // i % kCons, whatever came before it, so that the segment's sums do not depend on that.
  using Uses = Ring<kCons, kSlots>;
  static constexpr int kQPitch = 2 * DH + 16;                         // spreads the rows over the banks
  static constexpr int kQBytes = kRows * kQPitch;
  static constexpr int kQ = kSlots * kSlotBytes;
  static constexpr int kBuf = kQ + 2 * kQBytes;
  // merge of the warps: 16 rows x 32 columns, 8 x 64 or 4 x 128 (rows padded by 8 floats), or
  // the weights and partial sums of a join
  static constexpr int kMergeFloats = kCons * kRows * (32 + 8), kJoinFloats = 32 * kRows + 4 * 32 * kCons;
  static constexpr int kBufBytes = 4 * (kMergeFloats > kJoinFloats ? kMergeFloats : kJoinFloats);
  static constexpr int kStage = kBuf + 2 * kBufBytes;  // (segments alternate between two buffers)
  static constexpr int kHalf = (kCtas == 2 ? 8 : 20) * 1024;  // parts of a join arrive in two halves of this size
  static constexpr int kMl = kStage + 2 * kHalf;
  static constexpr int kBars = kMl + 2 * kCons * kRows * 8;
  static constexpr int kNumBars = 2 * kSlots + 6;
  static constexpr int kSeg = kBars + kNumBars * 8;
  static constexpr int kFlags = kSeg + 2 * (int)sizeof(Seg);
  static constexpr int kIssued = kFlags + 16;  // the log of tile copies
  static constexpr int kLens = (kIssued + 4 * kSlots + 15) / 16 * 16;  // the first kKeepLens requests' lengths
  static constexpr int kBytes = kLens + 4 * kKeepLens;
  static constexpr int kAlloc = kBytes + 1024;  // the base is aligned to 1024 (swizzle atom)
  static_assert(kCtas * (kAlloc + 1024) <= 233472, "shared memory of an SM");
};

__device__ __forceinline__ int clamp_len(const PagedArgs& a, int len) {
  return (int)min((int64_t)max(len, 0), (int64_t)a.width * a.page_size);
}
__device__ __forceinline__ int first_key(const PagedArgs& a, int len) {
  return a.window > 0 ? max(0, len - a.window) : 0;
}
__device__ __forceinline__ int granules_of(const PagedArgs& a, int len) {
  return len == 0 ? 0 : (len + kGran - 1) / kGran - first_key(a, len) / kGran;
}

// 64-bit quotient of non-negative numbers, by the 32-bit division wherever both fit.
__device__ __forceinline__ int64_t quot(int64_t x, int64_t y) {
  return (uint64_t)(x | y) >> 32 == 0 ? (int64_t)((uint32_t)x / (uint32_t)y) : x / y;
}

// U granules over C CTAs: the first U % C take one more.
struct Cut {
  int64_t q = 1, r = 0;
  __device__ void set(int64_t U, int64_t C) {
    q = quot(U, C);
    r = U - q * C;
  }
  __device__ int64_t start(int64_t c) const { return c * q + min(c, r); }
  __device__ int cta_of(int64_t x) const {  // the CTA that holds granule x
    const int64_t wide = r * (q + 1);
    return (int)(x < wide ? quot(x, q + 1) : r + quot(x - wide, q));
  }
};

// Offset of 16-byte chunk c of row r in a granule tile: 64-column boxes of 16 rows x 128 bytes,
// 128-byte swizzle.
__device__ __forceinline__ uint32_t tile_off(int r, int c) {
  return (uint32_t)((c >> 3) * (kGran * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

template <typename T>
__device__ __forceinline__ void store4(uint8_t* p, const float4& v, float f) {
  *reinterpret_cast<uint2*>(p) = make_uint2(ElemTraits<T>::pack2(v.x * f, v.y * f), ElemTraits<T>::pack2(v.z * f, v.w * f));
}
// Probabilities are held times 2^kShift, and so are the sums l and outputs o, which the final division
// undoes.  fp16 has steps of 2^-24 below 2^-14: unscaled, with the row's largest at 1, what lies 17
// nats below it would vanish from the output (but not from l).  At 2^15 (the largest still fits, the
// sums are fp32) the steps are 2^-39 of it.
template <typename T>
constexpr float kShift = std::is_same<T, __half>::value ? 15.f : 0.f;
template <typename T>
__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.f ? -INFINITY : (m + log2f(l * (std::is_same<T, __half>::value ? 0x1p-15f : 1.f))) * 0.6931471805599453f;
}

// Barrier of the consumer warps.  Every path of every warp between two of them ends by itself
// (waits for copies are bounded), so none waits for good.
template <int THREADS>
__device__ __forceinline__ void cons_sync() { named_bar_sync(1, THREADS); }
// The same, and whether any thread came with `bad`.
template <int THREADS>
__device__ __forceinline__ bool cons_any(bool bad) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, 1, %2, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)bad), "n"(THREADS)
      : "memory");
  return any != 0;
}

// WIDE: 9 to 16 query heads, the rows of the 16-row MMA.  Otherwise the heads are rows 0-7, and rows
// 8-15 of the P V product carry the low part of the probabilities.  A probability is held
// as hi + lo in the 16-bit type, scaled (kShift; relative error u^2 instead of u: rounding it once would add
// as much error to the output as its final rounding does); with at most 8 heads lo rides in rows
// that the MMA computes anyway, with more it costs a second MMA, which the memory hides.  The MMA
// cuts its fp32 sums off instead of rounding them, some hundreds of steps a warp and part: of 64
// requests with 65,536 tokens 0.37% of the bf16 results (2.1% in fp16) are the neighbours of the
// correctly rounded ones, of 400 tokens 0.12% (0.19%); fp32 arithmetic gives 0.06% (0.48%).
template <typename T, int DH, bool WIDE>
__global__ void __launch_bounds__(Layout<DH>::kThreads, Layout<DH>::kCtas)
    paged_decode_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const PagedArgs a) {
  using Lay = Layout<DH>;
  using Uses = typename Lay::Uses;
  constexpr int kCons = Lay::kCons;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + Lay::kBars);
  uint64_t* empty = full + Lay::kSlots;
  uint64_t* seg_full = empty + Lay::kSlots;
  uint64_t* seg_empty = seg_full + 2;
  uint64_t* stage_full = seg_empty + 2;
  Seg* segs = reinterpret_cast<Seg*>(sm + Lay::kSeg);
  volatile int* abort_flag = reinterpret_cast<int*>(sm + Lay::kFlags);
  volatile int* last_flag = abort_flag + 1;
  int* issued = reinterpret_cast<int*>(sm + Lay::kIssued);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // full and empty (one arrival), seg_full (one), seg_empty (each consumer warp), stage_full (one)
  for (int i = threadIdx.x; i < Lay::kNumBars; i += Lay::kThreads) {
    const int k = i - 2 * Lay::kSlots;
    mbar_init(full + i, k == 2 || k == 3 ? kCons : 1);
    fence_mbar_init();
    if (i < Lay::kSlots) issued[i] = 0;
  }
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    prefetch_tmap(&mk);
    prefetch_tmap(&mv);
  }
  __syncthreads();
  // every input may come from the previous kernel of the stream; the next one may be set up
  // once that kernel is done
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  auto wait = [&](uint64_t* bar, uint32_t parity, int site) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, kErrSite + site, a.err));
  };
  // Wait for a copy that is in flight, whatever went wrong elsewhere (20 ms at most): none may land in
  // the shared memory of a CTA that has ended.
  auto settle = [&](uint64_t* bar, uint32_t parity) {
    for (int tries = 0; tries < 1000; ++tries)
      if (mbar_try_wait_suspend(bar, parity, 20000u)) break;
  };

  if (warp == kCons) {
    // ------------------------------------------------------------------ producer
    const int per_b = a.Hkv * a.chunks;
    const int64_t grid = gridDim.x;
    int* lens = reinterpret_cast<int*>(sm + Lay::kLens);
    // The first claim of a pair goes out before it is known whether there is one to take: with
    // all CTAs claiming at once the answer takes 3 us.
    int* claims = reinterpret_cast<int*>(a.ws);
    int claim = lane == 0 ? atomicAdd(claims, 1) : 0;
    int64_t U = 0, N = 0;  // granules, and pairs that have any
    int longest = 0;
    auto count = [&](int len) {
      const int nt = granules_of(a, len);
      U += nt;
      N += nt > 0;
      longest = max(longest, nt);
    };
    for (int i0 = lane; i0 < a.B; i0 += 256) {  // eight loads in flight
      int len[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) len[x] = i0 + 32 * x < a.B ? a.lens[i0 + 32 * x] : 0;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        len[x] = clamp_len(a, len[x]);
        if (i0 + 32 * x < kKeepLens) lens[i0 + 32 * x] = len[x];
        count(len[x]);
      }
    }
    __syncwarp();
    if (__all_sync(0xffffffffu, U < 1 << 26)) {
      U = __reduce_add_sync(0xffffffffu, (unsigned)U);
    } else {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) U += __shfl_xor_sync(0xffffffffu, U, o);
    }
    N = __reduce_add_sync(0xffffffffu, (unsigned)N);
    longest = __reduce_max_sync(0xffffffffu, longest);
    U *= per_b;
    N *= per_b;
    // Whole pairs or an even cut?  In granules of work the fullest CTA gets the longest pair, or
    // an even share and about half a pair more; cutting costs the parts' way through memory
    // and their join, about 10 us, in which the SM could have read kCut granules.  Measured
    // whole / cut: 96 x 3 pairs of up to 1,000 keys (head_dim 64) 15 / 24 us; at head_dim 128, 256
    // pairs of 2,048 keys 47 / 50 us and 16 pairs of 2,048 keys 18 / 11 us.
    constexpr int kCut = 8192 / DH / Lay::kCtas;
    const float share = (float)U * __frcp_rn((float)grid), even = fmaxf(share, (float)kMinPart) + (float)kCut;
    const bool whole = (N <= grid ? (float)longest : share + 0.5f * (float)longest) <= even;
    // items: the pairs, or the stretches of C CTAs
    const int64_t C = whole ? N : max((int64_t)1, min(grid, quot(U + kMinPart - 1, kMinPart)));
    Cut cut;
    if (!whole) cut.set(U, C);

    // The line that items are cut from: granules, or whole pairs.  Window of 32 requests (lane i:
    // request wb + i): length, its stretch of the line, and the line up to that stretch's end.
    int wb = 0, len_w = 0;
    int64_t mine_w = 0, incl_w = 0, before = 0;
    auto load_window = [&]() {
      const int i = wb + lane;
      len_w = i >= a.B ? 0 : i < kKeepLens ? lens[i] : clamp_len(a, a.lens[i]);
      const int nt = granules_of(a, len_w);
      mine_w = incl_w = (int64_t)(whole ? (nt > 0) : nt) * per_b;
      if (__all_sync(0xffffffffu, mine_w < 1 << 26)) {
        int v = (int)mine_w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += x;
        }
        incl_w = v;
      } else {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t x = __shfl_up_sync(0xffffffffu, incl_w, o);
          if (lane >= o) incl_w += x;
        }
      }
    };
    if (blockIdx.x < C) load_window();
    // lane of the request, in the window moved to it, that holds place `at` of the line (-1: none,
    // if lengths changed under the call)
    auto find = [&](int64_t at) -> int {
      unsigned past;
      while (!(past = __ballot_sync(0xffffffffu, before + incl_w > at))) {
        before += __shfl_sync(0xffffffffu, incl_w, 31);
        wb += 32;
        if (wb >= a.B) {
          if (lane == 0 && a.err) atomicCAS(a.err, 0, 0x1000 | (kErrSite + 7));
          return -1;
        }
        load_window();
      }
      return __ffs(past) - 1;
    };
    // Segments (a pair, or the CTA's part of one) in their order, each with the pages of its first
    // 32 granules asked for.  Taking one starts the claim of the pair after it.
    struct Next {
      Seg s;
      int page, row;
    };
    auto look_up = [&](Next& x, int i) {
      if (i < x.s.n) {
        const int pos = (x.s.g0 + i) * kGran, pi = a.page_shift >= 0 ? pos >> a.page_shift : pos / a.page_size;
        x.row = pos - pi * a.page_size;
        x.page = a.table[x.s.b * a.table_stride + pi];
      }
    };
    int64_t item = blockIdx.x, cur = 0, end = 0;  // the next item, and what is left of the last one taken
    bool first = true, pending = true;
    // A claim comes with every CTA and with every pair claimed: the last of all finds nothing and
    // leaves the count as the next call needs it.
    const bool claiming = whole && C > grid && longest > kCons;
    const int64_t last_claim = (claiming ? C : grid) - 1;
    auto answer = [&]() -> int64_t {
      const int c = __shfl_sync(0xffffffffu, claim, 0);
      if (c == last_claim && lane == 0) *claims = 0;
      pending = false;
      return grid + c;
    };
    auto take = [&](Next& x) -> bool {
      if (cur >= end) {
        if (!first) {
          if (!claiming) {
            item = whole ? item + grid : C;
          } else {
            item = answer();
            if (item < C) {
              if (lane == 0) claim = atomicAdd(claims, 1);
              pending = true;
            }
          }
        }
        first = false;
        if (item >= C) return false;
        cur = whole ? item : cut.start(item);
        end = whole ? item + 1 : cut.start(item + 1);
      }
      const int f = find(cur);
      if (f < 0) return false;
      const int len = __shfl_sync(0xffffffffu, len_w, f), nt = granules_of(a, len);
      const int64_t local = cur - before - __shfl_sync(0xffffffffu, incl_w - mine_w, f);
      const int pair = whole ? (int)local : (int)quot(local, nt), t0 = whole ? 0 : (int)(local - (int64_t)pair * nt);
      Seg& s = x.s;
      s.b = wb + f;
      s.lo = first_key(a, len);
      s.hi = len;
      s.g0 = s.lo / kGran + t0;
      s.n = whole ? nt : (int)min((int64_t)(nt - t0), end - cur);
      x.page = -1;
      x.row = 0;
      look_up(x, lane);
      s.h = a.chunks == 1 ? pair : pair / a.chunks;
      s.r0 = (pair - s.h * a.chunks) * a.chunk_rows;
      s.rows = min(a.chunk_rows, a.G - s.r0);
      s.slot = -1;
      s.parts = 1;
      s.first_cta = 0;
      if (s.n < nt) {
        const int64_t p0 = cur - t0;
        s.first_cta = cut.cta_of(p0);
        s.parts = cut.cta_of(p0 + nt - 1) - s.first_cta + 1;
        s.slot = 2 * blockIdx.x + (t0 == 0 ? 1 : 0);
      }
      cur += whole ? 1 : s.n;
      return true;
    };
    int used = 0, nseg = 0;  // granules given to warp lane % kCons, and segments, so far
    int queries = 0;         // segments whose Q copies were issued
    bool ok = true;
    Next next;
    bool more = take(next);
    while (ok && more) {
      Next now = next;
      // the next one's page numbers arrive while this one's granules are issued (the first one's
      // copies go out at once)
      if (nseg > 0) more = take(next);
      const Seg& s = now.s;
      const int si = nseg & 1;
      if (!(ok = wait(seg_empty + si, (uint32_t)(((nseg >> 1) & 1) ^ 1), 0))) break;
      if (lane == 0) {
        segs[si] = s;
        mbar_arrive_expect_tx(seg_full + si, (uint32_t)(s.rows * 2 * DH));
      }
      __syncwarp();
      queries = nseg + 1;
      if (lane < s.rows)
        bulk_copy_g2s(sm + Lay::kQ + si * Lay::kQBytes + lane * Lay::kQPitch,
                      a.q + 2 * (s.b * a.q_b + (int64_t)(s.h * a.G + s.r0 + lane) * a.q_h), 2 * DH, seg_full + si);
      for (int i0 = 0; i0 < s.n && ok; i0 += 32) {
        const int m = min(32, s.n - i0), page = now.page, row = now.row;
        look_up(now, i0 + 32 + lane);
        // lane i issues granule i0 + i; several lanes at once, as one takes about 400 cycles a
        // granule and the memory delivers one in 350 (one lane: 758, eight: 615 us at 64 x 65,536)
        for (int w = 0; w < m && ok; w += kLanes) {
          bool mine = true;
          if (lane >= w && lane < w + kLanes && lane < m) {
            const int use = used + (i0 + lane) / kCons, slot = Uses::slot(use, lane % kCons);
            mine = mbar_wait(empty + slot, Uses::parity(use) ^ 1, abort_flag, kErrSite + 1, a.err);
            if (mine) {  // (a page number outside the pool fills the tile with zeros)
              Uses::log(issued, use, lane % kCons);
              uint8_t* dst = sm + slot * Lay::kSlotBytes;
              mbar_arrive_expect_tx(full + slot, Lay::kSlotBytes);
              tma_load_5d(dst, &mk, full + slot, 0, row, 0, s.h, page);
              tma_load_5d(dst + Lay::kSlotBytes / 2, &mv, full + slot, 0, row, 0, s.h, page);
            }
          }
          ok = __all_sync(0xffffffffu, mine);
        }
      }
      used += (s.n - lane % kCons + kCons - 1) / kCons;
      if (nseg == 0) more = take(next);
      ++nseg;
    }
    // the Q copies, while their barriers still stand at them (the end's mark comes next)
    if (lane < 2 && lane < queries) settle(seg_full + ((queries - 1 - lane) & 1), (uint32_t)((queries - 1 - lane) >> 1) & 1);
    __syncwarp();
    if (ok) {
      const int si = nseg & 1;
      if (wait(seg_empty + si, (uint32_t)(((nseg >> 1) & 1) ^ 1), 2) && lane == 0) {
        segs[si].n = -1;
        mbar_arrive(seg_full + si);
      }
    }
    if (pending) answer();
    // requests without keys
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
      if (clamp_len(a, a.lens[b]) != 0) continue;
      const int hq = a.Hkv * a.G;
      for (int i = lane; i < hq * (DH / 8); i += 32)
        st_128(a.out + 2 * (b * a.o_b + (int64_t)(i / (DH / 8)) * a.o_h) + 16 * (i % (DH / 8)), make_uint4(0, 0, 0, 0));
      if (a.lse)
        for (int i = lane; i < hq; i += 32) a.lse[b * a.ls_b + i * a.ls_h] = -INFINITY;
    }
    // no tile copy is in flight when the CTA ends, wherever this warp or the consumers gave up
    __syncwarp();
    Uses::settle(issued, lane, 32, [&](int slot, uint32_t parity) { settle(full + slot, parity); });
    return;
  }

  // -------------------------------------------------------------------- consumers
  constexpr int NT = DH / 8;   // 8-column output tiles
  constexpr int KS = DH / 16;  // 16-dim steps of the scores
  constexpr bool kKeepQ = DH <= 128;
  constexpr int kRowSets = WIDE ? 2 : 1;
  const uint32_t sm32 = smem_u32(sm);
  const int gid = lane >> 2, tig = lane & 3;
  const int tid = threadIdx.x;
  constexpr int kNT = 32 * kCons;
  // ldmatrix lane offsets: keys as B operand (plain), values as B operand (transposed)
  const int k_row = ((lane >> 4) << 3) + (lane & 7), k_chunk = (lane >> 3) & 1;
  const int v_row = (((lane >> 3) & 1) << 3) + (lane & 7), v_chunk = lane >> 4;

  int use = 0;      // granules taken by this warp so far
  int fetched = 0;  // batches of parts fetched for joins so far
  for (int nseg = 0;; ++nseg) {
    const int si = nseg & 1;
    // Every warp meets the others once a segment (the first barrier below), also when there is
    // none or it gave up a wait, and all leave together.
    bool bad = !wait(seg_full + si, (uint32_t)((nseg >> 1) & 1), 4);
    const Seg s = segs[si];
    if (bad || s.n < 0) {
      cons_any<kNT>(bad);
      return;
    }
    float* buf = reinterpret_cast<float*>(sm + Lay::kBuf + si * Lay::kBufBytes);
    const uint32_t q32 = sm32 + Lay::kQ + si * Lay::kQBytes;
    uint32_t qf[kKeepQ ? KS : 1][4];
    // Q fragment of step ks: rows 0-7 in registers 0 and 2, rows 8-15 in 1 and 3 (zero if !WIDE)
    auto load_q = [&](int ks, uint32_t (&f)[4]) {
      if (WIDE) {
        ldsm_x4(q32 + ((((lane >> 3) & 1) << 3) + (lane & 7)) * Lay::kQPitch + ks * 32 + (lane >> 4) * 16, f);
      } else {
        asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];"
                     : "=r"(f[0]), "=r"(f[2])
                     : "r"(q32 + (lane & 7) * Lay::kQPitch + ks * 32 + ((lane >> 3) & 1) * 16)
                     : "memory");
        f[1] = f[3] = 0;
      }
    };
    if (kKeepQ) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) load_q(ks, qf[ks]);
    }
    float o[NT][4], m[kRowSets], l[kRowSets];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
#pragma unroll
    for (int x = 0; x < kRowSets; ++x) {
      m[x] = -INFINITY;
      l[x] = 0.f;
    }
    const bool fresh = a.kn && (!a.active || a.active[s.b]);

    for (int i = warp; i < s.n; i += kCons, ++use) {
      const int slot = Uses::slot(use, warp);
      const uint32_t par = Uses::parity(use);
      const int pos = (s.g0 + i) * kGran;
      const bool edge = pos < s.lo || pos + kGran > s.hi;
      const bool owns_new = fresh && pos + kGran >= s.hi;  // the granule of key hi - 1
      // the new token's rows, asked for before the wait for the granule: 16-byte vector x of K, then V
      constexpr int kVecs = DH / 8, kNew = (2 * kVecs + 31) / 32;
      uint4 fresh_v[kNew];
      int64_t page = 0;
      if (owns_new) {
        page = a.table[s.b * a.table_stride + (s.hi - 1) / a.page_size];
#pragma unroll
        for (int y = 0; y < kNew; ++y) {
          const int x = lane + 32 * y;
          if (x < 2 * kVecs)
            fresh_v[y] = x >= kVecs ? ld_128(a.vn + 2 * (s.b * a.vn_b + s.h * a.vn_h) + 16 * (x - kVecs))
                                    : ld_128(a.kn + 2 * (s.b * a.kn_b + s.h * a.kn_h) + 16 * x);
        }
      }
      if (!wait(full + slot, par, 5)) {
        bad = true;
        break;
      }
      uint8_t* kt = sm + slot * Lay::kSlotBytes;
      const uint32_t k32 = sm32 + slot * Lay::kSlotBytes, v32 = k32 + Lay::kSlotBytes / 2;
      if (edge || owns_new) {
        // values of masked keys count as zero (0 times what the page holds could be NaN)
        if (edge)
          for (int x = lane; x < kGran * kVecs; x += 32) {
            const int r = x / kVecs, c = x % kVecs;
            if (pos + r < s.lo || pos + r >= s.hi)
              *reinterpret_cast<uint4*>(kt + Lay::kSlotBytes / 2 + tile_off(r, c)) = make_uint4(0, 0, 0, 0);
          }
        if (owns_new) {  // into the tile, and into the page
          const int r = s.hi - 1 - pos, off = (s.hi - 1) % a.page_size;
#pragma unroll
          for (int y = 0; y < kNew; ++y) {
            const int x = lane + 32 * y, c = x % kVecs;
            const bool isv = x >= kVecs;
            if (x >= 2 * kVecs) break;
            *reinterpret_cast<uint4*>(kt + (isv ? Lay::kSlotBytes / 2 : 0) + tile_off(r, c)) = fresh_v[y];
            if (s.r0 == 0 && page >= 0 && page < a.num_pages)
              st_128((isv ? a.vp + 2 * (page * a.vp_p + s.h * a.vp_h + off * a.vp_t)
                          : a.kp + 2 * (page * a.kp_p + s.h * a.kp_h + off * a.kp_t)) + 16 * c, fresh_v[y]);
          }
        }
        __syncwarp();
      }

      // scores of the 16 keys: two 8-key column tiles, even and odd steps in separate chains
      float sc[2][2][4];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[x][y][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t kf[4];
        ldsm_x4(k32 + tile_off(k_row, 2 * ks + k_chunk), kf);
        if (!kKeepQ) load_q(ks, qf[0]);
        const uint32_t(&qq)[4] = qf[kKeepQ ? ks : 0];
        mma_16816<T>(sc[ks & 1][0], qq, kf[0], kf[1]);
        mma_16816<T>(sc[ks & 1][1], qq, kf[2], kf[3]);
      }
      // online softmax of rows gid (and gid + 8): this lane's keys are pos + 8 y + 2 tig + {0, 1}
      uint32_t ph[4] = {0, 0, 0, 0}, pl[4] = {0, 0, 0, 0};  // P as A operand: high and low parts
      float al[kRowSets];
      bool moved = false;
#pragma unroll
      for (int x = 0; x < kRowSets; ++x) {
        float v[4];
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float t = (sc[0][y][2 * x + e] + sc[1][y][2 * x + e]) * a.scale_log2;
            const int key = pos + 8 * y + 2 * tig + e;
            if (edge && (key < s.lo || key >= s.hi)) t = -INFINITY;
            v[2 * y + e] = t;
          }
        float mx = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[x], mx), top = mn == -INFINITY ? 0.f : mn, base = top - kShift<T>;
        al[x] = ex2_approx(m[x] - top);
        moved |= mn != m[x];
        m[x] = mn;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = ex2_approx(v[e] - base);
        l[x] = l[x] * al[x] + ((v[0] + v[1]) + (v[2] + v[3]));
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t hi = ElemTraits<T>::pack2(v[2 * y], v[2 * y + 1]);
          const float2 f = ElemTraits<T>::unpack2(hi);
          const uint32_t lo = ElemTraits<T>::pack2(v[2 * y] - f.x, v[2 * y + 1] - f.y);
          if (WIDE) {
            ph[2 * y + x] = hi;
            pl[2 * y + x] = lo;
          } else {
            ph[2 * y] = hi;
            ph[2 * y + 1] = lo;
          }
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          o[j][0] *= al[0];
          o[j][1] *= al[0];
          o[j][2] *= al[kRowSets - 1];
          o[j][3] *= al[kRowSets - 1];
        }
      }
#pragma unroll
      for (int j = 0; j < NT; j += 2) {
        uint32_t vf[4];
        ldsm_x4_trans(v32 + tile_off(v_row, j + v_chunk), vf);
        mma_16816<T>(o[j], ph, vf[0], vf[1]);
        mma_16816<T>(o[j + 1], ph, vf[2], vf[3]);
        if (WIDE) {
          mma_16816<T>(o[j], pl, vf[0], vf[1]);
          mma_16816<T>(o[j + 1], pl, vf[2], vf[3]);
        }
      }
      if (edge || owns_new) fence_proxy_async_smem();  // the slot's next copy comes through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + slot);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(seg_empty + si);  // the descriptor and Q have been read

#pragma unroll
    for (int x = 0; x < kRowSets; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    }
    if (!WIDE) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {  // high and low parts
        o[j][0] += o[j][2];
        o[j][1] += o[j][3];
      }
    }
    if (s.n == 1 && s.slot < 0) {  // a pair of one granule: the first warp has all of it
      if (cons_any<kNT>(bad)) return;
#pragma unroll
      for (int x = 0; x < kRowSets; ++x) {
        const int r = gid + 8 * x;
        if (warp == 0 && r < s.rows) {
          const int64_t hq = s.h * a.G + s.r0 + r;
          uint8_t* dst = a.out + 2 * (s.b * a.o_b + hq * a.o_h + 2 * tig);
          const float f = l[x] == 0.f ? 0.f : 1.f / l[x];
#pragma unroll
          for (int j = 0; j < NT; ++j)
            *reinterpret_cast<uint32_t*>(dst + 16 * j) = ElemTraits<T>::pack2(o[j][2 * x] * f, o[j][2 * x + 1] * f);
          if (a.lse && tig == 0) a.lse[s.b * a.ls_b + hq * a.ls_h] = lse_of<T>(m[x], l[x]);
        }
      }
      continue;
    }

    // Join the warps: each leaves (m, l) and its outputs, which are scaled to the common maximum as
    // they are summed.  Two buffers: a warp may start on the next segment before all are done.
    float2* ml = reinterpret_cast<float2*>(sm + Lay::kMl) + si * kCons * kRows;
#pragma unroll
    for (int x = 0; x < kRowSets; ++x)
      if (tig == 0) ml[warp * kRows + gid + 8 * x] = make_float2(m[x], l[x]);
    // columns joined at a time: what the buffer holds of s.rows rows (rows padded by 8 floats
    // to spread the stores over the banks)
    const int shift = s.rows <= 4 ? (DH < 128 ? 6 : 7) : s.rows <= 8 ? 6 : 5, cw = 1 << shift;
    const int pitch = cw + 8;
    float* part_o = reinterpret_cast<float*>(a.ws + kWsO) + (int64_t)s.slot * kRows * DH;
    for (int c0 = 0; c0 < DH; c0 += cw) {
      if (c0 > 0) cons_sync<kNT>();  // the buffer has been read
#pragma unroll
      for (int x = 0; x < kRowSets; ++x)
        if (gid + 8 * x < s.rows) {
          float* dst = buf + (warp * s.rows + gid + 8 * x) * pitch + 2 * tig - c0;
#pragma unroll
          for (int j = 0; j < NT; ++j)
            if (8 * j >= c0 && 8 * j < c0 + cw) *reinterpret_cast<float2*>(dst + 8 * j) = make_float2(o[j][2 * x], o[j][2 * x + 1]);
        }
      if (c0 > 0) cons_sync<kNT>();
      else if (cons_any<kNT>(bad)) return;
      for (int it = tid; it < s.rows << (shift - 2); it += kNT) {
        const int r = it >> (shift - 2), c = (it << 2) & (cw - 1);
        float2 t[kCons];
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < kCons; ++w) {
          t[w] = ml[w * kRows + r];
          M = fmaxf(M, t[w].x);
        }
        const float base = M == -INFINITY ? 0.f : M;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kCons; ++w) {
          const float f = ex2_approx(t[w].x - base);
          L = fmaf(t[w].y, f, L);
          const float4 u = *reinterpret_cast<const float4*>(buf + (w * s.rows + r) * pitch + c);
          v.x = fmaf(u.x, f, v.x);
          v.y = fmaf(u.y, f, v.y);
          v.z = fmaf(u.z, f, v.z);
          v.w = fmaf(u.w, f, v.w);
        }
        if (s.slot < 0) {
          const int hq = s.h * a.G + s.r0 + r;
          store4<T>(a.out + 2 * (s.b * a.o_b + hq * a.o_h + c0 + c), v, L == 0.f ? 0.f : 1.f / L);
          if (a.lse && c0 + c == 0) a.lse[s.b * a.ls_b + hq * a.ls_h] = lse_of<T>(M, L);
        } else {
          *reinterpret_cast<float4*>(part_o + r * DH + c0 + c) = v;
          if (c0 + c == 0) reinterpret_cast<float2*>(a.ws + kWsMl)[s.slot * kRows + r] = make_float2(M, L);
        }
      }
    }
    if (s.slot < 0) continue;

    // A cut pair: the CTA whose part arrives last joins the parts.  Of many parts, groups of kFan
    // first: most groups are complete before the last CTA arrives, and a CTA reads only some
    // 30 GB/s here (74 parts of 4 heads at once took 8 us after the last arrival).
    const float2* gml = reinterpret_cast<const float2*>(a.ws + kWsMl);
    const float* go = reinterpret_cast<const float*>(a.ws + kWsO);
    bool final = s.parts <= kFan + 4;
    int base = final ? 0 : (int)(blockIdx.x - s.first_cta) / kFan * kFan;  // first part of the round's group,
    int members = final ? s.parts : min(kFan, s.parts - base), step = 1;   // their number, and their distance
    for (;;) {
      auto slot_of = [&](int p) {
        const int part = base + p * step;
        return (int64_t)(2 * (s.first_cta + part) + (part == 0 ? 1 : 0));
      };
      cons_sync<kNT>();
      if (tid == 0) {
        // release: the CTA's part (ordered before this by the barrier) before the count
        int arrived, *counter = reinterpret_cast<int*>(a.ws) + 1 + (final ? s.first_cta : kMaxCtas + (int)slot_of(0));
        asm volatile("atom.add.release.gpu.global.s32 %0, [%1], 1;" : "=r"(arrived) : "l"(counter) : "memory");
        const bool last = arrived + 1 == members;
        if (last) {
          *counter = 0;  // as the next call finds it
          asm volatile("fence.acq_rel.gpu;" ::: "memory");
        }
        *last_flag = last;
      }
      cons_sync<kNT>();
      if (!*last_flag) break;
      // The parts come to shared memory by bulk copies, in batches, two in flight; a thread sums
      // 4 columns of a row, and where the rows are few, groups of threads share the parts.
      constexpr int kItems = (kRows * DH / 4 + kNT - 1) / kNT;
      const int items = s.rows * (DH / 4);
      const int batch = Lay::kHalf / 16 / items, batches = (members + batch - 1) / batch;
      auto fetch = [&](int k) {  // by warp 0
        if (k >= batches) return;
        const int half = (fetched + k) & 1, n = min(batch, members - k * batch);
        if (lane == 0) mbar_arrive_expect_tx(stage_full + half, (uint32_t)(n * items * 16));
        __syncwarp();
        if (lane < n)
          bulk_copy_g2s(sm + Lay::kStage + half * Lay::kHalf + lane * items * 16, go + slot_of(k * batch + lane) * kRows * DH,
                        items * 16, stage_full + half);
      };
      if (warp == 0) {
        asm volatile("fence.proxy.async;" ::: "memory");  // the parts were written by plain stores
        fetch(0);
        fetch(1);
      }
      float* wt = buf;  // [members][rows] weights
      for (int r = warp; r < s.rows; r += kCons) {
        const float2 t = lane < members ? __ldcg(gml + slot_of(lane) * kRows + r) : make_float2(-INFINITY, 0.f);
        float M = t.x;
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
        const float f = ex2_approx(t.x - (M == -INFINITY ? 0.f : M));
        const float L = warp_sum(t.y * f);
        if (lane < members) wt[lane * s.rows + r] = f * (!final ? 1.f : L == 0.f ? 0.f : 1.f / L);
        if (lane == 0) {
          if (!final) const_cast<float2*>(gml)[slot_of(0) * kRows + r] = make_float2(M, L);
          else if (a.lse) a.lse[s.b * a.ls_b + (int64_t)(s.h * a.G + s.r0 + r) * a.ls_h] = lse_of<T>(M, L);
        }
      }
      cons_sync<kNT>();
      const int groups = items >= kNT ? 1 : kNT / items, grp = groups == 1 ? 0 : tid / items;
      const int it0 = groups == 1 ? tid : tid % items;
      float4 v[kItems];
#pragma unroll
      for (int x = 0; x < kItems; ++x) v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = 0; k < batches; ++k) {
        const int half = (fetched + k) & 1;
        const uint32_t par = (uint32_t)(((fetched + k) >> 1) & 1);
        if (!wait(stage_full + half, par, 6)) settle(stage_full + half, par);  // (the next segment's wait sees a failure)
        const float4* src = reinterpret_cast<const float4*>(sm + Lay::kStage + half * Lay::kHalf);
        const int n = min(batch, members - k * batch);
        if (grp < groups)
#pragma unroll
          for (int x = 0; x < kItems; ++x) {
            const int it = it0 + x * kNT;
            if (it < items)
              for (int p = grp; p < n; p += groups) {
                const float4 u = src[p * items + it];
                const float f = wt[(k * batch + p) * s.rows + it / (DH / 4)];
                v[x].x = fmaf(u.x, f, v[x].x);
                v[x].y = fmaf(u.y, f, v[x].y);
                v[x].z = fmaf(u.z, f, v[x].z);
                v[x].w = fmaf(u.w, f, v[x].w);
              }
          }
        if (k + 2 < batches) {
          cons_sync<kNT>();  // the half has been read
          if (warp == 0) fetch(k + 2);
        }
      }
      fetched += batches;
      if (groups > 1) {
        float4* red = reinterpret_cast<float4*>(wt + 32 * kRows);  // [group][item]
        if (grp < groups) red[grp * items + it0] = v[0];
        cons_sync<kNT>();
        if (grp == 0)
          for (int g = 1; g < groups; ++g) {
            const float4 w = red[g * items + it0];
            v[0].x += w.x;
            v[0].y += w.y;
            v[0].z += w.z;
            v[0].w += w.w;
          }
      }
      if (grp == 0)
#pragma unroll
        for (int x = 0; x < kItems; ++x) {
          const int it = it0 + x * kNT;
          if (it >= items) break;
          if (final)
            store4<T>(a.out + 2 * (s.b * a.o_b + (int64_t)(s.h * a.G + s.r0 + it / (DH / 4)) * a.o_h + (it % (DH / 4)) * 4), v[x], 1.f);
          else
            reinterpret_cast<float4*>(const_cast<float*>(go) + slot_of(0) * kRows * DH)[it] = v[x];
        }
      if (final) break;
      members = (s.parts + kFan - 1) / kFan;
      base = 0;
      step = kFan;
      final = true;
    }
  }
}

using EncodeFn = PFN_cuTensorMapEncodeTiled_v12000;
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    cudaDriverEntryPointQueryResult qr;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qr) != cudaSuccess ||
        qr != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// A pool [pages, Hkv, page_size, dh] as (64 columns, token, 64-column box, head, page), so that one
// copy brings 16 tokens of one head and page, all columns, in boxes of 16 rows x 128 bytes.
int encode_pool(CUtensorMap* m, const bna_tensor4* t, int dtype, const char* name) {
  EncodeFn enc = encode_fn();
  if (!enc) return fail(BNA_CUDA_ERROR, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t boxes = (cuuint64_t)t->size[3] / 64;
  const cuuint64_t dims[5] = {64, (cuuint64_t)t->size[2], boxes, (cuuint64_t)t->size[1], (cuuint64_t)t->size[0]};
  // a dim of size 1 is never stepped over: any valid stride will do
  auto st = [&](int d) { return t->size[d] > 1 ? (cuuint64_t)t->stride[d] * 2 : (cuuint64_t)t->size[3] * 2; };
  const cuuint64_t strides[4] = {st(2), 128, st(1), st(0)};
  const cuuint32_t box[5] = {64, kGran, (cuuint32_t)boxes, 1, 1};
  const cuuint32_t es[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(m, dtype == BNA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, t->data,
                         dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(BNA_BAD_STRIDE, std::string(name) + ": cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
  return BNA_OK;
}

int sm_count() {
  static std::mutex mu;
  static std::map<int, int> cache;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> g(mu);
  auto it = cache.find(dev);
  if (it != cache.end()) return it->second;
  int n = 0;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return cache[dev] = n;
}

template <typename T, int DH, bool WIDE>
int launch_decode(const CUtensorMap& mk, const CUtensorMap& mv, const PagedArgs& a, double most, cudaStream_t s) {
  auto kern = paged_decode_kernel<T, DH, WIDE>;
  static std::atomic<uint64_t> ready{0};  // devices (bits) whose kernel has its shared memory allowed
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !(ready.load() >> dev & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<DH>::kAlloc);
    if (e != cudaSuccess) return check_cuda(e, "paged_decode attributes");
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min((double)std::min(sm_count(), kMaxSms) * Layout<DH>::kCtas, most));
  cfg.blockDim = dim3(Layout<DH>::kThreads);
  cfg.dynamicSmemBytes = Layout<DH>::kAlloc;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, mk, mv, a), "paged_decode launch");
}

}  // namespace

int64_t paged_decode_workspace_bytes() { return kWsBytes; }

int launch_paged_decode(const bna_tensor4* q, bna_tensor4* kp, bna_tensor4* vp, const bna_tensor4* kn,
                        const bna_tensor4* vn, const uint8_t* active, bna_tensor4* out, float* lse, int64_t ls_b,
                        int64_t ls_h, int dtype, const int32_t* table, int64_t table_stride, int width,
                        const int32_t* lens, int window, float scale, void* ws, cudaStream_t s) {
  CUtensorMap mk, mv;
  if (int rc = encode_pool(&mk, kp, dtype, "k_pages")) return rc;
  if (int rc = encode_pool(&mv, vp, dtype, "v_pages")) return rc;
  PagedArgs a{};
  a.q = static_cast<const uint8_t*>(q->data);
  a.q_b = q->stride[0], a.q_h = q->stride[1];
  a.kp = static_cast<uint8_t*>(kp->data), a.vp = static_cast<uint8_t*>(vp->data);
  a.kp_p = kp->stride[0], a.kp_h = kp->stride[1], a.kp_t = kp->stride[2];
  a.vp_p = vp->stride[0], a.vp_h = vp->stride[1], a.vp_t = vp->stride[2];
  if (kn) {
    a.kn = static_cast<const uint8_t*>(kn->data), a.vn = static_cast<const uint8_t*>(vn->data);
    a.active = active;
    a.kn_b = kn->stride[0], a.kn_h = kn->stride[1], a.vn_b = vn->stride[0], a.vn_h = vn->stride[1];
  }
  a.out = static_cast<uint8_t*>(out->data);
  a.o_b = out->stride[0], a.o_h = out->stride[1];
  a.lse = lse, a.ls_b = ls_b, a.ls_h = ls_h;
  a.table = table, a.table_stride = table_stride, a.lens = lens;
  a.B = (int)q->size[0], a.Hkv = (int)kp->size[1], a.G = (int)(q->size[1] / kp->size[1]);
  a.width = width, a.num_pages = (int)kp->size[0], a.page_size = (int)kp->size[2], a.window = window;
  a.page_shift = (a.page_size & (a.page_size - 1)) == 0 ? __builtin_ctz((unsigned)a.page_size) : -1;
  a.chunks = (a.G + kRows - 1) / kRows;
  a.chunk_rows = (a.G + a.chunks - 1) / a.chunks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.ws = static_cast<uint8_t*>(ws);
  a.err = device_error_word();
  // no more CTAs than there could be pairs, or stretches of an even cut
  const int64_t keys = window > 0 ? std::min((int64_t)width * a.page_size, (int64_t)window + 2 * kGran) : (int64_t)width * a.page_size;
  const double pairs = (double)a.B * a.Hkv * a.chunks, stretches = std::ceil(pairs * (double)((keys + kGran - 1) / kGran) / kMinPart);
  const double most = std::max(pairs, stretches);
  const bool bf = dtype == BNA_BF16, wide = a.chunk_rows > 8;
#define BNA_PAGED(T_, DH_) \
  return wide ? launch_decode<T_, DH_, true>(mk, mv, a, most, s) : launch_decode<T_, DH_, false>(mk, mv, a, most, s)
  switch (q->size[3]) {
    case 64:
      if (bf) BNA_PAGED(__nv_bfloat16, 64);
      BNA_PAGED(__half, 64);
    case 128:
      if (bf) BNA_PAGED(__nv_bfloat16, 128);
      BNA_PAGED(__half, 128);
    case 256:
      if (bf) BNA_PAGED(__nv_bfloat16, 256);
      BNA_PAGED(__half, 256);
    default: return fail(BNA_UNSUPPORTED, "paged_decode_attention: head_dim must be 64, 128 or 256");
  }
#undef BNA_PAGED
}

}  // namespace bna
