// paged_cache.cu — the write side of a paged key/value cache: pages for the next tokens
// (block tables and slot maps from the requests' lengths) and the tokens' rows into them.
// Pools are [pages, kv heads, page_size, head_dim]; a request's tokens 0..len-1 lie in the pages
// its block-table row names, page_size to a page; slot = page * page_size + offset.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <string>

#include "common.cuh"
#include "int4.cuh"

namespace bna {
namespace {

constexpr int kMaxRequests = 4096;  // three prefix sums, the lengths and flags of a call: 68 KB of shared memory
constexpr int kReserveCtas = 148;
constexpr int kRequestBytes = 4 * 4 + 1;  // dynamic shared memory of a request
constexpr int kScanBytes = 3 * 32 * 8;  // static shared memory: a warp's part of each sum

struct ReserveArgs {
  const int32_t* lens;
  const int32_t* add;
  int32_t* table;
  int64_t table_stride;
  int32_t* free_pages;
  const int32_t* num_free;
  int32_t* lens_out;
  int32_t* num_free_out;
  uint8_t* granted;
  int64_t* slots;
  int32_t* positions;
  int64_t num_tokens;
  int B, width, num_pages, page_size;
  int vector_out;  // slots and positions are 16-byte aligned
};

// First index b in [0, n) with c[b] > x (c non-decreasing), n if there is none.
__device__ __forceinline__ int upper_bound(const int32_t* c, int n, int64_t x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (c[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ int pages_of(unsigned tokens, unsigned page_size) {
  return (int)((tokens + page_size - 1) / page_size);  // tokens <= INT_MAX, page_size <= INT_MAX
}

// What a request asks for: its length after the call, and pages taken (need) or given back.
enum : uint8_t { kGrows = 1, kNeeds = 2 };  // tokens are added and fit the table; they need pages
struct Ask {
  int want, old_pages, new_pages, need, back;
  bool fits;
};
__device__ __forceinline__ Ask ask_of(int len, int add, int capacity, int page_size) {
  Ask r;
  const int64_t want = (int64_t)len + add;
  r.fits = want <= capacity;
  r.want = (int)min(max(want, (int64_t)0), (int64_t)capacity);
  r.old_pages = pages_of(len, page_size);
  r.new_pages = r.fits ? pages_of(r.want, page_size) : r.old_pages;
  r.need = add > 0 ? r.new_pages - r.old_pages : 0;
  r.back = add < 0 ? r.old_pages - r.new_pages : 0;
  return r;
}

// Every CTA computes the prefix sums over the requests of the tokens added, the pages needed
// and the pages given back (shared memory; at most 4096 requests, read through L2), from which any
// table entry, slot and stack entry follows by a binary search, and the grid shares these
// out: no CTA waits for another.  Nothing that is read is written in the call: lengths and stack
// height go to other places, table entries written lie past those read, and stack entries
// are written only where pages stay given back (then none is taken from below them).
// The j-th page given back lies j below the new top of the stack and the i-th page taken
// comes from i below it, so a call followed by its opposite restores the stack.
// Bound by launch and dependent-read latency: the largest calls move about 1.6 MB (1,000 requests
// with 131,072 prompt tokens 8.9 us, one request 2.9 us on the GPU).  A thread takes K
// tokens in a row: one where the tokens are few, four (one search and one page for most of
// them) where there are many.
template <int K>
__global__ void __launch_bounds__(1024) reserve_kernel(const ReserveArgs a) {
  extern __shared__ int32_t sm[];
  // Inclusive prefix sums, capped at INT_MAX: exact for every token below num_tokens and every page
  // there is.  What a request asks for is not read off their differences, which the cap falsifies.
  int32_t* cum_add = sm;
  int32_t* cum_need = sm + a.B;
  int32_t* cum_back = sm + 2 * a.B;
  int32_t* lens = sm + 3 * a.B;     // cut to the table, so that no later index leaves a row
  uint8_t* asks = reinterpret_cast<uint8_t*>(sm + 4 * a.B);  // kGrows, kNeeds
  __shared__ int64_t warp_sums[3][32];
  static_assert(sizeof(warp_sums) == kScanBytes, "static shared memory");
  const int threads = blockDim.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int capacity = (int)min((int64_t)a.width * a.page_size, (int64_t)INT_MAX);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = min(max(a.num_free[0], 0), a.num_pages);

  // each thread sums a run of requests, then the runs are scanned
  const int per = (a.B + threads - 1) / threads;
  const int b0 = min((int)threadIdx.x * per, a.B), b1 = min(b0 + per, a.B);
  int64_t sum[3] = {0, 0, 0};
  for (int b = b0; b < b1; ++b) {
    const int len = min(max(a.lens[b], 0), capacity), add = a.add[b];
    const Ask r = ask_of(len, add, capacity, a.page_size);
    lens[b] = len;
    sum[0] += max(add, 0);
    sum[1] += r.need;
    sum[2] += r.back;
  }
  int64_t at[3];
#pragma unroll
  for (int x = 0; x < 3; ++x) {
    int64_t v = sum[x];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) warp_sums[x][warp] = v;
    at[x] = v - sum[x];
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < 3; ++x)
    for (int w = 0; w < warp; ++w) at[x] += warp_sums[x][w];
  for (int b = b0; b < b1; ++b) {
    const int add = a.add[b];
    const Ask r = ask_of(lens[b], add, capacity, a.page_size);
    at[0] += max(add, 0);
    at[1] += r.need;
    at[2] += r.back;
    asks[b] = (add > 0 && r.fits ? kGrows : 0) | (r.need > 0 ? kNeeds : 0);
    cum_add[b] = (int32_t)min(at[0], (int64_t)INT_MAX);
    cum_need[b] = (int32_t)min(at[1], (int64_t)INT_MAX);
    cum_back[b] = (int32_t)min(at[2], (int64_t)INT_MAX);
  }
  __syncthreads();

  const int R = cum_back[a.B - 1];
  const int64_t top = (int64_t)n + R;
  // requests are served in order while their pages last: pages taken = the largest prefix <= top
  const int served = cum_need[a.B - 1] <= top ? a.B : upper_bound(cum_need, a.B, top);
  const int A = served > 0 ? cum_need[served - 1] : 0;
  auto before = [](const int32_t* c, int b) { return b > 0 ? c[b - 1] : 0; };
  // Page x below the top of the stack with the pages given back on it.
  auto from_top = [&](int64_t x) -> int {
    if (x < R) {
      const int b = upper_bound(cum_back, a.B, x);
      const int first = pages_of(lens[b], a.page_size) - (cum_back[b] - before(cum_back, b));
      return a.table[b * a.table_stride + first + (x - before(cum_back, b))];
    }
    const int64_t i = top - 1 - x;
    return i >= 0 && i < n ? a.free_pages[i] : -1;
  };
  // Tokens were added to b and have slots: they fit, and need no page or were served.
  auto granted = [&](int b) { return (asks[b] & kGrows) && (b < served || !(asks[b] & kNeeds)); };
  const int64_t stride = (int64_t)gridDim.x * threads, tid = (int64_t)blockIdx.x * threads + threadIdx.x;

  // slots and positions of the added tokens, packed request by request, and the table entries
  // of the pages taken, each written with the page's first token
  for (int64_t t0 = tid * K; t0 < a.num_tokens; t0 += stride * K) {
    int b = upper_bound(cum_add, a.B, t0);
    int64_t slot[K];
    int pos[K], at_b = -1, at_page = -1, page = -1, have = 0, first = 0;
    bool ok = false;
#pragma unroll
    for (int x = 0; x < K; ++x) {
      const int64_t t = t0 + x;
      slot[x] = -1;
      pos[x] = -1;
      while (b < a.B && cum_add[b] <= t) ++b;
      if (b >= a.B) continue;
      if (b != at_b) {
        at_b = b;
        at_page = -1;
        ok = granted(b);
        have = pages_of(lens[b], a.page_size);
        first = before(cum_need, b);
      }
      if (!ok) continue;
      pos[x] = lens[b] + (int)(t - before(cum_add, b));
      const int pi = (unsigned)pos[x] / (unsigned)a.page_size, off = pos[x] - pi * a.page_size;
      if (pi != at_page) {
        at_page = pi;
        page = pi < have ? a.table[b * a.table_stride + pi] : from_top((int64_t)first + pi - have);
        if (pi >= have && off == 0) a.table[b * a.table_stride + pi] = page;
      }
      slot[x] = page < 0 ? -1 : (int64_t)page * a.page_size + off;
    }
    if (K == 4 && a.vector_out && t0 + K <= a.num_tokens) {
      st_128(a.slots + t0, make_uint4((uint32_t)slot[0], (uint32_t)(slot[0] >> 32), (uint32_t)slot[1 % K],
                                      (uint32_t)(slot[1 % K] >> 32)));
      st_128(a.slots + t0 + 2, make_uint4((uint32_t)slot[2 % K], (uint32_t)(slot[2 % K] >> 32), (uint32_t)slot[3 % K],
                                          (uint32_t)(slot[3 % K] >> 32)));
      st_128(a.positions + t0, make_uint4(pos[0], pos[1 % K], pos[2 % K], pos[3 % K]));
    } else {
#pragma unroll
      for (int x = 0; x < K; ++x)
        if (t0 + x < a.num_tokens) {
          a.slots[t0 + x] = slot[x];
          a.positions[t0 + x] = pos[x];
        }
    }
  }
  // more tokens than slot_map holds: the entries of the pages past it, page by page
  if (cum_add[a.B - 1] > a.num_tokens)
    for (int64_t i = tid; i < A; i += stride) {
      const int b = upper_bound(cum_need, a.B, i);
      const int64_t pi = pages_of(lens[b], a.page_size) + i - before(cum_need, b);
      if (before(cum_add, b) + pi * a.page_size - lens[b] >= a.num_tokens) a.table[b * a.table_stride + pi] = from_top(i);
    }
  for (int64_t b = tid; b < a.B; b += stride) {
    const bool ok = granted((int)b);
    const int add = a.add[b];
    a.lens_out[b] = add > 0 && !ok ? lens[b] : max(0, (int)((int64_t)lens[b] + add));
    a.granted[b] = ok;
  }
  if (tid == 0) a.num_free_out[0] = (int)min(top - A, (int64_t)a.num_pages);
  // stack entries of the pages given back and not taken again, from index n up
  for (int64_t i = n + tid; i < top - A && i < a.num_pages; i += stride) a.free_pages[i] = from_top(top - 1 - i);
}

// ------------------------------------------------------------------------------ append
struct PagedAppendArgs {
  const uint8_t *k, *v;
  uint8_t *kp, *vp;
  int64_t k_h, k_t, v_h, v_t;                    // element strides: head, token
  int64_t kp_p, kp_h, kp_t, vp_p, vp_h, vp_t;    // page, head, token in page
  const int64_t* slots;
  int64_t rows;  // tokens * heads
  int64_t num_slots;
  int heads, page_size, vec_shift;  // 2^vec_shift 16-byte vectors per row
};

// A thread moves one 16-byte vector of the keys and of the values of N (token, head) rows that lie a
// block apart, with all 2 N loads in flight before the first store (they do not wait for the
// slots).  Bound by HBM: each row is read and written once (131,072 tokens x 2 heads of 128:
// 42.0 us = 6.4 TB/s, the rate of a plain copy; one row a thread 53 us).
template <int N>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedAppendArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int c = threadIdx.x & ((1 << a.vec_shift) - 1);
  const int step = 256 >> a.vec_shift;  // rows of a block side by side
  const int64_t row0 = (int64_t)blockIdx.x * (N * step) + (threadIdx.x >> a.vec_shift);
  uint4 k[N], v[N];
  int64_t slot[N];
  int head[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t row = row0 + i * step;
    slot[i] = -1;
    if (row < a.rows) {
      const int64_t t = a.rows <= UINT_MAX ? (int64_t)((unsigned)row / (unsigned)a.heads) : row / a.heads;
      head[i] = (int)(row - t * a.heads);
      slot[i] = a.slots[t];
      k[i] = ld_nc_128(a.k + 2 * (t * a.k_t + head[i] * a.k_h) + 16 * c);
      v[i] = ld_nc_128(a.v + 2 * (t * a.v_t + head[i] * a.v_h) + 16 * c);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (slot[i] < 0 || slot[i] >= a.num_slots) continue;
    const int64_t page = a.num_slots <= UINT_MAX ? (int64_t)((unsigned)slot[i] / (unsigned)a.page_size) : slot[i] / a.page_size;
    const int64_t off = slot[i] - page * a.page_size;
    st_128(a.kp + 2 * (page * a.kp_p + head[i] * a.kp_h + off * a.kp_t) + 16 * c, k[i]);
    st_128(a.vp + 2 * (page * a.vp_p + head[i] * a.vp_h + off * a.vp_t) + 16 * c, v[i]);
  }
}

// ------------------------------------------------------------------------------ 4-bit rows
struct Int4RowsArgs {
  uint8_t* rows[2];      // keys, values: in (append) or out (read)
  int64_t h[2], t[2];    // their element strides: head, token
  uint8_t* pool;
  int64_t p_p, p_h, p_g;  // byte strides: page, head, block
  const int64_t* slots;
  int64_t count;  // tokens * heads
  int64_t num_slots;
  int heads, page_size;
  int wide;  // every 16 columns of the rows are 32-byte aligned
};

// A row is a token's of one head, and four lanes share it: lane t has columns 64 y + 16 t .. + 15 of every group y, whose code
// words lie side by side.  blockIdx.y: keys, values.
struct Int4Row {
  uint8_t *row, *half;  // the 16-bit row, its half of the block (null: no slot)
  int token;            // in the block
};
__device__ __forceinline__ bool int4_row(const Int4RowsArgs& a, int dh, Int4Row& r) {
  const int64_t i = (int64_t)blockIdx.x * (blockDim.x / 4) + threadIdx.x / 4;
  if (i >= a.count) return false;
  const bool x = blockIdx.y;
  const int64_t t = a.count <= UINT_MAX ? (int64_t)((unsigned)i / (unsigned)a.heads) : i / a.heads;
  const int head = (int)(i - t * a.heads);
  const int64_t slot = a.slots[t];
  r.row = x ? a.rows[1] + 2 * (t * a.t[1] + head * a.h[1]) : a.rows[0] + 2 * (t * a.t[0] + head * a.h[0]);
  if (slot >= 0 && slot < a.num_slots) {
    const int64_t page = a.num_slots <= UINT_MAX ? (int64_t)((unsigned)slot / (unsigned)a.page_size) : slot / a.page_size;
    const int off = (int)(slot - page * a.page_size);
    r.token = off % kInt4Tokens;
    r.half = a.pool + page * a.p_p + head * a.p_h + off / kInt4Tokens * a.p_g + x * int4_half_bytes(dh);
  }
  return true;
}
template <int N>  // N words, 4 N bytes aligned (16 at most)
__device__ __forceinline__ void move_words(uint32_t* dst, const uint32_t* src) {
  if constexpr (N == 2) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(src);
  else
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<uint4*>(dst + i) = *reinterpret_cast<const uint4*>(src + i);
}

// GR groups of 64 columns a row.  131,072 tokens x 2 heads of 128 in bf16: 42 us for 172 MB, 4.1 TB/s (0.63 of a copy), bound by
// instructions and their latency.  Ten CTAs of 128 threads an SM hold it to 48 registers; with 54 and four of 256 it takes 47 us, with twelve
// and 40 registers 41, but 8,000 tokens 5.4 us instead of 4.4.  The first form, with eight lanes to a group and a division for each
// code, took 182 us.
template <typename T, int GR>
__global__ void __launch_bounds__(128, GR == 4 ? 6 : 10) int4_append_kernel(const __grid_constant__ Int4RowsArgs a) {
  constexpr int DH = kInt4Group * GR;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int t = threadIdx.x & 3;
  Int4Row r{};
  const bool any = int4_row(a, DH, r);
  uint32_t u[GR][8];
#pragma unroll
  for (int y = 0; y < GR; ++y) {
    const uint8_t* src = r.row + 128 * y + 32 * t;
    if (any && a.wide) {
      ld_nc_256(src, u[y]);
    } else {
      const uint4 lo = any ? ld_nc_128(src) : make_uint4(0, 0, 0, 0), hi = any ? ld_nc_128(src + 16) : make_uint4(0, 0, 0, 0);
      u[y][0] = lo.x, u[y][1] = lo.y, u[y][2] = lo.z, u[y][3] = lo.w;
      u[y][4] = hi.x, u[y][5] = hi.y, u[y][6] = hi.z, u[y][7] = hi.w;
    }
  }
  uint32_t word[2 * GR], mine = 0;
#pragma unroll
  for (int y = 0; y < GR; ++y) {
    const uint32_t pair = int4_pair<T>(int4_extremes<T, 8, 4>(u[y]));
    const float2 sm = ElemTraits<T>::unpack2(pair);
    word[y] = int4_codes<T>(u[y], sm);
    word[GR + y] = int4_codes<T>(u[y] + 4, sm);
    if (y == t) mine = pair;
  }
  if (!any || !r.half) return;
  move_words<2 * GR>(reinterpret_cast<uint32_t*>(r.half + r.token * (DH / 2) + t * (8 * GR)), word);
  if (t < GR) *reinterpret_cast<uint32_t*>(r.half + 8 * DH + 4 * (r.token * GR + t)) = mine;
}

// Rows without a slot get zeros.  131,072 tokens x 2 heads of 128: 30 us for 172 MB, 5.8 TB/s (0.88 of a copy): HBM.
template <typename T, int GR>
__global__ void __launch_bounds__(128) int4_read_kernel(const __grid_constant__ Int4RowsArgs a) {
  constexpr int DH = kInt4Group * GR;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int t = threadIdx.x & 3;
  Int4Row r{};
  if (!int4_row(a, DH, r)) return;
  uint32_t word[2 * GR] = {}, pair[GR] = {};
  if (r.half) {
    move_words<2 * GR>(word, reinterpret_cast<const uint32_t*>(r.half + r.token * (DH / 2) + t * (8 * GR)));
    const uint32_t* p = reinterpret_cast<const uint32_t*>(r.half + 8 * DH + 4 * r.token * GR);
    if constexpr (GR == 1) pair[0] = *p;
    else move_words<GR>(pair, p);
  }
#pragma unroll
  for (int y = 0; y < GR; ++y) {
    const float2 sm = ElemTraits<T>::unpack2(pair[y]);
    uint32_t u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t w = word[(j >> 2) * GR + y];
      u[j] = ElemTraits<T>::pack2(int4_value(w, 2 * (j & 3), sm), int4_value(w, 2 * (j & 3) + 1, sm));
    }
    uint8_t* dst = r.row + 128 * y + 32 * t;
    if (a.wide) {
      st_256(dst, u);
    } else {
      st_128(dst, make_uint4(u[0], u[1], u[2], u[3]));
      st_128(dst + 16, make_uint4(u[4], u[5], u[6], u[7]));
    }
  }
}

// Launch that may be set up while the stream's previous kernel runs (the kernel waits for it).
template <typename Args>
int launch_dependent(void (*kern)(Args), const std::remove_const_t<Args>& a, dim3 grid, unsigned block, int smem, cudaStream_t s,
                     const char* what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, a), what);
}

}  // namespace

int launch_reserve(const int32_t* lens, const int32_t* add, int B, int32_t* table, int64_t table_stride, int width,
                   int32_t* free_pages, int num_pages, const int32_t* num_free, int page_size, int32_t* lens_out,
                   int32_t* num_free_out, uint8_t* granted, int64_t* slots, int32_t* positions, int64_t num_tokens,
                   cudaStream_t s) {
  if (B > kMaxRequests) return fail(BNA_UNSUPPORTED, "paged_reserve: at most 4096 requests per call");
  const bool aligned = ((reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(positions)) & 15) == 0;
  ReserveArgs a{lens, add, table, table_stride, free_pages, num_free, lens_out, num_free_out, granted, slots, positions,
                num_tokens, B, width, num_pages, page_size, aligned};
  // Four tokens a thread once one would need more than a CTA of 256 on every SM.  Small CTAs on many
  // SMs, as a token's searches keep the issue slots busy (33 CTAs of 1,024 threads took 6 us
  // over 131,072 tokens), unless the scan over the requests is the longer part.
  const int k = num_tokens > 256 * kReserveCtas ? 4 : 1;
  auto kern = k == 4 ? reserve_kernel<4> : reserve_kernel<1>;
  const unsigned threads = B > 1024 ? 1024 : 256;
  // What a launch may use unasked, 48 KB, covers the static warp sums too.
  const int smem = kRequestBytes * B;
  if (smem + kScanBytes > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRequestBytes * kMaxRequests);
    if (e != cudaSuccess) return check_cuda(e, "paged_reserve attributes");
  }
  // enough CTAs for the tokens and for every page the requests could give back (these in several
  // rounds: they are rarely many)
  const int64_t given = std::min((int64_t)num_pages, (int64_t)B * width) / 2;
  const int64_t items = std::max((num_tokens + k - 1) / k, std::max(given, (int64_t)B));
  const unsigned grid = (unsigned)std::min<int64_t>(kReserveCtas, (items + threads - 1) / threads);
  return launch_dependent(kern, a, dim3(grid), threads, smem, s, "paged_reserve launch");
}

int launch_paged_append(const bna_tensor4* k, const bna_tensor4* v, bna_tensor4* kp, bna_tensor4* vp,
                        const int64_t* slots, cudaStream_t s) {
  const int heads = (int)k->size[1];
  const int64_t rows = k->size[2] * heads;
  const int vecs = (int)(k->size[3] / 8), vec_shift = vecs == 8 ? 3 : vecs == 16 ? 4 : 5;
  PagedAppendArgs a{static_cast<const uint8_t*>(k->data), static_cast<const uint8_t*>(v->data),
                    static_cast<uint8_t*>(kp->data), static_cast<uint8_t*>(vp->data), k->stride[1], k->stride[2],
                    v->stride[1], v->stride[2], kp->stride[0], kp->stride[1], kp->stride[2], vp->stride[0],
                    vp->stride[1], vp->stride[2], slots, rows, kp->size[0] * kp->size[2], heads, (int)kp->size[2], vec_shift};
  // four rows a thread once that still fills the GPU; one row a thread has the shorter latency
  const int n = rows * vecs >= (int64_t)4 * 256 * 148 * 4 ? 4 : 1;
  const int64_t per = (int64_t)n * (256 >> vec_shift), blocks = (rows + per - 1) / per;
  if (blocks > INT_MAX) return fail(BNA_UNSUPPORTED, "paged_append: too many elements");
  return launch_dependent(n == 4 ? paged_append_kernel<4> : paged_append_kernel<1>, a, dim3((unsigned)blocks), 256, 0, s,
                          "paged_append launch");
}

// Rows of k / v into (append) or out of (read) 4-bit blocks.
int launch_int4_rows(bool append, const bna_tensor4* k, const bna_tensor4* v, bna_tensor4* pool, const int64_t* slots, int dtype, cudaStream_t s) {
  const bna_tensor4* x[2] = {k, v};
  Int4RowsArgs a{};
  a.pool = static_cast<uint8_t*>(pool->data);
  a.p_p = pool->stride[0], a.p_h = pool->stride[1], a.p_g = pool->stride[2];
  a.slots = slots;
  a.heads = (int)k->size[1], a.page_size = (int)pool->size[2] * kInt4Tokens;
  a.count = k->size[2] * a.heads, a.num_slots = pool->size[0] * a.page_size;
  a.wide = 1;
  for (int i = 0; i < 2; ++i) {
    a.rows[i] = static_cast<uint8_t*>(x[i]->data);
    a.h[i] = x[i]->stride[1], a.t[i] = x[i]->stride[2];
    if (reinterpret_cast<uintptr_t>(x[i]->data) % 32 || (x[i]->size[1] > 1 && a.h[i] % 16) || (x[i]->size[2] > 1 && a.t[i] % 16)) a.wide = 0;
  }
  // Short calls in small CTAs on many SMs (64 tokens x 2 heads: append 2.1, read 1.6 us with 64 threads, 2.3 and 1.8 with
  // 256); read of 131,072 tokens: 30 us with 128 threads, 36 with 64.
  const int block = a.count <= 64 * 148 ? 64 : 128;
  const int64_t blocks = (a.count + block / 4 - 1) / (block / 4);
  if (blocks > INT_MAX) return fail(BNA_UNSUPPORTED, "paged 4-bit rows: too many elements");
  auto pick = [&](auto t) -> void (*)(const Int4RowsArgs) {
    using T = decltype(t);
    switch (k->size[3]) {
      case 64: return append ? int4_append_kernel<T, 1> : int4_read_kernel<T, 1>;
      case 128: return append ? int4_append_kernel<T, 2> : int4_read_kernel<T, 2>;
      default: return append ? int4_append_kernel<T, 4> : int4_read_kernel<T, 4>;
    }
  };
  return launch_dependent(dtype == BNA_BF16 ? pick(__nv_bfloat16()) : pick(__half()), a, dim3((unsigned)blocks, 2), block, 0, s,
                          append ? "paged_append_int4 launch" : "paged_read_int4 launch");
}

}  // namespace bna
