// paged_cache.cu — the write side of a paged key/value cache: pages for the next tokens
// (block tables and slot maps from the requests' lengths) and the tokens' rows into them.
// Pools are [pages, kv heads, page_size, head_dim]; a request's tokens 0..len-1 lie in the pages
// its block-table row names, page_size to a page; slot = page * page_size + offset.
#include <cuda_runtime.h>

#include <climits>
#include <string>

#include "common.cuh"

namespace bna {
namespace {

constexpr int kMaxRequests = 4096;  // three prefix sums and the lengths of a call: 64 KB of shared memory
constexpr int kReserveThreads = 256;

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

__device__ __forceinline__ int pages_of(int64_t tokens, int page_size) {
  return (int)((tokens + page_size - 1) / page_size);
}

// What a request asks for: its length after the call, and pages taken (need) or given back.
struct Ask {
  int len, add, old_pages, new_pages, need, back;
  int64_t want;
  bool fits;
};
__device__ __forceinline__ Ask ask_of(const ReserveArgs& a, int b) {
  Ask r;
  // a length outside the table is cut to it, so that no later index leaves the row
  r.len = min(max(a.lens[b], 0), (int)min((int64_t)a.width * a.page_size, (int64_t)INT_MAX));
  r.add = a.add[b];
  r.want = max((int64_t)0, (int64_t)r.len + r.add);
  r.old_pages = pages_of(r.len, a.page_size);
  r.fits = r.want <= (int64_t)a.width * a.page_size && r.want <= INT_MAX;
  r.new_pages = r.fits ? pages_of(r.want, a.page_size) : r.old_pages;
  r.need = r.add > 0 && r.fits ? r.new_pages - r.old_pages : 0;
  r.back = r.add < 0 ? r.old_pages - r.new_pages : 0;
  return r;
}

// One CTA.  Prefix sums over the requests of the tokens added, the pages needed and the pages
// given back (shared memory), from which every table entry, slot and stack entry follows by a
// binary search; the j-th page given back lies j below the new top of the free stack and the
// i-th page taken comes from i below it, so a call followed by its opposite restores the stack.
__global__ void __launch_bounds__(kReserveThreads) reserve_kernel(const ReserveArgs a) {
  extern __shared__ int32_t sm[];
  int32_t* cum_add = sm;                 // inclusive prefix sums
  int32_t* cum_need = sm + a.B;
  int32_t* cum_back = sm + 2 * a.B;
  if (threadIdx.x == 0) {
    int64_t ca = 0, cn = 0, cb = 0;
    for (int b = 0; b < a.B; ++b) {
      const Ask r = ask_of(a, b);
      ca += max(r.add, 0);
      cn += r.need;
      cb += r.back;
      cum_add[b] = (int32_t)min(ca, (int64_t)INT_MAX);
      cum_need[b] = (int32_t)min(cn, (int64_t)INT_MAX);
      cum_back[b] = (int32_t)min(cb, (int64_t)INT_MAX);
    }
  }
  __syncthreads();
  const int n = min(max(a.num_free[0], 0), a.num_pages);
  const int R = cum_back[a.B - 1];
  const int64_t top = (int64_t)n + R;
  // requests are served in order while their pages last: pages taken = the largest prefix <= top
  const int served = upper_bound(cum_need, a.B, top);
  const int A = served > 0 ? cum_need[served - 1] : 0;

  // Page x below the top of the stack with the pages given back on it.
  auto from_top = [&](int64_t x) -> int {
    if (x < R) {
      const int b = upper_bound(cum_back, a.B, x);
      const Ask r = ask_of(a, b);
      return a.table[b * a.table_stride + r.new_pages + (x - (cum_back[b] - r.back))];
    }
    const int64_t i = top - 1 - x;
    return i >= 0 && i < n ? a.free_pages[i] : -1;
  };
  auto granted = [&](const Ask& r, int b) { return r.add > 0 && r.fits && (r.need == 0 || cum_need[b] <= top); };

  for (int b = threadIdx.x; b < a.B; b += blockDim.x) {
    const Ask r = ask_of(a, b);
    const bool ok = granted(r, b);
    a.lens_out[b] = ok || r.add <= 0 ? (int)r.want : r.len;
    a.granted[b] = ok;
  }
  if (threadIdx.x == 0) a.num_free_out[0] = (int)min(top - A, (int64_t)a.num_pages);
  // table entries of the pages taken
  for (int i = threadIdx.x; i < A; i += blockDim.x) {
    const int b = upper_bound(cum_need, a.B, i);
    const Ask r = ask_of(a, b);
    a.table[b * a.table_stride + r.old_pages + (i - (cum_need[b] - r.need))] = from_top(i);
  }
  // stack entries of the pages given back and not taken again (from index n up; a page taken
  // comes from below n only when every page given back was taken, so no entry is read here
  // that is written here)
  for (int64_t i = n + threadIdx.x; i < top - A && i < a.num_pages; i += blockDim.x) a.free_pages[i] = from_top(top - 1 - i);
  // slots and positions of the added tokens, packed request by request
  for (int64_t t = threadIdx.x; t < a.num_tokens; t += blockDim.x) {
    int64_t slot = -1;
    int pos = -1;
    const int b = upper_bound(cum_add, a.B, t);
    if (b < a.B) {
      const Ask r = ask_of(a, b);
      if (granted(r, b)) {
        pos = (int)(r.len + (t - (cum_add[b] - r.add)));
        const int pi = pos / a.page_size;
        const int page = pi < r.old_pages ? a.table[b * a.table_stride + pi]
                                          : from_top(cum_need[b] - r.need + pi - r.old_pages);
        slot = page < 0 ? -1 : (int64_t)page * a.page_size + pos % a.page_size;
      }
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
  }
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
  int heads, page_size, vecs;  // 16-byte vectors per row
};

// One thread per 16-byte vector of a (token, head) row, of the keys and of the values.
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedAppendArgs a) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t row = i / a.vecs;
  const int c = (int)(i - row * a.vecs);
  if (row >= a.rows) return;
  const int64_t t = row / a.heads;
  const int h = (int)(row - t * a.heads);
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.num_slots) return;
  const int64_t page = slot / a.page_size, off = slot - page * a.page_size;
  st_128(a.kp + 2 * (page * a.kp_p + h * a.kp_h + off * a.kp_t) + 16 * c, ld_128(a.k + 2 * (t * a.k_t + h * a.k_h) + 16 * c));
  st_128(a.vp + 2 * (page * a.vp_p + h * a.vp_h + off * a.vp_t) + 16 * c, ld_128(a.v + 2 * (t * a.v_t + h * a.v_h) + 16 * c));
}

}  // namespace

int launch_reserve(const int32_t* lens, const int32_t* add, int B, int32_t* table, int64_t table_stride, int width,
                   int32_t* free_pages, int num_pages, const int32_t* num_free, int page_size, int32_t* lens_out,
                   int32_t* num_free_out, uint8_t* granted, int64_t* slots, int32_t* positions, int64_t num_tokens,
                   cudaStream_t s) {
  if (B > kMaxRequests) return fail(BNA_UNSUPPORTED, "paged_reserve: at most 4096 requests per call");
  ReserveArgs a{lens, add, table, table_stride, free_pages, num_free, lens_out, num_free_out, granted, slots, positions,
                num_tokens, B, width, num_pages, page_size};
  const int smem = 3 * B * 4;
  cudaFuncSetAttribute(reserve_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * kMaxRequests * 4);
  reserve_kernel<<<1, kReserveThreads, smem, s>>>(a);
  return check_cuda(cudaGetLastError(), "paged_reserve launch");
}

int launch_paged_append(const bna_tensor4* k, const bna_tensor4* v, bna_tensor4* kp, bna_tensor4* vp,
                        const int64_t* slots, cudaStream_t s) {
  const int heads = (int)k->size[1];
  const int64_t rows = k->size[2] * heads;
  const int vecs = (int)(k->size[3] / 8);
  PagedAppendArgs a{static_cast<const uint8_t*>(k->data), static_cast<const uint8_t*>(v->data),
                    static_cast<uint8_t*>(kp->data), static_cast<uint8_t*>(vp->data), k->stride[1], k->stride[2],
                    v->stride[1], v->stride[2], kp->stride[0], kp->stride[1], kp->stride[2], vp->stride[0],
                    vp->stride[1], vp->stride[2], slots, rows, kp->size[0] * kp->size[2], heads, (int)kp->size[2], vecs};
  const int64_t blocks = (rows * vecs + 255) / 256;
  if (blocks > INT_MAX) return fail(BNA_UNSUPPORTED, "paged_append: too many elements");
  paged_append_kernel<<<(unsigned)blocks, 256, 0, s>>>(a);
  return check_cuda(cudaGetLastError(), "paged_append launch");
}

}  // namespace bna
