// logprobs.cu — log probability of a given token, entropy and likeliest alternatives of each row of logits:
//   lse = M + log Z,  Z = sum e^(x - M),  logprob = x[token] - lse,
//   H = -sum p log p = log Z - W / Z,  W = sum (x - M) e^(x - M),
// and the k largest entries, of equal ones the lowest index first.
//
// Each logit is read once from HBM and the rest is held in registers: a thread keeps (ref, Z, W) with a
// reference that moves only when an entry lies more than kSlack above it, and where its largest
// entry lies.  The k largest need no second pass over the row: of 64 groups of threads the k-th
// largest of their largest entries is a bound that at least k entries reach.  A thread keeps in mind which vector
// holds its largest entry and reads that one again (from L2), and the few threads whose second-best vector reaches
// the bound too have all their entries looked at, by all lanes of their warp.
// Many short rows take a warp each (logprob_short_kernel).
// A row is shared by a cluster of CTAs where there are few rows; the CTAs' sums and lists are joined
// through distributed shared memory by the cluster's first one.
//
// Measured, with the likeliest entry: 4,096 rows of 151,936 in bf16 212 us at 1,965 MHz for 1.24 GB, 5.9 TB/s (0.90 of a copy; the issue
// slots are 67% and the exponential's pipe 56% busy); call after call, under the power cap at 1,700 MHz, 232 to 250 us.  512 threads and three CTAs an SM, so that the end of one row (bound,
// candidates, ranks) lies beside the reads of two others.  One row with 20 alternatives 7.8 us: latency.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "sm100.cuh"

namespace bna {
namespace {
using namespace sm100;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kTop = 64;      // alternatives at most, and groups of threads
constexpr int kList = 4096;   // entries that reach the bound, as long as they fit
constexpr int kFew = 512;     // of more candidates than this, those that a second bound leaves are ranked
constexpr int kMaxCluster = 8;
constexpr float kSlack = 8.f;  // e^kSlack times the row's length stays far below the fp32 range
constexpr float kLog2e = 1.4426950408889634f;
// Entries are cut from below (Low) as they are summed, so that a masked one adds 0 to W and not 0 * inf: what lies so far
// below the reference adds nothing else.  Where the reference itself is about as low, differences are cut
// instead: e^kFloor is 0 in fp32.
constexpr float kFloor = -120.f;

struct LogprobArgs {
  const uint8_t* x;
  int64_t ld, ld_outer;  // elements between rows, and between runs of `inner` rows
  int inner, V;
  const void* tokens;  // or null
  int tokens64;
  float *logprob, *entropy;
  int64_t* top_ids;
  float* top_lp;
  int k;
};

// Order-preserving map of a float to an unsigned integer (-0 as 0, NaN as -inf), and back.
__device__ __forceinline__ uint32_t rank_of(float f) {
  f = f == f ? f + 0.f : -INFINITY;
  const uint32_t u = __float_as_uint(f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t r) { return __uint_as_float(r ^ ((r >> 31) ? 0x80000000u : 0xffffffffu)); }
// (value, lowest index first) as one number; 0: none
__device__ __forceinline__ uint64_t key_of(float f, uint32_t idx) { return (uint64_t)rank_of(f) << 32 | (uint32_t)~idx; }

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Where entries are cut, below which reference the differences are cut instead, and (16 bits) maxima of two entries in a
// register.  A cut entry less the largest finite one is still finite.
template <typename T> struct Low;
template <> struct Low<float> {
  static constexpr float kLowest = -0x1p100f, kNear = -0x1p99f;
};
template <> struct Low<__nv_bfloat16> {
  static constexpr uint32_t kLowest = 0xfb00fb00u;  // -2^119
  static constexpr float kNear = -0x1p118f;
  __device__ static uint32_t top(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static uint32_t cut(uint32_t a) {
    uint32_t b = kLowest;
    const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};
template <> struct Low<__half> {
  static constexpr uint32_t kLowest = 0xfbfffbffu;  // -65504
  static constexpr float kNear = -6e4f;
  __device__ static uint32_t top(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static uint32_t cut(uint32_t a) {
    uint32_t b = kLowest;
    const __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};

// Z and W around a reference.  ref = -inf: no entry but masked ones (Z = W = 0).
struct Sums {
  float ref, z, w;
};
// The same sums around M >= ref.
__device__ __forceinline__ Sums moved(const Sums& s, float M) {
  if (s.ref == -INFINITY) return {M, s.z, s.w};  // (z is 0, or NaN where an entry was)
  const float d = s.ref - M, f = ex2_approx(d * kLog2e);
  return {M, s.z * f, f == 0.f ? s.w * f : (s.w + d * s.z) * f};
}
// All lanes' sums as one (in every lane).
__device__ __forceinline__ Sums warp_join(const Sums& s) {
  float M = s.ref;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const Sums x = moved(s, M);
  return {M, warp_sum(x.z), warp_sum(x.w)};
}
static_assert(kThreads % kTop == 0, "");
// The warp's keys' ranks: of the keys list[0 .. n) the number above `key`, counted by the eight lanes 8 i .. 8 i + 7 that hold
// the same key.
__device__ __forceinline__ int rank_in(const uint64_t* list, int n, uint64_t key, int lane) {
  int above = 0;
  for (int i = lane & 7; i < n; i += 8) above += list[i] > key;
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
  return above;
}

template <typename T>
struct Row {
  static constexpr int E = 16 / (int)sizeof(T);  // entries of a 16-byte vector
  const uint8_t* base;  // the row's start, down to a multiple of 16 bytes
  int shift, V;         // entries between that and the row's start; vector v holds entries v E - shift ..
  int whole0, whole1;   // vectors [whole0, whole1) lie inside the row

  __device__ Row(const uint8_t* p, int n) : V(n) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    base = reinterpret_cast<const uint8_t*>(a & ~(uintptr_t)15);
    shift = (int)(a & 15) / (int)sizeof(T);
    whole0 = shift > 0;
    whole1 = (int)(((int64_t)shift + V) / E);
  }
  __device__ int vectors() const { return (int)(((int64_t)shift + V + E - 1) / E); }
  __device__ static void unpack(const uint4& r, float (&f)[E]) {
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        f[i] = __uint_as_float(u[i]);
      } else {
        const float2 p = ElemTraits<T>::unpack2(u[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
      }
    }
  }
  // A vector; entries before and after the row are -inf, and are not read.
  __device__ __forceinline__ uint4 load(int v) const {
    if (v >= whole0 && v < whole1) return ld_128(base + 16 * (int64_t)v);
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = (int64_t)v * E + j * (E / 4) - shift;
      if constexpr (sizeof(T) == 4) u[j] = __float_as_uint(entry(i));
      else u[j] = ElemTraits<T>::pack2(entry(i), entry(i + 1));
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  __device__ __forceinline__ float entry(int64_t i) const { return i >= 0 && i < V ? at(i) : -INFINITY; }
  __device__ __forceinline__ float at(int64_t i) const {
    if constexpr (sizeof(T) == 4) return reinterpret_cast<const float*>(base)[shift + i];
    else return static_cast<float>(reinterpret_cast<const T*>(base)[shift + i]);
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 3) logprob_kernel(const LogprobArgs a, int cluster) {
  constexpr int E = Row<T>::E;
  // Shared memory is read and written an element at a time, each of its array's type and by an index into that array, here
  // and (all_top, all_sums) from the cluster's other CTAs, whose arrays lie at the same offsets.  Global memory: the row by 16 bytes at
  // multiples of 16 (base) or by its elements, tokens and results by theirs; the C call checks their pointers.
  alignas(8) __shared__ uint64_t list[kList], group[kTop], top[kTop], few[kFew], bound, few_bound;
  alignas(8) __shared__ uint64_t all_top[kMaxCluster * kTop];  // of the cluster's CTAs, in the first one
  alignas(4) __shared__ float sums[3][kWarps];  // ref, Z, W of the warps, then of the CTA in column 0
  alignas(4) __shared__ float all_sums[3][kMaxCluster];
  alignas(4) __shared__ int few_count, count, owners[kThreads];
  static_assert(alignof(uint64_t) == 8 && alignof(float) == 4 && 16 % sizeof(T) == 0 && E * sizeof(T) == 16, "");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int part = cluster > 1 ? (int)cluster_ctarank() : 0;
  const int r = (int)blockIdx.x / cluster;
  if (cluster > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int outer = r / a.inner;
  const Row<T> row(a.x + (outer * a.ld_outer + (r - outer * a.inner) * a.ld) * (int64_t)sizeof(T), a.V);
  const int nv = row.vectors(), per = (nv + cluster - 1) / cluster;
  const int v0 = part * per, v1 = min(v0 + per, nv), first = v0 + tid;

  // the given token, asked for before the row's entries, and its logit after them
  int64_t token = -1;
  if (part == 0 && tid == 0 && a.tokens)
    token = a.tokens64 ? static_cast<const int64_t*>(a.tokens)[r] : static_cast<const int32_t*>(a.tokens)[r];

  float ref = -INFINITY;
  Two z2 = two(0.f, 0.f), w2 = two(0.f, 0.f);  // Z and W of the entries at even and at odd places
  // the largest entry, its vector, and the largest of the other vectors
  float best = -INFINITY, second = -INFINITY;
  int best_v = first;
  auto take = [&](const uint4& raw, int v) {
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
    float mx;
    if constexpr (sizeof(T) == 4) {
      mx = fmaxf(fmaxf(__uint_as_float(u[0]), __uint_as_float(u[1])), fmaxf(__uint_as_float(u[2]), __uint_as_float(u[3])));
    } else {
      const float2 m = ElemTraits<T>::unpack2(Low<T>::top(Low<T>::top(u[0], u[1]), Low<T>::top(u[2], u[3])));
      mx = fmaxf(m.x, m.y);
    }
    second = fmaxf(second, fminf(mx, best));
    if (mx > best) {
      best = mx;
      best_v = v;
    }
    if (mx > ref + kSlack) {
      const float2 z = apart(z2), w = apart(w2);
      const Sums x = moved({ref, z.x, w.x}, mx), y = moved({ref, z.y, w.y}, mx);
      z2 = two(x.z, y.z);
      w2 = two(x.w, y.w);
      ref = mx;
    }
    if (ref < Low<T>::kNear) {  // (nothing but masked entries so far, by either kind of mask)
      float f[E];
      Row<T>::unpack(raw, f);
      const float base = ref == -INFINITY ? 0.f : ref;
#pragma unroll
      for (int j = 0; j < E; j += 2) {
        const float d0 = max_nan(f[j] - base, kFloor), d1 = max_nan(f[j + 1] - base, kFloor);
        const Two e = two(ex2_approx(d0 * kLog2e), ex2_approx(d1 * kLog2e));
        z2 = add2(z2, e);
        w2 = fma2(two(d0, d1), e, w2);
      }
      return;
    }
    const Two log2e = two(kLog2e, kLog2e);
#pragma unroll
    for (int j = 0; j < E / 2; ++j) {
      Two d;
      if constexpr (sizeof(T) == 4) {
        d = add2(two(max_nan(__uint_as_float(u[2 * j]), Low<T>::kLowest), max_nan(__uint_as_float(u[2 * j + 1]), Low<T>::kLowest)),
                 two(-ref, -ref));
      } else {
        const float2 f = halves_plus<T>(Low<T>::cut(u[j]), -ref);
        d = two(f.x, f.y);
      }
      const float2 t = apart(mul2(d, log2e));
      const Two e = two(ex2_approx(t.x), ex2_approx(t.y));
      z2 = add2(z2, e);
      w2 = fma2(d, e, w2);
    }
  };
  constexpr int U = 4;  // vectors in flight
  const int inside = min(v1, row.whole1);
  int v = first;
  if (v < row.whole0 && v < v1) {
    take(row.load(v), v);
    v += kThreads;
  }
  for (; v + (U - 1) * kThreads < inside; v += U * kThreads) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = ld_128(row.base + 16 * (int64_t)(v + u * kThreads));
#pragma unroll
    for (int u = 0; u < U; ++u) take(raw[u], v + u * kThreads);
  }
  for (; v < v1; v += kThreads) take(row.load(v), v);
  const float2 z = apart(z2), w = apart(w2);
  float picked = -INFINITY;
  if (token >= 0 && token < a.V) picked = row.at(token);

  // sums of the CTA
  Sums t = warp_join({ref, z.x + z.y, w.x + w.y});
  auto keep = [&](int column) {
    sums[0][column] = t.ref;
    sums[1][column] = t.z;
    sums[2][column] = t.w;
  };
  if (lane == 0) keep(warp);
  auto join_warps = [&]() {  // by one warp, after a barrier
    t = {-INFINITY, 0.f, 0.f};
    if (lane < kWarps) t = {sums[0][lane], sums[1][lane], sums[2][lane]};
    t = warp_join(t);
    __syncwarp();
    if (lane == 0) keep(0);
  };

  if (a.k > 0) {
    // Keys of what a thread could hold at best (the first entry of its best vector), and of what its
    // largest is at least (the last one).
    const bool any = first < v1;
    auto key_at = [&](int v, int j) { return key_of(best, (uint32_t)max((int64_t)0, v * (int64_t)E + j - row.shift)); };
    const uint64_t most = any ? key_at(best_v, 0) : 0, least = any ? key_at(best_v, E - 1) : 0;
    uint64_t g = least;
    if (v1 - v0 < kThreads || a.k > 16) {
      // Of threads side by side whole groups would have no vector, and with fewer groups than k all entries would
      // count; and in a masked end the k-th group's bound would be 64 k entries into it.  Threads 64 apart instead, for one more
      // barrier (1,000 entries, 20 alternatives: 40 -> 4.6 us; five rows of 151,936, a seventh masked, 64 alternatives 558 -> 30).
      list[tid] = least;
      __syncthreads();
      g = list[tid / (kThreads / kTop) + kTop * (tid % (kThreads / kTop))];
    }
    constexpr int kShare = kThreads / kTop;  // threads of a group, and threads that count the groups above one
    auto leave = [&](uint64_t x) {  // the group's largest
#pragma unroll
      for (int o = kShare / 2; o > 0; o >>= 1) x = max(x, __shfl_xor_sync(0xffffffffu, x, o));
      if (lane % kShare == 0) group[tid / kShare] = x;
    };
    auto kth = [&](uint64_t& to) {  // the k-th largest of the groups', if so many have one
      const uint64_t mine = group[tid / kShare];
      int above = 0;
#pragma unroll
      for (int i = 0; i < kTop / kShare; ++i) above += group[i * kShare + tid % kShare] > mine;
#pragma unroll
      for (int o = 1; o < kShare; o <<= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
      if (tid % kShare == 0 && mine != 0 && above == a.k - 1) to = mine;
    };
    leave(g);
    if (tid == 0) {
      bound = 0;  // fewer than k threads have entries: all entries count
      count = 0;
    }
    if (tid < kTop) top[tid] = 0;
    __syncthreads();
    kth(bound);
    if (warp == kWarps - 1) join_warps();
    __syncthreads();
    // Entries that reach the bound.  If they do not fit, the k-th largest of those that did is a higher
    // bound; each round leaves at least kList - k of them out, so the rounds end.
    int n;
    for (;;) {
      const uint64_t b = bound;
      auto look = [&](const uint4& raw, int v) {
        float f[E];
        Row<T>::unpack(raw, f);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const int64_t i = v * (int64_t)E + j - row.shift;
          const uint64_t key = key_of(f[j], (uint32_t)i);
          if (i >= 0 && i < row.V && key >= b) {
            const int at = atomicAdd(&count, 1);
            if (at < kList) list[at] = key;
          }
        }
      };
      // the vectors with the threads' largest entries (but where there was no entry above -inf) ...
      const bool kept = best > -INFINITY;
      if (any && kept && most >= b) look(row.load(best_v), best_v);
      // ... and of threads that hold more, all vectors are read again, shared out over the warp's lanes
      const bool more = any && key_of(kept ? second : best, 0) >= b;
      const unsigned todo = __ballot_sync(0xffffffffu, more);
      if (more) owners[32 * warp + __popc(todo & ((1u << lane) - 1))] = tid;
      if (todo) {
        const int skip = kept ? best_v : -1;
        __syncwarp();
        const int span = (v1 - v0 + kThreads - 1) / kThreads, items = __popc(todo) * span;
        for (int it0 = 0; it0 < items; it0 += 32) {
          const int it = it0 + lane, who = min(it, items - 1) / span, owner = owners[32 * warp + who];
          const int v = v0 + owner + (it - who * span) * kThreads;
          const int done = __shfl_sync(0xffffffffu, skip, owner & 31);  // the vector looked at already
          if (it < items && v < v1 && v != done) look(row.load(v), v);
        }
        __syncwarp();
      }
      __syncthreads();
      n = min(count, kList);
      const bool fits = count <= kList;
      // Ranking takes n^2 steps; where masks left many groups without another entry n is large, and the k-th largest of 64
      // groups of candidates is a higher bound (2,939 rows of 4,233, 604 of them masked, 64 alternatives: 10.7 -> 0.12 ms).
      const uint64_t* from = list;
      if (n > kFew) {
        uint64_t x = 0;
        // (places 64 apart: the list is partly in order, and then the first k places are those of k groups)
        for (int c = tid / kShare + kTop * (tid % kShare); c < n; c += kThreads) x = max(x, list[c]);
        leave(x);
        if (tid == 0) few_count = 0;
        __syncthreads();
        kth(few_bound);
        __syncthreads();
        for (int c = tid; c < n; c += kThreads)
          if (list[c] >= few_bound) {
            const int at = atomicAdd(&few_count, 1);
            if (at < kFew) few[at] = list[c];
          }
        __syncthreads();
        if (few_count <= kFew) {
          from = few;
          n = few_count;
        }
      }
      for (int c0 = 0; c0 < n; c0 += kThreads / 8) {
        const int c = c0 + tid / 8;
        const uint64_t key = c < n ? from[c] : 0;
        const int above = rank_in(from, n, key, lane);
        if (c < n && (lane & 7) == 0 && above < a.k) top[above] = key;
      }
      __syncthreads();
      if (fits) break;
      if (tid == 0) {
        bound = top[a.k - 1];
        count = 0;
      }
      __syncthreads();
    }
  } else {
    __syncthreads();
    if (warp == kWarps - 1) join_warps();
  }
  if (cluster == 1) {
    __syncthreads();
  } else {
    // each CTA leaves its sums and its list in the first one's shared memory
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // (all of them run by now)
    if (tid < a.k)
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mapa_shared(smem_u32(&all_top[part * a.k + tid]), 0)), "l"(top[tid]) : "memory");
    if (tid == kThreads - 32) {  // (whose warp joined the sums)
      const float x[3] = {t.ref, t.z, t.w};
#pragma unroll
      for (int i = 0; i < 3; ++i)
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(smem_u32(&all_sums[i][part]), 0)), "f"(x[i]) : "memory");
    }
    cluster_sync_all();  // (every thread of every CTA comes here)
    if (part == 0) {
      if (warp == kWarps - 1) {
        t = {-INFINITY, 0.f, 0.f};
        if (lane < cluster) t = {all_sums[0][lane], all_sums[1][lane], all_sums[2][lane]};
        t = warp_join(t);
        if (lane == 0) keep(0);
      }
      for (int c0 = 0; c0 < cluster * a.k; c0 += kThreads / 8) {
        const int c = c0 + tid / 8;
        const uint64_t key = c < cluster * a.k ? all_top[c] : 0;
        const int above = rank_in(all_top, cluster * a.k, key, lane);
        if (key != 0 && (lane & 7) == 0 && above < a.k) top[above] = key;
      }
      __syncthreads();
    }
  }
  if (part == 0) {
    const Sums all{sums[0][0], sums[1][0], sums[2][0]};
    // a row of masked entries only: no distribution; log probabilities -inf, entropy 0
    const bool none = all.z == 0.f;
    const float base = none ? 0.f : all.ref, log_z = none ? 0.f : logf(all.z);
    if (tid == 0) {
      if (a.logprob) a.logprob[r] = token < 0 ? 0.f : (picked - base) - log_z;
      const float h = none ? 0.f : log_z - all.w / all.z;
      a.entropy[r] = h < 0.f ? 0.f : h;  // (a rounding below 0)
    }
    if (tid < a.k) {
      const uint64_t key = top[tid];
      a.top_ids[(int64_t)r * a.k + tid] = (int64_t)(uint32_t)~(uint32_t)key;
      a.top_lp[(int64_t)r * a.k + tid] = (value_of((uint32_t)(key >> 32)) - base) - log_z;
    }
  }
}

// Rows of up to kShort entries, a warp to each, held in registers: the sums around the row's maximum, then the rank of the k-th
// largest entry by bisection (a count over the warp each), the entries above it and the first of those that equal it.  65,536 rows of 1,000 in
// bf16: 82 us without alternatives, 242 with 5, 348 with 64 (131 MB: 20 us of a copy).  Without alternatives bound by loads that nothing
// covers (17 warps an SM, issue slots 38% busy), with them by four times the instructions and their fetch (50%).
constexpr int kShort = 1024, kShortWarps = 4;
template <typename T>
__global__ void __launch_bounds__(32 * kShortWarps) logprob_short_kernel(const LogprobArgs a, int rows) {
  constexpr int E = Row<T>::E, N = kShort / 32 / E;
  // ranks without the bits that no entry of the type sets
  constexpr int kDrop = std::is_same<T, __nv_bfloat16>::value ? 16 : std::is_same<T, __half>::value ? 13 : 0;
  alignas(8) __shared__ uint64_t picks[kShortWarps][kTop];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t r64 = (int64_t)blockIdx.x * kShortWarps + warp;
  if (r64 >= rows) return;
  const int r = (int)r64, outer = r / a.inner;
  const Row<T> row(a.x + (outer * a.ld_outer + (r - outer * a.inner) * a.ld) * (int64_t)sizeof(T), a.V);
  const int nv = row.vectors();  // (32 N at most)
  int64_t token = -1;
  if (a.tokens) token = a.tokens64 ? static_cast<const int64_t*>(a.tokens)[r] : static_cast<const int32_t*>(a.tokens)[r];
  float f[N][E];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int v = lane + 32 * i;
    if (v < nv) {
      Row<T>::unpack(row.load(v), f[i]);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) f[i][j] = -INFINITY;
    }
  }
  const float picked = token >= 0 && token < a.V ? row.at(token) : -INFINITY;
  float M = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < E; ++j) M = fmaxf(M, f[i][j]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  float base = M == -INFINITY ? 0.f : M;
  Two z2 = two(0.f, 0.f), w2 = two(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (32 * i >= nv) break;
#pragma unroll
    for (int j = 0; j < E; j += 2) {
      const float d0 = max_nan(f[i][j] - base, kFloor), d1 = max_nan(f[i][j + 1] - base, kFloor);
      const Two e = two(ex2_approx(d0 * kLog2e), ex2_approx(d1 * kLog2e));
      z2 = add2(z2, e);
      w2 = fma2(two(d0, d1), e, w2);
    }
  }
  const float2 za = apart(z2), wa = apart(w2);
  const float z = warp_sum(za.x + za.y), w = warp_sum(wa.x + wa.y);
  const bool none = z == 0.f;  // (a row of masked entries only)
  const float log_z = none ? 0.f : logf(z);
  if (none) base = 0.f;
  if (lane == 0) {
    if (a.logprob) a.logprob[r] = token < 0 ? 0.f : (picked - base) - log_z;
    const float h = none ? 0.f : log_z - w / z;
    a.entropy[r] = h < 0.f ? 0.f : h;  // (a rounding below 0)
  }
  if (a.k == 0) return;

  // ranks, 0 beside the row (any entry's is above that); the smallest of the largest of 32 or 64 groups is reached
  // by k entries
  uint32_t u[N][E], lo = 0, hi = 0, least = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = (lane + 32 * i) * E - row.shift;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      u[i][j] = at + j >= 0 && at + j < a.V ? rank_of(f[i][j]) >> kDrop : 0u;
      lo = max(lo, u[i][j]);
    }
    if (i % (N / 2) == N / 2 - 1) {
      least = a.k > 32 ? min(least, lo) : max(hi, lo);
      hi = max(hi, lo);
      lo = 0;
    }
  }
  lo = __reduce_min_sync(0xffffffffu, least);
  hi = __reduce_max_sync(0xffffffffu, hi);
  auto reach = [&](uint32_t x) {  // entries that reach x
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (32 * i < nv) {
#pragma unroll
        for (int j = 0; j < E; ++j) n += u[i][j] >= x;
      }
    return __reduce_add_sync(0xffffffffu, n);
  };
  int n = -1;  // of those that reach lo, where it has been counted
  while (lo < hi && n != a.k) {
    const uint32_t mid = lo + (hi - lo + 1) / 2;
    const int c = reach(mid);
    if (c >= a.k) {
      lo = mid;
      n = c;
    } else {
      hi = mid - 1;
    }
  }
  if (n < 0) n = reach(lo);
  // the k entries into the list: with ties too many first those above, then the ties in the order of their indices
  int count = 0;
  auto append = [&](bool ties, bool above) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (32 * i >= nv) break;
      int mine = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) mine += (above && u[i][j] > lo) || (ties && u[i][j] == lo);
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
      }
      int to = count + incl - mine;
#pragma unroll
      for (int j = 0; j < E; ++j)
        if ((above && u[i][j] > lo) || (ties && u[i][j] == lo)) {
          if (to < a.k) picks[warp][to] = key_of(f[i][j], (uint32_t)((lane + 32 * i) * E + j - row.shift));
          ++to;
        }
      count += __shfl_sync(0xffffffffu, incl, 31);
    }
  };
  if (n == a.k) {
    append(true, true);
  } else {
    append(false, true);
    append(true, false);
  }
  __syncwarp();
#pragma unroll
  for (int x = 0; x < kTop; x += 32) {
    if (x >= a.k) break;
    const uint64_t key = x + lane < a.k ? picks[warp][x + lane] : 0;
    int above = 0;
    for (int i = 0; i < a.k; ++i) above += picks[warp][i] > key;
    if (x + lane < a.k) {
      a.top_ids[(int64_t)r * a.k + above] = (int64_t)(uint32_t)~(uint32_t)key;
      a.top_lp[(int64_t)r * a.k + above] = (value_of((uint32_t)(key >> 32)) - base) - log_z;
    }
  }
}

template <typename T>
int launch(const LogprobArgs& a, int64_t rows, cudaStream_t s) {
  if (rows > INT_MAX) return fail(BNA_UNSUPPORTED, "token_logprobs: too many rows");
  const int64_t vectors = ((int64_t)a.V + Row<T>::E - 1) / Row<T>::E;
  constexpr int kWave = 3 * 148;  // rows that the CTAs of the other form hold at once
  // Short rows (one that begins inside a vector has E - 1 places before it at most) to a warp each where there are more of them than
  // CTAs at once, or alternatives for most of the groups, or groups without a vector; else the CTAs' latency is the shorter one.  A warp /
  // a CTA each, rows of 1,000: 65,536 with 64 alternatives 348 us / 15 ms, 444 with 64 12 / 28 us, 444 with 5 8.6 / 6.8, one in fp32
  // with 20 6.6 / 4.2.
  if (a.V <= kShort - (Row<T>::E - 1) && (rows > kWave || vectors < kTop || a.k > kTop / 2)) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((rows + kShortWarps - 1) / kShortWarps));
    cfg.blockDim = dim3(32 * kShortWarps);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return check_cuda(cudaLaunchKernelEx(&cfg, logprob_short_kernel<T>, a, (int)rows), "token_logprobs launch");
  }
  // A row to several CTAs as long as there is an SM for each and eight vectors a thread to share: 20 alternatives of one row of
  // 151,936 take 7.8 us with eight CTAs and 12.6 with one, of 40 rows 10.4 with two each and 13.3; 64 rows of 32,000 take
  // 6.5 us with one CTA each and 7.5 with two.
  int cluster = 1;
  while (cluster < kMaxCluster && rows * cluster * 2 <= 148 && vectors >= (int64_t)8 * cluster * kThreads) cluster *= 2;
  if (rows * cluster > INT_MAX) return fail(BNA_UNSUPPORTED, "token_logprobs: too many rows");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, logprob_kernel<T>, a, cluster), "token_logprobs launch");
}

}  // namespace

int launch_token_logprobs(const void* x, int64_t ld, int64_t ld_outer, int64_t rows, int64_t inner, int V, int dtype, const void* tokens,
                          int tokens64, float* logprob, float* entropy, int64_t* top_ids, float* top_lp, int k, cudaStream_t s) {
  const LogprobArgs a{static_cast<const uint8_t*>(x), ld, ld_outer, (int)std::min(inner, std::min(rows, (int64_t)INT_MAX)), V, tokens, tokens64, logprob, entropy, top_ids, top_lp, k};
  if (dtype == BNA_F32) return launch<float>(a, rows, s);
  return dtype == BNA_BF16 ? launch<__nv_bfloat16>(a, rows, s) : launch<__half>(a, rows, s);
}

}  // namespace bna
