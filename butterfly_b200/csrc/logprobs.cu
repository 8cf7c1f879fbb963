// logprobs.cu — log probability of a given token, entropy and likeliest alternatives of each row of logits:
//   lse = M + log Z,  Z = sum e^(x - M),  logprob = x[token] - lse,
//   H = -sum p log p = log Z - W / Z,  W = sum (x - M) e^(x - M),
// and the k largest entries, of equal ones the lowest index first.
//
// Each logit is read once from HBM and the rest is held in registers: a thread keeps (ref, Z, W) with a
// reference that moves only when an entry lies more than kSlack above it, and where its largest
// entry lies.  The k largest need no second pass over the row: of 64 groups of threads the k-th
// largest of their largest entries is a bound that at least k entries reach, and only the few threads
// whose own largest reaches it look at their entries again (from L2, a warp for each of them).
// A row is shared by a cluster of CTAs where there are few rows; the CTAs' sums and lists are joined
// through distributed shared memory by the cluster's first one.
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
constexpr int kMaxCluster = 8;
constexpr float kSlack = 8.f;  // e^kSlack times the row's length stays far below the fp32 range
constexpr float kLog2e = 1.4426950408889634f;
// e^kFloor is 0 in fp32; differences are cut there, so that a masked entry adds 0 to W and not 0 * inf
constexpr float kFloor = -120.f;
static_assert(kMaxCluster * kTop <= kList && kThreads % kTop == 0, "");

struct LogprobArgs {
  const uint8_t* x;
  int64_t ld, ld_outer;  // elements between rows, and between runs of `inner` rows
  int64_t inner;
  int V;
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
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b) {
  const float M = fmaxf(a.ref, b.ref);
  const Sums x = moved(a, M), y = moved(b, M);
  return {M, x.z + y.z, x.w + y.w};
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
    const T* row = reinterpret_cast<const T*>(base) + shift;
    uint32_t u[4];
    T* e = reinterpret_cast<T*>(u);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int64_t i = v * (int64_t)E + j - shift;
      e[j] = i >= 0 && i < V ? row[i] : static_cast<T>(-INFINITY);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  __device__ __forceinline__ float at(int64_t i) const {
    if constexpr (sizeof(T) == 4) return reinterpret_cast<const float*>(base)[shift + i];
    else return static_cast<float>(reinterpret_cast<const T*>(base)[shift + i]);
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) logprob_kernel(const LogprobArgs a, int cluster) {
  constexpr int E = Row<T>::E;
  __shared__ uint64_t list[kList];
  __shared__ uint64_t group[kTop], top[kTop];
  __shared__ Sums warp_sums[kWarps], cta_sums;
  __shared__ uint64_t bound;
  __shared__ int count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int part = cluster > 1 ? (int)cluster_ctarank() : 0;
  const int64_t r = blockIdx.x / cluster;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t outer = r / a.inner;
  const Row<T> row(a.x + (outer * a.ld_outer + (r - outer * a.inner) * a.ld) * (int64_t)sizeof(T), a.V);
  const int nv = row.vectors(), per = (nv + cluster - 1) / cluster;
  const int v0 = part * per, v1 = min(v0 + per, nv), first = v0 + tid;

  // the given token's logit, asked for first
  int64_t token = -1;
  float picked = -INFINITY;
  if (part == 0 && tid == 0 && a.tokens) {
    token = a.tokens64 ? static_cast<const int64_t*>(a.tokens)[r] : static_cast<const int32_t*>(a.tokens)[r];
    if (token >= 0 && token < a.V) picked = row.at(token);
  }

  Sums s{-INFINITY, 0.f, 0.f};
  float best = -INFINITY;
  int best_v = first;
  auto take = [&](const uint4& raw, int v) {
    float f[E];
    Row<T>::unpack(raw, f);
    float mx = f[0];
#pragma unroll
    for (int j = 1; j < E; ++j) mx = fmaxf(mx, f[j]);
    if (mx > best) {
      best = mx;
      best_v = v;
    }
    if (mx > s.ref + kSlack) s = moved(s, mx);
    const float base = s.ref == -INFINITY ? 0.f : s.ref;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float d = max_nan(f[j] - base, kFloor), e = ex2_approx(d * kLog2e);
      s.z += e;
      s.w = fmaf(d, e, s.w);
    }
  };
  constexpr int U = 4;  // vectors in flight
  for (int v = first; v < v1; v += U * kThreads) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * kThreads < v1) raw[u] = row.load(v + u * kThreads);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * kThreads < v1) take(raw[u], v + u * kThreads);
  }

  // sums of the CTA
  Sums t = s;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Sums other{__shfl_xor_sync(0xffffffffu, t.ref, o), __shfl_xor_sync(0xffffffffu, t.z, o), __shfl_xor_sync(0xffffffffu, t.w, o)};
    t = joined(t, other);
  }
  if (lane == 0) warp_sums[warp] = t;

  if (a.k > 0) {
    // Keys of what a thread could hold at best (the first entry of its best vector), and of what its
    // largest is at least (the last one).
    const bool any = first < v1;
    auto key_at = [&](int v, int j) { return key_of(best, (uint32_t)max((int64_t)0, v * (int64_t)E + j - row.shift)); };
    const uint64_t most = any ? key_at(best_v, 0) : 0, least = any ? key_at(best_v, E - 1) : 0;
    uint64_t g = least;
#pragma unroll
    for (int o = kThreads / kTop / 2; o > 0; o >>= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (lane % (kThreads / kTop) == 0) group[tid / (kThreads / kTop)] = g;
    if (tid == 0) {
      bound = 0;  // fewer than k threads have entries: all entries count
      count = 0;
    }
    if (tid < kTop) top[tid] = 0;
    __syncthreads();
    if (tid < kTop && group[tid] != 0) {
      int above = 0;
#pragma unroll 8
      for (int i = 0; i < kTop; ++i) above += group[i] > group[tid];
      if (above == a.k - 1) bound = group[tid];
    }
    __syncthreads();
    // Entries that reach the bound.  If they do not fit, the k-th largest of those that did is a higher
    // bound; each round leaves at least kList - k of them out, so the rounds end.
    int n;
    for (;;) {
      const uint64_t b = bound;
      unsigned todo = __ballot_sync(0xffffffffu, any && most >= b);
      while (todo) {
        const int owner = __ffs(todo) - 1;
        todo &= todo - 1;
        for (int v = v0 + warp * 32 + owner + lane * kThreads; v < v1; v += 32 * kThreads) {
          float f[E];
          Row<T>::unpack(row.load(v), f);
#pragma unroll
          for (int j = 0; j < E; ++j) {
            const int64_t i = v * (int64_t)E + j - row.shift;
            const uint64_t key = key_of(f[j], (uint32_t)i);
            if (i >= 0 && i < row.V && key >= b) {
              const int at = atomicAdd(&count, 1);
              if (at < kList) list[at] = key;
            }
          }
        }
      }
      __syncthreads();
      n = min(count, kList);
      const bool fits = count <= kList;
      for (int c = tid; c < n; c += kThreads) {
        int above = 0;
        for (int i = 0; i < n; ++i) above += list[i] > list[c];
        if (above < a.k) top[above] = list[c];
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
  }
  if (warp == 0) {
    t = lane < kWarps ? warp_sums[lane] : Sums{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Sums other{__shfl_xor_sync(0xffffffffu, t.ref, o), __shfl_xor_sync(0xffffffffu, t.z, o), __shfl_xor_sync(0xffffffffu, t.w, o)};
      t = joined(t, other);
    }
    if (lane == 0) cta_sums = t;
  }
  if (cluster == 1) {
    __syncthreads();
  } else {
    cluster_sync_all();  // (every thread of every CTA comes here)
    if (part == 0) {
      auto remote32 = [](const void* p, int rank) {
        uint32_t v;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
        return v;
      };
      for (int i = tid; i < cluster * a.k; i += kThreads) {
        const uint64_t* src = &top[i % a.k];
        uint64_t v;
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(smem_u32(src), i / a.k)) : "memory");
        list[i] = v;
      }
      Sums all = cta_sums;
      if (warp == 0) {
        const Sums mine = lane < cluster ? Sums{__uint_as_float(remote32(&cta_sums.ref, lane)), __uint_as_float(remote32(&cta_sums.z, lane)),
                                                __uint_as_float(remote32(&cta_sums.w, lane))}
                                         : Sums{-INFINITY, 0.f, 0.f};
        all = mine;
#pragma unroll
        for (int o = kMaxCluster / 2; o > 0; o >>= 1) {
          const Sums other{__shfl_xor_sync(0xffffffffu, all.ref, o), __shfl_xor_sync(0xffffffffu, all.z, o),
                           __shfl_xor_sync(0xffffffffu, all.w, o)};
          all = joined(all, other);
        }
      }
      __syncthreads();  // (the lists have been read before `top` is written again)
      if (tid == 0) cta_sums = all;
      for (int c = tid; c < cluster * a.k; c += kThreads) {
        int above = 0;
        for (int i = 0; i < cluster * a.k; ++i) above += list[i] > list[c];
        if (above < a.k && list[c] != 0) top[above] = list[c];
      }
      __syncthreads();
    }
  }
  if (part == 0) {
    const Sums all = cta_sums;
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
      a.top_ids[r * a.k + tid] = (int64_t)(uint32_t)~(uint32_t)key;
      a.top_lp[r * a.k + tid] = (value_of((uint32_t)(key >> 32)) - base) - log_z;
    }
  }
  if (cluster > 1) cluster_sync_all();  // no CTA ends while its shared memory may be read
}

template <typename T>
int launch(const LogprobArgs& a, int64_t rows, cudaStream_t s) {
  const int64_t vectors = ((int64_t)a.V + Row<T>::E - 1) / Row<T>::E;
  int cluster = 1;
  while (cluster < kMaxCluster && rows * cluster * 2 <= 2 * 148 && vectors >= (int64_t)2 * cluster * kThreads) cluster *= 2;
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
  const LogprobArgs a{static_cast<const uint8_t*>(x), ld, ld_outer, inner, V, tokens, tokens64, logprob, entropy, top_ids, top_lp, k};
  if (dtype == BNA_F32) return launch<float>(a, rows, s);
  return dtype == BNA_BF16 ? launch<__nv_bfloat16>(a, rows, s) : launch<__half>(a, rows, s);
}

}  // namespace bna
