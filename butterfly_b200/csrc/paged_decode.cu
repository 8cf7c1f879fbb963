// paged_decode.cu — attention of one new token per request over a paged key/value cache.
//   s_j = scale * q . k_j   for keys j in [max(0, len - window), len)
//   out = sum_j softmax(s)_j v_j,   lse = log sum_j exp(s_j);  no key: out = 0, lse = -inf
#include <cuda_runtime.h>

#include <cmath>
#include <string>
#include <type_traits>

#include "common.cuh"

namespace bna {
namespace {

constexpr int kWarps = 8;
// Query heads of one KV head served by a CTA (the partial outputs fit 32 KB of shared memory).
__host__ __device__ constexpr int rows_of(int dh) { return dh > 128 ? 4 : 8; }

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
  float scale_log2;
};

// One CTA per (request, KV head, group of up to 8 of its query heads); each warp walks every
// 8th key with an online softmax (a lane holds head_dim / 32 dims), and the warps' partial
// (max, sum, output) are joined through shared memory.
template <typename T, int DH>
__global__ void __launch_bounds__(kWarps * 32) paged_decode_kernel(const PagedArgs a) {
  constexpr int E = DH / 32, kRows = rows_of(DH);
  __shared__ float sm_m[kWarps][kRows], sm_l[kWarps][kRows], sm_o[kWarps][kRows][DH];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x, h = blockIdx.y, r0 = blockIdx.z * kRows;
  const int rows = min(kRows, a.G - r0);
  int64_t len = max(a.lens[b], 0);
  len = min(len, (int64_t)a.width * a.page_size);
  const int64_t lo = a.window > 0 ? max((int64_t)0, len - a.window) : 0;
  float q[kRows][E], o[kRows][E], m[kRows], l[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      o[r][e] = 0.f;
      const T* row = reinterpret_cast<const T*>(a.q) + b * a.q_b + (h * a.G + r0 + min(r, rows - 1)) * a.q_h;
      q[r][e] = (float)row[lane * E + e];
    }
  }
  for (int64_t j = lo + warp; j < len; j += kWarps) {
    const int page = a.table[b * a.table_stride + j / a.page_size];
    const int64_t off = j % a.page_size;
    const bool inside = page >= 0 && page < a.num_pages;  // a page outside the pool reads as zeros
    const bool fresh = a.kn && j == len - 1 && (!a.active || a.active[b]);
    T* kr = reinterpret_cast<T*>(a.kp) + page * a.kp_p + h * a.kp_h + off * a.kp_t + lane * E;
    T* vr = reinterpret_cast<T*>(a.vp) + page * a.vp_p + h * a.vp_h + off * a.vp_t + lane * E;
    float kf[E], vf[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (fresh) {
        const T kx = reinterpret_cast<const T*>(a.kn)[b * a.kn_b + h * a.kn_h + lane * E + e];
        const T vx = reinterpret_cast<const T*>(a.vn)[b * a.vn_b + h * a.vn_h + lane * E + e];
        kf[e] = (float)kx;
        vf[e] = (float)vx;
        if (inside && blockIdx.z == 0) {
          kr[e] = kx;
          vr[e] = vx;
        }
      } else {
        kf[e] = inside ? (float)kr[e] : 0.f;
        vf[e] = inside ? (float)vr[e] : 0.f;
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(q[r][e], kf[e], s);
      s = warp_sum(s) * a.scale_log2;
      const float mn = fmaxf(m[r], s), base = mn == -INFINITY ? 0.f : mn;
      const float alpha = ex2_approx(m[r] - base), p = ex2_approx(s - base);
      m[r] = mn;
      l[r] = l[r] * alpha + p;
#pragma unroll
      for (int e = 0; e < E; ++e) o[r][e] = fmaf(o[r][e], alpha, p * vf[e]);
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (lane == 0) {
      sm_m[warp][r] = m[r];
      sm_l[warp][r] = l[r];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sm_o[warp][r][lane * E + e] = o[r][e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * DH; i += blockDim.x) {
    const int r = i / DH, d = i - r * DH;
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w][r]);
    const float base = M == -INFINITY ? 0.f : M;
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2_approx(sm_m[w][r] - base);
      L += sm_l[w][r] * f;
      O += sm_o[w][r][d] * f;
    }
    const int hq = h * a.G + r0 + r;
    const uint32_t u = ElemTraits<T>::pack2(L == 0.f ? 0.f : O / L, 0.f);
    *reinterpret_cast<uint16_t*>(a.out + 2 * (b * a.o_b + hq * a.o_h + d)) = (uint16_t)u;
    if (a.lse && d == 0) a.lse[b * a.ls_b + hq * a.ls_h] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
  }
}

}  // namespace

int launch_paged_decode(const bna_tensor4* q, bna_tensor4* kp, bna_tensor4* vp, const bna_tensor4* kn,
                        const bna_tensor4* vn, const uint8_t* active, bna_tensor4* out, float* lse, int64_t ls_b, int64_t ls_h, int dtype,
                        const int32_t* table, int64_t table_stride, int width, const int32_t* lens, int window,
                        float scale, cudaStream_t s) {
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
  a.scale_log2 = scale * 1.4426950408889634f;
  const int kRows = rows_of((int)q->size[3]);
  const dim3 grid((unsigned)a.B, (unsigned)a.Hkv, (unsigned)((a.G + kRows - 1) / kRows));
  auto launch = [&](auto kern) { kern<<<grid, kWarps * 32, 0, s>>>(a); };
  const bool bf = dtype == BNA_BF16;
  switch (q->size[3]) {
    case 64: bf ? launch(paged_decode_kernel<__nv_bfloat16, 64>) : launch(paged_decode_kernel<__half, 64>); break;
    case 128: bf ? launch(paged_decode_kernel<__nv_bfloat16, 128>) : launch(paged_decode_kernel<__half, 128>); break;
    case 256: bf ? launch(paged_decode_kernel<__nv_bfloat16, 256>) : launch(paged_decode_kernel<__half, 256>); break;
    default: return fail(BNA_UNSUPPORTED, "paged_decode_attention: head_dim must be 64, 128 or 256");
  }
  return check_cuda(cudaGetLastError(), "paged_decode launch");
}

}  // namespace bna
