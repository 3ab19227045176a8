// paged_attention.cu — attention of one new token per request over its pages
// (sx_paged_attention).
//
// One CTA of 8 warps per (request, kv head). Each warp takes every eighth key: lanes split the
// head dimension, the scores of the group's query heads are shuffle sums, and a running
// maximum m, sum l and output o per head fold the keys in one pass:
//   m' = max(m, s), l' = l 2^(m - m') + 2^(s - m'), o' = o 2^(m - m') + 2^(s - m') v,
// with s in units of log 2. The warps' (m, l, o) are joined the same way through shared memory.
#include <cuda_runtime.h>

#include "paged.hpp"
#include "sx_device.cuh"
#include "sx_internal.hpp"

namespace sx {
namespace {

constexpr int kWarps = 8;

struct AttnK {
  const uint8_t* q;
  uint8_t* out;
  float* lse;
  const uint8_t *k, *v;
  const int *table, *lens;
  int* status;
  long long q_stride, out_stride;                    // elements
  long long page_stride, head_stride, token_stride;  // elements
  long long table_stride;
  int n, Hkv, G, H, page_shift, width, n_pages;
  float scale;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <int HD, typename QT, typename CT, int GM>
__global__ void __launch_bounds__(kWarps * 32) k_paged_attention(const AttnK a) {
  constexpr int E = HD / 32;
  extern __shared__ __align__(16) float smem[];  // [kWarps][GM][HD + 2]
  pdl_launch_dependents();
  pdl_wait();
  const int i = blockIdx.x / a.Hkv, h = blockIdx.x % a.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int len = max(0, ld_cg(a.lens + i));
  const long long cap = (long long)a.width << a.page_shift;
  if (len > cap) {
    len = (int)cap;
    if (a.status && threadIdx.x == 0) *a.status = SX_E_RANGE;
  }
  float q[GM][E], o[GM][E], m[GM], l[GM];
  const QT* qp = reinterpret_cast<const QT*>(a.q) + (size_t)i * a.q_stride + (size_t)h * a.G * HD;
#pragma unroll
  for (int g = 0; g < GM; g++) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) {
      q[g][e] = g < a.G ? to_f32(qp[(size_t)g * HD + lane + 32 * e]) : 0.f;
      o[g][e] = 0.f;
    }
  }
  const float sl2 = a.scale * 1.4426950408889634f;
  for (int t = warp; t < len; t += kWarps) {
    const int page = ld_cg(a.table + (size_t)i * a.table_stride + (t >> a.page_shift));
    const bool there = (unsigned)page < (unsigned)a.n_pages;
    if (!there && a.status && lane == 0) *a.status = SX_E_RANGE;
    const size_t at = there ? (size_t)page * a.page_stride + (size_t)h * a.head_stride +
                                  (size_t)(t & ((1 << a.page_shift) - 1)) * a.token_stride
                            : 0;
    float kv[E], vv[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
      kv[e] = there ? to_f32(reinterpret_cast<const CT*>(a.k)[at + lane + 32 * e]) : 0.f;
      vv[e] = there ? to_f32(reinterpret_cast<const CT*>(a.v)[at + lane + 32 * e]) : 0.f;
    }
#pragma unroll
    for (int g = 0; g < GM; g++) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; e++) s = fmaf(q[g][e], kv[e], s);
      s = warp_sum(s) * sl2;
      const float top = fmaxf(m[g], s), ref = top == -INFINITY ? 0.f : top;
      const float alpha = exp2f(m[g] - ref), p = exp2f(s - ref);
      m[g] = top;
      l[g] = fmaf(l[g], alpha, p);
#pragma unroll
      for (int e = 0; e < E; e++) o[g][e] = fmaf(p, vv[e], o[g][e] * alpha);
    }
  }
  float* mine = smem + (size_t)warp * GM * (HD + 2);
#pragma unroll
  for (int g = 0; g < GM; g++) {
#pragma unroll
    for (int e = 0; e < E; e++) mine[g * (HD + 2) + lane + 32 * e] = o[g][e];
    if (lane == 0) {
      mine[g * (HD + 2) + HD] = m[g];
      mine[g * (HD + 2) + HD + 1] = l[g];
    }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < a.G * HD; x += kWarps * 32) {
    const int g = x / HD, e = x % HD;
    float top = -INFINITY;
    for (int w = 0; w < kWarps; w++) top = fmaxf(top, smem[(w * GM + g) * (HD + 2) + HD]);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f, acc = 0.f;
    for (int w = 0; w < kWarps; w++) {
      const float* r = smem + (w * GM + g) * (HD + 2);
      const float f = exp2f(r[HD] - ref);
      sum = fmaf(r[HD + 1], f, sum);
      acc = fmaf(r[e], f, acc);
    }
    const int head = h * a.G + g;
    put(reinterpret_cast<QT*>(a.out) + (size_t)i * a.out_stride + (size_t)head * HD + e,
        sum == 0.f ? 0.f : __fdiv_rn(acc, sum));
    if (a.lse && e == 0)
      a.lse[(size_t)i * a.H + head] = sum == 0.f ? -INFINITY : 0.6931471805599453f * (ref + log2f(sum));
  }
}

template <int HD, typename QT, typename CT, int GM>
cudaError_t launch_g(const AttnK& a, cudaStream_t st) {
  const size_t smem = (size_t)kWarps * GM * (HD + 2) * 4;
  const cudaError_t e =
      cudaFuncSetAttribute(k_paged_attention<HD, QT, CT, GM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = launch_cfg(dim3(a.n * a.Hkv), dim3(kWarps * 32), smem, st, attr);
  return cudaLaunchKernelEx(&cfg, k_paged_attention<HD, QT, CT, GM>, a);
}

template <int HD, typename QT, typename CT>
cudaError_t launch_t(const AttnK& a, cudaStream_t st) {
  if (a.G <= 4) return launch_g<HD, QT, CT, 4>(a, st);
  if (a.G <= 8) return launch_g<HD, QT, CT, 8>(a, st);
  if constexpr (HD < 256) return launch_g<HD, QT, CT, 16>(a, st);
  return cudaErrorInvalidValue;
}

template <typename QT, typename CT>
cudaError_t launch_hd(const AttnK& a, int hd, cudaStream_t st) {
  switch (hd) {
    case 32: return launch_t<32, QT, CT>(a, st);
    case 64: return launch_t<64, QT, CT>(a, st);
    case 128: return launch_t<128, QT, CT>(a, st);
    default: return launch_t<256, QT, CT>(a, st);
  }
}

}  // namespace

size_t paged_attention_workspace(int, int, int) { return 256; }

cudaError_t launch_paged_attention(const sx_paged_attention_args& a, int, cudaStream_t st) {
  AttnK k;
  k.q = static_cast<const uint8_t*>(a.q);
  k.out = static_cast<uint8_t*>(a.out);
  k.lse = a.lse;
  k.k = static_cast<const uint8_t*>(a.cache.k);
  k.v = static_cast<const uint8_t*>(a.cache.v);
  k.table = a.table;
  k.lens = a.lens;
  k.status = a.status;
  k.q_stride = a.q_stride;
  k.out_stride = a.out_stride;
  k.page_stride = a.cache.page_stride;
  k.head_stride = a.cache.head_stride;
  k.token_stride = a.cache.token_stride;
  k.table_stride = a.table_stride;
  k.n = a.n_req;
  k.Hkv = a.cache.n_kv_heads;
  k.H = a.n_heads;
  k.G = a.n_heads / a.cache.n_kv_heads;
  k.page_shift = __builtin_ctz((unsigned)a.cache.page_size);
  k.width = a.table_width;
  k.n_pages = a.cache.n_pages;
  k.scale = a.scale;
  const int hd = a.cache.head_dim;
  const bool qf = a.q_dtype == SX_DTYPE_F32;
  switch (a.cache.dtype) {
    case SX_DTYPE_F32: return launch_hd<float, float>(k, hd, st);
    case SX_DTYPE_BF16:
      return qf ? launch_hd<float, __nv_bfloat16>(k, hd, st) : launch_hd<__nv_bfloat16, __nv_bfloat16>(k, hd, st);
    default: return qf ? launch_hd<float, __half>(k, hd, st) : launch_hd<__half, __half>(k, hd, st);
  }
}

}  // namespace sx
