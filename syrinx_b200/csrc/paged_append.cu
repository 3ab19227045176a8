// paged_append.cu — QK-norm, rotation and the scatter of new keys and values into pages
// (sx_paged_append).
//
// One pass over x: per head y = x / sqrt(mean(x^2) + eps) * gain, then per pair of elements
// (a, b) -> (a cos - b sin, b cos + a sin). Bound by memory: x read once, q and the cache rows
// written once. A group of lanes holds one head, E consecutive elements (16 bytes) a lane, so
// that loads and stores are whole 16-byte words, the norm is a shuffle sum over the group, an
// interleaved pair sits in one lane and a half-head pair in lanes half a group apart.
#include <cuda_runtime.h>

#include <type_traits>

#include "paged.hpp"
#include "sx_device.cuh"
#include "sx_internal.hpp"

namespace sx {
namespace {

constexpr int kAppendThreads = 128;

struct AppendK {
  const uint8_t* x;
  uint8_t* q;
  uint8_t *k, *v;
  const int *slots, *pos;
  const float *cosv, *sinv, *qn, *kn;
  int* status;
  long long x_stride, q_stride;                // bytes
  long long page_stride, head_stride, token_stride;  // elements
  float eps;
  int rows, H, Hkv, n_pos, page_shift, n_slots;
};

template <typename T, int E>
__device__ __forceinline__ void load_vec(const void* p, float (&v)[E]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const float4 r = __ldcg(reinterpret_cast<const float4*>(p) + i / 4);
      v[i] = r.x, v[i + 1] = r.y, v[i + 2] = r.z, v[i + 3] = r.w;
    }
  } else {
    static_assert(E == 8, "16-byte vectors");
    const uint4 r = __ldcg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
}

// E values rounded once to T, as 16-byte words (8-byte where four 16-bit values are held).
template <typename T, int E>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[E]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < E; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
    uint32_t w[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; i++) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    if constexpr (E == 4)
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int HD, typename XT, typename CT, bool IL, bool NORM, int U>
__global__ void __launch_bounds__(kAppendThreads) k_paged_append(const AppendK a) {
  constexpr int E = (sizeof(XT) == 4 && HD <= 128) ? 4 : 8;
  constexpr int LH = HD / E;     // lanes per head
  constexpr int HW = 32 / LH;    // heads per warp and step
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, sub = lane / LH, e0 = (lane % LH) * E;
  const int n_heads = a.H + 2 * a.Hkv;
  const int wpr = gridDim.y;  // warps that share a row
  const int row = blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  if (row >= a.rows) return;
  const uint8_t* xr = a.x + (size_t)row * a.x_stride;
  const int h_first = blockIdx.y * HW + sub, h_step = wpr * HW;
  float v[U][E];
  // the loads of U heads go out together, the first ones before the row's slot is known
  auto load = [&](int h0) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int h = h0 + u * h_step;
      if (h < n_heads && (h >= a.H || a.q)) {
        load_vec<XT, E>(xr + ((size_t)h * HD + e0) * sizeof(XT), v[u]);
      } else {
#pragma unroll
        for (int i = 0; i < E; i++) v[u][i] = 0.f;
      }
    }
  };
  const int slot = ld_cg(a.slots + row);
  const int pos = a.cosv ? ld_cg(a.pos + row) : 0;
  load(h_first);
  if (slot == -1) return;
  if ((unsigned)slot >= (unsigned)a.n_slots || (a.cosv && (unsigned)pos >= (unsigned)a.n_pos)) {
    if (a.status && lane == 0) *a.status = SX_E_RANGE;
    return;
  }
  // interleaved: E / 2 angles of this lane's own pairs; half-head: one angle per element
  constexpr int NA = IL ? E / 2 : E;
  float c[NA], s[NA];
#pragma unroll
  for (int i = 0; i < NA; i++) c[i] = 1.f, s[i] = 0.f;
  if (a.cosv) {
    const size_t at = (size_t)pos * (HD / 2) + (IL ? e0 / 2 : e0 % (HD / 2));
#pragma unroll
    for (int i = 0; i < NA; i += 2) {
      const float2 cc = *reinterpret_cast<const float2*>(a.cosv + at + i);
      const float2 ss = *reinterpret_cast<const float2*>(a.sinv + at + i);
      c[i] = cc.x, c[i + 1] = cc.y, s[i] = ss.x, s[i + 1] = ss.y;
    }
  }
  const size_t cache = (size_t)(slot >> a.page_shift) * a.page_stride +
                       (size_t)(slot & ((1 << a.page_shift) - 1)) * a.token_stride + e0;
  for (int h0 = h_first; h0 - sub < n_heads; h0 += U * h_step) {
    if (h0 != h_first) load(h0);
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int h = h0 + u * h_step;
      const bool on = h < n_heads && (h >= a.H || a.q);
      if (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < E; i++) ss = fmaf(v[u][i], v[u][i], ss);
#pragma unroll
        for (int o = LH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float* gain = h < a.H ? a.qn : h < a.H + a.Hkv ? a.kn : nullptr;
        if (gain) {
          const float inv = __fdiv_rn(1.f, sqrtf(fmaf(ss, 1.f / HD, a.eps)));
#pragma unroll
          for (int i = 0; i < E; i += 4) {
            const float4 g = *reinterpret_cast<const float4*>(gain + e0 + i);
            v[u][i] *= inv * g.x, v[u][i + 1] *= inv * g.y, v[u][i + 2] *= inv * g.z, v[u][i + 3] *= inv * g.w;
          }
        }
      }
      if (a.cosv) {
        if constexpr (IL) {
          if (h < a.H + a.Hkv) {
#pragma unroll
            for (int i = 0; i < E / 2; i++) {
              const float x0 = v[u][2 * i], x1 = v[u][2 * i + 1];
              v[u][2 * i] = x0 * c[i] - x1 * s[i];
              v[u][2 * i + 1] = x1 * c[i] + x0 * s[i];
            }
          }
        } else {
          const bool low = e0 < HD / 2;
#pragma unroll
          for (int i = 0; i < E; i++) {
            const float other = __shfl_xor_sync(0xffffffffu, v[u][i], LH / 2);
            const float turned = v[u][i] * c[i] + (low ? -other : other) * s[i];
            if (h < a.H + a.Hkv) v[u][i] = turned;
          }
        }
      }
      if (!on) continue;
      if (h < a.H) {
        store_vec<XT, E>(reinterpret_cast<XT*>(a.q + (size_t)row * a.q_stride) + (size_t)h * HD + e0, v[u]);
      } else {
        const bool key = h < a.H + a.Hkv;
        CT* base = reinterpret_cast<CT*>(key ? a.k : a.v);
        store_vec<CT, E>(base + cache + (size_t)(h - a.H - (key ? 0 : a.Hkv)) * a.head_stride, v[u]);
      }
    }
  }
}

template <int HD, typename XT, typename CT>
cudaError_t launch_t(const AppendK& a, bool il, int sms, cudaStream_t st) {
  constexpr int E = (sizeof(XT) == 4 && HD <= 128) ? 4 : 8;
  constexpr int HW = 32 * E / HD;
  constexpr int W = kAppendThreads / 32;
  const int heads = a.H + 2 * a.Hkv;
  const int steps = (heads + HW - 1) / HW;
  // few rows: a row's heads go to as many warps as fill the SMs
  const int gx = (a.rows + W - 1) / W;
  int gy = 1;
  while (gy < steps && (long long)gx * gy < 4ll * sms) gy *= 2;
  gy = gy < steps ? gy : steps;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = launch_cfg(dim3(gx, gy), dim3(kAppendThreads), 0, st, attr);
  const bool norm = a.qn || a.kn;
  auto go = [&](auto u) {
    constexpr int U = decltype(u)::value;
    if (il)
      return norm ? cudaLaunchKernelEx(&cfg, k_paged_append<HD, XT, CT, true, true, U>, a)
                  : cudaLaunchKernelEx(&cfg, k_paged_append<HD, XT, CT, true, false, U>, a);
    return norm ? cudaLaunchKernelEx(&cfg, k_paged_append<HD, XT, CT, false, true, U>, a)
                : cudaLaunchKernelEx(&cfg, k_paged_append<HD, XT, CT, false, false, U>, a);
  };
  // a warp with one step has nothing to load ahead
  return gy == steps ? go(std::integral_constant<int, 1>()) : go(std::integral_constant<int, 4>());
}

template <typename XT, typename CT>
cudaError_t launch_hd(const AppendK& a, int hd, bool il, int sms, cudaStream_t st) {
  switch (hd) {
    case 32: return launch_t<32, XT, CT>(a, il, sms, st);
    case 64: return launch_t<64, XT, CT>(a, il, sms, st);
    case 128: return launch_t<128, XT, CT>(a, il, sms, st);
    default: return launch_t<256, XT, CT>(a, il, sms, st);
  }
}

}  // namespace

cudaError_t launch_paged_append(const sx_paged_append_args& a, int sms, cudaStream_t st) {
  AppendK k;
  const size_t xe = a.x_dtype == SX_DTYPE_F32 ? 4 : 2;
  k.x = static_cast<const uint8_t*>(a.x);
  k.q = static_cast<uint8_t*>(a.q_out);
  k.k = static_cast<uint8_t*>(a.cache.k);
  k.v = static_cast<uint8_t*>(a.cache.v);
  k.slots = a.slots;
  k.pos = a.positions;
  k.cosv = a.cos;
  k.sinv = a.sin;
  k.qn = a.q_norm;
  k.kn = a.k_norm;
  k.status = a.status;
  k.x_stride = a.x_stride * (long long)xe;
  k.q_stride = a.q_stride * (long long)xe;
  k.page_stride = a.cache.page_stride;
  k.head_stride = a.cache.head_stride;
  k.token_stride = a.cache.token_stride;
  k.eps = a.eps;
  k.rows = a.n_rows;
  k.H = a.n_heads;
  k.Hkv = a.cache.n_kv_heads;
  k.n_pos = a.n_positions;
  k.page_shift = __builtin_ctz((unsigned)a.cache.page_size);
  k.n_slots = a.cache.n_pages * a.cache.page_size;
  const int hd = a.cache.head_dim;
  const bool il = a.interleaved != 0;
  const bool xf = a.x_dtype == SX_DTYPE_F32;
  switch (a.cache.dtype) {
    case SX_DTYPE_F32: return launch_hd<float, float>(k, hd, il, sms, st);
    case SX_DTYPE_BF16:
      return xf ? launch_hd<float, __nv_bfloat16>(k, hd, il, sms, st)
                : launch_hd<__nv_bfloat16, __nv_bfloat16>(k, hd, il, sms, st);
    default: return xf ? launch_hd<float, __half>(k, hd, il, sms, st) : launch_hd<__half, __half>(k, hd, il, sms, st);
  }
}

}  // namespace sx
