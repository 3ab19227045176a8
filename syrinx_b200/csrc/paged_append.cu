// paged_append.cu — QK-norm, rotation and the scatter of new keys and values into pages
// (sx_paged_append).
//
// One pass over x: per head y = x / sqrt(mean(x^2) + eps) * gain, then per pair of elements
// (a, b) -> (a cos - b sin, b cos + a sin). Bound by memory: x read once, q and the cache rows
// written once. A group of lanes holds one head, E consecutive elements (16 bytes) a lane, so
// that loads and stores are whole 16-byte words, the norm is a shuffle sum over the group, an
// interleaved pair sits in one lane and a half-head pair in lanes half a group apart.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "paged.hpp"
#include "paged_device.cuh"
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
  int first;  // the first head that is read: 0, or H where the query heads are dropped
};

using f32x2 = unsigned long long;  // two f32, the lower one first

// E elements of type T as they lie in memory: 16 bytes, or 32.
template <typename T, int E>
struct Raw {
  static constexpr int N = E * (int)sizeof(T) / 16;
  uint4 w[N];
  __device__ __forceinline__ void load(const void* p) {
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = __ldcg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void load_shared(const void* p) {
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void values(f32x2 (&v)[E / 2]) const {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
      if constexpr (sizeof(T) == 4) {
        v[2 * i] = pack2u(x[0], x[1]), v[2 * i + 1] = pack2u(x[2], x[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if constexpr (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[j]));
            v[j] = pack2(f.x, f.y);
          } else {
            v[j] = pack2u(x[j] << 16, x[j] & 0xffff0000u);
          }
        }
      }
    }
  }
};

// E values rounded once to T, as 16-byte words (8-byte where four 16-bit values are held).
template <typename T, int E>
__device__ __forceinline__ void store_vec(T* p, const f32x2 (&v)[E / 2]) {
  float x[E];
#pragma unroll
  for (int i = 0; i < E / 2; i++) unpack2(v[i], x[2 * i], x[2 * i + 1]);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < E; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  } else {
    uint32_t w[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; i++) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    if constexpr (E == 4)
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// What the two kernels share: lanes e0 .. e0 + E - 1 of head h, of the row's H query, Hkv key
// and Hkv value heads, once its sum of squares is known.
template <int HD, typename XT, typename CT, bool IL>
struct Head {
  static constexpr int E = (sizeof(XT) == 4 && HD <= 128) ? 4 : 8;
  static constexpr int LH = HD / E;   // lanes per head
  static constexpr int HW = 32 / LH;  // heads per warp and step
  static constexpr int STEP = 32 * E * (int)sizeof(XT);  // bytes of a step
  // interleaved: E / 2 angles, of this lane's own pairs; half-head: an angle per element, the
  // sine with the sign that the element's half takes
  static constexpr int NA = IL ? E / 2 : E;
  float c[NA], s[NA];

  __device__ __forceinline__ void angles(const float* cosv, const float* sinv, int e0) {
    const int at = IL ? e0 / 2 : e0 % (HD / 2);
    const float sign = !IL && e0 < HD / 2 ? -1.f : 1.f;
#pragma unroll
    for (int i = 0; i < NA; i += 2) {
      const float2 cc = *reinterpret_cast<const float2*>(cosv + at + i);
      const float2 ss = *reinterpret_cast<const float2*>(sinv + at + i);
      c[i] = cc.x, c[i + 1] = cc.y, s[i] = sign * ss.x, s[i + 1] = sign * ss.y;
    }
  }
  static __device__ __forceinline__ float squares(const f32x2 (&v)[E / 2]) {
    f32x2 sq = mul2(v[0], v[0]);
#pragma unroll
    for (int i = 1; i < E / 2; i++) sq = fma2(v[i], v[i], sq);
    float lo, hi;
    unpack2(sq, lo, hi);
    return lo + hi;
  }
  // All lanes of the warp take part; the ones whose head is beyond the row store nothing.
  __device__ __forceinline__ void put(const AppendK& a, f32x2 (&v)[E / 2], float mean_square, const float* gain, int h, int e0,
                                      XT* q, size_t cache) const {
    const bool is_q = h < a.H, is_k = !is_q && h < a.H + a.Hkv;
    if (gain) {
      const float inv = rsqrtf(mean_square + a.eps);
      const f32x2 by = pack2(inv, inv);
#pragma unroll
      for (int i = 0; i < E / 2; i += 2) {
        const float4 g = *reinterpret_cast<const float4*>(gain + e0 + 2 * i);
        v[i] = mul2(mul2(v[i], by), pack2(g.x, g.y));
        v[i + 1] = mul2(mul2(v[i + 1], by), pack2(g.z, g.w));
      }
    }
    if (a.cosv) {
      if constexpr (IL) {
        if (is_q || is_k) {
#pragma unroll
          for (int i = 0; i < E / 2; i++) {
            float x0, x1;
            unpack2(v[i], x0, x1);
            v[i] = pack2(x0 * c[i] - x1 * s[i], x1 * c[i] + x0 * s[i]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < E / 2; i++) {
          const f32x2 other = __shfl_xor_sync(0xffffffffu, v[i], LH / 2);
          if (is_q || is_k)
            v[i] = fma2(other, pack2(s[2 * i], s[2 * i + 1]), mul2(v[i], pack2(c[2 * i], c[2 * i + 1])));
        }
      }
    }
    if (h >= a.H + 2 * a.Hkv) return;
    if (is_q) {
      if (q) store_vec<XT, E>(q + (uint32_t)h * HD + e0, v);
    } else {
      CT* base = reinterpret_cast<CT*>(is_k ? a.k : a.v);
      store_vec<CT, E>(base + cache + e0 + (size_t)(h - a.H - (is_k ? 0 : a.Hkv)) * a.head_stride, v);
    }
  }
};

__device__ __forceinline__ bool refuses(const AppendK& a, int slot, int pos) {
  return (unsigned)slot >= (unsigned)a.n_slots || (a.cosv && (unsigned)pos >= (unsigned)a.n_pos);
}
__device__ __forceinline__ size_t place_of(const AppendK& a, int slot) {
  return (size_t)(slot >> a.page_shift) * a.page_stride + (size_t)(slot & ((1 << a.page_shift) - 1)) * a.token_stride;
}

// Few rows: a warp per row and step of HW heads (blockIdx.y), all of them resident at once.
template <int HD, typename XT, typename CT, bool IL>
__global__ void __launch_bounds__(kAppendThreads) k_paged_append(const AppendK a) {
  using P = Head<HD, XT, CT, IL>;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, e0 = lane % P::LH * P::E;
  const int row = blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
  if (row >= a.rows) return;
  const int h = a.first + blockIdx.y * P::HW + lane / P::LH;
  const int slot = ld_cg(a.slots + row), pos = a.cosv ? ld_cg(a.pos + row) : 0;
  Raw<XT, P::E> raw;  // requested before the slot is known
  if (h < a.H + 2 * a.Hkv)
    raw.load(a.x + (size_t)row * a.x_stride + ((uint32_t)h * HD + e0) * sizeof(XT));
  else
    raw.clear();
  if (slot == -1) return;
  if (refuses(a, slot, pos)) {
    if (a.status && lane == 0) *a.status = SX_E_RANGE;
    return;
  }
  P head;
  if (a.cosv) head.angles(a.cosv + (size_t)pos * (HD / 2), a.sinv + (size_t)pos * (HD / 2), e0);
  f32x2 v[P::E / 2];
  raw.values(v);
  float ss = 0.f;
  if (a.qn || a.kn) {
    ss = P::squares(v);
#pragma unroll
    for (int o = P::LH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  }
  head.put(a, v, ss * (1.f / HD), h < a.H ? a.qn : h < a.H + a.Hkv ? a.kn : nullptr, h, e0,
           a.q ? reinterpret_cast<XT*>(a.q + (size_t)row * a.q_stride) : nullptr, place_of(a, slot));
}

// Many rows: every warp walks an even run of units (kSteps steps of one row), copied ahead into
// a ring of its own by cp.async together with the row's angles. A warp that loads a row's heads
// into registers keeps too little in flight: 20 warps of 96 registers held 40 KB per SM and took
// 97 us for 16384 rows of 48 bf16 heads of 128 (403 MB), where 24 warps with a ring take 80 us
// (5.1 TB/s; without the norm it is the same: the mix of reads and writes bounds it).
constexpr int kSteps = 4;
constexpr int kRing = 3;
constexpr int kRingWarps = 8;
// CTAs per SM: of f32 rows two keep as many bytes in flight as of 16-bit rows three (16384 rows of
// 48 heads of 128: f32 158 us with three, 141 with two; bf16 80 and 87).
template <typename XT>
constexpr int ring_ctas() {
  return sizeof(XT) == 4 ? 2 : 3;
}

template <int HD, typename XT, typename CT, bool IL>
struct Unit {
  alignas(16) uint8_t x[kSteps * Head<HD, XT, CT, IL>::STEP];
  alignas(16) float angles[HD];  // cosines, sines
  int slot, pad[3];
};

template <int HD, typename XT, typename CT, bool IL>
__global__ void __launch_bounds__(kRingWarps * 32, ring_ctas<XT>()) k_paged_append_many(const AppendK a) {
  using P = Head<HD, XT, CT, IL>;
  using U = Unit<HD, XT, CT, IL>;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ __align__(16) float gains[2][HD];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, e0 = lane % P::LH * P::E;
  for (int i = tid; i < HD; i += kRingWarps * 32) {
    gains[0][i] = a.qn ? a.qn[i] : 1.f;
    gains[1][i] = a.kn ? a.kn[i] : 1.f;
  }
  __syncthreads();
  U* ring = reinterpret_cast<U*>(dyn) + warp * kRing;
  const int n_heads = a.H + 2 * a.Hkv, steps = (n_heads - a.first + P::HW - 1) / P::HW;
  const int per_row = (steps + kSteps - 1) / kSteps;
  const long long units = (long long)a.rows * per_row, warps = (long long)gridDim.x * kRingWarps;
  const long long w = (long long)blockIdx.x * kRingWarps + warp;
  const long long u0 = units / warps * w + units % warps * w / warps;
  const long long u1 = units / warps * (w + 1) + units % warps * (w + 1) / warps;
  const int row_bytes = n_heads * HD * (int)sizeof(XT);

  // the copying side: slots and positions of 32 rows, one per lane
  int row_p = (int)(u0 / per_row), unit_p = (int)(u0 % per_row), cached = -1, slots = 0, poss = 0;
  long long to_copy = u1 - u0;
  bool fresh = true;
  auto copy_next = [&](int at) {
    if (to_copy > 0) {
      if (cached < 0 || row_p >= cached + 32) {
        cached = row_p;
        const bool in = row_p + lane < a.rows;
        slots = in ? ld_cg(a.slots + row_p + lane) : -1;
        poss = in && a.cosv ? ld_cg(a.pos + row_p + lane) : 0;
        if (slots != -1 && refuses(a, slots, poss)) {
          slots = -1;
          if (a.status) *a.status = SX_E_RANGE;
        }
      }
      const int slot = __shfl_sync(0xffffffffu, slots, row_p - cached), pos = __shfl_sync(0xffffffffu, poss, row_p - cached);
      U& to = ring[at];
      if (lane == 0) to.slot = slot;
      if (slot != -1) {
        const int off = a.first * HD * (int)sizeof(XT) + unit_p * kSteps * P::STEP;
        const uint8_t* src = a.x + (size_t)row_p * a.x_stride + off;
#pragma unroll
        for (int x = 0; x < kSteps * P::STEP / 512; x++) {
          const int b = x * 512 + lane * 16;
          cp_async16(smem_addr(to.x + b), off + b < row_bytes ? src + b : a.x, off + b < row_bytes ? 16 : 0);
        }
        if (a.cosv && (fresh || unit_p == 0)) {
#pragma unroll
          for (int b = lane * 16; b < HD * 4; b += 512)
            cp_async16(smem_addr(to.angles) + b,
                       reinterpret_cast<const uint8_t*>((b < HD * 2 ? a.cosv : a.sinv) + (size_t)pos * (HD / 2)) + b % (HD * 2), 16);
        }
      }
      fresh = false;
      to_copy--;
      if (++unit_p == per_row) unit_p = 0, row_p++;
    }
    cp_commit();
  };
  int into = 0, from = 0;
#pragma unroll
  for (int x = 0; x < kRing - 1; x++) {
    copy_next(into);
    into = (into + 1) % kRing;
  }
  int row = (int)(u0 / per_row), unit = (int)(u0 % per_row);
  bool first = true;
  P head;
  for (long long todo = u1 - u0; todo > 0; todo--) {
    copy_next(into);
    into = (into + 1) % kRing;
    cp_wait<kRing - 1>();
    __syncwarp();
    const U& u = ring[from];
    from = (from + 1) % kRing;
    const int slot = u.slot;
    if (slot != -1) {
      if (a.cosv && (first || unit == 0)) head.angles(u.angles, u.angles + HD / 2, e0);
      float ss[kSteps];
      if (a.qn || a.kn) {
        // the sums of all steps first: their shuffles do not wait for one another
#pragma unroll
        for (int x = 0; x < kSteps; x++) {
          Raw<XT, P::E> raw;
          raw.load_shared(u.x + x * P::STEP + lane * (P::E * (int)sizeof(XT)));
          f32x2 v[P::E / 2];
          raw.values(v);
          ss[x] = P::squares(v);
        }
#pragma unroll
        for (int o = P::LH / 2; o > 0; o >>= 1)
#pragma unroll
          for (int x = 0; x < kSteps; x++) ss[x] += __shfl_xor_sync(0xffffffffu, ss[x], o);
      }
      XT* q = a.q ? reinterpret_cast<XT*>(a.q + (size_t)row * a.q_stride) : nullptr;
      const size_t cache = place_of(a, slot);
#pragma unroll
      for (int x = 0; x < kSteps; x++) {
        const int h0 = a.first + (unit * kSteps + x) * P::HW;
        if (h0 >= n_heads) break;
        const int h = h0 + lane / P::LH;
        Raw<XT, P::E> raw;
        raw.load_shared(u.x + x * P::STEP + lane * (P::E * (int)sizeof(XT)));
        f32x2 v[P::E / 2];
        raw.values(v);
        const float* gain = h < a.H ? (a.qn ? gains[0] : nullptr) : h < a.H + a.Hkv && a.kn ? gains[1] : nullptr;
        head.put(a, v, ss[x] * (1.f / HD), gain, h, e0, q, cache);
      }
    }
    first = false;
    if (++unit == per_row) unit = 0, row++;
    __syncwarp();  // every lane has read the unit before it is overwritten
  }
  cp_wait<0>();
}

template <int HD, typename XT, typename CT, bool IL>
cudaError_t launch_t(AppendK a, int sms, cudaStream_t st) {
  using P = Head<HD, XT, CT, IL>;
  a.first = a.q ? 0 : a.H;
  const int steps = (a.H - a.first + 2 * a.Hkv + P::HW - 1) / P::HW;
  cudaLaunchAttribute attr[1];
  // A warp per step up to about two waves of them; beyond, its start-up is paid too often (48 bf16
  // heads of 128: 300 rows 4.1 us against 5.6 with the ring, 600 6.2 / 6.8, 1200 10.8 / 10.0,
  // 5000 40 / 30).
  if ((long long)a.rows * steps <= 96ll * sms && steps <= 65535) {
    constexpr int W = kAppendThreads / 32;
    cudaLaunchConfig_t cfg = launch_cfg(dim3((a.rows + W - 1) / W, steps), dim3(kAppendThreads), 0, st, attr);
    return cudaLaunchKernelEx(&cfg, k_paged_append<HD, XT, CT, IL>, a);
  }
  constexpr int smem = kRingWarps * kRing * (int)sizeof(Unit<HD, XT, CT, IL>);
  static std::atomic<uint64_t> ready{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device >= 64 || !(ready.load(std::memory_order_acquire) >> device & 1)) {
    if ((e = cudaFuncSetAttribute(k_paged_append_many<HD, XT, CT, IL>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) !=
        cudaSuccess)
      return e;
    if (device < 64) ready.fetch_or(1ull << device, std::memory_order_release);
  }
  // beside the ring a CTA holds its gains and 1 KB of the system's
  const int per_sm = std::max(1, std::min(ring_ctas<XT>(), (226 * 1024) / (smem + 3072)));
  const long long units = (long long)a.rows * ((steps + kSteps - 1) / kSteps);
  const int grid = (int)std::min<long long>((long long)per_sm * sms, (units + kRingWarps - 1) / kRingWarps);
  cudaLaunchConfig_t cfg = launch_cfg(dim3(grid), dim3(kRingWarps * 32), smem, st, attr);
  return cudaLaunchKernelEx(&cfg, k_paged_append_many<HD, XT, CT, IL>, a);
}

template <typename XT, typename CT>
cudaError_t launch_hd(const AppendK& a, int hd, bool il, int sms, cudaStream_t st) {
  switch (hd) {
    case 32: return il ? launch_t<32, XT, CT, true>(a, sms, st) : launch_t<32, XT, CT, false>(a, sms, st);
    case 64: return il ? launch_t<64, XT, CT, true>(a, sms, st) : launch_t<64, XT, CT, false>(a, sms, st);
    case 128: return il ? launch_t<128, XT, CT, true>(a, sms, st) : launch_t<128, XT, CT, false>(a, sms, st);
    default: return il ? launch_t<256, XT, CT, true>(a, sms, st) : launch_t<256, XT, CT, false>(a, sms, st);
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
  k.first = 0;
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
