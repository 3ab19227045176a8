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
  __device__ __forceinline__ void store(void* p) const {
#pragma unroll
    for (int i = 0; i < N; i++) reinterpret_cast<uint4*>(p)[i] = w[i];
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

// E values rounded once to T, in as wide a word as they fill.
template <typename T, int E>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[E]) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (E == 2) {
      *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
    } else {
#pragma unroll
      for (int i = 0; i < E; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    }
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
    if constexpr (E == 2)
      *reinterpret_cast<uint32_t*>(p) = w[0];
    else if constexpr (E == 4)
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
template <typename T, int E>
__device__ __forceinline__ void store_vec(T* p, const f32x2 (&v)[E / 2]) {
  float x[E];
#pragma unroll
  for (int i = 0; i < E / 2; i++) unpack2(v[i], x[2 * i], x[2 * i + 1]);
  store_vec<T, E>(p, x);
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

// Many rows: every warp walks an even run of units (up to kSteps steps of HW heads of one kind, query,
// key or value, of one row), copied ahead into a ring of its own by cp.async together with the
// row's angles. A warp that loads a row's heads into registers keeps too little in flight: 20
// warps of 96 registers held 40 KB per SM and took 97 us for 16384 rows of 48 bf16 heads of 128
// (403 MB); with the ring, whose instructions came to 160 per step, it took 80. So a unit is of one
// kind and a head costs few instructions: gains, cosines and sines are multiplied together once
// per unit, and a lane holds both elements of each pair it turns. That takes 69 us, 5.9 TB/s,
// with two CTAs of rings of two units; more in flight is slower (three CTAs 79, three units 87:
// reads and writes get in each other's way in HBM), less too (one CTA 96).
constexpr int kSteps = 4;
constexpr int kRing = 2;
constexpr int kRingWarps = 8;
constexpr int kRingCtas = 2;  // per SM

template <int HD, typename XT, typename CT, bool IL>
struct Unit {
  alignas(16) uint8_t x[kSteps * Head<HD, XT, CT, IL>::STEP];
  alignas(16) float angles[HD];  // cosines, sines
};

// A lane's E elements of a head as pairs (a, b) that are turned together: a' = r (a A + b B),
// b' = r (b C + a D), r the head's norm factor. Interleaved pairs lie side by side, so the lane
// holds E neighbours; half-head pairs lie HD / 2 apart, so it holds E / 2 of each half.
template <int HD, typename XT, bool IL>
struct Turn {
  static constexpr int E = (sizeof(XT) == 4 && HD <= 128) ? 4 : 8;
  static constexpr int N = E / 4;  // packed values of each side
  f32x2 A[N], B[N], C[N], D[N];

  // side 0 / 1 of pair i of lane t: its element of the head
  static __device__ __forceinline__ int element(int t, int i, int side) {
    return IL ? t * E + 2 * i + side : t * (E / 2) + i + side * (HD / 2);
  }
  // gain: this kind's gains; angles: cosines and sines, null for no rotation; t: lane of the head
  __device__ __forceinline__ void set(const float* gain, const float* angles, int t) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      float k[2][4];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int p = 2 * i + j, at = t * (E / 2) + p;  // the pair, its angle
        const float c = angles ? angles[at] : 1.f, s = angles ? angles[HD / 2 + at] : 0.f;
        const float ga = gain[element(t, p, 0)], gb = gain[element(t, p, 1)];
        k[j][0] = c * ga, k[j][1] = -s * gb, k[j][2] = c * gb, k[j][3] = s * ga;
      }
      A[i] = pack2(k[0][0], k[1][0]), B[i] = pack2(k[0][1], k[1][1]);
      C[i] = pack2(k[0][2], k[1][2]), D[i] = pack2(k[0][3], k[1][3]);
    }
  }
  // The lane's elements of the head at `p` in shared memory, as a and b sides.
  static __device__ __forceinline__ void load(const uint8_t* p, int t, f32x2 (&a)[N], f32x2 (&b)[N]) {
    constexpr int W = E * (int)sizeof(XT) / 4;  // words
    uint32_t w[W];
    if constexpr (IL) {
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        const uint4 r = *reinterpret_cast<const uint4*>(p + t * (W * 4) + i * 4);
        w[i] = r.x, w[i + 1] = r.y, w[i + 2] = r.z, w[i + 3] = r.w;
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int i = 0; i < W / 2; i += 2) {
          const uint2 r = *reinterpret_cast<const uint2*>(p + t * (W * 2) + i * 4 + h * (HD / 2) * (int)sizeof(XT));
          w[h * (W / 2) + i] = r.x, w[h * (W / 2) + i + 1] = r.y;
        }
    }
    float x[E];
#pragma unroll
    for (int i = 0; i < W; i++) {
      if constexpr (sizeof(XT) == 4) {
        x[i] = __uint_as_float(w[i]);
      } else if constexpr (std::is_same<XT, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
      } else {
        x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
      a[i] = IL ? pack2(x[4 * i], x[4 * i + 2]) : pack2(x[2 * i], x[2 * i + 1]);
      b[i] = IL ? pack2(x[4 * i + 1], x[4 * i + 3]) : pack2(x[E / 2 + 2 * i], x[E / 2 + 2 * i + 1]);
    }
  }
  static __device__ __forceinline__ float squares(const f32x2 (&a)[N], const f32x2 (&b)[N]) {
    f32x2 q = mul2(a[0], a[0]);
#pragma unroll
    for (int i = 1; i < N; i++) q = fma2(a[i], a[i], q);
#pragma unroll
    for (int i = 0; i < N; i++) q = fma2(b[i], b[i], q);
    float lo, hi;
    unpack2(q, lo, hi);
    return lo + hi;
  }
  // The turned elements to head `p` in type T.
  template <typename T>
  __device__ __forceinline__ void put(T* p, int t, const f32x2 (&a)[N], const f32x2 (&b)[N], float r, bool rotate) const {
    const f32x2 by = pack2(r, r);
    float y[E];
#pragma unroll
    for (int i = 0; i < N; i++) {
      f32x2 u = mul2(a[i], A[i]), v = mul2(b[i], C[i]);
      if (rotate) u = fma2(b[i], B[i], u), v = fma2(a[i], D[i], v);
      u = mul2(u, by), v = mul2(v, by);
      if constexpr (IL) {
        unpack2(u, y[4 * i], y[4 * i + 2]);
        unpack2(v, y[4 * i + 1], y[4 * i + 3]);
      } else {
        unpack2(u, y[2 * i], y[2 * i + 1]);
        unpack2(v, y[E / 2 + 2 * i], y[E / 2 + 2 * i + 1]);
      }
    }
    if constexpr (IL) {
      store_vec<T, E>(p + t * E, y);
    } else {
      float lo[E / 2], hi[E / 2];
#pragma unroll
      for (int i = 0; i < E / 2; i++) lo[i] = y[i], hi[i] = y[E / 2 + i];
      store_vec<T, E / 2>(p + t * (E / 2), lo);
      store_vec<T, E / 2>(p + t * (E / 2) + HD / 2, hi);
    }
  }
};

template <int HD, typename XT, typename CT, bool IL>
__global__ void __launch_bounds__(kRingWarps * 32, kRingCtas) k_paged_append_many(const AppendK a) {
  using P = Head<HD, XT, CT, IL>;
  using U = Unit<HD, XT, CT, IL>;
  using T = Turn<HD, XT, IL>;
  constexpr int E = P::E, HW = P::HW, LH = P::LH, HB = HD * (int)sizeof(XT);  // bytes of a head
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ __align__(16) float gains[2][HD];
  __shared__ __align__(16) float row_angles[kRingWarps][HD];  // of each warp's row
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane / LH, t = lane % LH;
  for (int i = tid; i < HD; i += kRingWarps * 32) {
    gains[0][i] = a.qn ? a.qn[i] : 1.f;
    gains[1][i] = a.kn ? a.kn[i] : 1.f;
  }
  __syncthreads();
  U* ring = reinterpret_cast<U*>(dyn) + warp * kRing;
  // a row's units: nq of its query heads, nk of its key heads, nk of its value heads
  constexpr int HU = kSteps * HW;  // heads per unit
  const int nq = a.q ? (a.H + HU - 1) / HU : 0, nk = (a.Hkv + HU - 1) / HU, per_row = nq + 2 * nk;
  const long long units = (long long)a.rows * per_row, warps = (long long)gridDim.x * kRingWarps;
  const long long w = (long long)blockIdx.x * kRingWarps + warp;
  const long long u0 = units / warps * w + units % warps * w / warps;
  const long long u1 = units / warps * (w + 1) + units % warps * (w + 1) / warps;

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
      if (__shfl_sync(0xffffffffu, slots, row_p - cached) != -1) {
        U& to = ring[at];
        const int part = unit_p < nq ? 0 : unit_p < nq + nk ? 1 : 2;
        const int h = (part == 0 ? unit_p : part == 1 ? unit_p - nq : unit_p - nq - nk) * HU;  // first head, of its kind
        const int bytes = min(HU, (part == 0 ? a.H : a.Hkv) - h) * HB;
        const uint8_t* src = a.x + (size_t)row_p * a.x_stride + (uint32_t)(h + (part == 0 ? 0 : part == 1 ? a.H : a.H + a.Hkv)) * HB +
                             lane * 16;
        const uint32_t dst = smem_addr(to.x) + lane * 16;
        if (bytes == HU * HB) {
#pragma unroll
          for (int b = 0; b < HU * HB; b += 512) cp_async16(dst + b, src + b, 16);
        } else {
          for (int b = lane * 16; b < bytes; b += 512) cp_async16(dst + b - lane * 16, src + b - lane * 16, 16);
        }
        if (a.cosv && (fresh || unit_p == 0)) {
          const int pos = __shfl_sync(0xffffffffu, poss, row_p - cached);
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
#pragma unroll 1
  for (int x = 0; x < kRing - 1; x++) {
    copy_next(into);
    into = into + 1 == kRing ? 0 : into + 1;
  }
  int row = (int)(u0 / per_row), unit = (int)(u0 % per_row), held = -1, slot_of = 0;
  bool first = true;
  T turn;
  float* angles = row_angles[warp];
  for (long long todo = u1 - u0; todo > 0; todo--) {
    copy_next(into);
    into = into + 1 == kRing ? 0 : into + 1;
    cp_wait<kRing - 1>();
    __syncwarp();
    const U& u = ring[from];
    from = from + 1 == kRing ? 0 : from + 1;
    if (held < 0 || row >= held + 32) {  // as the copying side, which is ahead
      held = row;
      slot_of = row + lane < a.rows ? ld_cg(a.slots + row + lane) : -1;
      const int pos = row + lane < a.rows && a.cosv ? ld_cg(a.pos + row + lane) : 0;
      if (slot_of != -1 && refuses(a, slot_of, pos)) slot_of = -1;
    }
    const int slot = __shfl_sync(0xffffffffu, slot_of, row - held);
    if (slot != -1) {
      const int part = unit < nq ? 0 : unit < nq + nk ? 1 : 2;
      const int h0 = (part == 0 ? unit : part == 1 ? unit - nq : unit - nq - nk) * HU;
      const int left = (part == 0 ? a.H : a.Hkv) - h0 - sub;  // heads of this lane's: left > x HW
      if (a.cosv && (first || unit == 0)) {
        for (int i = lane; i < HD / 4; i += 32)
          reinterpret_cast<float4*>(angles)[i] = reinterpret_cast<const float4*>(u.angles)[i];
        __syncwarp();
      }
      CT* kv = reinterpret_cast<CT*>(part == 1 ? a.k : a.v) + place_of(a, slot) + (size_t)(h0 + sub) * a.head_stride;
      if (part == 2) {
#pragma unroll
        for (int x = 0; x < kSteps; x++) {
          if (left <= x * HW) break;
          Raw<XT, E> raw;
          raw.load_shared(u.x + (x * 32 + lane) * (E * (int)sizeof(XT)));
          CT* to = kv + (size_t)(x * HW) * a.head_stride + t * E;
          if constexpr (std::is_same<XT, CT>::value) {
            raw.store(to);
          } else {
            f32x2 v[E / 2];
            raw.values(v);
            store_vec<CT, E>(to, v);
          }
        }
      } else {
        const float* gain = part == 0 ? a.qn : a.kn;
        turn.set(gains[part], a.cosv ? angles : nullptr, t);
        const uint8_t* mine = u.x + sub * HB;
        float r[kSteps];
        if (gain) {
          // the sums of all steps first: their shuffles do not wait for one another
#pragma unroll
          for (int x = 0; x < kSteps; x++) {
            f32x2 va[T::N], vb[T::N];
            T::load(mine + x * HW * HB, t, va, vb);
            r[x] = T::squares(va, vb);
          }
#pragma unroll
          for (int o = LH / 2; o > 0; o >>= 1)
#pragma unroll
            for (int x = 0; x < kSteps; x++) r[x] += __shfl_xor_sync(0xffffffffu, r[x], o);
#pragma unroll
          for (int x = 0; x < kSteps; x++) r[x] = rsqrtf(fmaf(r[x], 1.f / HD, a.eps));
        } else {
#pragma unroll
          for (int x = 0; x < kSteps; x++) r[x] = 1.f;
        }
        XT* q = reinterpret_cast<XT*>(a.q + (size_t)row * a.q_stride) + (uint32_t)(h0 + sub) * HD;
#pragma unroll
        for (int x = 0; x < kSteps; x++) {
          if (left <= x * HW) break;
          f32x2 va[T::N], vb[T::N];
          T::load(mine + x * HW * HB, t, va, vb);
          if (part == 0)
            turn.template put<XT>(q + x * HW * HD, t, va, vb, r[x], a.cosv);
          else
            turn.template put<CT>(kv + (size_t)(x * HW) * a.head_stride, t, va, vb, r[x], a.cosv);
        }
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
  // A warp per step up to about three waves of them (48 bf16 heads of 128: 300 rows 4.1 us against
  // 5.6 with the ring, 600 6.2 / 5.9, 1200 10.8 / 8.9, 5000 40 / 25), and for narrow rows, which are
  // only a few units (14 + 2 x 2 bf16 heads of 64: 5000 rows 8.6 / 11.6, 16384 27.4 / 30.2, where the
  // bytes alone would take 12.4: a warp has one load in flight and ends).
  if (((long long)a.rows * steps <= 144ll * sms || steps <= 8) && steps <= 65535) {
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
  // beside the ring a CTA holds gains, its rows' angles and 1 KB of the system's
  const int per_sm = std::max(1, std::min(kRingCtas, (226 * 1024) / (smem + 1024 + (2 + kRingWarps) * HD * 4)));
  constexpr int HU = kSteps * P::HW;
  const long long units = (long long)a.rows * ((a.q ? (a.H + HU - 1) / HU : 0) + 2 * ((a.Hkv + HU - 1) / HU));
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
