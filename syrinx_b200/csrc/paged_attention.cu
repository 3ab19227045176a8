// paged_attention.cu — attention of one new token per request over its pages
// (sx_paged_attention).
//
// Mathematics. With scores in units of log 2, s_t = scale log2(e) q.k_t, one pass over the keys
// keeps a running maximum m, sum l and output o per query head:
//   m' = max(m, s), l' = l 2^(m - m') + 2^(s - m'), o' = o 2^(m - m') + 2^(s - m') v;
// partial results over disjoint keys join by the same rule. out = o / l, lse = ln 2 (m + log2 l).
//
// Bound. Every key and value is read once for its whole group of query heads: 2 len Hkv hd
// elements per request, a few operations each, so the kernel is bound by HBM when there is
// enough to read and by latency when there is not.
//
// Split. The keys of every (request, kv head) are cut into tiles of 8 KB (16 keys of 128 bf16
// elements; 16 KB for 16-bit pages with head_dim 256); all tiles of the batch, request by request and head by head, are one line that is
// cut into even shares, one per CTA (one CTA per SM), and a CTA's share into even runs, one per
// warp. However uneven the lengths are, every SM reads the same number of bytes (requests without
// keys are not as free: see Place::next). A warp copies
// its own tiles into a ring of its own (cp.async), so nothing in the main loop waits for
// another warp, and the ring runs on across the end of one request and the start of the next.
// A (request, kv head) that lies inside one warp's run is finished by that warp; runs that
// begin or end inside one leave a partial (m, l, o), joined in shared memory at the end of the
// CTA, and, where a share begins or ends inside one, through the workspace by a second kernel.
// Every partial is joined in key order, so results repeat bit for bit. 32 requests of
// 8001..32768 keys (8 kv heads of 128, bf16, 2.9 GB) take 431 us, 6.7 TB/s; one CTA per (request,
// kv head) took 4630. 64 requests of 1..4099 keys (177 MB) take 37.5 us, of which 10 are what a
// split call costs before its first tile and after its last one.
//
// Products. 16-bit pages: mma.sync.m16n8k16 with the keys as the 16 rows and up to 8 query heads
// as the 8 columns, S^T = K q^T, then O^T = V^T P^T, so the tiles are A operands as they lie in
// shared memory (ldmatrix, transposed for V) and an MMA is full for a group of 8; a group of up to
// 16 takes two. Every product starts from zero and is added in f32 outside the tensor core, which
// cuts its sums off; values and weights beyond 16 bits go through in parts. f32 pages would lose precision there; they use packed f32 FMAs, a key's row split
// over a few lanes. A kv head with more query heads than that is run as several groups.
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

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxSmem = 227 * 1024;

struct AttnK {
  const uint8_t* q;
  uint8_t* out;
  float* lse;
  const uint8_t *k, *v;
  const int *table, *lens;
  int* status;
  uint8_t* ws;
  long long q_stride, out_stride;                    // elements
  long long page_stride, head_stride, token_stride;  // bytes
  long long table_stride;
  // a kv head's Gall query heads are run as `share` groups of up to G; Hkv counts the groups of all
  int n, Hkv, G, H, page_shift, width, n_pages, Gall, share;
  int direct;  // 1: CTA c is (request c / Hkv, kv head c % Hkv); nothing is split over CTAs
  float scale;
};

// Of group h: its kv head, its first query head, and how many it has. SHARED: whether a kv head may
// have several groups (an instantiation of its own: the divisions cost short calls 5 %).
template <bool SHARED>
__device__ __forceinline__ int kv_head(const AttnK& a, int h) {
  return SHARED ? h / a.share : h;
}
template <bool SHARED>
__device__ __forceinline__ int first_head(const AttnK& a, int h) {
  return SHARED ? h / a.share * a.Gall + h % a.share * a.G : h * a.G;
}
template <bool SHARED>
__device__ __forceinline__ int group_heads(const AttnK& a, int h) {
  return SHARED ? min(a.G, a.Gall - h % a.share * a.G) : a.G;
}

// Workspace: per CTA a record of the partial that begins in it, then two partials per CTA
// (the one its share begins inside of, the one it ends inside of).
struct alignas(16) Joint {
  int i, h, pieces, pad;  // pieces: partials of (i, h), 0: none begins here
};
__host__ __device__ inline size_t ws_stats_off(int ctas) { return (size_t)ctas * sizeof(Joint); }
__host__ __device__ inline size_t ws_o_off(int ctas, int G) { return ws_stats_off(ctas) + (size_t)2 * ctas * G * 8; }
__host__ __device__ inline size_t ws_bytes(int ctas, int G, int hd) {
  return ws_o_off(ctas, G) + (size_t)2 * ctas * G * hd * 4 + 16;
}

__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Four neighbours; their 16-byte (f32) or 8-byte place is aligned.
__device__ __forceinline__ void put4(float* p, float x, float y, float z, float w) {
  *reinterpret_cast<float4*>(p) = make_float4(x, y, z, w);
}
template <typename T>
__device__ __forceinline__ void put4(T* p, float x, float y, float z, float w) {
  alignas(8) T v[4];
  put(v, x), put(v + 1, y), put(v + 2, z), put(v + 3, w);
  *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(v);
}

// 2^x; results below 2^-126 are zero.
__device__ __forceinline__ float pow2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// What a maximum of -inf (nothing seen, or only scores of -inf) is taken as.
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

// ---- 16-bit pages -----------------------------------------------------------------------

template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  } else {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
// The same with nothing to add to: d = a b. The tensor core cuts off what lies below the last place
// of the largest term, sums included (measured: towards zero every time, 0.9 steps on average and
// 2.3 at most where the sum is 100 times the product, 3.5 at 1000 times), so a sum that ran through
// a thousand products would drift by that much each time: 460 u (u = 2^-24) over a run of 16384 keys,
// 1600 at head_dim 256. Products start from zero therefore and are added in f32: 3 to 18 u.
template <typename T>
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  }
}
// x + d, and x f + d with f of elements 0 and 2 in f[0], of 1 and 3 in f[1].
__device__ __forceinline__ void add4(float (&x)[4], const float (&d)[4]) {
#pragma unroll
  for (int c = 0; c < 4; c += 2) unpack2(add2(pack2(x[c], x[c + 1]), pack2(d[c], d[c + 1])), x[c], x[c + 1]);
}
__device__ __forceinline__ void fma4(float (&x)[4], const float (&f)[2], const float (&d)[4]) {
#pragma unroll
  for (int c = 0; c < 4; c += 2)
    unpack2(fma2(pack2(x[c], x[c + 1]), pack2(f[0], f[1]), pack2(d[c], d[c + 1])), x[c], x[c + 1]);
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// v as NL values of type T that add up to it: each the rounding of what the ones before leave.
template <typename T, int NL>
__device__ __forceinline__ void split16(float lo, float hi, uint32_t (&w)[NL]) {
#pragma unroll
  for (int x = 0; x < NL; x++) {
    w[x] = pack16<T>(lo, hi);
    if (x + 1 < NL) {
      const float2 r = unpack16<T>(w[x]);
      lo -= r.x;
      hi -= r.y;
    }
  }
}

// The same for weights, which are not negative: every part but the last is cut off, not rounded,
// and no part of a weight above zero is zero, so that an infinite value times the parts is
// infinite and not inf - inf or 0 inf. A part is the type's least at least: f16's 2^-24 (2^-39 of
// the largest weight, which is 2^kLift), in bf16, whose range is f32's, 2^-126. (A floor in
// proportion to the weight, 2^-22 of it in f16, was below 2^-24 for weights under 2^-12.)
template <typename T, int NP>
__device__ __forceinline__ void split_weights(float lo, float hi, uint32_t (&w)[NP]) {
  constexpr bool f16 = std::is_same<T, __half>::value;
  // 0 for 0: pow2 gives nothing else below 2^-126
  const float least_lo = fminf(f16 ? lo * 0x1p102f : lo, f16 ? 0x1p-24f : 0x1p-126f);
  const float least_hi = fminf(f16 ? hi * 0x1p102f : hi, f16 ? 0x1p-24f : 0x1p-126f);
  if constexpr (f16) lo = fmaxf(lo, least_lo), hi = fmaxf(hi, least_hi);
#pragma unroll
  for (int x = 0; x < NP; x++) {
    if (x + 1 == NP) {
      w[x] = pack16<T>(lo, hi);
    } else {
      if constexpr (f16)
        asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(w[x]) : "f"(hi), "f"(lo));
      else
        w[x] = __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
      const float2 r = unpack16<T>(w[x]);
      lo = fmaxf(lo - r.x, least_lo);
      hi = fmaxf(hi - r.y, least_hi);
    }
  }
}

// One warp's online softmax over tiles of 16-bit keys and values. Lane (g = lane / 4, t = lane % 4)
// holds the scores of keys g and g + 8 of each 16 for heads 2t and 2t + 1 of each 8, and output
// elements g and g + 8 of each 16 for the same heads.
template <int HD_, typename QT_, typename CT_, int GM_, bool SHARED_ = false>
struct Mma {
  static constexpr bool SHARED = SHARED_;
  static constexpr int GM = GM_;
  using QT = QT_;
  using CT = CT_;
  static constexpr int HD = HD_;
  static constexpr int NW = HD == 256 ? 4 : 8;                   // warps per CTA
  static constexpr int TK = HD == 32 ? 64 : HD == 64 ? 32 : 16;  // keys per tile
  static constexpr int RB = HD * 2, CPR = RB / 16;
  static constexpr int NT = (GM + 7) / 8, MT = TK / 16, KS = HD / 16;
  static constexpr bool kF16 = std::is_same<CT, __half>::value;
  static constexpr bool kQ32 = sizeof(QT) == 4;
  // f32 queries and weights pass the tensor cores as sums of 16-bit values: three bf16 hold 24
  // bits; two f16 hold 22, of values that are first scaled to the top of f16's range. 16-bit
  // queries are exact. Their weights are split the same way, though a 16-bit result would hide two
  // bf16 values' 16 bits but for its ties: then 32 requests of 8001..32768 keys differ from the
  // rounded exact result by 1.1e-4 of its size, with three by 2.8e-5 (f32 sums in another order:
  // 1.05e-4). The third costs nothing up to 8 heads, 10 % at 9 to 16.
  static constexpr int NL = kQ32 ? (kF16 ? 2 : 3) : 1;
  static constexpr int NP = kF16 ? 2 : 3;
  // f16 weights are kept as 2^15 p, at the top of f16's range, so that as much as can be of their
  // low parts is above f16's smallest step
  static constexpr float kLift = kF16 ? 15.f : 0.f;
  static constexpr float kDrop = kF16 ? 0x1p-15f : 1.f;  // 2^-kLift, for the weights' sum

  uint32_t q[NT][NL][KS][2];
  float o[NT][KS][4];
  float m[NT][2], l[NT][2], lost[NT][2], sl2[NT][2];  // lost: what rounding has added to l

  static __device__ __forceinline__ uint32_t at(int row, int chunk) {  // byte of a 16-byte chunk in a tile
    if constexpr (CPR == 4) return row * RB + ((chunk ^ ((row >> 1) & 3)) << 4);
    return row * RB + ((chunk ^ (row & 7)) << 4);
  }

  __device__ __forceinline__ void start(const AttnK& a, int i, int h, int lane) {
    const int g = lane >> 2, t = lane & 3;
    const QT* qp = reinterpret_cast<const QT*>(a.q) + (size_t)i * a.q_stride + (size_t)first_head<SHARED>(a, h) * HD;
    const int heads = group_heads<SHARED>(a, h);
    const float base = a.scale * kLog2e;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int head = nt * 8 + g;
      const bool on = head < heads;
      float up = 1.f, down = 1.f;  // powers of two
      if constexpr (kQ32) {
        float2 x[KS][2];
        float top = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
          for (int c = 0; c < 2; c++) {
            x[ks][c] = on ? __ldcg(reinterpret_cast<const float2*>(qp + (size_t)head * HD + ks * 16 + c * 8 + 2 * t))
                          : make_float2(0.f, 0.f);
            top = fmaxf(top, fmaxf(fabsf(x[ks][c].x), fabsf(x[ks][c].y)));
          }
        if constexpr (kF16) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          if (top > 0.f && top < INFINITY) {
            const int ex = min(max(ilogbf(top), -100), 127) - 10;  // the head's largest lands in [2^10, 2^11)
            up = ldexpf(1.f, -ex);
            down = ldexpf(1.f, ex);
          }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
          for (int c = 0; c < 2; c++) {
            uint32_t w[NL];
            split16<CT, NL>(x[ks][c].x * up, x[ks][c].y * up, w);
#pragma unroll
            for (int y = 0; y < NL; y++) q[nt][y][ks][c] = w[y];
          }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
          for (int c = 0; c < 2; c++)
            q[nt][0][ks][c] =
                on ? __ldcg(reinterpret_cast<const uint32_t*>(qp + (size_t)head * HD + ks * 16 + c * 8 + 2 * t)) : 0u;
      }
      const float mine = base * down;
#pragma unroll
      for (int c = 0; c < 2; c++) {
        sl2[nt][c] = __shfl_sync(0xffffffffu, mine, 4 * (2 * t + c));
        m[nt][c] = -INFINITY;
        l[nt][c] = lost[nt][c] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < KS; j++)
#pragma unroll
        for (int c = 0; c < 4; c++) o[nt][j][c] = 0.f;
    }
  }

  // `valid` of the tile's keys count; the others' rows are zeros.
  __device__ __forceinline__ void tile(uint32_t ks_, uint32_t vs_, int valid, int lane) {
    const int g = lane >> 2;
    const int r16 = lane & 15, c1 = lane >> 4;  // ldmatrix: row and half chunk of this lane's address
    float s[MT][NT][4];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
      float low[NT][4];  // the products of a split query's lower parts
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        uint32_t a[4];
        ldsm4(a, ks_ + at(mt * 16 + r16, 2 * ks + c1));
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          if (ks == 0) {
            mma16816_first<CT>(s[mt][nt], a, q[nt][0][ks][0], q[nt][0][ks][1]);
          } else {
            float d[4];
            mma16816_first<CT>(d, a, q[nt][0][ks][0], q[nt][0][ks][1]);
            add4(s[mt][nt], d);
          }
#pragma unroll
          for (int y = 1; y < NL; y++) {  // 2^-8 of the score at most: their sum may lose a few bits
            if (ks == 0 && y == 1)
              mma16816_first<CT>(low[nt], a, q[nt][y][ks][0], q[nt][y][ks][1]);
            else
              mma16816<CT>(low[nt], a, q[nt][y][ks][0], q[nt][y][ks][1]);
          }
        }
      }
      if constexpr (NL > 1) {
        // an infinite key makes the lower parts' products infinite too, of either sign
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int c = 0; c < 4; c++) s[mt][nt][c] = isinf(s[mt][nt][c]) ? s[mt][nt][c] : s[mt][nt][c] + low[nt][c];
      }
    }
    uint32_t p[MT][NT][NP][2];
    float alpha[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int mt = 0; mt < MT; mt++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
          s[mt][nt][c] = mt * 16 + g + (c >> 1) * 8 < valid ? s[mt][nt][c] * sl2[nt][c & 1] : -INFINITY;
          top[c & 1] = fmaxf(top[c & 1], s[mt][nt][c]);
        }
#pragma unroll
      for (int c = 0; c < 2; c++) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], off));
        top[c] = fmaxf(top[c], m[nt][c]);
        const float ref = finite_or_zero(top[c]);
        alpha[nt][c] = pow2(m[nt][c] - ref);
        m[nt][c] = top[c];
        top[c] = ref - kLift;
      }
      float sum[2] = {0.f, 0.f};  // of the tile's weights
#pragma unroll
      for (int mt = 0; mt < MT; mt++) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
          s[mt][nt][c] = pow2(s[mt][nt][c] - top[c & 1]);
          sum[c & 1] += s[mt][nt][c];
        }
        uint32_t lo[NP], hi[NP];
        split_weights<CT, NP>(s[mt][nt][0], s[mt][nt][1], lo);
        split_weights<CT, NP>(s[mt][nt][2], s[mt][nt][3], hi);
#pragma unroll
        for (int y = 0; y < NP; y++) {
          p[mt][nt][y][0] = transpose8x8(lo[y]);
          p[mt][nt][y][1] = transpose8x8(hi[y]);
        }
      }
      // equal weights are rounded the same way tile after tile: what an addition loses goes to the next
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const float old = l[nt][c] * alpha[nt][c], x = fmaf(-lost[nt][c], alpha[nt][c], sum[c]);
        l[nt][c] = old + x;
        lost[nt][c] = (l[nt][c] - old) - x;
      }
    }
#pragma unroll
    for (int mt = 0; mt < MT; mt++)
#pragma unroll
      for (int j = 0; j < KS; j++) {
        uint32_t a[4];
        // rows: keys (lane & 7) + 8 (lane / 16); chunks: elements 16 j + 8 ((lane / 8) & 1)
        ldsm4_t(a, vs_ + at(mt * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * j + ((lane >> 3) & 1)));
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          float d[4];  // the weights' lower parts first: what a product cuts off is below the whole's last bits
          mma16816_first<CT>(d, a, p[mt][nt][NP - 1][0], p[mt][nt][NP - 1][1]);
#pragma unroll
          for (int y = NP - 2; y >= 0; y--) mma16816<CT>(d, a, p[mt][nt][y][0], p[mt][nt][y][1]);
          if (mt == 0)
            fma4(o[nt][j], alpha[nt], d);
          else
            add4(o[nt][j], d);
        }
      }
  }

  // f(head, element, o * by(l)) for every output of the group this lane holds and w(head, m, l)
  // by one lane per head; m and l over all keys the warp has seen.
  template <class B, class F, class W>
  __device__ __forceinline__ void finish(int G, int lane, B&& by, F&& f, W&& w) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        float sum = l[nt][c];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const int head = nt * 8 + 2 * t + c;
        if (head < G) {
          const float x = by(sum);
#pragma unroll
          for (int j = 0; j < KS; j++) {
            f(head, j * 16 + g, sum == 0.f ? 0.f : o[nt][j][c] * x);
            f(head, j * 16 + g + 8, sum == 0.f ? 0.f : o[nt][j][c + 2] * x);
          }
          if (g == 0) w(head, m[nt][c], sum);
        }
      }
  }
};

// ---- f32 pages --------------------------------------------------------------------------

// Sums over LPK neighbouring lanes of each of V values, left with every lane: halves of the
// values are exchanged while there are several (each lane adds up its own share), then gathered
// back in the opposite order.
template <int V, int MASK>
__device__ __forceinline__ void sum_over(float* a, int lane) {
  if constexpr (MASK > 0) {
    if constexpr (V > 1) {
      constexpr int HV = V / 2;
      const bool up = lane & MASK;
      float keep[HV];
#pragma unroll
      for (int i = 0; i < HV; i++) {
        const float send = up ? a[i] : a[i + HV];
        keep[i] = (up ? a[i + HV] : a[i]) + __shfl_xor_sync(0xffffffffu, send, MASK);
      }
      sum_over<HV, MASK / 2>(keep, lane);
#pragma unroll
      for (int i = 0; i < HV; i++) {
        const float other = __shfl_xor_sync(0xffffffffu, keep[i], MASK);
        a[i] = up ? other : keep[i];
        a[i + HV] = up ? keep[i] : other;
      }
    } else {
      a[0] += __shfl_xor_sync(0xffffffffu, a[0], MASK);
      sum_over<1, MASK / 2>(a, lane);
    }
  }
}

// One warp's online softmax over tiles of f32 keys and values on the FMA pipes. LPK lanes share
// a key, each E = HD / LPK of its elements (16-byte chunks LPK apart); the 32 / LPK lane groups
// take keys in turn, each with a running maximum of its own, and are joined at the end.
template <int HD_, int GM_, bool SHARED_ = false>
struct Fma {
  static constexpr bool SHARED = SHARED_;
  static constexpr int GM = GM_;
  using QT = float;
  using CT = float;
  static constexpr int HD = HD_;
  static constexpr int NW = 8;
  static constexpr int TK = 1024 / HD;  // keys per tile: 8 KB of keys and values
  static constexpr int RB = HD * 4, CPR = RB / 16;
  // at most 64 query elements and 64 output elements a lane
  static constexpr int LPK0 = GM * HD / 64 < 4 ? 4 : GM * HD / 64;
  static constexpr int LPK = LPK0 < HD / 16 ? HD / 16 : LPK0;
  static constexpr int E = HD / LPK, KG = 32 / LPK;
  static constexpr int NK = TK / KG;           // keys of a tile per lane group
  static constexpr int KB = NK < 4 ? 2 : 4;  // keys folded at a time
  static constexpr float kDrop = 1.f;
  static_assert(LPK <= 32 && E >= 4 && TK % KG == 0 && NK % KB == 0, "lane split");

  unsigned long long q[GM][E / 2], o[GM][E / 2];
  float m[GM], l[GM], sl2;

  static __device__ __forceinline__ uint32_t at(int row, int chunk) {
    if constexpr (LPK == 4) return row * RB + ((chunk ^ ((row & 1) << 2)) << 4);
    return row * RB + (chunk << 4);
  }

  __device__ __forceinline__ void start(const AttnK& a, int i, int h, int lane) {
    const int hs = lane % LPK;
    const float* qp = reinterpret_cast<const float*>(a.q) + (size_t)i * a.q_stride + (size_t)first_head<SHARED>(a, h) * HD;
    const int heads = group_heads<SHARED>(a, h);
    sl2 = a.scale * kLog2e;
#pragma unroll
    for (int g = 0; g < GM; g++) {
#pragma unroll
      for (int j = 0; j < E / 4; j++) {
        const float4 x = g < heads ? __ldcg(reinterpret_cast<const float4*>(qp + (size_t)g * HD) + hs + LPK * j)
                                 : make_float4(0.f, 0.f, 0.f, 0.f);
        q[g][2 * j] = pack2(x.x, x.y);
        q[g][2 * j + 1] = pack2(x.z, x.w);
      }
#pragma unroll
      for (int e = 0; e < E / 2; e++) o[g][e] = 0ull;
      m[g] = -INFINITY;
      l[g] = 0.f;
    }
  }

  static __device__ __forceinline__ void row(uint32_t addr, int r, int hs, unsigned long long (&x)[E / 2]) {
#pragma unroll
    for (int j = 0; j < E / 4; j++)
      asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];"
                   : "=l"(x[2 * j]), "=l"(x[2 * j + 1])
                   : "r"(addr + at(r, hs + LPK * j))
                   : "memory");
  }

  __device__ __forceinline__ void tile(uint32_t ks_, uint32_t vs_, int valid, int lane) {
    const int hs = lane % LPK, kg = lane / LPK;
#pragma unroll
    for (int b = 0; b < NK / KB; b++) {
      float s[GM * KB];
#pragma unroll
      for (int kk = 0; kk < KB; kk++) {
        unsigned long long x[E / 2];
        row(ks_, kg + KG * (b * KB + kk), hs, x);
#pragma unroll
        for (int g = 0; g < GM; g++) {
          unsigned long long d = mul2(q[g][0], x[0]);
#pragma unroll
          for (int e = 1; e < E / 2; e++) d = fma2(q[g][e], x[e], d);
          float lo, hi;
          unpack2(d, lo, hi);
          s[g * KB + kk] = lo + hi;
        }
      }
      sum_over<GM * KB, LPK / 2>(s, lane);
      bool turned = false;
      float alpha[GM];
#pragma unroll
      for (int g = 0; g < GM; g++) {
        float top = m[g];
#pragma unroll
        for (int kk = 0; kk < KB; kk++) {
          s[g * KB + kk] = kg + KG * (b * KB + kk) < valid ? s[g * KB + kk] * sl2 : -INFINITY;
          top = fmaxf(top, s[g * KB + kk]);
        }
        const float ref = finite_or_zero(top);
        alpha[g] = pow2(m[g] - ref);
        turned |= alpha[g] != 1.f;
        m[g] = top;
        l[g] *= alpha[g];
#pragma unroll
        for (int kk = 0; kk < KB; kk++) {
          s[g * KB + kk] = pow2(s[g * KB + kk] - ref);
          l[g] += s[g * KB + kk];
        }
      }
      if (__any_sync(0xffffffffu, turned)) {
#pragma unroll
        for (int g = 0; g < GM; g++) {
          const unsigned long long f = pack2(alpha[g], alpha[g]);
#pragma unroll
          for (int e = 0; e < E / 2; e++) o[g][e] = mul2(o[g][e], f);
        }
      }
#pragma unroll
      for (int kk = 0; kk < KB; kk++) {
        unsigned long long x[E / 2];
        row(vs_, kg + KG * (b * KB + kk), hs, x);
#pragma unroll
        for (int g = 0; g < GM; g++) {
          const unsigned long long f = pack2(s[g * KB + kk], s[g * KB + kk]);
#pragma unroll
          for (int e = 0; e < E / 2; e++) o[g][e] = fma2(f, x[e], o[g][e]);
        }
      }
    }
  }

  template <class B, class F, class W>
  __device__ __forceinline__ void finish(int G, int lane, B&& by, F&& f, W&& w) {
    const int hs = lane % LPK, kg = lane / LPK;
#pragma unroll
    for (int g = 0; g < GM; g++) {
      float top = m[g];
#pragma unroll
      for (int off = LPK; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      const float fac = pow2(m[g] - finite_or_zero(top));
      float sum = l[g] * fac;
#pragma unroll
      for (int off = LPK; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      float x[E];
#pragma unroll
      for (int e = 0; e < E / 2; e++) unpack2(o[g][e], x[2 * e], x[2 * e + 1]);
#pragma unroll
      for (int e = 0; e < E; e++) {
        x[e] *= fac;
#pragma unroll
        for (int off = LPK; off < 32; off <<= 1) x[e] += __shfl_xor_sync(0xffffffffu, x[e], off);
      }
      if (g < G && g % KG == kg) {
        const float inv = by(sum);
#pragma unroll
        for (int e = 0; e < E; e++) f(g, (hs + LPK * (e / 4)) * 4 + e % 4, sum == 0.f ? 0.f : x[e] * inv);
        if (hs == 0) w(g, top, sum);
      }
    }
  }
};

// ---- the walk over the tiles --------------------------------------------------------------

// What one (request, kv head) costs beside its tiles, in tiles: a query to load, a result to
// write. Shares are even in tiles plus these, so that a run of very short requests is not the
// last to finish (64 requests of 1..4099 keys: 54.6 us with 0, 39.6 with 1, 37.1 with 2, the same
// with 3 and 4).
constexpr uint32_t kSegTiles = kPagedSegTiles;
// Tiles in a warp's ring: one is computed while one is copied. With 8 warps that is 64 to 128 KB in
// flight per SM. Three took 2.6 us longer at 168 MB: the first tiles of all warps queue up, and
// every warp waits for them.
constexpr int kStages = 2;
// Requests whose lengths and running costs are kept in shared memory; more are kept in strips.
constexpr int kLine = 512;
// Up to this many requests every warp sums the costs itself.
constexpr int kFewRequests = 128;

template <int TK>
__device__ __forceinline__ int tiles_of(int len) {
  return len > 0 ? (len - 1) / TK + 1 : 0;
}

template <class M>
struct Smem {
  uint32_t before[kLine + 1];  // cost of the requests before each strip
  int lens[kLine];             // up to kLine requests: their lengths
  uint32_t part[M::NW];
  int4 piece[2 * M::NW];  // a partial's request, kv head, flags, tiles of the two behind it
  float2 ml[2 * M::NW][M::GM];
};
enum : int { kValid = 1, kBegins = 2, kEnds = 4 };

// A place in the line of tiles: tile t of kv head h of request i; i == n behind the last one.
// Every lane of a warp holds the same place.
template <class M>
struct Place {
  int i, h, t, len, tiles;

  __device__ __forceinline__ void at_request(const AttnK& a, const Smem<M>& sm, int cap, int req) {
    i = req;
    len = a.n <= kLine && !a.direct ? sm.lens[req] : min(max(ld_cg(a.lens + req), 0), cap);
    tiles = tiles_of<M::TK>(len);
  }
  // Requests without keys are stepped over one by one: at a read of shared memory each up to kLine
  // requests, at a load each beyond (5000 requests of which 16 hold 2000 keys: 180 us spread evenly,
  // 2015 side by side, where the last run walks the rest of the line; 29 without the empty ones).
  __device__ __forceinline__ void next(const AttnK& a, const Smem<M>& sm, int cap) {
    if (++t < tiles) return;
    t = 0;
    if (!a.direct && ++h < a.Hkv) return;
    h = 0;
    do {
      if (a.direct || ++i >= a.n) {
        i = a.n;
        return;
      }
      at_request(a, sm, cap, i);
    } while (len == 0);
  }
  // The place at cost g of `total`; `strip` requests per entry of sm.before.
  __device__ __forceinline__ void locate(const AttnK& a, const Smem<M>& sm, int cap, uint32_t g, uint32_t total, int strip,
                                         int lane) {
    h = t = 0;
    i = a.n;
    if (g >= total) return;
    int st = 16 * (__popc(__ballot_sync(0xffffffffu, sm.before[16 * lane] <= g)) - 1);
    st += __popc(__ballot_sync(0xffffffffu, lane < 16 && sm.before[st + (lane & 15)] <= g)) - 1;
    uint32_t off = g - sm.before[st];
    int r = st * strip;
    if (strip > 1) {
      for (;; r += 32) {
        const int tl = r + lane < a.n ? tiles_of<M::TK>(min(max(ld_cg(a.lens + r + lane), 0), cap)) : 0;
        const uint32_t own = tl ? (tl + kSegTiles) * (uint32_t)a.Hkv : 0u;
        uint32_t run = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t u = __shfl_up_sync(0xffffffffu, run, o);
          if (lane >= o) run += u;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, run > off);
        if (hit) {
          const int who = __ffs(hit) - 1;
          off -= __shfl_sync(0xffffffffu, run - own, who);
          r += who;
          break;
        }
        off -= __shfl_sync(0xffffffffu, run, 31);
        if (r + 32 >= a.n) return;  // not reached: sm.before holds the place
      }
    }
    at_cost(a, sm, cap, r, off);
  }
  // The place at cost `off` of request r (-1: behind the last one).
  __device__ __forceinline__ void at_cost(const AttnK& a, const Smem<M>& sm, int cap, int r, uint32_t off) {
    h = t = 0;
    i = a.n;
    if (r < 0) return;
    at_request(a, sm, cap, r);
    const uint32_t per = (uint32_t)tiles + kSegTiles;
    h = (int)(off / per);
    t = max(0, (int)(off - (uint32_t)h * per) - (int)kSegTiles);
  }
};

template <class M>
__global__ void __launch_bounds__(M::NW * 32, 1) k_paged_attention(const AttnK a) {
  constexpr int NW = M::NW, NT = NW * 32, TK = M::TK, HD = M::HD, RB = M::RB, CPR = M::CPR;
  constexpr int TILE = 2 * TK * RB;
  using QT = typename M::QT;
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ Smem<M> sm;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x, ctas = gridDim.x;
  pdl_launch_dependents();
  pdl_wait();

  const int cap = a.width << a.page_shift;
  Place<M> pc, last = {};  // this warp's run: [pc, last)
  uint32_t share = 1;  // cost per CTA
  bool some_empty = false;
  if (lane < 2) sm.piece[2 * warp + lane].z = 0;  // each warp its own: nothing orders the warps yet
  __syncwarp();

  // requests without keys get their result at once
  auto nothing = [&](long long i) {
    QT* out = reinterpret_cast<QT*>(a.out) + i * a.out_stride;
    for (int x = lane; x < a.H * HD; x += 32) put(out + x, 0.f);
    if (a.lse)
      for (int x = lane; x < a.H; x += 32) a.lse[i * a.H + x] = -INFINITY;
  };

  // this warp's part [lo, hi) of the CTA's even share of the total cost
  auto run_of = [&](uint32_t total, uint32_t& lo, uint32_t& hi) {
    share = max((total + ctas - 1) / ctas, (uint32_t)NW);
    const uint32_t c0 = min((unsigned long long)total, (unsigned long long)share * cta);
    const uint32_t c = min(total - c0, share);
    lo = c0 + c / NW * warp + c % NW * warp / NW;  // c warp / NW without leaving 32 bits
    hi = c0 + c / NW * (warp + 1) + c % NW * (warp + 1) / NW;
  };

  if (a.direct) {
    const int i = cta / a.Hkv;
    if (a.status && tid == 0 && ld_cg(a.lens + i) > cap) *a.status = SX_E_RANGE;
    pc.at_request(a, sm, cap, i);
    if (pc.tiles == 0 && cta % a.Hkv == 0 && warp == 0) nothing(i);
    const int w0 = (int)((long long)pc.tiles * warp / NW), w1 = (int)((long long)pc.tiles * (warp + 1) / NW);
    pc.h = last.h = cta % a.Hkv;
    pc.t = w0;
    last.i = i;
    last.t = w1;
    if (w1 == pc.tiles) last.i = a.n, last.h = last.t = 0;
    if (w0 == w1) pc.i = last.i, pc.h = last.h, pc.t = last.t;
  } else if (a.n <= kFewRequests) {
    // every warp for itself, 32 requests at a time and without a barrier: the running costs in
    // registers, the lengths in shared memory (all warps write the same)
    constexpr int R = kFewRequests / 32;
    uint32_t before[R], own[R], total = 0;
#pragma unroll
    for (int x = 0; x < R; x++) own[x] = x * 32 + lane < a.n ? (uint32_t)ld_cg(a.lens + x * 32 + lane) : 0u;
#pragma unroll
    for (int x = 0; x < R; x++) {
      if (x * 32 >= a.n) break;
      const bool in = x * 32 + lane < a.n;
      const int len = min(max((int)own[x], 0), cap), tl = tiles_of<TK>(len);
      if ((int)own[x] > cap && a.status) *a.status = SX_E_RANGE;
      some_empty |= __any_sync(0xffffffffu, in && len == 0);
      if (in) sm.lens[x * 32 + lane] = len;
      own[x] = tl ? (tl + kSegTiles) * (uint32_t)a.Hkv : 0u;
      uint32_t run = own[x];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += u;
      }
      before[x] = total + run - own[x];
      total += __shfl_sync(0xffffffffu, run, 31);
    }
    __syncwarp();
    uint32_t lo, hi;
    run_of(total, lo, hi);
#pragma unroll 1
    for (int y = 0; y < 2; y++) {
      const uint32_t g = y ? hi : lo;
      int r = -1;
      uint32_t off = 0;
      // the request with before <= g < before + own
#pragma unroll
      for (int x = 0; x < R; x++) {
        if (x * 32 >= a.n) break;
        const unsigned hit = __ballot_sync(0xffffffffu, g - before[x] < own[x]);
        if (hit) {
          r = x * 32 + __ffs(hit) - 1;
          off = g - __shfl_sync(0xffffffffu, before[x], __ffs(hit) - 1);
        }
      }
      pc = last;
      last.at_cost(a, sm, cap, r, off);
    }
  } else {
    // cost before each strip of requests and in all
    const int strip = (a.n + kLine - 1) / kLine;
    constexpr int SPT = kLine / NT;  // strips per thread
    uint32_t cost[SPT], mine = 0;
    bool none = false;
#pragma unroll
    for (int x = 0; x < SPT; x++) {
      cost[x] = 0;
      for (int y = 0; y < strip; y++) {
        const uint32_t i = (uint32_t)(tid * SPT + x) * strip + y;
        const int raw = i < (uint32_t)a.n ? ld_cg(a.lens + i) : 0;
        const int len = min(max(raw, 0), cap), tl = tiles_of<TK>(len);
        if (strip == 1) sm.lens[tid * SPT + x] = len;
        if (tl) cost[x] += (tl + kSegTiles) * (uint32_t)a.Hkv;
        none |= i < (uint32_t)a.n && len == 0;
        if (raw > cap && a.status) *a.status = SX_E_RANGE;
      }
      mine += cost[x];
    }
    uint32_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) sm.part[warp] = inc;
    some_empty = __syncthreads_or(none);
    uint32_t base = inc - mine, total = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) {
      const uint32_t v = sm.part[w];
      if (w < warp) base += v;
      total += v;
    }
#pragma unroll
    for (int x = 0; x < SPT; x++) {
      sm.before[tid * SPT + x] = base;
      base += cost[x];
    }
    __syncthreads();
    uint32_t lo, hi;
    run_of(total, lo, hi);
#pragma unroll 1
    for (int x = 0; x < 2; x++) {
      pc = last;
      last.locate(a, sm, cap, x ? hi : lo, total, strip, lane);
    }
  }
  auto before_last = [&](const Place<M>& x) { return x.i != last.i || x.h != last.h || x.t != last.t; };

  uint8_t* ring = dyn + (size_t)warp * kStages * TILE;
  const uint32_t ring_s = smem_addr(ring);
  // Where a partial at the start of a run goes. Warp 0's is the share's own first partial.
  Joint* joint = reinterpret_cast<Joint*>(a.ws);
  float2* ws_ml = reinterpret_cast<float2*>(a.ws + ws_stats_off(ctas));
  float* ws_o = reinterpret_cast<float*>(a.ws + ws_o_off(ctas, a.G));
  float* first_o = reinterpret_cast<float*>(dyn + (size_t)NW * kStages * TILE);  // [NW - 1][G][HD]

  // the copying side runs ahead of the computing side by the ring's depth
  Place<M> pp = pc;
  int page_of = -1, page_base = 0, pages = 0;  // request and first of the 32 pages held one per lane
  const int page_mask = (1 << a.page_shift) - 1;
  auto copy_next = [&](int stage) {
    if (before_last(pp)) {
      const int key0 = pp.t * TK, p0 = key0 >> a.page_shift;
      if (page_of != pp.i || p0 < page_base || p0 >= page_base + 32) {
        page_of = pp.i;
        page_base = p0 & ~31;
        const int idx = page_base + lane;
        pages = -1;
        if (idx <= (pp.len - 1) >> a.page_shift) {
          pages = ld_cg(a.table + (size_t)pp.i * a.table_stride + idx);
          if ((unsigned)pages >= (unsigned)a.n_pages) {
            pages = -1;
            if (a.status) *a.status = SX_E_RANGE;
          }
        }
      }
      const uint32_t dst = ring_s + stage * TILE;
      const int left = pp.len - key0;
      if (page_mask >= TK - 1) {  // the tile lies in one page
        const int page = __shfl_sync(0xffffffffu, pages, p0 - page_base);
        size_t off = (size_t)(page < 0 ? 0 : page) * a.page_stride + (size_t)kv_head<M::SHARED>(a, pp.h) * a.head_stride +
                     (size_t)((key0 & page_mask) + lane / CPR) * a.token_stride + lane % CPR * 16;
        const int rows = page < 0 ? 0 : left;
        const size_t down = (CPR <= 32 ? 32 / CPR : 1) * a.token_stride;
#pragma unroll
        for (int x = 0; x < TK * CPR / 32; x++) {
          const int idx = x * 32 + lane, r = idx / CPR, c = idx % CPR;
          const int bytes = r < rows ? 16 : 0;
          size_t at = off;
          if constexpr (CPR > 32) at += (x & 1) * 512;
          if (!bytes) at = 0;
          cp_async16(dst + M::at(r, c), a.k + at, bytes);
          cp_async16(dst + M::at(r, c) + TK * RB, a.v + at, bytes);
          if (CPR <= 32 || (x & 1)) off += down;
        }
      } else {
#pragma unroll 4
        for (int x = 0; x < TK * CPR / 32; x++) {
          const int idx = x * 32 + lane, r = idx / CPR, c = idx % CPR;
          const int key = key0 + r;
          const int page = __shfl_sync(0xffffffffu, pages, (key >> a.page_shift) - page_base);
          const int bytes = r < left && page >= 0 ? 16 : 0;
          const size_t at = bytes ? (size_t)page * a.page_stride + (size_t)kv_head<M::SHARED>(a, pp.h) * a.head_stride +
                                        (size_t)(key & page_mask) * a.token_stride + c * 16
                                  : 0;
          cp_async16(dst + M::at(r, c), a.k + at, bytes);
          cp_async16(dst + M::at(r, c) + TK * RB, a.v + at, bytes);
        }
      }
      pp.next(a, sm, cap);
    }
    cp_commit();
  };
  M mine;
  int stage = 0;
  bool lead = true, fresh = true, began = false;
  for (;;) {
    copy_next(stage);  // one tile ahead of the one computed
    stage ^= 1;
    if (lead) {
      lead = false;
      if (some_empty) {  // the warps of all CTAs take the requests in turn
        for (int i = cta * NW + warp; i < a.n; i += ctas * NW)
          if (ld_cg(a.lens + i) <= 0) nothing(i);
      }
      continue;
    }
    if (!before_last(pc)) break;
    if (fresh) {
      mine.start(a, pc.i, pc.h, lane);
      began = pc.t == 0;
      fresh = false;
    }
    cp_wait<1>();
    __syncwarp();
    const uint32_t tile = ring_s + stage * TILE;
    mine.tile(tile, tile + TK * RB, min(TK, pc.len - pc.t * TK), lane);
    __syncwarp();  // every lane has read the tile before it is overwritten
    const int i = pc.i, h = pc.h, rest = pc.tiles - pc.t - 1;
    pc.next(a, sm, cap);
    const bool done = !before_last(pc);
    if (rest == 0 || done) {
      if (rest == 0 && began) {
        const int head0 = first_head<M::SHARED>(a, h);
        QT* out = reinterpret_cast<QT*>(a.out) + (size_t)i * a.out_stride + (size_t)head0 * HD;
        mine.finish(
            group_heads<M::SHARED>(a, h), lane, [&](float sum) { return sum == 0.f ? 0.f : __fdiv_rn(1.f, sum); },
            [&](int head, int d, float v) { put(out + head * HD + d, v); },
            [&](int head, float top, float sum) {
              if (a.lse)
                a.lse[(size_t)i * a.H + head0 + head] =
                    sum == 0.f ? -INFINITY : kLn2 * (finite_or_zero(top) + log2f(sum * M::kDrop));
            });
      } else {
        // a partial: the run's last one may lie in the ring, which is then done with
        const int slot = 2 * warp + done;
        const bool out_of_cta = warp == 0 && !done;
        float* dst = done         ? reinterpret_cast<float*>(ring)
                     : out_of_cta ? ws_o + (size_t)2 * cta * a.G * HD
                                  : first_o + (size_t)(warp - 1) * a.G * HD;
        float2* ml = out_of_cta ? ws_ml + (size_t)2 * cta * a.G : sm.ml[slot];
        mine.finish(
            group_heads<M::SHARED>(a, h), lane, [](float) { return 1.f; }, [&](int head, int d, float v) { dst[head * HD + d] = v; },
            [&](int head, float top, float sum) { ml[head] = make_float2(top, sum); });
        if (lane == 0 && !out_of_cta)
          sm.piece[slot] = make_int4(i, h, kValid | (began ? kBegins : 0) | (rest == 0 ? kEnds : 0), rest);
      }
      fresh = true;
    }
  }
  cp_wait<0>();
  __syncthreads();

  // Join the warps' partials, in key order: neighbours of one (request, kv head) are a group.
  // Teams of G HD / 4 threads take the groups in turn, each thread four output elements.
  const int4 pz = lane < 2 * NW ? sm.piece[lane] : make_int4(0, 0, 0, 0);
  const unsigned valid = __ballot_sync(0xffffffffu, pz.z & kValid);
  const unsigned lower = valid & ((1u << lane) - 1);
  const int prev = lower ? 31 - __clz(lower) : 0;
  const int prev_i = __shfl_sync(0xffffffffu, pz.x, prev), prev_h = __shfl_sync(0xffffffffu, pz.y, prev);
  const bool same = prev_i == pz.x && prev_h == pz.y;
  unsigned firsts = __ballot_sync(0xffffffffu, (pz.z & kValid) && !(lower && same));  // first partial of each group
  const int team_size = min(NT, a.G * (HD / 4)), teams = NT / team_size, team = tid / team_size;
  bool leaves = false;
  for (int k = 0; firsts; k++) {
    const int x0 = __ffs(firsts) - 1;
    firsts &= firsts - 1;
    const unsigned group = valid & ~((1u << x0) - 1) & (firsts ? (1u << (__ffs(firsts) - 1)) - 1 : 0xffffffffu);
    const int4 head_piece = sm.piece[x0], tail_piece = sm.piece[31 - __clz(group)];
    const bool begins = head_piece.z & kBegins, ends = tail_piece.z & kEnds;
    const int i = head_piece.x, h = head_piece.y, slot = 2 * cta + begins;
    if (begins && !ends) {
      leaves = true;
      if (tid == 0)
        *reinterpret_cast<int4*>(joint + cta) = make_int4(i, h, 1 + (int)((tail_piece.w + share - 1) / share), 0);
    }
    if (team != k % teams) continue;
    const int head0 = first_head<M::SHARED>(a, h), heads = group_heads<M::SHARED>(a, h);
    for (int e = tid - team * team_size; e < heads * (HD / 4); e += team_size) {
      const int head = e / (HD / 4);
      float top = -INFINITY;
#pragma unroll 1
      for (unsigned g = group; g; g &= g - 1) top = fmaxf(top, sm.ml[__ffs(g) - 1][head].x);
      const float ref = finite_or_zero(top);
      float sum = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (unsigned g = group; g; g &= g - 1) {
        const int y = __ffs(g) - 1;
        const float2 ml = sm.ml[y][head];
        const float4 x = reinterpret_cast<const float4*>((y & 1) ? reinterpret_cast<const float*>(dyn + (size_t)(y >> 1) * kStages * TILE)
                                                                 : first_o + (size_t)((y >> 1) - 1) * a.G * HD)[e];
        const float f = pow2(ml.x - ref);
        sum = fmaf(ml.y, f, sum);
        v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
      }
      if (begins && ends) {
        const float inv = sum == 0.f ? 0.f : __fdiv_rn(1.f, sum);
        if (sum == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);
        put4(reinterpret_cast<QT*>(a.out) + (size_t)i * a.out_stride + (size_t)head0 * HD + 4 * e, v.x * inv, v.y * inv,
             v.z * inv, v.w * inv);
        if (a.lse && e % (HD / 4) == 0)
          a.lse[(size_t)i * a.H + head0 + head] =
              sum == 0.f ? -INFINITY : kLn2 * (ref + log2f(sum * M::kDrop));
      } else {
        reinterpret_cast<float4*>(ws_o)[(size_t)slot * a.G * (HD / 4) + e] = v;
        if (e % (HD / 4) == 0) ws_ml[(size_t)slot * a.G + head] = make_float2(top, sum);
      }
    }
  }
  if (!a.direct && !leaves && tid == 0) *reinterpret_cast<int4*>(joint + cta) = make_int4(0, 0, 0, 0);
}

// Joins the partials of one query head of the (request, kv head) that begins in CTA blockIdx.x's
// share and goes on behind it: the CTA's second partial, then the first ones of the CTAs after
// it. Groups of HD / 4 threads take the partials in turn and are added up in order.
constexpr int kJoinThreads = 128;
template <int HD, typename QT, bool SHARED>
__global__ void __launch_bounds__(kJoinThreads) k_paged_join(const AttnK a, int ctas, float drop) {
  constexpr int C = HD / 4, GROUPS = kJoinThreads / C;
  __shared__ float4 acc[kJoinThreads];
  __shared__ float sums[GROUPS], tops[kJoinThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int cta = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
  const float2* ml = reinterpret_cast<const float2*>(a.ws + ws_stats_off(ctas)) + head;
  const float4* o = reinterpret_cast<const float4*>(a.ws + ws_o_off(ctas, a.G)) + (size_t)head * C;
  auto slot = [&](int y) { return (size_t)(y == 0 ? 2 * cta + 1 : 2 * (cta + y)) * a.G; };
  const int c = tid % C, group = tid / C, most = ctas - cta;  // no more partials than CTAs from here on
  // The first partials are requested together with their number: what lies behind it is not used.
  const int4 joint = __ldcg(reinterpret_cast<const int4*>(a.ws) + cta);
  constexpr int AHEAD = 2;
  float4 x[AHEAD];
  float2 s[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; k++) {
    const int y = min(group + k * GROUPS, most - 1);
    s[k] = __ldcg(ml + slot(y));
    x[k] = __ldcg(o + slot(y) * C + c);
  }
  float top = __ldcg(ml + slot(min(tid, most - 1))).x;
  const int pieces = joint.z;
  if (pieces == 0 || head >= group_heads<SHARED>(a, joint.y)) return;
  if (tid >= pieces) top = -INFINITY;
  for (int y = tid + kJoinThreads; y < pieces; y += kJoinThreads) top = fmaxf(top, __ldcg(ml + slot(y)).x);
  top = warp_max(top);
  if ((tid & 31) == 0) tops[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; w++) top = fmaxf(top, tops[w]);
  const float ref = finite_or_zero(top);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  auto add = [&](const float2& s, const float4& x) {
    const float f = pow2(s.x - ref);
    sum = fmaf(s.y, f, sum);
    v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
  };
#pragma unroll
  for (int k = 0; k < AHEAD; k++)
    if (group + k * GROUPS < pieces) add(s[k], x[k]);
#pragma unroll 4
  for (int y = group + AHEAD * GROUPS; y < pieces; y += GROUPS) add(__ldcg(ml + slot(y)), __ldcg(o + slot(y) * C + c));
  acc[tid] = v;
  if (c == 0) sums[group] = sum;
  __syncthreads();
  const size_t row = (size_t)first_head<SHARED>(a, joint.y) + head;
  float total = 0.f;
#pragma unroll
  for (int g = 0; g < GROUPS; g++) total += sums[g];
  for (int d = tid; d < HD; d += kJoinThreads) {
    float x = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; g++) x += reinterpret_cast<const float*>(acc)[g * HD + d];
    put(reinterpret_cast<QT*>(a.out) + (size_t)joint.x * a.out_stride + row * HD + d,
        total == 0.f ? 0.f : __fdiv_rn(x, total));
  }
  if (a.lse && tid == 0)
    a.lse[(size_t)joint.x * a.H + row] = total == 0.f ? -INFINITY : kLn2 * (ref + log2f(total * drop));
}

// A CTA per (request, kv head), in one launch, where they are all resident at once and have at
// most this many tiles a warp. Measured either side of it, direct against split: 8 requests of
// 8 kv heads of 128 in bf16, 250 keys 7.3 / 9.5 us, 500 keys 9.5 / 10.6, 1000 keys (8 tiles a
// warp) 14.2 / 13.2; 300 requests of 1..400 keys, 16 CTAs an SM after one another, 77 / 26.
constexpr int kDirectTiles = 4;

template <class M>
cudaError_t launch_m(AttnK a, long long bound, int sms, cudaStream_t st) {
  constexpr int TILE = 2 * M::TK * M::RB;
  const int partials = (M::NW - 1) * a.G * M::HD * 4;
  a.direct = !a.ws || ((long long)a.n * a.Hkv <= sms && bound <= (long long)kDirectTiles * M::NW * M::TK);
  const size_t smem = (size_t)M::NW * kStages * TILE + partials;
  // the joining kernel asks for the same split of L1 and shared memory, so that it can be resident
  // (and wait) while the first one runs
  static std::atomic<uint64_t> ready{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device >= 64 || !(ready.load(std::memory_order_acquire) >> device & 1)) {
    constexpr int most = kMaxSmem - (int)sizeof(Smem<M>) - 128;
    if ((e = cudaFuncSetAttribute(k_paged_attention<M>, cudaFuncAttributeMaxDynamicSharedMemorySize, most)) != cudaSuccess ||
        (e = cudaFuncSetAttribute(k_paged_join<M::HD, typename M::QT, M::SHARED>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                  cudaSharedmemCarveoutMaxShared)) != cudaSuccess)
      return e;
    if (device < 64) ready.fetch_or(1ull << device, std::memory_order_release);
  }
  const int grid = a.direct ? a.n * a.Hkv : sms;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = launch_cfg(dim3(grid), dim3(M::NW * 32), smem, st, attr);
  e = cudaLaunchKernelEx(&cfg, k_paged_attention<M>, a);
  if (e != cudaSuccess || a.direct) return e;
  cfg = launch_cfg(dim3(sms, a.G), dim3(kJoinThreads), 0, st, attr);
  return cudaLaunchKernelEx(&cfg, k_paged_join<M::HD, typename M::QT, M::SHARED>, a, sms, M::kDrop);
}

template <int HD, typename QT, typename CT>
cudaError_t launch_hd(const AttnK& a, long long bound, int sms, cudaStream_t st) {
  if constexpr (sizeof(CT) == 4) {
    if (a.G <= 2) return launch_m<Fma<HD, 2>>(a, bound, sms, st);
    if (a.G <= 4) return launch_m<Fma<HD, 4>>(a, bound, sms, st);
    return a.share == 1 ? launch_m<Fma<HD, 8>>(a, bound, sms, st) : launch_m<Fma<HD, 8, true>>(a, bound, sms, st);
  } else {
    // several groups have more than half of the most heads each
    if constexpr (HD == 256)
      return a.share == 1 ? launch_m<Mma<HD, QT, CT, 8>>(a, bound, sms, st)
                          : launch_m<Mma<HD, QT, CT, 8, true>>(a, bound, sms, st);
    else
      return a.G <= 8        ? launch_m<Mma<HD, QT, CT, 8>>(a, bound, sms, st)
             : a.share == 1 ? launch_m<Mma<HD, QT, CT, 16>>(a, bound, sms, st)
                            : launch_m<Mma<HD, QT, CT, 16, true>>(a, bound, sms, st);
  }
}

template <typename QT, typename CT>
cudaError_t launch_t(const AttnK& a, int hd, long long bound, int sms, cudaStream_t st) {
  switch (hd) {
    case 32: return launch_hd<32, QT, CT>(a, bound, sms, st);
    case 64: return launch_hd<64, QT, CT>(a, bound, sms, st);
    case 128: return launch_hd<128, QT, CT>(a, bound, sms, st);
    default: return launch_hd<256, QT, CT>(a, bound, sms, st);
  }
}

}  // namespace

// Query heads that one pass over a kv head's tiles serves; more are run as groups, which read the
// tiles again (from L2, as neighbours in the line). f32 pages: 16 heads at once kept too little of
// their work in registers, 1.4 TB/s where two groups of 8 reach 2.4.
int paged_attention_group(int G, int hd, bool f32) {
  const int most = f32 || hd == 256 ? 8 : 16, share = (G + most - 1) / most;
  return (G + share - 1) / share;
}

size_t paged_attention_workspace(int G, int hd, int sms) { return ws_bytes(sms, paged_attention_group(G, hd, false), hd); }

cudaError_t launch_paged_attention(const sx_paged_attention_args& a, int sms, cudaStream_t st) {
  AttnK k;
  const long long ce = a.cache.dtype == SX_DTYPE_F32 ? 4 : 2;
  k.q = static_cast<const uint8_t*>(a.q);
  k.out = static_cast<uint8_t*>(a.out);
  k.lse = a.lse;
  k.k = static_cast<const uint8_t*>(a.cache.k);
  k.v = static_cast<const uint8_t*>(a.cache.v);
  k.table = a.table;
  k.lens = a.lens;
  k.status = a.status;
  k.ws = static_cast<uint8_t*>(a.workspace);
  k.q_stride = a.q_stride;
  k.out_stride = a.out_stride;
  k.page_stride = a.cache.page_stride * ce;
  k.head_stride = a.cache.head_stride * ce;
  k.token_stride = a.cache.token_stride * ce;
  k.table_stride = a.table_stride;
  k.n = a.n_req;
  k.H = a.n_heads;
  k.Gall = a.n_heads / a.cache.n_kv_heads;
  k.G = paged_attention_group(k.Gall, a.cache.head_dim, a.cache.dtype == SX_DTYPE_F32);
  k.share = (k.Gall + k.G - 1) / k.G;
  k.Hkv = a.cache.n_kv_heads * k.share;
  k.page_shift = __builtin_ctz((unsigned)a.cache.page_size);
  k.width = a.table_width;
  k.n_pages = a.cache.n_pages;
  k.direct = 0;
  k.scale = a.scale;
  long long bound = (long long)a.table_width * a.cache.page_size;
  if (a.max_len > 0) bound = std::min(bound, (long long)a.max_len);
  const int hd = a.cache.head_dim;
  const bool qf = a.q_dtype == SX_DTYPE_F32;
  switch (a.cache.dtype) {
    case SX_DTYPE_F32: return launch_t<float, float>(k, hd, bound, sms, st);
    case SX_DTYPE_BF16:
      return qf ? launch_t<float, __nv_bfloat16>(k, hd, bound, sms, st)
                : launch_t<__nv_bfloat16, __nv_bfloat16>(k, hd, bound, sms, st);
    default:
      return qf ? launch_t<float, __half>(k, hd, bound, sms, st) : launch_t<__half, __half>(k, hd, bound, sms, st);
  }
}

}  // namespace sx
