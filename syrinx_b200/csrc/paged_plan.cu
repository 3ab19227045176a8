// paged_plan.cu — block tables and slot maps from the requests' lengths (sx_paged_plan).
//
// Request i goes from L_i to N_i = max(0, L_i + d_i) positions, so its row of the block table
// goes from h_i = ceil(L_i / ps) to m_i = ceil(N_i / ps) pages: g_i = max(0, h_i - m_i) are
// pushed onto the stack of free pages, t_i = max(0, m_i - h_i) popped from it. With the
// exclusive sums of g, t and of the new tokens f_i = max(0, d_i) everything is independent:
//   page k taken by row i  = stack[F + G - 1 - (sum_{j<i} t_j + k)], where entries from F up are
//                            the pushes: table[r][m_r + q] of the row r the sum of g finds;
//   token j                = request r with start_r <= j < start_{r+1}, position L_r + j - start_r.
// No page is both written and read: a row gives or takes, and the stack changes only above the
// entries that are popped.
#include <cuda_runtime.h>

#include "paged.hpp"
#include "sx_device.cuh"
#include "sx_internal.hpp"

namespace sx {
namespace {

constexpr int kPlanThreads = 1024;

// Exclusive prefix of v over the CTA and its total. Two barriers; `part` is 33 words.
template <typename T>
__device__ T block_exclusive(T v, T* part, T* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) part[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const T s = part[lane];
    T run = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T u = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += u;
    }
    part[lane] = run - s;
    if (lane == 31) part[32] = run;
  }
  __syncthreads();
  *total = part[32];
  const T base = part[warp];
  __syncthreads();
  return base + inc - v;
}

// Largest r with a[r] <= x, a ascending with a[0] <= x, over a[0 .. n).
__device__ __forceinline__ int last_not_above(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) k_paged_plan(const sx_paged_plan_args a) {
  __shared__ long long part64[33];
  __shared__ int bad;
  extern __shared__ int dyn[];
  int* start = dyn;               // [n + 1] exclusive sums of the new tokens
  int* gs = dyn + a.n_req + 1;    // [n] of the pages given back
  int* ts = gs + a.n_req;         // [n] of the pages taken
  const int tid = threadIdx.x, n = a.n_req, ps = a.page_size;
  pdl_launch_dependents();
  pdl_wait();
  if (tid == 0) bad = 0;
  __syncthreads();
  const int F = ld_cg(a.n_free_in);
  const int strip = (n + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(n, tid * strip), i1 = min(n, i0 + strip);
  long long f = 0, g = 0, t = 0;
  int err = 0;  // bit 0: SX_E_INVALID, bit 1: SX_E_RANGE
  for (int i = i0; i < i1; i++) {
    const long long L = ld_cg(a.lens_in + i), d = ld_cg(a.delta + i);
    const long long N = max(0ll, L + d), h = (L + ps - 1) / ps, m = (N + ps - 1) / ps;
    if (L < 0) err |= 1;
    if (m > a.table_width || h > a.table_width) err |= 2;
    f += max(0ll, d);
    g += max(0ll, h - m);
    t += max(0ll, m - h);
  }
  long long fsum, gsum, tsum;
  long long f0 = block_exclusive(f, part64, &fsum);
  long long g0 = block_exclusive(g, part64, &gsum);
  long long t0 = block_exclusive(t, part64, &tsum);
  if (F < 0 || F > a.n_pages || F + gsum > a.n_pages) err |= 1;
  if (tsum > F + gsum || (a.slots && fsum > a.max_tokens) || fsum > 0x7fffffffll) err |= 2;
  if (err) atomicOr(&bad, err);
  __syncthreads();
  err = bad;
  if (!err) {
    for (int i = i0; i < i1; i++) {
      const int L = ld_cg(a.lens_in + i);
      const long long d = ld_cg(a.delta + i);
      const int N = (int)max(0ll, L + d), h = (L + ps - 1) / ps, m = (N + ps - 1) / ps;
      start[i] = (int)f0;
      gs[i] = (int)g0;
      ts[i] = (int)t0;
      f0 += max(0ll, d);
      g0 += max(0, h - m);
      t0 += max(0, m - h);
    }
    if (tid == 0) start[n] = (int)fsum;
  }
  __syncthreads();
  const int G = (int)gsum, T = (int)tsum;
  // a page id that is about to move must be one of the pool
  if (!err) {
    int wrong = 0;
    for (int k = tid; k < T; k += kPlanThreads) {
      const int r = last_not_above(ts, n, k), idx = F + G - 1 - k;
      const int h = (ld_cg(a.lens_in + r) + ps - 1) / ps;
      int page;
      if (idx < F) {
        page = ld_cg(a.free_pages + idx);
      } else {
        const int q = last_not_above(gs, n, idx - F);
        const int m = (int)((max(0ll, (long long)ld_cg(a.lens_in + q) + ld_cg(a.delta + q)) + ps - 1) / ps);
        page = ld_cg(a.table + (size_t)q * a.table_stride + m + (idx - F - gs[q]));
      }
      wrong |= (unsigned)page >= (unsigned)a.n_pages;
      (void)h;
    }
    if (wrong) atomicOr(&bad, 1);
  }
  __syncthreads();
  err = bad;
  if (!err) {
    for (int k = tid; k < T; k += kPlanThreads) {
      const int r = last_not_above(ts, n, k), idx = F + G - 1 - k;
      const int h = (ld_cg(a.lens_in + r) + ps - 1) / ps;
      int page;
      if (idx < F) {
        page = ld_cg(a.free_pages + idx);
      } else {
        const int q = last_not_above(gs, n, idx - F);
        const int m = (int)((max(0ll, (long long)ld_cg(a.lens_in + q) + ld_cg(a.delta + q)) + ps - 1) / ps);
        page = ld_cg(a.table + (size_t)q * a.table_stride + m + (idx - F - gs[q]));
      }
      a.table[(size_t)r * a.table_stride + h + (k - ts[r])] = page;
    }
    for (int k = tid; k < G - T; k += kPlanThreads) {  // pushes that stay
      const int q = last_not_above(gs, n, k);
      const int m = (int)((max(0ll, (long long)ld_cg(a.lens_in + q) + ld_cg(a.delta + q)) + ps - 1) / ps);
      a.free_pages[F + k] = ld_cg(a.table + (size_t)q * a.table_stride + m + (k - gs[q]));
    }
  }
  __syncthreads();  // the table is complete
  const int total = err ? 0 : (int)fsum;
  for (int j = tid; j < a.max_tokens; j += kPlanThreads) {
    int slot = -1, r = -1, p = -1;
    if (j < total) {
      r = last_not_above(start, n, j);
      p = ld_cg(a.lens_in + r) + j - start[r];
      const int page = ld_cg(a.table + (size_t)r * a.table_stride + p / ps);
      slot = page * ps + p % ps;
    }
    a.slots[j] = slot;
    if (a.tok_seq) a.tok_seq[j] = r;
    if (a.tok_pos) a.tok_pos[j] = p;
  }
  if (a.starts)
    for (int i = tid; i <= n; i += kPlanThreads) a.starts[i] = err ? 0 : start[i];
  __syncthreads();  // every read of the old lengths is done
  for (int i = tid; i < n; i += kPlanThreads) {
    const int L = ld_cg(a.lens_in + i);
    a.lens_out[i] = err ? L : (int)max(0ll, (long long)L + ld_cg(a.delta + i));
  }
  if (tid == 0) {
    *a.n_free_out = err ? F : F + G - T;
    a.status[0] = (err & 1) ? SX_E_INVALID : err ? SX_E_RANGE : SX_OK;
    a.status[1] = err ? 0 : total;
    a.status[2] = err ? 0 : T;
    a.status[3] = err ? F : F + G - T;
  }
}

}  // namespace

cudaError_t launch_paged_plan(const sx_paged_plan_args& a, cudaStream_t st) {
  const size_t smem = (size_t)(3 * a.n_req + 1) * sizeof(int);
  const cudaError_t e =
      cudaFuncSetAttribute(k_paged_plan, cudaFuncAttributeMaxDynamicSharedMemorySize, (3 * SX_PAGED_MAX_REQUESTS + 1) * 4);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = launch_cfg(dim3(1), dim3(kPlanThreads), smem, st, attr);
  return cudaLaunchKernelEx(&cfg, k_paged_plan, a);
}

}  // namespace sx
