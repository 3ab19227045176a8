// paged_plan.cu — block tables and slot maps from the requests' lengths (sx_paged_plan).
//
// Request i goes from L_i to N_i = max(0, L_i + d_i) positions, so its row of the block table
// goes from h_i = ceil(L_i / ps) to m_i = ceil(N_i / ps) pages: g_i = max(0, h_i - m_i) are
// pushed onto the stack of F free pages, t_i = max(0, m_i - h_i) popped from it. With the
// exclusive sums of g, t and of the new tokens f_i = max(0, d_i) everything is independent:
//   page k taken by row i  = stack[F + G - 1 - (sum_{j<i} t_j + k)], where entries from F up are
//                            the pushes: table[r][m_r + q] of the row r the sum of g finds;
//   token j                = request r with start_r <= j < start_{r+1}, position L_r + j - start_r.
// No page is both written and read: a row gives or takes, and the stack changes only above the
// entries that are popped. What it reads and writes is little (8 bytes per request, 8 per page
// that moves, 12 per token); it is bound by the latency of its chain of loads, so there is one
// launch of one cluster of CTAs. Each CTA forms the sums for itself, in shared memory; the pages
// that move and the tokens are spread over all threads of the cluster, each with several
// page searches and loads in flight; two cluster barriers order them (every length is read and
// every page id checked, those that moves leave in place but tokens fall into included, before
// anything is written; the table is complete before the slots).
// 2048 requests with 52k new tokens and 30k pages given back: 12.0 us (119 on one CTA, 17 on a
// cluster of 8): 1.4 for the first loads, 1.9 for the sums, 4 for the pages, 2.5 for the tokens.
// A thread searches for the first of its four tokens and walks to the requests of the others, so
// few growing requests far apart cost a read of shared memory for each idle one between them: 8 of
// 2048 take 28.8 us spread evenly against 8.0 side by side, 8 of 8192 104 against 21.7.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <utility>

#include "paged.hpp"
#include "sx_device.cuh"
#include "sx_internal.hpp"

namespace cg = cooperative_groups;

namespace sx {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanCtas = 16;  // of a cluster, more than the portable 8
constexpr int kKept = 4;      // page moves a thread keeps from the check to the write

__device__ __forceinline__ int pages_of(long long len, int shift) {
  return (int)((len + (1 << shift) - 1) >> shift);
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

// Four neighbouring entries of the token arrays, whole where they are aligned.
__device__ __forceinline__ void put_four(int* p, int j, int most, const int (&v)[4], bool whole) {
  if (whole && j + 4 <= most) {
    *reinterpret_cast<int4*>(p + j) = make_int4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (j + e < most) p[j + e] = v[e];
  }
}

// Tokens j .. j + 3 from the running sum of new tokens `start` and old lengths in `len`.
template <class Len>
__device__ __forceinline__ void four_tokens(const sx_paged_plan_args& a, const int* start, Len&& len, int shift, int j,
                                            int total, bool whole) {
  int slot[4], seq[4], pos[4];
  int r = j < total ? last_not_above(start, a.n_req, j) : -1;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    slot[e] = seq[e] = pos[e] = -1;
    if (j + e < total) {
      while (start[r + 1] <= j + e) r++;  // start[n_req] is the total
      seq[e] = r;
      pos[e] = len(r) + j + e - start[r];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (seq[e] >= 0) slot[e] = ld_cg(a.table + (size_t)seq[e] * a.table_stride + (pos[e] >> shift));
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (seq[e] >= 0) slot[e] = (int)((unsigned)slot[e] << shift) + (pos[e] & ((1 << shift) - 1));
  put_four(a.slots, j, a.max_tokens, slot, whole);
  if (a.tok_seq) put_four(a.tok_seq, j, a.max_tokens, seq, whole);
  if (a.tok_pos) put_four(a.tok_pos, j, a.max_tokens, pos, whole);
}

// Exclusive sums over the CTA of three values, and their totals. `part` is 3 x 33.
template <int THREADS>
__device__ __forceinline__ void block_exclusive3(long long (&v)[3], long long (&total)[3], long long (*part)[33]) {
  constexpr int W = THREADS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long inc[3] = {v[0], v[1], v[2]};
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
    for (int x = 0; x < 3; x++) {
      const long long u = __shfl_up_sync(0xffffffffu, inc[x], o);
      if (lane >= o) inc[x] += u;
    }
  }
  if (lane == 31)
#pragma unroll
    for (int x = 0; x < 3; x++) part[x][warp] = inc[x];
  __syncthreads();
  if (warp < 3) {
    const long long s = lane < W ? part[warp][lane] : 0;
    long long run = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += u;
    }
    part[warp][lane] = run - s;
    if (lane == 31) part[warp][32] = run;
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < 3; x++) {
    total[x] = part[x][32];
    v[x] = part[x][warp] + inc[x] - v[x];
  }
}

__global__ void __launch_bounds__(kPlanThreads) k_paged_plan(const sx_paged_plan_args a) {
  __shared__ long long part[3][33];
  __shared__ int refused;
  extern __shared__ int dyn[];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, n = a.n_req;
  const int all = ctas * kPlanThreads, me = rank * kPlanThreads + tid;
  int* start = dyn;          // [n + 1] exclusive sums of the new tokens
  int* gs = start + n + 1;   // [n + 1] of the pages given back
  int* ts = gs + n + 1;      // [n] of the pages taken
  int* len = ts + n;         // [n] old lengths
  const int shift = __ffs(a.page_size) - 1;
  pdl_launch_dependents();
  pdl_wait();
  if (tid == 0) refused = 0;
  auto started = cluster.barrier_arrive();  // waited for before another CTA's flag is written
  const int F = ld_cg(a.n_free_in);
  const int strip = (n + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(n, tid * strip), i1 = min(n, i0 + strip);
  long long v[3] = {0, 0, 0}, sum[3];  // new tokens, pages given back, pages taken
  int err = 0;                         // bit 0: SX_E_INVALID, bit 1: SX_E_RANGE
  int L0 = 0, d0 = 0;                  // one request per thread: kept
  // Pages that are neither given nor taken but get the first new tokens, the CTAs in turn; the last
  // one requested is looked at after the sums.
  unsigned open = 0, highest = 0;
  for (int i = i0; i < i1; i++) {
    const int L = L0 = ld_cg(a.lens_in + i), d = d0 = ld_cg(a.delta + i);
    highest = max(highest, open);
    if (d > 0 && L > 0 && (L & (a.page_size - 1)) && (L >> shift) < a.table_width && i % ctas == rank)
      open = (unsigned)ld_cg(a.table + (size_t)i * a.table_stride + (L >> shift));
    const long long N = max(0ll, (long long)L + d);
    const int h = pages_of(L, shift), m = pages_of(N, shift);
    len[i] = L;
    if (L < 0) err |= 1;
    if (m > a.table_width || h > a.table_width || N > 0x7fffffffll) err |= 2;
    v[0] += max(0, d);
    v[1] += max(0, h - m);
    v[2] += max(0, m - h);
  }
  block_exclusive3<kPlanThreads>(v, sum, part);
  if (F < 0 || F > a.n_pages || F + sum[1] > a.n_pages) err |= 1;
  if (sum[2] > F + sum[1] || (a.slots && sum[0] > a.max_tokens) || sum[0] > 0x7fffffffll) err |= 2;
  const bool kept = strip == 1;
  if (__syncthreads_or(err)) {
    // which of the two codes: a negative length or a broken stack comes first
    err = __syncthreads_or(err & 1) ? SX_E_INVALID : SX_E_RANGE;
  } else {
    for (int i = i0; i < i1; i++) {
      const int L = kept ? L0 : len[i], d = kept ? d0 : ld_cg(a.delta + i);
      const int h = pages_of(L, shift), m = pages_of(max(0ll, (long long)L + d), shift);
      start[i] = (int)v[0];
      gs[i] = (int)v[1];
      ts[i] = (int)v[2];
      v[0] += max(0, d);
      v[1] += max(0, h - m);
      v[2] += max(0, m - h);
    }
    if (tid == 0) start[n] = (int)sum[0], gs[n] = (int)sum[1];
    __syncthreads();
  }
  // every CTA has come to the same err, G and T here
  const int G = (int)sum[1], T = (int)sum[2], moves = max(G, T);  // T pops, then the G - T pushes that stay
  // entry k of the pushes: a page its row no longer needs
  auto pushed = [&](int k) {
    const int r = last_not_above(gs, n, k);
    // the row keeps its pages but for the ones it gives: the last gs[r + 1] - gs[r]
    return ld_cg(a.table + (size_t)r * a.table_stride + pages_of(len[r], shift) - (gs[r + 1] - k));
  };
  auto moved = [&](int k) {
    if (k >= T) return pushed(k - T);
    const int idx = F + G - 1 - k;
    return idx < F ? ld_cg(a.free_pages + idx) : pushed(idx - F);
  };
  int page[kKept], wrong = max(highest, open) >= (unsigned)a.n_pages;
  if (!err) {
#pragma unroll
    for (int x = 0; x < kKept; x++) {
      page[x] = me + x * all < moves ? moved(me + x * all) : 0;
      wrong |= (unsigned)page[x] >= (unsigned)a.n_pages;
    }
    for (int k = me + kKept * all; k < moves; k += all) wrong |= (unsigned)moved(k) >= (unsigned)a.n_pages;
  }
  wrong = __syncthreads_or(wrong);
  cluster.barrier_wait(std::move(started));
  if (wrong && tid < ctas) *cluster.map_shared_rank(&refused, tid) = 1;
  cluster.sync();  // every length, count and page id has been read, and every refusal is known
  if (refused) err = SX_E_INVALID;
  if (!err) {
    auto put = [&](int k, int p) {
      if (k < T) {
        const int r = last_not_above(ts, n, k);
        a.table[(size_t)r * a.table_stride + pages_of(len[r], shift) + (k - ts[r])] = p;
      } else {
        a.free_pages[F + k - T] = p;
      }
    };
    // pages beyond the kept ones are read again: pops and pushes touch none of what is read
    for (int k = me + kKept * all; k < moves; k += all) put(k, moved(k));
#pragma unroll
    for (int x = 0; x < kKept; x++)
      if (me + x * all < moves) put(me + x * all, page[x]);
  }
  const int total = err ? 0 : (int)sum[0];
  if (rank == ctas - 1) {
    if (a.starts)
      for (int i = tid; i <= n; i += kPlanThreads) a.starts[i] = err ? 0 : start[i];
    for (int i = i0; i < i1; i++) {
      const int L = kept ? L0 : len[i], d = kept ? d0 : ld_cg(a.delta + i);
      a.lens_out[i] = err ? L : (int)max(0ll, (long long)L + d);
    }
    if (tid == 0) {
      *a.n_free_out = err ? F : F + G - T;
      a.status[0] = err;
      a.status[1] = total;
      a.status[2] = err ? 0 : T;
      a.status[3] = err ? F : F + G - T;
    }
  }
  if (a.max_tokens == 0) return;
  cluster.sync();  // the table is complete
  const bool whole = ((reinterpret_cast<uintptr_t>(a.slots) | reinterpret_cast<uintptr_t>(a.tok_seq) |
                       reinterpret_cast<uintptr_t>(a.tok_pos)) & 15) == 0;
  for (long long j = 4ll * me; j < a.max_tokens; j += 4ll * all)
    four_tokens(a, start, [&](int r) { return len[r]; }, shift, (int)j, total, whole);
}

}  // namespace

cudaError_t launch_paged_plan(const sx_paged_plan_args& a, cudaStream_t st) {
  static std::atomic<uint64_t> ready{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device >= 64 || !(ready.load(std::memory_order_acquire) >> device & 1)) {
    constexpr int most = (4 * SX_PAGED_MAX_REQUESTS + 2) * 4;
    if ((e = cudaFuncSetAttribute(k_paged_plan, cudaFuncAttributeMaxDynamicSharedMemorySize, most)) != cudaSuccess ||
        (e = cudaFuncSetAttribute(k_paged_plan, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess)
      return e;
    if (device < 64) ready.fetch_or(1ull << device, std::memory_order_release);
  }
  // One CTA where its threads hold every page that can move and every token: 8 requests that grow by
  // one 4.6 us, against 5.7 on the cluster (which a table of 512 pages a row and more leads to).
  const bool small = (long long)a.n_req * a.table_width <= kKept * kPlanThreads && a.max_tokens <= 4 * kPlanThreads;
  const unsigned ctas = small ? 1 : kPlanCtas;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = launch_cfg(dim3(ctas), dim3(kPlanThreads), (size_t)(4 * a.n_req + 2) * 4, st, attr);
  if (ctas > 1) {
    cudaLaunchAttribute& c = attr[cfg.numAttrs++];
    c.id = cudaLaunchAttributeClusterDimension;
    c.val.clusterDim.x = ctas;
    c.val.clusterDim.y = c.val.clusterDim.z = 1;
  }
  return cudaLaunchKernelEx(&cfg, k_paged_plan, a);
}

}  // namespace sx
