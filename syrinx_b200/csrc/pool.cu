// pool.cu — the bookkeeping kernels of a pooled session (sx_session_create_pool): what a step's
// tokens ask of the page pool, the slots they get, and the rotation tables of sx_paged_append.
#include <cuda_runtime.h>

#include "paged.hpp"
#include "sx_device.cuh"
#include "sx_internal.hpp"

namespace sx {
namespace {

// Growth of each sequence so that every token of the step has a place: a sequence that already
// holds a token's position (one that stopped and runs on in its batch) grows by nothing.
__global__ void k_pool_begin(const PoolArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int i = threadIdx.x;
  if (i >= a.batch) return;
  const int held = ld_cg(a.lens + i);
  int target = held;
  for (int t = 0; t < a.M; t++)
    if (ld_cg(a.tok_seq + t) == i) target = max(target, ld_cg(a.tok_pos + t) + 1);
  a.delta[i] = target - held;
}

// Each token's slot, and the length its attention sees: its own position is the last one.
__global__ void k_pool_slots(const PoolArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int t = threadIdx.x;
  if (t >= a.M) return;
  const int seq = ld_cg(a.tok_seq + t), pos = ld_cg(a.tok_pos + t);
  int slot = -1;
  if (ld_cg(a.status) != SX_OK || pos / kPage >= a.pages_per_seq)
    *a.err = 4;
  else
    slot = ld_cg(a.table + (size_t)seq * a.pages_per_seq + pos / kPage) * kPage + pos % kPage;
  a.slots[t] = slot;
  a.att_len[t] = pos + 1;
}

// The angles that the decode attention computes per token (attention.cu), for every position.
__global__ void k_rope_table(const float* inv_freq, int half, int n_pos, float* cosv, float* sinv) {
  const size_t n = (size_t)n_pos * half;
  for (size_t x = blockIdx.x * (size_t)blockDim.x + threadIdx.x; x < n; x += (size_t)gridDim.x * blockDim.x) {
    float s, c;
    sincosf(__fmul_rn((float)(x / half), inv_freq[x % half]), &s, &c);
    cosv[x] = c;
    sinv[x] = s;
  }
}

}  // namespace

cudaError_t launch_pool_begin(const PoolArgs& a, cudaStream_t st) {
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = launch_cfg(dim3(1), dim3(32), 0, st, attr);
  return cudaLaunchKernelEx(&cfg, k_pool_begin, a);
}
cudaError_t launch_pool_slots(const PoolArgs& a, cudaStream_t st) {
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = launch_cfg(dim3(1), dim3(kMaxPrefillTok), 0, st, attr);
  return cudaLaunchKernelEx(&cfg, k_pool_slots, a);
}
cudaError_t launch_rope_table(const float* inv_freq, int half, int n_pos, float* cosv, float* sinv, cudaStream_t st) {
  (void)cudaGetLastError();
  k_rope_table<<<592, 256, 0, st>>>(inv_freq, half, n_pos, cosv, sinv);
  return cudaGetLastError();
}

}  // namespace sx
