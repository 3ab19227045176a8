// paged.hpp — launch interfaces of the paged key/value operators (include/syrinx_paged.h).
#pragma once
#include <cuda_runtime.h>

#include "../../include/syrinx_dualar.h"
#include "../../include/syrinx_paged.h"

namespace sx {

// The argument checks of the C ABI: SX_OK, or a status with its message set.
int paged_check(const sx_paged_plan_args& a);
int paged_check(const sx_paged_append_args& a);
int paged_check(const sx_paged_attention_args& a, int sms);

// Launches on the current device. The arguments have passed paged_check.
cudaError_t launch_paged_plan(const sx_paged_plan_args& a, cudaStream_t st);
cudaError_t launch_paged_append(const sx_paged_append_args& a, int sms, cudaStream_t st);
cudaError_t launch_paged_attention(const sx_paged_attention_args& a, int sms, cudaStream_t st);
// A (request, kv head)'s share of the attention's work beside its tiles, in tiles.
constexpr int kPagedSegTiles = 2;
// Most tiles and (request, kv head) pairs that the call's table can hold: they are counted in 32 bits.
int64_t paged_attention_cost(const sx_paged_attention_args& a);
// Query heads of a kv head (of G) that are run together.
int paged_attention_group(int G, int hd, bool f32);
size_t paged_attention_workspace(int G, int hd, int sms);

// ---- pooled sessions (pool.cu) --------------------------------------------------------------
struct PoolArgs {
  const int* tok_seq = nullptr;  // [M] sequence and position of each token of the step
  const int* tok_pos = nullptr;
  int M = 0;
  int batch = 0;          // sequences of the session
  int pages_per_seq = 0;  // width of the table
  const int* lens = nullptr;    // [batch] positions each sequence holds pages for
  int* delta = nullptr;         // [batch] what the step adds to them
  const int* table = nullptr;   // [batch][pages_per_seq]
  const int* status = nullptr;  // of sx_paged_plan
  int* slots = nullptr;         // [M]
  int* att_len = nullptr;       // [M]
  int* err = nullptr;           // the session's device error flag (4: the pool could not grow)
};
cudaError_t launch_pool_begin(const PoolArgs& a, cudaStream_t st);
cudaError_t launch_pool_slots(const PoolArgs& a, cudaStream_t st);
// cos / sin [n_pos][half] of (float)position * inv_freq, rounded to f32 before the functions
cudaError_t launch_rope_table(const float* inv_freq, int half, int n_pos, float* cosv, float* sinv, cudaStream_t st);

int paged_sms(int device);  // SMs of a device (0: there is no such device)

}  // namespace sx
