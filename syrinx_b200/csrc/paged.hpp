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
size_t paged_attention_workspace(int G, int hd, int sms);

int paged_sms(int device);  // SMs of a device (0: there is no such device)

}  // namespace sx
