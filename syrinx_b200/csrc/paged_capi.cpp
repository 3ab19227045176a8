// paged_capi.cpp — the extern "C" boundary declared in include/syrinx_paged.h: argument checks
// and the selection of the caller's device for the length of the call.
#include <cuda_runtime.h>

#include <atomic>
#include <exception>
#include <string>

#include "paged.hpp"
#include "sx_internal.hpp"

namespace sx {

namespace {

int refuse(int code, const std::string& msg) {
  set_error(msg);
  return code;
}

size_t elem_bytes(int dtype) { return dtype == SX_DTYPE_F32 ? 4 : 2; }
bool known(int dtype) { return dtype == SX_DTYPE_F32 || dtype == SX_DTYPE_BF16 || dtype == SX_DTYPE_F16; }
bool pow2_page(int p) { return p >= 8 && p <= 1024 && (p & (p - 1)) == 0; }
bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) % to) == 0; }

int check_cache(const sx_paged_cache& c, const char* who) {
  const std::string w(who);
  if (!c.k || !c.v) return refuse(SX_E_INVALID, w + ": null cache");
  if (!known(c.dtype)) return refuse(SX_E_UNSUPPORTED, w + ": the cache holds f32, bf16 or f16");
  if (c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
    return refuse(SX_E_UNSUPPORTED, w + ": head_dim must be 32, 64, 128 or 256");
  if (!pow2_page(c.page_size)) return refuse(SX_E_UNSUPPORTED, w + ": page_size must be a power of two, 8 .. 1024");
  if (c.n_pages < 1 || c.n_kv_heads < 1 || c.reserved != 0)
    return refuse(SX_E_INVALID, w + ": non-positive pages or kv heads, or reserved is not 0");
  if ((int64_t)c.n_pages * c.page_size > INT32_MAX)
    return refuse(SX_E_RANGE, w + ": n_pages * page_size must be below 2^31");
  const int64_t per = 16 / (int64_t)elem_bytes(c.dtype);
  if (!aligned(c.k, 16) || !aligned(c.v, 16) || c.page_stride % per || c.head_stride % per || c.token_stride % per)
    return refuse(SX_E_INVALID, w + ": cache pointers and strides must be multiples of 16 bytes");
  if (c.page_stride < 0 || c.head_stride < 0 || c.token_stride < c.head_dim)
    return refuse(SX_E_INVALID, w + ": cache strides must not be negative, and a token's head must be contiguous");
  return SX_OK;
}

int check_row(const void* p, int64_t stride, int64_t width, int dtype, const std::string& what) {
  if (!aligned(p, 16) || stride % (16 / (int64_t)elem_bytes(dtype)))
    return refuse(SX_E_INVALID, what + " and its row stride must be multiples of 16 bytes");
  if (stride < width) return refuse(SX_E_INVALID, what + ": the row stride is shorter than a row");
  return SX_OK;
}

}  // namespace

int paged_check(const sx_paged_plan_args& a) {
  if (!a.lens_in || !a.delta || !a.n_free_in || !a.lens_out || !a.n_free_out || !a.table || !a.free_pages || !a.status)
    return refuse(SX_E_INVALID, "sx_paged_plan: null argument");
  if (a.n_req < 1 || a.n_req > SX_PAGED_MAX_REQUESTS)
    return refuse(SX_E_RANGE, "sx_paged_plan: n_req must be 1.." + std::to_string(SX_PAGED_MAX_REQUESTS));
  if (!pow2_page(a.page_size))
    return refuse(SX_E_UNSUPPORTED, "sx_paged_plan: page_size must be a power of two, 8 .. 1024");
  if (a.n_pages < 1 || a.table_width < 1 || a.max_tokens < 0 || a.reserved != 0)
    return refuse(SX_E_INVALID, "sx_paged_plan: non-positive pages or table width, negative max_tokens, or reserved is not 0");
  if (a.max_tokens > INT32_MAX - 4) return refuse(SX_E_RANGE, "sx_paged_plan: max_tokens must be below 2^31 - 4");
  if (a.max_tokens > 0 && !a.slots) return refuse(SX_E_INVALID, "sx_paged_plan: null slots");
  if (a.max_tokens == 0 && (a.slots || a.tok_seq || a.tok_pos))
    return refuse(SX_E_INVALID, "sx_paged_plan: token arrays without max_tokens");
  if (a.table_stride < a.table_width) return refuse(SX_E_INVALID, "sx_paged_plan: table_stride is below table_width");
  if ((int64_t)a.n_pages * a.page_size > INT32_MAX || (int64_t)a.table_width * a.page_size > INT32_MAX ||
      (int64_t)a.n_req * a.table_width > INT32_MAX)
    return refuse(SX_E_RANGE, "sx_paged_plan: pages, a row's positions and the table's entries must be below 2^31");
  return SX_OK;
}

int paged_check(const sx_paged_append_args& a) {
  int rc = check_cache(a.cache, "sx_paged_append");
  if (rc) return rc;
  const sx_paged_cache& c = a.cache;
  if (a.n_rows < 0 || a.n_heads < 0) return refuse(SX_E_INVALID, "sx_paged_append: negative rows or heads");
  if (a.n_rows > 0 && (!a.x || !a.slots)) return refuse(SX_E_INVALID, "sx_paged_append: null x or slots");
  if (a.x_dtype != SX_DTYPE_F32 && a.x_dtype != c.dtype)
    return refuse(SX_E_UNSUPPORTED, "sx_paged_append: x is f32 or of the cache's type");
  const int64_t heads = (int64_t)a.n_heads + 2 * (int64_t)c.n_kv_heads;
  if (heads * c.head_dim > INT32_MAX || a.n_heads > (1 << 20) || c.n_kv_heads > (1 << 20))
    return refuse(SX_E_RANGE, "sx_paged_append: too many heads");
  if ((rc = check_row(a.x, a.x_stride, heads * c.head_dim, a.x_dtype, "sx_paged_append: x"))) return rc;
  if (a.q_out && (rc = check_row(a.q_out, a.q_stride, (int64_t)a.n_heads * c.head_dim, a.x_dtype, "sx_paged_append: q_out")))
    return rc;
  if ((a.cos == nullptr) != (a.sin == nullptr)) return refuse(SX_E_INVALID, "sx_paged_append: cos and sin go together");
  if (a.cos && (!a.positions || a.n_positions < 1))
    return refuse(SX_E_INVALID, "sx_paged_append: a rotation needs positions and n_positions >= 1");
  if (!aligned(a.cos, 16) || !aligned(a.sin, 16) || !aligned(a.q_norm, 16) || !aligned(a.k_norm, 16))
    return refuse(SX_E_INVALID, "sx_paged_append: cos, sin and the gains must be 16-byte aligned");
  if (!(a.eps >= 0.f)) return refuse(SX_E_INVALID, "sx_paged_append: eps must not be negative");
  return SX_OK;
}

int paged_check(const sx_paged_attention_args& a, int sms) {
  int rc = check_cache(a.cache, "sx_paged_attention");
  if (rc) return rc;
  const sx_paged_cache& c = a.cache;
  if (a.n_req < 0) return refuse(SX_E_INVALID, "sx_paged_attention: negative n_req");
  if (a.n_req > 0 && (!a.q || !a.out || !a.table || !a.lens))
    return refuse(SX_E_INVALID, "sx_paged_attention: null argument");
  if (a.q_dtype != SX_DTYPE_F32 && a.q_dtype != c.dtype)
    return refuse(SX_E_UNSUPPORTED, "sx_paged_attention: q is f32 or of the cache's type");
  if (a.n_heads < 1 || a.n_heads % c.n_kv_heads)
    return refuse(SX_E_UNSUPPORTED, "sx_paged_attention: n_heads must be a multiple of n_kv_heads");
  if (a.n_heads > (1 << 16)) return refuse(SX_E_RANGE, "sx_paged_attention: too many heads");
  if (a.table_width < 1 || a.table_stride < a.table_width || a.max_len < 0)
    return refuse(SX_E_INVALID, "sx_paged_attention: bad table width or stride, or negative max_len");
  if ((int64_t)a.table_width * c.page_size > INT32_MAX)
    return refuse(SX_E_RANGE, "sx_paged_attention: a row's positions must be below 2^31");
  if ((int64_t)a.n_req * a.n_heads > INT32_MAX)
    return refuse(SX_E_RANGE, "sx_paged_attention: n_req * n_heads must be below 2^31");
  if (paged_attention_cost(a) > UINT32_MAX - (1 << 16))
    return refuse(SX_E_RANGE, "sx_paged_attention: requests x kv heads x a row's positions is too large for one call");
  const int64_t width = (int64_t)a.n_heads * c.head_dim;
  if ((rc = check_row(a.q, a.q_stride, width, a.q_dtype, "sx_paged_attention: q"))) return rc;
  if ((rc = check_row(a.out, a.out_stride, width, a.q_dtype, "sx_paged_attention: out"))) return rc;
  if (!aligned(a.workspace, 16)) return refuse(SX_E_INVALID, "sx_paged_attention: workspace must be 16-byte aligned");
  const size_t need = paged_attention_workspace(a.n_heads / c.n_kv_heads, c.head_dim, sms);
  if (a.workspace && a.workspace_bytes < need)
    return refuse(SX_E_RANGE, "sx_paged_attention: workspace holds " + std::to_string(a.workspace_bytes) + " bytes, " +
                                  std::to_string(need) + " needed");
  return SX_OK;
}

int64_t paged_attention_cost(const sx_paged_attention_args& a) {
  const int hd = a.cache.head_dim;
  const int keys = a.cache.dtype == SX_DTYPE_F32 ? 1024 / hd : hd == 32 ? 64 : hd == 64 ? 32 : 16;
  const int64_t tiles = ((int64_t)a.table_width * a.cache.page_size + keys - 1) / keys + kPagedSegTiles;
  const int G = a.n_heads / a.cache.n_kv_heads, run = paged_attention_group(G, hd, a.cache.dtype == SX_DTYPE_F32);
  const int64_t rows = (int64_t)a.n_req * a.cache.n_kv_heads * ((G + run - 1) / run);
  return rows > INT64_MAX / tiles ? INT64_MAX : rows * tiles;
}

int paged_sms(int device) {
  static std::atomic<int> cached[64];
  if (device < 0) return 0;
  if (device < 64 && cached[device].load(std::memory_order_relaxed)) return cached[device].load(std::memory_order_relaxed);
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  if (device < 64) cached[device].store(n, std::memory_order_relaxed);
  return n;
}

namespace {

// The caller's device for the length of a call: the thread's current device comes back.
struct OnDevice {
  int before = -1;
  bool ok = false;
  explicit OnDevice(int device) {
    int now = -1;
    if (cudaGetDevice(&now) != cudaSuccess) return;
    if (now != device) {
      if (cudaSetDevice(device) != cudaSuccess) return;
      before = now;
    }
    ok = true;
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

template <class F>
int enqueue(const char* who, int device, F&& launch) {
  OnDevice on(device);
  if (!on.ok) return refuse(SX_E_CUDA, std::string(who) + ": cudaSetDevice failed");
  const cudaError_t e = launch();
  if (e != cudaSuccess) {
    cudaGetLastError();
    return refuse(SX_E_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
  }
  return SX_OK;
}

template <class F>
int guarded(F&& f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return SX_E_OOM;
  } catch (const std::exception& e) {
    return refuse(SX_E_INVALID, std::string("internal error: ") + e.what());
  } catch (...) {
    return SX_E_INVALID;
  }
}

}  // namespace
}  // namespace sx

using namespace sx;

extern "C" {

int sx_paged_plan(const sx_paged_plan_args* args, int32_t device, void* cuda_stream) {
  return guarded([&]() -> int {
    if (!args) return refuse(SX_E_INVALID, "sx_paged_plan: null argument");
    if (int rc = paged_check(*args)) return rc;
    if (!paged_sms(device)) return refuse(SX_E_INVALID, "sx_paged_plan: no such CUDA device");
    return enqueue("sx_paged_plan", device,
                   [&] { return launch_paged_plan(*args, static_cast<cudaStream_t>(cuda_stream)); });
  });
}

int sx_paged_append(const sx_paged_append_args* args, int32_t device, void* cuda_stream) {
  return guarded([&]() -> int {
    if (!args) return refuse(SX_E_INVALID, "sx_paged_append: null argument");
    if (int rc = paged_check(*args)) return rc;
    const int sms = paged_sms(device);
    if (!sms) return refuse(SX_E_INVALID, "sx_paged_append: no such CUDA device");
    if (args->n_rows == 0) return SX_OK;
    return enqueue("sx_paged_append", device,
                   [&] { return launch_paged_append(*args, sms, static_cast<cudaStream_t>(cuda_stream)); });
  });
}

int sx_paged_attention(const sx_paged_attention_args* args, int32_t device, void* cuda_stream) {
  return guarded([&]() -> int {
    if (!args) return refuse(SX_E_INVALID, "sx_paged_attention: null argument");
    const int sms = paged_sms(device);
    // a machine without the device still refuses bad arguments by their own names
    if (int rc = paged_check(*args, sms ? sms : 1)) return rc;
    if (!sms) return refuse(SX_E_INVALID, "sx_paged_attention: no such CUDA device");
    if (args->n_req == 0) return SX_OK;
    return enqueue("sx_paged_attention", device,
                   [&] { return launch_paged_attention(*args, sms, static_cast<cudaStream_t>(cuda_stream)); });
  });
}

int sx_paged_attention_workspace(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int32_t device,
                                 size_t* bytes_out) {
  return guarded([&]() -> int {
    if (!bytes_out) return refuse(SX_E_INVALID, "sx_paged_attention_workspace: null argument");
    if (n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads || n_heads > (1 << 16) ||
        (head_dim != 32 && head_dim != 64 && head_dim != 128 && head_dim != 256))
      return refuse(SX_E_UNSUPPORTED, "sx_paged_attention_workspace: heads or head_dim not supported");
    const int sms = paged_sms(device);
    if (!sms) return refuse(SX_E_INVALID, "sx_paged_attention_workspace: no such CUDA device");
    *bytes_out = paged_attention_workspace(n_heads / n_kv_heads, head_dim, sms);
    return SX_OK;
  });
}

}  // extern "C"
