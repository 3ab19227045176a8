/*
 * syrinx_paged.h — C ABI of the operators that serve a paged key/value pool on a B200: block
 * tables and slot maps from the requests' lengths, the append of new keys and values, and the
 * attention of one new token per request over its pages.
 *
 * A session (include/syrinx_dualar.h) runs them inside a pooled session
 * (sx_session_create_pool); here a program calls them on its own cache. Every call enqueues
 * one or two kernels on `cuda_stream` (a cudaStream_t of `device`; NULL is the legacy default
 * stream) and returns without waiting. All pointers are device pointers on `device`. Nothing
 * is allocated, kept between calls or copied to the host, so every call can be captured into
 * a CUDA graph. The current device of the calling thread is left as it was.
 *
 * Status codes and sx_last_error() are those of include/syrinx_dualar.h. What a call can see
 * on the host (null pointers, sizes, types, alignment) it refuses with a status code before
 * anything is enqueued. What only the device sees (a length beyond its row, a page id or a
 * slot outside the cache) is never used as an address: it is written to the call's `status`
 * words, as each operator says.
 */
#ifndef SYRINX_PAGED_H
#define SYRINX_PAGED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * One layer's keys and values: n_pages pages of page_size positions. Element (page, head,
 * position, d) is at page * page_stride + head * head_stride + position * token_stride + d
 * elements from k (and from v), so [page][head][position][d] (the session's layout) and
 * [page][position][head][d] are both described. Base pointers and strides are multiples of 16
 * bytes. A slot is page * page_size + position.
 */
typedef struct sx_paged_cache {
  void* k;
  void* v;
  int64_t page_stride, head_stride, token_stride; /* in elements, the same for k and v */
  int32_t dtype;                                  /* SX_DTYPE_F32, SX_DTYPE_BF16 or SX_DTYPE_F16 */
  int32_t n_pages;                                /* n_pages * page_size < 2^31 */
  int32_t page_size;                              /* a power of two, 8 .. 1024 */
  int32_t n_kv_heads;
  int32_t head_dim; /* 32, 64, 128 or 256 */
  int32_t reserved; /* 0 */
} sx_paged_cache;

/*
 * Block tables and slot maps. Request i holds lens_in[i] positions and changes by delta[i]:
 * it grows by that many new tokens, or, where delta is negative, is cut back (to nothing at
 * most), so its new length is max(0, lens_in[i] + delta[i]). Row i of `table` holds
 * ceil(length / page_size) page ids. The free pages are a stack: free_pages[0 .. n_free), the
 * top last. Pages that rows no longer need are pushed in (row, page) order, then the pages
 * that rows lack are popped in (row, page) order; the other entries of `table` and of
 * `free_pages` are left as they were.
 *
 * The new tokens of all requests, request by request, get their slot, request and position;
 * the entries of the three arrays behind the last token, up to max_tokens, become -1. starts
 * (n_req + 1) holds where each request's tokens begin.
 *
 * status[0] is SX_OK or why nothing was changed: SX_E_RANGE (too few free pages, more than
 * max_tokens new tokens, a row longer than table_width pages) or SX_E_INVALID (a negative
 * length, a stack larger than n_pages, a page id outside the pool). In that case the lengths,
 * the stack and the table stay as they were, every slot, request and position is -1, so that a
 * following append writes nothing, and `starts` is 0. status[1 .. 3]: new tokens, pages popped, pages
 * free afterwards.
 */
typedef struct sx_paged_plan_args {
  const int32_t* lens_in; /* [n_req] */
  const int32_t* delta;   /* [n_req] */
  const int32_t* n_free_in;
  int32_t* lens_out;   /* [n_req]; may be lens_in */
  int32_t* n_free_out; /* may be n_free_in */
  int32_t* table;      /* [n_req][table_stride] */
  int32_t* free_pages; /* [n_pages] */
  int32_t* slots;      /* [max_tokens]; null with max_tokens == 0 */
  int32_t* tok_seq;    /* [max_tokens], nullable */
  int32_t* tok_pos;    /* [max_tokens], nullable */
  int32_t* starts;     /* [n_req + 1], nullable */
  int32_t* status;     /* [4] */
  int64_t table_stride;
  int32_t table_width; /* pages a row can hold */
  int32_t n_req;       /* 1 .. SX_PAGED_MAX_REQUESTS */
  int32_t n_pages;
  int32_t page_size; /* a power of two, 8 .. 1024 */
  int32_t max_tokens;
  int32_t reserved; /* 0 */
} sx_paged_plan_args;

#define SX_PAGED_MAX_REQUESTS 8192

int sx_paged_plan(const sx_paged_plan_args* args, int32_t device, void* cuda_stream);

/*
 * Append of new rows. Row j of x is [n_heads query | n_kv_heads key | n_kv_heads value heads]
 * of head_dim elements. Per query and key head: RMSNorm with the gains q_norm / k_norm
 * (x / sqrt(mean(x^2) + eps) * gain; null: none), then a rotation of the pairs (2i, 2i + 1)
 * (interleaved) or (i, i + head_dim / 2) by the angle whose cosine and sine stand in row
 * positions[j] of `cos` / `sin` (null: none). Query heads go to q_out (null: they are
 * dropped), keys and values into the cache at slots[j]. A row with slot -1 writes nothing.
 * Arithmetic is f32. Rows must not share a slot. q_out may be the query part of x itself.
 *
 * A slot outside the cache or a position outside the tables writes nothing for that row and
 * sets *status (nullable) to SX_E_RANGE; status is not written otherwise.
 */
typedef struct sx_paged_append_args {
  sx_paged_cache cache;
  const void* x;            /* [n_rows][x_stride] */
  void* q_out;              /* [n_rows][q_stride], the type of x; nullable */
  const int32_t* slots;     /* [n_rows] */
  const int32_t* positions; /* [n_rows]; null without cos / sin */
  const float* cos;         /* [n_positions][head_dim / 2] */
  const float* sin;
  const float* q_norm; /* [head_dim] */
  const float* k_norm;
  int32_t* status;
  int64_t x_stride, q_stride; /* elements, multiples of 16 bytes */
  float eps;
  int32_t x_dtype; /* SX_DTYPE_F32, or the cache's type */
  int32_t n_rows;  /* 0: nothing is done */
  int32_t n_heads; /* query heads in x, >= 0 */
  int32_t n_positions;
  int32_t interleaved;
} sx_paged_append_args;

int sx_paged_append(const sx_paged_append_args* args, int32_t device, void* cuda_stream);

/*
 * Attention of one new token per request: out[i][h] = sum_t softmax_t(scale * q[i][h].k_t) v_t
 * over the lens[i] positions of request i's pages, for kv head h / (n_heads / n_kv_heads).
 * lse[i][h] = log sum_t exp(scale * q.k_t). A request of length 0 gets zeros and -inf, as does
 * a row whose scores are all -inf. Positions behind a request's length are never read. Scores,
 * softmax and sums are f32 whatever the types are; over f16 pages the weights meet the values
 * with 22 bits, or to 2^-39 of the largest. The result does not depend on the other
 * requests' values; it is the same from call to call.
 *
 * A length beyond table_width pages is cut to it, and a page id outside the cache reads as
 * zeros; either sets *status (nullable) to SX_E_RANGE, which is not written otherwise.
 *
 * The key axis of all requests is cut into even shares for the GPU's SMs (so the last bits of
 * a result depend on the lengths of all of them); partial results pass through `workspace`,
 * whose content means nothing before and after the call. Calls that may run at the same time
 * (on two streams, or two captured graphs) need a workspace each. `out` may be `q` itself.
 */
typedef struct sx_paged_attention_args {
  sx_paged_cache cache;
  const void* q;        /* [n_req][q_stride]: n_heads heads of head_dim */
  void* out;            /* [n_req][out_stride], the type of q */
  float* lse;           /* [n_req][n_heads], nullable */
  const int32_t* table; /* [n_req][table_stride] page ids */
  const int32_t* lens;  /* [n_req] */
  int32_t* status;
  void* workspace; /* 16-byte aligned; null: no request is split, which short ones are not anyway */
  size_t workspace_bytes;
  int64_t q_stride, out_stride; /* elements, multiples of 16 bytes */
  int64_t table_stride;
  int32_t table_width;
  int32_t n_req;   /* 0: nothing is done; n_req x kv heads x tiles of a row below 2^32 */
  int32_t n_heads; /* a multiple of n_kv_heads */
  int32_t q_dtype; /* SX_DTYPE_F32, or the cache's type */
  int32_t max_len; /* what no length exceeds, as far as the host knows (0: table_width pages);
                      it chooses the launch and never the result's meaning */
  float scale;
} sx_paged_attention_args;

int sx_paged_attention(const sx_paged_attention_args* args, int32_t device, void* cuda_stream);

/* Workspace bytes that any sx_paged_attention call with these heads and head_dim needs
 * (whatever its requests, lengths and types are). */
int sx_paged_attention_workspace(int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int32_t device,
                                 size_t* bytes_out);

#ifdef __cplusplus
}
#endif

#endif /* SYRINX_PAGED_H */
