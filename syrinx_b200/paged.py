"""The paged key/value operators behind include/syrinx_paged.h, on torch CUDA tensors.

`plan` turns the requests' lengths into block tables and slot maps, `append` norms, rotates and
scatters new rows into the pages, `attend` is the attention of one new token per request. One
decode step of many requests is

    plan(lens, delta, table, free_pages, n_free, page_size=64, slots=slots, tok_pos=pos, ...)
    q = append(qkv, k, v, slots, n_heads=H, positions=pos, cos=cos, sin=sin)
    out = attend(q.view(n, H, hd), k, v, table, lens)

Everything is enqueued on torch's current stream of the tensors' device; nothing waits for the
GPU, so the calls can be captured into a CUDA graph. A wrong shape, type or device raises
ValueError, what the library refuses raises SyrinxError; what only the GPU can see ends up in
the `status` tensors (include/syrinx_paged.h).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .configs import (SX_DTYPE_BF16, SX_DTYPE_F32, SxPagedAppendArgs, SxPagedAttentionArgs, SxPagedCache,
                      SxPagedPlanArgs)

SX_DTYPE_F16 = 1
_DTYPES = {torch.float32: SX_DTYPE_F32, torch.float16: SX_DTYPE_F16, torch.bfloat16: SX_DTYPE_BF16}
_WORKSPACE = {}  # (heads, kv heads, head_dim, device) -> bytes


def _need(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


def _device(t: torch.Tensor, *others) -> int:
    dev = t.device
    _need(dev.type == "cuda", "the tensors must be on a CUDA device")
    for o in others:
        _need(o is None or o.device == dev, "the tensors must be on one device")
    return dev.index


def _stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


def _ints(t: torch.Tensor, name: str, least: int) -> int:
    _need(t.dtype == torch.int32 and t.is_contiguous() and t.numel() >= least,
          f"{name}: a contiguous int32 tensor of at least {least} entries")
    return t.data_ptr()


def _row(t: torch.Tensor) -> int:
    """Elements from one row to the next (of a single row: its own)."""
    return t.stride(0) if t.shape[0] > 1 else t.numel()


def _table(t: torch.Tensor, n: int) -> int:
    _need(t.dtype == torch.int32 and t.dim() == 2 and t.shape[0] >= n and t.shape[1] >= 1 and t.stride(1) == 1,
          "table: int32 [requests, pages] with contiguous rows")
    return t.data_ptr()


def _cache(c: SxPagedCache, k: torch.Tensor, v: torch.Tensor, layout: str) -> None:
    """k and v pages: [pages, kv heads, page, head_dim] ("hnd") or [pages, page, kv heads, head_dim] ("nhd")."""
    _need(k.dim() == 4 and v.shape == k.shape and v.dtype == k.dtype and v.stride() == k.stride(),
          "k and v: four dimensions, with the same shape, type and strides")
    dtype = _DTYPES.get(k.dtype)
    _need(dtype is not None, "k and v must be float32, float16 or bfloat16")
    s, st = k.shape, k.stride()
    _need(st[3] == 1 or s[3] == 1, "k and v: the head dimension must be contiguous")
    if layout == "hnd":
        heads, page, head_stride, token_stride = s[1], s[2], st[1], st[2]
    else:
        _need(layout == "nhd", 'layout must be "hnd" or "nhd"')
        heads, page, head_stride, token_stride = s[2], s[1], st[2], st[1]
    c.k, c.v = k.data_ptr(), v.data_ptr()
    c.page_stride, c.head_stride, c.token_stride = st[0], head_stride, token_stride
    c.dtype, c.n_pages, c.page_size, c.n_kv_heads, c.head_dim = dtype, s[0], page, heads, s[3]


def plan(lens, delta, table, free_pages, n_free, *, page_size: int, slots=None, tok_seq=None, tok_pos=None,
         starts=None, lens_out=None, n_free_out=None, status=None) -> torch.Tensor:
    """Grow and cut the requests by `delta` (sx_paged_plan). `lens`, `delta` [n], `table` [n, width],
    `free_pages` [pages] and `n_free` [1] are int32; `lens_out` and `n_free_out` default to updating
    `lens` and `n_free` in place. Returns `status` [4]: code, new tokens, pages taken, pages free.
    `check(status)` raises if the code is not SX_OK."""
    n = lens.shape[0]
    lens_out = lens if lens_out is None else lens_out
    n_free_out = n_free if n_free_out is None else n_free_out
    dev = _device(lens, delta, table, free_pages, n_free, slots, tok_seq, tok_pos, starts, lens_out, n_free_out, status)
    if status is None:
        status = torch.empty(4, dtype=torch.int32, device=lens.device)
    most = 0 if slots is None else slots.shape[0]
    a = SxPagedPlanArgs()
    a.lens_in, a.delta, a.n_free_in = _ints(lens, "lens", n), _ints(delta, "delta", n), _ints(n_free, "n_free", 1)
    a.lens_out, a.n_free_out = _ints(lens_out, "lens_out", n), _ints(n_free_out, "n_free_out", 1)
    a.table, a.free_pages = _table(table, n), _ints(free_pages, "free_pages", 1)
    if most:
        a.slots = _ints(slots, "slots", most)
    if tok_seq is not None:
        a.tok_seq = _ints(tok_seq, "tok_seq", max(1, most))
    if tok_pos is not None:
        a.tok_pos = _ints(tok_pos, "tok_pos", max(1, most))
    if starts is not None:
        a.starts = _ints(starts, "starts", n + 1)
    a.status = _ints(status, "status", 4)
    a.table_stride, a.table_width = _row(table), table.shape[1]
    a.n_req, a.n_pages, a.page_size, a.max_tokens = n, free_pages.shape[0], page_size, most
    _lib.check(_lib.lib().sx_paged_plan(C.byref(a), dev, _stream(dev)))
    return status


def append(x, k, v, slots, *, n_heads: int, positions=None, cos=None, sin=None, interleaved: bool = True,
           q_norm=None, k_norm=None, eps: float = 1e-6, layout: str = "hnd", out=None, status=None):
    """Norm, rotate and scatter the rows [query heads | key heads | value heads] of `x` (sx_paged_append).
    Keys and values go to `k` / `v` at `slots`; the query heads are returned, in `out` [rows, n_heads *
    head_dim] where it is given. Rows with slot -1 are left out of both."""
    c = SxPagedAppendArgs()
    _cache(c.cache, k, v, layout)
    dev = _device(x, k, v, slots, positions, cos, sin, q_norm, k_norm, out, status)
    rows, hd = x.shape[0], c.cache.head_dim
    _need(x.dim() == 2 and x.stride(1) == 1 and x.dtype in _DTYPES, "x: floating [rows, heads * head_dim]")
    _need(x.shape[1] == (n_heads + 2 * c.cache.n_kv_heads) * hd, "x: a row is n_heads + 2 kv heads of head_dim")
    if out is None:
        out = torch.empty((rows, n_heads * hd), dtype=x.dtype, device=x.device)
    else:
        _need(out.dim() == 2 and out.shape[0] >= rows and out.shape[1] == n_heads * hd and out.dtype == x.dtype
              and (out.stride(1) == 1 or out.shape[1] == 1), "out: [rows, n_heads * head_dim] of x's type")
    c.x, c.x_stride, c.x_dtype = x.data_ptr(), _row(x), _DTYPES[x.dtype]
    if n_heads:
        c.q_out, c.q_stride = out.data_ptr(), _row(out)
    c.slots = _ints(slots, "slots", rows)
    if positions is not None:
        c.positions = _ints(positions, "positions", rows)
    if cos is not None or sin is not None:
        for t in (cos, sin):
            _need(t is not None and t.dtype == torch.float32 and t.is_contiguous() and t.dim() == 2
                  and t.shape == cos.shape and t.shape[1] == hd // 2, "cos and sin: float32 [positions, head_dim / 2]")
        c.cos, c.sin, c.n_positions = cos.data_ptr(), sin.data_ptr(), cos.shape[0]
    for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t is not None:
            _need(t.dtype == torch.float32 and t.is_contiguous() and t.numel() == hd, f"{name}: float32 [head_dim]")
            setattr(c, name, t.data_ptr())
    if status is not None:
        c.status = _ints(status, "status", 1)
    c.eps, c.n_rows, c.n_heads, c.interleaved = eps, rows, n_heads, int(interleaved)
    _lib.check(_lib.lib().sx_paged_append(C.byref(c), dev, _stream(dev)))
    return out


def workspace_bytes(n_heads: int, n_kv_heads: int, head_dim: int, device: int = 0) -> int:
    """Bytes of the workspace that `attend` with these heads needs (sx_paged_attention_workspace)."""
    key = (n_heads, n_kv_heads, head_dim, device)
    if key not in _WORKSPACE:
        b = C.c_size_t()
        _lib.check(_lib.lib().sx_paged_attention_workspace(n_heads, n_kv_heads, head_dim, device, C.byref(b)))
        _WORKSPACE[key] = b.value
    return _WORKSPACE[key]


def attend(q, k, v, table, lens, *, scale: float | None = None, layout: str = "hnd", out=None, lse=None,
           max_len: int = 0, workspace=None, status=None):
    """Attention of one new token per request (sx_paged_attention): `q` [n, heads, head_dim] over the first
    `lens[i]` positions of the pages in `table[i]`; returns `out`, of q's shape and type. `scale` defaults to
    1 / sqrt(head_dim), `lse` [n, heads] float32 receives log sum exp. Without `workspace` (a tensor of
    `workspace_bytes`) one is taken from torch's allocator for the call."""
    a = SxPagedAttentionArgs()
    _cache(a.cache, k, v, layout)
    dev = _device(q, k, v, table, lens, out, lse, workspace, status)
    hd = a.cache.head_dim
    _need(q.dim() == 3 and q.shape[2] == hd and q.dtype in _DTYPES, "q: floating [requests, heads, head_dim]")
    n, heads = q.shape[0], q.shape[1]
    _need(q.stride(2) == 1 and (heads == 1 or q.stride(1) == hd), "q: a request's heads must be contiguous")
    if out is None:
        out = torch.empty((n, heads, hd), dtype=q.dtype, device=q.device)
    else:
        _need(out.shape == q.shape and out.dtype == q.dtype and out.stride(2) == 1
              and (heads == 1 or out.stride(1) == hd), "out: q's shape and type, a request's heads contiguous")
    if n == 0:
        return out
    bytes_ = workspace_bytes(heads, a.cache.n_kv_heads, hd, dev)
    if workspace is None:
        workspace = torch.empty(bytes_, dtype=torch.uint8, device=q.device)
    else:
        _need(workspace.is_contiguous(), "workspace must be contiguous")
    a.q, a.out, a.q_stride, a.out_stride = q.data_ptr(), out.data_ptr(), _row(q), _row(out)
    if lse is not None:
        _need(lse.dtype == torch.float32 and lse.is_contiguous() and lse.numel() == n * heads,
              "lse: float32 [requests, heads]")
        a.lse = lse.data_ptr()
    a.table, a.lens = _table(table, n), _ints(lens, "lens", n)
    if status is not None:
        a.status = _ints(status, "status", 1)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    a.table_stride, a.table_width, a.n_req, a.n_heads = _row(table), table.shape[1], n, heads
    a.q_dtype, a.max_len, a.scale = _DTYPES[q.dtype], max_len, hd ** -0.5 if scale is None else scale
    _lib.check(_lib.lib().sx_paged_attention(C.byref(a), dev, _stream(dev)))
    return out


def check(status: torch.Tensor) -> None:
    """Raise SyrinxError if a status tensor holds a code (waits for the GPU)."""
    code = int(status.view(-1)[0])
    if code:
        raise _lib.SyrinxError(code, "a paged operator refused its input on the device")
