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
import struct

import torch

from . import _lib
from .configs import SX_DTYPE_BF16, SX_DTYPE_F32, SxPagedAppendArgs, SxPagedAttentionArgs, SxPagedPlanArgs

SX_DTYPE_F16 = 1
_DTYPES = {torch.float32: SX_DTYPE_F32, torch.float16: SX_DTYPE_F16, torch.bfloat16: SX_DTYPE_BF16}
_WORKSPACE = {}  # (heads, kv heads, head_dim, device) -> bytes


def _need(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


# cudaStream_t of torch's current stream on a device; the public call builds a Stream object for it,
# a quarter of a small operator's host time
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_I32, _F32 = torch.int32, torch.float32


# The argument structs of include/syrinx_paged.h, packed in one go (native sizes and alignment; the
# ctypes structures of configs.py spell the same fields out).
_CACHE = "PPqqqiiiiii"
_PLAN_ARGS = struct.Struct("@12Pq6i0q")
_APPEND_ARGS = struct.Struct("@" + _CACHE + "9P2qf5i0q")
_ATTEND_ARGS = struct.Struct("@" + _CACHE + "7PN3q5if0q")
for _s, _c in ((_PLAN_ARGS, SxPagedPlanArgs), (_APPEND_ARGS, SxPagedAppendArgs), (_ATTEND_ARGS, SxPagedAttentionArgs)):
    assert _s.size == C.sizeof(_c), "argument struct out of step with include/syrinx_paged.h"


def _on(dev: int, *tensors) -> None:
    """Every tensor (None: left out) is on CUDA device `dev`."""
    if dev < 0:
        raise ValueError("the tensors must be on a CUDA device")
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError("the tensors must be on one device")


def _ints(dev: int, t: torch.Tensor, name: str, least: int) -> int:
    """Address of a contiguous int32 tensor of at least `least` entries on device `dev`."""
    if t.dtype is _I32 and t.get_device() == dev and t.is_contiguous() and t.numel() >= least:
        return t.data_ptr()
    raise ValueError(f"{name}: a contiguous int32 tensor of at least {least} entries on the same CUDA device")


def _table(dev: int, t: torch.Tensor, n: int) -> tuple:
    """Address, elements from row to row and pages a row of a block table."""
    s = t.shape
    if t.dtype is not _I32 or len(s) != 2 or s[0] < n or s[1] < 1 or t.get_device() != dev:
        raise ValueError("table: int32 [requests, pages] on the same CUDA device")
    row, step = t.stride()
    if step != 1:
        raise ValueError("table: a row's pages must be contiguous")
    return t.data_ptr(), row if s[0] > 1 else s[1], s[1]


def _cache(k: torch.Tensor, v: torch.Tensor, layout: str) -> tuple:
    """The fields of sx_paged_cache: k and v pages are [pages, kv heads, page, head_dim] ("hnd") or
    [pages, page, kv heads, head_dim] ("nhd")."""
    s, st, dtype = k.shape, k.stride(), _DTYPES.get(k.dtype)
    if len(s) != 4 or v.shape != s or v.dtype is not k.dtype or v.stride() != st:
        raise ValueError("k and v: four dimensions, with the same shape, type and strides")
    if dtype is None or st[3] != 1:
        raise ValueError("k and v: float32, float16 or bfloat16, the head dimension contiguous")
    if layout == "hnd":
        return k.data_ptr(), v.data_ptr(), st[0], st[1], st[2], dtype, s[0], s[2], s[1], s[3], 0
    _need(layout == "nhd", 'layout must be "hnd" or "nhd"')
    return k.data_ptr(), v.data_ptr(), st[0], st[2], st[1], dtype, s[0], s[1], s[2], s[3], 0


def plan(lens, delta, table, free_pages, n_free, *, page_size: int, slots=None, tok_seq=None, tok_pos=None,
         starts=None, lens_out=None, n_free_out=None, status=None) -> torch.Tensor:
    """Grow and cut the requests by `delta` (sx_paged_plan). `lens`, `delta` [n], `table` [n, width],
    `free_pages` [pages] and `n_free` [1] are int32; `lens_out` and `n_free_out` default to updating
    `lens` and `n_free` in place. Returns `status` [4]: code, new tokens, pages taken, pages free.
    `check(status)` raises if the code is not SX_OK."""
    n, most = lens.shape[0], 0 if slots is None else slots.shape[0]
    lens_out = lens if lens_out is None else lens_out
    n_free_out = n_free if n_free_out is None else n_free_out
    if status is None:
        status = torch.empty(4, dtype=_I32, device=lens.device)
    dev, least = lens.get_device(), max(1, most)
    if dev < 0:
        raise ValueError("the tensors must be on a CUDA device")
    address, stride, width = _table(dev, table, n)
    args = _PLAN_ARGS.pack(
        _ints(dev, lens, "lens", n), _ints(dev, delta, "delta", n), _ints(dev, n_free, "n_free", 1),
        _ints(dev, lens_out, "lens_out", n), _ints(dev, n_free_out, "n_free_out", 1), address,
        _ints(dev, free_pages, "free_pages", 1), _ints(dev, slots, "slots", most) if most else 0,
        0 if tok_seq is None else _ints(dev, tok_seq, "tok_seq", least),
        0 if tok_pos is None else _ints(dev, tok_pos, "tok_pos", least),
        0 if starts is None else _ints(dev, starts, "starts", n + 1), _ints(dev, status, "status", 4),
        stride, width, n, free_pages.shape[0], page_size, most, 0)
    _lib.check(_lib.lib().sx_paged_plan(args, dev, _stream(dev)))
    return status


def append(x, k, v, slots, *, n_heads: int, positions=None, cos=None, sin=None, interleaved: bool = True,
           q_norm=None, k_norm=None, eps: float = 1e-6, layout: str = "hnd", out=None, status=None):
    """Norm, rotate and scatter the rows [query heads | key heads | value heads] of `x` (sx_paged_append).
    Keys and values go to `k` / `v` at `slots`; the query heads are returned, in `out` [rows, n_heads *
    head_dim] where it is given. Rows with slot -1 are left out of both."""
    cache = _cache(k, v, layout)
    (rows, width), (x_row, x_step) = x.shape, x.stride()
    hkv, hd, dtype = cache[8], cache[9], x.dtype
    q_width = n_heads * hd
    if dtype not in _DTYPES or x_step != 1 or width != q_width + 2 * hkv * hd:
        raise ValueError("x: floating [rows, (n_heads + 2 kv heads) * head_dim], rows contiguous")
    if out is None:
        out = torch.empty((rows, q_width), dtype=dtype, device=x.device)
    q_rows, q_row, q_step = *out.shape[:1], *out.stride()
    if out.shape[1] != q_width or q_rows < rows or out.dtype is not dtype or (q_step != 1 and q_width > 1):
        raise ValueError("out: [rows, n_heads * head_dim] of x's type, rows contiguous")
    if rows < 2:  # the one row's stride says nothing
        x_row, q_row = width, q_width
    n_pos = 0
    if cos is not None or sin is not None:
        if (cos is None or sin is None or cos.dtype is not _F32 or sin.dtype is not _F32 or not cos.is_contiguous()
                or not sin.is_contiguous() or sin.shape != (table := cos.shape) or len(table) != 2
                or table[1] != hd // 2 or not table[0]):
            raise ValueError("cos and sin: float32 [positions, head_dim / 2], one position at least")
        n_pos = table[0]
    dev = x.get_device()
    _on(dev, k, v, cos, sin, q_norm, k_norm, out)
    for t in (q_norm, k_norm):
        if t is not None and (t.dtype is not _F32 or t.numel() != hd or not t.is_contiguous()):
            raise ValueError("q_norm and k_norm: float32 [head_dim]")
    args = _APPEND_ARGS.pack(
        *cache, x.data_ptr(), out.data_ptr() if n_heads else 0, _ints(dev, slots, "slots", rows),
        0 if positions is None else _ints(dev, positions, "positions", rows), cos.data_ptr() if n_pos else 0,
        sin.data_ptr() if n_pos else 0, 0 if q_norm is None else q_norm.data_ptr(),
        0 if k_norm is None else k_norm.data_ptr(), 0 if status is None else _ints(dev, status, "status", 1),
        x_row, q_row, eps, _DTYPES[dtype], rows, n_heads, n_pos, int(interleaved))
    _lib.check(_lib.lib().sx_paged_append(args, dev, _stream(dev)))
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
    `workspace_bytes`) one is taken from torch's allocator for the call, where the requests are split at all."""
    cache = _cache(k, v, layout)
    hkv, hd, dtype, shape = cache[8], cache[9], q.dtype, q.shape
    if len(shape) != 3 or shape[2] != hd or dtype not in _DTYPES:
        raise ValueError("q: floating [requests, heads, head_dim]")
    n, heads, _ = shape
    q_row, q_head, q_step = q.stride()
    if q_step != 1 or (q_head != hd and heads > 1):
        raise ValueError("q: a request's heads must be contiguous")
    if out is None:
        out = torch.empty((n, heads, hd), dtype=dtype, device=q.device)
        out_row = heads * hd
    else:
        if out.shape != shape or out.dtype is not dtype:
            raise ValueError("out: q's shape and type")
        out_row, out_head, out_step = out.stride()
        if out_step != 1 or (out_head != hd and heads > 1):
            raise ValueError("out: a request's heads must be contiguous")
    if n == 1:  # the one row's stride says nothing
        q_row = out_row = heads * hd
    dev = q.get_device()
    _on(dev, k, v, out, lse, workspace)
    if n == 0:
        return out
    address, stride, width = _table(dev, table, n)
    pointer = size = 0  # few and short requests are not split, so they need no workspace
    if workspace is not None:
        _need(workspace.is_contiguous(), "workspace must be contiguous")
        pointer, size = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    elif n * hkv > 64 or (max_len or width * cache[7]) > 256:
        size = _WORKSPACE.get((heads, hkv, hd, dev)) or workspace_bytes(heads, hkv, hd, dev)
        workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
        pointer = workspace.data_ptr()
    if lse is not None and (lse.dtype is not _F32 or lse.numel() != n * heads or not lse.is_contiguous()):
        raise ValueError("lse: float32 [requests, heads]")
    args = _ATTEND_ARGS.pack(
        *cache, q.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), address,
        _ints(dev, lens, "lens", n), 0 if status is None else _ints(dev, status, "status", 1), pointer, size,
        q_row, out_row, stride, width, n, heads, _DTYPES[dtype], max_len, hd ** -0.5 if scale is None else scale)
    _lib.check(_lib.lib().sx_paged_attention(args, dev, _stream(dev)))
    return out


def check(status: torch.Tensor) -> None:
    """Raise SyrinxError if a status tensor holds a code (waits for the GPU)."""
    code = int(status.view(-1)[0])
    if code:
        raise _lib.SyrinxError(code, "a paged operator refused its input on the device")
