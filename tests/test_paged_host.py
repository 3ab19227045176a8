"""Host-side checks of the paged key/value operators (include/syrinx_paged.h) without a GPU:
every refusal that the library makes before it touches the device, and the Python layer's."""
import ctypes as C

import pytest

import syrinx_b200 as sx
from syrinx_b200 import _lib
from syrinx_b200.configs import (SX_DTYPE_BF16, SX_DTYPE_F32, SX_DTYPE_Q8_0, SxPagedAppendArgs, SxPagedAttentionArgs,
                                 SxPagedPlanArgs)

P = 0x10000  # an aligned address that nothing reads: every call here is refused on the host
INVALID, UNSUPPORTED, RANGE = -1, -6, -7


def cache(c, **kw):
    vals = dict(k=P, v=P, page_stride=8 * 64 * 128, head_stride=64 * 128, token_stride=128, dtype=SX_DTYPE_BF16,
                n_pages=10, page_size=64, n_kv_heads=8, head_dim=128, reserved=0)
    vals.update(kw)
    for n, v in vals.items():
        setattr(c, n, v)


def call(fn, args):
    rc = getattr(_lib.lib(), fn)(C.byref(args), 0, None)
    return rc, _lib.lib().sx_last_error().decode()


def plan_args(**kw):
    a = SxPagedPlanArgs()
    vals = dict(lens_in=P, delta=P, n_free_in=P, lens_out=P, n_free_out=P, table=P, free_pages=P, slots=P, tok_seq=P,
                tok_pos=P, starts=P, status=P, table_stride=32, table_width=32, n_req=4, n_pages=100, page_size=64,
                max_tokens=16, reserved=0)
    vals.update(kw)
    for n, v in vals.items():
        setattr(a, n, v)
    return a


def append_args(c=None, **kw):
    a = SxPagedAppendArgs()
    cache(a.cache, **(c or {}))
    vals = dict(x=P, q_out=P, slots=P, positions=P, cos=P, sin=P, q_norm=P, k_norm=P, status=P, x_stride=48 * 128,
                q_stride=32 * 128, eps=1e-6, x_dtype=SX_DTYPE_F32, n_rows=3, n_heads=32, n_positions=100, interleaved=1)
    vals.update(kw)
    for n, v in vals.items():
        setattr(a, n, v)
    return a


def attention_args(c=None, **kw):
    a = SxPagedAttentionArgs()
    cache(a.cache, **(c or {}))
    vals = dict(q=P, out=P, lse=P, table=P, lens=P, status=P, workspace=P, workspace_bytes=1 << 40, q_stride=32 * 128,
                out_stride=32 * 128, table_stride=16, table_width=16, n_req=3, n_heads=32, q_dtype=SX_DTYPE_BF16,
                max_len=0, scale=0.1)
    vals.update(kw)
    for n, v in vals.items():
        setattr(a, n, v)
    return a


PLAN = [
    (dict(lens_in=None), INVALID), (dict(delta=None), INVALID), (dict(n_free_in=None), INVALID),
    (dict(lens_out=None), INVALID), (dict(n_free_out=None), INVALID), (dict(table=None), INVALID),
    (dict(free_pages=None), INVALID), (dict(status=None), INVALID), (dict(slots=None), INVALID),
    (dict(max_tokens=0), INVALID), (dict(max_tokens=-1), INVALID), (dict(max_tokens=2 ** 31 - 1), RANGE), (dict(n_req=0), RANGE), (dict(n_req=8193), RANGE),
    (dict(page_size=48), UNSUPPORTED), (dict(page_size=4), UNSUPPORTED), (dict(page_size=2048), UNSUPPORTED),
    (dict(n_pages=0), INVALID), (dict(table_width=0), INVALID), (dict(table_stride=31), INVALID),
    (dict(n_pages=1 << 26), RANGE), (dict(reserved=1), INVALID),
    (dict(n_req=8192, table_width=1 << 19, table_stride=1 << 19, page_size=8), RANGE),
]
CACHE = [
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(k=P + 8), INVALID), (dict(v=P + 2), INVALID),
    (dict(dtype=SX_DTYPE_Q8_0), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED), (dict(page_size=24), UNSUPPORTED),
    (dict(n_pages=0), INVALID), (dict(n_kv_heads=0), INVALID), (dict(n_pages=1 << 25), RANGE),
    (dict(token_stride=132), INVALID), (dict(page_stride=-8), INVALID), (dict(token_stride=64), INVALID),
    (dict(reserved=7), INVALID),
]
APPEND = [
    (dict(x=None), INVALID), (dict(slots=None), INVALID), (dict(n_rows=-1), INVALID), (dict(n_heads=-1), INVALID),
    (dict(x_dtype=SX_DTYPE_Q8_0), UNSUPPORTED), (dict(x_dtype=1), UNSUPPORTED), (dict(x_stride=47 * 128), INVALID),
    (dict(x_stride=48 * 128 + 2), INVALID), (dict(q_stride=31 * 128), INVALID), (dict(x=P + 4), INVALID),
    (dict(cos=None), INVALID), (dict(sin=None), INVALID), (dict(positions=None), INVALID), (dict(n_positions=0), INVALID),
    (dict(cos=P + 4), INVALID), (dict(q_norm=P + 8), INVALID), (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID),
    (dict(n_heads=1 << 21), RANGE),
]
ATTENTION = [
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(table=None), INVALID), (dict(lens=None), INVALID),
    (dict(workspace_bytes=0), RANGE), (dict(workspace=P + 4), INVALID),
    (dict(n_req=-1), INVALID), (dict(q_dtype=1), UNSUPPORTED), (dict(n_heads=0), UNSUPPORTED),
    (dict(n_heads=33), UNSUPPORTED), (dict(n_heads=1 << 17), RANGE), (dict(table_width=0), INVALID),
    (dict(table_stride=15), INVALID), (dict(max_len=-1), INVALID), (dict(q_stride=31 * 128), INVALID),
    (dict(out_stride=32 * 128 + 4), INVALID), (dict(q=P + 8), INVALID), (dict(table_width=1 << 26, table_stride=1 << 26), RANGE),
    (dict(n_req=1 << 29), RANGE), (dict(n_req=1 << 20, table_width=1 << 15, table_stride=1 << 15), RANGE),
]


@pytest.mark.parametrize("kw,code", PLAN, ids=lambda v: str(v)[:48])
def test_plan_refuses(kw, code):
    rc, msg = call("sx_paged_plan", plan_args(**kw))
    assert rc == code and "sx_paged_plan" in msg


@pytest.mark.parametrize("kw,code", CACHE, ids=lambda v: str(v)[:48])
def test_cache_descriptions_refused(kw, code):
    for fn, args in (("sx_paged_append", append_args(c=kw)), ("sx_paged_attention", attention_args(c=kw))):
        rc, msg = call(fn, args)
        assert rc == code and fn in msg


@pytest.mark.parametrize("kw,code", APPEND, ids=lambda v: str(v)[:48])
def test_append_refuses(kw, code):
    rc, msg = call("sx_paged_append", append_args(**kw))
    assert rc == code and "sx_paged_append" in msg


@pytest.mark.parametrize("kw,code", ATTENTION, ids=lambda v: str(v)[:48])
def test_attention_refuses(kw, code):
    rc, msg = call("sx_paged_attention", attention_args(**kw))
    assert rc == code and "sx_paged_attention" in msg


def test_null_arguments_and_devices():
    L = _lib.lib()
    for fn in ("sx_paged_plan", "sx_paged_append", "sx_paged_attention"):
        assert getattr(L, fn)(None, 0, None) == INVALID
    b = C.c_size_t()
    assert L.sx_paged_attention_workspace(32, 8, 128, 0, None) == INVALID
    assert L.sx_paged_attention_workspace(32, 7, 128, 0, C.byref(b)) == UNSUPPORTED
    assert L.sx_paged_attention_workspace(32, 8, 100, 0, C.byref(b)) == UNSUPPORTED
    assert L.sx_paged_attention_workspace(32, 8, 128, -1, C.byref(b)) == INVALID
    # well-formed arguments on a device that is not there
    for fn, args in (("sx_paged_plan", plan_args()), ("sx_paged_append", append_args()),
                     ("sx_paged_attention", attention_args())):
        assert getattr(L, fn)(C.byref(args), 63, None) == INVALID
        assert "no such CUDA device" in L.sx_last_error().decode()


def test_python_layer_refuses_what_is_not_on_a_gpu():
    import torch

    from syrinx_b200 import paged

    i = torch.zeros(4, dtype=torch.int32)
    kv = torch.zeros(2, 8, 16, 64)
    with pytest.raises(ValueError):
        paged.plan(i, i, i.view(4, 1), i, i[:1], page_size=16)
    with pytest.raises(ValueError):
        paged.attend(torch.zeros(4, 8, 64), kv, kv, i.view(4, 1), i)
    with pytest.raises(ValueError):
        paged.append(torch.zeros(4, 24 * 64), kv, kv, i, n_heads=8)
    with pytest.raises(ValueError):
        paged.attend(torch.zeros(4, 8, 64), kv, kv.transpose(1, 2), i.view(4, 1), i)
    with pytest.raises(sx.SyrinxError):
        paged.check(torch.tensor([-7, 0, 0, 0], dtype=torch.int32))
    paged.check(torch.zeros(4, dtype=torch.int32))
