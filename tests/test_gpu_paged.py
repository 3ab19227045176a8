"""The paged key/value operators (include/syrinx_paged.h) on a B200 against float64.

Tolerances. u = 2^-24 is half a step of f32. A sum of n terms in any order, with roundings that
do not conspire, is off by at most 8 sqrt(n) u times the sum of the terms' sizes. For the
attention: a score s = scale * q.k is off by ds = (8 sqrt(hd) + 4) u scale sum|q k|, a weight by
the factor 1 + ds + 4u, and o = sum p v / sum p by both errors of the quotient, so by at most
2 (ds + 4u + (8 sqrt(len) + 8) u) sum p|v| / sum p. 16-bit pages pass the weights to the tensor
cores in pieces that keep 2^-17 (bf16) or 2^-22 (f16) of them at least; a 16-bit result is rounded once, by at
most eps / 2 of its value (2^-25 at the bottom of f16's range).
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def paged():
    from syrinx_b200 import paged as m
    return m


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def pages_of(length, ps):
    return -(-length // ps)


def empty_cache(n_pages, hkv, ps, hd, dtype, layout, fill=float("nan")):
    shape = (n_pages, hkv, ps, hd) if layout == "hnd" else (n_pages, ps, hkv, hd)
    return torch.full(shape, fill, dtype=dtype, device="cuda")


def rows_of(cache, ids, length, ps, layout):
    """[length, kv heads, hd] of one request's pages."""
    r = cache[ids.long()]
    if layout == "hnd":
        r = r.permute(0, 2, 1, 3)
    return r.reshape(-1, r.shape[2], r.shape[3])[:length]


def filled(lens, hkv, ps, hd, dtype, layout, seed, k_gain=1.0, spare=2):
    """Caches that hold the requests' rows on shuffled pages and NaN everywhere else, and a table
    whose unused entries are not page ids."""
    g = gen(seed)
    need = [pages_of(x, ps) for x in lens]
    n_pages = sum(need) + spare
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    k, v = (empty_cache(n_pages, hkv, ps, hd, dtype, layout) for _ in range(2))
    table = torch.full((len(lens), max(need + [1]) + 2), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    at = 0
    for i, x in enumerate(lens):
        mine = ids[at:at + need[i]]
        at += need[i]
        table[i, :need[i]] = mine
        for c, gain in ((k, k_gain), (v, 1.0)):
            rows = (gain * torch.randn((x, hkv, hd), generator=g, device="cuda")).to(dtype)
            put_rows(c, mine, rows, ps, layout)
    return k, v, table


def put_rows(cache, ids, rows, ps, layout, first=0):
    p = torch.arange(first, first + rows.shape[0], device="cuda")
    page, off = ids.long()[p // ps], p % ps
    if layout == "hnd":
        cache[page, :, off] = rows
    else:
        cache[page, off] = rows


def ref_attend(q, k, v, table, lens, scale, ps, layout):
    """(out, lse, bound of |out - its f32 computation|, bound of lse) in float64."""
    n, H, hd = q.shape
    out = torch.zeros(n, H, hd, dtype=torch.float64, device="cuda")
    lse = torch.full((n, H), -math.inf, dtype=torch.float64, device="cuda")
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for i, x in enumerate(lens):
        if x == 0:
            continue
        ids = table[i, :pages_of(x, ps)]
        K, V = (rows_of(c, ids, x, ps, layout).double() for c in (k, v))
        G = H // K.shape[1]
        K, V = K.repeat_interleave(G, 1), V.repeat_interleave(G, 1)
        Q = q[i].double()
        s = scale * torch.einsum("hd,thd->ht", Q, K)
        ds = abs(scale) * (8 * math.sqrt(hd) + 4) * U * torch.einsum("hd,thd->ht", Q.abs(), K.abs()).amax(1)
        lse[i] = torch.logsumexp(s, 1)
        w = torch.softmax(s, 1)
        out[i] = torch.einsum("ht,thd->hd", w, V)
        size = torch.einsum("ht,thd->hd", w, V.abs())
        some = (8 * math.sqrt(x) + 12) * U
        low = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -17, torch.float16: 2.0 ** -22}[k.dtype]
        if q.dtype == torch.float32:
            low = min(low, 2 * U)
        tol[i] = 2 * (ds[:, None] + some + low) * size
        ltol[i] = ds + some + 4 * U * (1 + lse[i].abs())
    if q.dtype != torch.float32:
        tol = tol + out.abs() * torch.finfo(q.dtype).eps / 2 + 2.0 ** -25
    return out, lse, tol, ltol


def assert_attends(paged, q, k, v, table, lens, ps, layout, scale=None, **kw):
    n, H, hd = q.shape
    sc = hd ** -0.5 if scale is None else scale
    out = kw.pop("out", torch.full_like(q, float("nan")))
    lse = torch.full((n, H), float("nan"), device="cuda")
    d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.attend(q, k, v, table, d, scale=scale, layout=layout, out=out, lse=lse, status=status, **kw)
    want, wl, tol, ltol = ref_attend(q, k, v, table, lens, sc, ps, layout)
    assert int(status) == 0
    assert torch.isfinite(out).all()
    err = (out.double() - want).abs()
    assert (err <= tol).all(), f"out: {float((err - tol).max())} over, worst error {float(err.max())}"
    empty = torch.isinf(wl)
    assert torch.equal(torch.isinf(lse), empty) and (out[empty] == 0).all()
    le = (lse.double() - wl)[~empty].abs()
    assert (le <= ltol[~empty]).all(), f"lse: {float((le - ltol[~empty]).max())} over"
    return out, lse


TYPES = [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")]
HEADS = [(2, 2, 64), (14, 2, 64), (32, 8, 128), (8, 1, 128), (16, 1, 128), (4, 2, 256), (8, 1, 256), (9, 3, 32), (5, 1, 32),
         (16, 1, 64), (16, 1, 32), (11, 1, 128)]


# ---- attend -------------------------------------------------------------------------------

@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("H,hkv,hd", HEADS)
def test_attend_short_and_odd_lengths(paged, qt, ct, H, hkv, hd):
    lens = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 0, 127, 130, 257, 0]
    for ps, layout in ((16, "hnd"), (64, "nhd")):
        k, v, table = filled(lens, hkv, ps, hd, DT[ct], layout, 7 + ps)
        q = torch.randn((len(lens), H, hd), generator=gen(3), device="cuda").to(DT[qt])
        assert_attends(paged, q, k, v, table, lens, ps, layout)


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("H,hkv,hd", [(17, 1, 64), (71, 1, 64), (66, 2, 128), (9, 1, 256), (40, 2, 256), (24, 1, 32), (128, 1, 128)])
def test_attend_wide_groups_are_run_in_parts(paged, qt, ct, H, hkv, hd):
    lens = [0, 1, 40, 333, 2500]
    k, v, table = filled(lens, hkv, 16, hd, DT[ct], "nhd", 3)
    q = torch.randn((len(lens), H, hd), generator=gen(3), device="cuda").to(DT[qt])
    assert_attends(paged, q, k, v, table, lens, 16, "nhd")
    assert_attends(paged, q[:3], k, v, table, lens[:3], 16, "nhd", max_len=40)


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("n,H,hkv,hd,ps", [(1, 32, 8, 128, 64), (1, 8, 1, 64, 8), (3, 14, 2, 64, 16), (2, 4, 4, 256, 128),
                                            (5, 16, 1, 128, 32), (1, 2, 1, 32, 1024)])
def test_attend_long_lengths_are_split_and_joined(paged, qt, ct, n, H, hkv, hd, ps):
    lens = [20011, 1, 4097, 0, 9999][:n]
    k, v, table = filled(lens, hkv, ps, hd, DT[ct], "hnd", 11)
    q = 2 * torch.randn((n, H, hd), generator=gen(5), device="cuda")
    assert_attends(paged, q.to(DT[qt]), k, v, table, lens, ps, "hnd")


@pytest.mark.parametrize("ps", [8, 16, 32, 64, 128, 256, 512, 1024])
@pytest.mark.parametrize("qt,ct,hd", [("f32", "f32", 128), ("bf16", "bf16", 32), ("f32", "f16", 64), ("f16", "f16", 256)])
def test_attend_page_sizes(paged, qt, ct, hd, ps):
    lens = [ps - 1, ps, ps + 1, 3 * ps + 5, 1]
    for layout in ("hnd", "nhd"):
        k, v, table = filled(lens, 2, ps, hd, DT[ct], layout, ps)
        q = torch.randn((len(lens), 4, hd), generator=gen(ps), device="cuda").to(DT[qt])
        assert_attends(paged, q, k, v, table, lens, ps, layout)


@pytest.mark.parametrize("qt,ct", TYPES)
def test_attend_many_uneven_requests(paged, qt, ct):
    r = np.random.default_rng(0)
    lens = [int(x) for x in np.exp(r.uniform(0, 7.5, 300))]
    lens[5] = lens[77] = lens[299] = 0
    k, v, table = filled(lens, 2, 16, 64, DT[ct], "nhd", 1)
    q = torch.randn((300, 6, 64), generator=gen(2), device="cuda").to(DT[qt])
    assert_attends(paged, q, k, v, table, lens, 16, "nhd")


@pytest.mark.parametrize("n", [32, 33, 127, 128, 129, 512, 513, 1025])
@pytest.mark.parametrize("qt,ct,hd", [("f32", "f32", 64), ("bf16", "bf16", 128)])
def test_attend_request_counts(paged, qt, ct, hd, n):
    """Either side of the counts at which the requests are summed up in another way."""
    lens = [(37 * i * i + 11 * i) % 290 if i % 7 else 0 for i in range(n)]
    lens[n // 2] = 3000
    k, v, table = filled(lens, 2, 16, hd, DT[ct], "hnd", n)
    q = torch.randn((n, 4, hd), generator=gen(n), device="cuda").to(DT[qt])
    assert_attends(paged, q, k, v, table, lens, 16, "hnd")


def test_attend_on_two_streams_at_once(paged):
    """Eager calls on two streams take a workspace each from the allocator."""
    lens = [5000, 300, 2000]
    k, v, table = filled(lens, 2, 16, 128, torch.bfloat16, "hnd", 5)
    d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    qs = [torch.randn((3, 8, 128), generator=gen(s), device="cuda").bfloat16() for s in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(30):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                outs[s].append(paged.attend(qs[s], k, v, table, d))
    torch.cuda.synchronize()
    for s in range(2):
        want, _, tol, _ = ref_attend(qs[s], k, v, table, lens, 128 ** -0.5, 16, "hnd")
        assert ((outs[s][0].double() - want).abs() <= tol).all()
        assert all(torch.equal(o, outs[s][0]) for o in outs[s])


def test_attend_thousands_of_requests(paged):
    lens = [(7 * i) % 5 for i in range(5000)]
    k, v, table = filled([0] * 5000, 1, 8, 32, torch.float32, "hnd", 1)
    k, v = (torch.randn((64, 1, 8, 32), generator=gen(s), device="cuda") for s in (1, 2))
    table[:, 0] = torch.arange(5000, device="cuda") % 64  # pages may be shared: they are only read
    q = torch.randn((5000, 1, 32), generator=gen(3), device="cuda")
    assert_attends(paged, q, k, v, table, lens, 8, "hnd")


@pytest.mark.parametrize("scale", [0.0, -0.3, 8.0, 1e-3])
@pytest.mark.parametrize("qt,ct", TYPES)
def test_attend_scales(paged, qt, ct, scale):
    lens = [1, 40, 700, 0]
    k, v, table = filled(lens, 2, 16, 64, DT[ct], "hnd", 4)
    q = torch.randn((4, 8, 64), generator=gen(5), device="cuda").to(DT[qt])
    assert_attends(paged, q, k, v, table, lens, 16, "hnd", scale=scale)


@pytest.mark.parametrize("qt,ct,size", [("f32", "f32", 1e15), ("f32", "bf16", 1e15), ("f32", "f16", 1e15), ("f32", "f16", 1e-15),
                                        ("f32", "bf16", 1e-15), ("f16", "f16", 1e3)])
def test_attend_large_and_small_queries(paged, qt, ct, size):
    """The queries' size comes off again in the scale, so nothing but their range differs."""
    lens = [300, 17, 1]
    k, v, table = filled(lens, 2, 16, 128, DT[ct], "hnd", 6)
    q = (size * torch.randn((3, 8, 128), generator=gen(7), device="cuda")).to(DT[qt])
    q[1, 3] = 0
    assert_attends(paged, q, k, v, table, lens, 16, "hnd", scale=0.1 / size)


@pytest.mark.parametrize("qt,ct", TYPES)
def test_attend_rows_whose_scores_are_all_minus_infinity(paged, qt, ct):
    """Keys of -inf against positive queries leave nothing: zeros and -inf, as for no key at all;
    single such keys are left out."""
    lens = [40, 40, 900]
    k, v, table = filled(lens, 1, 16, 64, DT[ct], "hnd", 8)
    q = (0.5 + torch.rand((3, 4, 64), generator=gen(9), device="cuda")).to(DT[qt])
    for i, spots in ((0, range(40)), (1, (0, 17, 39)), (2, range(0, 900, 2))):
        for t in spots:
            k[table[i, t // 16].long(), 0, t % 16, 5] = -math.inf
    out, lse = torch.empty_like(q), torch.empty(3, 4, device="cuda")
    d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    paged.attend(q, k, v, table, d, out=out, lse=lse)
    assert (out[0] == 0).all() and (lse[0] == -math.inf).all()
    for i, keep in ((1, [t for t in range(40) if t not in (0, 17, 39)]), (2, list(range(1, 900, 2)))):
        K, V = (rows_of(c, table[i, :pages_of(lens[i], 16)], lens[i], 16, "hnd")[keep, 0].double() for c in (k, v))
        s = q[i].double() @ K.T / 8
        want = torch.softmax(s, 1) @ V
        eps = torch.finfo(q.dtype).eps if qt != "f32" else 0
        # sum |q k| / 8 <= 1.5 * 64 * 4.5 / 8 = 54, so ds <= 68 * 54 u = 2.2e-4 and |out| <= 4.5
        assert (out[i].double() - want).abs().max() <= 2 * (2.2e-4 + 2 ** -16) * 4.5 + eps / 2 * 4.5


@pytest.mark.parametrize("qt,ct", TYPES)
def test_attend_infinite_and_nan_values_stay_in_their_element(paged, qt, ct):
    """An infinite value under an ordinary weight makes its own output element infinite, a NaN one
    NaN, and no other; a NaN key makes its head group's outputs NaN and no other request's."""
    lens = [20, 20, 300]
    k, v, table = filled(lens, 2, 16, 64, DT[ct], "hnd", 21)
    q = (0.1 * torch.randn((3, 4, 64), generator=gen(22), device="cuda")).to(DT[qt])
    clean = paged.attend(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    v[table[0, 0].long(), 0, 3, 9] = math.inf
    v[table[0, 1].long(), 0, 1, 10] = -math.inf
    v[table[0, 0].long(), 1, 5, 11] = math.nan
    k[table[1, 0].long(), 1, 7, 0] = math.nan
    out = paged.attend(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert (out[0, :2, 9] == math.inf).all() and (out[0, :2, 10] == -math.inf).all() and out[0, 2:, 11].isnan().all()
    assert out[1, 2:].isnan().all()
    out[0, :2, 9:11], out[0, 2:, 11], out[1, 2:] = clean[0, :2, 9:11], clean[0, 2:, 11], clean[1, 2:]
    assert torch.equal(out, clean)


def test_attend_strided_rows_and_neighbours_left_alone(paged):
    """Queries inside fused rows, results into a wider buffer, k and v halves of one tensor."""
    lens = [33, 0, 200]
    kv = torch.full((9 + 14, 2, 2, 16, 128), float("nan"), device="cuda")
    k0, v0, table = filled(lens, 2, 16, 128, torch.float32, "hnd", 10, spare=23 - 3 - 13)
    kv[:, 0], kv[:, 1] = k0, v0
    fused = torch.randn((3, 12 * 128), generator=gen(1), device="cuda")
    q = fused.view(3, 12, 128)[:, :8]
    wide = torch.full((3, 10, 128), 5.0, device="cuda")
    big = torch.cat((table, torch.full((3, 7), -9, dtype=torch.int32, device="cuda")), 1)
    assert_attends(paged, q, kv[:, 0], kv[:, 1], big[:, : table.shape[1]], lens, 16, "hnd", out=wide[:, 1:9])
    assert (wide[:, 0] == 5).all() and (wide[:, 9] == 5).all()


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("lens,H,hkv", [([1, 0, 60, 130], 8, 2), ([9000], 8, 2), ([700, 0, 1, 3000, 33] * 30, 8, 2),
                                        ([400] * 9, 40, 1)])
def test_attend_over_its_own_queries(paged, qt, ct, lens, H, hkv):
    """out may be q: in one CTA per request, split and joined, and with several groups a kv head."""
    k, v, table = filled(lens, hkv, 32, 64, DT[ct], "hnd", 41)
    q = torch.randn((len(lens), H, 64), generator=gen(42), device="cuda").to(DT[qt])
    d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = paged.attend(q, k, v, table, d)
    got = q.clone()
    assert paged.attend(got, k, v, table, d, out=got) is got
    assert torch.equal(got, want)


@pytest.mark.parametrize("requests", [2, 40])
def test_first_calls_of_a_process_can_be_captured(requests):
    """Nothing of a call has to have run before it is captured: a new process captures its first plan,
    append (of few and of many rows) and attention, and the replay equals calls made afterwards."""
    import os
    import subprocess
    import sys

    code = f"""
import torch
from syrinx_b200 import paged
n, H, hkv, hd, ps, width = {requests}, 32, 8, 128, 16, 40
g0 = torch.Generator(device="cuda"); g0.manual_seed(3)
k = torch.randn(n * width + 200, hkv, ps, hd, generator=g0, device="cuda").bfloat16()
v = torch.randn(k.shape, generator=g0, device="cuda").bfloat16()
lens = torch.arange(1, n + 1, dtype=torch.int32, device="cuda") % 20 * ps  # every request needs a page
table = torch.arange(n * width, dtype=torch.int32, device="cuda").view(n, width).contiguous()
free = torch.arange(k.shape[0], dtype=torch.int32, device="cuda").roll(200)  # the spare pages lie lowest
left = torch.full((1,), n, dtype=torch.int32, device="cuda")
delta, slots = torch.ones_like(lens), torch.empty_like(lens)
x = torch.randn((n, (H + 2 * hkv) * hd), generator=g0, device="cuda").bfloat16()
spare = torch.arange((n * width + 100) * ps, (n * width + 200) * ps, dtype=torch.int32, device="cuda")
many = torch.randn((spare.numel(), (H + 2 * hkv) * hd), generator=g0, device="cuda").bfloat16()
work = torch.empty(paged.workspace_bytes(H, hkv, hd), dtype=torch.uint8, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    status = paged.plan(lens, delta, table, free, left, page_size=ps, slots=slots)
    q = paged.append(x, k, v, slots, n_heads=H)
    q2 = paged.append(many, k, v, spare, n_heads=H)
    out = paged.attend(q.view(n, H, hd), k, v, table, lens, workspace=work)
graph.replay()
torch.cuda.synchronize()
assert status.tolist() == [0, n, n, 0], status.tolist()
assert torch.equal(q, x[:, : H * hd])
assert torch.equal(q2, many[:, : H * hd])
assert torch.equal(out, paged.attend(q.view(n, H, hd), k, v, table, lens))
print("same")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), r.stderr[-2000:]


@pytest.mark.parametrize("ct", ["bf16", "f32"])
def test_attend_offsets_past_32_bits(paged, ct):
    """Pages whose elements lie beyond 2^31 (and bytes beyond 2^32) from the base."""
    ps, hkv, hd = 64, 8, 128
    n_pages = (1 << 31) // (ps * hkv * hd) + 40
    k = torch.empty((n_pages, hkv, ps, hd), dtype=DT[ct], device="cuda")
    v = torch.empty_like(k)
    lens = [150, 64]
    table = torch.tensor([[n_pages - 1, 3, n_pages - 9], [n_pages - 30, 0, 0]], dtype=torch.int32, device="cuda")
    for p in table.flatten().tolist():
        for c, s in ((k, p), (v, p + 1)):
            c[p] = torch.randn((hkv, ps, hd), generator=gen(s), device="cuda").to(DT[ct])
    q = torch.randn((2, 32, hd), generator=gen(4), device="cuda")
    assert_attends(paged, q, k, v, table, lens, ps, "hnd")


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("max_len", [0, 1, 100, 5000])
def test_attend_the_hint_never_changes_the_meaning(paged, qt, ct, max_len):
    lens = [5000, 3, 0, 77]
    k, v, table = filled(lens, 2, 16, 128, DT[ct], "hnd", 12)
    q = torch.randn((4, 8, 128), generator=gen(13), device="cuda").to(DT[qt])
    assert_attends(paged, q, k, v, table, lens, 16, "hnd", max_len=max_len)


@pytest.mark.parametrize("qt,ct", TYPES)
def test_attend_repeats_and_does_not_mix_requests(paged, qt, ct):
    lens = [3000, 1, 500, 0, 64, 1200]
    k, v, table = filled(lens, 2, 16, 64, DT[ct], "hnd", 14)
    q = torch.randn((6, 8, 64), generator=gen(15), device="cuda").to(DT[qt])
    a, la = assert_attends(paged, q, k, v, table, lens, 16, "hnd")
    b, lb = assert_attends(paged, q, k, v, table, lens, 16, "hnd")
    assert torch.equal(a, b) and torch.equal(la, lb)
    q2 = q.clone()
    q2[2] += 1
    k2 = k.clone()
    k2[table[2, 0].long()] = 3
    c, _ = assert_attends(paged, q2, k2, v, table, lens, 16, "hnd")
    keep = [0, 1, 3, 4, 5]
    assert torch.equal(a[keep], c[keep]) and not torch.equal(a[2], c[2])


def test_attend_reports_bad_pages_and_lengths(paged):
    lens = [100, 40]
    k, v, table = filled(lens, 2, 16, 64, torch.float32, "hnd", 16)
    q = torch.randn((2, 4, 64), generator=gen(17), device="cuda")
    d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for bad in (-1, k.shape[0], 2 ** 31 - 1):
        t, status = table.clone(), torch.zeros(1, dtype=torch.int32, device="cuda")
        t[0, 2] = bad
        out = paged.attend(q, k, v, t, d, status=status)
        assert int(status) == -7
        want, _, tol, _ = ref_attend(q[1:], k, v, table[1:], lens[1:], 0.125, 16, "hnd")
        assert ((out[1:].double() - want).abs() <= tol).all()
    width = pages_of(100, 16)
    for n0 in (width * 16 + 1, 2 ** 31 - 1):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        long = torch.tensor([n0, 40], dtype=torch.int32, device="cuda")
        k1, v1, t1 = filled([width * 16, 40], 2, 16, 64, torch.float32, "hnd", 16)
        t1 = t1[:, :width].contiguous()
        out = paged.attend(q, k1, v1, t1, long, status=status)
        assert int(status) == -7
        want, _, tol, _ = ref_attend(q, k1, v1, t1, [width * 16, 40], 0.125, 16, "hnd")
        assert ((out.double() - want).abs() <= tol).all()
    neg = torch.tensor([-5, 40], dtype=torch.int32, device="cuda")
    assert (paged.attend(q, k, v, table, neg)[0] == 0).all()


@pytest.mark.parametrize("qt,ct", TYPES)
def test_attend_without_a_workspace(paged, qt, ct):
    """The library call with a null workspace: nothing is split, whatever the lengths are."""
    import ctypes as C

    from syrinx_b200 import _lib
    from syrinx_b200.configs import SxPagedAttentionArgs

    lens = [5000, 0, 17, 900]
    k, v, table = filled(lens, 2, 16, 64, DT[ct], "hnd", 31)
    q = torch.randn((4, 8, 64), generator=gen(32), device="cuda").to(DT[qt])
    out, d = torch.full_like(q, float("nan")), torch.tensor(lens, dtype=torch.int32, device="cuda")
    a = SxPagedAttentionArgs()
    c = a.cache
    c.k, c.v, c.page_stride, c.head_stride, c.token_stride = k.data_ptr(), v.data_ptr(), *k.stride()[:3]
    kinds = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
    c.dtype, c.n_pages, c.page_size, c.n_kv_heads, c.head_dim = kinds[k.dtype], k.shape[0], 16, 2, 64
    a.q, a.out, a.table, a.lens = q.data_ptr(), out.data_ptr(), table.data_ptr(), d.data_ptr()
    a.q_stride = a.out_stride = 8 * 64
    a.table_stride = a.table_width = table.shape[1]
    a.n_req, a.n_heads, a.q_dtype, a.scale = 4, 8, kinds[q.dtype], 0.125
    _lib.check(_lib.lib().sx_paged_attention(C.byref(a), 0, torch.cuda.current_stream().cuda_stream))
    want, _, tol, _ = ref_attend(q, k, v, table, lens, 0.125, 16, "hnd")
    assert ((out.double() - want).abs() <= tol).all()


def test_attend_refusals(paged):
    import syrinx_b200 as sx

    k, v, table = filled([40], 2, 16, 64, torch.float32, "hnd", 16)
    q = torch.randn((1, 4, 64), device="cuda")
    d = torch.tensor([40], dtype=torch.int32, device="cuda")
    for bad in (lambda: paged.attend(q[:, :, :32], k, v, table, d), lambda: paged.attend(q.cpu(), k, v, table, d),
                lambda: paged.attend(q, k, v[:1], table, d), lambda: paged.attend(q, k, v, table.long(), d),
                lambda: paged.attend(q, k, v, table, d.long()), lambda: paged.attend(q, k, v, table, d, layout="dhn"),
                lambda: paged.attend(q, k, v, table, d[:0]), lambda: paged.attend(q.double(), k, v, table, d),
                lambda: paged.attend(q, k, v, table, d, lse=torch.empty(3, device="cuda")),
                lambda: paged.attend(q.transpose(1, 2).contiguous().transpose(1, 2), k, v, table, d),
                lambda: paged.attend(q, k, v, table, d, out=torch.empty(1, 4, 32, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: paged.attend(q[:, :3], k, v, table, d), lambda: paged.attend(q.half(), k, v, table, d),
                lambda: paged.attend(q, k, v, table, d, workspace=torch.empty(8, device="cuda"))):
        with pytest.raises(sx.SyrinxError):
            bad()
    assert paged.attend(q[:0], k, v, table, d).shape == (0, 4, 64)


def test_attend_on_another_stream_and_in_two_graphs_at_once(paged):
    """Two captured calls, each with a workspace of its own, replayed on two streams at once; the
    lengths are read when the graph runs."""
    n, H, hkv, hd, ps = 3, 8, 2, 128, 16
    full = [4000, 700, 2500]
    k, v, table = filled(full, hkv, ps, hd, torch.bfloat16, "hnd", 18)
    work = []
    for s in range(2):
        q = torch.randn((n, H, hd), generator=gen(30 + s), device="cuda").bfloat16()
        lens = torch.tensor(full, dtype=torch.int32, device="cuda")
        out = torch.zeros_like(q)
        ws = torch.empty(paged.workspace_bytes(H, hkv, hd), dtype=torch.uint8, device="cuda")
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            paged.attend(q, k, v, table, lens, out=out, workspace=ws)
        st.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            paged.attend(q, k, v, table, lens, out=out, workspace=ws)
        work.append((q, lens, out, st, graph))
    for now in (full, [1, 0, 2500], [3999, 64, 1]):
        for _, lens, out, st, _ in work:
            with torch.cuda.stream(st):
                lens.copy_(torch.tensor(now, dtype=torch.int32))
                out.fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(20):
            for _, _, _, st, graph in work:
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for q, _, out, _, _ in work:
            want, _, tol, _ = ref_attend(q, k, v, table, now, hd ** -0.5, ps, "hnd")
            assert ((out.double() - want).abs() <= tol).all()


# ---- append -------------------------------------------------------------------------------

def ref_append(x, H, hkv, hd, pos, cos, sin, il, qn, kn, eps):
    """Rows [T, heads, hd] in float64 and the bound of their f32 computation."""
    T = x.shape[0]
    y = x.double().view(T, H + 2 * hkv, hd).clone()
    tol = torch.zeros_like(y)
    for part, gain in ((slice(0, H), qn), (slice(H, H + hkv), kn)):
        if gain is not None:
            z = y[:, part]
            y[:, part] = z / torch.sqrt((z * z).mean(-1, keepdim=True) + eps) * gain.double()
            # the mean is off by 8 sqrt(hd) u, its root by half of that; root, quotient, product: 4 u
            tol[:, part] = y[:, part].abs() * (4 * math.sqrt(hd) + 4) * U
    if cos is not None:
        c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
        rot = slice(0, H + hkv)
        z, t = y[:, rot], tol[:, rot]
        pairs = ((slice(0, None, 2), slice(1, None, 2)) if il else (slice(0, hd // 2), slice(hd // 2, None)))
        a, b = z[..., pairs[0]].clone(), z[..., pairs[1]].clone()
        ta, tb = t[..., pairs[0]].clone(), t[..., pairs[1]].clone()
        z[..., pairs[0]], z[..., pairs[1]] = a * c - b * s, b * c + a * s
        more = ta * 1.01 + tb * 1.01 + 2 * U * (a.abs() + b.abs())
        t[..., pairs[0]], t[..., pairs[1]] = more, more
    return y, tol


def rope(n_pos, hd):
    inv = 1.0 / (1e6 ** (torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd))
    ang = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def rounding(dtype, y):
    return 0 if dtype == torch.float32 else y.abs() * torch.finfo(dtype).eps / 2 + 2.0 ** -25


def assert_appends(paged, T, pad, H, hkv, hd, ps, xt, ct, layout, norm, rot, il, seed, strided=False):
    g = gen(seed)
    width = (H + 2 * hkv) * hd
    x = torch.randn((T + pad, width + (64 if strided else 0)), generator=g, device="cuda").to(DT[xt])[:, :width]
    n_pages = pages_of(T, ps) + 3
    slots = torch.randperm(n_pages * ps, generator=g, device="cuda")[: T + pad].to(torch.int32)
    if pad:
        slots[T:] = -1
        x[T:] = float("nan")
    if T > 4:
        slots[2] = -1
    cos, sin = rope(700, hd) if rot else (None, None)
    pos = torch.randint(0, 700, (T + pad,), generator=g, device="cuda").to(torch.int32)
    pos[T:] = -1
    qn, kn = ((0.5 + torch.rand(hd, generator=g, device="cuda")) if w else None for w in norm)
    k, v = (empty_cache(n_pages, hkv, ps, hd, DT[ct], layout, 7.0) for _ in range(2))
    wide = torch.full((T + pad, H * hd + (64 if strided else 0)), 3.0, dtype=DT[xt], device="cuda")
    out = wide[:, : H * hd]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.append(x, k, v, slots, n_heads=H, positions=pos if rot else None, cos=cos, sin=sin, interleaved=il,
                 q_norm=qn, k_norm=kn, eps=1e-6, layout=layout, out=out, status=status)
    assert int(status) == 0
    live = (slots >= 0)
    y, tol = ref_append(x[live], H, hkv, hd, pos[live], cos, sin, il, qn, kn, 1e-6)
    assert (wide[:, H * hd:] == 3).all() and (out[~live] == 3).all()
    got = out[live].double().view(y.shape[0], H, hd)
    assert ((got - y[:, :H]).abs() <= tol[:, :H] + rounding(DT[xt], y[:, :H])).all()
    s = slots[live].long()
    for c, part in ((k, slice(H, H + hkv)), (v, slice(H + hkv, None))):
        rows = c[s // ps, :, s % ps] if layout == "hnd" else c[s // ps, s % ps]
        assert ((rows.double() - y[:, part]).abs() <= tol[:, part] + rounding(DT[ct], y[:, part])).all()
        flat = (c.permute(0, 2, 1, 3) if layout == "hnd" else c).reshape(-1, hkv, hd)
        rest = torch.ones(flat.shape[0], dtype=torch.bool, device="cuda")
        rest[s] = False
        assert (flat[rest] == 7).all()


@pytest.mark.parametrize("xt,ct", TYPES)
@pytest.mark.parametrize("H,hkv,hd", [(14, 2, 64), (32, 8, 128), (3, 1, 256), (5, 5, 32), (1, 1, 64)])
@pytest.mark.parametrize("norm,rot,il", [((1, 1), 1, 1), ((1, 1), 1, 0), ((0, 0), 1, 0), ((0, 1), 0, 0), ((1, 0), 1, 1),
                                         ((0, 0), 0, 1)])
def test_append(paged, xt, ct, H, hkv, hd, norm, rot, il):
    assert_appends(paged, 37, 3, H, hkv, hd, 16, xt, ct, "hnd", norm, rot, bool(il), 1)
    assert_appends(paged, 1, 0, H, hkv, hd, 64, xt, ct, "nhd", norm, rot, bool(il), 2, strided=True)


@pytest.mark.parametrize("xt,ct", TYPES)
def test_append_many_rows(paged, xt, ct):
    assert_appends(paged, 3001, 5, 16, 8, 64, 32, xt, ct, "nhd", (1, 1), 1, False, 3, strided=True)


@pytest.mark.parametrize("xt,ct", TYPES)
@pytest.mark.parametrize("H,hkv,hd", [(70, 5, 32), (40, 3, 64), (21, 5, 128), (9, 2, 256)])
@pytest.mark.parametrize("norm,rot,il", [((1, 1), 1, 1), ((1, 1), 1, 0), ((0, 1), 0, 0), ((1, 0), 1, 0), ((0, 0), 0, 1)])
def test_append_many_wide_rows(paged, xt, ct, H, hkv, hd, norm, rot, il):
    """Heads that do not fill the last step or unit of their kind, over many rows."""
    assert_appends(paged, 3000, 2, H, hkv, hd, 16, xt, ct, "nhd" if il else "hnd", norm, rot, bool(il), 5, strided=True)


@pytest.mark.parametrize("xt,ct", [("f32", "bf16"), ("bf16", "bf16")])
def test_append_many_rows_with_bad_ones(paged, xt, ct):
    """Rows without a slot, and with a slot or a position that is none."""
    H, hkv, hd, T = 6, 20, 128, 2000
    x = torch.randn((T, (H + 2 * hkv) * hd), generator=gen(3), device="cuda").to(DT[xt])
    k, v = (empty_cache(pages_of(T, 16), hkv, 16, hd, DT[ct], "nhd", 7.0) for _ in range(2))
    slots = torch.arange(T, device="cuda", dtype=torch.int32)
    pos = torch.arange(T, device="cuda", dtype=torch.int32) % 50
    slots[5::97], slots[6::97], pos[7::97] = -1, pages_of(T, 16) * 16, 50
    cos, sin = rope(50, hd)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.append(x, k, v, slots, n_heads=H, positions=pos, cos=cos, sin=sin, layout="nhd", status=status)
    assert int(status) == -7
    good = (slots >= 0) & (slots < pages_of(T, 16) * 16) & (pos < 50)
    y, tol = ref_append(x[good], H, hkv, hd, pos[good], cos, sin, True, None, None, 1e-6)
    flat = k.view(-1, hkv, hd)[:T]
    assert ((flat[good].double() - y[:, H:H + hkv]).abs() <= tol[:, H:H + hkv] + rounding(DT[ct], y[:, H:H + hkv])).all()
    assert (flat[~good] == 7).all() and (v.view(-1, hkv, hd)[:T][~good] == 7).all()


@pytest.mark.parametrize("T", [70, 3000])
def test_append_drops_queries(paged, T):
    """The library call with a null q_out: keys and values as with one."""
    import ctypes as C

    from syrinx_b200 import _lib
    from syrinx_b200.configs import SxPagedAppendArgs

    H, hkv, hd = 6, 12, 128
    x = torch.randn((T, (H + 2 * hkv) * hd), generator=gen(3), device="cuda")
    slots = torch.randperm(pages_of(T, 64) * 64, generator=gen(4), device="cuda")[:T].to(torch.int32)
    pos = torch.arange(T, device="cuda", dtype=torch.int32) % 50
    cos, sin = rope(50, hd)
    gain = 0.5 + torch.rand(hd, generator=gen(2), device="cuda")
    k, v, k2, v2 = (empty_cache(pages_of(T, 64), hkv, 64, hd, torch.float32, "hnd", 7.0) for _ in range(4))
    paged.append(x, k, v, slots, n_heads=H, positions=pos, cos=cos, sin=sin, k_norm=gain)
    a = SxPagedAppendArgs()
    c = a.cache
    c.k, c.v, c.page_stride, c.head_stride, c.token_stride = k2.data_ptr(), v2.data_ptr(), *k2.stride()[:3]
    c.dtype, c.n_pages, c.page_size, c.n_kv_heads, c.head_dim = 0, k2.shape[0], 64, hkv, hd
    a.x, a.slots, a.positions, a.cos, a.sin = (t.data_ptr() for t in (x, slots, pos, cos, sin))
    a.k_norm, a.x_stride, a.eps = gain.data_ptr(), x.shape[1], 1e-6
    a.x_dtype, a.n_rows, a.n_heads, a.n_positions, a.interleaved = 0, T, H, 50, 1
    _lib.check(_lib.lib().sx_paged_append(C.byref(a), 0, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(k, k2) and torch.equal(v, v2)


@pytest.mark.parametrize("T", [3, 4000])
@pytest.mark.parametrize("il", [True, False])
def test_append_queries_in_place(paged, T, il):
    """The query part of x may be its own output."""
    H, hkv, hd = 4, 2, 64
    x = torch.randn((T, 8 * 64), generator=gen(1), device="cuda")
    cos, sin = rope(100, hd)
    pos = torch.arange(T, device="cuda", dtype=torch.int32) % 100
    slots = torch.arange(T, device="cuda", dtype=torch.int32)
    k, v, k2, v2 = (empty_cache(pages_of(T, 16), hkv, 16, hd, torch.float32, "hnd", 0.0) for _ in range(4))
    gain = 0.5 + torch.rand(hd, generator=gen(2), device="cuda")
    opts = dict(n_heads=H, positions=pos, cos=cos, sin=sin, interleaved=il, q_norm=gain, k_norm=gain)
    want = paged.append(x.clone(), k, v, slots, **opts)
    y = x.clone()
    paged.append(y, k2, v2, slots, out=y[:, : H * hd], **opts)
    assert torch.equal(y[:, : H * hd], want) and torch.equal(y[:, H * hd:], x[:, H * hd:])
    assert torch.equal(k, k2) and torch.equal(v, v2)


def test_append_without_query_heads(paged):
    assert_appends(paged, 9, 0, 0, 2, 128, 16, "f32", "bf16", "hnd", (0, 1), 1, True, 4)
    assert_appends(paged, 2500, 1, 0, 12, 128, 16, "f32", "bf16", "hnd", (0, 1), 1, True, 4)


def test_append_reports_bad_slots_and_positions(paged):
    cos, sin = rope(50, 64)
    x = torch.randn((4, 8 * 64), device="cuda")
    for slots, pos in (([0, 80, 2, 3], [0, 1, 2, 3]), ([0, -2, 2, 3], [0, 1, 2, 3]), ([0, 1, 2, 3], [0, 50, 2, 3]),
                       ([0, 1, 2, 3], [0, -1, 2, 3])):
        k, v = (torch.full((5, 2, 16, 64), 7.0, device="cuda") for _ in range(2))
        s, p = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in (slots, pos))
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = torch.full((4, 4 * 64), 3.0, device="cuda")
        paged.append(x, k, v, s, n_heads=4, positions=p, cos=cos, sin=sin, out=out, status=status)
        assert int(status) == -7
        assert (out[1] == 3).all() and (out[[0, 2, 3]] != 3).any(1).all()
        assert (k[0, :, 1] == 7).all() and (k[1:] == 7).all() and (v[0, 0, [0, 2, 3]] != 7).any(1).all()


def test_append_offsets_past_32_bits(paged):
    ps, hkv, hd = 64, 8, 128
    n_pages = (1 << 31) // (ps * hkv * hd) + 5
    k, v = (torch.empty((n_pages, hkv, ps, hd), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots = torch.tensor([n_pages * ps - 1, 5, (n_pages - 2) * ps + 7], dtype=torch.int32, device="cuda")
    x = torch.randn((3, 18 * hd), generator=gen(2), device="cuda").bfloat16()
    paged.append(x, k, v, slots, n_heads=2)
    s = slots.long()
    assert torch.equal(k[s // ps, :, s % ps].view(3, -1), x[:, 2 * hd:10 * hd])
    assert torch.equal(v[s // ps, :, s % ps].view(3, -1), x[:, 10 * hd:])


# ---- plan ---------------------------------------------------------------------------------

class Model:
    """The bookkeeping in Python: rows of page ids and a stack of free ones."""

    def __init__(self, n, n_pages, width, ps, seed):
        self.ps, self.width = ps, width
        self.stack = [int(p) for p in np.random.default_rng(seed).permutation(n_pages)]
        self.rows, self.lens, self.n_pages = [[] for _ in range(n)], [0] * n, n_pages

    def step(self, delta, max_tokens):
        new = [max(0, a + d) for a, d in zip(self.lens, delta)]
        need = [pages_of(x, self.ps) for x in new]
        fresh = [max(0, d) for d in delta]
        pushes = [p for r, m in zip(self.rows, need) for p in r[m:]]
        takes = sum(max(0, m - len(r)) for r, m in zip(self.rows, need))
        if takes > len(self.stack) + len(pushes) or sum(fresh) > max_tokens or max(need) > self.width:
            return None
        self.stack += pushes
        tokens = []
        for i, (r, m) in enumerate(zip(self.rows, need)):
            del r[m:]
            while len(r) < m:
                r.append(self.stack.pop())
            for p in range(self.lens[i], self.lens[i] + fresh[i]):
                tokens.append((r[p // self.ps] * self.ps + p % self.ps, i, p))
        self.lens = new
        return tokens, takes


def on_gpu(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Pool:
    """The device's side of Model."""

    def __init__(self, m, max_tokens):
        n = len(m.rows)
        self.m, self.most = m, max_tokens
        self.lens, self.n_free, self.free = on_gpu([0] * n), on_gpu([len(m.stack)]), on_gpu(m.stack)
        self.table = torch.full((n, m.width), -5, dtype=torch.int32, device="cuda")
        self.slots, self.seqs, self.pos = (torch.full((max_tokens + 4,), -77, dtype=torch.int32, device="cuda") for _ in range(3))
        self.starts = torch.zeros(n + 1, dtype=torch.int32, device="cuda")

    def args(self):
        t = slice(0, self.most)
        return dict(page_size=self.m.ps, slots=self.slots[t], tok_seq=self.seqs[t], tok_pos=self.pos[t], starts=self.starts)

    def compare(self, tokens, takes, status):
        m, T = self.m, len(tokens)
        assert status.tolist() == [0, T, takes, len(m.stack)]
        assert self.lens.tolist() == m.lens and int(self.n_free) == len(m.stack)
        assert self.free[: len(m.stack)].tolist() == m.stack
        for got, at in ((self.slots, 0), (self.seqs, 1), (self.pos, 2)):
            assert got[:T].tolist() == [t[at] for t in tokens]
            assert (got[T:self.most] == -1).all() and (got[self.most:] == -77).all()
        table = self.table.tolist()
        assert all(table[i][: len(r)] == r for i, r in enumerate(m.rows))
        fresh = [0] * len(m.rows)
        for _, i, _ in tokens:
            fresh[i] += 1
        assert self.starts.tolist() == [0] + list(np.cumsum(fresh))


@pytest.mark.parametrize("n,ps,n_pages,width,longest,seed", [(1, 16, 40, 40, 600, 0), (8, 64, 60, 24, 1500, 1),
                                                              (300, 16, 2500, 64, 1000, 2), (1500, 8, 9000, 30, 200, 3),
                                                              (8192, 8, 20000, 4, 32, 4)])
def test_plan_through_many_steps(paged, n, ps, n_pages, width, longest, seed):
    """Requests that arrive, grow by one, are cut back and leave, in place, step after step."""
    r = np.random.default_rng(seed)
    m = Model(n, n_pages, width, ps, seed)
    pool = Pool(m, n * 2 + longest)
    done = refused = 0
    for step in range(40 if n < 5000 else 8):
        kind = r.random(n)
        delta = np.where(kind < 0.6, (np.array(m.lens) > 0).astype(int), 0)
        some = kind > 0.97
        delta = np.where(some & (np.array(m.lens) == 0), r.integers(1, longest, n), delta)
        delta = np.where((kind > 0.9) & (kind < 0.95), -r.integers(0, longest, n), delta)
        if step % 7 == 6:
            delta = -np.array(m.lens) * (r.random(n) < 0.5)
        delta = [int(d) for d in delta]
        before = (pool.lens.clone(), pool.n_free.clone(), pool.free.clone(), pool.table.clone())
        got = m.step(delta, pool.most)
        status = paged.plan(pool.lens, on_gpu(delta), pool.table, pool.free, pool.n_free, **pool.args())
        if got is None:
            refused += 1
            assert status.tolist() == [-7, 0, 0, len(m.stack)]
            for a, b in zip(before, (pool.lens, pool.n_free, pool.free, pool.table)):
                assert torch.equal(a, b)
            assert (pool.slots[: pool.most] == -1).all() and (pool.starts == 0).all()
        else:
            done += 1
            pool.compare(*got, status)
    assert done >= 3  # of the model: enough steps that were not refused


def test_plan_out_of_place_repeats(paged):
    m = Model(5, 50, 20, 16, 1)
    pool = Pool(m, 400)
    m.step([100, 0, 37, 16, 1], 400)
    paged.plan(pool.lens, on_gpu([100, 0, 37, 16, 1]), pool.table, pool.free, pool.n_free, **pool.args())
    got = m.step([1, 200, -30, -99, 16], 400)
    lens, n_free = torch.empty_like(pool.lens), torch.empty_like(pool.n_free)
    old, old_free = pool.lens, pool.n_free
    for _ in range(3):
        status = paged.plan(old, on_gpu([1, 200, -30, -99, 16]), pool.table, pool.free, old_free, lens_out=lens,
                            n_free_out=n_free, **pool.args())
        pool.lens, pool.n_free = lens, n_free
        pool.compare(*got, status)


def test_plan_without_tokens_and_pages_to_the_last_one(paged):
    """Every page in use, and not one token array."""
    lens, table = on_gpu([0, 0]), torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    free, n_free = on_gpu([3, 1, 0, 2]), on_gpu([4])
    assert paged.plan(lens, on_gpu([48, 1]), table, free, n_free, page_size=16).tolist() == [0, 49, 4, 0]
    assert table.tolist() == [[2, 0, 1, -1], [3, -1, -1, -1]] and lens.tolist() == [48, 1]
    assert paged.plan(lens, on_gpu([1, 0]), table, free, n_free, page_size=16).tolist() == [-7, 0, 0, 0]
    # one leaves in the step in which the other needs its page
    assert paged.plan(lens, on_gpu([1, -1]), table, free, n_free, page_size=16).tolist() == [0, 1, 1, 0]
    assert table[0].tolist() == [2, 0, 1, 3] and lens.tolist() == [49, 0]
    assert paged.plan(lens, on_gpu([-2 ** 31, -2 ** 31]), table, free, n_free, page_size=16).tolist() == [0, 0, 0, 4]
    assert sorted(free.tolist()) == [0, 1, 2, 3] and lens.tolist() == [0, 0]


@pytest.mark.parametrize("lens,delta,n_free,stack,code", [
    ([-1, 0], [1, 0], 2, [0, 1], -1), ([0, 0], [1, 0], 3, [0, 1], -1), ([0, 0], [1, 0], -1, [0, 1], -1),
    ([0, 0], [1, 0], 2, [0, 9], -1), ([0, 0], [1, 0], 2, [0, -3], -1), ([0, 0], [65, 0], 2, [0, 1], -7),
    ([0, 0], [2 ** 31 - 1, 2 ** 31 - 1], 2, [0, 1], -7), ([2 ** 31 - 1, 0], [2 ** 31 - 1, 1], 2, [0, 1], -7),
    ([0, 0], [9, 0], 2, [0, 1], -7),
])
def test_plan_refuses_on_the_device(paged, lens, delta, n_free, stack, code):
    lens, delta, n_free, free = on_gpu(lens), on_gpu(delta), on_gpu([n_free]), on_gpu(stack)
    table, slots = on_gpu([[0, 1, 0, 1], [1, 0, 1, 0]]), on_gpu([5] * 8)
    keep = [t.clone() for t in (lens, n_free, free, table)]
    status = paged.plan(lens, delta, table, free, n_free, page_size=16, slots=slots)
    assert status.tolist() == [code, 0, 0, int(n_free)]
    for a, b in zip(keep, (lens, n_free, free, table)):
        assert torch.equal(a, b)
    assert (slots == -1).all()


def test_plan_refusals(paged):
    import syrinx_b200 as sx

    i = on_gpu([0, 0])
    table = on_gpu([[0], [0]])
    with pytest.raises(sx.SyrinxError):
        paged.plan(i, i, table, i, i[:1], page_size=12)
    for bad in (lambda: paged.plan(i, i[:1], table, i, i, page_size=16), lambda: paged.plan(i.long(), i, table, i, i, page_size=16),
                lambda: paged.plan(i, i, table[:1], i, i, page_size=16),
                lambda: paged.plan(i, i, table, i, i, page_size=16, slots=i, tok_pos=i[:1]),
                lambda: paged.plan(i, i, table, i, i, page_size=16, starts=i)):
        with pytest.raises(ValueError):
            bad()


# ---- together -----------------------------------------------------------------------------

@pytest.mark.parametrize("ct,layout,captured", [("f32", "hnd", False), ("bf16", "nhd", False), ("f32", "nhd", True),
                                                ("f16", "hnd", True)])
def test_plan_append_attend_as_a_decode_loop(paged, ct, layout, captured):
    """Requests of different ages decode over one pool; every step's result equals dense float64
    attention over all rows the request has seen. `captured`: the decode steps replay one graph."""
    n, H, hkv, hd, ps, width, n_pages = 6, 8, 2, 64, 16, 8, 40
    g = gen(42)
    lens, n_free, free = on_gpu([0] * n), on_gpu([n_pages]), torch.randperm(n_pages, device="cuda").to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    k, v = (empty_cache(n_pages, hkv, ps, hd, DT[ct], layout) for _ in range(2))
    cos, sin = rope(width * ps, hd)
    qn, kn = (0.5 + torch.rand(hd, generator=g, device="cuda") for _ in range(2))
    seen_k, seen_v = [[] for _ in range(n)], [[] for _ in range(n)]
    opts = dict(n_heads=H, cos=cos, sin=sin, interleaved=True, q_norm=qn, k_norm=kn, layout=layout)

    def note(x, tokens):
        """Dense rows, rounded as the cache holds them; the queries in float64."""
        y, _ = ref_append(x, H, hkv, hd, on_gpu([p for _, p in tokens]), cos, sin, True, qn, kn, 1e-6)
        for j, (i, _) in enumerate(tokens):
            seen_k[i].append(y[j, H:H + hkv].to(DT[ct]).double())
            seen_v[i].append(y[j, H + hkv:].to(DT[ct]).double())
        return y[:, :H]

    # prompts
    prompts = [5, 0, 33, 16, 1, 60]
    T = sum(prompts)
    slots, pos = (torch.empty(T + 3, dtype=torch.int32, device="cuda") for _ in range(2))
    paged.check(paged.plan(lens, on_gpu(prompts), table, free, n_free, page_size=ps, slots=slots, tok_pos=pos))
    x = torch.randn((T + 3, (H + 2 * hkv) * hd), generator=g, device="cuda")
    paged.append(x, k, v, slots, positions=pos, **opts)
    note(x[:T], [(i, p) for i, c in enumerate(prompts) for p in range(c)])

    delta, status = on_gpu([0] * n), torch.zeros(4, dtype=torch.int32, device="cuda")
    slots, pos, seqs = (torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(3))
    x = torch.zeros((n, (H + 2 * hkv) * hd), device="cuda")
    q, out = torch.zeros((n, H * hd), device="cuda"), torch.zeros((n, H, hd), device="cuda")
    by_req = torch.zeros((n, H, hd), device="cuda")
    starts = torch.zeros(n + 1, dtype=torch.int32, device="cuda")

    def step():
        paged.plan(lens, delta, table, free, n_free, page_size=ps, slots=slots, tok_seq=seqs, tok_pos=pos, starts=starts,
                   status=status)
        paged.append(x, k, v, slots, positions=pos, out=q, **opts)
        by_req.copy_(q.view(n, H, hd)[starts[:n].clamp(max=n - 1).long()])
        paged.attend(by_req, k, v, table, lens, layout=layout, out=out)

    graph = None
    if captured:
        keep = [t.clone() for t in (lens, n_free, free, table)]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for a, b in zip((lens, n_free, free, table), keep):
            a.copy_(b)
    for it in range(25):
        grow = [1] * n if it % 3 else [1, 0, 1, 1, 0, 1]
        if it == 10:
            grow[2] = -100000
            seen_k[2], seen_v[2] = [], []
        delta.copy_(on_gpu(grow))
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        old = lens.tolist()
        graph.replay() if graph else step()
        paged.check(status)
        tokens = [(i, old[i]) for i in range(n) if grow[i] > 0]
        Q = note(x[: len(tokens)], tokens)
        for j, (i, p) in enumerate(tokens):
            assert len(seen_k[i]) == p + 1
            K, V = (torch.stack(c[i]).repeat_interleave(H // hkv, 1) for c in (seen_k, seen_v))
            want = torch.einsum("ht,thd->hd", torch.softmax(torch.einsum("hd,thd->ht", Q[j], K) / 8, 1), V)
            # a key that rounds the other way after the f32 norm is off by one step of the cache's
            # type, 2^-8 (bf16): |ds| <= 2^-8 sum|q k| / 8 with |q|, |k| <= 1.5 * sqrt(2) * 4.5 each
            # would be the worst; rows that differ are few, the typical |ds| is 2^-9 * sqrt(64) / 8
            step_ = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[ct]
            assert (out[i].double() - want).abs().max() <= (4 * step_ + 2e-5) * V.abs().max()
    assert int(n_free) + sum(pages_of(x, ps) for x in lens.tolist()) == n_pages
