"""What sx_paged_attention's arithmetic holds over 16-bit pages on a B200, against float64.
u = 2^-24 is half a step of f32.

A tensor-core product of 16 terms cuts the terms off (and what it adds them to) at the last place
of the largest one, always towards zero, so one result is off by at most 17 quarter steps, 9 u of
its terms' sizes, where nothing larger is added to."""
import math

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


TYPES = [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")]


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("hd", [64, 256])
def test_infinite_values_under_small_weights(paged, qt, ct, hd):
    """An infinite value under a weight of exp(-x), down to 2^-115 of the largest, makes its own output
    element infinite with its sign, and no other: no part of such a weight may be zero.

    The other elements: two to six values of size below 8 under weights below one, off by at most
    (8 sqrt(6) + 12) u and the scores' error, which are exact products of one element here (x log2(e)
    is off by 2 u of 115, so a weight by 160 u); a 16-bit result is rounded once."""
    sizes = [0.0, 1.0, 5.0, 8.5, 9.0, 10.0, 12.0, 15.0, 17.0, 20.0, 27.0, 40.0, 60.0, 72.0, 79.5]
    n, ps, length = len(sizes), 8, 6
    g = gen(hd)
    k = torch.zeros((n, 1, ps, hd), device="cuda")
    v = torch.randn((n, 1, ps, hd), generator=g, device="cuda").clamp(-8, 8).to(DT[ct])
    for i, x in enumerate(sizes):
        k[i, 0, 1:, 7] = -x
    clean = v[:, 0, :length].double()
    v[:, 0, 3, 5], v[:, 0, 4, 20], v[:, 0, 2, 31], v[:, 0, 5, 31] = math.inf, -math.inf, math.inf, math.inf
    q = torch.zeros((n, 3, hd), device="cuda")
    q[:, :, 7] = 1.0
    table = torch.arange(n, dtype=torch.int32, device="cuda").view(n, 1)
    lens = torch.full((n,), length, dtype=torch.int32, device="cuda")
    out = paged.attend(q.to(DT[qt]), k.to(DT[ct]), v, table, lens, scale=1.0)
    assert (out[:, :, 5] == math.inf).all() and (out[:, :, 20] == -math.inf).all() and (out[:, :, 31] == math.inf).all()
    w = torch.exp(-torch.tensor(sizes, dtype=torch.float64, device="cuda"))[:, None].repeat(1, length)
    w[:, 0] = 1.0
    want = (w[:, :, None] * clean).sum(1) / w.sum(1, keepdim=True)
    rest = [d for d in range(hd) if d not in (5, 20, 31)]
    low = {"f32": 0.0, "bf16": 2.0 ** -17, "f16": 2.0 ** -22}[ct]
    tol = 2 * (8 * math.sqrt(6) + 12 + 160) * U * 8 + low * 16
    if qt != "f32":
        tol = tol + want.abs() * torch.finfo(DT[qt]).eps / 2 + 2.0 ** -25
        tol = tol[:, rest][:, None]
    err = (out.double() - want[:, None])[:, :, rest].abs()
    assert (err <= tol).all(), float(err.max())


@pytest.mark.parametrize("ct", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_sums_over_long_runs_do_not_drift(paged, ct, hd):
    """A thousand tiles and more in one warp's run, values of one sign: what every tile's addition
    lost would add up. All keys but the first have one weight p = exp(-0.3), so the result is
    (v_0 + p sum v) / (1 + p (n - 1)), whose last bits do not depend on p's own rounding.

    Bound. A tile's sum is off by 9 u (above) + 4 u (the weights' split, 2^-22). The T additions
    of a run are off by at most u of the partial sum each; as independent ones, of variance a third
    of that squared, they come to u sqrt(T) / 3 of the sum, and six times that are allowed for; the
    join of the runs, the sum of the weights (the same additions, on one lane) and the quotient are
    allowed 2 sqrt(T) + 16 once more."""
    ps, length = 64, 131072
    g = gen(hd)
    n = torch.cuda.get_device_properties(0).multi_processor_count  # a CTA's share is one request
    v = (1 + torch.rand((length // ps, 1, ps, hd), generator=g, device="cuda")).to(DT[ct])
    k = torch.zeros_like(v)
    k[:, :, :, 3] = -0.5
    k[0, 0, 0, 3] = 0.0
    q = torch.zeros((n, 2, hd), device="cuda")
    q[:, :, 3] = 0.6
    table = torch.arange(length // ps, dtype=torch.int32, device="cuda").expand(n, -1).contiguous()
    lens = torch.full((n,), length, dtype=torch.int32, device="cuda")
    out = paged.attend(q, k, v, table, lens, scale=1.0)
    w = torch.full((length, 1), math.exp(0.6 * -0.5), dtype=torch.float64, device="cuda")
    w[0] = 1.0
    want = (w * v.view(length, hd).double()).sum(0) / w.sum()
    keys = (1024 // hd if ct == "f32" else {32: 64, 64: 32}.get(hd, 16))  # of a tile
    T = length // keys // (4 if hd == 256 and ct != "f32" else 8)
    err = ((out.double() - want) / want).abs().max()
    assert err <= (4 * math.sqrt(T) + 13 + 16) * U, f"{float(err / U):.1f} u, {T} tiles"


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_scores_of_one_sign(paged, qt, ct, hd):
    """A request of one key has lse = scale q.k; all products positive, so that what they lose adds up.

    Bound. The products of 16 elements are cut off by at most 8 u of their sum (above; f32 pages: a
    product is rounded once), their hd / 16 (f32 pages: hd / 4 and more) additions come to 2 sqrt(hd / 4) u
    as in the runs above; queries' parts, scale and the two logarithms 8 u."""
    n, ps = 512, 8
    g = gen(hd)
    k = torch.randn((n, 1, ps, hd), generator=g, device="cuda").abs().to(DT[ct])
    q = torch.randn((n, 4, hd), generator=g, device="cuda").abs().to(DT[qt])
    table = torch.arange(n, dtype=torch.int32, device="cuda").view(n, 1)
    lens = torch.ones(n, dtype=torch.int32, device="cuda")
    lse = torch.empty((n, 4), device="cuda")
    paged.attend(q, k, torch.zeros_like(k), table, lens, scale=1.0, lse=lse)
    want = torch.einsum("nhd,nd->nh", q.double(), k[:, 0, 0].double())
    err = ((lse.double() - want) / want).abs().max()
    assert err <= (8 + 2 * math.sqrt(hd / 4) + 8) * U, f"{float(err / U):.1f} u"


@pytest.mark.parametrize("qt,ct", [("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
def test_weights_keep_their_bits(paged, qt, ct):
    """Requests of two keys, over many: a 16-bit result is the rounding of one that is f32's but for a few
    u, so it is off by more than half a step only where the exact result is that near to a tie.

    Bound. The scores are one exact product each, below 4 in size: in units of log 2 they are off by two
    roundings, so a weight by 4 * 2 u and pow2's own 4 u. Its parts hold 24 bits in bf16 (u), 22 in f16
    (4 u). Two products (9 u of their sizes), two sums, a quotient: 14 u; and the sum of the weights is
    off by 12 u. 40 u of sum p|v| / sum p in all, and half a step of the result."""
    n, H, hd, ps = 4096, 8, 64, 8
    g = gen(5)
    k = torch.zeros((n, 1, ps, hd), device="cuda")
    k[:, 0, 1, 9] = -1.0
    v = torch.randn((n, 1, ps, hd), generator=g, device="cuda").to(DT[ct])
    q = torch.zeros((n, H, hd), device="cuda")
    q[:, :, 9] = 4 * torch.rand((n, H), generator=g, device="cuda")
    q = q.to(DT[qt])
    table = torch.arange(n, dtype=torch.int32, device="cuda").view(n, 1)
    lens = torch.full((n,), 2, dtype=torch.int32, device="cuda")
    out = paged.attend(q, k.to(DT[ct]), v, table, lens, scale=1.0)
    p = torch.exp(-q[:, :, 9].double())[:, :, None]
    a, b = v[:, 0, 0].double()[:, None], v[:, 0, 1].double()[:, None]
    want = (a + p * b) / (1 + p)
    tol = 40 * U * (a.abs() + p * b.abs()) / (1 + p)
    if qt != "f32":
        step = torch.exp2(torch.floor(torch.log2(out.double().abs()))) * torch.finfo(DT[qt]).eps
        tol = tol + torch.clamp(step, min=2.0 ** -24 if qt == "f16" else 0.0) / 2
    over = ((out.double() - want).abs() > tol).sum()
    assert over == 0, f"{int(over)} of {out.numel()}"


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("longest", [40, 6000])
def test_lse_of_equal_scores(paged, qt, ct, longest):
    """Scores of zero: lse = log n, whatever power of two the weights are kept at. Their sum is exact, so
    what is left is log2, half a step and a bit, and a product: 4 u of the result. 6000: joined runs."""
    hkv, hd, ps = 1, 128, 16
    lens = list(range(1, 40)) + [longest]
    pages = -(-longest // ps)
    k = torch.zeros((pages, hkv, ps, hd), device="cuda").to(DT[ct])
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(len(lens), -1).contiguous()
    q = torch.randn((len(lens), 4, hd), generator=gen(1), device="cuda").to(DT[qt])
    lse = torch.empty((len(lens), 4), device="cuda")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    paged.attend(q, k, k, table, n, lse=lse)
    want = n.double().log()[:, None]
    assert ((lse.double() - want).abs() <= 4 * U * want).all(), float(((lse.double() - want).abs() / U).max())
