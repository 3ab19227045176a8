"""What sx_paged_attention's arithmetic holds over 16-bit pages on a B200, against float64.
u = 2^-24 is half a step of f32."""
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
