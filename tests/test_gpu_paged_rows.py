"""sx_paged_append over many wide rows on a B200, in the forms that tests of few or narrow rows do not reach."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def paged():
    from syrinx_b200 import paged as m
    return m


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("il", [True, False])
@pytest.mark.parametrize("H,hkv,hd,T", [(30, 5, 128, 3000), (32, 8, 128, 5001), (45, 3, 64, 4000), (9, 2, 256, 6000)])
def test_queries_in_place_over_many_rows(paged, dtype, il, H, hkv, hd, T):
    """The query part of x may be its own output where rows are copied ahead of the heads that are being
    stored: the same results as into another tensor, the key and value parts of x left alone."""
    x = torch.randn((T, (H + 2 * hkv) * hd), generator=gen(1), device="cuda").to(dtype)
    ang = torch.rand((100, hd // 2), generator=gen(2), device="cuda") * 6.28
    cos, sin = ang.cos(), ang.sin()
    pos = torch.arange(T, device="cuda", dtype=torch.int32) % 100
    slots = torch.randperm(-(-T // 16) * 16, generator=gen(3), device="cuda")[:T].to(torch.int32)
    slots[7::131] = -1
    k, v, k2, v2 = (torch.zeros((-(-T // 16), hkv, 16, hd), dtype=dtype, device="cuda") for _ in range(4))
    gain = 0.5 + torch.rand(hd, generator=gen(4), device="cuda")
    opts = dict(n_heads=H, positions=pos, cos=cos, sin=sin, interleaved=il, q_norm=gain, k_norm=gain)
    apart = x[:, : H * hd].clone()  # rows without a slot keep what the output holds
    paged.append(x, k, v, slots, out=apart, **opts)
    y = x.clone()
    paged.append(y, k2, v2, slots, out=y[:, : H * hd], **opts)
    assert torch.equal(y[:, : H * hd], apart) and torch.equal(y[:, H * hd:], x[:, H * hd:])
    assert torch.equal(k, k2) and torch.equal(v, v2)
    assert not torch.equal(apart[0], x[0, : H * hd]) and torch.equal(apart[7], x[7, : H * hd])
