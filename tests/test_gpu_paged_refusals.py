"""Inputs of the paged key/value operators that only the GPU can refuse, or that are given in a form
that says nothing, on a B200."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def paged():
    from syrinx_b200 import paged as m
    return m


def on_gpu(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("n,who", [(4, 2), (700, 0), (700, 699), (5000, 4321), (8192, 8191)])
@pytest.mark.parametrize("bad", [2 ** 26 + 5, 2 ** 31 - 1, -1, 60000])
def test_plan_checks_the_page_that_a_token_falls_into(paged, n, who, bad):
    """A row's last page is not full, and its id is none of the pool's: shifted in 32 bits, 2^26 + 5
    would be the slots of page 5. Refused as a whole; a request that does not grow may hold anything."""
    ps, pages = 64, 60000
    lens, delta = on_gpu([100 + i % 27 for i in range(n)]), on_gpu([1 if i % 3 == who % 3 else 0 for i in range(n)])
    table = torch.arange(4 * n, dtype=torch.int32, device="cuda").view(n, 4).contiguous()
    free, n_free = torch.arange(pages, dtype=torch.int32, device="cuda"), on_gpu([0])
    slots = on_gpu([7] * n)
    table[who, 1] = bad
    keep = [t.clone() for t in (lens, n_free, free, table)]
    status = paged.plan(lens, delta, table, free, n_free, page_size=ps, slots=slots)
    assert status.tolist() == [-1, 0, 0, 0]
    for a, b in zip(keep, (lens, n_free, free, table)):
        assert torch.equal(a, b)
    assert (slots == -1).all()
    delta[who] = 0
    status = paged.plan(lens, delta, table, free, n_free, page_size=ps, slots=slots)
    grown = int((delta > 0).sum())
    assert status.tolist() == [0, grown, 0, 0]
    where = (delta > 0).nonzero()[:, 0]
    want = table[where, 1] * ps + keep[0][where] % ps
    assert torch.equal(slots[:grown], want.to(torch.int32)) and (slots[grown:] == -1).all()


def test_append_refuses_rotation_tables_without_rows(paged):
    x, none = torch.randn((4, 8 * 64), device="cuda"), torch.zeros((0, 32), device="cuda")
    k, v = (torch.full((5, 2, 16, 64), 7.0, device="cuda") for _ in range(2))
    with pytest.raises(ValueError):
        paged.append(x, k, v, on_gpu([0, 1, 2, 3]), n_heads=4, positions=on_gpu([0, 1, 2, 3]), cos=none, sin=none)
    assert (k == 7).all() and (v == 7).all()
