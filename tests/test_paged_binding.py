"""Arguments that syrinx_b200.paged has to refuse by their shape, without a GPU."""
import pytest

torch = pytest.importorskip("torch")


def test_append_refuses_rotation_tables_without_rows():
    """Tables of no position are not the same as no tables: every position is outside them."""
    from syrinx_b200 import paged

    i, kv = torch.zeros(4, dtype=torch.int32), torch.zeros(2, 8, 16, 64)
    x, none = torch.zeros(4, 24 * 64), torch.zeros(0, 32)
    for cos, sin in ((none, none), (none, None), (None, none), (torch.zeros(9, 32), none)):
        with pytest.raises(ValueError, match="one position at least"):
            paged.append(x, kv, kv, i, n_heads=8, positions=i, cos=cos, sin=sin)
    with pytest.raises(ValueError, match="CUDA device"):
        paged.append(x, kv, kv, i, n_heads=8, positions=i, cos=torch.zeros(9, 32), sin=torch.zeros(9, 32))
