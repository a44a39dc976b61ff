"""The numbers that dropout takes, without a GPU: what reaches the library."""
import numpy as np
import pytest

from rgpu_amd import gpu as G


class Calls:
    """Stands where a Gpu would: keeps the last call."""

    _h = None

    def _call(self, *args):
        self.last = args


class Handle:
    handle = None


@pytest.mark.parametrize("kind", [int, np.int32, np.int64, np.uint32, np.uint64])
def test_seeds_and_draws_of_any_whole_type(kind):
    g = Calls()
    G.Gpu.dropout(g, Handle, Handle, 0.5, kind(7), kind(9))
    assert g.last[-2:] == (7, 9)
    if kind not in (np.uint32, np.uint64):
        G.Gpu.dropout(g, Handle, Handle, 0.5, kind(-1), kind(-2))
        assert g.last[-2:] == ((1 << 64) - 1, (1 << 64) - 2)
    for bad in (1.5, "1", None):
        with pytest.raises(TypeError):
            G.Gpu.dropout(g, Handle, Handle, 0.5, bad)
