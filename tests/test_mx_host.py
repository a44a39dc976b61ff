"""Microscaled tensors without a GPU: sizes, the host decoder, and null handles."""
import numpy as np
import pytest

from rgpu_amd import gpu as G
from tests import mx_common as X


@pytest.mark.parametrize("fmt", [G.MXFP4, G.MXFP8])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 129), (64, 256), (65, 1000), (4100, 77)])
def test_tensor_bytes_and_decoder_agree_with_the_definition(fmt, rows, cols):
    x = X.values(np.random.default_rng(rows * cols), rows, cols)
    code, byte, want = X.quantize(x, fmt)
    data = X.pack(code, byte, fmt)
    assert G.tensor_bytes((rows, cols), fmt) == data.size
    assert np.array_equal(G.mx_decode(data, (rows, cols), fmt), want.astype(np.float32))


def test_error_of_a_block_is_half_a_step():
    # e2m1 has steps of a half at least and a third of its value at most; e4m3 an eighth of its exponent
    x = X.values(np.random.default_rng(3), 100, 256)
    amax = np.abs(x).reshape(100, -1, 32).max(axis=2, keepdims=True)
    for fmt, eps, least in ((G.MXFP4, 2.0 ** -2, 0.25 / 3), (G.MXFP8, 2.0 ** -4, 2.0 ** -10 / 224)):
        got = X.quantize(x, fmt)[2]
        err = np.abs(got - x).reshape(100, -1, 32)
        # amax > MAX/2 · scale, so a scale is below 2 amax / MAX
        assert np.all(err <= np.maximum(eps * np.abs(x).reshape(100, -1, 32), least * amax))


def test_tensor_bytes_of_bad_shapes():
    for shape in ((), (3,), (2, 3, 4)):
        assert G.tensor_bytes(shape, G.MXFP4) == 0
    assert G.tensor_bytes((0, 5), G.MXFP8) == 0 and G.tensor_bytes((5, 0), G.MXFP8) == 0
    assert G.tensor_bytes((2 ** 40, 2 ** 40), G.MXFP4) == 0
    assert G.lib().rt_tensor_bytes(6, None, 0) == 0
    assert G.lib().rt_tensor_bytes(G.F32, None, 0) == 4


def test_null_handles():
    L = G.lib()
    assert L.rt_convert_t(None, None, None) == 2
    assert L.rt_wrap(None, G.F32, None, 0, None, None) == 2


@pytest.mark.parametrize("fmt", [G.MXFP4, G.MXFP8])
@pytest.mark.parametrize("shape", [(0, 5), (5, 0), (0, 0)])
def test_decoder_of_no_elements(shape, fmt):
    got = G.mx_decode(np.zeros(0, np.uint8), shape, fmt)
    assert got.shape == shape and got.dtype == np.float32
