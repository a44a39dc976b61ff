"""Microscaled tensors at the ends of what they take: batches of no rows, the widest layers."""
import numpy as np
import pytest

from rgpu_amd import autograd as A
from rgpu_amd import gpu as G
from tests import mx_common as X

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    g = G.Gpu(0)
    yield g
    g.close()


@pytest.mark.parametrize("k,n", [(2 ** 22 + 1, 1), (1, 2 ** 22 + 1)])
def test_a_checkpointed_layer_too_wide_is_refused_before_it_runs(gpu, k, n):
    layer = A.Dense(gpu, k, n, "linear", weights=np.zeros((k, n), np.float32), checkpoint=True)
    with pytest.raises(ValueError):
        layer.forward(A.Tape(gpu).constant(np.zeros((1, k), np.float32)))


def test_a_batch_of_no_rows(gpu):
    rng = np.random.default_rng(0)
    one = A.Dense(gpu, 40, 30, "relu", weights=rng.normal(size=(40, 30)).astype(np.float32), checkpoint=True)
    two = A.Dense(gpu, 30, 5, "linear", weights=rng.normal(size=(30, 5)).astype(np.float32), checkpoint=True)
    tape = A.Tape(gpu)
    x = tape.constant(np.zeros((0, 40), np.float32))
    grads = two.forward(one.forward(x)).sum().backward()
    for layer in (one, two):
        for p in layer.params():
            assert not gpu.download(grads.of(p)).any()
    served = A.QuantizedSequential(A.Sequential([one, two]))
    assert gpu.download(served.predict(np.zeros((0, 40), np.float32))).shape == (0, 5)
    mask, out = gpu.zeros((0, 30), G.MXFP8), gpu.zeros((0, 30))
    gpu.matmul_a_bt(gpu.zeros((0, 7)), gpu.zeros((30, 7)), out, relu_mask_from=mask)
    gpu.relu_bwd(mask, out)
    gpu.map_vjp("relu", gpu.zeros((0, 30)), mask, None, out)
    for fmt in (G.MXFP4, G.MXFP8):
        assert gpu.download_f32(gpu.zeros((0, 7), fmt)).shape == (0, 7)
    gpu.sync()
