"""Routing where its 32-bit steps could decide otherwise than 64 bits."""
import numpy as np
import pytest

from rgpu_amd import gpu as G
from tests import token_common as T

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    g = G.Gpu(0)
    yield g
    g.close()


FEW = np.r_[0:8, 32:40]  # of 128 experts, two groups of 8 whose members are 32 apart


def few_left(kind, k, n, seed):
    """Logits and a bias of 128 experts of which FEW's alone can be chosen, by their groups or by biases of -inf, so that
    they stand in the same columns modulo 16: of each such pair one c is above 0.75, the least of them 0.75; k - 9 of the
    others are above it too; the rest lie within 2^-23 of where a threshold of 32 bits below 0.75 would be."""
    rng = np.random.default_rng(seed)
    bias = np.full(128, -0.25 if kind == "groups" else -np.inf, np.float32)
    bias[FEW] = 0.25 + rng.normal(size=16) * 0.01
    high, low = 0.75 + rng.uniform(0.01, 0.2, (n, 8)), 0.75 + rng.uniform(0.001, 0.009, (n, 8))
    high[:, 7] = 0.75
    low[:, k - 9:] = 0.75 - 2.0 ** -20 - 0.75 * 2.0 ** -22 + rng.uniform(-2, 2, (n, 17 - k)) * 2.0 ** -24
    turn = rng.uniform(size=(n, 8)) < 0.5
    s = np.concatenate([np.where(turn, high, low), np.where(turn, low, high)], axis=1) - bias[FEW].astype(np.float64)
    x = rng.normal(size=(n, 128))
    x[:, FEW] = np.log(s / (1 - s))
    return x.astype(np.float32), bias


@pytest.mark.parametrize("kind", ["groups", "biases"])
@pytest.mark.parametrize("k", [9, 10, 11, 12, 14, 16])
def test_route_of_more_choices_than_columns(gpu, kind, k):
    n = 8000
    x, bias = few_left(kind, k, n, k)
    ids, weights = gpu.empty((n, k), G.U32), gpu.empty((n, k))
    how = {"groups": 16, "kept": 2} if kind == "groups" else {}
    gpu.route(gpu.upload(x), ids, weights, gpu.upload(bias), score="sigmoid", **how)
    s = T.scores(x, "sigmoid")
    c = np.full(x.shape, -np.inf)
    c[:, FEW] = s[:, FEW] + bias[FEW].astype(np.float64)
    want = np.argsort(-c, axis=1, kind="stable")[:, :k]
    for t in range(0, n, 997):
        assert np.array_equal(T.route(x[t:t + 1], k, "sigmoid", bias, **how)[0][0], want[t])
    got = gpu.download(ids).astype(np.int64)
    # where the plain form's own c differ by its rounding only, either order is right
    same = got == want
    assert np.all(same | (abs(np.take_along_axis(c, got, 1) - np.take_along_axis(c, want, 1)) <= 2.0 ** -51))
    w = np.take_along_axis(s, want, 1)
    w /= w.sum(axis=1, keepdims=True)
    rows = same.all(axis=1)
    assert rows.mean() > 0.99 and np.all(abs(gpu.download(weights) - w)[rows] <= 2.0 ** -23 * w[rows])
