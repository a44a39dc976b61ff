"""Routing where its 32-bit steps could decide otherwise than 64 bits, and its gradient where it is a small difference of large
terms."""
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


def gradient(x, ids, g, score, renormalise, scale):
    """(dx, what its terms add up to without their signs), from sums that hold no difference of nearly equal numbers but
    those of the given g: with e the powers, T their sum over all experts (or over the chosen, if renormalised),
    g_j - sum_i w_i g_i = (g_j sum of the e not chosen + sum_i e_i (g_j - g_i)) / T; 1 - sigmoid(z) = sigmoid(-z)."""
    x, g = x.astype(np.float64), g.astype(np.float64)
    e = T.scores(x, "sigmoid") if score == "sigmoid" else np.exp(x - x.max(axis=1, keepdims=True))
    ej = np.take_along_axis(e, ids, axis=1)
    left = e.copy()
    np.put_along_axis(left, ids, 0, axis=1)
    left = left.sum(axis=1, keepdims=True)
    apart = g[:, :, None] - g[:, None, :]
    if renormalise:
        total = ej.sum(axis=1, keepdims=True)
        d, size = ej * (ej[:, None] * apart).sum(axis=2) / total ** 2, ej * (ej[:, None] * abs(apart)).sum(axis=2) / total ** 2
    elif score == "softmax":
        total = ej.sum(axis=1, keepdims=True) + left
        d = ej * (g * left + (ej[:, None] * apart).sum(axis=2)) / total ** 2
        size = ej * (abs(g) * left + (ej[:, None] * abs(apart)).sum(axis=2)) / total ** 2
    else:
        d, size = ej * g, ej * abs(g)
    if score == "sigmoid":
        rest = T.scores(-np.take_along_axis(x, ids, axis=1), "sigmoid")
        d, size = d * rest, size * rest
    dx, big = np.zeros_like(e), np.zeros_like(e)
    if score == "softmax" and not renormalise:
        dx, big = -e * (ej * g).sum(axis=1, keepdims=True) / total ** 2, e * (ej * abs(g)).sum(axis=1, keepdims=True) / total ** 2
    np.put_along_axis(dx, ids, d, axis=1)
    np.put_along_axis(big, ids, size, axis=1)
    return scale * dx, scale * big


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("experts,k", [(2, 1), (8, 1), (8, 2), (8, 8), (64, 4), (256, 8), (300, 20), (1024, 64)])
@pytest.mark.parametrize("gap", [0, 8, 12, 17, 30, 60])
def test_route_backward_of_a_confident_router(gpu, score, renormalise, experts, k, gap):
    """One logit `gap` above the others: the chosen ones' gradients are as small as what is left of 1, and as exact."""
    rng = np.random.default_rng(experts + k + gap)
    n = 40
    x = (rng.normal(size=(n, experts)) * 0.5).astype(np.float32)
    x[np.arange(n), rng.integers(0, experts, n)] += gap
    if score == "sigmoid" and renormalise:
        x -= np.float32(gap)  # scores from 0.5 down
    ids = T.route(x, k, score)[0]
    g = rng.normal(size=(n, k)).astype(np.float32)
    g[::3] = g[::3, :1]  # one gradient for all: nothing but what the others' scores leave
    dx = gpu.empty((n, experts))
    gpu.route_backward(gpu.upload(x), T.words(gpu, ids), gpu.upload(g), dx, score=score, renormalise=renormalise, scale=2.5)
    want, size = gradient(x, ids, g, score, renormalise, 2.5)
    # f32 powers: the difference from the greatest logit rounded (half a step of at most gap + 4), two steps of their
    # own, at most 22 additions: once in what was not chosen, twice in the sum (there without the gap, whose terms are as
    # much smaller); a dozen roundings beside
    err = (gap + 3 * (4 + 4 + 22) + 12) * 2.0 ** -24 * size
    assert np.all(abs(gpu.download(dx) - want) <= err + T.LEAST[G.F32])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
def test_route_backward_of_an_expert_named_twice(gpu, score, renormalise):
    """A program's own choice may name an expert more than once: each time counts."""
    rng = np.random.default_rng(0)
    x, g = rng.normal(size=(30, 20)).astype(np.float32), rng.normal(size=(30, 5)).astype(np.float32)
    ids = rng.integers(0, 4, (30, 5))
    ids[::5, 1] = G.PADDING
    dx = gpu.empty((30, 20))
    gpu.route_backward(gpu.upload(x), T.words(gpu, ids), gpu.upload(g), dx, score=score, renormalise=renormalise, scale=1.5)
    s = T.scores(x, score)
    want, size = np.zeros((30, 20)), np.zeros((30, 20))
    for t in range(30):
        on = [j for j in range(5) if ids[t, j] < 20]
        sj = s[t, ids[t, on]]
        z = sj.sum() if renormalise else 1.0
        ds, big = np.zeros(20), np.zeros(20)  # of the scores
        np.add.at(ds, ids[t, on], 1.5 * g[t, on] / z - (1.5 * (g[t, on] * sj).sum() / z ** 2 if renormalise else 0))
        np.add.at(big, ids[t, on], 1.5 * abs(g[t, on]) / z + (1.5 * (abs(g[t, on]) * sj).sum() / z ** 2 if renormalise else 0))
        if score == "sigmoid":
            want[t], size[t] = s[t] * (1 - s[t]) * ds, s[t] * big
        else:
            want[t], size[t] = s[t] * (ds - (s[t] * ds).sum()), s[t] * (big + (s[t] * big).sum())
    # as without repetitions: powers and their sum to a few steps, a dozen roundings, at most 5 f32 additions
    assert np.all(abs(gpu.download(dx) - want) <= 50 * 2.0 ** -24 * size + T.LEAST[G.F32])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,k", [(8, 1), (64, 3), (100, 20), (600, 4)])
def test_weights_of_scores_whose_reciprocal_is_infinite(gpu, score, experts, k):
    """A bias takes out the experts with the great scores; those left are below 2^-1022, and weigh `scale` together."""
    rng = np.random.default_rng(experts)
    low = (-709.7, -709.0) if score == "sigmoid" else (-718.0, -709.0)
    x = rng.uniform(*low, (5, experts)).astype(np.float32)
    x[:, :experts // 2] = 0
    bias = np.zeros(experts, np.float32)
    bias[:experts // 2] = -np.inf
    ids, weights, dx = gpu.empty((5, k), G.U32), gpu.empty((5, k)), gpu.empty((5, experts))
    gpu.route(gpu.upload(x), ids, weights, gpu.upload(bias), score=score, scale=2.5)
    got = gpu.download(ids).astype(np.int64)
    assert got.min() >= experts // 2
    z = np.take_along_axis(x, got, 1).astype(np.float64)  # 1 / (1 + e^-z) is e^z here, to 300 places
    w = np.exp(z - z.max(axis=1, keepdims=True))
    w *= 2.5 / w.sum(axis=1, keepdims=True)
    # one rounding; a score is a whole number of 2^-1074, at least 2^36 of them
    assert np.all(abs(gpu.download(weights) - w) <= 2.0 ** -23 * w)
    g = rng.normal(size=(5, k)).astype(np.float32)
    gpu.route_backward(gpu.upload(x), ids, gpu.upload(g), dx, score=score, scale=2.5)
    want = np.zeros((5, experts))
    np.put_along_axis(want, got, w * (g - (w / 2.5 * g).sum(axis=1, keepdims=True)), axis=1)
    assert np.all(abs(gpu.download(dx) - want) <= 2.0 ** -22 * 2.5 * abs(g).max())


@pytest.mark.parametrize("dtype", T.TYPES, ids=T.NAMES.get)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("tokens,experts,k", [(1, 8, 2), (37, 64, 4), (1000, 256, 8), (9, 1000, 30)])
def test_route_backward_in_place(gpu, dtype, score, renormalise, tokens, experts, k):
    rng = np.random.default_rng(tokens)
    x, v = T.put(gpu, rng.normal(size=(tokens, experts)), dtype)
    ids = T.words(gpu, T.route(v, k, score)[0])
    g, dx = gpu.upload(rng.normal(size=(tokens, k)).astype(np.float32)), gpu.empty((tokens, experts), dtype)
    gpu.route_backward(x, ids, g, dx, score=score, renormalise=renormalise)
    want = gpu.download_f32(dx)
    gpu.route_backward(x, ids, g, x, score=score, renormalise=renormalise)
    assert np.array_equal(gpu.download_f32(x), want)
