"""Layers over the microscaled operators: the tape's Dense with its activations kept in 8 bits, and a model served with
weights in 4 bits."""
import weakref

import numpy as np
import pytest

from rgpu_amd import autograd as A
from rgpu_amd import gpu as G
from tests import mx_common as X

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24  # half a step of f32


@pytest.fixture(scope="module")
def gpu():
    g = G.Gpu(0)
    yield g
    g.close()


def dense(gpu, rng, k, n, activation, **kw):
    return A.Dense(gpu, k, n, activation, weights=rng.normal(size=(k, n)).astype(np.float32) / np.sqrt(k),
                   bias=rng.normal(size=(1, n)).astype(np.float32) * 0.1, **kw)


def weighted_sum(z, c):
    """Σ c ⊙ z: a loss whose gradient with respect to z is c."""
    return z.mul(A.constant(z.tape, c)).sum()


@pytest.mark.parametrize("rows,k,h,n", [(1, 3, 5, 2), (33, 100, 70, 10), (300, 256, 129, 64)])
def test_checkpointed_layers_against_the_formula(gpu, rows, k, h, n):
    rng = np.random.default_rng(rows)
    one, two = dense(gpu, rng, k, h, "relu", checkpoint=True), dense(gpu, rng, h, n, "linear", checkpoint=True)
    x, c = X.values(rng, rows, k), rng.normal(size=(rows, n)).astype(np.float32)
    tape = A.Tape(gpu)
    vx = tape.constant(x)
    a = one.forward(vx)
    z = two.forward(a)
    grads = weighted_sum(z, c).backward()
    plain = A.Sequential([A.Dense(gpu, k, h, "relu", weights=one.w.value(), bias=one.b.value()),
                          A.Dense(gpu, h, n, weights=two.w.value(), bias=two.b.value())])
    assert np.array_equal(z.numpy(), gpu.download(plain.predict(x)))  # the forward pass is the f32 one
    av, w1, w2 = a.numpy().astype(np.float64), one.w.value().astype(np.float64), two.w.value().astype(np.float64)
    c64, x64 = c.astype(np.float64), x.astype(np.float64)
    # The mask is that of the f32 activation, sums of n products in f32 are off by at most n half steps of their sizes
    # (three planes a product for dW), and each factor of a later product carries its own.
    d1, s1 = (c64 @ w2.T) * (av > 0), (np.abs(c64) @ np.abs(w2).T) * (av > 0)
    xq, aq = X.quantize(x, G.MXFP8)[2], X.quantize(av, G.MXFP8)[2]
    e1 = (n + 8) * 2 * EPS * s1
    for got, want, tol in (
            (two.w, aq.T @ c64, (3 * rows + 40) * 2 * EPS * (np.abs(aq).T @ np.abs(c64))),
            (two.b, c64.sum(0, keepdims=True), (rows + 8) * 2 * EPS * np.abs(c64).sum(0, keepdims=True)),
            (one.w, xq.T @ d1, (3 * rows + 40) * 2 * EPS * (np.abs(xq).T @ s1) + np.abs(xq).T @ e1),
            (one.b, d1.sum(0, keepdims=True), (rows + 8) * 2 * EPS * s1.sum(0, keepdims=True) + e1.sum(0, keepdims=True))):
        assert np.all(np.abs(gpu.download(grads.of(got)) - want) <= tol)
    dx = gpu.download(grads.of_var(vx))
    assert np.all(np.abs(dx - d1 @ w1.T) <= (h + 8) * 2 * EPS * (s1 @ np.abs(w1).T) + e1 @ np.abs(w1).T)


@pytest.mark.parametrize("activation", ["linear", "relu", "tanh", "sigmoid", ("leaky_relu", 0.1)])
def test_checkpointed_gradients_against_the_f32_node_and_differences(gpu, activation):
    rows, k, n = 40, 70, 24
    rng = np.random.default_rng(7)
    kept = dense(gpu, rng, k, n, activation, checkpoint=True)
    full = A.Dense(gpu, k, n, activation, weights=kept.w.value(), bias=kept.b.value())
    x, c = X.values(rng, rows, k), rng.normal(size=(rows, n)).astype(np.float32)
    out = []
    for layer in (kept, full):
        tape = A.Tape(gpu)
        vx = tape.constant(x)
        z = layer.forward(vx)
        g = weighted_sum(z, c).backward()
        out.append([z.numpy(), gpu.download(g.of_var(vx)), gpu.download(g.of(layer.b)), gpu.download(g.of(layer.w))])
    (z8, dx8, db8, dw8), (z, dx, db, dw) = out
    assert np.array_equal(z8, z)
    # the same δ goes into both; dX is summed by the same kernels or their paired form, db in another order
    size = np.abs(dx).max(initial=0)
    assert np.all(np.abs(dx8 - dx) <= 64 * EPS * np.maximum(size, 1) * n)
    assert np.all(np.abs(db8 - db) <= 2 * (rows + 8) * EPS * np.abs(c).sum(0))
    # dW differs by what the 8 bits leave out, times a δ that is at most |c| (every slope here is at most 1)
    left = np.abs(x - X.quantize(x, G.MXFP8)[2])
    assert np.all(np.abs(dw8 - dw) <= left.T @ np.abs(c) + 8 * rows * EPS * (np.abs(x).T @ np.abs(c)))
    if activation == "linear":
        # L is linear in each weight: its difference over a step of 2 is exact up to the sums' rounding
        for i, j in ((0, 0), (13, 5), (69, 23)):
            w = full.w.value()
            ends = []
            for step in (-1, 1):
                moved = w.copy()
                moved[i, j] += step
                layer = A.Dense(gpu, k, n, activation, weights=moved, bias=full.b.value())
                ends.append((layer.forward(A.Tape(gpu).constant(x)).numpy().astype(np.float64) * c).sum())
            bound = left[:, i] @ np.abs(c[:, j]) + (k + rows + 16) * 8 * EPS * (
                (np.abs(x) @ (np.abs(w) + 1) + 1) * np.abs(c)).sum()
            assert abs((ends[1] - ends[0]) / 2 - dw8[i, j]) <= bound


def test_checkpointed_layers_hold_no_f32_activation(gpu):
    rng = np.random.default_rng(1)
    model = A.Sequential([dense(gpu, rng, 64, 96, "relu", checkpoint=True), dense(gpu, rng, 96, 96, "relu", checkpoint=True),
                          dense(gpu, rng, 96, 8, "linear", checkpoint=True)])
    tape = A.Tape(gpu)
    v, seen, saved = tape.constant(X.values(rng, 50, 64)), [], []
    for layer in model.layers:
        v = layer.forward(v)
        seen.append(weakref.ref(v.value))
        saved.append(v._saved8)
    assert seen[0]() is None and seen[1]() is None and seen[2]() is v.value
    assert saved[0] is not None and saved[1] is not None and saved[2] is None  # one copy for mask and next layer, none unused
    loss = A.softmax_cross_entropy(v, A.one_hot(rng.integers(0, 8, 50), 8))
    grads = loss.backward()
    assert all(np.isfinite(gpu.download(grads.of(p))).all() for p in model.params())


def test_training_with_checkpoints_runs_and_shares_an_input(gpu):
    rng = np.random.default_rng(2)
    left, right = dense(gpu, rng, 32, 16, "relu", checkpoint=True), dense(gpu, rng, 32, 16, "tanh", checkpoint=True)
    opt = A.Adam(1e-2)
    x = X.values(rng, 90, 32)
    for _ in range(3):
        tape = A.Tape(gpu)
        vx = tape.constant(x)
        a, b = left.forward(vx), right.forward(vx)
        q = vx.saved8()
        grads = a.mul(b).sum().backward()
        assert vx.saved8() is q
        # both layers' gradients reach the shared input
        da, db = b.numpy().astype(np.float64), a.numpy().astype(np.float64)
        d1 = da * (a.numpy() > 0)
        d2 = db * (1 - b.numpy().astype(np.float64) ** 2)
        w1, w2 = left.w.value().astype(np.float64), right.w.value().astype(np.float64)
        want, size = d1 @ w1.T + d2 @ w2.T, np.abs(d1) @ np.abs(w1).T + np.abs(d2) @ np.abs(w2).T
        assert np.all(np.abs(gpu.download(grads.of_var(vx)) - want) <= 64 * 2 * EPS * (size + np.abs(db) @ np.abs(w2).T))
        opt.step(left.params() + right.params(), grads)
    assert all(np.isfinite(p.value()).all() for p in left.params() + right.params())


def test_checkpoint_refusals(gpu):
    rng = np.random.default_rng(3)
    with pytest.raises(ValueError):
        dense(gpu, rng, 4, 4, "relu", fused=False, checkpoint=True)
    layer = dense(gpu, rng, 4, 4, "relu", checkpoint=True)
    with pytest.raises(ValueError):
        layer.forward(A.Tape(gpu).constant(np.zeros((2, 3, 4), np.float32)))
    with pytest.raises(ValueError):
        A.Tape(gpu).constant(np.zeros(4, np.float32)).saved8()
    with pytest.raises(ValueError):
        A.dense_node(A.Tape(gpu).constant(np.zeros((2, 4), np.float32)), layer.w.watch(A.Tape(gpu)),
                     layer.b.watch(A.Tape(gpu)), True, True)


@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("activations", [G.MXFP4, G.MXFP8])
def test_quantized_model_is_its_operators_in_a_row(gpu, rows, activations):
    rng = np.random.default_rng(rows)
    model = A.Sequential([dense(gpu, rng, 100, 130, "relu"), dense(gpu, rng, 130, 64, "linear"),
                          dense(gpu, rng, 64, 48, ("leaky_relu", 0.25)), dense(gpu, rng, 48, 10, "linear")])
    served = A.QuantizedSequential(model, activations)
    x = X.values(rng, rows, 100)
    got = gpu.download(served.predict(x))
    # by hand, and the first layer against numpy
    v = gpu.upload(x)
    for i, layer in enumerate(model.layers):
        k, n = layer.w.shape
        w4, q = gpu.zeros((n, k), G.MXFP4), gpu.zeros((rows, k), activations)
        gpu.convert_t(layer.w.tensor, w4)
        gpu.convert(v, q)
        assert np.array_equal(gpu.download_f32(w4), X.quantize(layer.w.value().T, G.MXFP4)[2].astype(np.float32))
        v = gpu.zeros((rows, n), G.BF16 if i in (0, 1) else G.F32)
        gpu.gemm(G.NT, q, w4, v, G.EPI_BIAS_RELU if i == 0 else G.EPI_BIAS, layer.b.tensor)
        if i == 0:
            xv, wv, b = X.quantize(x, activations)[2], X.quantize(layer.w.value().T, G.MXFP4)[2], layer.b.value()
            size = np.abs(xv) @ np.abs(wv).T + np.abs(b)
            want = np.maximum(xv @ wv.T + b, 0)
            # sums in f32, an 8-bit operand's neighbours (7 · 2^-13 of their sizes), one rounding to bf16
            assert np.all(np.abs(gpu.download_f32(v) - want) <= 108 * 2 * EPS * size + 7 * 2.0 ** -13 * size + 2.0 ** -8 * want)
        if i == 2:
            gpu.map("leaky_relu", v, v, 0.25)
    assert got.shape == (rows, 10) and np.array_equal(got, gpu.download(v))
    # inputs in half precision, and what does not fit
    half = gpu.upload(x, G.BF16)
    assert served.predict(half).shape == (rows, 10)
    with pytest.raises(ValueError):
        served.predict(np.zeros((rows, 99), np.float32))
    with pytest.raises(ValueError):
        served.predict(np.float32(1.0))
    with pytest.raises(ValueError):
        A.QuantizedSequential(model, G.F32)
    with pytest.raises(ValueError):
        A.QuantizedSequential(A.Sequential([]))
    # the served weights are a copy
    model.layers[0].w.set(np.zeros((100, 130), np.float32))
    model.layers[0].b.set(np.zeros((1, 130), np.float32))
    assert np.array_equal(gpu.download(served.predict(x)), got)
