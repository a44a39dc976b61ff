"""Microscaled tensors at the ends of what they take: batches of no rows, the widest layers, every bf16 value, the smallest
values, tall tensors."""
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


@pytest.mark.parametrize("rows,K,N", [(100, 60, 50), (300, 2000, 2048)])
@pytest.mark.parametrize("dtype,power", [("bf16", 100), ("f32", 100), ("bf16", 0), ("f32", 20), ("f16", 10)])
def test_gradient_from_the_smallest_values(gpu, rows, K, N, dtype, power):
    """Values of X whose bits reach below 2^-133, the last of a bf16 (scale bytes 0 to 2): a product keeps those from 2^-133
    on; beside an f16 gradient values up to 2^-118 may count as zeros."""
    rng = np.random.default_rng(17)
    x = (rng.normal(size=(rows, K)) * np.exp2(rng.integers(-130, -117, size=(rows, -(-K // 32))).repeat(32, 1)[:, :K])).astype(
        np.float32)
    code, byte, xv = X.quantize(x, G.MXFP8)
    assert (byte == 0).any() and (byte == 1).any() and (byte == 2).any() and np.any(xv % 2.0 ** -133)
    q = gpu.upload(X.pack(code, byte, G.MXFP8), G.MXFP8, x.shape)
    d = np.ldexp(rng.normal(size=(rows, N)), power).astype(np.float32)
    if dtype == "bf16":
        d = G.bf16_bits_to_f32(G.f32_to_bf16_bits(d))
    elif dtype == "f16":
        d = d.astype(np.float16).astype(np.float32)
    d64 = d.astype(np.float64)
    dw = gpu.empty((K, N))
    gpu.matmul_at_b(q, gpu.upload(d, {"f32": G.F32, "bf16": G.BF16, "f16": G.F16}[dtype]), dw)
    # the sums as elsewhere; each product short of at most 2^-133 of its factor of X; f32 results that are subnormal
    # themselves (power 0) are rounded to 2^-149 in each of the sum's steps
    kept = np.where(np.abs(xv) <= 2.0 ** -118, np.abs(xv), 0) if dtype == "f16" else np.minimum(np.abs(xv), 2.0 ** -133)
    tol = (3 * rows + 40) * (2.0 ** -23 * (np.abs(xv).T @ np.abs(d64)) + 2.0 ** -149) + kept.T @ np.abs(d64)
    err = np.abs(gpu.download(dw).astype(np.float64) - xv.T @ d64)
    assert np.all(err <= tol), (err / tol).max()


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("fmt", [G.MXFP4, G.MXFP8])
@pytest.mark.parametrize("beside", [None, 0x3F80, 0x4049, 0x0080, 0x7F00])
def test_every_finite_bf16_value(gpu, fmt, beside, transposed):
    """All 65280 of them, as they come (blocks of 32 neighbours) or each in a block with one given value."""
    bits = np.concatenate([np.arange(0x7F80), np.arange(0x8000, 0xFF80)]).astype(np.uint16)
    if beside is None:
        bits = bits.reshape(-1, 32 * 8)
    else:
        pairs = np.zeros((bits.size, 32), np.uint16)
        pairs[:, 5], pairs[:, 20] = bits, beside
        bits = pairs.reshape(-1, 32 * 16)
    x = G.bf16_bits_to_f32(bits).astype(np.float64)
    q = gpu.zeros(x.shape, fmt)
    if transposed:
        gpu.convert_t(gpu.upload(bits.T.copy(), G.BF16), q)
    else:
        gpu.convert(gpu.upload(bits, G.BF16), q)
    code, byte, _ = X.quantize(x, fmt)
    assert np.array_equal(gpu.download(q), X.pack(code, byte, fmt))


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("fmt", [G.MXFP4, G.MXFP8])
@pytest.mark.parametrize("rows,cols", [(4100, 77), (77, 4100), (70001, 5), (5, 70001)])
def test_tall_and_wide_tensors(gpu, rows, cols, fmt, transposed):
    x = X.values(np.random.default_rng(rows), rows, cols)
    t = gpu.upload(x.T.copy() if transposed else x)
    q, back = gpu.zeros((rows, cols), fmt), gpu.empty((rows, cols))
    gpu.convert_t(t, q) if transposed else gpu.convert(t, q)
    gpu.convert(q, back)
    code, byte, want = X.quantize(x, fmt)
    assert np.array_equal(gpu.download(q), X.pack(code, byte, fmt))
    assert np.array_equal(gpu.download(back), want.astype(np.float32))
