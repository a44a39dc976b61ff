"""The product of microscaled tensors where its kernels could answer differently: its two output types."""
import numpy as np
import pytest

from rgpu_amd import gpu as G
from tests import mx_common as X

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    g = G.Gpu(0)
    yield g
    g.close()


def mx_upload(gpu, x, fmt):
    code, byte, values = X.quantize(x, fmt)
    return gpu.upload(X.pack(code, byte, fmt), fmt, x.shape), values


@pytest.mark.parametrize("fa", [G.MXFP4, G.MXFP8])
@pytest.mark.parametrize("M,N,K", [(1, 33, 500), (48, 100, 129), (49, 130, 1000), (64, 64, 1030), (300, 257, 640),
                                   (1500, 1800, 260), (1000, 4100, 130)])
def test_a_bf16_product_is_the_f32_one_rounded(gpu, M, N, K, fa):
    rng = np.random.default_rng(M + N + K)
    a, _ = mx_upload(gpu, X.values(rng, M, K), fa)
    b, _ = mx_upload(gpu, X.values(rng, N, K, spread=0.3), G.MXFP4)
    bias = gpu.upload(rng.normal(size=(1, N)).astype(np.float32))
    full, half = gpu.empty((M, N)), gpu.empty((M, N), G.BF16)
    for epi in (G.EPI_NONE, G.EPI_BIAS_RELU):
        gpu.gemm(G.NT, a, b, full, epi, bias if epi else None)
        gpu.gemm(G.NT, a, b, half, epi, bias if epi else None)
        assert np.array_equal(gpu.download(half), G.f32_to_bf16_bits(gpu.download(full)))


@pytest.mark.parametrize("M", [3, 60, 300, 2000])
def test_a_bf16_product_keeps_small_neighbours(gpu, M):
    """Large products that cancel beside small ones: the small ones are what is left."""
    rng = np.random.default_rng(M)
    x = np.zeros((M, 256))
    x[:, 0::8], x[:, 1::8] = 448, -448
    x[:, 2:8] = np.ldexp(1.0, rng.integers(-9, -4, size=(M, 6)))
    w = np.ones((1700, 256))
    a, av = mx_upload(gpu, x, G.MXFP8)
    b, bv = mx_upload(gpu, w, G.MXFP4)
    c = gpu.empty((M, 1700), G.BF16)
    gpu.gemm(G.NT, a, b, c)
    # every sum is a multiple of 2^-9 below 2^8, so f32 holds it on its way; bf16 rounds it by 2^-8 of itself at most
    want = av @ bv.T
    assert np.all(want > 0) and np.all(np.abs(gpu.download_f32(c) - want) <= 2.0 ** -8 * np.abs(want))
