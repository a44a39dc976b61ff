"""The product of microscaled tensors where its kernels could answer differently: its two output types, the
edges of its largest tile, scales of any size."""
import os

import numpy as np
import pytest
import torch

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


def exact64(av, bv, bias=None):
    """A·Bᵀ + b and the sums of the sizes of its terms, in 64 bits on the device."""
    a, b = torch.from_numpy(av).cuda(), torch.from_numpy(bv).cuda()
    want, size = a @ b.T.contiguous(), a.abs() @ b.abs().T.contiguous()
    if bias is not None:
        c = torch.from_numpy(bias.astype(np.float64)).cuda()
        want, size = want + c, size + c.abs()
    return want.cpu().numpy(), size.cpu().numpy()


@pytest.mark.parametrize("M,N,K", [(4090, 4090, 300), (4090, 4088, 1300), (4090, 4093, 100), (4095, 4096, 640),
                                   (65500, 250, 260), (250, 65500, 130)])
def test_edges_of_the_256_tile(gpu, M, N, K):
    """Rows past M and N, scale groups past the end, K of fewer steps than stages and of no multiple of them."""
    # the sizes are ones that the dispatch sends to that tile; if its rule changes, so must they
    tiles = -(-M // 256) * -(-N // 256)
    places = -(-tiles // 256) * 256
    source = open(os.path.join(os.path.dirname(G.__file__), "csrc", "mx_gemm.hip")).read()
    assert "if (t >= 256 && 2 * places <= 3 * t) return launch_tiles<4, 256, 256," in source
    assert tiles >= 256 and 2 * places <= 3 * tiles
    rng = np.random.default_rng(M + K)
    a, av = mx_upload(gpu, X.values(rng, M, K), G.MXFP4)
    b, bv = mx_upload(gpu, X.values(rng, N, K, spread=0.3), G.MXFP4)
    bias = rng.normal(size=(1, N)).astype(np.float32)
    gb = gpu.upload(bias)
    want, size = exact64(av, bv, bias)
    guard = torch.full((M * N + 512,), float("nan"), device="cuda")
    torch.cuda.synchronize()
    c = gpu.wrap(guard.data_ptr() + 1024, (M, N), owner=guard)
    gpu.gemm(G.NT, a, b, c, G.EPI_BIAS, gb)
    # K + 1 additions in f32, each off by at most one unit in the last place of what is summed so far
    tol = (K + 8) * 2.0 ** -23 * size
    assert np.all(np.abs(gpu.download(c).astype(np.float64) - want) <= tol)
    assert bool(guard[:256].isnan().all()) and bool(guard[256 + M * N:].isnan().all())
    half = gpu.upload(np.full((M, N), 7.0, np.float32), G.BF16)
    gpu.gemm(G.NT, a, b, half, G.EPI_BIAS_RELU, gb)
    want = np.maximum(want, 0)
    assert np.all(np.abs(gpu.download_f32(half).astype(np.float64) - want) <= tol + 2.0 ** -8 * (want + tol))


@pytest.mark.parametrize("fa", [G.MXFP4, G.MXFP8])
@pytest.mark.parametrize("M", [5, 60, 300, 4096])
def test_scales_of_any_size(gpu, M, fa):
    """Blocks from 2^-100 to 2^100 in the rows of A, their inverses in B: every product is near one."""
    rng = np.random.default_rng(M)
    N, K = (4096 if M == 4096 else 150), 200
    e = rng.integers(-100, 101, size=-(-K // 32)).repeat(32)[:K]
    x, w = np.ldexp(rng.normal(size=(M, K)), e), np.ldexp(rng.normal(size=(N, K)), -e)
    a, av = mx_upload(gpu, x.astype(np.float32), fa)
    b, bv = mx_upload(gpu, w.astype(np.float32), G.MXFP4)
    c = gpu.empty((M, N))
    gpu.gemm(G.NT, a, b, c)
    want, size = exact64(av, bv)
    assert np.all(np.abs(gpu.download(c).astype(np.float64) - want) <= (K + 8) * 2.0 ** -23 * size)
