"""Every kind of call on wrapped tensors that start on any element of the caller's memory, with NaN before and behind them:
the same results as on the library's own buffers, and nothing written beside the tensor."""
import numpy as np
import pytest
import torch

from rgpu_amd import gpu as G

pytestmark = pytest.mark.gpu

TORCH = {G.F32: torch.float32, G.BF16: torch.bfloat16, G.F16: torch.float16, G.U32: torch.int32}
PAD = 64


@pytest.fixture(scope="module")
def gpu():
    g = G.Gpu(0)
    yield g
    g.close()


class Odd:
    """Makes wrapped copies `shift` elements into their memory, and looks at what lies around them afterwards."""

    def __init__(self, gpu, shift):
        self.gpu, self.shift, self.made = gpu, shift, []

    def __call__(self, a, dtype=G.F32):
        a = np.asarray(a)
        t = torch.full((a.size + 2 * PAD,), float("nan") if dtype != G.U32 else -1, dtype=TORCH[dtype], device="cuda")
        at = slice(PAD + self.shift, PAD + self.shift + a.size)
        t[at] = torch.from_numpy(a.astype(np.int32 if dtype == G.U32 else np.float32).reshape(-1)).to(t)
        torch.cuda.synchronize()
        self.made.append((t, at))
        return self.gpu.wrap(t[at].data_ptr(), a.shape, dtype, owner=t)

    def check(self):
        self.gpu.sync()
        for t, at in self.made:
            rest = torch.cat([t[:at.start], t[at.stop:]])
            assert bool((rest == -1).all() if t.dtype == torch.int32 else rest.isnan().all())


def both(gpu, shift, call, ins, outs):
    """call(inputs..., outputs...) on buffers of the library and on wrapped ones; ins and outs: (array, dtype)."""
    odd = Odd(gpu, shift)
    got = []
    for make in (lambda a, t: gpu.upload(a, t), odd):
        i, o = [make(a, t) for a, t in ins], [make(a, t) for a, t in outs]
        call(*i, *o)
        got.append([gpu.download_f32(t) if t.dtype != G.U32 else gpu.download(t).astype(np.float64) for t in o])
    odd.check()
    return got


SIZES = [(1, 1, 1), (3, 5, 7), (37, 64, 10), (64, 128, 128), (100, 96, 130), (256, 512, 256), (300, 257, 131), (512, 1024, 512)]


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("dtype", [G.F32, G.BF16, G.F16])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_products(gpu, M, K, N, dtype, shift):
    rng = np.random.default_rng(M + K + N)
    draw = lambda *s: rng.normal(size=s).astype(np.float32)
    as_held = {G.F32: lambda a: a, G.BF16: lambda a: G.bf16_bits_to_f32(G.f32_to_bf16_bits(a)),
               G.F16: lambda a: a.astype(np.float16).astype(np.float32)}[dtype]
    bias, mask = draw(1, N), draw(M, N)
    for out in (G.F32,) if dtype == G.F32 else (G.F32, G.BF16):
        for layout, sa, sb in ((G.NN, (M, K), (K, N)), (G.TN, (K, M), (K, N)), (G.NT, (M, K), (N, K))):
            a, b = as_held(draw(*sa)), as_held(draw(*sb))
            wide = [m.astype(np.float64) for m in (a, b)]
            wide = [wide[0].T if layout == G.TN else wide[0], wide[1].T if layout == G.NT else wide[1]]
            full, size = wide[0] @ wide[1], np.abs(wide[0]) @ np.abs(wide[1])
            for epi, aux in ((G.EPI_NONE, None), (G.EPI_BIAS, (bias, G.F32)), (G.EPI_BIAS_RELU, (bias, G.F32)),
                             (G.EPI_RELU_MASK, (mask, out))):
                cs = layout == G.TN and epi == G.EPI_NONE

                def call(x, y, *rest):
                    rest = list(rest)
                    u = rest.pop(0) if aux else None
                    gpu.gemm(layout, x, y, rest[0], epi, u, rest[1] if cs else None)

                ins = [(a, dtype), (b, dtype)] + ([aux] if aux else [])
                outs = [(np.zeros((M, N), np.float32), out)] + ([(np.zeros((1, N), np.float32), G.F32)] if cs else [])
                want = full + bias if epi in (G.EPI_BIAS, G.EPI_BIAS_RELU) else full
                want = np.maximum(want, 0) if epi == G.EPI_BIAS_RELU else want
                if epi == G.EPI_RELU_MASK:  # as the mask's type holds it: no value rounds to zero
                    want = np.where(mask > 0, want, 0)
                # f32 additions (six products an element where f32 goes in as planes), and one rounding to bf16
                tol = (6 * K + 40) * 2.0 ** -23 * (size + np.abs(bias)) + (2.0 ** -8 * np.abs(want) if out == G.BF16 else 0)
                for got in both(gpu, shift, call, ins, outs):
                    assert np.all(np.abs(got[0] - want) <= tol), (layout, epi, out)
                    if cs:
                        b64 = b.astype(np.float64)
                        assert np.all(np.abs(got[1] - b64.sum(0)) <= (K + 8) * 2.0 ** -23 * np.abs(b64).sum(0))


@pytest.mark.parametrize("shift", [1, 2])
@pytest.mark.parametrize("dtype", [G.F32, G.BF16, G.F16])
@pytest.mark.parametrize("K,M,N,slices", [(1000, 60, 130, 3), (2048, 128, 64, 8), (4100, 64, 16, 16)])
def test_split_products_and_backward(gpu, K, M, N, slices, dtype, shift):
    rng = np.random.default_rng(K + M)
    hold = {G.F32: np.float32, G.BF16: None, G.F16: np.float16}[dtype]
    held = lambda a: (G.bf16_bits_to_f32(G.f32_to_bf16_bits(a)) if hold is None else a.astype(hold).astype(np.float32))
    a, b, w = (held(rng.normal(size=s).astype(np.float32)) for s in ((K, M), (K, N), (M, N)))
    a64, b64, w64 = (m.astype(np.float64) for m in (a, b, w))
    want, size = a64.T @ b64, np.abs(a64).T @ np.abs(b64)
    tol = (6 * K + 40) * 2.0 ** -23 * size
    sums, sums_tol = b64.sum(0), (K + 8) * 2.0 ** -23 * np.abs(b64).sum(0)
    zeros = lambda *s: (np.zeros(s, np.float32), G.F32)
    for got in both(gpu, shift, lambda x, y, p, c, s: gpu.split_k(x, y, c, p, slices, True, colsum=s),
                    [(a, dtype), (b, dtype), zeros(slices * (M * N + N))], [zeros(M, N), zeros(1, N)]):
        assert np.all(np.abs(got[0] - want) <= tol) and np.all(np.abs(got[1] - sums) <= sums_tol)
    for got in both(gpu, shift, lambda x, d, v, dx, dw, db: gpu.linear_backward(x, d, v, dx, dw, db),
                    [(a, dtype), (b, dtype), (w, dtype)], [zeros(K, M), zeros(M, N), zeros(1, N)]):
        assert np.all(np.abs(got[1] - want) <= tol) and np.all(np.abs(got[2] - sums) <= sums_tol)
        assert np.all(np.abs(got[0] - b64 @ w64.T) <= (6 * N + 40) * 2.0 ** -23 * (np.abs(b64) @ np.abs(w64).T))


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 10), (65, 130), (200, 1000), (40, 2304)])
def test_rows_columns_and_elements(gpu, rows, cols, shift):
    """Kernels whose results do not depend on alignment: the same bits."""
    rng = np.random.default_rng(rows + cols)
    x, y = rng.normal(size=(rows, cols)).astype(np.float32), rng.normal(size=(rows, cols)).astype(np.float32)
    row, one = rng.normal(size=(1, cols)).astype(np.float32), np.zeros((1,), np.float32)
    labels, target = rng.integers(0, cols, rows), np.abs(y) / np.abs(y).sum(1, keepdims=True)
    f = lambda a: (a, G.F32)
    u, v = f(x), f(y)
    cases = [(lambda a, o: gpu.relu(a, o), [u], [v]), (lambda a, o: gpu.relu_bwd(a, o), [u], [v]),
             (lambda b, o: gpu.bias_add(o, b), [f(row)], [u]),
             (lambda a, o: gpu.map("exp", a, o), [u], [v]), (lambda g, a, o: gpu.map_vjp("relu", g, a, None, o), [u, v], [u]),
             (lambda a, b, o: gpu.zip("mul", a, b, o), [u, v], [u]), (lambda a, b, o: gpu.zip("add", a, b, o), [u, f(row)], [u]),
             (lambda a, o: gpu.reduce_to(a, o), [u], [f(row)]), (lambda a, o: gpu.sum_all(a, o, 3.0), [u], [f(one)]),
             (lambda s, a, o: gpu.fill_scaled(s, o, 2.0, a), [f(row[0, :1]), u], [v]),
             (lambda a, o: gpu.softmax_rows(a, o), [u], [v]), (lambda a, b, o: gpu.softmax_rows_vjp(a, b, o), [u, v], [u]),
             (lambda a, l, d, r: gpu.softmax_xent(a, l, d, r), [u, (labels, G.U32)], [v, f(np.zeros(rows, np.float32))]),
             (lambda a, o: gpu.argmax_rows(a, o), [u], [(labels, G.U32)]),
             (lambda a, t, o, d: gpu.loss(G.LOSS_SOFTMAX_XENT_LOGITS, a, t, o, d), [u, f(target)], [f(one), v])]
    for half in (G.BF16, G.F16):
        cases += [(lambda a, o: gpu.convert(a, o), [u], [(y, half)]), (lambda a, o: gpu.convert(a, o), [(x, half)], [v]),
                  (lambda a, o: gpu.relu_bwd(a, o), [(x, half)], [v])]
    for i, (call, ins, outs) in enumerate(cases):
        plain, odd = both(gpu, shift, call, ins, outs)
        for p, q in zip(plain, odd):
            assert np.array_equal(p, q, equal_nan=True), i
    # column sums: other loads, the same order of additions
    for dtype in (G.F32, G.BF16, G.F16):
        plain, odd = both(gpu, shift, lambda a, o: gpu.colsum(a, o), [(x, dtype)], [f(row)])
        assert np.array_equal(plain[0], odd[0])


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("n", [1, 5, 1000, 4099, 300000])
def test_optimizers(gpu, n, shift):
    rng = np.random.default_rng(n)
    w, m, g = (rng.normal(size=n).astype(np.float32) for _ in range(3))
    v = np.abs(rng.normal(size=n)).astype(np.float32)
    f = lambda a: (a, G.F32)
    for call, ins, outs in (
            (lambda d, a, b, c: gpu.adam(a, b, c, d, 1e-3, t=3), [f(g)], [f(w), f(m), f(v)]),
            (lambda d, a, b, c: gpu.adam_many([a], [b], [c], [d], 1e-3, t=3), [f(g)], [f(w), f(m), f(v)]),
            (lambda d, a, b: gpu.sgd(a, d, 0.1, 0.9, b), [f(g)], [f(w), f(m)]),
            (lambda d, a: gpu.sgd_many([a], [d], 0.1), [f(g)], [f(w)])):
        plain, odd = both(gpu, shift, call, ins, outs)
        assert all(np.array_equal(p, q) for p, q in zip(plain, odd))


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("dtype", [G.F32, G.BF16, G.F16])
@pytest.mark.parametrize("rows,k,n", [(1, 7, 3), (37, 130, 64), (70, 256, 129), (300, 1003, 1000)])
def test_microscaled(gpu, rows, k, n, dtype, shift):
    """Values, bias, outputs and gradients on any element; the packed tensors are the library's.  The same bits, as every
    path adds in the same order (the gradient's tile goes by the alignment of δ: see the tolerance)."""
    rng = np.random.default_rng(rows + k)
    x, w, d = (rng.normal(size=s).astype(np.float32) for s in ((rows, k), (k, n), (rows, n)))
    q, w4 = gpu.empty((rows, k), G.MXFP8), gpu.empty((n, k), G.MXFP4)
    f = lambda a, t=G.F32: (a, t)
    held = []
    for fmt in (G.MXFP4, G.MXFP8):
        a, at = gpu.empty((rows, k), fmt), gpu.empty((k, rows), fmt)

        def convert(v, back):
            gpu.convert(v, a)
            gpu.convert(a, back)
            held.append(gpu.download_f32(a))
            gpu.convert_t(v, at)
            held.append(gpu.download_f32(at))

        plain, odd = both(gpu, shift, convert, [f(x, dtype)], [f(np.zeros_like(x), dtype)])
        assert np.array_equal(plain[0], odd[0])
        assert np.array_equal(held[-4], held[-2]) and np.array_equal(held[-3], held[-1])
    gpu.convert(gpu.upload(x), q)
    gpu.convert_t(gpu.upload(w), w4)
    for out in (G.F32, G.BF16):
        plain, odd = both(gpu, shift, lambda b, c: gpu.gemm(G.NT, q, w4, c, G.EPI_BIAS_RELU, b), [f(d[:1])],
                          [f(np.zeros((rows, n), np.float32), out)])
        assert np.array_equal(plain[0], odd[0])
    x64 = gpu.download_f32(q).astype(np.float64)
    d64 = {G.F32: d, G.BF16: G.bf16_bits_to_f32(G.f32_to_bf16_bits(d)), G.F16: d.astype(np.float16)}[dtype].astype(np.float64)
    for got in both(gpu, shift, lambda v, c, s: gpu.matmul_at_b(q, v, c, colsum=s), [f(d, dtype)],
                    [f(np.zeros((k, n), np.float32)), f(np.zeros((1, n), np.float32))]):
        assert np.all(np.abs(got[0] - x64.T @ d64) <= (3 * rows + 40) * 2.0 ** -23 * (np.abs(x64).T @ np.abs(d64)))
        assert np.all(np.abs(got[1] - d64.sum(0)) <= (rows + 8) * 2.0 ** -23 * np.abs(d64).sum(0))
    plain, odd = both(gpu, shift, lambda v: gpu.relu_bwd(q, v), [], [f(np.resize(d, (rows, k)))])
    assert np.array_equal(plain[0], odd[0])
    plain, odd = both(gpu, shift, lambda g, v: gpu.map_vjp("relu", g, q, None, v), [f(np.resize(d, (rows, k)))], [f(x)])
    assert np.array_equal(plain[0], odd[0])
