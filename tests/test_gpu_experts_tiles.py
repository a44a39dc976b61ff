"""The experts' products in every tile that a size can take: several stages and a tail, whole tiles and edges, unequal
experts, one of them without rows, rows behind the last, against 64 bits.  Each case's comment gives the rule that picks its
kernel: `rows` are the rows in the order of the experts, `mean` those of an expert."""
import numpy as np
import pytest
import torch

from rgpu_amd import gpu as G
from tests import token_common as T

pytestmark = pytest.mark.gpu

KIND = {G.F32: torch.float32, G.BF16: torch.bfloat16, G.F16: torch.float16}


@pytest.fixture(scope="module")
def gpu():
    g = G.Gpu(0)
    yield g
    g.close()
    torch.cuda.empty_cache()


def routed(rng, tokens, k, experts):
    """(order, offsets) of choices that like some experts more, go nowhere now and then, and leave one without rows."""
    p = rng.exponential(size=experts) + 0.2
    if experts > 2:
        p[experts // 2] = 0
    ids = rng.choice(experts, size=(tokens, k), p=p / p.sum())
    if tokens > 2:
        ids[rng.uniform(size=ids.shape) < 0.02] = -1
    order, offsets, _ = T.by_expert(ids, experts)
    return order, offsets


class Case:
    """Operands on the device, and what is held of them in 64 bits."""

    def __init__(self, gpu, dtype, tokens, k, experts, K, N):
        self.gpu, self.dtype, self.K, self.N, self.experts, self.n = gpu, dtype, K, N, experts, tokens * k
        self.rng = np.random.default_rng(tokens + K)
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(tokens + N)
        order, self.offsets = routed(self.rng, tokens, k, experts)
        self.end = int(self.offsets[-1])
        self.token = torch.tensor(order // k, device="cuda")
        self.d_order, self.d_off = T.words(gpu, order), T.words(gpu, self.offsets)
        self.x, self.w = self.normal(tokens, K), self.normal(experts, K, N)
        self.rows = self.x[self.token]
        if self.end < self.n:
            self.rows[self.end:] = float("nan")  # rows that no expert has are read by nothing

    def normal(self, *shape, dtype=None):
        return torch.randn(shape, generator=self.gen, device="cuda").to(KIND[self.dtype if dtype is None else dtype])

    def held(self, t):
        torch.cuda.synchronize()
        code = next(c for c, v in KIND.items() if v == t.dtype)
        return self.gpu.wrap(t.data_ptr(), tuple(t.shape), code, owner=t)

    def seven(self, *shape, dtype=G.F32):
        return torch.full(shape, 7.0, device="cuda", dtype=KIND[dtype])

    def each(self):
        for e in range(self.experts):
            yield e, int(self.offsets[e]), int(self.offsets[e + 1])

    def gemm(self, *args, **how):
        self.gpu.experts_gemm(*args, **how)
        self.gpu.sync()


def near(got, want, size, adds, out):
    """Each of the products and additions is rounded in f32 (of six-product f32 what is left out is below one of them more),
    then the result once."""
    err = (adds + 4) * 2.0 ** -24 * size
    worst = ((got.double() - want).abs() - (err + T.HALF_STEP[out] * (want.abs() + err) + T.LEAST[out])).max().item()
    assert worst <= 0, worst


def check_nn(c, out, ordered, epi):
    bias, mask = c.normal(c.experts, c.N, dtype=G.F32), c.normal(c.n, c.N, dtype=out)
    y = c.seven(c.n, c.N, dtype=out)
    aux = {G.EPI_NONE: None, G.EPI_RELU_MASK: mask}.get(epi, bias)
    c.gemm(G.NN, c.held(c.x if ordered else c.rows), c.held(c.w), c.held(y), c.d_off, c.d_order if ordered else None, epi,
           None if aux is None else c.held(aux))
    for e, a, b in c.each():
        if a == b:
            continue
        rows, w = c.rows[a:b].double(), c.w[e].double()
        want, size = rows @ w, rows.abs() @ w.abs()
        if epi in (G.EPI_BIAS, G.EPI_BIAS_RELU):
            want, size = want + bias[e].double(), size + bias[e].double().abs()
        if epi == G.EPI_BIAS_RELU:
            want = want.clamp_min(0)
        if epi == G.EPI_RELU_MASK:
            want = want * (mask[a:b] > 0)
        near(y[a:b], want, size, c.K + 1, out)
    assert bool((y[c.end:] == 7).all())


def check_nt(c, out):
    dz, mask = c.normal(c.n, c.N), c.normal(c.n, c.K, dtype=out)
    if c.end < c.n:
        dz[c.end:] = float("nan")
    y = c.seven(c.n, c.K, dtype=out)
    c.gemm(G.NT, c.held(dz), c.held(c.w), c.held(y), c.d_off, None, G.EPI_RELU_MASK, c.held(mask))
    for e, a, b in c.each():
        if a < b:
            rows, w = dz[a:b].double(), c.w[e].double().T.contiguous()
            near(y[a:b], rows @ w * (mask[a:b] > 0), rows.abs() @ w.abs(), c.N, out)
    assert bool((y[c.end:] == 7).all())


def check_tn(c, out, ordered):
    dz = c.normal(c.n, c.N)
    if c.end < c.n:
        dz[c.end:] = float("nan")
    dw, db = c.seven(c.experts, c.K, c.N, dtype=out), c.seven(c.experts, c.N)
    c.gemm(G.TN, c.held(c.x if ordered else c.rows), c.held(dz), c.held(dw), c.d_off, c.d_order if ordered else None,
           colsum=c.held(db))
    for e, a, b in c.each():
        rows, d = c.rows[a:b].double(), dz[a:b].double()
        near(dw[e], rows.T.contiguous() @ d, rows.abs().T.contiguous() @ d.abs(), b - a + 32, out)
        near(db[e], d.sum(0), d.abs().sum(0), b - a + 32, G.F32)


HALVES = [G.BF16, G.F16]
NAMES = T.NAMES.get


# 16 bits, widths of whole 16 bytes.  256x256: 512 such tiles and mean 256 or more (57 x 9 here); 128x128 in two stages: more
# than 256 of those (31 x 9), in four: fewer (13 x 5).
@pytest.mark.parametrize("dtype", HALVES, ids=NAMES)
@pytest.mark.parametrize("tokens,k,experts,wide,deep", [(7001, 2, 5, 2056, 328), (1500, 2, 16, 1032, 200), (700, 2, 5, 584, 328),
                                                        # any width: 128x128 tiles where more than 256 (31 x 9), else 64x64
                                                        (1500, 2, 16, 1031, 203), (700, 2, 5, 583, 203)])
@pytest.mark.parametrize("f32_out", [True, False])
def test_forward_and_input_gradient_in_16_bits(gpu, dtype, tokens, k, experts, wide, deep, f32_out):
    out = G.F32 if f32_out else dtype
    c = Case(gpu, dtype, tokens, k, experts, deep, wide)
    for ordered in (True, False):
        check_nn(c, out, ordered, G.EPI_BIAS_RELU)
    check_nn(c, out, True, G.EPI_NONE)
    check_nn(c, out, True, G.EPI_RELU_MASK)
    check_nt(Case(gpu, dtype, tokens, k, experts, wide, deep), out)


# 256x256 tiles where 256 of them (9 x 5 x 6; 2 slices of 130), else 128x128: whole, in four slices (120 tiles), and
# of padded copies (odd widths, 1.25 2^30 multiply-adds) in 25 slices, in two and in one; a little less work, without copies.
@pytest.mark.parametrize("dtype", HALVES, ids=NAMES)
@pytest.mark.parametrize("tokens,k,experts,K,N", [(1500, 2, 9, 1032, 1288), (33800, 2, 130, 72, 40), (1500, 2, 9, 520, 776),
                                                  (4400, 2, 8, 264, 520), (40400, 2, 5, 203, 131), (2000, 2, 4, 515, 1027),
                                                  (900, 2, 5, 1003, 777), (800, 2, 5, 1003, 777)])
@pytest.mark.parametrize("f32_out", [True, False])
def test_weight_gradient_in_16_bits(gpu, dtype, tokens, k, experts, K, N, f32_out):
    c = Case(gpu, dtype, tokens, k, experts, K, N)
    for ordered in (True, False):
        check_tn(c, G.F32 if f32_out else dtype, ordered)


# f32, mean above 32: 128x64 where 1024 of them (64 x 16), 64x64 where 256 (34 x 8), else 64x32.
@pytest.mark.parametrize("tokens,k,experts,wide,deep", [(3900, 2, 8, 1000, 50), (1000, 2, 5, 500, 75), (1000, 2, 5, 501, 75),
                                                        (500, 2, 5, 130, 75)])
def test_forward_and_input_gradient_in_f32(gpu, tokens, k, experts, wide, deep):
    c = Case(gpu, G.F32, tokens, k, experts, deep, wide)
    for ordered in (True, False):
        check_nn(c, G.F32, ordered, G.EPI_BIAS_RELU)
    check_nn(c, G.F32, True, G.EPI_RELU_MASK)
    check_nt(Case(gpu, G.F32, tokens, k, experts, wide, deep), G.F32)


# f32 weight gradients: 64x64 tiles (300, and 150 of 128x64) in one slice; two slices of 128x64 tiles; four of 64x32, whose
# columns are whole 16 bytes or not.
@pytest.mark.parametrize("tokens,k,experts,K,N", [(1000, 2, 5, 330, 640), (4400, 2, 8, 512, 512), (3150, 2, 3, 100, 72),
                                                  (3150, 2, 3, 101, 71)])
def test_weight_gradient_in_f32(gpu, tokens, k, experts, K, N):
    c = Case(gpu, G.F32, tokens, k, experts, K, N)
    for ordered in (True, False):
        check_tn(c, G.F32, ordered)


# Up to 64 rows: of 16 bits from K 2048 on and up to 512 blocks of 64 columns, f32 always; 32 columns a block up to 128
# blocks.  2048 columns of A are held at a time.
@pytest.mark.parametrize("dtype", T.TYPES, ids=NAMES)
@pytest.mark.parametrize("tokens,k", [(1, 1), (1, 2), (4, 2), (11, 3), (32, 2)])
@pytest.mark.parametrize("K", [513, 2048, 2051, 4096, 4107])
@pytest.mark.parametrize("experts,N", [(4, 70), (30, 1029), (30, 1024), (3, 1)])
def test_few_rows(gpu, dtype, tokens, k, K, experts, N):
    c = Case(gpu, dtype, tokens, k, experts, K, N)
    for out in {G.F32, dtype}:
        for ordered, epi in ((True, G.EPI_NONE), (False, G.EPI_BIAS), (True, G.EPI_BIAS_RELU), (False, G.EPI_RELU_MASK)):
            check_nn(c, out, ordered, epi)


@pytest.mark.parametrize("dtype", T.TYPES, ids=NAMES)
@pytest.mark.parametrize("rows", [50, 300])
@pytest.mark.parametrize("wide", [72, 131])
def test_products_of_no_inner_dimension(gpu, dtype, rows, wide):
    off = T.words(gpu, [0, rows // 3, rows - 2])
    bias = np.random.default_rng(rows).normal(size=(2, wide)).astype(np.float32)
    c = gpu.upload(np.full((rows, wide), 7, np.float32))
    gpu.experts_gemm(G.NN, gpu.empty((rows, 0), dtype), gpu.empty((2, 0, wide), dtype), c, off, None, G.EPI_BIAS, gpu.upload(bias))
    want = np.full((rows, wide), 7, np.float32)
    want[:rows // 3], want[rows // 3:rows - 2] = bias
    assert np.array_equal(gpu.download(c), want)
    c = gpu.upload(np.full((rows, wide), 7, np.float32))
    gpu.experts_gemm(G.NT, gpu.empty((rows, 0), dtype), gpu.empty((2, wide, 0), dtype), c, off)
    want[:rows - 2] = 0
    assert np.array_equal(gpu.download(c), want)


# Matrices of more than 2^21 a side, f32: 128x128 register tiles, mean above 32.  Whole numbers, so sums are exact.
@pytest.mark.parametrize("ordered", [True, False])
def test_f32_matrices_of_more_than_2_21_a_side(gpu, ordered):
    rows, long = 74, (1 << 21) + 5
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    whole = lambda *s: torch.randint(-1, 2, s, generator=gen, device="cuda").float()  # noqa: E731
    held = lambda t: gpu.wrap(t.data_ptr(), tuple(t.shape), G.F32, owner=t)  # noqa: E731
    order = torch.randperm(rows, generator=gen, device="cuda")
    off, d_order = T.words(gpu, [0, 40, rows - 1]), T.words(gpu, order.cpu().numpy()) if ordered else None
    a, d, w, wt = whole(rows, long), whole(rows, 6), whole(2, long, 6), whole(2, 6, long)
    pick = a[order] if ordered else a
    c, dx, dw = (torch.full(s, 7.0, device="cuda") for s in ((rows, 6), (rows, 6), (2, long, 6)))
    torch.cuda.synchronize()
    gpu.experts_gemm(G.NN, held(a), held(w), held(c), off, d_order)
    gpu.experts_gemm(G.NT, held(a), held(wt), held(dx), off)
    gpu.experts_gemm(G.TN, held(a), held(d), held(dw), off, d_order)
    gpu.sync()
    for e, (s, t) in enumerate(((0, 40), (40, rows - 1))):
        assert torch.equal(c[s:t], (pick[s:t].double() @ w[e].double()).float())
        assert torch.equal(dx[s:t], (a[s:t].double() @ wt[e].double().T.contiguous()).float())
        assert torch.equal(dw[e], (pick[s:t].double().T.contiguous() @ d[s:t].double()).float())
    assert bool((c[rows - 1] == 7).all()) and bool((dx[rows - 1] == 7).all())


@pytest.mark.parametrize("dtype", T.TYPES, ids=NAMES)
@pytest.mark.parametrize("tokens,k,experts,K,N", [(4, 2, 3, 2100, 70), (40, 2, 8, 100, 72), (130, 2, 3, 136, 264), (130, 2, 3, 133, 131),
                                                  (1500, 2, 4, 75, 501), (1500, 2, 4, 200, 1032)])
def test_infinities_and_nan_stay_in_their_rows(gpu, dtype, tokens, k, experts, K, N):
    """An infinity or NaN in a row of A or a matrix: what 64 bits give, and the other rows and experts as without it."""
    c = Case(gpu, dtype, tokens, k, experts, K, N)
    c.x[0, 3], c.x[tokens // 2, K - 1], c.x[tokens - 1, 0] = float("inf"), float("nan"), -float("inf")
    c.rows = c.x[c.token]
    c.w[0, 5, 1] = float("inf")
    dz = c.normal(c.n, N)
    y, dw = c.seven(c.n, N), c.seven(experts, K, N)
    c.gemm(G.NN, c.held(c.x), c.held(c.w), c.held(y), c.d_off, c.d_order)
    c.gemm(G.TN, c.held(c.x), c.held(dz), c.held(dw), c.d_off, c.d_order)
    for e, a, b in c.each():
        rows, w, d = c.rows[a:b].double(), c.w[e].double(), dz[a:b].double()
        for got, m, o, adds in ((y[a:b], rows, w, K), (dw[e], rows.T.contiguous(), d, b - a + 32)):
            if 0 in got.shape:
                continue
            want = m @ o
            on = want.isfinite()
            assert torch.equal(torch.where(on, 0.0, got.double()).nan_to_num(7.0, 8.0, 9.0),
                               torch.where(on, 0.0, want).nan_to_num(7.0, 8.0, 9.0))
            near(torch.where(on, got, 0.0), torch.where(on, want, 0.0),
                 torch.where(on, m.abs().nan_to_num(0, 0, 0) @ o.abs().nan_to_num(0, 0, 0), 0.0), adds, G.F32)
