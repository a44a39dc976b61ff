"""Operators of layers that learn from tokens, as cases that can be timed and compared: their plain forms in elementary torch
operations, or, where ``own`` is true, the calls that a program makes of this package.

Kinds
-----
embed    rows of a table looked up by token and scaled; for training also the table's gradient: the rows of dy added up for
         each token, whole table out.  A token of all ones (-1 as a 32-bit whole number) is padding: a row of zeros, no
         gradient.
dropout  y = x m / (1 - q) and, with the same mask m, dx = dy m / (1 - q).  The mask comes from the numbers of the elements
         alone: Philox4x32 with 10 rounds (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011), key = the
         seed's two words, counter = (low and high word of i // 8, low and high word of the draw); element i takes the
         (i % 8)-th 16 bits of the four words (low half first) and is dropped where they are below 65536 q, a whole number.
route    tokens to experts: scores s = softmax or sigmoid of the logits; the choice goes by s + bias (64 bits: two of them
         are often next to each other) among the experts of the kept groups, a group's rank being the sum of its two
         greatest; weights are the chosen scores, divided by their sum if renormalised, times a scale.  For training also
         the gradient of the logits.
experts  the products of the experts that the tokens were routed to.
         "serve": y = sum over the choices j of w_j (relu(x W1 + b1) W2 + b2) with the chosen expert's weights.
         "train": its backward pass in f32: every gradient from dy and what the forward pass kept, h = relu(x W1 + b1) and
         o = h W2 + b2 in the order of the experts.
         "products": one layer of a bf16 or f16 step: relu(x W + b) for each token and choice, in the order of the experts,
         and from the gradient dz of such rows dW, db and dx (summed over a token's choices).
"""
import math

import torch

own = False

# ------------------------------------------------------------------ the cases

_LISTED = [
    # Some tokens of a request: latency.
    {"name": "embed_serve_64", "kind": "embed", "train": False, "dtype": "bf16", "vocab": 32768, "dim": 1024,
     "tokens": 64, "padded": False},
    # A training batch over a large vocabulary: tokens as frequent as words are, a few of them most of the batch.
    {"name": "embed_train_65536", "kind": "embed", "train": True, "dtype": "bf16", "vocab": 131072, "dim": 1024,
     "tokens": 65536, "padded": True},
    # A small vocabulary and an odd width, f16.
    {"name": "embed_train_odd", "kind": "embed", "train": True, "dtype": "f16", "vocab": 1003, "dim": 777,
     "tokens": 5000, "padded": True},
    # The small model's hidden layer at batch 32.
    {"name": "dropout_32x1024_f32", "kind": "dropout", "dtype": "f32", "rows": 32, "cols": 1024, "drop": 32768,
     "seed": 7, "draw": 3},
    # The wide layer's activations at the batch that it is trained on.
    {"name": "dropout_8192x4096", "kind": "dropout", "dtype": "bf16", "rows": 8192, "cols": 4096, "drop": 6554,
     "seed": 123456789012345, "draw": 5000000000},
    # One token's choice of experts.
    {"name": "route_1x64", "kind": "route", "train": False, "dtype": "f32", "tokens": 1, "experts": 64, "k": 4,
     "score": "softmax", "groups": 1, "kept": 1, "bias": False, "renormalise": True, "scale": 1.0, "masked": False},
    # A batch of tokens over few experts, as a bf16 product leaves their logits; some experts switched off.
    {"name": "route_train_2048x16", "kind": "route", "train": True, "dtype": "bf16", "tokens": 2048, "experts": 16, "k": 2,
     "score": "softmax", "groups": 1, "kept": 1, "bias": False, "renormalise": False, "scale": 1.0, "masked": True},
    # Many experts in groups, balanced by a bias.
    {"name": "route_train_16384x256", "kind": "route", "train": True, "dtype": "f32", "tokens": 16384, "experts": 256,
     "k": 8, "score": "sigmoid", "groups": 8, "kept": 4, "bias": True, "renormalise": True, "scale": 2.5, "masked": False},
    # Four tokens through wide experts: the chosen experts' weights are the work.
    {"name": "experts_serve_4", "kind": "experts", "mode": "serve", "dtype": "bf16", "tokens": 4, "experts": 16, "k": 2,
     "din": 1024, "dout": 4096},
    # The small model's batch and width, the backward pass in f32.
    {"name": "experts_train_2048_f32", "kind": "experts", "mode": "train", "dtype": "f32", "tokens": 2048, "experts": 8,
     "k": 2, "din": 1024, "dout": 1024},
    # Sizes that are multiples of nothing, f16.
    {"name": "experts_odd_f16", "kind": "experts", "mode": "products", "dtype": "f16", "tokens": 1500, "experts": 5,
     "k": 2, "din": 1003, "dout": 777},
    # A wide layer's training step over many experts.
    {"name": "experts_bf16_8192", "kind": "experts", "mode": "products", "dtype": "bf16", "tokens": 8192, "experts": 32,
     "k": 4, "din": 2048, "dout": 2048},
]


def listed():
    return [dict(c) for c in _LISTED]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of the range: half of them multiples of 64 (as layers are mostly chosen), the others any number."""
    n = _log(rng, lo, hi)
    return min(hi, max(64, (n + 32) // 64 * 64)) if rng.random() < 0.5 else n


def draw(rng):
    kind = rng.choice(["embed", "embed", "dropout", "route", "route", "experts", "experts"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if kind == "embed":
        dim = _size(rng, 16, 4096)
        return {"kind": kind, "train": rng.random() < 0.7, "dtype": dtype, "vocab": _log(rng, 64, min(131072, (1 << 27) // dim)),
                "dim": dim, "tokens": _log(rng, 1, min(65536, (1 << 26) // dim)), "padded": rng.random() < 0.5}
    if kind == "dropout":
        return {"kind": kind, "dtype": dtype, "rows": _size(rng, 1, 8192), "cols": _size(rng, 10, 4096),
                "drop": rng.choice([6554, 13107, 32768, rng.randrange(1, 65536)]), "seed": rng.randrange(1 << 63),
                "draw": rng.randrange(1 << 40)}
    if kind == "route":
        experts = rng.choice([_log(rng, 4, 256), 8, 64, 128, 256])
        # Groups go with a bias.  (Without one, sums of two scores of a few bits may agree in 64 bits by their roundings only.)
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if experts % g == 0 and experts // g >= 2])
        kept = rng.randint(1, groups)
        return {"kind": kind, "train": rng.random() < 0.6, "dtype": dtype, "tokens": _log(rng, 1, 16384),
                "experts": experts, "k": rng.randint(1, min(8, experts // groups * kept)),
                "score": rng.choice(["softmax", "sigmoid"]), "groups": groups, "kept": kept, "bias": groups > 1 or rng.random() < 0.5,
                "renormalise": rng.random() < 0.6, "scale": rng.choice([1.0, 2.5]), "masked": groups == 1 and rng.random() < 0.3}
    experts = _log(rng, 2, 64)
    mode = rng.choice(["serve", "train" if dtype == "f32" else "products"])
    return {"kind": kind, "mode": mode, "dtype": dtype, "tokens": _log(rng, 1, 8192 if mode != "train" else 2048),
            "experts": experts, "k": rng.randint(1, min(4, experts)), "din": _size(rng, 64, 1024), "dout": _size(rng, 64, 1024)}


_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------ the plain form

def _mulhilo(a, m):
    """The high and the low 32 bits of a m, for whole numbers below 2^32 held in 64 bits."""
    low, high = (a & 0xffff) * m, (a >> 16) * m
    low = low + ((high & 0xffff) << 16)
    return (high >> 16) + (low >> 32), low & 0xffffffff


def _keep(n, drop, seed, draw_, device):
    """The mask of n elements."""
    i = torch.arange(-(-n // 8), dtype=torch.int64, device=device)
    c = [i & 0xffffffff, i >> 32, torch.full_like(i, draw_ & 0xffffffff), torch.full_like(i, draw_ >> 32)]
    k0, k1 = seed & 0xffffffff, seed >> 32
    for _ in range(10):
        hi0, lo0 = _mulhilo(c[0], 0xD2511F53)
        hi1, lo1 = _mulhilo(c[2], 0xCD9E8D57)
        c = [hi1 ^ c[1] ^ k0, lo1, hi0 ^ c[3] ^ k1, lo0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xffffffff, (k1 + 0xBB67AE85) & 0xffffffff
    words = torch.stack(c, dim=1)
    halves = torch.stack([words & 0xffff, words >> 16], dim=2).reshape(-1)[:n]
    return halves >= drop


def _scores(x, case):
    """The scores of the logits (a row of nothing but -inf has scores of zero)."""
    if case["score"] == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    top = x.amax(dim=1, keepdim=True)
    e = torch.exp(x - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = e.sum(dim=1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total))


def _plain_route(s):
    case = s["case"]
    x = s["logits"].double()
    score = _scores(x, case)
    choice = score + s["bias"].double() if case["bias"] else score
    t, e, g = x.shape[0], x.shape[1], case["groups"]
    if case["kept"] < g:
        grouped = choice.reshape(t, g, e // g)
        rank = torch.sort(grouped, dim=2, descending=True).values[:, :, :2].sum(dim=2)
        kept = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :case["kept"]]
        on = (kept[:, :, None] == torch.arange(g, device=x.device)).any(dim=1)
        choice = torch.where(on[:, :, None], grouped, torch.full_like(grouped, -math.inf)).reshape(t, e)
    ids = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, :case["k"]]
    chosen = torch.gather(score, 1, ids)
    total = chosen.sum(dim=1, keepdim=True) if case["renormalise"] else torch.ones_like(chosen[:, :1])
    total = torch.where(total > 0, total, torch.ones_like(total))
    weights = case["scale"] * chosen / total
    out = {"ids": ids.int(), "weights": weights.float()}
    if case["train"]:
        g_ = s["dweights"].double()
        ds = case["scale"] * g_ / total
        if case["renormalise"]:
            ds = ds - (ds * chosen).sum(dim=1, keepdim=True) / total
        if case["score"] == "sigmoid":
            dx = torch.zeros_like(x).scatter(1, ids, chosen * (1 - chosen) * ds)
        else:
            dx = torch.zeros_like(x).scatter(1, ids, chosen * ds) - score * (chosen * ds).sum(dim=1, keepdim=True)
        out["dlogits"] = dx.to(s["logits"].dtype)
    return out


def _by_expert(ids, experts):
    """The (token, choice) pairs in the order of their experts, each one's expert, and its place among that expert's."""
    flat = ids.reshape(-1).long()
    order = torch.sort(flat, stable=True).indices
    of = flat[order]
    counts = (flat[:, None] == torch.arange(experts, device=ids.device)).sum(dim=0)
    first = counts.cumsum(0) - counts
    return order, of, torch.arange(flat.numel(), device=ids.device) - first[of], int(counts.max())


def _padded(rows, of, place, experts, most):
    """Rows in the order of their experts as [experts, most, ...], zeros behind each expert's."""
    out = torch.zeros(experts, most, rows.shape[1], device=rows.device)
    out[of, place] = rows
    return out


def _plain_experts(s):
    case = s["case"]
    k, e, t = case["k"], case["experts"], case["tokens"]
    order, of, place, most = _by_expert(s["ids"], e)
    x = s["x"].float()
    xp = _padded(x[order // k], of, place, e, most)

    def back(rows):
        """Rows in the order of their experts as [tokens, k, ...]."""
        out = torch.empty_like(rows)
        out[order] = rows
        return out.reshape(t, k, -1)

    w1, b1 = s["w1"].float(), s["b1"]
    if case["mode"] == "train":
        w2, w, dy = s["w2"], s["weights"], s["dy"]
        hp = _padded(s["h"], of, place, e, most)
        do = (dy[:, None] * w[:, :, None]).reshape(t * k, -1)[order]
        dop = _padded(do, of, place, e, most)
        dhp = torch.bmm(dop, w2.transpose(1, 2).contiguous()) * (hp > 0)
        dx = torch.bmm(dhp, w1.transpose(1, 2).contiguous())[of, place]
        return {"dx": back(dx).sum(dim=1), "dweights": (dy[:, None] * back(s["o"])).sum(dim=2),
                "dw1": torch.bmm(xp.transpose(1, 2).contiguous(), dhp), "db1": dhp.sum(dim=1),
                "dw2": torch.bmm(hp.transpose(1, 2).contiguous(), dop), "db2": dop.sum(dim=1)}
    hp = torch.relu(torch.bmm(xp, w1) + b1[:, None])
    if case["mode"] == "products":
        dzp = _padded(s["dz"].float(), of, place, e, most)
        dx = torch.bmm(dzp, w1.transpose(1, 2).contiguous())[of, place]
        dtype = s["x"].dtype
        return {"rows": hp[of, place].to(dtype), "dw": torch.bmm(xp.transpose(1, 2).contiguous(), dzp), "db": dzp.sum(dim=1),
                "dx": back(dx).sum(dim=1).to(dtype)}
    w2, b2, w = s["w2"].float(), s["b2"], s["weights"]
    o = back((torch.bmm(hp, w2) + b2[:, None])[of, place])
    return {"y": (o * w[:, :, None]).sum(dim=1).to(s["x"].dtype)}


def _plain(s):
    case = s["case"]
    if case["kind"] == "route":
        return _plain_route(s)
    if case["kind"] == "experts":
        return _plain_experts(s)
    t = _TORCH[case["dtype"]]
    if case["kind"] == "dropout":
        keep = _keep(s["x"].numel(), case["drop"], case["seed"], case["draw"], s["x"].device).reshape(s["x"].shape)
        scale = 65536 / (65536 - case["drop"])
        zero = torch.zeros((), device=keep.device)
        return {"y": torch.where(keep, s["x"].float() * scale, zero).to(t),
                "dx": torch.where(keep, s["dy"].float() * scale, zero).to(t)}
    on = (s["ids"] >= 0)[:, None]
    ids = s["ids"].clamp_min(0).long()
    out = {"y": (s["table"][ids].float() * on * s["scale"]).to(t)}
    if case["train"]:
        dtable = torch.zeros(case["vocab"], case["dim"], device=ids.device)
        out["dtable"] = dtable.index_add_(0, ids, s["dy"].float() * on) * s["scale"]
    return out


# ------------------------------------------------------------------ inputs (from the seed alone)

def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))

    def normal(shape, scale=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * scale

    def uniform(shape):
        return torch.rand(shape, generator=gen, device="cuda", dtype=torch.float64)

    t = _TORCH[case["dtype"]]
    if case["kind"] == "embed":
        # The n-th most frequent token 1/n as frequent as the first, the tokens' numbers in no order.
        nth = torch.exp(uniform(case["tokens"]) * math.log(case["vocab"] + 1)).long() - 1
        ids = torch.randperm(case["vocab"], generator=gen, device="cuda")[nth.clamp(0, case["vocab"] - 1)]
        if case["padded"]:
            ids[uniform(case["tokens"]) < 0.05] = -1
        v = {"table": normal((case["vocab"], case["dim"]), case["dim"] ** -0.5).to(t), "ids": ids.int(),
             "scale": math.sqrt(case["dim"])}
        if case["train"]:
            v["dy"] = normal((case["tokens"], case["dim"]), 1 / 64).to(t)
        return v
    if case["kind"] == "dropout":
        shape = (case["rows"], case["cols"])
        return {"x": normal(shape).relu().to(t), "dy": normal(shape, 1 / 64).to(t)}  # behind a ReLU
    e, n = case["experts"], case["tokens"]
    # Some experts are liked more than others.
    logits = normal((n, e)) + normal((1, e), 0.5)
    if case["kind"] == "route":
        if case["masked"]:
            logits[:, 1::max(2, e // (e - case["k"] + 1))] = -math.inf
        v = {"logits": logits.to(t), "bias": normal((1, e), 0.1)}
        if case["train"]:
            v["dweights"] = normal((n, case["k"]))
        return v
    weights, ids = torch.topk(torch.softmax(logits, dim=1), case["k"], dim=1)
    din, dout = case["din"], case["dout"]
    v = {"x": normal((n, din)).to(t), "ids": ids.int(), "weights": weights / weights.sum(dim=1, keepdim=True),
         "w1": normal((e, din, dout), math.sqrt(2 / din)).to(t), "b1": normal((e, dout), 0.1)}
    if case["mode"] == "products":
        v["dz"] = normal((n * case["k"], dout), 1 / 64).to(t)
    else:
        v["w2"], v["b2"] = normal((e, dout, din), math.sqrt(1 / dout)).to(t), normal((e, din), 0.1)
    if case["mode"] == "train":
        v["dy"] = normal((n, din), 1 / 64)
        v["h"], v["o"] = normal((n * case["k"], dout)).relu(), normal((n * case["k"], din))
    return v


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    t = _TORCH[case["dtype"]]

    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="cuda")

    out = s["out"] = {}
    if case["kind"] == "embed":
        out["y"] = empty(case["tokens"], case["dim"], dtype=t)
        if case["train"]:
            out["dtable"] = empty(case["vocab"], case["dim"])
    elif case["kind"] == "dropout":
        out["y"], out["dx"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
    elif case["kind"] == "route":
        out["ids"] = empty(case["tokens"], case["k"], dtype=torch.int32)
        out["weights"] = empty(case["tokens"], case["k"])
        if case["train"]:
            out["dlogits"] = torch.empty_like(s["logits"])
    else:
        e, n, din, dout = case["experts"], case["tokens"], case["din"], case["dout"]
        rows = n * case["k"]
        s["order"], s["rank"] = empty(rows, dtype=torch.int32), empty(n, case["k"], dtype=torch.int32)
        s["offsets"] = empty(e + 1, dtype=torch.int32)
        if case["mode"] == "products":
            s["dxr"] = empty(rows, din, dtype=t)
            out.update(rows=empty(rows, dout, dtype=t), dw=empty(e, din, dout), db=empty(e, dout),
                       dx=empty(n, din, dtype=t))
        elif case["mode"] == "serve":
            s["h"], s["o"] = empty(rows, dout, dtype=t), empty(rows, din, dtype=t)
            out["y"] = empty(n, din, dtype=t)
        else:
            s["do"], s["dh"], s["dxr"] = empty(rows, din), empty(rows, dout), empty(rows, din)
            out.update(dx=empty(n, din), dweights=empty(n, case["k"]), dw1=empty(e, din, dout), db1=empty(e, dout),
                       dw2=empty(e, dout, din), db2=empty(e, din))
    return s


# ------------------------------------------------------------------ the framework's calls

_device = []


def _gpu():
    """The program's one context."""
    if not _device:
        from rgpu_amd import gpu as G

        _device.append(G.Gpu(0))
    return _device[0]


def _handles(s):
    """Handles on the program's device memory, made once for its life."""
    from rgpu_amd import gpu as G

    gpu = _gpu()
    code = {torch.float32: G.F32, torch.bfloat16: G.BF16, torch.float16: G.F16, torch.int32: G.U32}

    def wrap(v):
        return gpu.wrap(v.data_ptr(), tuple(v.shape), code[v.dtype], owner=v)

    h = {k: wrap(v) for k, v in s.items() if torch.is_tensor(v)}
    h["out"] = {k: wrap(v) for k, v in s["out"].items()}
    return h


def _call_experts(case, h, out):
    from rgpu_amd import gpu as G

    gpu = _gpu()
    order, offsets, rank = h["order"], h["offsets"], h["rank"]
    gpu.sort_ids(h["ids"], case["experts"], order, offsets, rank)
    if case["mode"] == "products":
        gpu.experts_gemm(G.NN, h["x"], h["w1"], out["rows"], offsets, order, G.EPI_BIAS_RELU, h["b1"])
        gpu.experts_gemm(G.TN, h["x"], h["dz"], out["dw"], offsets, order, colsum=out["db"])
        gpu.experts_gemm(G.NT, h["dz"], h["w1"], h["dxr"], offsets)
        gpu.combine(h["dxr"], rank, None, out["dx"])
        return
    if case["mode"] == "serve":
        gpu.experts_gemm(G.NN, h["x"], h["w1"], h["h"], offsets, order, G.EPI_BIAS_RELU, h["b1"])
        gpu.experts_gemm(G.NN, h["h"], h["w2"], h["o"], offsets, None, G.EPI_BIAS, h["b2"])
        gpu.combine(h["o"], rank, h["weights"], out["y"])
        return
    gpu.combine_backward(h["dy"], h["o"], rank, h["weights"], h["do"], out["dweights"])
    gpu.experts_gemm(G.TN, h["h"], h["do"], out["dw2"], offsets, colsum=out["db2"])
    gpu.experts_gemm(G.NT, h["do"], h["w2"], h["dh"], offsets, None, G.EPI_RELU_MASK, h["h"])
    gpu.experts_gemm(G.TN, h["x"], h["dh"], out["dw1"], offsets, order, colsum=out["db1"])
    gpu.experts_gemm(G.NT, h["dh"], h["w1"], h["dxr"], offsets)
    gpu.combine(h["dxr"], rank, None, out["dx"])


def _call(s):
    case, gpu = s["case"], _gpu()
    if "handles" not in s:
        s["handles"] = _handles(s)
        # The inputs were made on torch's stream, which the context's is not ordered with; what the calls below write is
        # read by others once the device has been waited for.
        gpu.order_after(torch.cuda.current_stream().cuda_stream)
    h = s["handles"]
    out = h["out"]
    if case["kind"] == "embed":
        gpu.embed(h["table"], h["ids"], out["y"], s["scale"])
        if case["train"]:
            gpu.embed_backward(h["dy"], h["ids"], out["dtable"], s["scale"])
    elif case["kind"] == "dropout":
        q = case["drop"] / 65536
        gpu.dropout(h["x"], out["y"], q, case["seed"], case["draw"])
        gpu.dropout(h["dy"], out["dx"], q, case["seed"], case["draw"])
    elif case["kind"] == "route":
        how = {"score": case["score"], "renormalise": case["renormalise"], "scale": case["scale"]}
        gpu.route(h["logits"], out["ids"], out["weights"], h["bias"] if case["bias"] else None, groups=case["groups"],
                  kept=case["kept"], **how)
        if case["train"]:
            gpu.route_backward(h["logits"], out["ids"], h["dweights"], out["dlogits"], **how)
    else:
        _call_experts(case, h, out)
    return s["out"]


def run(s):
    return _call(s) if own else _plain(s)


# ------------------------------------------------------------------ work

def work(case):
    i = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": 4 * i * n, "flops": 2.0 * n}
    n = case["tokens"]
    if case["kind"] == "embed":
        # At most every token's row is read; a vocabulary smaller than the batch is read once.
        b = i * case["dim"] * (min(n, case["vocab"]) + n) + 4 * n
        if case["train"]:
            b += i * n * case["dim"] + 4 * case["vocab"] * case["dim"]
        return {"bytes": b, "flops": n * case["dim"] * (2.0 if case["train"] else 1.0)}
    e, k = case["experts"], case["k"]
    if case["kind"] == "route":
        b = i * n * e + 8 * n * k + (4 * e if case["bias"] else 0)
        if case["train"]:
            b += i * n * e + 4 * n * k
        return {"bytes": b, "flops": 10.0 * n * e * (2 if case["train"] else 1)}
    din, dout = case["din"], case["dout"]
    one, used = 2.0 * n * k * din * dout, min(e, n * k)  # at most as many experts as there are choices
    if case["mode"] == "serve":
        return {"bytes": i * n * din + 2 * used * (i * din * dout) + 4 * used * (din + dout) + 8 * n * k + i * n * din,
                "flops": 2 * one}
    if case["mode"] == "products":
        return {"bytes": i * (n * din + used * din * dout + n * k * dout) + 4 * (used * dout + n * k)
                + i * (n * k * dout + n * din) + 4 * e * (din * dout + dout), "flops": 3 * one}
    return {"bytes": 4 * (3 * n * din + n * k * (din + dout) + 2 * used * din * dout + 2 * e * din * dout + e * (din + dout)
                          + 3 * n * k), "flops": 4 * one}


# ------------------------------------------------------------------ 64-bit results

def _exact_keep(n, drop, seed, draw_):
    """The mask by the generator's definition, 32-bit words as unsigned numbers in f64 halves and whole 64-bit ones."""
    i = torch.arange((n + 7) // 8, device="cuda")
    word = 1 << 32
    c0, c1, c2, c3 = i % word, i // word, torch.zeros_like(i) + draw_ % word, torch.zeros_like(i) + draw_ // word
    for r in range(10):
        k0 = (seed % word + r * 0x9E3779B9) % word
        k1 = (seed // word + r * 0xBB67AE85) % word
        # A product of two words, by the words' halves: a m = (a m1) 2^16 + a m0 with m = m1 2^16 + m0.
        p = [(a * (m >> 16), a * (m & 0xffff)) for a, m in ((c0, 0xD2511F53), (c2, 0xCD9E8D57))]
        low = [((h % 65536) * 65536 + l) % word for h, l in p]
        high = [(h + l // 65536) // 65536 for h, l in p]
        c0, c1, c2, c3 = high[1] ^ c1 ^ k0, low[1], high[0] ^ c3 ^ k1, low[0]
    bits = torch.stack([c0 % 65536, c0 // 65536, c1 % 65536, c1 // 65536, c2 % 65536, c2 // 65536, c3 % 65536,
                        c3 // 65536], dim=1)
    return (bits.reshape(-1)[:n] >= drop).double()


def _exact_route(case, v):
    x = v["logits"].double()
    if case["score"] == "softmax":
        s = torch.softmax(x, dim=1).nan_to_num(0.0)
    else:
        s = torch.sigmoid(x)
    c = s.clone() if not case["bias"] else s + v["bias"].double()
    if case["kept"] < case["groups"]:
        per = case["experts"] // case["groups"]
        best = torch.stack([torch.topk(c[:, g * per:(g + 1) * per], 2, dim=1).values.sum(dim=1)
                            for g in range(case["groups"])], dim=1)
        for g in range(case["groups"]):
            better = (best > best[:, g:g + 1]).sum(dim=1) + (best[:, :g] == best[:, g:g + 1]).sum(dim=1)
            c[better >= case["kept"], g * per:(g + 1) * per] = -math.inf
    ids = []
    n = torch.arange(case["experts"], device="cuda")
    for _ in range(case["k"]):  # the greatest that is left, the first of equals
        first = torch.where(c == c.amax(dim=1, keepdim=True), n, case["experts"]).amin(dim=1)
        ids.append(first)
        c[torch.arange(c.shape[0], device="cuda"), first] = -math.inf
    ids = torch.stack(ids, dim=1)
    with torch.enable_grad():
        z = x.clone().requires_grad_(case["train"])
        s = torch.softmax(z, dim=1) if case["score"] == "softmax" else torch.sigmoid(z)
        w = torch.gather(s, 1, ids)
        if case["renormalise"]:
            w = w / w.sum(dim=1, keepdim=True)
        w = case["scale"] * w
        out = {"ids": ids.int(), "weights": w.detach()}
        if case["train"]:
            out["dlogits"] = torch.autograd.grad(w, z, v["dweights"].double())[0]
    return out


def _exact_experts(case, v):
    x, w1, b1 = v["x"].double(), v["w1"].double(), v["b1"].double()
    n, k, e = case["tokens"], case["k"], case["experts"]
    ids = v["ids"].long()
    if case["mode"] == "products":
        dz = v["dz"].double()
        out = {"rows": torch.empty_like(dz), "dw": torch.zeros_like(w1), "db": torch.zeros_like(b1), "dx": torch.zeros_like(x)}
        at = 0
        for g in range(e):
            t = (ids == g).nonzero()[:, 0]
            d = dz[at:at + t.numel()]
            out["rows"][at:at + t.numel()] = (x[t] @ w1[g] + b1[g]).clamp_min(0)
            out["dw"][g], out["db"][g] = x[t].T @ d, d.sum(0)
            out["dx"].index_add_(0, t, d @ w1[g].T)
            at += t.numel()
        return out
    w2, b2, w = v["w2"].double(), v["b2"].double(), v["weights"].double()
    if case["mode"] == "serve":
        y = torch.zeros_like(x)
        for g in range(e):
            t, j = (ids == g).nonzero(as_tuple=True)
            y.index_add_(0, t, ((x[t] @ w1[g] + b1[g]).clamp_min(0) @ w2[g] + b2[g]) * w[t, j][:, None])
        return {"y": y}
    out = {"dx": torch.zeros_like(x), "dweights": torch.zeros_like(w), "dw1": torch.zeros_like(w1),
           "db1": torch.zeros_like(b1), "dw2": torch.zeros_like(w2), "db2": torch.zeros_like(b2)}
    at = 0
    for g in range(e):
        t, j = (ids == g).nonzero(as_tuple=True)
        h, o = v["h"][at:at + t.numel()].double(), v["o"][at:at + t.numel()].double()
        dy = v["dy"].double()[t]
        out["dweights"][t, j] = (dy * o).sum(dim=1)
        do = dy * w[t, j][:, None]
        dh = (do @ w2[g].T) * (h > 0)
        out["dw2"][g], out["db2"][g], out["dw1"][g], out["db1"][g] = h.T @ do, do.sum(0), x[t].T @ dh, dh.sum(0)
        out["dx"].index_add_(0, t, dh @ w1[g].T)
        at += t.numel()
    return out


def exact(case, seed):
    v = _inputs(case, seed)
    if case["kind"] == "route":
        return _exact_route(case, v)
    if case["kind"] == "experts":
        return _exact_experts(case, v)
    if case["kind"] == "dropout":
        keep = _exact_keep(v["x"].numel(), case["drop"], case["seed"], case["draw"]).reshape(v["x"].shape)
        keep = keep / (1 - case["drop"] / 65536)
        return {"y": v["x"].double() * keep, "dx": v["dy"].double() * keep}
    on = v["ids"] >= 0
    y = torch.zeros(case["tokens"], case["dim"], dtype=torch.float64, device="cuda")
    y[on] = v["table"].double()[v["ids"][on].long()] * v["scale"]
    out = {"y": y}
    if case["train"]:
        out["dtable"] = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device="cuda").index_put_(
            (v["ids"][on].long(),), v["dy"].double()[on] * v["scale"], accumulate=True)
    return out
