"""The low-bit operators of a Linear layer, as cases that can be timed and compared: their plain forms in elementary torch
operations, or, where ``own`` is true, the calls that a program makes of this package.

Kinds
-----
quantize    values into microscaled floating point (blocks of 32 that share a power-of-two scale; e2m1 in 4 bits or e4m3
            in 8) along the rows, or transposed along the columns as a weight [in, out] is laid out for the product, and
            back to the values that the codes stand for.
linear      a Dense layer as it is served: the activations into 8 or 4 bits, their product with weights held in 4 bits,
            then bias and ReLU.
checkpoint  a Dense layer's training step around a saved activation: the input into 8 bits after the forward pass, and the
            backward pass from those 8 bits (dW, db, dX; for a hidden layer dX with the ReLU mask of the saved input).

The packed form of a [rows, cols] tensor is one buffer of bytes.  First the codes: each row padded with zeros to whole 128
columns; 4-bit codes two to a byte, the even column in the low half.  Then, from the next multiple of 256 bytes on, the
scales, one byte e for 32 columns, standing for 2^(e - 127): for each 128 columns and each 64 rows 256 bytes, where byte
4 (16 g + r) + t belongs to row 16 t + r and to columns 32 g to 32 g + 31.
"""
import math

import torch

own = False

# ------------------------------------------------------------------ the cases

_LISTED = [
    # A wide layer's weights [in, out] laid out for serving, once a checkpoint is loaded or after an optimizer step.
    {"name": "weights_4bit_4096", "kind": "quantize", "bits": 4, "dtype": "f32", "rows": 4096, "cols": 4096,
     "transposed": True},
    # The activations of that layer at the batch that it is trained on.
    {"name": "activations_8bit_8192", "kind": "quantize", "bits": 8, "dtype": "bf16", "rows": 8192, "cols": 4096,
     "transposed": False},
    # Sizes that a data set gave: no row on a 16-byte boundary, the last block of a row cut.
    {"name": "odd_4bit_f16", "kind": "quantize", "bits": 4, "dtype": "f16", "rows": 1500, "cols": 1003,
     "transposed": False},
    # One request: a row through a wide layer, bound by the weights' bytes and by launches.
    {"name": "serve_1x4096", "kind": "linear", "bits": 8, "dtype": "bf16", "rows": 1, "din": 4096, "dout": 4096},
    # A small batch through the small model's hidden layer, in f32.
    {"name": "serve_32x1024_f32", "kind": "linear", "bits": 8, "dtype": "f32", "rows": 32, "din": 1024, "dout": 1024},
    # A batch whose sizes are multiples of no tile.
    {"name": "serve_ragged", "kind": "linear", "bits": 8, "dtype": "bf16", "rows": 4100, "din": 4000, "dout": 1000},
    # The wide layer at a training batch, both operands in 4 bits: the largest product.
    {"name": "serve_8192_4bit", "kind": "linear", "bits": 4, "dtype": "bf16", "rows": 8192, "din": 4096, "dout": 16384},
    # The small model's first hidden layer at batch 2048, f32 gradients.
    {"name": "train_f32_b2048", "kind": "checkpoint", "dtype": "f32", "rows": 2048, "din": 1024, "dout": 1024,
     "hidden": True},
    # Odd widths in f32.
    {"name": "train_f32_odd", "kind": "checkpoint", "dtype": "f32", "rows": 1500, "din": 1003, "dout": 777,
     "hidden": True},
    # The Linear 4096 -> 4096 backward at batch 8192.
    {"name": "train_bf16_b8192", "kind": "checkpoint", "dtype": "bf16", "rows": 8192, "din": 4096, "dout": 4096,
     "hidden": False},
    # A narrow layer over a very long batch: few tiles of dW, all of the work along the batch.
    {"name": "train_f16_b262144", "kind": "checkpoint", "dtype": "f16", "rows": 262144, "din": 512, "dout": 512,
     "hidden": False},
    # The last batch of an epoch: a few rows, so launches count.
    {"name": "train_bf16_b37", "kind": "checkpoint", "dtype": "bf16", "rows": 37, "din": 1024, "dout": 1000,
     "hidden": True},
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
    kind = rng.choice(["quantize", "linear", "linear", "checkpoint", "checkpoint"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if kind == "quantize":
        return {"kind": kind, "bits": rng.choice([4, 8]), "dtype": dtype, "rows": _size(rng, 1, 8192),
                "cols": _size(rng, 32, 4096), "transposed": rng.random() < 0.5}
    if kind == "linear":
        return {"kind": kind, "bits": rng.choice([4, 8]), "dtype": dtype, "rows": _size(rng, 1, 8192),
                "din": _size(rng, 64, 4096), "dout": _size(rng, 10, 8192)}
    return {"kind": kind, "dtype": dtype, "rows": _size(rng, 1, 8192), "din": _size(rng, 64, 2048),
            "dout": _size(rng, 10, 2048), "hidden": rng.random() < 0.5}


_TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _wide(dtype):
    """What results are written as: bf16 where the inputs are, else f32."""
    return "bf16" if dtype == "bf16" else "f32"


# ------------------------------------------------------------------ the plain form

# Per width: mantissa bits, smallest exponent, and the largest value's mantissa bits (as an f32) and exponent.
_MINIFLOAT = {4: (1, 0, 0x400000, 2), 8: (3, -6, 0x600000, 8)}


def _power(e):
    """2^e in f32, exactly, for whole e from -127 to 127."""
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 0x400000)).view(torch.float32)


def _blocks(x):
    """[rows, cols] as [rows, blocks, 32], padded with zeros to whole 128 columns."""
    rows, cols = x.shape
    pad = -cols % 128
    if pad:
        x = torch.cat([x, x.new_zeros(rows, pad)], dim=1)
    return x.reshape(rows, -1, 32)


def _round_blocks(x, bits):
    """f32 blocks in units of their scales, rounded to the values of the format, and the scales' bytes.  The scale is the
    least power of two, from 2^-127 on, at which the block's largest magnitude does not pass the format's largest value."""
    mantissa, least, top_mantissa, top_exponent = _MINIFLOAT[bits]
    amax = x.abs().amax(dim=2).view(torch.int32)
    byte = (amax >> 23) - top_exponent + ((amax & 0x7fffff) > top_mantissa)
    byte = byte.clamp_min(0)
    q = x * _power(127 - byte)[..., None]
    exponent = ((q.view(torch.int32) >> 23) & 0xff) - 127
    step = _power(exponent.clamp_min(least) - mantissa)
    return torch.round(q / step) * step, byte


def _quantized(x, bits):
    """The values that the format holds for the f32 rows of x."""
    q, byte = _round_blocks(_blocks(x), bits)
    return (q * _power(byte - 127)[..., None]).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _scale_order(rows, blocks):
    """Where the bytes of a [rows, blocks] scale table go in the packed form, as a shape and an order of its axes."""
    return (-(-rows // 64), 4, 16, blocks // 4, 4), (3, 0, 4, 2, 1)


def _packed_sizes(rows, cols, bits):
    wide = -(-cols // 128) * 128
    codes = rows * wide * bits // 8
    at = -(-codes // 256) * 256
    return codes, at, at + wide // 128 * -(-rows // 64) * 256


def _packed(x, bits):
    """The packed form of the rows of x (4 bits)."""
    rows, cols = x.shape
    q, byte = _round_blocks(_blocks(x), bits)
    m = q.abs()
    code = ((m >= 0.5).int() + (m >= 1) + (m >= 1.5) + (m >= 2) + (m >= 3) + (m >= 4) + (m >= 6)) | ((q < 0).int() << 3)
    code = code.reshape(rows, -1)
    codes, at, total = _packed_sizes(rows, cols, bits)
    out = torch.zeros(total, dtype=torch.uint8, device=x.device)
    out[:codes] = (code[:, 0::2] | (code[:, 1::2] << 4)).to(torch.uint8).reshape(-1)
    shape, order = _scale_order(rows, byte.shape[1])
    full = torch.zeros(shape[0] * 64, byte.shape[1], dtype=torch.uint8, device=x.device)
    full[:rows] = byte.to(torch.uint8)
    out[at:] = full.reshape(shape).permute(order).reshape(-1)
    return out


def _unpacked(data, rows, cols):
    """The f32 values of a packed 4-bit tensor."""
    codes, at, _ = _packed_sizes(rows, cols, 4)
    pair = data[:codes].reshape(rows, -1)
    code = torch.stack([pair & 15, pair >> 4], dim=2).reshape(rows, -1).int()
    exponent, mantissa = (code >> 1) & 3, (code & 1).float()
    m = torch.where(exponent == 0, mantissa * 0.5, (1 + mantissa * 0.5) * _power(exponent - 1))
    m = torch.where(code >= 8, -m, m)
    blocks = m.shape[1] // 32
    shape, order = _scale_order(rows, blocks)
    table = data[at:].reshape([shape[k] for k in order])
    back = [order.index(k) for k in range(5)]
    byte = table.permute(back).reshape(-1, blocks)[:rows].int()
    return (m.reshape(rows, blocks, 32) * _power(byte - 127)[..., None]).reshape(rows, -1)[:, :cols]


def _plain(s):
    case = s["case"]
    x = s["x"].float()
    if case["kind"] == "quantize":
        y = _quantized(x.T.contiguous() if case["transposed"] else x, case["bits"])
        return {"values": y.to(s["values"].dtype)}
    if case["kind"] == "linear":
        w = _unpacked(s["w"], case["dout"], case["din"])
        y = torch.relu(_quantized(x, case["bits"]) @ w.T + s["b"])
        return {"y": y.to(s["y"].dtype)}
    dy, w = s["dy"].float(), s["w"].float()
    dx = dy @ w.T
    if case["hidden"]:
        dx = dx * (x > 0)
    return {"dw": _quantized(x, 8).T @ dy, "db": dy.sum(0, keepdim=True), "dx": dx.to(s["dx"].dtype)}


# ------------------------------------------------------------------ inputs (from the seed alone)

def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))

    def normal(shape, scale=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * scale

    t = _TORCH[case["dtype"]]
    if case["kind"] == "quantize":
        shape = (case["rows"], case["cols"])
        if case["transposed"]:  # a trained layer's weights
            return {"x": normal(shape, case["rows"] ** -0.5).to(t)}
        # Activations: some features larger than others, some rows of padding.
        x = normal(shape) * normal((1, shape[1]), 0.7).exp()
        x[torch.rand(shape[0], generator=gen, device="cuda") < 0.02] = 0
        return {"x": x.to(t)}
    rows, din, dout = case["rows"], case["din"], case["dout"]
    x = (normal((rows, din)) * normal((1, din), 0.5).exp()).relu()  # the layer below ends in a ReLU
    w = normal((din, dout), math.sqrt(2 / din))
    if case["kind"] == "linear":
        return {"x": x.to(t), "w": w, "b": normal((1, dout), 0.1)}
    return {"x": x.to(t), "w": w.to(t), "dy": normal((rows, dout), 1 / 64).to(t)}


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    kind, wide = case["kind"], _TORCH[_wide(case["dtype"])]

    def empty(shape, dtype):
        return torch.empty(shape, dtype=dtype, device="cuda")

    if kind == "quantize":
        shape = (case["cols"], case["rows"]) if case["transposed"] else (case["rows"], case["cols"])
        s["packed"] = empty(_packed_sizes(*shape, case["bits"])[2], torch.uint8)
        s["values"] = empty(shape, wide)
    elif kind == "linear":
        s["w"] = _packed(s["w"].T.contiguous(), 4)  # the weights, laid out once
        s["packed"] = empty(_packed_sizes(case["rows"], case["din"], case["bits"])[2], torch.uint8)
        s["y"] = empty((case["rows"], case["dout"]), wide)
    else:
        s["packed"] = empty(_packed_sizes(case["rows"], case["din"], 8)[2], torch.uint8)
        s["dw"], s["db"] = empty((case["din"], case["dout"]), torch.float32), empty((1, case["dout"]), torch.float32)
        s["dx"] = empty((case["rows"], case["din"]), wide)
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

    case, gpu = s["case"], _gpu()
    code = {torch.float32: G.F32, torch.bfloat16: G.BF16, torch.float16: G.F16}
    h = {k: gpu.wrap(v.data_ptr(), tuple(v.shape), code[v.dtype], owner=v)
         for k, v in s.items() if torch.is_tensor(v) and v.dtype in code}
    fmt = G.MXFP4 if case.get("bits") == 4 else G.MXFP8
    if case["kind"] == "quantize":
        shape = tuple(s["values"].shape)
    else:
        shape = tuple(s["x"].shape)
    h["packed"] = gpu.wrap(s["packed"].data_ptr(), shape, fmt, owner=s["packed"])
    if case["kind"] == "linear":
        h["w"] = gpu.wrap(s["w"].data_ptr(), (case["dout"], case["din"]), G.MXFP4, owner=s["w"])
    return h


def _call(s):
    from rgpu_amd import gpu as G

    case, gpu = s["case"], _gpu()
    if "handles" not in s:
        s["handles"] = _handles(s)
        # The inputs were made on torch's stream, which the context's is not ordered with; what the calls below write is
        # read by others once the device has been waited for.
        gpu.order_after(torch.cuda.current_stream().cuda_stream)
    h = s["handles"]
    if case["kind"] == "quantize":
        if case["transposed"]:
            gpu.convert_t(h["x"], h["packed"])
        else:
            gpu.convert(h["x"], h["packed"])
        gpu.convert(h["packed"], h["values"])
        return {"values": s["values"]}
    gpu.convert(h["x"], h["packed"])
    if case["kind"] == "linear":
        gpu.gemm(G.NT, h["packed"], h["w"], h["y"], G.EPI_BIAS_RELU, h["b"])
        return {"y": s["y"]}
    if case["hidden"]:
        gpu.matmul_at_b(h["packed"], h["dy"], h["dw"], colsum=h["db"])
        gpu.matmul_a_bt(h["dy"], h["w"], h["dx"], relu_mask_from=h["packed"])
    else:
        gpu.linear_backward(h["packed"], h["dy"], h["w"], h["dx"], h["dw"], h["db"])
    return {"dw": s["dw"], "db": s["db"], "dx": s["dx"]}


def run(s):
    return _call(s) if own else _plain(s)


# ------------------------------------------------------------------ work

def work(case):
    i, o = 4 if case["dtype"] == "f32" else 2, 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "quantize":
        shape = (case["cols"], case["rows"]) if case["transposed"] else (case["rows"], case["cols"])
        n = case["rows"] * case["cols"]
        # The values in, the packed form out, the values that it stands for out.
        return {"bytes": (i + o) * n + _packed_sizes(*shape, case["bits"])[2], "flops": 8.0 * n}
    rows, din, dout = case["rows"], case["din"], case["dout"]
    one = 2.0 * rows * din * dout
    if case["kind"] == "linear":
        return {"bytes": i * rows * din + _packed_sizes(dout, din, 4)[2] + 4 * dout + o * rows * dout, "flops": one}
    grads = o * rows * din + 4 * (din * dout + dout)
    return {"bytes": i * (rows * din + rows * dout + din * dout) + _packed_sizes(rows, din, 8)[2] + grads,
            "flops": 2 * one}


# ------------------------------------------------------------------ 64-bit results

def _exact_quantized(x, bits):
    """Every element to the nearest of the format's values (written out as a list; a tie goes to the even code) in units of
    the block's scale, in 64 bits."""
    if bits == 4:
        table = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    else:
        table = [c / 512 for c in range(8)] + [(8 + c % 8) / 8 * 2.0 ** (c // 8 - 7) for c in range(8, 127)]
    values = torch.tensor(table, dtype=torch.float64, device=x.device)
    middle = (values[1:] + values[:-1]) / 2
    rows, cols = x.shape
    out = torch.empty_like(x)
    for c in range(0, cols, 32):
        block = x[:, c:c + 32]
        top = block.abs().amax(dim=1, keepdim=True)
        m, e = torch.frexp(top)
        mt, et = math.frexp(table[-1])
        e = torch.where(m > mt, e - et + 1, e - et)
        e = torch.where(top > 0, e, torch.zeros_like(e)).clamp_min(-127).long()
        scale = ((e + 1023) << 52).view(torch.float64)
        q = block.abs() / scale
        below = torch.bucketize(q, middle)  # middles under q
        at = middle[below.clamp_max(len(table) - 2)]
        code = below + ((q == at) & (below % 2 == 1)).long()
        out[:, c:c + 32] = values[code.clamp_max(len(table) - 1)] * scale * torch.sign(block)
    return out


def exact(case, seed):
    v = _inputs(case, seed)
    x = v["x"].double()
    if case["kind"] == "quantize":
        return {"values": _exact_quantized(x.T.contiguous() if case["transposed"] else x, case["bits"])}
    if case["kind"] == "linear":
        w = _exact_quantized(v["w"].double().T.contiguous(), 4)
        return {"y": torch.relu(_exact_quantized(x, case["bits"]) @ w.T + v["b"].double())}
    dy = v["dy"].double()
    dx = dy @ v["w"].double().T
    return {"dw": _exact_quantized(x, 8).T @ dy, "db": dy.sum(0, keepdim=True), "dx": dx * (x > 0) if case["hidden"] else dx}
