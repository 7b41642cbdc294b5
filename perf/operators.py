"""What the microscaled operators are measured on: the passes of a decoder layer with 4-bit weights.

The format: a row is cut into blocks of 32 elements, a block has one power-of-two scale byte ``s`` (the factor is
2^(s - 127)) and an element is a 4-bit float (e2m1) or an 8-bit one (e4m3).  ``s`` is the biased binary exponent of the
block's largest magnitude less that of the element type's largest power of two (2 or 8); elements round to nearest even
and saturate.  Rows are padded with zeros to whole chunks of 128 elements; two 4-bit codes share a byte, the even one in
the low half; the scales of 128 rows and one chunk lie together, 512 bytes as ``[row % 32][row / 32 % 4][block % 4]``.

Four operators, each case one pass through one of them:

``quantize``  rows of numbers into the format;
``norm``      ``x += delta``, then the root-mean-square norm of ``x`` as 8-bit rows;
``linear``    ``out (+)= a w^T`` with 8- or 4-bit rows ``a`` and 4-bit weights ``w``;
``glu``       ``silu(a g^T) * (a u^T)`` as 8-bit rows, ``w`` holding strips of 32 gate rows and their 32 up rows.

What is held in the format is returned as the numbers it stands for.
"""
import math

import torch

own = False
DEVICE = "cuda:0"
BLOCK, CHUNK, TILE = 32, 128, 128
EMAX = {4: 2, 8: 8}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # a feed-forward's matrix when a checkpoint is loaded: the largest quantisation
        {"name": "quantize 4 bit weights", "op": "quantize", "rows": 12288, "k": 4096, "bits": 4, "type": "bfloat16", "gap": 0},
        # the attention's output of eight decoding requests, on its way into the output projection
        {"name": "quantize 8 bit decode", "op": "quantize", "rows": 8, "k": 4096, "bits": 8, "type": "bfloat16", "gap": 0},
        # float32 columns out of a wider buffer, an odd number of rows and a row that ends inside a chunk
        {"name": "quantize 4 bit columns", "op": "quantize", "rows": 517, "k": 2888, "bits": 4, "type": "float32", "gap": 20},
        # between the two halves of a layer, eight decoding requests
        {"name": "norm decode", "op": "norm", "rows": 8, "k": 4096, "delta": "float32"},
        # ... and a prompt
        {"name": "norm prompt", "op": "norm", "rows": 2048, "k": 4096, "delta": "float32"},
        # the query, key and value projection of one request's next token
        {"name": "linear one token", "op": "linear", "rows": 1, "n": 6144, "k": 4096, "bits": 8, "add": False},
        # the down projection of a busy decode step, added to the residual
        {"name": "linear 64 tokens", "op": "linear", "rows": 64, "n": 4096, "k": 12288, "bits": 8, "add": True},
        # sizes that fill no tile: a short portion into a small projection
        {"name": "linear odd sizes", "op": "linear", "rows": 77, "n": 520, "k": 1000, "bits": 8, "add": False},
        # a prompt's down projection
        {"name": "linear prompt 8 bit", "op": "linear", "rows": 2048, "n": 4096, "k": 12288, "bits": 8, "add": True},
        # a prompt's query, key and value projection with its rows in 4 bits too
        {"name": "linear prompt 4 bit", "op": "linear", "rows": 4096, "n": 6144, "k": 4096, "bits": 4, "add": False},
        # the gated half of the feed-forward, eight decoding requests
        {"name": "glu decode", "op": "glu", "rows": 8, "n": 12288, "k": 4096, "bits": 8},
        # ... and a prompt, rows in 4 bits
        {"name": "glu prompt 4 bit", "op": "glu", "rows": 2048, "n": 12288, "k": 4096, "bits": 4},
    ]


def _between(rng, low, high):
    """A whole number, even over the logarithm; about half of them odd."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("quantize", "norm", "linear", "glu"))
    if op == "quantize":
        case = {"op": op, "rows": _between(rng, 1, 12288), "k": _between(rng, 100, 8192), "bits": rng.choice((4, 8)),
                "type": rng.choice(("bfloat16", "float32")), "gap": rng.choice((0, 0, 8, 20, 33))}
    elif op == "norm":
        case = {"op": op, "rows": _between(rng, 1, 4096), "k": _between(rng, 100, 8192),
                "delta": rng.choice(("none", "bfloat16", "float32"))}
    else:
        # rows of activations end where a head or a width ends: mostly whole blocks, sometimes not
        k = _between(rng, 100, 12288)
        case = {"op": op, "rows": _between(rng, 1, 4096), "n": _between(rng, 64, 8192),
                "k": k if rng.random() < 0.5 else max(128, k // 128 * 128), "bits": rng.choice((4, 8))}
        if op == "linear":
            case["add"] = rng.choice((False, True))
    big = max(work(c)["flops"] for c in listed())
    while work(case)["flops"] > big or work(case)["bytes"] > (1 << 28):
        case["rows"] = max(1, case["rows"] // 2)
    return case


def _up(n, to):
    return -(-n // to) * to


def work(case):
    rows, k = case["rows"], case["k"]
    held = {4: 0.5 + 1 / BLOCK, 8: 1 + 1 / BLOCK}
    if case["op"] == "quantize":
        return {"bytes": rows * k * ((2 if case["type"] == "bfloat16" else 4) + 2), "flops": 3 * rows * k}
    if case["op"] == "norm":
        return {"bytes": rows * k * (6 + {"none": 0, "bfloat16": 6, "float32": 8}[case["delta"]]) + 4 * k,
                "flops": 7 * rows * k}
    n = case["n"] * (2 if case["op"] == "glu" else 1)
    read = rows * k * held[case["bits"]] + n * k * held[4]
    wrote = rows * case["n"] * 2 if case["op"] == "glu" else rows * n * (8 if case["add"] else 4)
    return {"bytes": read + wrote, "flops": 2 * rows * n * k}


# ---- the format in elementary operations ---------------------------------------------------------
def _scale(s):
    """2^(s - 127) in float32, from the bits."""
    bits = torch.where(s == 0, torch.full_like(s, 1 << 22), s << 23)
    return bits.view(torch.float32)


def _round(y, bits):
    """Nearest e2m1 or e4m3 number of float32 ``y``, ties to even, saturating."""
    if bits == 8:
        return y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).to(torch.float32)
    a = y.abs()
    q = torch.where(a < 2, (a * 2).round() / 2, torch.where(a < 4, a.round(), (a / 2).round() * 2)).clamp(max=6.0)
    return torch.copysign(q, y)


def _quantized(x, bits):
    """Elements ``[rows, blocks, 32]`` before their scale and scale bytes ``[rows, blocks]`` (int32) of float32 rows."""
    rows, k = x.shape
    x = torch.nn.functional.pad(x, (0, _up(k, CHUNK) - k)).view(rows, -1, BLOCK)
    top = x.abs().amax(dim=2)
    s = ((top.view(torch.int32) >> 23) - EMAX[bits]).clamp(min=0)
    inverse = _scale(254 - s)
    return _round(x * inverse[:, :, None], bits), s


def _values(x, bits):
    """float32 rows as the format holds them."""
    q, s = _quantized(x, bits)
    return (q * _scale(s)[:, :, None]).view(x.shape[0], -1)[:, : x.shape[1]]


def _stored(x, bits):
    """Codes and tiled scales of float32 rows, as they lie in memory."""
    q, s = _quantized(x, bits)
    rows, blocks = s.shape
    q = q.view(rows, -1)
    if bits == 8:
        codes = q.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        a = q.abs()
        c = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
        c = c | ((q < 0).to(torch.uint8) << 3)
        codes = c[:, 0::2] | (c[:, 1::2] << 4)
    s = torch.nn.functional.pad(s, (0, 0, 0, _up(rows, TILE) - rows)).to(torch.uint8)
    s = s.view(-1, 4, 32, blocks // 4, 4).permute(0, 3, 2, 1, 4)       # tile, chunk, row % 32, row / 32 % 4, block % 4
    return codes.contiguous(), s.reshape(-1, blocks // 4, 512).contiguous()


def _loaded(codes, scales, bits, k):
    """The float32 numbers that codes and tiled scales stand for."""
    rows = codes.shape[0]
    if bits == 8:
        q = codes.view(torch.float8_e4m3fn).to(torch.float32)
    else:
        table = torch.tensor(E2M1, device=codes.device)
        q = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), dim=2).view(rows, -1)
    s = scales.view(scales.shape[0], -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, scales.shape[1] * 4)[:rows].int()
    return (q.view(rows, -1, BLOCK) * _scale(s)[:, :, None]).view(rows, -1)[:, :k]


# ---- inputs --------------------------------------------------------------------------------------
def _rows(g, rows, k):
    """Activations: a few channels are much larger than the rest, and rows differ in size."""
    x = torch.randn(rows, k, device=DEVICE, generator=g)
    channel = torch.exp(0.5 * torch.randn(k, device=DEVICE, generator=g))
    channel[torch.randint(0, k, (max(1, k // 200),), device=DEVICE, generator=g)] *= 12.0
    return x * channel * torch.exp(0.3 * torch.randn(rows, 1, device=DEVICE, generator=g))


def _weights(g, n, k):
    return torch.randn(n, k, device=DEVICE, generator=g) * (k ** -0.5)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    op, rows, k = case["op"], case["rows"], case["k"]
    s = dict(case)
    if op == "quantize":
        wide = _rows(g, rows, k + case["gap"]).to(TYPES[case["type"]])
        s["x"] = wide[:, case["gap"]:]
    elif op == "norm":
        s["x"] = _rows(g, rows, k)
        s["weight"] = 1.0 + 0.2 * torch.randn(k, device=DEVICE, generator=g)
        s["delta_rows"] = None if case["delta"] == "none" else (0.1 * _rows(g, rows, k)).to(TYPES[case["delta"]])
    else:
        n = case["n"]
        s["a"] = _stored(_rows(g, rows, k), case["bits"])
        if op == "glu":          # strips of 32 gate rows and their 32 up rows, whole chunks of columns with zero rows
            pad = _up(n, CHUNK) - n
            both = [torch.nn.functional.pad(_weights(g, n, k), (0, 0, 0, pad)).view(-1, BLOCK, k) for _ in range(2)]
            s["w"] = _stored(torch.stack(both, dim=1).view(-1, k), 4)
        else:
            s["w"] = _stored(_weights(g, n, k), 4)
            s["out"] = torch.randn(rows, n, device=DEVICE, generator=g)
    return s


# ---- one pass ------------------------------------------------------------------------------------
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from tinyinfer_b200.kernels import MxRows, cuda_ops
    ops, op = cuda_ops(DEVICE), s["op"]
    if op == "quantize":
        return ops.mx_dequantize(ops.mx_quantize(s["x"], s["bits"]))
    if op == "norm":
        h = ops.mx_rmsnorm(s["x"], s["weight"], 1e-6, bits=8, delta=s["delta_rows"])
        return s["x"], ops.mx_dequantize(h)
    a, w = MxRows(*s["a"], s["bits"], s["k"]), MxRows(*s["w"], 4, s["k"], settled=True)
    if op == "glu":
        return ops.mx_dequantize(ops.mx_linear_glu(a, w, s["n"], bits=8))
    ops.mx_linear(a, w, s["out"], accumulate=s["add"])
    return s["out"]


def _run_plain(s):
    op = s["op"]
    if op == "quantize":
        return _values(s["x"].float(), s["bits"]).to(torch.bfloat16)
    if op == "norm":
        x = s["x"]
        if s["delta_rows"] is not None:
            x.add_(s["delta_rows"].float())
        h = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + 1e-6) * s["weight"]
        return x, _values(h, 8).to(torch.bfloat16)
    a, w = _loaded(*s["a"], s["bits"], s["k"]), _loaded(*s["w"], 4, s["k"])
    if op == "glu":
        gate, up = (a @ w.T).view(a.shape[0], -1, 2, BLOCK).unbind(dim=2)
        h = (gate / (1 + torch.exp(-gate)) * up).reshape(a.shape[0], -1)[:, : s["n"]]
        return _values(h, 8).to(torch.bfloat16)
    if s["add"]:
        s["out"].add_(a @ w.T)
    else:
        s["out"].copy_(a @ w.T)
    return s["out"]


# ---- the definition in 64 bits -------------------------------------------------------------------
def _power(e):
    """2^e in float64 for whole numbers e, from the bits."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _exact_values(x, bits):
    """Each number of float64 rows as the format holds it: through exponents, not bits."""
    rows, k = x.shape
    blocks = torch.zeros(rows, _up(k, BLOCK), dtype=torch.float64, device=x.device)
    blocks[:, :k] = x
    blocks = blocks.view(rows, -1, BLOCK)
    power = torch.frexp(blocks.abs().amax(dim=2, keepdim=True))[1] - 1 - EMAX[bits]
    unit = _power(power.clamp(min=-127))
    y = blocks / unit
    digits, lowest, top = (1, 0, 6.0) if bits == 4 else (3, -6, 448.0)
    step = _power((torch.frexp(y)[1] - 1).clamp(min=lowest) - digits)
    y = ((y / step).round() * step).clamp(-top, top)
    return (y * unit).view(rows, -1)[:, :k]


def _exact_loaded(codes, scales, bits, k):
    """The float64 numbers of stored rows, element by element from the codes' fields."""
    rows, width = codes.shape[0], scales.shape[1] * CHUNK
    if bits == 4:
        c = torch.empty(rows, width, dtype=torch.int64, device=codes.device)
        c[:, 0::2], c[:, 1::2] = (codes % 16).long(), (codes // 16).long()
        digits, lowest = 1, 1
    else:
        c = codes.long()
        digits, lowest = 3, 7
    sign, e, m = c // (1 << (bits - 1)), c // (1 << digits) % (1 << (bits - 1 - digits)), c % (1 << digits)
    m = torch.where(e == 0, m, m + (1 << digits)).double()
    row, block = torch.arange(rows, device=codes.device)[:, None], torch.arange(width // BLOCK, device=codes.device)[None, :]
    s = scales[row // TILE, block // 4, row % 32 * 16 + row // 32 % 4 * 4 + block % 4].long()
    power = e.clamp(min=1) - lowest - digits + (s - 127).repeat_interleave(BLOCK, dim=1)
    return (m * _power(power) * (1 - 2 * sign))[:, :k]


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "quantize":
        return _exact_values(s["x"].double(), case["bits"])
    if op == "norm":                                   # the rows before their rounding to 8 bits
        x = s["x"].double()
        if s["delta_rows"] is not None:
            x = x + s["delta_rows"].double()
        return x, x / (x.square().sum(dim=1, keepdim=True) / case["k"] + 1e-6).sqrt() * s["weight"].double()
    a, w = _exact_loaded(*s["a"], case["bits"], case["k"]), _exact_loaded(*s["w"], 4, case["k"])
    if op == "linear":
        product = torch.nn.functional.linear(a, w)
        return product + s["out"].double() if case["add"] else product
    rows = torch.arange(w.shape[0], device=w.device).view(-1, 2, BLOCK)
    gate, up = (torch.nn.functional.linear(a, w[rows[:, i].reshape(-1)])[:, : case["n"]] for i in range(2))
    return gate * torch.sigmoid(gate) * up             # the rows before their rounding to 8 bits
