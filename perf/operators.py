"""The microscaled 4-bit operators, as they are used: tensors rounded to E2M1
blocks and back, products of blocks, a served linear layer and a trained one.

A block is 16 or 32 consecutive elements along the contraction with one 8-bit
scale: UE4M3 (16 elements, with a power-of-two multiplier per tensor where
asked for) or UE8M0 (16 or 32 elements).  Held operands are what a program
keeps: E2M1 codes two to a byte, low nibble first, rows padded with zeros to a
multiple of 16 bytes, and scale bytes in tiles of 128 rows by 4 blocks (byte
(r % 32) * 16 + (r % 128) // 32 * 4 + b % 4 of tile (r // 128, b // 4)).
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = {"ue4m3/4": 16, "ue8m0/2": 32, "ue8m0/4": 16}


def listed():
    return [
        # one token's activations, rounded with a static scale: launch latency
        {"name": "round-token", "op": "round", "rows": 1, "k": 4096, "type": "bf16", "scale": "ue4m3/4",
         "auto": False, "columns": False, "up": False},
        # a training step's activations, scaled by their own largest value
        {"name": "round-activations", "op": "round", "rows": 8192, "k": 8192, "type": "bf16", "scale": "ue4m3/4",
         "auto": True, "columns": False, "up": False},
        # an f32 tensor whose rows end inside a block and start unaligned
        {"name": "round-ragged", "op": "round", "rows": 1003, "k": 4999, "type": "f32", "scale": "ue8m0/2",
         "auto": False, "columns": False, "up": True},
        # the same tensor's blocks down the columns, for a gradient's contraction over tokens
        {"name": "round-columns", "op": "round", "rows": 8192, "k": 4096, "type": "bf16", "scale": "ue4m3/4",
         "auto": True, "columns": True, "up": False},
        # decoding one sequence: one token through a layer held in 4 bits
        {"name": "serve-one", "op": "serve", "tokens": 1, "n": 8192, "k": 8192, "type": "bf16", "scale": "ue4m3/4"},
        # decoding a batch of sequences
        {"name": "serve-batch", "op": "serve", "tokens": 48, "n": 14336, "k": 4096, "type": "bf16",
         "scale": "ue8m0/2"},
        # a small layer of odd sizes
        {"name": "serve-odd", "op": "serve", "tokens": 7, "n": 1003, "k": 2055, "type": "f16", "scale": "ue8m0/4"},
        # a large product of held operands: the tensor cores' rate
        {"name": "mm-square", "op": "mm", "m": 8192, "n": 8192, "k": 8192, "type": "bf16", "scale": "ue4m3/4",
         "add": False},
        # odd sizes with an addend, in 16-element UE8M0 blocks
        {"name": "mm-odd-add", "op": "mm", "m": 777, "n": 2051, "k": 4101, "type": "f16", "scale": "ue8m0/4",
         "add": True},
        # a weight gradient's shape: few tiles, a long contraction
        {"name": "mm-long", "op": "mm", "m": 512, "n": 384, "k": 65536, "type": "bf16", "scale": "ue8m0/2",
         "add": False},
        # a linear layer's training step: output, input gradient, weight gradient
        {"name": "train", "op": "train", "tokens": 8192, "n": 4096, "k": 4096, "type": "bf16", "scale": "ue4m3/4"},
        # the same with token and feature counts that fill no block or tile
        {"name": "train-odd", "op": "train", "tokens": 1501, "n": 1999, "k": 1002, "type": "f16",
         "scale": "ue8m0/2"},
    ]


def _spread(rng, low, high):
    """A size spread over the logarithm of its range; one in three is a multiple of 128 where that fits."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return v // 128 * 128 if v >= 256 and rng.random() < 1 / 3 else v


def draw(rng):
    op = rng.choice(["round", "serve", "mm", "train"])
    case = {"op": op, "type": rng.choice(["bf16", "bf16", "f16", "f32"]),
            "scale": rng.choice(["ue4m3/4", "ue8m0/2", "ue8m0/4"])}
    if op == "round":
        case |= {"rows": _spread(rng, 1, 8192), "k": _spread(rng, 33, 8192),
                 "auto": case["scale"] == "ue4m3/4" and rng.random() < 0.5, "columns": rng.random() < 0.4,
                 "up": case["scale"] != "ue4m3/4" and rng.random() < 0.5}
        return case
    if case["type"] == "f32":
        case["type"] = "bf16"
    if op == "serve":
        case |= {"tokens": _spread(rng, 1, 64), "n": _spread(rng, 500, 14336), "k": _spread(rng, 500, 8192)}
    elif op == "mm":
        case |= {"m": _spread(rng, 33, 8192), "n": _spread(rng, 33, 8192), "k": _spread(rng, 65, 8192),
                 "add": rng.random() < 0.3}
    else:
        case |= {"tokens": _spread(rng, 100, 8192), "n": _spread(rng, 100, 4096), "k": _spread(rng, 100, 4096)}
    return case


# ------------------------------------------------------------- inputs


def _activations(g, rows, k, dtype):
    """Normal values whose channels differ in size, a few of them far larger, and some rows of zeros (padding)."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(k, generator=g, device="cuda"))
    x *= torch.where(torch.rand(k, generator=g, device="cuda") < 0.004, 24.0, 1.0)
    if rows > 16:
        x *= (torch.rand(rows, 1, generator=g, device="cuda") > 0.02).float()
    return x.to(dtype)


def _weights(g, n, k, dtype):
    return (torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)).to(dtype)


def _held(w, scale):
    """A matrix as a program holds it in 4 bits: packed codes and tiled scales."""
    values, steps = _blocks(w, scale, 1.0, False)
    rows, k = w.shape
    half = values.reshape(rows, -1)[:, :k].abs() * 2
    code = half - (half > 4).float() * (half - 4) / 2 - (half > 8).float()
    code = (code.to(torch.int32) + 8 * (torch.signbit(values.reshape(rows, -1)[:, :k])).int()).to(torch.uint8)
    width = (k + 31) // 32 * 32
    nibbles = torch.zeros(rows, width, dtype=torch.uint8, device=w.device)
    nibbles[:, :k] = code
    data = nibbles[:, 0::2] | (nibbles[:, 1::2] << 4)
    if scale.startswith("ue4m3"):
        words = steps.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        words = (torch.frexp(steps)[1] + 126).to(torch.uint8)
    blocks = words.shape[1]
    full = torch.zeros((rows + 127) // 128 * 128, (blocks + 3) // 4 * 4, dtype=torch.uint8, device=w.device)
    full[:rows, :blocks] = words
    tiles = full.view(-1, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()
    return {"data": data, "scales": tiles.view(tiles.shape[0], tiles.shape[1], 512), "k": k}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["type"]]
    state = dict(case)
    if op == "round":
        state["x"] = _activations(g, case["rows"], case["k"], dtype)
    elif op == "serve":
        state["x"] = _activations(g, case["tokens"], case["k"], dtype)
        state["w"] = _held(torch.randn(case["n"], case["k"], generator=g, device="cuda"), case["scale"])
    elif op == "mm":
        state["a"] = _held(_activations(g, case["m"], case["k"], torch.float32), case["scale"])
        state["b"] = _held(torch.randn(case["n"], case["k"], generator=g, device="cuda"), case["scale"])
        state["c"] = torch.randn(case["m"], case["n"], generator=g, device="cuda").to(dtype) if case["add"] else None
    else:
        state["x"] = _activations(g, case["tokens"], case["k"], dtype).requires_grad_()
        state["w"] = _weights(g, case["n"], case["k"], dtype).requires_grad_()
        size = 1.0 if dtype == torch.float16 else 1e-4  # f16 gradients come scaled
        state["g"] = (torch.randn(case["tokens"], case["n"], generator=g, device="cuda") * size).to(dtype)
    return state


# --------------------------------------------------------- plain forms


def _multiplier(x):
    """The largest power of two that keeps 6 * 448 / m above every value."""
    f, e = torch.frexp(x.float().abs().amax())
    power = 11 - (e - 1) - (2 * f > 1.3125).int()
    return torch.where(f > 0, torch.ldexp(torch.ones_like(f), power.clamp(-126, 126)), torch.ones_like(f))


def _blocks(x, scale, m, up):
    """Rounded E2M1 values [rows, blocks, block] and scales [rows, blocks] of x's rows, in units of 1 / m."""
    rows, k = x.shape
    block = BLOCK[scale]
    u = torch.nn.functional.pad(x.float() * m, (0, -k % block)).view(rows, -1, block)
    top = u.abs().amax(-1)
    if scale.startswith("ue4m3"):
        s = (top / 6).clamp(max=448).to(torch.float8_e4m3fn).float()
    else:
        f, e = torch.frexp(top)  # top = f * 2^e, f in [0.5, 1)
        e = e - 3 + (f > 0.75).int() if up else e - 3
        s = torch.ldexp(torch.ones_like(top), torch.where(top > 0, e, -127).clamp(-127, 127))
    y = torch.where(s[..., None] > 0, u / s[..., None], 0.0)
    size = y.abs().clamp(max=6)
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    return torch.copysign(torch.round(size / step) * step, y), s


def _rounded(x, scale, m=1.0, up=False):
    """x after rounding to blocks along its rows, in 32 bits."""
    v, s = _blocks(x, scale, m, up)
    return (v * s[..., None] / m).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _opened(h, scale):
    """A held matrix's values, in 32 bits."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=h["data"].device)
    data, k, block = h["data"], h["k"], BLOCK[scale]
    v = table[torch.stack([data & 15, data >> 4], -1).int()].reshape(data.shape[0], -1)[:, :k]
    t = h["scales"]
    words = t.view(t.shape[0], t.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(t.shape[0] * 128, -1)
    if scale.startswith("ue4m3"):
        s = words.contiguous().view(torch.float8_e4m3fn).float()
    else:
        s = torch.ldexp(torch.ones((), device=words.device), words.int() - 127)
    return v * s[:data.shape[0]].repeat_interleave(block, 1)[:, :k]


def _auto(x, scale):
    return _multiplier(x) if scale == "ue4m3/4" else 1.0


def _plain(s):
    op, scale, dtype = s["op"], s["scale"], DTYPES[s["type"]]
    if op == "round":
        m = _multiplier(s["x"]) if s["auto"] else 1.0
        return _rounded(s["x"].t() if s["columns"] else s["x"], scale, m, s["up"]).to(dtype)
    if op == "serve":
        return (_rounded(s["x"], scale) @ _opened(s["w"], scale).t()).to(dtype)
    if op == "mm":
        d = _opened(s["a"], scale) @ _opened(s["b"], scale).t()
        return (d if s["c"] is None else d + s["c"].float()).to(dtype)
    x, w, g = s["x"].detach(), s["w"].detach(), s["g"]
    mx, mw, mg = _auto(x, scale), _auto(w, scale), _auto(g, scale)
    y = _rounded(x, scale, mx) @ _rounded(w, scale, mw).t()
    dx = _rounded(g, scale, mg) @ _rounded(w.t(), scale, mw).t()
    dw = _rounded(g.t(), scale, mg) @ _rounded(x.t(), scale, mx).t()
    return {"y": y.to(dtype), "dx": dx.to(dtype), "dw": dw.to(dtype)}


# ------------------------------------------------- the framework's calls


def _own(s):
    import tcgen05_b200 as t5

    op, dtype = s["op"], DTYPES[s["type"]]
    scaling, vec = s["scale"].split("/")
    form = {"scaling": scaling, "scale_vec": int(vec)}
    if op == "round":
        if scaling == "ue8m0":
            form["scale_rounding"] = "ceil" if s["up"] else "floor"
        q = t5.quantize_blocks(s["x"], axis=0 if s["columns"] else -1, multiplier="auto" if s["auto"] else None, **form)
        return t5.dequantize_blocks(q, dtype=dtype)
    if op == "serve":
        w = t5.BlockScaledRows(s["w"]["data"], s["w"]["scales"], s["w"]["k"], **form)
        return t5.block_scaled_mm(t5.quantize_blocks(s["x"], **form), w, dtype=dtype)
    if op == "mm":
        a = t5.BlockScaledRows(s["a"]["data"], s["a"]["scales"], s["a"]["k"], **form)
        b = t5.BlockScaledRows(s["b"]["data"], s["b"]["scales"], s["b"]["k"], **form)
        return t5.block_scaled_mm(a, b, s["c"], dtype=dtype)
    y = t5.block_scaled_linear(s["x"], s["w"], **form)
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["g"])
    return {"y": y, "dx": dx, "dw": dw}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# -------------------------------------------------------------- work


def work(case):
    op, size = case["op"], DTYPES[case["type"]].itemsize
    held = 0.5 + 1 / BLOCK[case["scale"]]
    if op == "round":
        n = case["rows"] * case["k"]
        return {"bytes": n * (2 * size + 2 * held), "flops": 4 * n}
    if op == "serve":
        t, n, k = case["tokens"], case["n"], case["k"]
        return {"bytes": t * k * size + n * k * held + t * n * size, "flops": 2 * t * n * k}
    if op == "mm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * k * held + m * n * size * (2 if case["add"] else 1), "flops": 2 * m * n * k}
    t, n, k = case["tokens"], case["n"], case["k"]
    return {"bytes": 2 * size * (t * k + n * k + t * n), "flops": 6 * t * n * k}


# ------------------------------------------------- the definition, in 64 bits


def _grid(v, digits, lowest):
    """v rounded to `digits` significand bits (no quantum below 2^lowest), ties to even, in 64 bits."""
    exponent = torch.floor(torch.log2(torch.where(v > 0, v, 1.0)))
    exponent += (torch.exp2(exponent + 1) <= v).double() - (torch.exp2(exponent) > torch.where(v > 0, v, 1.0)).double()
    quantum = torch.exp2(torch.clamp(exponent - (digits - 1), min=lowest))
    return torch.round(v / quantum) * quantum


def _exact_rounded(x, scale, m, up):
    rows, k = x.shape
    block = BLOCK[scale]
    count = -(-k // block)
    u = torch.zeros(rows, count * block, dtype=torch.float64, device=x.device)
    u[:, :k] = (x.double() * m).float().double()  # the product with m is rounded to 32 bits by definition
    u = u.view(rows, count, block)
    a = u.abs().amax(2, keepdim=True)
    if scale == "ue4m3/4":
        s = _grid(torch.clamp(a / 6, max=448.0), 4, -9)
    else:
        lead = torch.floor(torch.log2(torch.where(a > 0, a, 1.0)))
        lead += (torch.exp2(lead + 1) <= a).double() - (torch.exp2(lead) > torch.where(a > 0, a, 1.0)).double()
        shift = lead - 2
        if up:
            shift = shift + (a > 6 * torch.exp2(shift)).double()
        s = torch.exp2(torch.clamp(torch.where(a > 0, shift, -127.0), -127, 127))
    size = torch.where(s > 0, u.abs() / torch.where(s > 0, s, 1.0), 0.0)
    q = torch.clamp(_grid(torch.clamp(size, max=6.0), 2, -1), max=6.0)
    return (torch.sign(u) * q * s / m).view(rows, count * block)[:, :k]


def _exact_multiplier(x):
    top = float(x.abs().max())
    return 2.0 ** max(-126, min(126, math.floor(math.log2(2688.0) - math.log2(top)))) if top > 0 else 1.0


def _exact_held(h, scale):
    data, k, block = h["data"].long(), h["k"], BLOCK[scale]
    nibble = torch.empty(data.shape[0], 2 * data.shape[1], dtype=torch.int64, device=data.device)
    nibble[:, 0::2], nibble[:, 1::2] = data % 16, data // 16
    e, f = nibble // 2 % 4, nibble % 2
    v = torch.where(e == 0, 0.5 * f, (1 + 0.5 * f) * torch.exp2(e.double() - 1)) * (1 - 2 * (nibble // 8))
    r = torch.arange(data.shape[0], device=data.device)[:, None]
    b = torch.arange(k, device=data.device)[None] // block
    w = h["scales"][r // 128, b // 4, r % 32 * 16 + r % 128 // 32 * 4 + b % 4].long()
    if scale == "ue4m3/4":
        s = torch.where(w // 8 == 0, w % 8 * 2.0 ** -9, (8 + w % 8) * torch.exp2((w // 8).double() - 10))
    else:
        s = torch.exp2(w.double() - 127)
    return v[:, :k] * s


def exact(case, seed):
    s = prepare(case, seed)
    op, scale = case["op"], case["scale"]
    if op == "round":
        m = _exact_multiplier(s["x"]) if case["auto"] else 1.0
        return _exact_rounded(s["x"].t() if case["columns"] else s["x"], scale, m, case["up"])
    if op == "serve":
        return _exact_rounded(s["x"], scale, 1.0, False) @ _exact_held(s["w"], scale).t()
    if op == "mm":
        d = _exact_held(s["a"], scale) @ _exact_held(s["b"], scale).t()
        return d if s["c"] is None else d + s["c"].double()
    x, w, g = s["x"].detach(), s["w"].detach(), s["g"]
    m = [_exact_multiplier(t) if scale == "ue4m3/4" else 1.0 for t in (x, w, g)]
    r = _exact_rounded
    return {"y": r(x, scale, m[0], False) @ r(w, scale, m[1], False).t(),
            "dx": r(g, scale, m[2], False) @ r(w.t(), scale, m[1], False).t(),
            "dw": r(g.t(), scale, m[2], False) @ r(x.t(), scale, m[0], False).t()}
