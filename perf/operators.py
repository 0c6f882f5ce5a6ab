"""Microscaled LoRA operators: MXFP4 base weights and MXINT8 activation checkpoints.

Both formats share one power-of-two scale X among 32 consecutive features of a
row (the last block of a row may be shorter); with e = floor(log2 max|x|) over
the block:

* MXFP4:  X = 2^max(e - 2, -127), value = X * e2m1(x / X), round to nearest
  even on {0, .5, 1, 1.5, 2, 3, 4, 6}, saturating at 6;
* MXINT8: X = 2^max(e, -127), value = X / 64 * clamp(rint(64 x / X), -127, 127).

Operators: quantise and dequantise (weights to MXFP4, activations to MXINT8);
the LoRA linear over an MXFP4 base, ``Q4(x).W^T + s (x.A^T).B^T``, where the
base product multiplies MXFP4 by MXFP4; the LoRA gradients taken from the
8-bit checkpoint of x; and the training step made of them.

A case runs in its plain form (elementary torch operations) where ``own`` is
False and through the framework's entry points where it is True.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------- cases --

def listed():
    """Sizes: the layer shapes of this repository's benchmark (4096 -> 4096,
    4096 -> 11008 rank 64, 4096 -> 14336) and its 8192-token training batch."""
    return [
        # a short prompt's activations kept for the backward: latency
        {"name": "checkpoint 64x4096 bf16", "op": "act", "m": 64, "k": 4096, "dt": "bf16"},
        # the training batch's input of one layer
        {"name": "checkpoint 8192x4096 bf16", "op": "act", "m": 8192, "k": 4096, "dt": "bf16"},
        # a ragged batch, a feature count that ends inside a block
        {"name": "checkpoint 2001x1000 fp16", "op": "act", "m": 2001, "k": 1000, "dt": "fp16"},
        # loading a base weight
        {"name": "weight 11008x4096 bf16", "op": "weight", "m": 11008, "k": 4096, "dt": "bf16"},
        # one generated token; a small decoding batch
        {"name": "forward 1 tok 4096-11008", "op": "fwd", "m": 1, "k": 4096, "n": 11008, "r": 64, "dt": "bf16"},
        {"name": "forward 16 tok 4096-4096", "op": "fwd", "m": 16, "k": 4096, "n": 4096, "r": 16, "dt": "bf16"},
        # a ragged prompt into a wide layer, fp16
        {"name": "forward 333 tok 4096-14336", "op": "fwd", "m": 333, "k": 4096, "n": 14336, "r": 8, "dt": "fp16"},
        # prefill
        {"name": "forward 4096 tok 4096-11008", "op": "fwd", "m": 4096, "k": 4096, "n": 11008, "r": 64, "dt": "bf16"},
        # the adapter's gradients of the training batch, from the checkpoint
        {"name": "grads 8192 tok 4096-4096", "op": "grads", "m": 8192, "k": 4096, "n": 4096, "r": 16, "dt": "bf16"},
        # the same for a ragged fp16 batch, a wide layer and a larger rank
        {"name": "grads 1001 tok 4096-11008", "op": "grads", "m": 1001, "k": 4096, "n": 11008, "r": 64, "dt": "fp16"},
        # forward and backward of one layer, MXFP4 base and checkpoint together
        {"name": "step 2048 tok 4096-4096", "op": "step", "m": 2048, "k": 4096, "n": 4096, "r": 16, "dt": "bf16"},
        {"name": "step 8192 tok 4096-4096", "op": "step", "m": 8192, "k": 4096, "n": 4096, "r": 16, "dt": "bf16"},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["act", "weight", "fwd", "fwd", "grads", "step"])
    dt = rng.choice(["bf16", "fp16"])
    m = _log_uniform(rng, 1, 8192)
    if op == "act":
        return {"op": op, "m": m, "k": 8 * _log_uniform(rng, 8, 1376), "dt": dt}
    if op == "weight":
        return {"op": op, "m": _log_uniform(rng, 64, 11008), "k": 32 * _log_uniform(rng, 2, 344), "dt": dt}
    k, n = 32 * _log_uniform(rng, 4, 256), 8 * _log_uniform(rng, 16, 1376)
    r = rng.choice([4, 8, 16, 24, 32, 64, 128])
    if op == "step":
        m, n, k = max(8, min(m, 4096)), min(n, 4096), min(k, 4096)
    elif op == "grads":
        m, k = max(8, m), 8 * _log_uniform(rng, 16, 1024)
        r = max(8, r)
    return {"op": op, "m": m, "k": k, "n": n, "r": r, "dt": dt}


# ------------------------------------------------------------ plain formats --

def _blocks(x):
    """[rows, blocks, 32] in 32 bits (rows padded with zeros) and each block's
    floor(log2 max|x|), -200 for an all-zero block.  Scaling by a power of two
    is exact, so values next to a rounding border stay on their side of it."""
    m, k = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -k % 32)).view(m, -1, 32)
    amax = v.abs().amax(-1)
    e = torch.frexp(amax)[1] - 1
    return v, torch.where(amax > 0, e, torch.full_like(e, -200))


def _pow2(e):
    """2^e in 32 bits (formed in 64: exact for every exponent)."""
    return torch.exp2(e.double()).float()


def _mxfp4_codes(x):
    """(codes [m, k/2] with the even feature in the low nibble, scale bytes [m, k/32])."""
    v, e = _blocks(x)
    e = (e - 2).clamp_min(-127)
    u = v * _pow2(-e)[..., None]
    a = u.abs()
    mag = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
           + (a >= 3.5) + (a > 5.0))
    code = (mag + 8 * (u < 0)).to(torch.uint8).reshape(x.shape[0], -1)[:, : x.shape[1]]
    return code[:, 0::2] | (code[:, 1::2] << 4), (e + 127).to(torch.uint8)


def _mxfp4_values(codes, scales, dtype):
    """The values of codes and scale bytes, in ``dtype``."""
    grid = torch.tensor(_GRID, device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1).long()
    v = grid[c & 7] * (1 - 2 * (c >> 3))
    x = _pow2(scales.int() - 127).repeat_interleave(32, -1)[:, : c.shape[1]]
    return (v * x).to(dtype)


def _mxint8_codes(x):
    """(codes [m, k] int8, exponents [m, ceil(k/32)])."""
    v, e = _blocks(x)
    e = e.clamp_min(-127)
    q = torch.round(v * _pow2(-e)[..., None] * 64).clamp(-127, 127)
    return q.reshape(x.shape[0], -1)[:, : x.shape[1]].to(torch.int8), e


def _mxint8_values(codes, e, dtype):
    x = _pow2(e - 6).repeat_interleave(32, -1)[:, : codes.shape[1]]
    return (codes.float() * x).to(dtype)


# --------------------------------------------------------------------- state --

def _randn(gen, *shape, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale


def _acts(gen, m, k, dtype):
    """Activations as they come out of a normalisation: unit variance, tokens of
    different size and a few strong feature channels."""
    x = _randn(gen, m, k) * (1 + 3 * (torch.rand((m, 1), generator=gen, device="cuda") > 0.9))
    strong = torch.rand((1, k), generator=gen, device="cuda") > 0.995
    return (x * (1 + 15 * strong)).to(dtype)


def _tile_rank(r):
    t = 16
    while t < r:
        t *= 2
    return t


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, m, k = _DT[case["dt"]], case["m"], case["k"]
    s = {"case": case}
    if case["op"] == "act":
        s["x"] = _acts(gen, m, k, dt)
        return s
    if case["op"] == "weight":
        s["w"] = _randn(gen, m, k, scale=0.02).to(dt)
        return s
    n, r = case["n"], case["r"]
    s["alpha"] = 2.0 * r
    s["a"] = ((torch.rand((r, k), generator=gen, device="cuda") * 2 - 1) / math.sqrt(k)).to(dt)
    s["b"] = _randn(gen, n, r, scale=0.05).to(dt)
    x = _acts(gen, m, k, dt)
    if case["op"] == "grads":
        s["dy"] = _randn(gen, m, n, scale=0.1).to(dt)
        codes, e = _mxint8_codes(x)
        # the checkpoint: rows of codes start on 16 bytes; a word of four scale
        # bytes per 128 features and row, the rows rounded up to 4
        s["codes"] = torch.zeros((m, -(-k // 16) * 16), dtype=torch.int8, device="cuda")[:, :k]
        s["codes"].copy_(codes)
        g = -(-k // 128)
        words = torch.zeros((-(-m // 4) * 4, g * 4), dtype=torch.uint8, device="cuda")
        words[:m, : e.shape[1]] = (e + 127).to(torch.uint8)
        s["scales"] = words.view(-1, g, 4).transpose(0, 1).contiguous()
        # the forward's (alpha/r) x.A^T, as it keeps it: [rank tile, tokens rounded to 8]
        s["saved"] = torch.zeros((_tile_rank(r), -(-m // 8) * 8), dtype=dt, device="cuda")
        s["saved"][:r, :m] = (2.0 * (x.float() @ s["a"].float().t())).t().to(dt)
        return s
    s["wcodes"], s["wscales"] = _mxfp4_codes(_randn(gen, n, k, scale=0.02).to(dt))
    s["x"] = x
    if case["op"] == "step":
        s["dy"] = _randn(gen, m, n, scale=0.1).to(dt)
        for t in ("x", "a", "b"):
            s[t].requires_grad_(True)
    return s


def _weight(s):
    """The base weight as a program holds it: wrapped when it is loaded."""
    from metallora_b200 import quant
    if "qw" not in s:
        c = s["case"]
        s["qw"] = quant.from_reference_layout("mxfp4", s["wcodes"], s["wscales"], None,
                                              (c["n"], c["k"]), 32)
    return s["qw"]


def _run_own(s):
    from metallora_b200 import ops, quant
    op = s["case"]["op"]
    if op == "act":
        return quant.checkpoint_activation(s["x"]).dequantize()
    if op == "weight":
        return quant.quantize(s["w"], "mxfp4").dequantize(s["w"].dtype)
    if op == "fwd":
        with torch.no_grad():
            return ops.qlora_forward(s["x"], _weight(s), s["a"], s["b"], s["alpha"])
    if op == "grads":
        ckpt = quant.ActivationCheckpoint(s["codes"], s["scales"],
                                          (s["case"]["m"], s["case"]["k"]), s["dy"].dtype)
        return ops.lora_backward(s["dy"], ckpt, s["a"], s["b"], s["alpha"], clip_value=None,
                                 saved_xa=s["saved"])
    y = ops.qlora_forward(s["x"], _weight(s), s["a"], s["b"], s["alpha"], checkpoint="mxint8")
    return (y.detach(), *torch.autograd.grad(y, (s["x"], s["a"], s["b"]), s["dy"]))


def _run_plain(s):
    case = s["case"]
    op, dt = case["op"], _DT[case["dt"]]
    if op == "act":
        return _mxint8_values(*_mxint8_codes(s["x"]), dt)
    if op == "weight":
        return _mxfp4_values(*_mxfp4_codes(s["w"]), dt)
    a, b, sc = s["a"].detach().float(), s["b"].detach().float(), s["alpha"] / case["r"]
    if op == "grads":
        dy = s["dy"].float()
        words = s["scales"].transpose(0, 1).flatten(1)[: case["m"], : -(-case["k"] // 32)]
        xh = _mxint8_values(s["codes"], words.int() - 127, torch.float32)
        da = (sc * (dy @ b)).t() @ xh
        db = dy.t() @ s["saved"][: case["r"], : case["m"]].t().float()
        return da.to(dt), db.to(dt)
    x = s["x"].detach().float()
    w = _mxfp4_values(s["wcodes"], s["wscales"], torch.float32)
    xq = _mxfp4_values(*_mxfp4_codes(s["x"].detach()), torch.float32)
    xa = sc * (x @ a.t())
    y = (xq @ w.t() + xa @ b.t()).to(dt)
    if op == "fwd":
        return y
    dy = s["dy"].float()
    u = sc * (dy @ b)
    xh = _mxint8_values(*_mxint8_codes(s["x"].detach()), torch.float32)
    return y, (dy @ w + u @ a).to(dt), (u.t() @ xh).to(dt), (dy.t() @ xa).to(dt)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    m, k = case["m"], case["k"]
    if case["op"] in ("act", "weight"):  # values in, values out
        return {"bytes": 4 * m * k, "flops": 2 * m * k}
    n, r = case["n"], case["r"]
    weight = n * k // 2 + n * (k // 32) + 2 * r * (n + k)
    fwd = {"bytes": 2 * m * k + weight + 2 * m * n, "flops": 2 * m * n * k + 2 * m * r * (n + k)}
    if case["op"] == "fwd":
        return fwd
    if case["op"] == "grads":
        return {"bytes": 2 * m * n + m * k + m * -(-k // 32) + 2 * m * r + 2 * r * (2 * n + k),
                "flops": 2 * m * r * (2 * n + k)}
    # y, dx, dA and dB from x, dy and the weights
    return {"bytes": 4 * m * (k + n) + weight + 2 * r * (n + k),
            "flops": 4 * m * n * k + 2 * m * r * (2 * n + k) + 4 * m * r * k + 2 * m * r * n}


# ------------------------------------------------------- 64-bit definitions --

def _exact_mx(x, top, grid):
    """Values of the block format by its definition, in 64 bits: block scale
    2^max(floor(log2 max) - top, -127) and ``grid`` rounding on the scaled values."""
    m, k = x.shape
    pad = -k % 32
    v = torch.nn.functional.pad(x.double(), (0, pad)).unflatten(-1, (-1, 32))
    big = v.abs().max(-1, keepdim=True).values
    ex = torch.floor(torch.log2(big.clamp_min(1e-300)))
    ex = torch.where(torch.exp2(ex) > big, ex - 1, ex)  # log2 rounded up to the next power
    ex = torch.where(torch.exp2(ex + 1) <= big, ex + 1, ex)
    scale = torch.exp2((ex - top).clamp_min(-127.0))
    return (grid(v / scale) * scale).flatten(1)[:, :k]


def _round_fp4(u):
    a = u.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return torch.sign(u) * (torch.round(a / step) * step).clamp_max(6.0)


def _round_int8(u):
    return torch.round(u * 64).clamp(-127, 127) / 64


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "act":
        return _exact_mx(s["x"], 0, _round_int8)
    if op == "weight":
        return _exact_mx(s["w"], 2, _round_fp4)
    m, k, r = case["m"], case["k"], case["r"]
    a, b, sc = s["a"].detach().double(), s["b"].detach().double(), s["alpha"] / r
    if op == "grads":
        by = s["scales"].permute(1, 0, 2).flatten(1)[:m, torch.arange(k, device="cuda") // 32]
        xh = s["codes"].double() / 64 * torch.exp2(by.double() - 127)
        dy = s["dy"].double()
        return sc * (b.t() @ (dy.t() @ xh)), (s["saved"][:r, :m].double() @ dy).t()
    nib = torch.stack((s["wcodes"] % 16, s["wcodes"] // 16), 2).flatten(1)
    mag = nib % 8
    half = torch.where(mag < 2, mag.double() / 2,
                       (2 + mag % 2).double() * torch.exp2((mag // 2).double() - 2))
    sign = torch.where(nib > 7, -1.0, 1.0)
    w = half * sign * torch.exp2(s["wscales"].double() - 127).repeat_interleave(32, 1)
    x = s["x"].detach().double()
    xa = sc * (x @ a.t())
    y = _exact_mx(s["x"].detach(), 2, _round_fp4) @ w.t() + xa @ b.t()
    if op == "fwd":
        return y
    dy = s["dy"].double()
    xh = _exact_mx(s["x"].detach(), 0, _round_int8)
    return y, dy @ w + sc * (dy @ b) @ a, sc * (b.t() @ (dy.t() @ xh)), dy.t() @ xa
