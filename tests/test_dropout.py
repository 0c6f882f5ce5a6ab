"""Counter-based dropout (ops.dropout) and the LoRA linear with it: the generator
against its published vectors and numpy, values bit for bit, gradients, refusals."""
import math

import numpy as np
import pytest
import torch

from metallora_b200 import _lib, ops
from metallora_b200.exceptions import ConfigurationError, DeviceError, ShapeError
from metallora_b200.layers import LoRALinear

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def philox(key, counter):
    """Philox4x32-10 in Python's integers (Salmon, Moraes, Dror and Shaw, 2011):
    key of two and counter of four 32-bit words."""
    m = 0xFFFFFFFF
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & m, (a >> 32) ^ c[3] ^ k[1], a & m]
        k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
    return c


def halves(n, seed, call):
    """The 16 bits of n elements."""
    out = []
    for b in range(-(-n // 8)):
        ctr = (b & 0xFFFFFFFF, b >> 32, call & 0xFFFFFFFF, call >> 32)
        for w in philox((seed & 0xFFFFFFFF, seed >> 32), ctr):
            out += [w & 0xFFFF, w >> 16]
    return np.array(out[:n])


def factor(shape, p, seed, call):
    t = round(65536 * p)
    kept = torch.from_numpy(halves(math.prod(shape), seed, call) >= t).reshape(shape)
    return kept, np.float32(65536) / np.float32(65536 - t) if t < 65536 else np.float32(0)


# ------------------------------------------------------------------ CPU --

def test_generator_vectors():
    """The known-answer vectors that the generator's authors publish."""
    f = 0xFFFFFFFF
    assert philox((0, 0), (0,) * 4) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox((f, f), (f,) * 4) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox((0xA4093822, 0x299F31D0), (0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344)) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_refusals():
    x = torch.zeros(4, 8)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ConfigurationError):
            ops.dropout(x, p, 1)
    with pytest.raises(DeviceError):
        ops.dropout(x, 0.5, 1)
    assert ops.dropout(x, 0.5, 1, training=False) is x
    w, a, b = torch.zeros(16, 8, requires_grad=True), torch.zeros(8, 8), torch.zeros(16, 8)
    with pytest.raises(ConfigurationError):  # a trained base
        ops.lora_forward(x, w, a, b, dropout=0.5, training=True, dropout_seed=1)
    lib = _lib.load()
    good = dict(x=4096, out=4096, n=8, t=100, seed=1, dev=None, call=0, dtype=0)
    for kw in ({"n": 0}, {"t": -1}, {"t": 65537}, {"dtype": 3}, {"x": None}, {"out": 4097}, {"dev": 4}):
        v = {**good, **kw}
        assert lib.mlora_dropout(v["x"], v["out"], v["n"], v["t"], 1, v["seed"], v["dev"], v["call"],
                                 v["dtype"], None) < 0, kw
    p = 1 << 20

    def lora(K=64, N=64, t=100, dtype=0, saved=p, ws=p, ws_bytes=1 << 30, w0=p):
        return lib.mlora_lora_forward_dropout(p, w0, p, p, p, saved, 16, K, N, 8, 16.0, t, 1, None, 0,
                                              dtype, ws, ws_bytes, None)
    for kw in ({"K": 60}, {"N": 60}, {"t": 65537}, {"dtype": 2}, {"saved": None}, {"ws_bytes": 8},
               {"ws": None}, {"w0": p + 2}):
        assert lora(**kw) < 0, kw


def test_layer_with_a_quantised_base_refuses():
    layer = LoRALinear(64, 64, rank=8, dropout=0.1, dropout_seed=3)
    layer.qweight = object()
    with pytest.raises(ConfigurationError):
        layer(torch.zeros(2, 64))


# ------------------------------------------------------------------ GPU --

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (33, 5), (3, 50, 17), (128, 264)])
@pytest.mark.parametrize("p,seed,call", [(0.1, 1, 0), (0.5, (1 << 63) + 12345, (1 << 40) + 7),
                                         (0.0, 5, 1), (1.0, 5, 1), (1e-6, 2, 3)])
def test_values_bit_for_bit(cuda, dtype, shape, p, seed, call):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(dtype)
    kept, scale = factor(shape, p, seed, call)
    # one product in 32 bits, rounded once to the type
    want = torch.where(kept, (x.float() * float(scale)).to(dtype), torch.zeros((), dtype=dtype))
    xg = x.to(cuda).requires_grad_(True)
    got = ops.dropout(xg, p, seed, call=call)
    assert got.dtype == dtype and torch.equal(got.detach().cpu(), want)
    dx = torch.autograd.grad(got, xg, torch.ones_like(got))[0].cpu()  # the same mask
    assert torch.equal(dx, torch.where(kept, torch.tensor(float(scale)).to(dtype), torch.zeros((), dtype=dtype)))


@pytest.mark.gpu
def test_dropped_elements_are_zero_whatever_they_were(cuda):
    x = torch.full((64,), float("inf"), device=cuda)
    x[::2] = float("nan")
    kept, _ = factor((64,), 0.5, 9, 0)
    got = ops.dropout(x, 0.5, 9).cpu()
    assert torch.count_nonzero(got[~kept]) == 0 and not torch.isfinite(got[kept]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_orders_strides_and_alignment(cuda, dtype):
    base = torch.randn(40, 70, device=cuda).to(dtype)
    flat = base.flatten()
    for x in (base.t(), base[:, 3:20], base[::2], flat[1:1000], flat[3:]):
        assert torch.equal(ops.dropout(x, 0.3, 4), ops.dropout(x.contiguous().clone(), 0.3, 4))
    assert ops.dropout(base[:0], 0.3, 4).shape == (0, 70)
    wide = torch.randn(70, device=cuda).to(dtype).expand(40, 70).requires_grad_(True)
    assert torch.equal(ops.dropout(wide, 0.3, 4), ops.dropout(wide.contiguous(), 0.3, 4))


@pytest.mark.gpu
def test_rate_calls_and_seeds(cuda):
    """A kept share within five deviations; other calls and seeds, other masks."""
    n = 1 << 22
    x = torch.ones(n, device=cuda)
    seen = []
    for seed, call in ((1, 0), (1, 1), (2, 0), (1 + (1 << 32), 0)):
        kept = ops.dropout(x, 0.25, seed, call=call) > 0
        assert abs(float(kept.float().mean()) - 0.75) < 5 * math.sqrt(0.25 * 0.75 / n)
        seen.append(kept)
    for i in range(4):
        for j in range(i):
            both = float((seen[i] & seen[j]).float().mean())
            assert abs(both - 0.75 ** 2) < 5 * math.sqrt(0.5 / n)


@pytest.mark.gpu
def test_seed_tensor_in_a_graph(cuda):
    seed = torch.tensor([77], device=cuda)
    x = torch.randn(100, 33, device=cuda, dtype=BF16).requires_grad_(True)
    assert torch.equal(ops.dropout(x, 0.2, seed), ops.dropout(x, 0.2, 77))
    neg = torch.tensor([-5], device=cuda)  # the same 64 bits
    assert torch.equal(ops.dropout(x, 0.2, neg), ops.dropout(x, 0.2, -5))
    assert torch.equal(ops.dropout(x, 0.2, neg), ops.dropout(x, 0.2, 2 ** 64 - 5))
    dy = torch.randn_like(x).detach()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.dropout(x, 0.2, seed, call=6)
        dx = torch.autograd.grad(out, x, dy)[0]
    for s in (77, 123456789):
        seed.fill_(s)
        graph.replay()
        want = ops.dropout(x, 0.2, s, call=6)
        assert torch.equal(out, want) and torch.equal(dx, torch.autograd.grad(want, x, dy)[0])
    y = ops.dropout(x, 0.2, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError):  # another mask than the forward's: noticed
        y.sum().backward()
    with pytest.raises(ShapeError):
        ops.dropout(x, 0.2, torch.zeros(2, dtype=torch.int64, device=cuda))
    with pytest.raises(DeviceError):
        ops.dropout(x, 0.2, torch.zeros(1, dtype=torch.int64))


def _lora_case(m, k, n, r, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*s):
        return torch.randn(s, generator=g, device="cuda")
    return ((randn(m, k)).to(dtype), (randn(n, k) / math.sqrt(k)).to(dtype),
            (randn(r, k) / math.sqrt(k)).to(dtype), (randn(n, r) * 0.2).to(dtype),
            randn(m, n).to(dtype))


def _lora_check(x, w, a, b, dy, got, p, seed, call, alpha, grads=True):
    """Against 64 bits, every element within the roundings' bound: s x A^T, dropout(dy)
    and s dropout(dy) B are 16-bit operands, the LoRA term a 16-bit value at most, and
    the results are rounded once more."""
    h = torch.finfo(x.dtype).eps / 2
    sub = 2.0 ** -24 if x.dtype == FP16 else 0.0
    eps = 2.0 ** -19  # of sums in 32 bits
    kept, scale = factor(dy.shape, p, seed, call)
    f = kept.to(x.device).double() * float(scale)
    xd, wd, ad, bd, dyd = (t.detach().double() for t in (x, w, a, b, dy))
    sc = alpha / a.shape[0]
    xa = sc * xd @ ad.T
    z = xa @ bd.T
    y = xd @ wd.T + f * z
    ez = f * (h * xa.abs() @ bd.abs().T + 2 * h * z.abs() + sub)
    bound = ez + h * (y.abs() + ez) + eps * (xd.abs() @ wd.abs().T + f * (xa.abs() @ bd.abs().T)) + sub
    assert ((got[0].double() - y).abs() - bound).max() <= 0
    if not grads:
        return
    dz = f * dyd
    u = sc * dz @ bd
    eu = sc * (h + eps) * dz.abs() @ bd.abs() + h * u.abs() + sub
    dx = dyd @ wd + u @ ad
    bound = eu @ ad.abs() + h * dx.abs() * 1.01 + eps * (dyd.abs() @ wd.abs() + u.abs() @ ad.abs()) + sub
    assert ((got[1].double() - dx).abs() - bound).max() <= 0
    da, db = u.T @ xd, dz.T @ xa
    assert ((got[2].double() - da).abs() - (eu.T @ xd.abs() + h * da.abs() * 1.01 + sub
                                            + eps * (u.abs().T @ xd.abs()))).max() <= 0
    assert ((got[3].double() - db).abs() - ((2 * h + eps) * dz.abs().T @ xa.abs() * 1.01
                                            + h * db.abs() * 1.01 + sub)).max() <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,k,n,r,p", [(1, 64, 8, 8, 0.5), (16, 256, 128, 16, 0.1), (130, 72, 264, 5, 0.3),
                                       (257, 512, 520, 64, 0.05), (300, 136, 1000, 200, 0.9),
                                       (515, 64, 256, 8, 1.0)])
def test_lora_linear(cuda, dtype, m, k, n, r, p):
    x, w, a, b, dy = _lora_case(m, k, n, r, dtype, seed=m)
    for t in (x, a, b):
        t.requires_grad_(True)
    y = ops.lora_forward(x, w, a, b, alpha=2.0 * r, dropout=p, training=True, dropout_seed=11,
                         dropout_call=4)
    got = (y.detach(), *torch.autograd.grad(y, (x, a, b), dy))
    _lora_check(x, w, a, b, dy, got, p, 11, 4, 2.0 * r)
    assert _lib.device_status(reset=True) == 0


@pytest.mark.gpu
def test_lora_linear_corner_calls(cuda):
    x, w, a, b, dy = _lora_case(96, 128, 256, 16, BF16, seed=3)
    kw = dict(alpha=32.0, dropout=0.2, training=True, dropout_seed=5)
    e = ops.lora_forward(x[:0], w, a.requires_grad_(True), b.requires_grad_(True), **kw)
    assert e.shape == (0, 256)
    for g in torch.autograd.grad(e, (a, b), dy[:0]):
        assert torch.count_nonzero(g) == 0
    # strides and leading axes; gradients of A and B alone; fp32 factors
    y3 = ops.lora_forward(x.reshape(4, 24, 128), w, a, b, **kw)
    xt = x.t().contiguous().t()
    a32, b32 = a.detach().float().requires_grad_(True), b.detach().float().requires_grad_(True)
    yt = ops.lora_forward(xt, w.t().contiguous().t(), a32, b32, **kw)
    assert y3.shape == (4, 24, 256) and torch.equal(y3.reshape(96, 256), yt)
    ga = torch.autograd.grad(y3, (a, b), dy.reshape(4, 24, 256))
    gt = torch.autograd.grad(yt, (a32, b32), dy)
    assert gt[0].dtype == FP32
    for u, v in zip(ga, gt):  # the fp32 ones before their rounding
        assert torch.equal(u, v.to(BF16))
    # without training, or without a seed, the forward is the one that it was
    plain = ops.lora_forward(x, w, a, b, alpha=32.0)
    assert torch.equal(ops.lora_forward(x, w, a, b, alpha=32.0, dropout=0.2, dropout_seed=5), plain)
    assert torch.equal(ops.lora_forward(x, w, a, b, alpha=32.0, dropout=0.0, training=True,
                                        dropout_seed=5), plain)


@pytest.mark.gpu
def test_lora_layer_calls_and_graph(cuda):
    layer = LoRALinear(128, 264, rank=8, alpha=16.0, dropout=0.25, device=cuda, dtype=BF16,
                       dropout_seed=21)
    with torch.no_grad():
        layer.W0.normal_(0, 0.1)
        layer.B.normal_(0, 0.1)
    x = torch.randn(50, 128, device=cuda, dtype=BF16)
    outs = [layer(x) for _ in range(2)]
    assert layer.dropout_call == 2 and not torch.equal(*outs)
    layer.dropout_call = 0
    assert torch.equal(layer(x), outs[0])
    for i, out in enumerate(outs):
        _lora_check(x, layer.W0, layer.A, layer.B, torch.zeros(50, 264, device=cuda, dtype=BF16),
                    (out.detach(),), 0.25, 21, i, 16.0, grads=False)
    layer.eval()
    layer(x)
    assert layer.dropout_call == 1
    layer.train()
    seed = torch.tensor([21], device=cuda)
    layer.dropout_seed, layer.dropout_call = seed, 0
    del outs, out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x)
        ga, gb = torch.autograd.grad(y, (layer.A, layer.B), torch.ones_like(y))
    for s in (21, 22):
        seed.fill_(s)
        graph.replay()
        layer.dropout_call = 0
        want = layer(x)
        wa, wb = torch.autograd.grad(want, (layer.A, layer.B), torch.ones_like(want))
        assert torch.equal(y, want) and torch.equal(ga, wa) and torch.equal(gb, wb)


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    n = 2 ** 31 + 43
    x = torch.ones(n, device=cuda, dtype=BF16)
    got = ops.dropout(x, 0.25, 12, call=3)
    t = round(65536 * 0.25)
    for first in (0, 2 ** 31 - 16, n // 8 * 8 - 64):
        want = []
        for b in range(first // 8, min(first // 8 + 9, -(-n // 8))):
            for w in philox((12, 0), (b & 0xFFFFFFFF, b >> 32, 3, 0)):
                want += [w & 0xFFFF, w >> 16]
        part = got[first:first + 72].cpu()
        assert torch.equal(part > 0, torch.tensor([u >= t for u in want])[:part.numel()])

