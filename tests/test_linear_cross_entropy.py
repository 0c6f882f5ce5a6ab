"""Cross entropy of a linear head from the hidden states (ops.linear_cross_entropy):
refusals on the CPU; losses and gradients against 64 bits on the GPU, with bounds
derived from the roundings."""
import math

import pytest
import torch

from metallora_b200 import _lib, ops
from metallora_b200.exceptions import ConfigurationError, DeviceError, ShapeError

BF16, FP16 = torch.bfloat16, torch.float16
IGNORE = -100


# ------------------------------------------------------------------ CPU --

def test_refusals():
    x, w = torch.zeros(4, 16, dtype=BF16), torch.zeros(32, 16, dtype=BF16)
    y = torch.zeros(4, dtype=torch.int64)
    a, b = torch.zeros(8, 16, dtype=BF16), torch.zeros(32, 8, dtype=BF16)
    with pytest.raises(DeviceError):
        ops.linear_cross_entropy(x, w, y)
    for kw in ({"reduction": "avg"}, {"A": a}, {"B": b}):
        with pytest.raises(ConfigurationError):
            ops.linear_cross_entropy(x, w, y, **kw)
    with pytest.raises(ConfigurationError):  # a gradient per token reaches x alone
        ops.linear_cross_entropy(x, w.requires_grad_(True), y, reduction="none")
    w = w.detach()
    with pytest.raises(ShapeError):
        ops.linear_cross_entropy(x[:, :8], w, y)
    with pytest.raises(ShapeError):
        ops.linear_cross_entropy(x, w, y[:3])


def test_c_entry_refusals():
    """Sizes, flags, pointers and buffers are checked before a device is touched."""
    lib = _lib.load()
    p = 1 << 20  # an aligned address that is never read

    def call(M=16, K=64, V=100, r=0, dtype=0, grads=1, w=p, a=None, b=None, loss=p, rows=None,
             state=p, state_bytes=1 << 40, ws=p, ws_bytes=1 << 40):
        return lib.mlora_linear_cross_entropy(p, w, a, b, p, loss, rows, state, state_bytes, M, K,
                                              V, r, 16.0, IGNORE, 1, dtype, grads, ws, ws_bytes,
                                              None)

    bad, unsupported, space = (_lib.MLORA_ERR_INVALID_ARG, _lib.MLORA_ERR_UNSUPPORTED,
                               _lib.MLORA_ERR_WORKSPACE)
    for want, kw in ((bad, {"M": 0}), (bad, {"V": -1}), (unsupported, {"K": 60}),
                     (unsupported, {"dtype": 2}), (bad, {"grads": 8}), (bad, {"grads": 4}),
                     (unsupported, {"r": 8, "V": 100, "a": p, "b": p}), (bad, {"r": 8, "V": 104}),
                     (bad, {"r": 257}), (unsupported, {"M": 1 << 31}), (bad, {"w": None}),
                     (bad, {"w": p + 2}), (bad, {"loss": None}), (space, {"state_bytes": 10}),
                     (space, {"state": p + 16}), (space, {"ws_bytes": 10}), (space, {"ws": None})):
        assert call(**kw) == want, kw
    back = (p, 1 << 40, p, 1, 0, p, p, p, p, 0, 0, None, 16, 64, 104, 8, 0)
    assert lib.mlora_linear_cross_entropy_backward(*back, 5, None) == unsupported
    assert lib.mlora_linear_cross_entropy_backward(*back, 1, None) == bad  # da without its flag
    assert lib.mlora_linear_cross_entropy_state_bytes(0, 64, 100, 0, 0, 1) == 0
    assert lib.mlora_linear_cross_entropy_workspace_bytes(16, 60, 100, 0, 0, 1) == 0


def test_memory_does_not_grow_with_the_logits():
    lib = _lib.load()
    for grads, bound in ((0, 5 << 29), (1, 5 << 29)):
        ws = lib.mlora_linear_cross_entropy_workspace_bytes(32768, 4096, 128000, 0, 0, grads)
        assert ws < bound + 32768 * 4096 * 2 < 32768 * 128000 * 2
    state = lib.mlora_linear_cross_entropy_state_bytes(32768, 4096, 128000, 0, 0, 1)
    assert state < 2 * 32768 * 4096 * 4


# ------------------------------------------------------------------ GPU --

def _case(m, k, v, dtype, r=0, seed=0, size=1.3, lean=12.0, dev="cuda"):
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*s):
        return torch.randn(s, generator=g, device=dev)
    w = (randn(v, k) * size / math.sqrt(k)).to(dtype)
    y = torch.randint(0, v, (m,), generator=g, device=dev)
    x = (randn(m, k) + lean * torch.rand((m, 1), generator=g, device=dev) * w[y].float()).to(dtype)
    if not r:
        return x, w, y, None, None
    a = (randn(r, k) / math.sqrt(k)).to(dtype)
    return x, w, y, a, (randn(v, r) * 0.1).to(dtype)


def _check(x, w, y, a=None, b=None, alpha=16.0, upstream=1.0, reduction="mean"):
    """Loss and gradients of the call against 64 bits."""
    dtype = x.dtype
    h = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -31 if dtype == FP16 else 0.0  # half a subnormal step of 64 g in fp16
    sub = 2.0 ** -25 if dtype == FP16 else 0.0   # of the outputs
    leaves = [t for t in (x, w, a, b) if t is not None and t.requires_grad]
    loss = ops.linear_cross_entropy(x, w, y, A=a, B=b, alpha=alpha, reduction=reduction)
    assert loss.dtype == torch.float32
    xd, wd = x.detach().double(), w.detach().double()
    m, k = x.shape
    counted = (y >= 0) & (y < w.shape[0])
    n = int(counted.sum())
    at = y.clamp(0, w.shape[0] - 1)[:, None]
    logits = xd @ wd.T
    # fp32 sums of exact products: a random walk of K roundings, four deviations
    dl = 2.0 ** -24 * 4 * math.sqrt(k) * float((xd.norm(dim=1).max() * wd.norm(dim=1).max())) + 2e-6
    if a is not None:
        ad, bd, sc = a.detach().double(), b.detach().double(), alpha / a.shape[0]
        xa = sc * (xd @ ad.T)
        logits = logits + xa @ bd.T
        dl += float((h * (xa.abs() @ bd.abs().T)).max())  # s x A^T enters in 16 bits
    nll = (torch.logsumexp(logits, 1) - logits.gather(1, at)[:, 0]) * counted
    # a loss is off by at most twice its logits, a probability by that fraction
    tol = 2 * dl + 2.0 ** -22 * float(nll.abs().max())
    if reduction == "none":
        assert (loss.double() - nll).abs().max() <= tol
        per = upstream
    else:
        want = nll.sum() / (n if reduction == "mean" else 1)
        if reduction == "mean" and n == 0:
            assert torch.isnan(loss)
        else:
            assert (loss.double() - want).abs() <= tol * (1 if reduction == "mean" else max(n, 1))
        per = torch.full((m,), upstream / (n if reduction == "mean" and n else 1),
                         dtype=torch.float64, device=x.device)
    if not leaves:
        return loss
    up = per.float() if reduction == "none" else torch.tensor(upstream, device=x.device)
    got = dict(zip([id(t) for t in leaves], torch.autograd.grad(loss, leaves, up)))
    p = torch.softmax(logits, 1)
    keep = (counted * per)[:, None]
    g = (p - torch.zeros_like(p).scatter_(1, at, 1.0)) * keep
    # g in 16 bits, once or by way of an 11-bit exp; the target's rounding is given back to dx
    rel = h + 2.0 ** -11 + 2 * dl
    off = (p * rel + tiny) * keep.abs()
    eg = off + h * g.abs()  # where it is not
    eps = 2.0 ** -20
    if a is not None:
        u = sc * (g @ bd)
        eu = sc * (eg @ bd.abs()) + h * u.abs() + eps * sc * (g.abs() @ bd.abs())
    if x.requires_grad:
        dx, bound = g @ wd, off @ wd.abs() + eps * (g.abs() @ wd.abs())
        if a is not None:
            dx, bound = dx + u @ ad, bound + eu @ ad.abs() + eps * (u.abs() @ ad.abs())
        e = (got[id(x)].double() - dx).abs() - (bound + h * dx.abs() * 1.01 + sub)
        assert e.max() <= 0, f"dx beyond its bound by {e.max()}"
        assert torch.count_nonzero(got[id(x)][~counted]) == 0
    if w.requires_grad:
        dw = g.T @ xd
        e = (got[id(w)].double() - dw).abs() - (eg.T @ xd.abs() + h * dw.abs() * 1.01 + sub
                                                + eps * (g.abs().T @ xd.abs()))
        assert e.max() <= 0, f"dW beyond its bound by {e.max()}"
    if a is not None and a.requires_grad:
        ho = h if a.dtype == dtype else 2.0 ** -24
        da, db = u.T @ xd, g.T @ xa
        e = (got[id(a)].double() - da).abs() - (eu.T @ xd.abs() + ho * da.abs() * 1.01 + sub
                                                + eps * (u.abs().T @ xd.abs()))
        assert e.max() <= 0, f"dA beyond its bound by {e.max()}"
        e = (got[id(b)].double() - db).abs() - ((eg + (h + eps) * g.abs()).T @ xa.abs()
                                                + ho * db.abs() * 1.01 + sub)
        assert e.max() <= 0, f"dB beyond its bound by {e.max()}"
    assert _lib.device_status(reset=True) == 0
    return loss


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,k,v", [(1, 8, 1), (1, 64, 7), (3, 128, 257), (16, 4096, 1000),
                                   (255, 72, 300), (257, 1032, 5003), (700, 256, 20001),
                                   (1030, 512, 4096)])
def test_frozen_head(cuda, dtype, m, k, v):
    x, w, y, _, _ = _case(m, k, v, dtype, seed=m + v)
    y[: m // 3] = IGNORE
    _check(x.requires_grad_(True), w, y, upstream=0.7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,k,v", [(1, 8, 1), (5, 64, 33), (130, 264, 1001), (300, 512, 2000),
                                   (1100, 136, 777)])
def test_trained_head(cuda, dtype, m, k, v):
    x, w, y, _, _ = _case(m, k, v, dtype, seed=m)
    y[::5] = IGNORE
    _check(x.requires_grad_(True), w.requires_grad_(True), y, reduction="sum")
    _check(x.detach(), w, y)  # of the weight alone


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,k,v,r", [(1, 64, 8, 8), (40, 256, 1000, 16), (300, 136, 504, 5),
                                     (513, 512, 4096, 64), (260, 64, 800, 200)])
def test_lora_head(cuda, dtype, m, k, v, r):
    x, w, y, a, b = _case(m, k, v, dtype, r, seed=r)
    y[m // 2:m // 2 + m // 4] = IGNORE
    _check(x.requires_grad_(True), w, y, a.requires_grad_(True), b.requires_grad_(True),
           alpha=2.0 * r)
    x, a, b = x.detach(), a.detach().float().requires_grad_(True), b.detach().float().requires_grad_(True)
    loss = ops.linear_cross_entropy(x, w, y, A=a, B=b, alpha=2.0 * r)  # master factors in fp32
    da, db = torch.autograd.grad(loss, (a, b))
    assert da.dtype == db.dtype == torch.float32 and da.shape == a.shape and db.shape == b.shape
    _check(x, w, y, a, b, alpha=2.0 * r)


@pytest.mark.gpu
def test_lora_and_trained_weight_together(cuda):
    x, w, y, a, b = _case(200, 128, 640, BF16, 8, seed=3)
    _check(x.requires_grad_(True), w.requires_grad_(True), y, a.requires_grad_(True),
           b.requires_grad_(True))


@pytest.mark.gpu
def test_rows_in_pieces(cuda):
    """A vocabulary so large that 256 rows fill the workspace: three pieces, the
    last of them with uncounted rows alone, dW summed over them."""
    x, w, y, _, _ = _case(700, 16, 1_000_003, BF16, seed=5, lean=2.0)
    y[20:220] = IGNORE
    x.requires_grad_(True)
    _check(x, w, y)
    _check(x, w[:600_000].clone().requires_grad_(True), y % 600_000)


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_nothing_counts(cuda, reduction):
    x, w, y, _, _ = _case(70, 64, 100, BF16)
    y[:] = IGNORE
    x.requires_grad_(True)
    w.requires_grad_(reduction != "none")
    loss = ops.linear_cross_entropy(x, w, y, reduction=reduction)
    if reduction == "mean":
        assert torch.isnan(loss)
    else:
        assert torch.count_nonzero(loss) == 0
    for g in torch.autograd.grad(loss.sum(), [x] + ([w] if w.requires_grad else [])):
        assert torch.count_nonzero(g) == 0  # and none is NaN
    e = ops.linear_cross_entropy(x[:0], w, y[:0], reduction=reduction)
    assert e.shape == ((0,) if reduction == "none" else ())
    assert torch.isnan(e) if reduction == "mean" else torch.count_nonzero(e) == 0
    g = torch.autograd.grad(e.sum(), x)[0]
    assert g.shape == x.shape and torch.count_nonzero(g) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_per_token_losses_and_gradients(cuda, dtype):
    x, w, y, _, _ = _case(333, 128, 1003, dtype, seed=8)
    y[5:50] = IGNORE
    up = torch.randn(333, dtype=torch.float64, device=cuda)
    _check(x.requires_grad_(True), w, y, upstream=up.float().double(), reduction="none")
    x3, y3 = x.detach().reshape(3, 111, 128), y.reshape(3, 111).int()
    rows = ops.linear_cross_entropy(x3, w, y3, reduction="none")
    assert rows.shape == (3, 111)
    assert torch.equal(rows.reshape(-1), ops.linear_cross_entropy(x, w, y, reduction="none"))


@pytest.mark.gpu
def test_labels_outside_the_vocabulary(cuda):
    x, w, y, _, _ = _case(64, 64, 500, BF16, seed=9)
    x.requires_grad_(True)
    good = y.clone()
    y[3], y[40] = 500, -1
    good[[3, 40]] = IGNORE
    _lib.device_status(reset=True)
    loss = ops.linear_cross_entropy(x, w, y)
    g = torch.autograd.grad(loss, x)[0]
    torch.cuda.synchronize()
    assert _lib.device_status(reset=False) == 0x107
    again = ops.linear_cross_entropy(x, w, good)  # runs as ever while the code stands
    assert torch.equal(loss, again) and torch.equal(g, torch.autograd.grad(again, x)[0])
    assert _lib.device_status(reset=True) == 0x107


@pytest.mark.gpu
def test_large_logits_infinities_and_nan(cuda):
    x, w, y, _, _ = _case(300, 64, 700, BF16, seed=10, size=40.0, lean=0.0)
    _check(x.requires_grad_(True), w, y)  # logits in the hundreds
    x = x.detach().clone()
    x[2, 0], x[7, 3], x[9] = float("inf"), float("nan"), 0.0
    y[2], y[7] = 1, 2
    rows = ops.linear_cross_entropy(x, w, y, reduction="none")
    assert torch.isnan(rows[[2, 7]]).all() and torch.isfinite(rows[torch.arange(300) >= 10]).all()
    assert abs(float(rows[9]) - math.log(700)) < 1e-5
    y[[2, 7]] = IGNORE  # in a row that does not count they are not seen
    x.requires_grad_(True)
    g = torch.autograd.grad(ops.linear_cross_entropy(x, w, y), x)[0]
    assert torch.isfinite(g).all() and torch.count_nonzero(g[[2, 7]]) == 0


@pytest.mark.gpu
def test_gradient_against_differences(cuda):
    """Of the operator's own losses: moving x along d changes the loss by <dx, d>."""
    x, w, y, _, _ = _case(64, 512, 3001, BF16, seed=11)
    y[:9] = IGNORE
    x.requires_grad_(True)
    dx = torch.autograd.grad(ops.linear_cross_entropy(x, w, y, reduction="sum"), x)[0].double()
    d = torch.zeros_like(x)
    d.copy_(dx.sign() * 2.0 ** -4)
    hi, lo = (x + d).detach(), (x - d).detach()
    moved = (hi.double() - lo.double())  # as bf16 took it
    got = (ops.linear_cross_entropy(hi, w, y, reduction="sum").double()
           - ops.linear_cross_entropy(lo, w, y, reduction="sum").double())
    want = (dx * moved).sum()
    # central difference: third-order term of logits that move by at most 2^-4 |W| sums
    assert abs(float(got / want) - 1) < 0.05


@pytest.mark.gpu
def test_strides_streams_graphs_and_repeats(cuda):
    x, w, y, _, _ = _case(400, 256, 3000, BF16, seed=12)
    xt = x.t().contiguous().t()
    wt = torch.cat([w, w], 1)[:, :256]
    yt = torch.stack([y, y], 1)[:, 0]
    x.requires_grad_(True)
    xt.requires_grad_(True)
    a, b = ops.linear_cross_entropy(x, w, y), ops.linear_cross_entropy(xt, wt, yt)
    ga, gb = torch.autograd.grad(a, x)[0], torch.autograd.grad(b, xt)[0]
    assert torch.equal(a, b) and torch.equal(ga, gb)
    loss = ops.linear_cross_entropy(x, w, y)  # the state outlives a first backward
    one = torch.autograd.grad(loss, x, retain_graph=True)[0]
    assert torch.equal(one, torch.autograd.grad(loss, x)[0]) and torch.equal(one, ga)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = ops.linear_cross_entropy(x, w, y)
        gc = torch.autograd.grad(c, x)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(c, a) and torch.equal(gc, ga)
    del a, b, c, loss
    # captured once, replayed with other inputs and another number of counted tokens
    xs, ys = x.detach().clone().requires_grad_(True), y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lg = ops.linear_cross_entropy(xs, w, ys)
        gg = torch.autograd.grad(lg, xs)[0]
    with torch.no_grad():
        xs.copy_(x.flip(0))
    ys.copy_(y.flip(0))
    ys[:123] = IGNORE
    graph.replay()
    want = ops.linear_cross_entropy(xs, w, ys)
    assert torch.equal(lg, want) and torch.equal(gg, torch.autograd.grad(want, xs)[0])


@pytest.mark.gpu
def test_threads_at_once(cuda):
    """Two host threads with their own streams."""
    import threading
    x, w, y, _, _ = _case(300, 256, 5000, BF16, seed=13)
    want = ops.linear_cross_entropy(x.requires_grad_(True), w, y)
    gw = torch.autograd.grad(want, x)[0]
    torch.cuda.synchronize()
    out = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                xi = x.detach().clone().requires_grad_(True)
                loss = ops.linear_cross_entropy(xi, w, y)
                g = torch.autograd.grad(loss, xi)[0]
                out.append(torch.equal(g, gw) and torch.equal(loss, want))

    threads = [threading.Thread(target=work) for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert out == [True] * 20


@pytest.mark.gpu
def test_differentiable_once(cuda):
    """A gradient that is to be differentiated again comes out right and refuses that."""
    x, w, y, a, b = _case(40, 64, 304, BF16, 8, seed=14)
    x.requires_grad_(True)
    a.requires_grad_(True)
    b.requires_grad_(True)
    for kw in ({}, {"A": a, "B": b}):
        leaves = (x, a, b) if kw else (x,)
        want = torch.autograd.grad(ops.linear_cross_entropy(x, w, y, **kw), leaves)
        got = torch.autograd.grad(ops.linear_cross_entropy(x, w, y, **kw), leaves, create_graph=True)
        assert all(torch.equal(g, h) for g, h in zip(got, want))
        with pytest.raises(RuntimeError):
            torch.autograd.grad(got[0].float().sum(), x)
    tab = torch.randn(20, 16, device=cuda, requires_grad=True)
    for out, leaf in ((ops.dropout(x, 0.5, 3), x), (ops.embedding(y[:9] % 20, tab), tab)):
        got = torch.autograd.grad(out.float().square().sum(), leaf, create_graph=True)[0]
        with pytest.raises(RuntimeError):
            torch.autograd.grad(got.float().sum(), leaf)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_losses_without_a_gradient(cuda, dtype):
    """Nothing asked for: the same losses, from less memory."""
    x, w, y, a, b = _case(600, 128, 5000, dtype, 16, seed=15)
    y[::7] = IGNORE
    for kw in ({}, {"A": a, "B": b, "alpha": 32.0}):
        want = ops.linear_cross_entropy(x.requires_grad_(True), w, y, reduction="none", **kw)
        with torch.no_grad():
            assert torch.equal(ops.linear_cross_entropy(x, w, y, reduction="none", **kw), want)
        _check(x.detach(), w, y, kw.get("A"), kw.get("B"), kw.get("alpha", 16.0))


@pytest.mark.gpu
def test_lora_head_with_frozen_factors(cuda):
    x, w, y, a, b = _case(300, 128, 1000, BF16, 16, seed=16)
    y[4:90] = IGNORE
    _check(x.requires_grad_(True), w, y, a, b, alpha=32.0)
    _check(x, w, y, a, b, alpha=32.0, reduction="sum")


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    """More than 2^31 hidden values: rows at both ends against 64 bits."""
    m, k, v = 530_000, 4096, 72
    g = torch.Generator(device=cuda).manual_seed(17)
    w = (torch.randn(v, k, generator=g, device=cuda) / 64).to(BF16)
    x = torch.randn(m, k, generator=g, device=cuda, dtype=BF16).requires_grad_(True)
    y = torch.randint(0, v, (m,), generator=g, device=cuda)
    y[::3] = IGNORE
    loss = ops.linear_cross_entropy(x, w, y, reduction="none")
    dx = torch.autograd.grad(loss, x, torch.ones_like(loss))[0]
    pick = torch.cat([torch.arange(100), torch.arange(m - 100, m)]).to(cuda)
    xs, ys = x.detach()[pick].requires_grad_(True), y[pick]
    want = ops.linear_cross_entropy(xs, w, ys, reduction="none")  # checked against 64 bits elsewhere
    assert (loss[pick] - want).abs().max() < 1e-5
    few = torch.autograd.grad(want, xs, torch.ones_like(want))[0].double()
    assert ((dx[pick].double() - few).abs() <= 2.0 ** -7 * few.abs() + 1e-5).all()
    assert torch.count_nonzero(dx[::3][-50:]) == 0

