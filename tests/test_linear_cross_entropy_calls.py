"""What a linear cross entropy asks of its kernels, how it cuts its tokens into pieces,
and how exact it is where tokens are few: the forms that the sizes of
test_linear_cross_entropy.py do not reach."""
import pytest
import torch

from metallora_b200 import _lib, ops

BF16, FP16 = torch.bfloat16, torch.float16
IGNORE = -100


# ------------------------------------------------------------------ CPU --

def test_gradients_are_made_where_they_are_wanted(monkeypatch):
    """Every set of leaves, with gradients and under no_grad, where a LoRA head's factors
    are parameters still: there none are made."""
    asked = []

    def fwd(x2d, w, labels, a=None, b=None, alpha=16.0, ignore_index=-100, reduction="mean", grads=0):
        asked.append(grads)
        return torch.zeros(()), torch.zeros(1)
    monkeypatch.setattr(ops._k, "linear_cross_entropy_fwd", fwd)
    monkeypatch.setattr(_lib, "autograd", lambda: type("Fake", (), {
        "attach_linear_cross_entropy": staticmethod(lambda *a: None)}))
    x, w = torch.zeros(4, 16, dtype=BF16), torch.zeros(32, 16, dtype=BF16)
    a, b = torch.zeros(8, 16, dtype=BF16), torch.zeros(32, 8, dtype=BF16)
    y = torch.zeros(4, dtype=torch.int64)
    for dx in (False, True):
        for dw in (False, True):
            for dab in (False, True):
                x, w, a, b = (t.detach().requires_grad_(on)
                              for t, on in ((x, dx), (w, dw), (a, dab), (b, dab)))
                plain = _lib.HEAD_GRAD_X * dx + _lib.HEAD_GRAD_W * dw
                ops.linear_cross_entropy(x, w, y)
                ops.linear_cross_entropy(x, w, y, A=a, B=b)
                with torch.no_grad():
                    ops.linear_cross_entropy(x, w, y)
                    ops.linear_cross_entropy(x, w, y, A=a, B=b)
                assert asked[-4:] == [plain, plain + _lib.HEAD_GRAD_AB * dab, 0, 0]


# ------------------------------------------------------------------ GPU --

@pytest.mark.gpu
def test_a_lora_head_under_no_grad_takes_less_memory(cuda):
    """The exponentials, [tokens, entries] in 16 bits, are for gradients alone."""
    gen = torch.Generator(device=cuda).manual_seed(0)
    x, w, a, b = (torch.randn(*s, device=cuda, generator=gen).to(BF16).requires_grad_(i != 1)
                  for i, s in enumerate(((2048, 64), (16384, 64), (8, 64), (16384, 8))))
    y = torch.randint(0, 16384, (2048,), device=cuda, generator=gen)

    def peak():
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        loss = ops.linear_cross_entropy(x, w, y, A=a, B=b)
        return torch.cuda.max_memory_allocated() - before, loss.detach()
    most, want = peak()
    with torch.no_grad():
        least, got = peak()
    assert torch.equal(got, want) and most > 2048 * 16384 * 2 > 8 * least


def _few(cuda, dtype, m, seed, v=2000, k=64, r=8):
    """A few tokens, one of them not counted, two of one label, and what 64 bits make of them."""
    gen = torch.Generator(device=cuda).manual_seed(seed)

    def randn(*s, scale):
        return (torch.randn(*s, device=cuda, generator=gen) * scale).to(dtype)
    x, w = randn(m, k, scale=1.0), randn(v, k, scale=0.2)
    a, b = randn(r, k, scale=0.1), randn(v, r, scale=0.3)
    y = torch.randint(0, v, (m,), device=cuda, generator=gen)
    if m > 2:
        y[2], y[1] = y[0], IGNORE
    return x, w, a, b, y


def _gradient(x, w, a, b, y, s):
    """Logits' gradient of the summed loss, its part at the labels, and s x A^T, in 64 bits."""
    xa = s * x.double() @ a.double().T
    rows = (y != IGNORE).nonzero()[:, 0]
    g = torch.softmax(x.double() @ w.double().T + xa @ b.double().T, 1)
    at = torch.zeros_like(g)
    g[rows, y[rows]] -= 1
    at[rows, y[rows]] = g[rows, y[rows]]
    g[y == IGNORE] = 0
    return g, at, xa


# relative error of softmax's values: ex2.approx, logits of up to 15 cut by 2^-19 at each of
# the sum's few steps, exp and log of them
SOFT = 2.0 ** -14


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m", [1, 2, 5])
def test_gradients_of_weights_from_few_tokens(cuda, dtype, m):
    """The label's entry of the logits' gradient, nearly all of a row of dW and dB where its
    label has one token, is not seen rounded: those rows are off by their own rounding."""
    half = torch.finfo(dtype).eps / 2
    # entries but the label's are rounded twice: the exponentials are fp16 values (off by
    # 2^-11 at most), and g, that times the row's factor, is one of the type's
    twice = half + 2.0 ** -11 + SOFT
    tiny = torch.finfo(dtype).smallest_normal * half if dtype == FP16 else 0.0
    for seed in range(8):
        x, w, a, b, y = _few(cuda, dtype, m, seed)
        no = torch.zeros_like(a), torch.zeros_like(b)
        g, at, _ = _gradient(x, w, *no, y, 0.0)
        w1 = w.clone().requires_grad_(True)
        dw = torch.autograd.grad(ops.linear_cross_entropy(x, w1, y, reduction="sum"), w1)[0].double()
        want = g.T @ x.double()
        # (fp16: 64 g is kept, its subnormals are off by 2^-31 of g)
        rest = (g - at).abs().T @ x.double().abs()
        bound = (half + SOFT) * want.abs() + twice * rest * (1 + half) + 2 * tiny + SOFT * (
            at.abs().T @ x.double().abs())
        assert bool(((dw - want).abs() <= bound).all()), (seed, m)
        # a LoRA head: the others' roundings are many and of random sign, six deviations
        s = 2.0
        g, at, xa = _gradient(x, w, a, b, y, s)
        leaves = [t.clone().requires_grad_(True) for t in (a, b)]
        loss = ops.linear_cross_entropy(x, w, y, A=leaves[0], B=leaves[1], alpha=s * 8, reduction="sum")
        da, db = (t.double() for t in torch.autograd.grad(loss, leaves))
        want = g.T @ xa
        rest = (g - at).abs().T @ xa.abs()
        part = 2.0 ** -14  # s x A^T in two parts of 8 bits or more
        bound = (half + SOFT + part) * want.abs() + twice * rest * (1 + half) + 2 * tiny + \
            (SOFT + part) * (at.abs().T @ xa.abs())
        assert bool(((db - want).abs() <= bound).all()), (seed, m)
        u = s * g @ b.double()
        want = u.T @ x.double()
        off = 6 * twice / 3 ** 0.5 * s * ((g - at).square() @ b.double().square()).sqrt()
        size = s * g.abs() @ b.double().abs()
        bound = half * want.abs() + (1 + half) * ((off + (SOFT + part) * size).T @ x.double().abs()) + tiny
        assert bool(((da - want).abs() <= bound).all()), (seed, m)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,k", [(40, 64), (60, 2056), (4096, 136), (4097, 520), (9000, 2184)])
def test_gradients_of_weights_from_tokens_that_recur(cuda, dtype, m, k):
    """Three tokens over and over, so that their roundings add up, around the 16 that a
    label's tokens are many from, the ranges of 4096 tokens and 2048 columns: the rows of
    their labels are off by their own rounding still, and by m additions, each of which
    cuts at most 2^-23 of what is summed by then, on average half of the sum."""
    half = torch.finfo(dtype).eps / 2
    soft = SOFT + m * 2.0 ** -24
    twice = half + 2.0 ** -11 + soft
    x, w, _, _, y = _few(cuda, dtype, 3, 7, v=300, k=k)
    x, w = x / 4, w * (8 / k ** 0.5)
    y = torch.stack([y[0], (y[0] + 1) % 300, (y[0] + 2) % 300])
    gen = torch.Generator(device=cuda).manual_seed(m)
    which = torch.randint(0, 3, (m,), device=cuda, generator=gen)
    x, y = x[which], y[which]
    y[::50] = IGNORE
    w1 = w.clone().requires_grad_(True)
    dw = [torch.autograd.grad(ops.linear_cross_entropy(x, w1, y, reduction="sum"), w1)[0]
          for _ in range(2)]
    assert torch.equal(*dw)
    no = torch.zeros(8, k, device=cuda, dtype=dtype), torch.zeros(300, 8, device=cuda, dtype=dtype)
    g, at, _ = _gradient(x, w, *no, y, 0.0)
    want = g.T @ x.double()
    tiny = m * 2.0 ** -31 * float(x.abs().max()) + 2.0 ** -25 if dtype == FP16 else 0.0
    bound = half * want.abs() + (1 + half) * (
        twice * (g - at).abs().T @ x.double().abs() + soft * (at.abs().T @ x.double().abs())) + tiny
    assert bool(((dw[0].double() - want).abs() <= bound).all())


def _workspace(m, k, v, r, dtype, grads):
    code = _lib.DTYPE_BF16 if dtype == BF16 else _lib.DTYPE_F16
    return _lib.load().mlora_linear_cross_entropy_workspace_bytes(m, k, v, r, code, grads)


def _check_in_blocks(x, w, y, a=None, b=None, s=2.0, rows=256):
    """Summed loss and gradients against 64 bits, 256 tokens at a time; the bounds are
    those of each rounding, elementwise."""
    dtype, (m, k), v = x.dtype, x.shape, w.shape[0]
    h = torch.finfo(dtype).eps / 2
    tiny, sub = (2.0 ** -31, 2.0 ** -25) if dtype == FP16 else (0.0, 0.0)
    eps = 2.0 ** -20
    leaves = [t for t in (x, w, a, b) if t is not None and t.requires_grad]
    r = 0 if a is None else a.shape[0]
    loss = ops.linear_cross_entropy(x, w, y, A=a, B=b, alpha=s * max(r, 1), reduction="sum")
    got = dict(zip([id(t) for t in leaves], torch.autograd.grad(loss, leaves)))
    xs, wd = x.detach().double(), w.detach().double()
    dw, bw = torch.zeros_like(wd), torch.zeros_like(wd)
    if r:
        ad, bd = a.detach().double(), b.detach().double()
        da, ba, db, bb = (torch.zeros_like(t) for t in (ad, ad, bd, bd))
    total = most = 0.0
    # logits: a random walk of K fp32 roundings, four deviations
    dl = 2.0 ** -24 * 4 * k ** 0.5 * float(xs.norm(dim=1).max() * wd.norm(dim=1).max()) + 2e-6
    if r:  # s x A^T in two parts of 16 bits
        xa_all = s * xs @ ad.T
        dl += 2.0 ** -14 * float((xa_all.abs().max(1).values).max() * bd.abs().sum(1).max())
    rel = h + 2.0 ** -11 + 2 * dl
    for part in torch.arange(m, device=x.device).split(rows):
        xd, yd = xs[part], y[part]
        counted = yd != IGNORE
        at = yd.clamp_min(0)[:, None]
        logits = xd @ wd.T
        if r:
            logits += xa_all[part] @ bd.T
        nll = (torch.logsumexp(logits, 1) - logits.gather(1, at)[:, 0]) * counted
        total, most = total + float(nll.sum()), max(most, float(nll.max()))
        g = torch.softmax(logits, 1, out=logits)
        off = (g * rel + tiny) * counted[:, None]
        g.scatter_add_(1, at, torch.full_like(at, -1, dtype=g.dtype)).mul_(counted[:, None])
        eg = off + h * g.abs()
        dx, bx = g @ wd, off @ wd.abs() + eps * (g.abs() @ wd.abs())
        if r:
            u = s * g @ bd
            eu = s * (eg @ bd.abs()) + h * u.abs() + eps * s * (g.abs() @ bd.abs())
            dx, bx = dx + u @ ad, bx + eu @ ad.abs() + eps * (u.abs() @ ad.abs())
            xa = xa_all[part]
            da += u.T @ xd
            ba += (eu + eps * u.abs()).T @ xd.abs()
            db += g.T @ xa
            bb += (eg + (h + eps) * g.abs()).T @ xa.abs()
        if x.requires_grad:
            e = (got[id(x)][part].double() - dx).abs() - (bx + h * dx.abs() * 1.01 + sub)
            assert e.max() <= 0, f"dx of tokens {int(part[0])}.. beyond its bound by {e.max()}"
            assert torch.count_nonzero(got[id(x)][part][~counted]) == 0
        if w.requires_grad:
            dw += g.T @ xd
            bw += (eg + eps * g.abs()).T @ xd.abs()
    assert abs(float(loss.detach()) - total) <= (2 * dl + 2.0 ** -22 * most) * m
    for t, want, bound in ((w, dw, bw),) + (((a, da, ba), (b, db, bb)) if r else ()):
        if t.requires_grad:
            e = (got[id(t)].double() - want).abs() - (bound + h * want.abs() * 1.01 + sub)
            assert e.max() <= 0, f"beyond its bound by {e.max()}"
    assert _lib.device_status(reset=True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("counted", [2050, 1200, 700])
@pytest.mark.parametrize("head,dtype", [("frozen", BF16), ("frozen", FP16), ("trained", BF16),
                                        ("lora", BF16), ("lora", FP16)])
def test_more_tokens_than_a_piece(cuda, head, dtype, counted):
    """Vocabularies of which 768 tokens are a piece: three of them, the last or the last two
    without counted tokens, the last counted one inside a piece."""
    m, k = 2100, 16
    v = (1 << 20) - (8 if head == "lora" else 5)
    gen = torch.Generator(device=cuda).manual_seed(counted)

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, device=cuda, generator=gen) * scale).to(dtype)
    x, w = randn(m, k).requires_grad_(True), randn(v, k, scale=0.4).requires_grad_(head == "trained")
    y = torch.randint(0, v, (m,), device=cuda, generator=gen)
    y[1::3] = y[::3][: y[1::3].numel()]  # labels that recur, within a piece and across
    y[1500:1600] = y[:100]
    y[torch.randperm(m, device=cuda, generator=gen)[: m - counted]] = IGNORE
    a = b = None
    if head == "lora":
        a = randn(8, k, scale=0.3).requires_grad_(True)
        b = randn(v, 8, scale=0.1).requires_grad_(True)
    grads = 1 + 2 * (head == "trained") + 4 * (head == "lora")
    # all exponentials at once would take more than the whole workspace, twice over
    assert 2 * _workspace(m, k, v, 8 if a is not None else 0, dtype, grads) < 2 * m * v * 2
    _check_in_blocks(x, w, y, a, b)


@pytest.mark.gpu
def test_losses_of_more_tokens_than_a_piece(cuda):
    """Without a gradient a token costs a piece 8 bytes for each 96 entries or more; the
    losses are those of calls with fewer tokens, but for the order of sums over tiles."""
    m, k, v = 50_000, 16, (1 << 20) - 5
    gen = torch.Generator(device=cuda).manual_seed(0)
    x = torch.randn(m, k, device=cuda, generator=gen).to(BF16)
    w = (torch.randn(v, k, device=cuda, generator=gen) * 0.4).to(BF16)
    y = torch.randint(0, v, (m,), device=cuda, generator=gen)
    y[::5] = IGNORE
    assert _workspace(m, k, v, 0, BF16, 0) < m * v // 128 * 8
    got = ops.linear_cross_entropy(x, w, y, reduction="none")
    for lo in range(0, m, 6250):
        part = slice(lo, lo + 6250)
        want = ops.linear_cross_entropy(x[part], w, y[part], reduction="none")
        # sums of 8192 tiles in another order and by another reference
        assert bool(((got[part] - want).abs() <= 2.0 ** -18 * want.abs()).all())
        assert torch.equal(got[part] == 0, y[part] == IGNORE)


def _loss_error(x, w, y):
    """|error| of the mean loss; the mean softmax-weighted |logit| of the other entries, what
    a relative error of the logits is seen times; the fp32 steps' share: ex2.approx and
    l log2(e) - n, rounded at 2^-24 of |l| log2(e) + 1 twice, and the result."""
    got = ops.linear_cross_entropy(x, w, y).double()
    logits = x.double() @ w.double().T
    want = torch.nn.functional.cross_entropy(logits, y)
    sens = torch.softmax(logits, 1).scatter_(1, y[:, None], 0.0).mul_(logits.abs()).sum(1).mean()
    fp32 = 2.0 ** -22 * (float(logits.abs().max()) + 4) + 2.0 ** -23 * float(want)
    return abs(float(got - want)), float(sens), fp32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("k", [256, 1024, 4096, 8192])
def test_loss_of_dense_hidden_states(cuda, dtype, k):
    """What the tensor cores cut off the logits, 1e-9 K of them, is given back to within
    half: without that the loss would be off by all of it."""
    gen = torch.Generator(device=cuda).manual_seed(k)
    x, w = (torch.randn(*s, device=cuda, generator=gen) for s in ((512, k), (3000, k)))
    y = torch.randint(0, 3000, (512,), device=cuda, generator=gen)
    off, sens, fp32 = _loss_error(x.to(dtype), (w * 6 / k ** 0.5).to(dtype), y)
    assert off <= 0.5e-9 * k * sens + 2.0 ** -24 * 20
    assert k < 4096 or 0.5e-9 * k * sens > 2.0 ** -24 * 20  # the bound is the cut's


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("k", [256, 4096, 65536])
def test_loss_of_sparse_hidden_states(cuda, dtype, k):
    """One feature a token: the logits are single products, of which nothing is cut."""
    gen = torch.Generator(device=cuda).manual_seed(k)
    x = torch.zeros(200, k, device=cuda, dtype=dtype)
    at = torch.randint(0, k, (200,), device=cuda, generator=gen)
    x[torch.arange(200, device=cuda), at] = 1.5
    x[::2] *= -1  # the zeros beside them negative
    w = (torch.randn(1000, k, device=cuda, generator=gen) * 6).to(dtype)
    y = torch.randint(0, 1000, (200,), device=cuda, generator=gen)
    off, _, fp32 = _loss_error(x, w, y)
    assert off <= fp32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_loss_of_more_features_than_were_measured(cuda, dtype):
    """Exact sums of 2^17 features of one size: what is given back stops at 8192 features'."""
    k = 1 << 17
    gen = torch.Generator(device=cuda).manual_seed(0)
    x, w = (torch.randint(0, 2, s, device=cuda, generator=gen).mul_(2).sub_(1).to(dtype)
            for s in ((200, k), (1000, k)))
    y = torch.randint(0, 1000, (200,), device=cuda, generator=gen)
    off, sens, fp32 = _loss_error(x, w * 2.0 ** -5, y)
    assert off <= 1.0e-9 * 8192 * sens + fp32 < 1.0e-9 * k * sens / 4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("k", [1024, 4096])
def test_loss_of_products_of_one_sign(cuda, dtype, k):
    """Sums that only grow lose most.  Each of K additions cuts at most 2^-23 of what is
    summed by then, on average half of the sum: K 2^-24 of it.  (Measured 3.5e-9 K in
    bf16 and 6.3e-9 K in fp16, of which 1e-9 K are given back.)"""
    gen = torch.Generator(device=cuda).manual_seed(k)
    x = torch.rand(300, k, device=cuda, generator=gen).to(dtype)
    w = (torch.rand(1000, k, device=cuda, generator=gen) * torch.rand(1000, 1, device=cuda, generator=gen)
         * 100 / k).to(dtype)
    y = torch.randint(0, 1000, (300,), device=cuda, generator=gen)
    off, sens, fp32 = _loss_error(x, w, y)
    assert off <= k * 2.0 ** -24 * sens + fp32
