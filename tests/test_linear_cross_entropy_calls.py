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
