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
