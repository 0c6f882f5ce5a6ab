"""The backward nodes that torch's engine runs without Python: dropout, token embedding,
the loss of a frozen head."""
import shutil
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

from metallora_b200 import _lib, ops
from metallora_b200.exceptions import MetalLoRAError

BF16 = torch.bfloat16


def test_extension_is_built():
    nodes = _lib.autograd()
    assert nodes is _lib.autograd()
    assert all(hasattr(nodes, "attach_" + n) for n in ("dropout", "embedding", "linear_cross_entropy"))


def test_forward_and_backward_are_of_one_library(tmp_path):
    """Loaded from another path, the kernels of both directions are that path's."""
    other = tmp_path / "other.so"
    shutil.copy(_lib.LIB_PATH, other)
    out = subprocess.run(
        [sys.executable, "-c", "import sys; from metallora_b200 import _lib; _lib.load(sys.argv[1]); "
         "_lib.autograd(); print(open('/proc/self/maps').read())", str(other)],
        capture_output=True, text=True, cwd=Path(__file__).resolve().parent.parent, timeout=300)
    assert out.returncode == 0, out.stderr
    assert str(other) in out.stdout and str(_lib.LIB_PATH) not in out.stdout


def _calls(cuda):
    """(name, leaf, call of the leaf, what the backward reads besides) of each operator."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(40, 64, device=cuda, generator=g).to(BF16)
    w = torch.randn(304, 64, device=cuda, generator=g).to(BF16)
    y = torch.randint(0, 304, (40,), device=cuda, generator=g)
    table = torch.randn(304, 64, device=cuda, generator=g)
    seed = torch.tensor([11], device=cuda)
    return [("dropout", x.float(), lambda t: ops.dropout(t, 0.4, seed, 2), seed),
            ("embedding", table, lambda t: ops.embedding(y, t, 2.0, 5), y),
            ("loss", x, lambda t: ops.linear_cross_entropy(t, w, y), w),
            ("losses", x, lambda t: ops.linear_cross_entropy(t, w, y, reduction="none"), w)]


NAMES = ("dropout", "embedding", "loss", "losses")


def _case(cuda, name):
    _, leaf, call, kept = next(c for c in _calls(cuda) if c[0] == name)
    return leaf.clone().requires_grad_(True), call, kept


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_kept_tensors_are_guarded_and_let_go(cuda, name):
    leaf, call, kept = _case(cuda, name)
    out = call(leaf)
    up = torch.randn_like(out)
    first = torch.autograd.grad(out, leaf, up, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(out, leaf, up)[0], first)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, leaf, up)
    out = call(leaf)
    kept.add_(0)  # written over before the backward
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(out, leaf, up)
    del out, first
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    for _ in range(3):
        out = call(leaf)
        torch.autograd.grad(out, leaf, up)
        del out
        del_only = call(leaf)
        del del_only
    assert torch.cuda.memory_allocated() == held


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_upstream_gradients_of_any_layout(cuda, name):
    """Expanded, transposed or absent; through a view, on a second stream, in a thread."""
    leaf, call, _ = _case(cuda, name)
    out = call(leaf)
    up = torch.randn_like(out)
    want = torch.autograd.grad(out, leaf, up)[0]
    if out.dim() == 2:
        turned = up.t().contiguous().t()
        assert not turned.is_contiguous()
        assert torch.equal(torch.autograd.grad(call(leaf), leaf, turned)[0], want)
    ones = torch.autograd.grad(call(leaf).sum(), leaf)[0]  # one expanded element
    assert torch.equal(torch.autograd.grad(call(leaf), leaf, torch.ones_like(up))[0], ones)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call(leaf)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(torch.autograd.grad(other, leaf, up)[0], want)
    torch.cuda.synchronize()
    got = []
    work = [threading.Thread(target=lambda: got.append(torch.autograd.grad(call(leaf), leaf, up)[0]))
            for _ in range(3)]
    [t.start() for t in work]
    [t.join() for t in work]
    torch.cuda.synchronize()
    assert len(got) == 3 and all(torch.equal(g, want) for g in got)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_grad_modes_and_checkpoints(cuda, name):
    leaf, call, _ = _case(cuda, name)
    out = call(leaf)
    up = torch.randn_like(out)
    want = torch.autograd.grad(out, leaf, up)[0]
    with torch.no_grad():
        quiet = call(leaf)
    assert not quiet.requires_grad and torch.equal(quiet, out)
    assert not call(leaf.detach()).requires_grad
    again = checkpoint(call, leaf, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(again, leaf, up)[0], want)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        call(forward_ad.make_dual(leaf.detach(), torch.ones_like(leaf)))


@pytest.mark.gpu
def test_differentiating_again(cuda):
    """The linear operators' gradients depend on the upstream gradient alone, the loss's
    on the hidden states too: with create_graph it refuses to be a constant."""
    for name in NAMES:
        leaf, call, _ = _case(cuda, name)
        out = call(leaf)
        up = torch.randn_like(out)
        grad = torch.autograd.grad(out, leaf, up, create_graph=True)[0]
        assert grad.requires_grad == name.startswith("loss")
        if grad.requires_grad:
            with pytest.raises(RuntimeError, match="twice"):
                grad.float().square().sum().backward()
        up.requires_grad_(True)
        grad = torch.autograd.grad(call(leaf), leaf, up, create_graph=True)[0]
        with pytest.raises(RuntimeError, match="twice"):
            grad.float().sum().backward()


@pytest.mark.gpu
def test_refusals_are_the_packages_own(cuda):
    """The C ABI's refusal of a backward (here of a threshold that the forward would not
    have let through) comes out of torch's engine as the package's exception."""
    x = torch.randn(8, 8, device=cuda, requires_grad=True)
    out = torch.empty_like(x, requires_grad=False)
    _lib.autograd().attach_dropout(out, x, 64, -1, True, 1, 0, _lib.DTYPE_F32, None)
    with pytest.raises(MetalLoRAError, match="mlora_dropout"):
        out.sum().backward()
    y = ops.dropout(x, 0.5, 1)  # and the next call is as it was
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0] != 0, y != 0)
