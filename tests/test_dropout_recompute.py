"""Counter-based LoRA dropout where torch.utils.checkpoint runs the forward again: the
masks are the first run's."""
import copy
import pickle

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from metallora_b200 import layers as layers_module
from metallora_b200.exceptions import ConfigurationError
from metallora_b200.layers import LoRALinear

BF16 = torch.bfloat16


def _restated(x, w0, a, b, alpha=16.0, dropout=0.0, training=False, dropout_seed=None, dropout_call=0,
              **_):
    """The layer's arithmetic with a mask that is a function of the seed and the call."""
    gen = torch.Generator().manual_seed(1000 * dropout_seed + dropout_call)
    kept = torch.rand(x.shape[:-1] + (w0.shape[0],), generator=gen, dtype=x.dtype) >= dropout
    return x @ w0.T + kept * (x @ a.T @ b.T) * (alpha / a.shape[0] / (1 - dropout))


def _pair(device="cpu", dtype=torch.float64):
    torch.manual_seed(0)
    made = [LoRALinear(64, 64, rank=8, dropout=0.5, device=device, dtype=dtype, dropout_seed=3 + i)
            for i in range(2)]
    with torch.no_grad():
        for m in made:
            m.W0.normal_(0, 0.1)
            m.B.normal_(0, 0.3)
    return made


def _gradients(pair, how, rounds=2):
    """The gradients of `rounds` forwards (all of them before the first backward) of two
    layers, the first one used twice, with nonlinearities between."""
    p, q = pair
    for m in pair:
        m.dropout_call = 0

    def block(h):
        return torch.tanh(p(torch.tanh(q(torch.tanh(p(h))))))

    torch.manual_seed(1)
    x = torch.randn(24, 64, dtype=torch.float64).to(p.W0.device, p.W0.dtype).requires_grad_(True)
    outs = [block(x * (i + 1)) if how is None else
            checkpoint(block, x * (i + 1), use_reentrant=how) for i in range(rounds)]
    made = []
    for out in outs:  # the first one's backward after the second one's forward
        leaves = (x, p.A, p.B, q.A, q.B)
        for t in leaves:
            t.grad = None
        (out * out).sum().backward()
        made += [t.grad for t in leaves]
    assert (p.dropout_call, q.dropout_call) == (2 * rounds, rounds)
    return [t.detach() for t in (*outs, *made)]


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_forwards_use_the_first_ones_masks(monkeypatch, reentrant):
    monkeypatch.setattr(layers_module, "lora_forward", _restated)
    pair = _pair()
    plain = _gradients(pair, None)
    again = _gradients(pair, reentrant)
    assert len(plain) == len(again) == 12
    for u, v in zip(again, plain):
        assert torch.equal(u, v)
    assert not torch.equal(plain[0], plain[1])


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputation_without_the_generators_state_is_refused(monkeypatch, reentrant):
    monkeypatch.setattr(layers_module, "lora_forward", _restated)
    p, _ = _pair()
    x = torch.randn(4, 64, dtype=torch.float64, requires_grad=True)
    out = checkpoint(lambda h: torch.tanh(p(h)), x, use_reentrant=reentrant, preserve_rng_state=False)
    with pytest.raises(ConfigurationError, match="CPU generator"):
        out.sum().backward()
    # seeded alike before two forwards: which of them is run again is not known
    for _ in range(2):
        torch.manual_seed(5)
        out = checkpoint(lambda h: torch.tanh(p(h)), x, use_reentrant=reentrant)
    with pytest.raises(ConfigurationError, match="CPU generator"):
        out.sum().backward()


def test_what_a_layer_keeps_is_bounded_and_copied(monkeypatch):
    monkeypatch.setattr(layers_module, "lora_forward", _restated)
    monkeypatch.setattr(layers_module, "_KEPT_CALLS", 4)
    p, _ = _pair()
    x = torch.randn(4, 64, dtype=torch.float64, requires_grad=True)
    outs = [checkpoint(lambda h: torch.tanh(p(h)), x, use_reentrant=False) for _ in range(5)]
    assert len(p._calls_by_draw) == 4
    outs[1].sum().backward()
    with pytest.raises(ConfigurationError):
        outs[0].sum().backward()
    p.eval()
    with torch.no_grad():
        monkeypatch.setattr(layers_module, "lora_forward", lambda x, *a, **k: x)
        p(x)
    assert p.dropout_call == 5 and len(p._calls_by_draw) == 4
    for twin in (copy.deepcopy(p), pickle.loads(pickle.dumps(p))):
        assert twin.dropout_call == 5
        twin.train()
        assert twin._mask_call() == 5 and p.dropout_call == 5


# ------------------------------------------------------------------ GPU --

@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_forwards_on_the_gpu(cuda, reentrant):
    pair = _pair(cuda, BF16)
    for u, v in zip(_gradients(pair, reentrant), _gradients(pair, None)):
        assert torch.equal(u, v)
