"""Counter-based LoRA dropout where torch.utils.checkpoint runs the forward again, and
where a run is saved and resumed: the masks are those of the unbroken run."""
import copy
import json
import pickle

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from metallora_b200 import layers as layers_module
from metallora_b200.exceptions import ConfigurationError
from metallora_b200.layers import LoRALinear
from metallora_b200.trainer import LoRATrainer, TrainingConfig
from tests.test_training_ends import Model

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
    # one with the draw and the number of another takes its place among the youngest
    p.dropout_call, outs = 0, []
    for seed in (1, 2, 3, 4, 1, 5):
        torch.manual_seed(seed)
        p.dropout_call = seed - 1
        outs.append(checkpoint(lambda h: torch.tanh(p(h)), x, use_reentrant=False))
    outs[4].sum().backward()
    with pytest.raises(ConfigurationError):
        outs[1].sum().backward()
    p.eval()
    with torch.no_grad():
        monkeypatch.setattr(layers_module, "lora_forward", lambda x, *a, **k: x)
        p(x)
    assert p.dropout_call == 5 and len(p._calls_by_draw) == 4
    for twin in (copy.deepcopy(p), pickle.loads(pickle.dumps(p))):
        assert twin.dropout_call == 5
        twin.train()
        assert twin._mask_call() == 5 and p.dropout_call == 5


def _trainer(path, seed=5, device="cpu", **kw):
    torch.manual_seed(0)
    return LoRATrainer(Model(device=device, **kw),
                       TrainingConfig(rank=8, dropout=0.3, dropout_seed=seed, loss_head="lm_head",
                                      learning_rate=1e-2, output_dir=str(path)))


def test_numbers_of_masks_are_saved(tmp_path):
    trainer = _trainer(tmp_path)
    for i, (_, m) in enumerate(trainer.params.layers):
        m.dropout_call = 7 + i
    trainer.save(tmp_path / "c")
    other = _trainer(tmp_path)
    other.load(tmp_path / "c")
    assert [m.dropout_call for _, m in other.params.layers] == [7, 8]
    # what was saved without them loads as it did
    config = json.loads((tmp_path / "c" / "config.json").read_text())
    assert config.pop("dropout_calls") == {"q_proj": 7, "v_proj": 8}
    (tmp_path / "c" / "config.json").write_text(json.dumps(config))
    again = _trainer(tmp_path)
    again.load(tmp_path / "c")
    (tmp_path / "c" / "config.json").unlink()
    again.load(tmp_path / "c")
    assert [m.dropout_call for _, m in again.params.layers] == [0, 0]
    # layers without counted masks leave the file as it was
    plain = _trainer(tmp_path, seed=None)
    plain.save(tmp_path / "p")
    assert set(json.loads((tmp_path / "p" / "config.json").read_text())) == \
        {"rank", "alpha", "global_step"}


# ------------------------------------------------------------------ GPU --

@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_forwards_on_the_gpu(cuda, reentrant):
    pair = _pair(cuda, BF16)
    for u, v in zip(_gradients(pair, reentrant), _gradients(pair, None)):
        assert torch.equal(u, v)


@pytest.mark.gpu
def test_a_resumed_run_is_the_unbroken_one(cuda, tmp_path):
    def batch(i):
        gen = torch.Generator(device=cuda).manual_seed(i)
        ids = torch.randint(0, 1003, (2, 40), device=cuda, generator=gen)
        return {"input_ids": ids, "labels": ids}

    runs = []
    for broken in (False, True):
        trainer = _trainer(tmp_path, device=cuda)
        for i in range(4):
            if broken and i == 2:
                trainer.save(tmp_path / "c")
                trainer = _trainer(tmp_path, device=cuda)
                trainer.load(tmp_path / "c")
            trainer._training_step(batch(i))
        runs.append(trainer.params.master.clone())
    assert torch.equal(*runs)
