"""The operators together, as a training step uses them: token embedding, LoRA layers
with counter-based dropout, and the loss from a head's input; and the trainer's
settings for them."""
import math

import pytest
import torch
from torch import nn

from metallora_b200 import ops
from metallora_b200.exceptions import ConfigurationError
from metallora_b200.layers import LoRALinear, TokenEmbedding
from metallora_b200.trainer import LoRATrainer, TrainingConfig
from tests.test_dropout import factor

BF16, FP32 = torch.bfloat16, torch.float32


class Model(nn.Module):
    """Two residual projections between a token table and a head."""

    def __init__(self, vocab=1003, dim=128, hidden=264, dtype=BF16, device="cpu", head_bias=False,
                 tail=False):
        super().__init__()
        fk = {"device": device, "dtype": dtype}
        self.embed = TokenEmbedding(vocab, dim, scale=math.sqrt(dim), **fk)
        self.q_proj = nn.Linear(dim, hidden, bias=False, **fk)
        self.v_proj = nn.Linear(hidden, dim, bias=False, **fk)
        self.lm_head = nn.Linear(dim, vocab, bias=head_bias, **fk)
        self.tail = tail

    def forward(self, ids):
        h = self.embed(ids)
        h = h + self.v_proj(torch.tanh(self.q_proj(h)))
        out = self.lm_head(h)
        return out * 2 if self.tail else out


def test_settings_are_refused_before_the_model_changes(tmp_path):
    def refused(model, **kw):
        with pytest.raises(ConfigurationError):
            LoRATrainer(model, TrainingConfig(output_dir=str(tmp_path / "out"), **kw))
        assert not any(isinstance(m, LoRALinear) for m in model.modules())
        assert not (tmp_path / "out").exists()

    refused(Model(), loss_head="nothing")
    refused(Model(), loss_head="embed")
    refused(Model(head_bias=True), loss_head="lm_head")
    refused(Model(dtype=FP32), loss_head="lm_head")
    refused(Model(dim=132), loss_head="lm_head")
    refused(Model(), loss_head="lm_head", dropout=0.1, target_modules=["lm_head"])
    refused(Model(dtype=FP32), dropout=0.1, dropout_seed=1)
    refused(Model(hidden=260), dropout=0.1, dropout_seed=1)
    head = LoRALinear(128, 64, dtype=BF16)
    head.qweight = object()
    model = nn.Sequential(head)
    with pytest.raises(ConfigurationError):
        LoRATrainer(model, TrainingConfig(output_dir=str(tmp_path / "out"), loss_head="0"))
    assert head.dropout_seed is None


# ------------------------------------------------------------------ GPU --

@pytest.mark.gpu
def test_embedding_layer_dropout_and_loss(cuda):
    """Loss and every gradient of the chain against 64 bits at the same roundings'
    scale: each step's result is a bf16 value, 2^-8 off at most, and passes through
    at most three more products."""
    g = torch.Generator(device=cuda).manual_seed(0)

    def randn(*s, scale=1.0):
        return torch.randn(s, generator=g, device=cuda) * scale
    v, d, n, r, t, p = 2003, 256, 512, 16, 330, 0.2
    table = randn(v, d, scale=1 / 16).to(BF16).requires_grad_(True)
    w1 = randn(n, d, scale=1 / 16).to(BF16)
    a = randn(r, d, scale=1 / 16).to(BF16).requires_grad_(True)
    b = randn(n, r, scale=0.3).to(BF16).requires_grad_(True)
    w2 = randn(v, n, scale=1.5 / math.sqrt(n)).to(BF16)
    ids = torch.randint(0, v, (t,), generator=g, device=cuda)
    labels = torch.randint(0, v, (t,), generator=g, device=cuda)
    labels[:30] = -100

    h = ops.embedding(ids, table, scale=16.0)
    y = ops.lora_forward(h, w1, a, b, alpha=32.0, dropout=p, training=True, dropout_seed=9,
                         dropout_call=2)
    loss = ops.linear_cross_entropy(y, w2, labels)
    got = torch.autograd.grad(loss, (table, a, b))

    leaves = [x.detach().double().requires_grad_(True) for x in (table, a, b)]
    td, ad, bd = leaves
    kept, scale = factor((t, n), p, 9, 2)
    mask = kept.to(cuda).double() * float(scale)
    hd = 16.0 * td[ids]
    yd = hd @ w1.double().T + mask * (2.0 * (hd @ ad.T) @ bd.T)
    want_loss = nn.functional.cross_entropy(yd @ w2.double().T, labels)
    want = torch.autograd.grad(want_loss, leaves)
    eps = 2.0 ** -8
    # y is off by 2^-8 of itself, logits by as much of |y| |W2| as errors of random sign
    # leave, six deviations; the gradients by six roundings normwise
    dev = 6 * eps / math.sqrt(3) * float((yd.abs().square() @ w2.double().T.square()).sqrt().max())
    assert abs(float(loss.detach() - want_loss)) < dev / math.sqrt(300) * 2
    for x, ref in zip(got, want):
        assert float((x.double() - ref).norm() / ref.norm()) < 6 * eps


@pytest.mark.gpu
def test_trainer_takes_its_loss_from_the_head(cuda, tmp_path):
    """Loss and LoRA gradients of the two forms of the trainer's loss: the one from
    16-bit logits is off by their rounding."""
    for target in (["q_proj", "v_proj"], ["q_proj", "v_proj", "lm_head"]):
        runs = []
        for head in (None, "lm_head"):
            torch.manual_seed(0)
            model = Model(vocab=1000, device=cuda)
            trainer = LoRATrainer(model, TrainingConfig(
                rank=8, target_modules=target, output_dir=str(tmp_path), loss_head=head))
            with torch.no_grad():
                for _, m in trainer.params.layers:
                    m.B.normal_(0, 0.1, generator=torch.Generator(device=cuda).manual_seed(1))
                trainer.params.refresh_compute()
            ids = torch.randint(0, 1000, (4, 65), device=cuda,
                                generator=torch.Generator(device=cuda).manual_seed(2))
            labels = ids.clone()
            labels[:, :10] = -100
            loss = trainer.backward({"input_ids": ids, "labels": labels})
            runs.append((loss, trainer.params.grad.clone(), trainer))
            assert "forward" not in vars(model.lm_head)
        (l0, g0, _), (l1, g1, trainer) = runs
        # logits |l| <= 16 rounded to 2^-5 at most there, of random sign over 216 tokens
        assert abs(float(l0 - l1)) < 2.0 ** -5
        # 16-bit probabilities' gradients and logits' rounding, normwise
        assert float((g0 - g1).norm() / g1.norm()) < 2.0 ** -5
        assert g1.abs().sum() > 0
        metrics = trainer._training_step({"input_ids": ids, "labels": labels})
        assert math.isfinite(metrics["loss"])
        # the gradient buffer accumulates: two micro-batches, twice the gradient
        trainer.params.grad.zero_()
        trainer.backward({"input_ids": ids, "labels": labels})
        once = trainer.params.grad.clone()
        trainer.backward({"input_ids": ids, "labels": labels})
        assert torch.allclose(trainer.params.grad, 2 * once, rtol=1e-6, atol=0)


@pytest.mark.gpu
def test_trainer_refuses_a_head_that_is_not_last(cuda, tmp_path):
    model = Model(device=cuda, tail=True)
    trainer = LoRATrainer(model, TrainingConfig(output_dir=str(tmp_path), loss_head="lm_head"))
    ids = torch.zeros((1, 8), dtype=torch.int64, device=cuda)
    with pytest.raises(ConfigurationError):
        trainer.backward({"input_ids": ids, "labels": ids})
    assert model(ids).shape == (1, 8, 1003)  # the head is itself again
    out = trainer.backward({"input_ids": ids})  # no labels: the logits' loss, as ever
    assert float(out) == 0.0


@pytest.mark.gpu
def test_trainer_with_dropout_seed(cuda, tmp_path):
    """Masks differ from layer to layer and from step to step, and the same settings
    give the same run."""
    states = []
    for seed in (5, 5, 6):
        torch.manual_seed(0)
        model = Model(device=cuda)
        trainer = LoRATrainer(model, TrainingConfig(rank=8, dropout=0.3, dropout_seed=seed,
                                                    loss_head="lm_head", output_dir=str(tmp_path)))
        seeds = [m.dropout_seed for _, m in trainer.params.layers]
        assert seeds == [seed, seed + 1]
        ids = torch.randint(0, 1003, (2, 40), device=cuda,
                            generator=torch.Generator(device=cuda).manual_seed(2))
        for _ in range(3):
            trainer._training_step({"input_ids": ids, "labels": ids})
        assert [m.dropout_call for _, m in trainer.params.layers] == [3, 3]
        states.append(trainer.params.master.clone())
    assert torch.equal(states[0], states[1]) and not torch.equal(states[0], states[2])
