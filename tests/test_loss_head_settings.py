"""Loss heads that the trainer cannot take its loss from are refused before the model is
changed, or, where only the batch shows it, before a loss is made."""
import pytest
import torch
from torch import nn

from metallora_b200.exceptions import ConfigurationError
from metallora_b200.layers import LoRALinear
from metallora_b200.trainer import LoRATrainer, TrainingConfig
from tests.test_training_ends import Model

BF16 = torch.bfloat16


def test_heads_of_sizes_that_the_loss_refuses(tmp_path):
    def make(model, **kw):
        return LoRATrainer(model, TrainingConfig(output_dir=str(tmp_path / "out"), loss_head="lm_head",
                                                 **kw))
    adapted = ["q_proj", "lm_head"]
    large = Model(vocab=8, dim=8, hidden=8)
    large.lm_head = nn.Linear(8, (1 << 20) + 8, bias=False, dtype=BF16)
    for model, kw in ((Model(vocab=1003), {"target_modules": adapted}), (large, {}),
                      (large, {"target_modules": adapted})):
        with pytest.raises(ConfigurationError, match="out_features"):
            make(model, **kw)
        assert not any(isinstance(m, LoRALinear) for m in model.modules())
        assert not (tmp_path / "out").exists()
    make(Model(vocab=1003))  # an odd head takes no factors
    make(Model(vocab=1000), target_modules=adapted)
    # a head that is a LoRALinear already; merged, its factors take no part
    model = Model(vocab=1003)
    model.lm_head = LoRALinear(128, 1003, dtype=BF16)
    with pytest.raises(ConfigurationError, match="out_features"):
        make(model)
    model.lm_head.merged = True
    make(model)


def _loss_of(monkeypatch, head, tmp_path, ready=lambda model: None):
    """The trainer's loss with the operator replaced by torch's, on the CPU."""
    def loss(x, weight, labels, A=None, B=None, alpha=16.0, _compute=None, _sink=None):  # noqa: N803
        return nn.functional.cross_entropy((x @ weight.T).float().flatten(0, 1), labels.flatten())
    monkeypatch.setattr("metallora_b200.trainer.linear_cross_entropy", loss)
    monkeypatch.setattr("metallora_b200.layers.lora_forward", lambda x, w0, *a, **kw: x @ w0.T)
    model = nn.Sequential()
    model.embed, model.lm_head = nn.Embedding(64, 16, dtype=BF16), head
    ready(model)
    trainer = LoRATrainer(model, TrainingConfig(output_dir=str(tmp_path), loss_head="lm_head",
                                                target_modules=["lm_head"]))
    ids = torch.arange(8).reshape(2, 4)
    return trainer, lambda: trainer._compute_loss({"input_ids": ids, "labels": ids})


def test_a_head_with_dropout_is_refused_when_it_trains(monkeypatch, tmp_path):
    """Put to train() after the trainer was made; in eval() its dropout takes no part."""
    head = LoRALinear(16, 64, rank=8, dropout=0.5, dtype=BF16)
    _, loss = _loss_of(monkeypatch, head, tmp_path, ready=lambda model: model.eval())
    assert torch.isfinite(loss())
    head.train()
    with pytest.raises(ConfigurationError, match="dropout"):
        loss()
    head.merged = True
    assert torch.isfinite(loss())


def test_a_heads_own_forward_is_given_back(monkeypatch, tmp_path):
    head = LoRALinear(16, 64, rank=8, dtype=BF16)
    _, loss = _loss_of(monkeypatch, head, tmp_path)
    loss()
    assert "forward" not in vars(head)
    head.forward = wrapped = lambda x: LoRALinear.forward(head, x)
    loss()
    assert vars(head)["forward"] is wrapped
