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
