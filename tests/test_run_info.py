"""The run description of a training report says which model ran: the reference's keys, and what
sets the model apart from the reference's."""

import torch

from llm_training_b200.config import ModelConfig
from llm_training_b200.train import Trainer

REFERENCE_KEYS = {"block_size", "vocab_size", "n_layer", "n_head", "n_embd", "dropout", "bias",
                  "attention"}


def model_config(**kw):
    cfg = ModelConfig(block_size=16, vocab_size=97, n_layer=1, n_head=2, n_embd=32, bias=False,
                      attention="tests.cpu_attention:CausalAttentionCPU", **kw)
    tr = Trainer(cfg, torch.device("cpu"))
    return tr.run_info(cfg, 2, 16, max_steps=1, lr=1e-3, seed=0)["model_config"]


def test_the_reference_s_model_has_its_keys_alone():
    assert set(model_config()) == REFERENCE_KEYS


def test_other_models_are_told_apart():
    got = model_config(post_norm=True, layer_scale=0.1)
    assert set(got) == REFERENCE_KEYS | {"post_norm", "layer_scale"}
    assert got["post_norm"] is True and got["layer_scale"] == 0.1
    assert model_config(layer_scale=0.0)["layer_scale"] == 0.0
    assert "layer_scale" not in model_config(post_norm=True)
