"""Checkpoints whose q/k norms are not per head."""
import pytest
import torch

from phung5_b200.config import preset
from phung5_b200.models.llama import pack_weights
from phung5_b200.weights.init import random_weights
from phung5_b200.weights.loader import load_model, save_checkpoint


def test_norms_over_the_whole_projection_are_refused_on_loading(tmp_path):
    """Weights [num_heads * head_dim] are a norm over all heads at once, which the operator does not compute."""
    cfg = preset("tiny", num_layers=2, qk_norm=True)
    w = random_weights(cfg, seed=3)
    pack_weights(cfg, w, "cpu")
    for k in list(w):
        if k.endswith("q_norm.weight"):
            w[k] = torch.ones(cfg.q_size)
        elif k.endswith("k_norm.weight"):
            w[k] = torch.ones(cfg.kv_size)
    save_checkpoint(w, cfg, str(tmp_path))
    with pytest.raises(ValueError, match="per head"):
        load_model(str(tmp_path), "cpu")
    w["model.layers.0.self_attn.q_norm.weight"] = torch.ones(cfg.head_dim)
    with pytest.raises(ValueError, match="k_norm"):
        pack_weights(cfg, w, "cpu")
