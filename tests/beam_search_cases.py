"""Models for the tests of beam search: per architecture a configuration, weights and the plain logits behind some tokens."""

from __future__ import annotations

import lunelorn_cases
import nogatar_cases
import nukodra_cases
import plain_gpt
import vumotar_cases
import zenedra_cases
from harness import make_tensors, tiny_config, tokens_for

from mini_gpt_inference_b200 import LunelornConfig, NogatarConfig, NukodraConfig, VumotarConfig, ZenedraConfig
from mini_gpt_inference_b200.engine.build import load_model

OTHERS = {"zenedra": (zenedra_cases, ZenedraConfig), "nukodra": (nukodra_cases, NukodraConfig), "lunelorn": (lunelorn_cases, LunelornConfig),
          "nogatar": (nogatar_cases, NogatarConfig), "vumotar": (vumotar_cases, VumotarConfig)}


def model(which: str, dtype: str, device: str):
    """(loaded model, last_logits(tokens), tokens(length, seed), vocabulary)."""
    if which in ("A", "B"):
        cfg = tiny_config(which)
        tensors = make_tensors(cfg, 5, dtype, sharp=True)
        loaded = load_model(config=cfg, tensors=tensors, dtype=dtype, device=device)
        last = lambda tokens: plain_gpt.forward_logits(tokens, tensors, cfg.n_layer, cfg.n_head, cfg.layer_norm_epsilon)[-1]  # noqa: E731
        return loaded, last, lambda n, seed: tokens_for(cfg, n, seed), cfg.vocab_size
    cases, kind = OTHERS[which]
    raw = cases.config("A")
    import torch

    tensors = cases.random_weights(raw, 7, torch.bfloat16 if dtype == "bfloat16" else torch.float32)
    loaded = load_model(config=kind.from_dict(raw), tensors=tensors, dtype=dtype, device=device)
    return loaded, lambda tokens: cases.plain_logits(raw, tensors, tokens)[-1], lambda n, seed: cases.tokens_for(raw, n, seed), raw["vocab"]
