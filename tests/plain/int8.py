"""The dense decoder of ``plain/model.py`` with the matrices of its layers, and the inputs of their products, rounded to 8 bits a
row: v becomes step * rint(v / step) with step = max |v| / 127 of its row."""
from __future__ import annotations

import numpy as np

from . import model as pm


def coded(v: np.ndarray) -> np.ndarray:
    v = v.astype(np.float64)
    step = np.maximum(np.abs(v).max(axis=-1, keepdims=True) / 127, 2.0 ** -126)
    return np.rint(v / step) * step


def forward_logits(raw_config: dict, weights: dict, token_ids) -> np.ndarray:
    """``plain.model.forward_logits`` of that decoder; embedding, norms and output matrix are as they are."""
    cfg = pm.normalise_config(raw_config)
    held = {n: coded(w) if ".layers." in n and w.ndim == 2 else w for n, w in weights.items()}
    positions = np.arange(len(token_ids))
    x = pm.embedding(held["model.embed_tokens.weight"], token_ids)
    linear = pm.linear
    pm.linear = lambda rows, weight: linear(coded(rows), weight)
    try:
        for layer in range(cfg["num_hidden_layers"]):
            x = pm.decoder_block(x, held, layer, cfg, positions)
    finally:
        pm.linear = linear
    x = pm.rmsnorm(x, held["model.norm.weight"], cfg["rms_norm_eps"])
    return linear(x, held["model.embed_tokens.weight"] if cfg["tie_word_embeddings"] else held["lm_head.weight"])
