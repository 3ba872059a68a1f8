"""Log-probabilities of given tokens, entropy, best alternatives and their gradient, in fp64 from the definitions."""
from __future__ import annotations

import numpy as np


def rows(x: np.ndarray, targets: np.ndarray, top_k: int = 0, ignore_index: int = -100, softcap: float | None = None,
         temperature: float = 1.0, dlogp: np.ndarray | None = None, dentropy: np.ndarray | None = None) -> dict:
    """``x`` ``[rows, vocab]``; a target outside the vocabulary counts as ignored."""
    raw = np.asarray(x, dtype=np.float64)
    n, vocab = raw.shape
    with np.errstate(all="ignore"):
        y = softcap * np.tanh(raw / softcap) if softcap else raw
        y = y / temperature
        big = y.max(1, keepdims=True)
        z = np.exp(y - big)
        z[np.isneginf(y) & np.isfinite(big)] = 0.0
        log_sum = np.log(z.sum(1))
        lse = big[:, 0] + log_sum
        lp = (y - big) - log_sum[:, None]       # not y - lse: rows of the type's lowest value would absorb the logarithm
        p = np.exp(lp)
        plp = np.where(p == 0, 0.0, p * lp)
        entropy = -plp.sum(1)
    keep = (targets != ignore_index) & (targets >= 0) & (targets < vocab)
    t = np.where(keep, targets, 0)
    out = {"lse": lse, "entropy": np.where(keep, entropy, 0.0), "logp": np.where(keep, lp[np.arange(n), t], 0.0), "keep": keep}
    if top_k:
        rank = np.where(np.isnan(raw), -np.inf, raw)
        # descending value, then ascending index
        out["top_ids"] = np.argsort(-rank, axis=1, kind="stable")[:, :top_k]
        out["top_logp"] = np.take_along_axis(lp, out["top_ids"], 1)
    if dlogp is not None or dentropy is not None:
        a = np.zeros(n) if dlogp is None else np.asarray(dlogp, dtype=np.float64)
        b = np.zeros(n) if dentropy is None else np.asarray(dentropy, dtype=np.float64)
        one = np.zeros_like(p)
        one[np.arange(n), t] = 1.0
        d = a[:, None] * (one - p) - b[:, None] * (plp + p * entropy[:, None])
        if softcap:
            d = d * (1.0 - np.tanh(raw / softcap) ** 2)
        out["dx"] = np.where(keep[:, None], d / temperature, 0.0)
        out["p"], out["lp"] = p, lp
    return out
