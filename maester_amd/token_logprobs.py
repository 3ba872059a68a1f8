"""Log-probabilities of given tokens, entropy and top alternatives: the per-token form of the model's loss.

``linear_cross_entropy`` ends a supervised step with one scalar (maester/models/gemma/model.py:762-769).  Objectives that
weigh tokens themselves -- policy and preference losses, distillation, filtering and scoring of packed batches -- need the
log-probability of every label, the entropy of every position and, to look at or to distil from, the best alternatives.
``token_logprobs`` computes them from rows of logits in one pass over the row, with the gradient of the first two.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` returns.  ``logp`` and ``entropy`` fp32 of the shape of the targets, ``top_ids`` int64 and
    ``top_logp`` fp32 with ``top_k`` more entries each (best first), ``None`` with ``top_k=0``."""
    logp: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor | None
    top_logp: torch.Tensor | None


def check_softmax_arguments(softcap, temperature) -> tuple[float, float]:
    """(softcap, 0.0 for none; temperature) as the library takes them."""
    softcap = 0.0 if softcap is None else float(softcap)
    if softcap != 0.0 and not 1e-30 <= softcap <= 1e30:      # (the kernels take its reciprocal in fp32)
        raise ValueError(f"softcap must be in [1e-30, 1e30], or None, got {softcap}")
    if not 1e-6 < float(temperature) <= 1e6:
        raise ValueError(f"temperature must be in (1e-6, 1e6], got {temperature}")
    return softcap, float(temperature)


def token_logprobs_forward(logits, targets, top_k=0, ignore_index=-100, softcap=None, temperature=1.0, need_stats=True):
    """``(logp, entropy, stats, top_ids, top_logp)`` of ``logits`` ``[rows, vocab]`` (rows may be strided) and int64
    ``targets`` ``[rows]``; ``stats`` ``[rows, 2]`` is what the gradient needs of the forward (``need_stats=False``: None)."""
    _lib.require_gpu(logits, "token_logprobs")
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError("logits must be [rows, vocab] with unit stride along the vocabulary")
    rows, vocab = logits.shape
    dev = logits.device
    if targets.shape != (rows,) or targets.dtype != torch.int64 or targets.device != dev:
        raise ValueError("targets must be int64 [rows] on the device of the logits")
    top_k = int(top_k)
    if not 0 <= top_k <= min(_lib.MA_LOGPROBS_MAX_TOP, vocab):
        raise ValueError(f"top_k must be in 0 .. {_lib.MA_LOGPROBS_MAX_TOP} and at most the vocabulary of {vocab}, got {top_k}")
    softcap, temperature = check_softmax_arguments(softcap, temperature)
    code = _lib.dtype_code(logits.dtype)
    logits, targets = _apart(logits), targets.contiguous()
    logp, entropy = (torch.empty(rows, dtype=torch.float32, device=dev) for _ in range(2))
    stats = torch.empty(rows, 2, dtype=torch.float32, device=dev) if need_stats else None
    top_ids = torch.empty(rows, top_k, dtype=torch.int64, device=dev) if top_k else None
    top_logp = torch.empty(rows, top_k, dtype=torch.float32, device=dev) if top_k else None
    if rows:
        L = _lib.lib()
        ws_bytes = L.ma_token_logprobs_workspace_bytes(rows, vocab, top_k)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
        _lib.launch(dev, L.ma_token_logprobs_fwd, logits.data_ptr(), _row_pitch(logits), targets.data_ptr(), rows, vocab, int(ignore_index),
                    softcap, temperature, top_k, logp.data_ptr(), entropy.data_ptr(), stats.data_ptr() if need_stats else None,
                    top_ids.data_ptr() if top_k else None, top_logp.data_ptr() if top_k else None, ws.data_ptr() if ws_bytes else None,
                    ws_bytes, code)
    return logp, entropy, stats, top_ids, top_logp


def _apart(x: torch.Tensor) -> torch.Tensor:
    """``x`` itself, or a copy where its rows share memory (a broadcast row)."""
    return x.contiguous() if x.shape[0] > 1 and x.stride(0) < x.shape[1] else x


def _row_pitch(x: torch.Tensor) -> int:
    """Elements between rows (a single row has no meaningful stride)."""
    return x.stride(0) if x.shape[0] > 1 else max(x.stride(0), x.shape[1])


def token_logprobs_backward(logits, targets, stats, entropy, dlogp, dentropy, ignore_index=-100, softcap=None, temperature=1.0):
    """Gradient of the logits, contiguous, from those of ``logp`` and ``entropy`` (either may be None)."""
    softcap, temperature = check_softmax_arguments(softcap, temperature)
    logits, targets = _apart(logits), targets.contiguous()
    dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    rows, vocab = logits.shape
    dlogp, dentropy = (None if t is None else t.float().contiguous() for t in (dlogp, dentropy))
    if rows:
        _lib.launch(logits.device, _lib.lib().ma_token_logprobs_bwd, _lib.ptr(logits), _row_pitch(logits), _lib.ptr(targets), rows, vocab,
                    int(ignore_index), softcap, temperature, _lib.ptr(stats), _lib.ptr(entropy), _lib.ptr(dlogp), _lib.ptr(dentropy),
                    _lib.ptr(dlogits), vocab, _lib.dtype_code(logits.dtype))
    return dlogits


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k, ignore_index, softcap, temperature):
        logp, entropy, stats, top_ids, top_logp = token_logprobs_forward(logits, targets, top_k, ignore_index, softcap, temperature)
        ctx.save_for_backward(logits, targets, stats, entropy.clone())       # (the caller may edit the output)
        ctx.args = (ignore_index, softcap, temperature)
        ctx.set_materialize_grads(False)
        if top_k:
            ctx.mark_non_differentiable(top_ids, top_logp)
        return logp, entropy, top_ids, top_logp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dlogp, dentropy, dids, dtop):
        if dlogp is None and dentropy is None:
            return (None,) * 6
        logits, targets, stats, entropy = ctx.saved_tensors
        return (token_logprobs_backward(logits, targets, stats, entropy, dlogp, dentropy, *ctx.args),) + (None,) * 5


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top_k: int = 0, ignore_index: int = -100,
                   softcap: float | None = None, temperature: float = 1.0) -> TokenLogprobs:
    """Log-probability of every target, entropy and the ``top_k`` (at most 64) best alternatives of rows of logits.

    ``logits`` ``[..., V]`` bf16 or fp32, ``targets`` int64 of the leading shape.  Entries of a row are neighbours in memory (a
    transposed matrix is refused); rows may lie apart, anywhere, in a matrix, while more dimensions whose rows are not
    evenly spaced, such as ``logits[:, :-1]`` of a batch, and rows that share memory are copied first.  Logits are capped as
    ``softcap * tanh(x / softcap)`` where a cap is given, then divided by ``temperature``.  Rows whose target is
    ``ignore_index`` (or outside the vocabulary) get 0 for both and no gradient; the alternatives come for every row,
    equal logits in the order of their index.  Logits of ``-inf`` have probability 0 (a soft cap makes them
    ``-softcap`` first: mask after capping); a row with a NaN or ``+inf``, or with nothing but ``-inf``, gives NaN.
    ``logp`` and ``entropy`` are differentiable in the logits (once), the alternatives are not."""
    if logits.dim() < 1 or targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets shape {tuple(targets.shape)} != leading shape of logits {tuple(logits.shape[:-1])}")
    _lib.require_plain("token_logprobs", logits, targets)
    _lib.refuse_tangents("token_logprobs", logits)
    lead, vocab = targets.shape, logits.shape[-1]
    if vocab < 1:
        raise ValueError("empty vocabulary")
    if len(lead) != 1:
        logits, targets = logits.reshape(targets.numel(), vocab), targets.reshape(-1)
    if logits.requires_grad and torch.is_grad_enabled():
        logp, entropy, top_ids, top_logp = _TokenLogprobsFn.apply(logits, targets, int(top_k), int(ignore_index), softcap, temperature)
    else:
        logp, entropy, _, top_ids, top_logp = token_logprobs_forward(logits, targets, top_k, ignore_index, softcap, temperature, False)
    if len(lead) != 1:
        logp, entropy = logp.view(lead), entropy.view(lead)
        if top_ids is not None:
            top_ids, top_logp = (x.view(*lead, x.shape[1]) for x in (top_ids, top_logp))
    return TokenLogprobs(logp, entropy, top_ids, top_logp)
