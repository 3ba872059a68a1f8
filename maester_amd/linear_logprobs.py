"""Log-probabilities of given tokens and entropy from hidden states and the classifier, without the logits.

``token_logprobs`` of ``e @ c.T`` in one matrix-core kernel whose epilogue keeps the softmax statistics of every token: the
``[tokens, vocab]`` matrix never exists and its entries stay in fp32 (``linear_cross_entropy`` rounds a block of them to the
activation dtype between its GEMM and its softmax kernel).  The backward forms the gradient of the logits a block of rows
at a time, from the statistics that the forward kept, in the activation dtype, and multiplies it with the classifier and
the hidden states in matrix-core kernels that read both as they lie in memory.
"""
from __future__ import annotations

import torch

from . import _lib
from .linear_ce import default_chunk_rows
from .token_logprobs import check_softmax_arguments


def _check(e, c, targets):
    _lib.require_gpu(e, "linear_token_logprobs")
    if e.dim() != 2 or c.dim() != 2 or e.shape[1] != c.shape[1]:
        raise ValueError(f"e {tuple(e.shape)} and c {tuple(c.shape)} must be [N, K] and [V, K]")
    if e.dtype != c.dtype or e.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("e and c must share a dtype, bf16 or fp32")
    if targets.shape != (e.shape[0],) or targets.dtype != torch.int64:
        raise ValueError("targets must be int64 [N]")
    if c.device != e.device or targets.device != e.device:
        raise ValueError("e, c and targets must be on one device")
    unit = 16 // e.element_size()
    if e.shape[1] == 0 or e.shape[1] % unit or c.shape[0] == 0:
        raise ValueError(f"K must be a positive multiple of {unit} in {e.dtype} and V positive, got K={e.shape[1]}, V={c.shape[0]}")


def _rows_in_place(x: torch.Tensor) -> torch.Tensor:
    """``x`` itself where the kernels can read its rows where they are, else a contiguous copy."""
    unit = 16 // x.element_size()
    ok = x.stride(1) == 1 and (x.shape[0] <= 1 or (x.stride(0) >= x.shape[1] and x.stride(0) % unit == 0 and x.stride(0) <= 1 << 20))
    return x if ok and x.data_ptr() % 16 == 0 else x.contiguous().clone() if x.data_ptr() % 16 and x.is_contiguous() else x.contiguous()


def _pitch(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def linear_token_logprobs_forward(e, c, targets, ignore_index=-100, softcap=None, temperature=1.0):
    """``(logp, entropy, stats)`` for ``e`` ``[N, K]``, ``c`` ``[V, K]``, int64 ``targets`` ``[N]``."""
    _check(e, c, targets)
    softcap, temperature = check_softmax_arguments(softcap, temperature)
    e, c, targets = _rows_in_place(e), _rows_in_place(c), targets.contiguous()
    n, vocab = e.shape[0], c.shape[0]
    logp, entropy = (torch.empty(n, dtype=torch.float32, device=e.device) for _ in range(2))
    stats = torch.empty(n, 2, dtype=torch.float32, device=e.device)
    if n:
        L = _lib.lib()
        ws_bytes = L.ma_linear_logprobs_workspace_bytes(n, vocab)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=e.device)
        _lib.launch(e.device, L.ma_linear_logprobs_fwd, e.data_ptr(), _pitch(e), c.data_ptr(), _pitch(c), targets.data_ptr(), n, vocab,
                    e.shape[1], int(ignore_index), softcap, temperature, logp.data_ptr(), entropy.data_ptr(), stats.data_ptr(),
                    ws.data_ptr(), ws_bytes, _lib.dtype_code(e.dtype))
    return logp, entropy, stats


def _dlogits(e, c, targets, stats, entropy, dlogp, dentropy, ignore_index, softcap, temperature, out):
    """Gradient of the logits of a block of rows into ``out`` ``[rows, pitch]`` (``[2 rows, pitch]``: with what the rounding left)."""
    _lib.launch(e.device, _lib.lib().ma_linear_logprobs_dlogits, _lib.ptr(e), _pitch(e), _lib.ptr(c), _pitch(c), _lib.ptr(targets),
                e.shape[0], c.shape[0], e.shape[1], int(ignore_index), softcap, temperature, _lib.ptr(stats), _lib.ptr(entropy),
                _lib.ptr(dlogp), _lib.ptr(dentropy), _lib.ptr(out), out.shape[1], out.shape[0] // e.shape[0], _lib.dtype_code(e.dtype))


# Up to so many rows a bf16 gradient of the logits is kept in two parts of bf16: its rounding is the same for all results of a
# row's largest coefficient and does not average out among so few (the gradients' error is up to 2.5 times that of rounding
# them alone).  The products of so few rows are bound by memory: 2560 x 262208, 8 rows 798 -> 838 us, 64 rows 872 -> 975; 128
# rows would take 1168 for 983.
_TWO_PARTS_TO = 64
MAX_GRAD_VOCAB = 1 << 21                    # ma_linear_grads addresses 256 rows of the logits' gradient with 31 bits


def _products(x, e, c, de, dc, add, parts=1):
    """``de = x c`` (sums of ``parts`` rows of ``x``) and ``dc = x^T e`` (``add``: added to an fp32 ``dc``), either may be None;
    the rows of ``x`` are padded."""
    L, code = _lib.lib(), _lib.dtype_code(e.dtype)
    ws_bytes = 0 if de is None else L.ma_linear_grads_workspace_bytes(x.shape[0], c.shape[0], e.shape[1], parts, code)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=e.device) if ws_bytes else None
    _lib.launch(e.device, L.ma_linear_grads, x.data_ptr(), x.shape[1], e.data_ptr(), _pitch(e), c.data_ptr(), _pitch(c), x.shape[0],
                c.shape[0], e.shape[1], parts, _lib.ptr(de), _lib.ptr(dc), int(add), _lib.ptr(ws), ws_bytes,
                code)


def _counted_rows(e, targets, vocab, ignore_index, copies):
    """``copies`` copies of ``e``, one after the other, with zeros for the rows that do not count."""
    out = torch.empty(copies * e.shape[0], e.shape[1], dtype=e.dtype, device=e.device)
    _lib.launch(e.device, _lib.lib().ma_linear_counted_rows, _lib.ptr(e), _pitch(e), _lib.ptr(targets), e.shape[0], vocab, e.shape[1],
                int(ignore_index), copies, _lib.ptr(out), _lib.dtype_code(e.dtype))
    return out


def linear_token_logprobs_backward(e, c, targets, stats, entropy, dlogp, dentropy, ignore_index=-100, softcap=None,
                                   temperature=1.0, chunk_rows=None, need_de=True, need_dc=True, all_count=False):
    """``(de, dc)`` (None where not needed) from the gradients of ``logp`` and ``entropy`` (either may be None).
    ``all_count``: every target is known to count, so that ``dc`` may take the rows of ``e`` as they are."""
    softcap, temperature = check_softmax_arguments(softcap, temperature)
    e, c, targets = _rows_in_place(e), _rows_in_place(c), targets.contiguous()
    dlogp, dentropy = (None if t is None else t.float().contiguous() for t in (dlogp, dentropy))
    n, k = e.shape
    vocab = c.shape[0]
    de = torch.empty(n, k, dtype=e.dtype, device=e.device) if need_de else None
    if n == 0:
        return de, torch.zeros(vocab, k, dtype=c.dtype, device=c.device) if need_dc else None
    step = int(chunk_rows) if chunk_rows else default_chunk_rows(vocab, e.element_size(), n)
    step = max(1, min(step, n))
    parts = 2 if e.dtype == torch.bfloat16 and step <= _TWO_PARTS_TO else 1
    block = torch.empty(parts * step, -(-vocab // 8) * 8, dtype=e.dtype, device=e.device)
    # several blocks: dc is summed in fp32 and rounded once at the end
    dc = None
    if need_dc:
        dc = torch.empty(vocab, k, dtype=c.dtype, device=c.device) if n <= step else torch.zeros(vocab, k, dtype=torch.float32, device=c.device)
    for r0 in range(0, n, step):
        whole, rows = n <= step, slice(r0, min(n, r0 + step))
        buf = block[: parts * (rows.stop - r0)]
        e_rows, rest = e, (targets, stats, entropy, dlogp, dentropy)
        if not whole:
            e_rows, rest = e[rows], tuple(None if t is None else t[rows] for t in rest)
        _dlogits(e_rows, c, *rest, ignore_index, softcap, temperature, buf)
        if need_de or need_dc:
            if need_dc and (parts > 1 or not all_count):
                e_rows = _counted_rows(e_rows, rest[0], vocab, ignore_index, parts)
            _products(buf, e_rows, c, de if whole or de is None else de[rows], dc, not whole, parts)
    return de, dc.to(c.dtype) if need_dc else None


# Ignored rows are dropped from 257 rows on (up to 256 fill one block of the kernel's anyway) and from products of 2^36
# multiply-adds (fp32: 2^33) on: finding and gathering the others costs some 100 us with the wait (300 rows x 888 x 2064, forward and
# gradients: 283 us with, 140 without), a third of four such products as much.
_FILTER_FROM, _FILTER_WORK = 257, {torch.bfloat16: 1 << 36, torch.float32: 1 << 33}


def _kept_rows(targets, ignore_index, vocab):
    """Indices of the rows that count, or None for all of them (the one host synchronisation of a filtered call)."""
    valid = (targets != ignore_index) & (targets >= 0) & (targets < vocab)
    keep = torch.nonzero(valid).squeeze(1)
    return None if keep.numel() == targets.numel() else keep


class _LinearTokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, e, c, targets, ignore_index, softcap, temperature, chunk_rows, keep, all_count):
        ctx.rows, ctx.all_count = e.shape[0], all_count
        if keep is not None:
            e, targets = e.index_select(0, keep), targets.index_select(0, keep)
        logp, entropy, stats = linear_token_logprobs_forward(e, c, targets, ignore_index, softcap, temperature)
        # (the caller may edit the outputs: spread ones are copies, others share no memory with what is saved)
        ctx.save_for_backward(e, c, targets, stats, entropy.clone() if keep is None else entropy, keep)
        ctx.args = (ignore_index, softcap, temperature, chunk_rows)
        ctx.set_materialize_grads(False)
        return _spread(logp, keep, ctx.rows), _spread(entropy, keep, ctx.rows)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dlogp, dentropy):
        if dlogp is None and dentropy is None:
            return (None,) * 9
        e, c, targets, stats, entropy, keep = ctx.saved_tensors
        if keep is not None:
            dlogp, dentropy = (None if t is None else t.index_select(0, keep) for t in (dlogp, dentropy))
        de, dc = linear_token_logprobs_backward(e, c, targets, stats, entropy, dlogp, dentropy, *ctx.args,
                                                ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.all_count)
        return None if de is None else _spread(de, keep, ctx.rows), dc, None, None, None, None, None, None, None


def _spread(x, keep, rows):
    """``x`` of the kept rows as all rows', zeros elsewhere."""
    return x if keep is None else x.new_zeros((rows, *x.shape[1:])).index_copy_(0, keep, x)


def linear_token_logprobs(e: torch.Tensor, c: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100,
                          softcap: float | None = None, temperature: float = 1.0, chunk_rows: int | None = None,
                          filter_ignored: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """``(logp, entropy)`` of ``token_logprobs(e @ c.T, targets)``, fp32 of the shape of ``targets``, differentiable (once)
    in ``e`` and ``c``.

    ``e`` ``[..., K]`` hidden states, ``c`` ``[V, K]`` classifier (Gemma: the tied embedding table), bf16 or fp32 alike,
    ``K`` a multiple of 8 (fp32: 4); the logits are products of the inputs summed in fp32 and never stored (fp32: an infinity
    in ``e`` or ``c`` makes them NaN, where bf16 may give an infinity).  ``softcap``,
    ``temperature`` and ignored targets as in ``token_logprobs``.  ``chunk_rows``: rows per block of the backward (default:
    about 4 GiB of gradient of the logits at a time; V is at most 2^21 with gradients).  In bf16 a block's gradient of the
    logits is rounded to bf16 for the products with ``c`` and ``e``, which makes the gradients' error 1.4 times that of
    rounding them alone (2.4e-3 relative against 1.7e-3); a block of up to 64 rows keeps it in two parts, 16 bits, so that
    few rows, or more with ``chunk_rows=64`` at one pass over the classifier for each block, have the latter.  In fp32 operands
    below 2^-103 may lose their last bits.  ``filter_ignored``: a large call
    (more than 256 rows, 2^36 multiply-adds a product; fp32 2^33) drops the rows whose target does not count before any
    product, which costs its one host synchronisation; not under graph capture.  Either way such rows have no part in the
    results, whatever their hidden states hold."""
    if e.dim() < 1 or targets.shape != e.shape[:-1]:
        raise ValueError(f"targets shape {tuple(targets.shape)} != leading shape of e {tuple(e.shape[:-1])}")
    if chunk_rows is not None and int(chunk_rows) < 0:
        raise ValueError(f"chunk_rows must be positive, or None, got {chunk_rows}")
    _lib.require_plain("linear_token_logprobs", e, c, targets)
    _lib.refuse_tangents("linear_token_logprobs", e, c)
    lead = targets.shape
    if len(lead) != 1:
        e, targets = e.reshape(targets.numel(), e.shape[-1]), targets.reshape(-1)
    _check(e, c, targets)
    if c.shape[0] > MAX_GRAD_VOCAB and torch.is_grad_enabled() and (e.requires_grad or c.requires_grad):
        raise ValueError(f"gradients for vocabularies up to {MAX_GRAD_VOCAB}, got V={c.shape[0]}")
    keep, all_count = None, False
    if filter_ignored and e.shape[0] >= _FILTER_FROM and e.numel() * c.shape[0] >= _FILTER_WORK[e.dtype] and not torch.cuda.is_current_stream_capturing():
        keep, all_count = _kept_rows(targets, ignore_index, c.shape[0]), True
    if torch.is_grad_enabled() and (e.requires_grad or c.requires_grad):
        logp, entropy = _LinearTokenLogprobsFn.apply(e, c, targets, int(ignore_index), softcap, temperature, chunk_rows, keep, all_count)
    else:
        if keep is not None:
            e, targets = e.index_select(0, keep), targets.index_select(0, keep)
        logp, entropy, _ = linear_token_logprobs_forward(e, c, targets, ignore_index, softcap, temperature)
        logp, entropy = (_spread(t, keep, lead.numel()) for t in (logp, entropy))
    return (logp, entropy) if len(lead) == 1 else (logp.view(lead), entropy.view(lead))
