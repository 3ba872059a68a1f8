"""The two gradient products of ``linear_token_logprobs`` on the MI355X: ``de = x c`` and ``dc = x^T e``.

Operands are small whole numbers: every sum stays below 2^24 and is exact in fp32 in any order, so the results have to equal
the 64-bit products rounded once, bit for bit."""
from __future__ import annotations

import pytest
import torch

from maester_amd import _lib
from maester_amd import linear_logprobs as LL

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _whole(*shape, seed, top=6):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-top, top + 1, shape, generator=g).double()


def _on_device(x, dtype, pitch=None):
    """``x`` in ``dtype`` with rows ``pitch`` apart, 1e4 between them."""
    pitch = x.shape[1] if pitch is None else pitch
    out = torch.full((x.shape[0], pitch), 1e4, dtype=dtype, device=DEV)
    out[:, : x.shape[1]] = x.to(DEV, dtype)
    return out[:, : x.shape[1]]


def _guarded(rows, dim, dtype, value=-7.0):
    """``[rows, dim]`` inside a buffer of ``value``, and the buffer."""
    room = torch.full((rows * dim + 2048,), value, dtype=dtype, device=DEV)
    return room[1024: 1024 + rows * dim].view(rows, dim), room


def _products(rows, vocab, dim, dtype, pitch_e=None, pitch_c=None, seed=0):
    x, e, c = _whole(rows, vocab, seed=seed), _whole(rows, dim, seed=seed + 1), _whole(vocab, dim, seed=seed + 2)
    assert 36 * max(rows, vocab) < 1 << 24
    padded = torch.zeros(rows, -(-vocab // 8) * 8, dtype=dtype, device=DEV)
    padded[:, :vocab] = x.to(DEV, dtype)
    return x, e, c, padded, _on_device(e, dtype, pitch_e), _on_device(c, dtype, pitch_c)


# around the edges of the tiles (256 by 256) and of a step of the contraction (64, fp32: 32), and one of several ranges
SHAPES = [(1, 1, 8), (1, 300, 8), (3, 64, 40), (31, 63, 264), (32, 65, 256), (33, 257, 248), (64, 256, 512), (65, 255, 520),
          (255, 1000, 136), (256, 2048, 64), (257, 2051, 72), (300, 40001, 304), (700, 513, 1048), (1025, 7, 8), (70001, 9, 16),
          (5, 40, 65536), (2, 300001, 16)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows,vocab,dim", SHAPES)
def test_whole_numbers_are_exact(rows, vocab, dim, dtype):
    x, e, c, xd, ed, cd = _products(rows, vocab, dim, dtype, seed=rows + vocab)
    de, room_e = _guarded(rows, dim, dtype)
    dc, room_c = _guarded(vocab, dim, dtype)
    LL._products(xd, ed, cd, de, dc, False)
    assert torch.equal(de.cpu(), (x @ c).to(dtype))
    assert torch.equal(dc.cpu(), (x.t() @ e).to(dtype))
    for room in (room_e, room_c):
        assert bool((room[:1024] == -7).all()) and bool((room[-1024:] == -7).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_strided_operands_one_output_and_sums_of_blocks(dtype):
    rows, vocab, dim = 130, 391, 328
    x, e, c, xd, ed, cd = _products(rows, vocab, dim, dtype, pitch_e=352, pitch_c=336, seed=5)
    de, _ = _guarded(rows, dim, dtype)
    LL._products(xd, ed, cd, de, None, False)
    assert torch.equal(de.cpu(), (x @ c).to(dtype))
    dc, room = _guarded(vocab, dim, torch.float32)
    dc.zero_()
    for part in (slice(0, 64), slice(64, 129), slice(129, 130)):
        LL._products(xd[part], ed[part], cd, None, dc, True)
    assert torch.equal(dc.double().cpu(), x.t() @ e)
    assert bool((room[:1024] == -7).all()) and bool((room[-1024:] == -7).all())


def test_non_finite_values_stay_where_they_belong():
    rows, vocab, dim = 70, 300, 264
    x, e, c, xd, ed, cd = _products(rows, vocab, dim, torch.bfloat16, seed=9)
    ed[3, 5] = float("nan")
    cd[17, 260] = float("inf")
    xd[:, 17] = 1.0
    de, _ = _guarded(rows, dim, torch.bfloat16)
    dc, _ = _guarded(vocab, dim, torch.bfloat16)
    LL._products(xd, ed, cd, de, dc, False)
    bad_e, bad_c = torch.zeros(rows, dim, dtype=torch.bool), torch.zeros(vocab, dim, dtype=torch.bool)
    bad_e[:, 260] = True
    bad_c[:, 5] = True
    assert torch.equal(~torch.isfinite(de.cpu()), bad_e)
    assert torch.equal(~torch.isfinite(dc.cpu()), bad_c)


def test_padding_of_the_vocabulary_takes_no_part():
    """All logits far below zero: exp(0 - lse) overflows in the padding behind the vocabulary."""
    rows, vocab, dim = 9, 1003, 64
    e = torch.ones(rows, dim, device=DEV, dtype=torch.bfloat16).requires_grad_()
    c = torch.full((vocab, dim), -40.0, device=DEV, dtype=torch.bfloat16).requires_grad_()
    targets = torch.arange(rows, device=DEV) * 100
    logp, entropy = LL.linear_token_logprobs(e, c, targets)
    (logp.sum() + entropy.sum()).backward()
    assert bool(torch.isfinite(e.grad).all()) and bool(torch.isfinite(c.grad).all())
    # every alternative is as likely: d logit = (target) - 1 / V, the entropy's gradient is 0
    want = torch.full((vocab, dim), -rows / vocab, dtype=torch.float64)
    want[targets.cpu()] += 1.0
    # each of x's rows and then dc is rounded to bf16, and 1 / V of nine rows is summed: 2^-8 (rows of x) + 2^-8
    assert float(((c.grad.double().cpu() - want).abs() / want.abs()).max()) <= 2 * 2.0 ** -8 + 1e-4


def test_refusals():
    rows, vocab, dim = 4, 24, 16
    _, _, _, xd, ed, cd = _products(rows, vocab, dim, torch.float32, seed=1)
    de = torch.empty(rows, dim, device=DEV)
    with pytest.raises((RuntimeError, ValueError), match="both outputs"):
        LL._products(xd, ed, cd, None, None, False)
    with pytest.raises((RuntimeError, ValueError), match="aligned"):
        LL._products(xd.view(-1)[1:65].view(4, 16), ed, cd[:16], de, None, False)
    L = _lib.lib()
    with pytest.raises((RuntimeError, ValueError), match="workspace"):
        need = L.ma_linear_grads_workspace_bytes(8, 40000, 64, 1, _lib.dtype_code(torch.float32))
        assert need > 0
        x, e, c = torch.zeros(8, 40000, device=DEV), torch.zeros(8, 64, device=DEV), torch.zeros(40000, 64, device=DEV)
        out = torch.empty(8, 64, device=DEV)
        _lib.launch(x.device, L.ma_linear_grads, x.data_ptr(), 40000, e.data_ptr(), 64, c.data_ptr(), 64, 8, 40000, 64, 1, out.data_ptr(), None, 0,
                    None, 0, _lib.dtype_code(torch.float32))
    meta = torch.empty(LL.MAX_GRAD_VOCAB + 1, 8, device=DEV, dtype=torch.bfloat16).requires_grad_()
    with pytest.raises(ValueError, match="vocabularies"):
        LL.linear_token_logprobs(torch.zeros(2, 8, device=DEV, dtype=torch.bfloat16), meta, torch.zeros(2, dtype=torch.int64, device=DEV))


def test_blocks_of_rows_under_another_default_dtype():
    """Several blocks sum the classifier's gradient in fp32 whatever new tensors are by default."""
    rows, vocab, dim = 37, 515, 64
    e, c = torch.randn(rows, dim, device=DEV), torch.randn(vocab, dim, device=DEV)
    targets = torch.randint(0, vocab, (rows,), device=DEV)
    grads = []
    for default in (torch.float32, torch.float64, torch.bfloat16):
        torch.set_default_dtype(default)
        try:
            a, b = e.clone().requires_grad_(), c.clone().requires_grad_()
            logp, entropy = LL.linear_token_logprobs(a, b, targets, chunk_rows=16)
            (logp.sum() + entropy.sum()).backward()
        finally:
            torch.set_default_dtype(torch.float32)
        grads.append((a.grad, b.grad))
    for g in grads[1:]:
        assert torch.equal(g[0], grads[0][0]) and torch.equal(g[1], grads[0][1])


def test_beyond_32_bits_of_offset():
    """The classifier and its gradient take 4.3 GB each; then the logits' gradient does."""
    rows, vocab, dim = 40, 262144, 8200
    torch.manual_seed(3)
    c = torch.randint(-3, 4, (vocab, dim), device=DEV, dtype=torch.int8).to(torch.bfloat16)
    x = torch.randint(-3, 4, (rows, vocab), device=DEV).to(torch.bfloat16)
    e = torch.randint(-3, 4, (rows, dim), device=DEV).to(torch.bfloat16)
    assert c.numel() * 2 > 1 << 32 and 9 * vocab < 1 << 24
    de, dc = torch.empty(rows, dim, device=DEV, dtype=torch.bfloat16), torch.empty_like(c)
    LL._products(x, e, c, de, dc, False)
    want = torch.zeros(rows, dim, device=DEV, dtype=torch.float64)
    for part in torch.arange(vocab, device=DEV).split(16384):
        lo, hi = int(part[0]), int(part[-1]) + 1
        want += x[:, lo:hi].double() @ c[lo:hi].double()
        assert torch.equal(dc[lo:hi], (x[:, lo:hi].double().t().contiguous() @ e.double()).to(torch.bfloat16)), lo
    assert torch.equal(de, want.to(torch.bfloat16))
    del c, dc, x

    rows, dim, last = 8300, 16, 70
    x = torch.zeros(rows, vocab, device=DEV, dtype=torch.bfloat16)
    assert (rows - last) * vocab * 2 > 1 << 32
    x[-last:] = torch.randint(-3, 4, (last, vocab), device=DEV).to(torch.bfloat16)
    e, c = (torch.randint(-3, 4, (n, dim), device=DEV).to(torch.bfloat16) for n in (rows, vocab))
    de, dc = torch.empty_like(e), torch.empty_like(c)
    LL._products(x, e, c, de, dc, False)
    tail = x[-last:].double()
    assert bool((de[:-last] == 0).all()) and torch.equal(de[-last:], (tail @ c.double()).to(torch.bfloat16))
    assert torch.equal(dc, (tail.t().contiguous() @ e[-last:].double()).to(torch.bfloat16))


def test_all_bits_of_fp32_operands_count():
    """Against one-hot rows the products are the other operand's values, 24 bits of them."""
    rows, vocab, dim = 67, 515, 132
    g = torch.Generator().manual_seed(11)
    x = torch.randn(rows, vocab, generator=g) * torch.exp2(torch.randint(-30, 30, (rows, vocab), generator=g).float())
    pick = torch.randint(0, vocab, (dim,), generator=g)
    c = torch.zeros(vocab, dim)
    c[pick, torch.arange(dim)] = 1.0
    pad = torch.zeros(rows, 520, device=DEV)
    pad[:, :vocab] = x.to(DEV)
    e = torch.zeros(rows, dim)
    e[torch.randint(0, rows, (dim,), generator=g), torch.arange(dim)] = -2.0
    de, dc = torch.empty(rows, dim, device=DEV), torch.empty(vocab, dim, device=DEV)
    LL._products(pad, e.to(DEV), c.to(DEV), de, dc, False)
    assert torch.equal(de.cpu(), x[:, pick])
    assert torch.equal(dc.cpu(), (x.double().t() @ e.double()).float())
    # and the other way round: one-hot logits' gradients pick rows of full e and c
    full_e, full_c = torch.randn(rows, dim, generator=g) * 1e-9, torch.randn(vocab, dim, generator=g) * 1e9
    x = torch.zeros(rows, vocab)
    order = torch.randperm(vocab, generator=g)[:rows]
    x[torch.arange(rows), order] = 1.0
    pad[:, :vocab] = x.to(DEV)
    LL._products(pad, full_e.to(DEV), full_c.to(DEV), de, dc, False)
    want = torch.zeros(vocab, dim)
    want[order] = full_e
    assert torch.equal(de.cpu(), full_c[order]) and torch.equal(dc.cpu(), want)


@pytest.mark.parametrize("rows,chunk", [(1, None), (2, None), (5, 3), (33, None), (64, None), (100, 50)])
def test_gradients_of_few_bf16_rows_are_rounded_once(rows, chunk):
    """Up to 64 rows at a time the gradient of the logits counts with 16 bits: what is left is the results' own rounding."""
    vocab, dim, g = 1003, 64, torch.Generator().manual_seed(rows)
    e = torch.randn(rows, dim, generator=g).to(torch.bfloat16)
    c = (torch.randn(vocab, dim, generator=g) * 3 / 8).to(torch.bfloat16)
    targets = torch.randint(0, vocab, (rows,), generator=g)
    a, b = torch.randn(rows, generator=g), 0.1 * torch.randn(rows, generator=g)
    ed, cd = e.to(DEV).requires_grad_(), c.to(DEV).requires_grad_()
    out = LL.linear_token_logprobs(ed, cd, targets.to(DEV), chunk_rows=chunk)
    de, dc = torch.autograd.grad(out, (ed, cd), (a.to(DEV), b.to(DEV)))
    lp = torch.log_softmax(e.double() @ c.double().t(), 1)
    p, h = lp.exp(), -(lp.exp() * lp).sum(1, keepdim=True)
    x = -p * (b[:, None].double() * (lp + h) + a[:, None].double())
    x[torch.arange(rows), targets] += a.double()
    for got, want, size in ((de, x @ c.double(), x.abs() @ c.double().abs()), (dc, x.t() @ e.double(), x.t().abs() @ e.double().abs())):
        # 2^-8 of the result; of its terms 2^-16 (the second part's rounding) and p's error, that of a logit: (K + 3) 2^-24 of
        # the sizes of its 64 products (some ten in all), with the factor of the entropy's gradient: 2^-13 together
        assert bool(((got.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -13 * size).all())
