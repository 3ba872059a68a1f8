"""Log-probabilities of given tokens, entropy, top alternatives and their gradient against the fp64 oracle.

Tolerances, with u = 2^-24 (half a step of fp32, relative): every exponential is taken of a difference d that went
through three roundings (difference, temperature, log2 e) and an exp2 of at most two half steps, so its relative error
is at most (3 |d| + 2) u; terms with |d| > 40 weigh less than 1e-11 of the sum even a million of them together.  A
thread sums its vocab / 512 elements and the partial sums are joined in about 30 more steps, each adding at most u
(all terms have one sign).  The sum l, and likewise s = sum (y - m) exp(y - m), is therefore right to
    c = (3 * 40 + 2 + vocab / 512 + 30 + joins of split rows) u
relative: logp = (y_t - m) - log l to c + 4 u (|logp| + log l), the entropy log l - s / l to c + 2 c |s / l| + 4 u log l.
"""
import numpy as np
import pytest
import torch

import maester_amd
from maester_amd import token_logprobs
from oracle import token_logprobs as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def rel_of_sums(vocab):
    return (3 * 40 + 2 + vocab / 512 + 30 + 64) * U


def check_rows(got, want, vocab, tag=""):
    c = rel_of_sums(vocab)
    logp, entropy = got.logp.detach().double().cpu().numpy(), got.entropy.detach().double().cpu().numpy()
    log_v = np.log(vocab) + 1
    assert np.all(np.abs(logp - want["logp"]) <= c + 4 * U * (np.abs(want["logp"]) + log_v)), tag
    assert np.all(np.abs(entropy - want["entropy"]) <= c + 2 * c * log_v + 4 * U * log_v), tag
    if got.top_ids is not None:
        assert np.array_equal(got.top_ids.cpu().numpy(), want["top_ids"]), tag
        t, w = got.top_logp.double().cpu().numpy(), want["top_logp"]
        fine = np.isfinite(w)
        assert np.array_equal(t[~fine], w[~fine], equal_nan=True), tag
        assert np.all(np.abs(t - w)[fine] <= (c + 4 * U * (np.abs(w) + log_v))[fine]), tag


def make(rows, vocab, dtype, seed, ignore=0.25):
    g = torch.Generator().manual_seed(seed)
    x = (3 * torch.randn(rows, vocab, generator=g)).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g)
    t[torch.rand(rows, generator=g) < ignore] = -100
    t[0] = vocab - 1
    return x, t


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 64, 1003, 4095, 4097, 4096 * 3 + 5, 50257])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_forward(gpu, vocab, dtype):
    x, t = make(13, vocab, dtype, vocab)
    k = min(20, vocab)
    got = token_logprobs(x.to(gpu), t.to(gpu), top_k=k)
    check_rows(got, O.rows(x.float().numpy(), t.numpy(), top_k=k), vocab)


@pytest.mark.parametrize("rows,vocab,k", [(1, 262208, 20), (1, 262208, 64), (3, 262209, 1), (40, 128257, 5), (700, 3001, 64), (1500, 300, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_forward_row_counts(gpu, rows, vocab, k, dtype):
    # one row over the whole chip, few rows, more rows than the chip holds; bf16 rows of this width have ties at the top
    x, t = make(rows, vocab, dtype, rows)
    got = token_logprobs(x.to(gpu), t.to(gpu), top_k=k)
    check_rows(got, O.rows(x.float().numpy(), t.numpy(), top_k=k), vocab)


@pytest.mark.parametrize("softcap,temperature", [(30.0, 1.0), (None, 0.7), (5.0, 1.3)])
def test_softcap_and_temperature(gpu, softcap, temperature):
    # tanh of a library: 2 steps (4 u) of the cap on every logit, divided by the temperature
    x, t = make(21, 5003, torch.float32, 3)
    got = token_logprobs(x.to(gpu), t.to(gpu), top_k=9, softcap=softcap, temperature=temperature)
    want = O.rows(x.numpy(), t.numpy(), 9, softcap=softcap, temperature=temperature)
    extra = 4 * U * (softcap or 0) / temperature * 4
    c = rel_of_sums(5003) + extra
    assert np.abs(got.logp.cpu().numpy() - want["logp"]).max() <= c + 4 * U * 40
    assert np.abs(got.entropy.cpu().numpy() - want["entropy"]).max() <= 25 * c
    assert np.array_equal(got.top_ids.cpu().numpy(), want["top_ids"])


@pytest.mark.parametrize("vocab", [1, 3, 9, 4099])
@pytest.mark.parametrize("offset", [0, 1])
def test_small_caps_on_ragged_rows(gpu, vocab, offset):
    # a cap so low that an element beside the row, taken for a logit of -cap, would weigh as much as one of the row's
    buf = torch.randn(7, vocab + 5, generator=torch.Generator().manual_seed(vocab))
    x, t = buf[:, offset:offset + vocab], torch.arange(7) % vocab
    got = token_logprobs(buf.to(gpu)[:, offset:offset + vocab], t.to(gpu), top_k=1, softcap=0.5)
    want = O.rows(x.numpy(), t.numpy(), 1, softcap=0.5)
    tol = rel_of_sums(vocab) + 16 * U
    assert np.abs(got.logp.cpu().numpy() - want["logp"]).max() <= 4 * tol
    assert np.abs(got.entropy.cpu().numpy() - want["entropy"]).max() <= 25 * tol
    assert np.array_equal(got.top_ids.cpu().numpy(), want["top_ids"])
    # tanh(-inf) = -1: a soft cap gives banned tokens -cap, as the formula says
    x = x.clone()
    x[:, 0] = float("-inf")
    t = torch.full((7,), vocab - 1)
    got = token_logprobs(x.contiguous().to(gpu), t.to(gpu), softcap=0.5)
    assert np.abs(got.logp.cpu().numpy() - O.rows(x.numpy(), t.numpy(), softcap=0.5)["logp"]).max() <= 4 * tol


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_rows(gpu, dtype):
    vocab = 9001
    g = torch.Generator().manual_seed(5)
    x = torch.randn(8, vocab, generator=g).to(dtype)
    low = torch.finfo(dtype).min
    x[0] = float("-inf")                                  # nothing left: NaN
    x[1] = low                                            # the type's lowest value everywhere: uniform
    x[2, 1:] = float("-inf")                              # one token left: logp 0, entropy 0
    x[3, torch.randperm(vocab, generator=g)[:8990]] = float("-inf")
    x[4, ::2] = low
    x[5, 17] = float("nan")
    x[6, 4000] = float("inf")
    x[7, :] = 2.5                                         # all equal: the lowest indices lead
    t = torch.tensor([3, 4, 0, 5, 1, 7, 8, 9])
    t[3] = int(torch.isfinite(x[3]).nonzero()[0])
    got = token_logprobs(x.to(gpu), t.to(gpu), top_k=20)
    want = O.rows(x.float().numpy(), t.numpy(), 20)
    logp, ent = got.logp.cpu().numpy(), got.entropy.cpu().numpy()
    for r in (0, 5, 6):
        assert np.isnan(logp[r]) and np.isnan(ent[r])
    for r in (1, 2, 3, 4, 7):
        assert abs(logp[r] - want["logp"][r]) <= rel_of_sums(vocab) + 4 * U * 20
        assert abs(ent[r] - want["entropy"][r]) <= 25 * rel_of_sums(vocab)
    assert np.array_equal(got.top_ids.cpu().numpy(), want["top_ids"])       # -inf and NaN rank last, by index
    assert logp[2] == 0 and ent[2] == 0
    # a target that the mask excludes has probability 0
    out = token_logprobs(x[2:3].to(gpu), torch.tensor([5], device=gpu))
    assert float(out.logp) == float("-inf") and float(out.entropy) == 0


@pytest.mark.parametrize("vocab,stride", [(40000, 4096), (40000, 512), (262208, 4096), (5000, 8)])
@pytest.mark.parametrize("k", [3, 64])
def test_alternatives_in_clusters(gpu, vocab, stride, k):
    # the largest logits all in a few congruence classes of the index, ascending, descending and tied runs
    x = torch.zeros(6, vocab)
    n = len(x[0, ::stride])
    x[0, ::stride] = torch.arange(n).float() + 1
    x[1, 3::stride] = torch.arange(len(x[1, 3::stride])).flip(0).float() + 1
    x[2] = torch.arange(vocab).float()
    x[3] = -torch.arange(vocab).float()
    x[4, -700:] = 7.0
    for o in range(8):
        if o < vocab:
            x[5, o::stride] = 2.0 + o
    t = torch.zeros(6, dtype=torch.long)
    got = token_logprobs(x.to(gpu), t.to(gpu), top_k=k)
    assert np.array_equal(got.top_ids.cpu().numpy(), O.rows(x.numpy(), t.numpy(), k)["top_ids"])


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_and_misaligned_rows(gpu, offset, dtype):
    buf = torch.full((11, 1301), float("inf"), dtype=dtype)
    x, t = make(11, 1201, dtype, offset)
    buf[:, offset:offset + 1201] = x
    view = buf.to(gpu)[:, offset:offset + 1201]
    a, b = token_logprobs(view, t.to(gpu), top_k=8), token_logprobs(x.to(gpu), t.to(gpu), top_k=8)
    check_rows(a, O.rows(x.float().numpy(), t.numpy(), 8), 1201)
    assert torch.equal(a.top_ids, b.top_ids)
    leaf = buf.to(gpu).requires_grad_()
    leaf2 = x.to(gpu).requires_grad_()
    w = torch.randn(11, generator=torch.Generator().manual_seed(1)).to(gpu)
    (token_logprobs(leaf[:, offset:offset + 1201], t.to(gpu)).logp * w).sum().backward()
    (token_logprobs(leaf2, t.to(gpu)).logp * w).sum().backward()
    assert torch.all(leaf.grad[:, :offset] == 0) and torch.all(leaf.grad[:, offset + 1201:] == 0)
    # the rows' sums are formed in another order: c on the log-sum-exp, then one rounding to the type each
    lim = 2 * torch.finfo(dtype).eps * leaf2.grad.abs() + 2 * rel_of_sums(1201) * w.abs()[:, None]
    assert torch.all((leaf.grad[:, offset:offset + 1201] - leaf2.grad).abs().float() <= lim.float())


def gradient_limit(want, a, b, x, dtype, softcap, temperature, vocab):
    """One rounding to the type; lse and log p right to c + 4 u (|lse| + |y|); p relative to that and 2 steps of exp2; the
    factors of the formula one rounding each (8 u); a tanh 2 steps of its value and of the cap on y."""
    y = np.abs(np.where(np.isfinite(x), x, 0)) / temperature
    lp = np.where(want["p"] > 0, np.abs(want["lp"]), 0)
    e = rel_of_sums(vocab) + 4 * U * (np.abs(want["lse"])[:, None] + y + 1) + 16 * U * (softcap or 0) / temperature
    coef = np.abs(a)[:, None] + np.abs(b)[:, None] * (lp + np.log(vocab) + 1)
    one = np.zeros_like(want["p"])
    return (torch.finfo(dtype).eps / 2 * np.abs(want["dx"]) + (want["p"] * coef * (e + 8 * U) + want["p"] * np.abs(b)[:, None] * 2 * np.log(vocab + 1) * e
            + one + np.abs(a)[:, None] * 4 * U + coef * (16 * U if softcap else 0) * want["p"] + 1e-37) / temperature)


@pytest.mark.parametrize("rows,vocab", [(5, 3), (17, 1003), (9, 50257), (2, 262209), (300, 640)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("softcap,temperature", [(None, 1.0), (30.0, 0.7)])
def test_gradient(gpu, rows, vocab, dtype, softcap, temperature):
    x, t = make(rows, vocab, dtype, rows + vocab)
    g = torch.Generator().manual_seed(9)
    a, b = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    leaf = x.to(gpu).requires_grad_()
    out = token_logprobs(leaf, t.to(gpu), softcap=softcap, temperature=temperature)
    got, = torch.autograd.grad((out.logp, out.entropy), leaf, (a.to(gpu), b.to(gpu)))
    want = O.rows(x.float().numpy(), t.numpy(), 0, softcap=softcap, temperature=temperature, dlogp=a.numpy(), dentropy=b.numpy())
    err = np.abs(got.double().cpu().numpy() - want["dx"])
    lim = gradient_limit(want, a.numpy(), b.numpy(), x.double().numpy(), dtype, softcap, temperature, vocab)
    assert got.dtype == dtype and np.all(err <= lim), float((err / lim).max())
    assert torch.all(got[t.to(gpu) == -100] == 0)


def test_gradient_against_differences(gpu):
    # (f(x + h v) - f(x - h v)) / 2h of logp and entropy in fp64 from the oracle, along random directions
    x, t = make(6, 200, torch.float32, 11, ignore=0.0)
    leaf = x.to(gpu).requires_grad_()
    out = token_logprobs(leaf, t.to(gpu), softcap=20.0, temperature=0.8)
    g = torch.Generator().manual_seed(2)
    v = torch.randn(6, 200, generator=g, dtype=torch.float64)
    h = 1e-4
    hi, lo = (O.rows((x.double() + s * h * v).numpy(), t.numpy(), softcap=20.0, temperature=0.8) for s in (1, -1))
    for name, y in (("logp", out.logp), ("entropy", out.entropy)):
        d, = torch.autograd.grad(y.sum(), leaf, retain_graph=True)
        got = (d.double().cpu() * v).sum(1).numpy()
        want = (hi[name] - lo[name]) / (2 * h)
        # third derivatives of order 10 times h^2 |v|^3, fp32 gradients of order 1 over 200 terms
        assert np.abs(got - want).max() <= 1e-4, name


def test_gradient_of_masked_rows_and_single_outputs(gpu):
    x = torch.randn(4, 500, generator=torch.Generator().manual_seed(4))
    x[:, 100:400] = float("-inf")
    x[3] = float("-inf")
    t = torch.tensor([1, 2, 499, -100])
    leaf = x.to(gpu).requires_grad_()
    out = token_logprobs(leaf, t.to(gpu), top_k=3)
    d, = torch.autograd.grad(out.logp.sum(), leaf, retain_graph=True)
    want = O.rows(x.numpy(), t.numpy(), dlogp=np.ones(4), dentropy=np.zeros(4))["dx"]
    assert torch.all(d[:, 100:400] == 0) and np.abs(d.cpu().numpy()[:3] - want[:3]).max() <= 1e-6      # p <= 1, few u each
    assert torch.all(d[3] == 0)
    d, = torch.autograd.grad(out.entropy.sum(), leaf)
    want = O.rows(x.numpy(), t.numpy(), dlogp=np.zeros(4), dentropy=np.ones(4))["dx"]
    assert torch.isfinite(d).all() and np.abs(d.cpu().numpy()[:3] - want[:3]).max() <= 1e-5
    low = torch.full((2, 64), torch.finfo(torch.float32).min, device=gpu, requires_grad=True)
    token_logprobs(low, torch.tensor([0, 63], device=gpu)).logp.sum().backward()
    assert float((low.grad[0, 1:] + 1 / 64).abs().max()) <= 1e-6 and abs(float(low.grad[1, 63]) - 63 / 64) <= 1e-6
    assert not out.top_logp.requires_grad and not out.top_ids.requires_grad


def test_shapes_targets_and_empty_batches(gpu):
    x, t = make(12, 100, torch.float32, 6)
    t[3], t[4] = 100, -5                                   # outside the vocabulary: like ignore_index
    flat = token_logprobs(x.to(gpu), t.to(gpu), top_k=4)
    assert float(flat.logp[3]) == 0 and float(flat.entropy[4]) == 0 and float(flat.entropy[0]) > 0
    shaped = token_logprobs(x.view(3, 4, 100).to(gpu), t.view(3, 4).to(gpu), top_k=4)
    assert shaped.top_ids.shape == (3, 4, 4) and torch.equal(shaped.logp.view(-1), flat.logp)
    one = token_logprobs(x[0].to(gpu), t[0].to(gpu))       # a single row without a batch dimension
    assert one.logp.shape == () and float(one.logp) == float(flat.logp[0]) and one.top_ids is None
    empty = token_logprobs(torch.empty(0, 100, device=gpu), torch.empty(0, dtype=torch.long, device=gpu), top_k=2)
    assert empty.logp.shape == (0,) and empty.top_ids.shape == (0, 2)
    leaf = torch.empty(0, 100, device=gpu, requires_grad=True)
    token_logprobs(leaf, torch.empty(0, dtype=torch.long, device=gpu)).logp.sum().backward()
    assert leaf.grad.shape == (0, 100)


def test_refusals(gpu):
    x, t = torch.zeros(4, 10, device=gpu), torch.zeros(4, dtype=torch.long, device=gpu)
    for kw in (dict(top_k=11), dict(top_k=-1), dict(temperature=0.0), dict(temperature=float("nan")), dict(softcap=-1.0)):
        with pytest.raises(ValueError):
            token_logprobs(x, t, **kw)
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(4, 100, device=gpu), t, top_k=65)
    with pytest.raises(ValueError):
        token_logprobs(x, t[:3])
    with pytest.raises(ValueError):
        token_logprobs(x, t.int())
    with pytest.raises(ValueError):
        token_logprobs(x, t.cpu())
    with pytest.raises(ValueError):
        token_logprobs(x.t().contiguous().t(), t)
    with pytest.raises(TypeError):
        token_logprobs(x.half(), t)
    with pytest.raises(RuntimeError):
        token_logprobs(x.cpu(), t.cpu())


def test_beyond_32_bits_of_offset(gpu):
    # 8300 x 262208 bf16 is 2^31 elements and more: its last rows as a batch of their own
    rows, vocab = 8300, 262208
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=gpu)
    t = torch.randint(0, vocab, (rows,), device=gpu)
    x[-3:].normal_()
    x[-3:] *= 3
    a = torch.ones(rows, device=gpu)
    whole = x.requires_grad_()
    out = token_logprobs(whole, t, top_k=4)
    d, = torch.autograd.grad((out.logp, out.entropy), whole, (a, a))
    part = x[-3:].detach().clone().requires_grad_()
    want = token_logprobs(part, t[-3:], top_k=4)
    e, = torch.autograd.grad((want.logp, want.entropy), part, (a[-3:], a[-3:]))
    # (few rows are cut into parts: another order of the sums)
    c = rel_of_sums(vocab)
    assert float((out.logp[-3:] - want.logp).abs().max()) <= 2 * c and float((out.entropy[-3:] - want.entropy).abs().max()) <= 50 * c
    assert torch.equal(out.top_ids[-3:], want.top_ids)
    assert float((d[-3:].float() - e.float()).abs().max()) <= 2 * 2.0 ** -8 * float(e.abs().max())
    assert abs(float(out.logp[0]) + np.log(vocab)) <= 2 * c * 13


def test_gradient_in_place_of_the_logits(gpu):
    # the C entry point may write the gradient over the logits themselves
    from maester_amd import _lib
    from maester_amd.token_logprobs import token_logprobs_backward, token_logprobs_forward
    for vocab in (1003, 4096):
        x, t = make(9, vocab, torch.bfloat16, vocab)
        xg, tg = x.to(gpu), t.to(gpu)
        a = torch.randn(9, device=gpu)
        _, entropy, stats, _, _ = token_logprobs_forward(xg, tg)
        want = token_logprobs_backward(xg, tg, stats, entropy, a, a)
        rc = _lib.lib().ma_token_logprobs_bwd(xg.data_ptr(), vocab, tg.data_ptr(), 9, vocab, -100, 0.0, 1.0, stats.data_ptr(), entropy.data_ptr(),
                                              a.data_ptr(), a.data_ptr(), xg.data_ptr(), vocab, _lib.MA_DTYPE_BF16, _lib.current_stream(xg.device))
        _lib.check(rc)
        assert torch.equal(xg, want)


def test_other_stream_and_graph_replay(gpu):
    x, t = make(33, 30011, torch.bfloat16, 8)
    xg, tg = x.to(gpu), t.to(gpu)
    w = torch.randn(33, device=gpu)
    leaf = xg.clone().requires_grad_()

    def step():
        out = token_logprobs(leaf, tg, top_k=5)
        d, = torch.autograd.grad((out.logp, out.entropy), leaf, (w, w))
        return out.logp.detach(), out.entropy.detach(), out.top_ids, d

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n in range(3):
        with torch.no_grad():
            leaf.copy_(xg * (n + 1))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager)), n
    with torch.no_grad():
        leaf.copy_(xg)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_large_entropy_gradients_on_masked_rows(gpu):
    """A masked alternative has probability 0 and no gradient, however large the entropy's is."""
    x = torch.randn(3, 700, dtype=torch.float64)
    x[:, 300:] = -float("inf")
    x[1, 5:300] = torch.finfo(torch.float32).min
    leaf = x.float().to(gpu).requires_grad_()
    out = token_logprobs(leaf, torch.tensor([3, 1, 299], device=gpu))
    (out.entropy * 1e12).sum().backward()
    got = leaf.grad.double().cpu()
    assert bool(torch.isfinite(got).all()) and bool((got[:, 300:] == 0).all())
    p = torch.softmax(x.float().double(), 1)
    lp = torch.where(p > 0, torch.log(p.clamp_min(1e-300)), torch.zeros_like(p))
    h = -(p * lp).sum(1, keepdim=True)
    # p, log p + H and their product: errors of 2^-24 relative to |log p| + H + 1, some tens of operations
    assert bool(((got + 1e12 * p * (lp + h)).abs() <= 1e12 * 64 * 2.0 ** -24 * (p * (lp.abs() + h + 1) ** 2 + 1e-30)).all())
