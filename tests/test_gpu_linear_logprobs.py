"""Log-probabilities and entropy from hidden states and the classifier, and their gradients, against fp64.

The logits are sums of K products of the inputs (exact in fp32 for bf16 inputs) in fp32: each off by at most
K u sum |e_k c_k| worst case, and by sqrt(K) u times that sum's root mean square in earnest; the inputs here have
logits of order 1 to 10 built from terms of either sign, and 4 sqrt(K) u max|x| + 1e-6 bounds the error of every one of
them with room (u = 2^-24).  After that the tolerance of the form on logits holds (c below).  Gradients: the gradient
of the logits is rounded to the activation dtype (half a step each) and multiplied by the library, and the result is
rounded again: relative L2 two half steps of the type; fp32 1e-5."""
import math

import numpy as np
import pytest
import torch

from maester_amd import linear_token_logprobs, token_logprobs
from oracle import token_logprobs as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def problem(n, k, vocab, dtype, seed, ignore=0.25, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    e = torch.randn(n, k, generator=g).to(dtype)
    c = (torch.randn(vocab, k, generator=g) * scale / math.sqrt(k)).to(dtype)
    t = torch.randint(0, vocab, (n,), generator=g)
    t[torch.rand(n, generator=g) < ignore] = -100
    t[0] = vocab - 1
    return e, c, t


def limits(k, vocab, x, softcap, temperature):
    dx = (4 * math.sqrt(k) * U * np.abs(x).max() + 1e-6 + 16 * U * (softcap or 0)) / temperature
    c = (3 * 40 + 2 + 512 + 60) * U + 2 * dx
    log_v = math.log(vocab) + 1
    return c + 4 * U * (np.abs(x).max() / temperature + log_v), c + 2 * c * log_v + 4 * U * log_v


def check(gpu, e, c, t, softcap=None, temperature=1.0):
    logp, entropy = linear_token_logprobs(e.to(gpu), c.to(gpu), t.to(gpu), softcap=softcap, temperature=temperature)
    x = (e.double() @ c.double().t()).numpy()
    want = O.rows(x, t.numpy(), softcap=softcap, temperature=temperature)
    tol_p, tol_h = limits(e.shape[1], c.shape[0], x, softcap, temperature)
    a, b = np.abs(logp.cpu().numpy() - want["logp"]).max(), np.abs(entropy.cpu().numpy() - want["entropy"]).max()
    assert a <= tol_p and b <= tol_h, (a, tol_p, b, tol_h)
    assert torch.all(logp[t.to(gpu) == -100] == 0) and torch.all(entropy[t.to(gpu) == -100] == 0)


# rows around every block width, widths with ragged last steps, vocabularies around tile and range edges
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 65, 127, 129, 255, 256, 257, 700])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_row_counts(gpu, n, dtype):
    check(gpu, *problem(n, 136, 1003, dtype, n))


@pytest.mark.parametrize("k", [8, 16, 56, 64, 72, 128, 200, 640, 2560])
@pytest.mark.parametrize("n", [5, 150, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_widths(gpu, k, n, dtype):
    check(gpu, *problem(n, k, 777, dtype, k))


@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 255, 256, 257, 8192, 65537])
@pytest.mark.parametrize("n", [3, 60, 260])
def test_vocabularies(gpu, vocab, n):
    check(gpu, *problem(n, 64, vocab, torch.bfloat16, vocab + n))


@pytest.mark.parametrize("softcap,temperature", [(30.0, 1.0), (None, 0.5), (8.0, 1.7)])
@pytest.mark.parametrize("n", [9, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_softcap_and_temperature(gpu, softcap, temperature, n, dtype):
    check(gpu, *problem(n, 128, 5000, dtype, n, scale=10.0), softcap, temperature)


@pytest.mark.parametrize("n", [4, 520])
def test_full_vocabulary(gpu, n):
    # 262208 x 256 against the form on fp32 logits, itself held to the oracle elsewhere: each within its tolerance
    e, c, t = (x.to(gpu) for x in problem(n, 256, 262208, torch.bfloat16, n))
    logp, entropy = linear_token_logprobs(e, c, t)
    want = token_logprobs(e.float() @ c.float().t(), t)
    assert float((logp - want.logp).abs().max()) <= 1e-4 and float((entropy - want.entropy).abs().max()) <= 2e-3


def test_beyond_32_bits_of_offset(gpu):
    # a classifier of 4.9 GB: log-probabilities of its last entries against a product taken a slice at a time
    vocab, k, n = 300_000, 8192, 40
    c = torch.zeros(vocab, k, dtype=torch.bfloat16, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(0)
    for r in range(0, vocab, 50_000):
        c[r:r + 50_000] = torch.randn(50_000, k, generator=g, device=gpu) * (3 / k ** 0.5)
    e = torch.randn(n, k, generator=g, device=gpu).bfloat16()
    t = torch.arange(vocab - n, vocab, device=gpu)
    logp, entropy = linear_token_logprobs(e, c, t)
    x = torch.cat([e.float() @ c[r:r + 50_000].float().t() for r in range(0, vocab, 50_000)], 1)
    want = torch.log_softmax(x.double(), 1)
    assert float((logp - want[torch.arange(n), t]).abs().max()) <= 1e-4
    assert float((entropy + (want.exp() * want).sum(1)).abs().max()) <= 1e-3


def test_every_target_is_found(gpu):
    # all vocabulary entries as targets once: logp is the log-softmax row by row
    vocab, k = 1111, 64
    e, c, _ = problem(vocab, k, vocab, torch.float32, 1)
    e[:] = e[0]
    logp, _ = linear_token_logprobs(e.to(gpu), c.to(gpu), torch.arange(vocab, device=gpu))
    want = torch.log_softmax(e[0].double() @ c.double().t(), 0)
    assert float((logp.cpu().double() - want).abs().max()) <= 1e-4


def test_strided_hidden_states_and_classifier(gpu):
    e, c, t = problem(40, 64, 500, torch.bfloat16, 2)
    big_e, big_c = torch.randn(40, 200).bfloat16(), torch.randn(500, 72).bfloat16()
    big_e[:, 8:72], big_c[:, :64] = e, c
    want = linear_token_logprobs(e.to(gpu), c.to(gpu), t.to(gpu))
    got = linear_token_logprobs(big_e.to(gpu)[:, 8:72], big_c.to(gpu)[:, :64], t.to(gpu))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd_e = torch.zeros(40, 67).bfloat16()                    # rows that do not start on 16 bytes: copied
    odd_e[:, 1:65] = e
    got = linear_token_logprobs(odd_e.to(gpu)[:, 1:65], c.to(gpu), t.to(gpu))
    assert torch.equal(got[0], want[0])
    flat = torch.zeros(40 * 64 + 1).bfloat16()
    flat[1:] = e.reshape(-1)
    got = linear_token_logprobs(flat.to(gpu)[1:].view(40, 64), c.t().contiguous().to(gpu).t(), t.to(gpu))
    assert torch.equal(got[0], want[0])
    three = linear_token_logprobs(e.to(gpu).view(5, 8, 64), c.to(gpu), t.to(gpu).view(5, 8))
    assert three[0].shape == (5, 8) and torch.equal(three[0].view(-1), want[0])


def test_overflowing_hidden_states(gpu):
    e, c, t = problem(70, 64, 300, torch.float32, 3, ignore=0.0)
    e[5] = float("nan")
    e[6, 0] = float("inf")
    logp, entropy = linear_token_logprobs(e.to(gpu), c.to(gpu), t.to(gpu))
    ok = torch.ones(70, dtype=torch.bool)
    ok[5:7] = False
    assert torch.isfinite(logp[ok.to(gpu)]).all() and torch.isnan(logp[~ok.to(gpu)]).all() and torch.isnan(entropy[~ok.to(gpu)]).all()


@pytest.mark.parametrize("shape", [(7, 64, 100, None), (300, 136, 1003, None), (300, 136, 1003, 128), (70, 72, 5001, 33), (513, 64, 2050, None)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("softcap,temperature", [(None, 1.0), (10.0, 0.7)])
def test_gradients(gpu, shape, dtype, softcap, temperature):
    n, k, vocab, chunk = shape
    e, c, t = problem(n, k, vocab, dtype, n)
    g = torch.Generator().manual_seed(8)
    a, b = torch.randn(n, generator=g), torch.randn(n, generator=g)
    eg, cg = e.to(gpu).requires_grad_(), c.to(gpu).requires_grad_()
    out = linear_token_logprobs(eg, cg, t.to(gpu), softcap=softcap, temperature=temperature, chunk_rows=chunk)
    de, dc = torch.autograd.grad(out, (eg, cg), (a.to(gpu), b.to(gpu)))
    x = (e.double() @ c.double().t()).numpy()
    d = torch.from_numpy(O.rows(x, t.numpy(), softcap=softcap, temperature=temperature, dlogp=a.numpy(), dentropy=b.numpy())["dx"])
    tol = 2 * 2.0 ** -8 if dtype == torch.bfloat16 else 1e-5
    for got, want in ((de, d @ c.double()), (dc, d.t() @ e.double())):
        assert got.dtype == dtype
        assert float((got.double().cpu() - want).norm() / want.norm()) <= tol
    assert torch.all(de[t.to(gpu) == -100] == 0)


def test_gradient_against_differences(gpu):
    e, c, t = problem(6, 16, 50, torch.float32, 12, ignore=0.0)
    eg, cg = e.to(gpu).requires_grad_(), c.to(gpu).requires_grad_()
    logp, entropy = linear_token_logprobs(eg, cg, t.to(gpu), temperature=0.9)
    g = torch.Generator().manual_seed(1)
    ve, vc, h = torch.randn(6, 16, generator=g, dtype=torch.float64), torch.randn(50, 16, generator=g, dtype=torch.float64), 1e-5
    ends = [O.rows(((e.double() + s * h * ve) @ (c.double() + s * h * vc).t()).numpy(), t.numpy(), temperature=0.9) for s in (1, -1)]
    for name, y in (("logp", logp), ("entropy", entropy)):
        de, dc = torch.autograd.grad(y.sum(), (eg, cg), retain_graph=True)
        got = float((de.double().cpu() * ve).sum() + (dc.double().cpu() * vc).sum())
        want = float((ends[0][name] - ends[1][name]).sum() / (2 * h))
        assert abs(got - want) <= 1e-4 * max(1.0, abs(want)), name


def test_single_outputs_and_inputs(gpu):
    e, c, t = problem(40, 64, 300, torch.float32, 4)
    eg, cg = e.to(gpu).requires_grad_(), c.to(gpu).requires_grad_()
    logp, entropy = linear_token_logprobs(eg, cg, t.to(gpu))
    de, dc = torch.autograd.grad(logp.sum() + entropy.sum(), (eg, cg), retain_graph=True)
    one, = torch.autograd.grad(logp.sum(), eg, retain_graph=True)
    two, = torch.autograd.grad(entropy.sum(), eg)
    assert float((one + two - de).norm()) <= 1e-5 * float(de.norm()) + 1e-6
    frozen = linear_token_logprobs(eg, c.to(gpu), t.to(gpu))[0]
    only, = torch.autograd.grad(frozen.sum(), eg)
    assert torch.equal(only, one) and dc.shape == c.shape
    leaf = torch.empty(0, 64, device=gpu, requires_grad=True)
    cl = c.to(gpu).requires_grad_()
    linear_token_logprobs(leaf, cl, torch.empty(0, dtype=torch.long, device=gpu))[0].sum().backward()
    assert leaf.grad.shape == (0, 64) and torch.all(cl.grad == 0)


def test_same_bits_every_time_other_stream_and_graph(gpu):
    e, c, t = (x.to(gpu) for x in problem(300, 200, 5003, torch.bfloat16, 5))
    leaf = e.clone().requires_grad_()

    def step():
        logp, entropy = linear_token_logprobs(leaf, c, t)
        de, = torch.autograd.grad(logp.sum() + entropy.sum(), leaf)
        return logp.detach(), entropy.detach(), de

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            leaf.copy_(e * (1 + i))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager)), i


@pytest.mark.parametrize("n,ignore", [(256, 0.5), (257, 0.5), (900, 0.9), (400, 1.0), (300, 0.0)])
def test_dropped_rows_change_nothing(gpu, n, ignore, monkeypatch):
    from maester_amd import linear_logprobs
    monkeypatch.setitem(linear_logprobs._FILTER_WORK, torch.bfloat16, 0)   # also where it would not pay
    e, c, t = problem(n, 64, 1003, torch.bfloat16, n, ignore=ignore)
    t[0] = -100 if ignore == 1.0 else 5
    if n == 900:
        t[7], t[9] = 1003, -3                                 # out of the vocabulary: dropped as well
    a = torch.randn(n, device=gpu)
    out = []
    for flag in (True, False):
        eg, cg = e.to(gpu).requires_grad_(), c.to(gpu).requires_grad_()
        logp, entropy = linear_token_logprobs(eg, cg, t.to(gpu), filter_ignored=flag)
        de, dc = torch.autograd.grad((logp * a + entropy).sum(), (eg, cg))
        with torch.no_grad():
            again = linear_token_logprobs(eg, cg, t.to(gpu), filter_ignored=flag)
        assert torch.equal(again[0], logp) and torch.equal(again[1], entropy)
        out.append((logp, entropy, de, dc))
    # a row's own results do not depend on the others up to the order in which the vocabulary's parts are joined; dc sums
    # the same terms in another order of rows
    assert float((out[0][0] - out[1][0]).abs().max()) <= 1e-4 and float((out[0][1] - out[1][1]).abs().max()) <= 1e-3
    for x, y in zip(out[0][2:], out[1][2:]):
        assert float((x.float() - y.float()).norm()) <= 2 * 2.0 ** -8 * float(y.float().norm()) + 1e-6
    dead = (t == -100).to(gpu)
    assert torch.all(out[0][0][dead] == 0) and torch.all(out[0][2][dead] == 0)


def test_refusals(gpu):
    e, c, t = (x.to(gpu) for x in problem(4, 64, 30, torch.bfloat16, 6))
    for args, kw in [((e[:, :60], c[:, :60], t), {}), ((e, c.float(), t), {}), ((e, c[:, :32], t), {}), ((e, c, t[:3]), {}), ((e, c, t.int()), {}),
                     ((e, c, t.cpu()), {}), ((e, c, t), dict(temperature=0.0)), ((e, c, t), dict(softcap=-2.0)), ((e.half(), c.half(), t), {}),
                     ((e, c[:0], t), {})]:
        with pytest.raises(ValueError):
            linear_token_logprobs(*args, **kw)
    with pytest.raises(RuntimeError):
        linear_token_logprobs(e.cpu(), c.cpu(), t.cpu())


def test_infinities_in_fp32(gpu):
    """An infinity makes NaN of the tokens whose logits it takes part in, and of no others."""
    e, c = torch.randn(5, 64, device=gpu), torch.randn(300, 64, device=gpu)
    t = torch.arange(5, device=gpu)
    want = linear_token_logprobs(e, c, t)
    for sign in (1.0, -1.0):
        bad = e.clone()
        bad[2, 7] = sign * float("inf")
        for got, ref in zip(linear_token_logprobs(bad, c, t), want):
            assert bool(torch.isnan(got[2])) and torch.equal(got[[0, 1, 3, 4]], ref[[0, 1, 3, 4]])
        bad = c.clone()
        bad[299, 0] = sign * float("inf")
        assert all(bool(torch.isnan(x).all()) for x in linear_token_logprobs(e, bad, t))


def test_fp32_operands_of_any_size(gpu):
    """24 bits of both operands over 60 binades: against 64 bits of the same values, as the fp32 sum of K products."""
    torch.manual_seed(5)
    n, k, v = 70, 132, 515
    up = torch.exp2(torch.randint(-30, 30, (k,)).float())
    e, c = (torch.randn(n, k) * up).to(gpu), (torch.randn(v, k) / up).to(gpu)
    t = torch.randint(0, v, (n,), device=gpu)
    logp, entropy = linear_token_logprobs(e, c, t)
    x = e.double() @ c.double().t()
    size = e.double().abs() @ c.double().abs().t()
    lse = torch.logsumexp(x, 1)
    # a logit is off by at most (K + 3) 2^-24 of the sum of its products' sizes, the statistics by some 40 roundings of theirs
    off = ((k + 3) * 2.0 ** -24 * size).amax(1) * 2 + 40 * 2.0 ** -24 * (x.abs().amax(1) + 10)
    assert bool(((logp.double() - (x.gather(1, t[:, None])[:, 0] - lse)).abs() <= off).all())
