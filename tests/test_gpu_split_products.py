"""fp32 products through the bf16 matrix instructions: how much of a single product is lost.

A product x y is formed from three parts each, x = h + m + l with |m| <= 2^-7 |x| (what 8 bits cut off leave) and
|l| <= 2^-16 |x| (of either sign: m is rounded), without m l + l m + l l: 2 * 2^-23 + 2^-32 of it at most, and 0 on average.
Here a second term of the contraction takes h'_x h'_y away again (x and y rounded to bf16, which have one part each).  What is
left of the sum is 2^-6 of the product at most, so that only the first of three instructions, which sums h h + m m - h' h',
works on numbers as large as the product: a whole last place of its largest term at most, 2^-23, whichever way it rounds, and
half of that on average; the other two add terms of 2^-6 and less, four roundings of such sums, 4 * 2^-23 * 2^-6 = 2^-27.  Together
2 * 2^-23 + 2^-32 + 2^-23 + 2^-27 < 6.2 * 2^-24 of the product, and 2^-24 of it on average over pairs of one sign.  (With m cut off
7.8 * 2^-24 of the worst pair are left out, beside those roundings.)"""
import pytest
import torch

from maester_amd import linear_logprobs as LL
from maester_amd import linear_token_logprobs

pytestmark = pytest.mark.gpu
BOUND, MEAN = 6.2 * 2.0 ** -24, 2.0 ** -24


def _values(count, seed):
    """Mantissas whose lower parts are as large as they get, cut off or rounded, and random ones; of one sign."""
    g = torch.Generator().manual_seed(seed)
    worst = torch.tensor([1 + 2.0 ** -7 - 2.0 ** -23, 1 + 2.0 ** -8 - 2.0 ** -23, 1 + 2.0 ** -8 + 2.0 ** -16, 1 + 2.0 ** -7 - 2.0 ** -16 - 2.0 ** -23,
                          2 - 2.0 ** -23, 1 + 2.0 ** -23, 1 + 2.0 ** -8 + 2.0 ** -17, 1.5], dtype=torch.float64)
    rest = 1 + torch.randint(0, 1 << 23, (count - len(worst),), generator=g).double() * 2.0 ** -23
    return torch.cat((worst, rest)).float()


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_single_products(sign, seed):
    # 512 x 512 pairs: de = x c over a vocabulary of two, dc = x^T e over two rows
    a, b = _values(512, seed), sign * _values(512, seed + 10)
    two_a, two_b = torch.stack((a, -a.bfloat16().float())), torch.stack((b, b.bfloat16().float()))
    x = torch.zeros(512, 8, device="cuda")
    x[:, :2] = two_a.t().cuda()
    de, dc = torch.empty(512, 512, device="cuda"), torch.empty(512, 512, device="cuda")
    LL._products(x, torch.zeros(512, 512, device="cuda"), two_b.cuda(), de, None, False)
    LL._products(two_a.cuda(), two_b.cuda(), torch.zeros(512, 512, device="cuda"), None, dc, False)
    whole = a.double()[:, None] * b.double()
    want = whole + two_a[1].double()[:, None] * two_b[1].double()
    for got in (de, dc):
        off = (got.double().cpu() - want) / whole
        assert float(off.abs().max()) <= BOUND and abs(float(off.mean())) <= MEAN


@pytest.mark.parametrize("start", [-1.0, 1.0])
def test_the_largest_values(start):
    # up to fp32's largest magnitudes, times powers of two: their 24 bits are the result; h + m of a product above
    # 2^128 (1 - 2^-17) may round up to 2^128 before l is added, so that it may overflow
    top = torch.finfo(torch.float32).max
    values = [top * (1 - n * 2.0 ** -24) for n in (0, 1, 2, 3, 2 ** 7, 2 ** 8, 2 ** 14, 2 ** 15 - 1, 2 ** 15, 2 ** 16, 2 ** 17 + 5)]
    c = start * torch.tensor([[*values, torch.finfo(torch.bfloat16).max, 2.0 ** 127 * 1.25, 2.0 ** 127]], device="cuda")
    c = torch.cat((c, torch.zeros(1, 2, device="cuda")), 1)
    x = torch.zeros(3, 8, device="cuda")
    x[:, 0] = torch.tensor([1.0, -2.0 ** -40, 2.0 ** -120])
    de, dc = torch.empty(3, 16, device="cuda"), torch.empty(3, 16, device="cuda")
    LL._products(x, torch.zeros(3, 16, device="cuda"), c, de, None, False)
    LL._products(torch.cat((x[:, :1].t(), torch.zeros(1, 1, device="cuda")), 1), c, torch.zeros(3, 16, device="cuda"), None, dc, False)
    want = (x[:, :1].double() * c.double()).float()
    for got in (de, dc):
        same = got == want
        assert bool((same | ((want.abs().double() > 2.0 ** 128 * (1 - 2.0 ** -17)) & (got == torch.sign(want) * float("inf")))).all())
        assert bool(same[1:].all())


def test_a_ban_by_the_lowest_value():
    # a column of ones in the hidden states and a column of 0 or the lowest value in the classifier
    n, k, vocab = 40, 64, 515
    e, c = torch.randn(n, k, device="cuda"), torch.randn(vocab, k, device="cuda")
    e[:, 7], c[:, 7] = 1.0, 0.0
    c[100:400, 7] = torch.finfo(torch.float32).min
    t = torch.randint(0, 100, (n,), device="cuda")
    e.requires_grad_()
    logp, entropy = linear_token_logprobs(e, c, t)
    want = torch.log_softmax(torch.cat((e.detach() @ c[:100].t(), e.detach() @ c[400:].t()), 1).double(), 1)
    assert float((logp - want.gather(1, t[:, None])[:, 0]).abs().max()) <= 1e-4
    assert float((entropy + (want.exp() * want).sum(1)).abs().max()) <= 1e-3
    logp.sum().backward()
    assert bool(torch.isfinite(e.grad).all())
