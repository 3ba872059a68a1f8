"""fp32 products through the bf16 matrix instructions: how much of a single product is lost.

A product x y is formed from three parts each, x = h + m + l with |m| <= 2^-8 |x| and |l| <= 2^-16 |x| (rounded to the nearest of
8 bits), without m l + l m + l l: 2 * 2^-24 + 2^-32 of it.  Here a second term of the contraction takes h_x h_y away again, whose
factors are bf16 values and have one part each.  What is left of the sum is 2^-7 of the product at most, so that only the first
of three instructions, which sums h h + m m - h h, works on numbers as large as the product: a whole last place of its largest
term at most, 2^-23, whichever way it rounds; the other two add terms of 2^-7 (1 + 2^-7) and less, four roundings of such sums,
4 * 2^-23 * 2^-7 < 2^-28.  Together 2^-23 + 2^-32 + 2^-23 + 2^-28 < 4.2 * 2^-24 of the product.  (Parts cut off instead of rounded
leave out 7.8 * 2^-24 of the worst pair's.)"""
import pytest
import torch

from maester_amd import linear_logprobs as LL

pytestmark = pytest.mark.gpu
BOUND = 4.2 * 2.0 ** -24


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
        assert float(((got.double().cpu() - want) / whole).abs().max()) <= BOUND


def test_the_largest_values():
    # magnitudes that bf16 still holds are exact, larger ones count as infinities
    top = torch.finfo(torch.bfloat16).max
    x = torch.zeros(3, 8, device="cuda")
    x[:, 0] = torch.tensor([1.0, -2.0 ** -40, 2.0 ** -120])
    c = torch.tensor([[top, -top, torch.finfo(torch.float32).max, 2.0 ** 127 * 1.25]], device="cuda")
    de = torch.empty(3, 4, device="cuda")
    LL._products(x, torch.zeros(3, 4, device="cuda"), c, de, None, False)
    want = x[:, :1].double() * c.double()
    keep = torch.tensor([0, 1, 3], device="cuda")
    assert torch.equal(de[:, keep].double(), want[:, keep]) and bool(torch.isnan(de[:, 2]).all())
