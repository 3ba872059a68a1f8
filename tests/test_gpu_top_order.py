"""The order of equal alternatives: -0 and +0 are one value, by ascending index like any other tie."""
import numpy as np
import pytest
import torch

from maester_amd import token_logprobs
from oracle import token_logprobs as O

pytestmark = pytest.mark.gpu


def _zeros(*shape, generator):
    return torch.where(torch.rand(*shape, generator=generator) < 0.5, -0.0, 0.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_three_logits(gpu, dtype):
    x = torch.tensor([[-0.0, 0.0, -1.0], [0.0, -0.0, -1.0], [-1.0, -0.0, 0.0]], dtype=dtype, device=gpu)
    for k in (1, 2, 3):
        got = token_logprobs(x, torch.zeros(3, dtype=torch.long, device=gpu), top_k=k).top_ids.cpu()
        assert torch.equal(got, torch.tensor([[0, 1, 2], [0, 1, 2], [1, 2, 0]])[:, :k]), k


# rows cut into parts (few rows), whole rows (600 of them), a vocabulary within one group of a thread and many groups each
@pytest.mark.parametrize("rows,vocab", [(1, 262208), (5, 40001), (40, 9001), (600, 9001), (600, 50), (7, 4097)])
@pytest.mark.parametrize("k", [1, 5, 50])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_zeros_of_both_signs_tie(gpu, rows, vocab, k, dtype):
    g = torch.Generator().manual_seed(rows + vocab + k)
    x = -1 - torch.rand(rows, vocab, generator=g)
    some = torch.rand(rows, vocab, generator=g) < min(1.0, 3 * k / vocab)        # around the border of the k best
    x = torch.where(some, _zeros(rows, vocab, generator=g), x)
    x[0] = _zeros(vocab, generator=g)                                             # a row of nothing else
    if rows > 2:
        x[1, :] = -0.0
        x[1, vocab // 2] = 0.0
        x[2, ::2] = _zeros(len(x[2, ::2]), generator=g)
        x[2, 7] = 3.0
    x = x.to(dtype)
    got = token_logprobs(x.to(gpu), torch.zeros(rows, dtype=torch.long, device=gpu), top_k=k)
    assert np.array_equal(got.top_ids.cpu().numpy(), O.rows(x.float().numpy(), np.zeros(rows, np.int64), k)["top_ids"])


def test_a_thread_with_both_zeros(gpu):
    # one thread's groups are 4096 elements apart: -0 in an earlier one, +0 in a later, and the other way round
    x = torch.full((600, 20000), -2.0)
    x[::2, 16], x[::2, 16 + 4096], x[::2, 16 + 2 * 4096] = -0.0, 0.0, -0.0
    x[1::2, 24], x[1::2, 24 + 4096] = 0.0, -0.0
    x[:, 19999] = -0.0
    for dtype in (torch.bfloat16, torch.float32):
        got = token_logprobs(x.to(gpu, dtype), torch.zeros(600, dtype=torch.long, device=gpu), top_k=3).top_ids.cpu()
        assert torch.equal(got[::2], torch.tensor([16, 16 + 4096, 16 + 2 * 4096]).expand(300, 3))
        assert torch.equal(got[1::2], torch.tensor([24, 24 + 4096, 19999]).expand(300, 3))
