"""Argument checks of the log-probability entry points, before any launch (no GPU), and the oracle's own pins."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from maester_amd import _lib, token_logprobs
from oracle import token_logprobs as O

P = 0x1000
NAN = float("nan")


def _fwd(logits=P, pitch=100, targets=P, rows=4, vocab=100, cap=0.0, temp=1.0, k=0, logp=P, ent=P, ids=P, top=P, ws=P, ws_bytes=1 << 20, dtype=1):
    return _lib.lib().ma_token_logprobs_fwd(logits, pitch, targets, rows, vocab, -100, cap, temp, k, logp, ent, None, ids, top, ws, ws_bytes, dtype, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(logits=None), -1, "NULL"), (dict(targets=None), -1, "NULL"), (dict(logp=None), -1, "logp"), (dict(rows=0), -1, "rows"),
    (dict(rows=1 << 23), -2, "rows"), (dict(vocab=0), -1, "vocab"), (dict(vocab=1 << 30, pitch=1 << 31), -1, "vocab"),
    (dict(pitch=99), -1, "pitch"), (dict(cap=-1.0), -1, "softcap"), (dict(cap=NAN), -1, "softcap"), (dict(temp=0.0), -1, "temperature"),
    (dict(temp=NAN), -1, "temperature"), (dict(k=65), -1, "top_k"), (dict(k=-1), -1, "top_k"), (dict(k=6, vocab=5), -1, "top_k"),
    (dict(k=2, ids=None), -1, "top_ids"), (dict(vocab=50000, pitch=50000, ws=None), -1, "workspace"),
    (dict(vocab=50000, pitch=50000, ws_bytes=8), -1, "workspace"), (dict(vocab=50000, pitch=50000, ws=P + 8), -1, "aligned"), (dict(dtype=7), -1, "dtype"), (dict(logits=P + 1), -1, "aligned")])
def test_forward_refusals(kw, code, text):
    assert _fwd(**kw) == code and text in _lib.lib().ma_last_error().decode()


def _bwd(logits=P, pitch=100, rows=4, vocab=100, stats=P, ent=P, dx=P, dpitch=100, dtype=0):
    return _lib.lib().ma_token_logprobs_bwd(logits, pitch, P, rows, vocab, -100, 0.0, 1.0, stats, ent, P, P, dx, dpitch, dtype, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(logits=None), -1, "NULL"), (dict(stats=None), -1, "stats"), (dict(dx=None), -1, "dlogits"), (dict(dpitch=99), -1, "dpitch"),
    (dict(dx=P + 2), -1, "aligned"), (dict(rows=1 << 20, vocab=262208, pitch=262208, dpitch=262208), -2, "grid")])
def test_backward_refusals(kw, code, text):
    assert _bwd(**kw) == code and text in _lib.lib().ma_last_error().decode()


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError):
        token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.long))
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(2, 5), torch.zeros(3, dtype=torch.long))


@pytest.mark.parametrize("softcap,temperature", [(None, 1.0), (4.0, 0.6)])
def test_oracle_against_torch(softcap, temperature):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(7, 31, generator=g, dtype=torch.float64).requires_grad_()
    t = torch.randint(0, 31, (7,), generator=g)
    t[2] = -100
    a, b = torch.randn(7, generator=g, dtype=torch.float64), torch.randn(7, generator=g, dtype=torch.float64)
    y = (softcap * torch.tanh(x / softcap) if softcap else x) / temperature
    logp = -F.cross_entropy(y, t, ignore_index=-100, reduction="none")
    entropy = torch.distributions.Categorical(logits=y).entropy() * (t != -100)
    dx, = torch.autograd.grad((logp * a).sum() + (entropy * b).sum(), x)
    out = O.rows(x.detach().numpy(), t.numpy(), 5, softcap=softcap, temperature=temperature, dlogp=a.numpy(), dentropy=b.numpy())
    assert np.allclose(out["logp"], logp.detach().numpy(), atol=1e-12) and np.allclose(out["entropy"], entropy.detach().numpy(), atol=1e-12)
    assert np.allclose(out["dx"], dx.numpy(), atol=1e-12)
    assert np.array_equal(out["top_ids"], torch.sort(x.detach(), dim=1, descending=True, stable=True).indices[:, :5].numpy())


def _lin(e=P, es=64, c=P, cs=64, targets=P, rows=4, vocab=100, dim=64, cap=0.0, temp=1.0, logp=P, stats=P, ws=P, ws_bytes=1 << 20, dtype=1):
    return _lib.lib().ma_linear_logprobs_fwd(e, es, c, cs, targets, rows, vocab, dim, -100, cap, temp, logp, P, stats, ws, ws_bytes, dtype, None)


LINEAR = [(dict(e=None), -1, "NULL"), (dict(c=P + 8), -1, "aligned"), (dict(rows=0), -1, "rows"), (dict(rows=(1 << 26) + 1), -1, "rows"),
          (dict(vocab=0), -1, "vocab"), (dict(dim=60), -2, "dim"), (dict(dim=65544, es=65544, cs=65544), -2, "dim"), (dict(es=56), -1, "strides"),
          (dict(cs=68), -1, "strides"), (dict(es=(1 << 20) + 8), -2, "strides"), (dict(cap=-1.0), -1, "softcap"), (dict(temp=NAN), -1, "temperature"),
          (dict(dtype=3), -1, "dtype")]


@pytest.mark.parametrize("kw,code,text", LINEAR + [(dict(logp=None), -1, "logp"), (dict(stats=P + 4), -1, "stats"), (dict(ws=None), -1, "workspace"),
                                                   (dict(ws_bytes=20), -1, "workspace"), (dict(ws=P + 8), -1, "aligned")])
def test_linear_forward_refusals(kw, code, text):
    assert _lin(**kw) == code and text in _lib.lib().ma_last_error().decode()


def _dlogits(e=P, es=64, c=P, cs=64, targets=P, rows=4, vocab=100, dim=64, cap=0.0, temp=1.0, stats=P, out=P, pitch=104, parts=1, dtype=1):
    return _lib.lib().ma_linear_logprobs_dlogits(e, es, c, cs, targets, rows, vocab, dim, -100, cap, temp, stats, P, P, P, out, pitch, parts, dtype, None)


@pytest.mark.parametrize("kw,code,text", LINEAR + [(dict(stats=None), -1, "stats"), (dict(out=P + 8), -1, "aligned"), (dict(pitch=100), -1, "pitch"),
                                                   (dict(pitch=96), -1, "pitch"), (dict(parts=0), -1, "parts"), (dict(parts=3), -1, "parts"),
                                                   (dict(parts=2, rows=65), -1, "parts"), (dict(parts=2, dtype=0), -1, "parts")])
def test_linear_gradient_refusals(kw, code, text):
    assert _dlogits(**kw) == code and text in _lib.lib().ma_last_error().decode()


def test_linear_workspace():
    L = _lib.lib()
    assert L.ma_linear_logprobs_workspace_bytes(0, 100) == 0
    assert L.ma_linear_logprobs_workspace_bytes(5, 600) == 32 + 3 * 5 * 12          # targets' logits, three ranges' statistics
    assert L.ma_linear_logprobs_workspace_bytes(8, 262208) == 32 + 256 * 8 * 12


def _grads(x=P, xs=304, e=P, es=64, c=P, cs=64, rows=9, vocab=300, dim=64, parts=1, de=P, dc=P, add=0, ws=P, ws_bytes=1 << 20, dtype=1):
    return _lib.lib().ma_linear_grads(x, xs, e, es, c, cs, rows, vocab, dim, parts, de, dc, add, ws, ws_bytes, dtype, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(x=None), -1, "NULL"), (dict(c=None), -1, "NULL"), (dict(e=None), -1, "NULL"), (dict(de=None, dc=None), -1, "both outputs"),
    (dict(x=P + 8), -1, "aligned"), (dict(dc=P + 8), -1, "aligned"), (dict(rows=0), -1, "rows"), (dict(vocab=0), -1, "vocab"),
    (dict(dim=60, es=64, cs=64), -2, "dim"), (dict(dim=1 << 17, es=1 << 17, cs=1 << 17), -2, "dim"), (dict(xs=300), -1, "strides"),
    (dict(xs=296), -1, "strides"), (dict(es=56), -1, "strides"), (dict(cs=68), -1, "strides"), (dict(xs=(1 << 21) + 8), -2, "2^21"),
    (dict(vocab=1 << 22, xs=1 << 22), -2, "2^21"), (dict(es=(1 << 20) + 8), -2, "2^20"), (dict(dtype=7), -1, "dtype"),
    (dict(parts=0), -1, "parts"), (dict(parts=2), -1, "parts"), (dict(rows=18, parts=9), -1, "parts"),
    (dict(rows=8, vocab=64, parts=2, ws=None), -1, "workspace"), (dict(vocab=40000, xs=40000, ws=None), -1, "workspace"), (dict(vocab=40000, xs=40000, ws_bytes=16), -1, "workspace"),
    (dict(vocab=40000, xs=40000, ws=P + 8), -1, "workspace")])
def test_gradient_products_refuse(kw, code, text):
    assert _grads(**kw) == code and text in _lib.lib().ma_last_error().decode()


def test_workspace_of_the_gradient_products():
    L = _lib.lib()
    assert L.ma_linear_grads_workspace_bytes(0, 100, 64, 1, 1) == 0 and L.ma_linear_grads_workspace_bytes(9, 64, 64, 1, 1) == 0
    assert L.ma_linear_grads_workspace_bytes(10, 64, 64, 2, 1) == 10 * 64 * 4
    for rows, vocab, dim, dtype in ((9, 40000, 64, 1), (2047, 262208, 2560, 1), (210, 32003, 640, 0), (1 << 20, 32003, 640, 1)):
        need = L.ma_linear_grads_workspace_bytes(rows, vocab, dim, 1, dtype)
        assert need % (rows * dim * 4) == 0 and need // (rows * dim * 4) <= 128
