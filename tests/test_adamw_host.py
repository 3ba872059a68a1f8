"""Argument checks of the AdamW entry points before any launch (no GPU), and the oracle's own pins."""
import ctypes

import numpy as np
import pytest
import torch

from maester_amd import Blocks8, _lib, adamw_step
from oracle import adamw as O

P = 0x10000


def _table(tensors=1, **kw):
    t = (_lib.MaAdamwTensor * tensors)()
    for row in t:
        for k in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
            setattr(row, k, P)
        row.n, row.param_dtype, row.grad_dtype = 100, 0, 0
        for k, v in kw.items():
            setattr(row, k, v)
    return t


def _step(table=None, count=1, bits=32, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, max_norm=-1.0, step=P, ws=P, ws_bytes=1 << 20, **kw):
    table = _table(**kw) if table is None else table
    return _lib.lib().ma_adamw_step(table, count, bits, lr, None, b1, b2, eps, wd, max_norm, None, None, step, 0, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(bits=16), -1, "state_bits"), (dict(count=-1), -1, "count"), (dict(b1=1.0), -1, "betas"), (dict(b2=float("nan")), -1, "betas"),
    (dict(lr=-1.0), -1, "lr"), (dict(eps=-1.0), -1, "eps"), (dict(wd=-1.0), -1, "weight_decay"), (dict(max_norm=float("nan")), -1, "max_norm"),
    (dict(step=None), -1, "step"), (dict(step=P + 4), -1, "step"), (dict(ws=None), -1, "workspace"), (dict(ws_bytes=16), -1, "workspace"),
    (dict(ws=P + 8), -1, "aligned"), (dict(n=-1), -1, "n=-1"), (dict(n=(1 << 34) + 1), -2, "2^34"), (dict(param=None), -1, "param"),
    (dict(grad=None), -1, "grad"), (dict(exp_avg_sq=None), -1, "exp_avg_sq"), (dict(bits=8, exp_avg_scale=None), -1, "scales"),
    (dict(param_dtype=5), -1, "dtype"), (dict(grad_dtype=5), -1, "dtype"), (dict(master=P), -1, "master"),
    (dict(param=P + 2), -1, "aligned"), (dict(grad=P + 2), -1, "aligned"), (dict(exp_avg=P + 1), -1, "aligned"),
    (dict(param_dtype=1, param=P + 1), -1, "aligned"), (dict(bits=8, exp_avg_scale=P + 2), -1, "aligned")])
def test_refusals(kw, code, text):
    assert _step(**kw) == code and text in _lib.lib().ma_last_error().decode()


def test_too_many_elements_and_norm_refusals():
    L = _lib.lib()
    assert _step(table=_table(9, n=1 << 34), count=9) == -2 and "2^37" in L.ma_last_error().decode()
    assert L.ma_grad_norm(_table(), 1, -1.0, None, None, P, 1 << 20, None) == -1 and "outputs" in L.ma_last_error().decode()
    assert L.ma_adamw_workspace_bytes(-1) == 0 and L.ma_adamw_workspace_bytes(1) < L.ma_adamw_workspace_bytes(1000)
    assert ctypes.sizeof(_lib.MaAdamwTensor) == 80


def test_cpu_tensors_are_refused():
    p = torch.zeros(4)
    with pytest.raises(RuntimeError):
        adamw_step([p], [p], [p.clone()], [p.clone()], torch.zeros((), dtype=torch.int64))


def test_oracle_codes_are_torchs_float8():
    codes = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(codes.copy()).view(torch.float8_e4m3fn).float().numpy()
    fine = np.isfinite(want)
    assert np.array_equal(O.value_of(codes)[fine], want[fine])


def test_oracle_rounds_between_neighbours_with_the_right_weight():
    g = np.random.default_rng(0)
    x = np.abs(g.standard_normal(128 * 50)).astype(np.float32) * np.exp(g.uniform(-9, 0, 128 * 50)).astype(np.float32)
    for sign in (1, -1):
        low, s0 = O.pack(sign * x, np.zeros(len(x), np.int64), False)
        high, s1 = O.pack(sign * x, np.full(len(x), (1 << 20) - 1), False)
        assert np.array_equal(s0, s1) and np.array_equal(np.log2(s0), np.round(np.log2(s0)))
        a, b = np.abs(O.spread(low, s0)), np.abs(O.spread(high, s0))
        assert np.all(a <= x) and np.all((x <= b) | (x < 2.0 ** -29)) and np.all(high.astype(int) - low.astype(int) <= 1)
        total = np.zeros(len(x))
        for r in range(64):
            c, _ = O.pack(sign * x, np.full(len(x), (2 * r + 1) << 13), False)
            total += np.abs(O.spread(c, s0))
        assert np.all(np.abs(total / 64 - x) <= (b - a) / 64 + 1e-12)
    blocks = x.reshape(-1, 128).max(1) / s0
    assert np.all(blocks <= 448) and np.all(blocks > 224)


@pytest.mark.parametrize("wd", [0.0, 0.1])
def test_oracle_against_torchs_optimizer(wd):
    g = torch.Generator().manual_seed(0)
    p = torch.randn(500, generator=g).requires_grad_()
    opt = torch.optim.AdamW([p], lr=1e-2, betas=(0.8, 0.95), eps=1e-6, weight_decay=wd, foreach=False)
    q, m, v = p.detach().numpy().copy(), np.zeros(500, np.float32), np.zeros(500, np.float32)
    for t in range(1, 5):
        p.grad = torch.randn(500, generator=g)
        q, m, v = O.step(q, p.grad.numpy(), m, v, t, lr=1e-2, betas=(0.8, 0.95), eps=1e-6, weight_decay=wd)
        opt.step()
        assert np.abs(q - p.detach().numpy()).max() <= t * 1e-6


def test_hash_bits_look_random():
    h = O.mix((np.arange(1 << 18, dtype=np.int64) * 0x9E3779B9 & 0xFFFFFFFF).astype(np.uint32)).astype(np.int64)
    for u in ((h & 0xFFFF) / 65536, (h >> 16) / 65536):
        assert abs(u.mean() - 0.5) < 6 * (1 / 12) ** 0.5 / 512 and abs(u.std() - (1 / 12) ** 0.5) < 0.003
        assert abs(np.corrcoef(u[1:], u[:-1])[0, 1]) < 6 / 512
    assert abs(np.corrcoef(h & 0xFFFF, h >> 16)[0, 1]) < 6 / 512


def test_blocks8_values():
    b = Blocks8.zeros_like(torch.zeros(3, 100))
    assert b.codes.shape == (3, 100) and b.scales.shape == (3,) and torch.all(b.float() == 0)
    b.scales[2] = 4.0
    b.codes.view(-1).view(torch.uint8)[256:] = 0x38          # 1.0
    assert torch.all(b.float().view(-1)[256:] == 4.0) and torch.all(b.float().view(-1)[:256] == 0)


def test_buffers_that_share_memory_are_refused():
    L = _lib.lib()

    def table(**moved):
        t = (_lib.MaAdamwTensor * 2)()
        for i, row in enumerate(t):
            for j, k in enumerate(("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")):
                setattr(row, k, P + 0x100000 * (i + 1) + 400 * j)
            row.n, row.param_dtype, row.grad_dtype = 100, 0, 0
        for k, v in moved.items():
            setattr(t[1], k, v)
        return t

    first = table()[0]
    for bits, moved in [(32, dict(param=first.param)), (32, dict(param=first.param + 396)), (32, dict(exp_avg=first.exp_avg_sq - 396)),
                        (32, dict(grad=first.param + 4)), (32, dict(param=first.grad - 200)), (32, dict(exp_avg=first.grad + 399 // 4 * 4)),
                        (8, dict(exp_avg_scale=first.exp_avg_sq_scale)), (8, dict(exp_avg=first.exp_avg + 99)),
                        (32, dict(param_dtype=1, master=first.exp_avg))]:
        assert _step(table=table(**moved), count=2, bits=bits) == -1, moved
        assert "overlaps" in L.ma_last_error().decode(), moved
