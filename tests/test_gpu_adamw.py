"""AdamW over many tensors against the oracle in IEEE single precision and against torch's.

The states are compared bit for bit: the kernels evaluate the formulas operation by operation in fp32, as the oracle does.
A parameter goes through p d - s (m / (r c + eps)) with at most one more rounding per operation on either side (six
operations, u = 2^-24 relative each, and s, c rounded from doubles of the same formula): 8 u (|p| + |update|), plus half a
step of its own type where it is stored in bf16 and the two sides straddle a rounding border (one step, 2^-8 relative)."""
import copy

import numpy as np
import pytest
import torch

from maester_amd import AdamW, Blocks8, adamw_step, global_grad_norm
from oracle import adamw as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
SIZES = [1, 7, 8, 9, 127, 128, 129, 1000, 2047, 2048, 2049, 4096, 5003, 0, 131]


def close(got, want, dtype):
    got, want = got.double().cpu().numpy(), want.astype(np.float64)
    lim = 8 * U * (np.abs(want) + 0.1) + (2.0 ** -8 * np.abs(want) if dtype == torch.bfloat16 else 0)
    return bool(np.all(np.abs(got - want) <= lim))


def bits(t):
    return t.view(torch.uint8).cpu().numpy().reshape(-1)


@pytest.mark.parametrize("pdt,gdt,master", [(torch.float32, torch.float32, False), (torch.float32, torch.bfloat16, False),
                                            (torch.bfloat16, torch.bfloat16, False), (torch.bfloat16, torch.float32, False),
                                            (torch.bfloat16, torch.bfloat16, True), (torch.bfloat16, torch.float32, True)])
@pytest.mark.parametrize("state_bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 3])
def test_steps_against_the_oracle(gpu, pdt, gdt, master, state_bits, offset):
    # every size a view of a larger buffer (offset 0: 16-byte aligned, 3: not), whose rest stays as it is
    g = torch.Generator().manual_seed(state_bits + offset)
    at, spans = 0, []
    for n in SIZES:
        spans.append((at + offset, n))
        at += -(-(n + offset) // 128) * 128 + 128

    def views(t):
        return [t[a:a + n] for a, n in spans]

    w0 = (0.1 * torch.randn(at, generator=g)).to(pdt)
    params, keep_p = w0.clone().to(gpu), w0.clone()
    masters = w0.float().to(gpu) if master else None
    if state_bits == 32:
        m, v = torch.zeros(at, device=gpu), torch.zeros(at, device=gpu)
        ms, vs = views(m), views(v)
    else:
        m, v = (torch.full((at,), 0, dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn) for _ in "mv")
        sm, sv = (torch.ones(at // 128 + 2 * len(SIZES), device=gpu) for _ in "mv")
        starts = np.cumsum([0] + [-(-n // 128) + 1 for n in SIZES])
        ms, vs = ([Blocks8(c, s[b:b + -(-n // 128)]) for c, b, n in zip(views(x), starts, SIZES)] for x, s in ((m, sm), (v, sv)))
    step = torch.zeros((), dtype=torch.int64, device=gpu)
    ref = [dict(p=w0[a:a + n].float().numpy(), m=np.zeros(n, np.float32 if state_bits == 32 else np.uint8),
                v=np.zeros(n, np.float32 if state_bits == 32 else np.uint8), s=(np.ones(-(-n // 128), np.float32),) * 2) for a, n in spans]
    for t in range(1, 4):
        grads = (1e-2 * torch.randn(at, generator=g)).to(gdt)
        if t == 2:
            grads[::5] = 0
        adamw_step(views(params), views(grads.to(gpu)), ms, vs, step, **HYPER, masters=views(masters) if master else None, seed=77)
        for i, ((a, n), r) in enumerate(zip(spans, ref)):
            gr = grads[a:a + n].float().numpy()
            if state_bits == 32:
                p, r["m"], r["v"] = O.step(r["p"], gr, r["m"], r["v"], t, i, **HYPER, seed=77)
                assert np.array_equal(ms[i].cpu().numpy(), r["m"]) and np.array_equal(vs[i].cpu().numpy(), r["v"]), (t, n)
            else:
                p, r["m"], r["v"], r["s"] = O.step(r["p"], gr, r["m"], r["v"], t, i, **HYPER, seed=77, scales=r["s"])
                assert np.array_equal(bits(ms[i].codes), r["m"]) and np.array_equal(bits(vs[i].codes), r["v"]), (t, n)
                assert np.array_equal(ms[i].scales.cpu().numpy(), r["s"][0]) and np.array_equal(vs[i].scales.cpu().numpy(), r["s"][1])
            got = views(params)[i]
            assert close(got, p, pdt), (t, n)
            if master:
                assert close(views(masters)[i], p, torch.float32) and torch.equal(got, views(masters)[i].bfloat16())
                r["p"] = views(masters)[i].cpu().numpy()       # continue from the same weights
            else:
                r["p"] = got.float().cpu().numpy()
    assert int(step) == 3
    inside = torch.zeros(at, dtype=torch.bool)
    for a, n in spans:
        inside[a:a + n] = True
    assert torch.equal(params.cpu()[~inside], keep_p[~inside])
    if state_bits == 8:
        assert not bits(m)[~inside.numpy()].any() and not bits(v)[~inside.numpy()].any()


def test_more_tensors_than_one_launch_takes(gpu):
    g = torch.Generator().manual_seed(0)
    ps = [torch.randn(1 + 37 * i % 700, generator=g) for i in range(131)]
    gs = [torch.randn(p.shape, generator=g) for p in ps]
    pg, gg = [p.to(gpu) for p in ps], [x.to(gpu) for x in gs]
    m = [Blocks8.zeros_like(p) for p in pg]
    v = [Blocks8.zeros_like(p) for p in pg]
    step = torch.zeros((), dtype=torch.int64, device=gpu)
    adamw_step(pg, gg, m, v, step, **HYPER, seed=5)
    assert int(step) == 1
    for i, (p, x) in enumerate(zip(ps, gs)):
        zero, one = np.zeros(p.numel(), np.uint8), np.ones(-(-p.numel() // 128), np.float32)
        want, mc, rc, _ = O.step(p.numpy(), x.numpy(), zero, zero, 1, i, **HYPER, seed=5, scales=(one, one))
        assert np.array_equal(bits(m[i].codes), mc) and np.array_equal(bits(v[i].codes), rc) and close(pg[i], want, torch.float32), i


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sizes", [[1], [5000, 3, 70001], [2049] * 60, [3_000_001]])
def test_norm(gpu, dtype, sizes):
    # fp64 sums of exact squares, one rounding to fp32 at the end
    g = torch.Generator().manual_seed(1)
    grads = [torch.randn(n, generator=g).to(dtype) for n in sizes]
    want = float(sum(x.double().square().sum() for x in grads).sqrt())
    got, clip = global_grad_norm([x.to(gpu) for x in grads], max_norm=1.0)
    assert abs(float(got) - want) <= 2 * U * want and abs(float(clip) - min(1.0, 1.0 / (want + 1e-6))) <= 2 * U
    assert float(global_grad_norm([x.to(gpu) for x in grads])) == float(got)
    again, _ = global_grad_norm([x.to(gpu) for x in grads], max_norm=1.0)
    assert float(again) == float(got)
    zero, clip = global_grad_norm([torch.zeros(5, device=gpu), torch.zeros(0, device=gpu)], max_norm=1.0)
    assert float(zero) == 0 and float(clip) == 1


@pytest.mark.parametrize("max_norm", [0.5, 1e9, 0.0])
def test_clipping(gpu, max_norm):
    g = torch.Generator().manual_seed(2)
    ps, gs = ([torch.randn(n, generator=g) for n in (300, 4000)] for _ in "pg")
    pg, gg = [p.to(gpu) for p in ps], [x.to(gpu) for x in gs]
    m, v = ([torch.zeros_like(p) for p in pg] for _ in "mv")
    step = torch.zeros((), dtype=torch.int64, device=gpu)
    norm = adamw_step(pg, gg, m, v, step, **HYPER, max_grad_norm=max_norm)
    want = float(sum(x.double().square().sum() for x in gs).sqrt())
    assert abs(float(norm) - want) <= 2 * U * want
    clip = np.float32(min(1.0, max_norm / (float(norm) + 1e-6)))
    for i, (p, x) in enumerate(zip(ps, gs)):
        w, wm, wv = O.step(p.numpy(), x.numpy(), np.zeros(len(p), np.float32), np.zeros(len(p), np.float32), 1, i, **HYPER, clip=clip)
        assert np.array_equal(m[i].cpu().numpy(), wm) and np.array_equal(v[i].cpu().numpy(), wv) and close(pg[i], w, torch.float32)
        assert torch.equal(gg[i].cpu(), x)                   # the gradients themselves stay as they are
    # the same through a factor on the device
    p2, m2, v2 = ([t.clone().to(gpu) for t in ts] for ts in (ps, [torch.zeros_like(p) for p in ps], [torch.zeros_like(p) for p in ps]))
    step.zero_()
    adamw_step(p2, gg, m2, v2, step, **HYPER, clip=torch.tensor(float(clip), device=gpu))
    assert all(torch.equal(a, b) for a, b in zip(p2, pg))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_gradients_that_are_not_finite(gpu, bad):
    p = torch.ones(1024, device=gpu)
    grad = torch.full((1024,), 1e-3, device=gpu)
    grad[300] = bad
    m, v = Blocks8.zeros_like(p), Blocks8.zeros_like(p)
    step = torch.zeros((), dtype=torch.int64, device=gpu)
    adamw_step([p], [grad], [m], [v], step, **HYPER)
    hit = torch.zeros(1024, dtype=torch.bool)
    hit[256:384] = True                                      # its block of 128
    assert torch.equal(torch.isnan(m.float()).cpu(), hit) and torch.equal(torch.isnan(v.float()).cpu(), hit)
    assert torch.isfinite(p[~hit.to(gpu)]).all() and int((~torch.isfinite(p)).sum()) == 1
    norm = adamw_step([p.clone().nan_to_num()], [grad], [Blocks8.zeros_like(p)], [Blocks8.zeros_like(p)], step, **HYPER, max_grad_norm=1.0)
    assert not np.isfinite(float(norm))


def test_blocks_of_zeros_and_wide_ranges(gpu):
    # one block of zeros, one with a single element, one whose magnitudes span 2^-60 .. 2^20, one of subnormals
    grad = torch.zeros(512)
    grad[200] = 3.0
    grad[256:384] = 2.0 ** torch.linspace(-60, 20, 128)
    grad[384:] = 2.0 ** -140
    p = torch.zeros(512, device=gpu)
    m, v = Blocks8.zeros_like(p), Blocks8.zeros_like(p)
    step = torch.zeros((), dtype=torch.int64, device=gpu)
    adamw_step([p], [grad.to(gpu)], [m], [v], step, **HYPER)
    zero, one = np.zeros(512, np.uint8), np.ones(4, np.float32)
    _, mc, rc, (ms, rs) = O.step(np.zeros(512, np.float32), grad.numpy(), zero, zero, 1, 0, **HYPER, scales=(one, one))
    assert np.array_equal(bits(m.codes), mc) and np.array_equal(bits(v.codes), rc)
    assert np.array_equal(m.scales.cpu().numpy(), ms) and np.array_equal(v.scales.cpu().numpy(), rs)
    assert torch.all(v.float()[256:384] > 0)                 # however small beside its block's largest
    assert torch.all(m.float()[:128] == 0) and float(m.scales[0]) == 1.0
    # a zero gradient after it moves no parameter by more than a few learning rates
    before = p.clone()
    adamw_step([p], [torch.zeros(512, device=gpu)], [m], [v], step, **HYPER)
    assert float((p - before).abs().max()) <= 20 * HYPER["lr"]


def test_rounding_is_unbiased_and_small_changes_accumulate(gpu):
    # the mean of N codes of one value: each off by at most a step of 2^-3 relative, so N of them by six standard deviations
    # of 2^-4 / sqrt(N) at most
    n = 1 << 20
    p, grad = torch.zeros(n, device=gpu), torch.full((n,), 1.03e-3, device=gpu)
    m, v = Blocks8.zeros_like(p), Blocks8.zeros_like(p)
    step = torch.zeros((), dtype=torch.int64, device=gpu)
    adamw_step([p], [grad], [m], [v], step, **HYPER)
    for state, want in ((m, 1.03e-4), (v, 1.03e-3 * 0.05 ** 0.5)):
        assert abs(float(state.float().double().mean()) / want - 1) <= 6 * 2.0 ** -4 / n ** 0.5
    assert len(m.float().unique()) == 2                       # the two neighbours
    # sqrt(v) of 500 steps without a gradient at b2 = 0.999 falls by 0.999^250, though one step changes it by 0.05 % and a
    # code by 6 % at least; a rounded walk of 500 steps of at most 0.125 * sqrt(5e-4) each stays within 6 of its deviations
    before = v.float().double().mean()
    for _ in range(500):
        adamw_step([p], [torch.zeros_like(grad)], [m], [v], step, lr=0.0, betas=(0.9, 0.999), seed=3)
    fall = float(v.float().double().mean() / before)
    assert abs(fall / 0.999 ** 250 - 1) <= 6 * 0.125 * (5e-4 * 500) ** 0.5 / n ** 0.5 + 1e-3


def test_same_call_same_bits_and_seeds_differ(gpu):
    g = torch.Generator().manual_seed(3)
    grad = torch.randn(100_000, generator=g).to(gpu)
    out = []
    for seed in (1, 1, 2):
        p = torch.zeros_like(grad)
        m, v = Blocks8.zeros_like(p), Blocks8.zeros_like(p)
        adamw_step([p], [grad], [m], [v], torch.zeros((), dtype=torch.int64, device=gpu), **HYPER, seed=seed)
        out.append(bits(m.codes))
    assert np.array_equal(out[0], out[1]) and not np.array_equal(out[0], out[2])


# ---- the optimizer ------------------------------------------------------------------------------------------------
def _net(gpu, dtype=torch.float32):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(33, 65), torch.nn.Tanh(), torch.nn.Linear(65, 17)).to(gpu, dtype)


@pytest.mark.parametrize("clip", [None, 0.1])
def test_optimizer_against_torch(gpu, clip):
    # fp32: each step differs by a few roundings of values of order 1
    a, b = _net(gpu), _net(gpu)
    groups = lambda n: [{"params": [n[0].weight, n[2].weight], "weight_decay": 0.1}, {"params": [n[0].bias, n[2].bias], "weight_decay": 0.0, "lr": 1e-3}]  # noqa: E731
    ours = AdamW(groups(a), lr=5e-3, max_grad_norm=clip)
    theirs = torch.optim.AdamW(groups(b), lr=5e-3, foreach=False)
    sched = [torch.optim.lr_scheduler.StepLR(o, 2, 0.5) for o in (ours, theirs)]
    for i in range(6):
        x = torch.randn(20, 33, device=gpu, generator=torch.Generator(device=gpu).manual_seed(i))
        for net in (a, b):
            net.zero_grad()
            net(x).square().mean().backward()
        if clip is not None:
            norm = torch.nn.utils.clip_grad_norm_(b.parameters(), clip)
        ours.step()
        theirs.step()
        if clip is not None:
            assert abs(float(ours.grad_norm) - float(norm)) <= 1e-6 * float(norm) + 1e-7 + 1e-4 * i * float(norm)
        for s in sched:
            s.step()
        if i == 0:
            # one step from equal weights: 8 u of weights of order 0.2, and the update m / (sqrt v + eps) of elements whose
            # gradient is tiny beside eps moves with the roundings of the gradients' clipping
            assert all(torch.allclose(p, q, rtol=1e-5, atol=1e-6) for p, q in zip(a.parameters(), b.parameters()))
    assert all(float((p - q).abs().max()) <= 6 * 5e-3 * 0.02 for p, q in zip(a.parameters(), b.parameters()))


@pytest.mark.parametrize("state_bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
def test_state_dict_continues_bit_for_bit(gpu, state_bits, master):
    a = _net(gpu, torch.bfloat16)
    opt = AdamW(a.parameters(), lr=1e-2, state_bits=state_bits, master_weights=master, seed=9)

    def train(net, o, seeds):
        for s in seeds:
            x = torch.randn(8, 33, device=gpu, generator=torch.Generator(device=gpu).manual_seed(s)).bfloat16()
            o.zero_grad()
            net(x).float().square().mean().backward()
            o.step()

    train(a, opt, range(3))
    state = opt.state[a[0].weight]
    assert ("master" in state) == master and state["exp_avg"].dtype == (torch.float32 if state_bits == 32 else torch.float8_e4m3fn)
    b = copy.deepcopy(a)
    opt2 = AdamW(b.parameters(), lr=5e-1, state_bits=state_bits, master_weights=master)
    import io
    f = io.BytesIO()
    torch.save(opt.state_dict(), f)
    f.seek(0)
    opt2.load_state_dict(torch.load(f, weights_only=True, map_location="cpu"))
    train(a, opt, range(3, 6))
    train(b, opt2, range(3, 6))
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    for p, q in zip(a.parameters(), b.parameters()):
        for k, t in opt.state[p].items():
            u = opt2.state[q][k]
            assert t.dtype == u.dtype and torch.equal(t.view(torch.uint8), u.view(torch.uint8)), k


def test_takes_over_a_state_of_torchs(gpu):
    a = _net(gpu)
    theirs = torch.optim.AdamW(a.parameters(), lr=5e-3, foreach=False)

    def train(net, o, seeds):
        for s in seeds:
            x = torch.randn(8, 33, device=gpu, generator=torch.Generator(device=gpu).manual_seed(s))
            o.zero_grad()
            net(x).square().mean().backward()
            o.step()

    train(a, theirs, range(3))
    b = copy.deepcopy(a)
    ours = AdamW(b.parameters(), lr=1.0)
    ours.load_state_dict(theirs.state_dict())
    assert int(ours.param_groups[0]["step"]) == 3 and ours.param_groups[0]["lr"] == 5e-3
    train(a, theirs, [3])
    train(b, ours, [3])
    assert all(torch.allclose(p, q, rtol=1e-5, atol=1e-6) for p, q in zip(a.parameters(), b.parameters()))


def test_beyond_32_bits_of_offset(gpu):
    # 2^31 + 5 bf16 weights with fp32 states: the last elements as a tensor of their own gets them
    n, tail = (1 << 31) + 5, 4101
    p = torch.full((n,), 0.5, dtype=torch.bfloat16, device=gpu)
    grad = torch.zeros(n, dtype=torch.bfloat16, device=gpu)
    m, v = torch.zeros(n, device=gpu), torch.zeros(n, device=gpu)
    g = torch.Generator().manual_seed(1)
    p[-tail:] = torch.randn(tail, generator=g).to(gpu)
    grad[-tail:] = torch.randn(tail, generator=g).to(gpu)
    q, h = p[-tail:].clone(), grad[-tail:].clone()
    mq, vq = torch.zeros(tail, device=gpu), torch.zeros(tail, device=gpu)
    for args in ((p, grad, m, v), (q, h, mq, vq)):
        step = torch.zeros((), dtype=torch.int64, device=gpu)
        norm = adamw_step(*([t] for t in args), step, **HYPER, max_grad_norm=1.0)
    assert abs(float(norm) - float(h.double().norm())) <= 1e-5 * float(norm)
    # (the norms of both calls are the same number up to the order of an fp64 sum)
    assert torch.allclose(m[-tail:], mq, rtol=1e-6, atol=0) and torch.allclose(p[-tail:].float(), q.float(), rtol=2 ** -8, atol=0)
    assert float(m[:-tail].abs().max()) == 0 and torch.all(p[:4096] == p[0])


def test_optimizer_corners(gpu):
    a = _net(gpu)
    opt = AdamW(a.parameters())
    opt.step()                                               # no gradients: nothing happens
    assert opt.grad_norm is None and not opt.state
    a[0].weight.grad = torch.ones((), device=gpu).expand_as(a[0].weight)       # an expanded gradient
    before = a[2].weight.clone()
    loss = opt.step(lambda: 7.0)
    assert loss == 7.0 and torch.equal(a[2].weight, before) and not opt.state.get(a[2].weight)
    lr = torch.tensor(0.0, device=gpu)
    opt = AdamW(a.parameters(), lr=lr, weight_decay=0.0)
    w = a[0].weight.clone()
    opt.step()
    assert torch.equal(a[0].weight, w)                       # a rate of 0 from the device
    lr.fill_(1e-2)
    opt.step()
    assert not torch.equal(a[0].weight, w)


@pytest.mark.parametrize("state_bits", [32, 8])
def test_graph_replay_counts_steps(gpu, state_bits):
    n = 70_001
    g = torch.Generator().manual_seed(4)
    grad = torch.randn(n, generator=g).to(gpu)
    lr = torch.tensor(1e-2, device=gpu)

    def fresh():
        p = torch.zeros(n, device=gpu, requires_grad=True)
        p.grad = grad.clone()
        return p, AdamW([p], lr=lr, state_bits=state_bits, max_grad_norm=1.0, seed=2)

    p, opt = fresh()
    q, ref = fresh()
    opt.step()
    ref.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for i in range(4):
        lr.fill_(1e-2 / (i + 1))
        p.grad.copy_(grad * (i - 1))
        q.grad.copy_(grad * (i - 1))
        graph.replay()
        torch.cuda.synchronize()
        ref.step()
        torch.cuda.synchronize()
        assert torch.equal(p, q) and float(opt.grad_norm) == float(ref.grad_norm), i
        for k, t in opt.state[p].items():
            assert torch.equal(t.view(torch.uint8), ref.state[q][k].view(torch.uint8)), (i, k)
    assert int(opt.param_groups[0]["step"]) == 5


def test_other_stream(gpu):
    grad = torch.randn(300_000, device=gpu)
    want = None
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            p, m, v = (torch.zeros_like(grad) for _ in "pmv")
            step = torch.zeros((), dtype=torch.int64, device=gpu)
            adamw_step([p], [grad], [m], [v], step, **HYPER, max_grad_norm=1.0)
        torch.cuda.synchronize()
        want = p if want is None else want
    assert torch.equal(p, want)


def test_refusals(gpu):
    p, g = torch.zeros(256, device=gpu), torch.zeros(256, device=gpu)
    m, v, step = torch.zeros_like(p), torch.zeros_like(p), torch.zeros((), dtype=torch.int64, device=gpu)
    ok = dict(params=[p], grads=[g], exp_avgs=[m], exp_avg_sqs=[v], step=step)
    b8 = Blocks8.zeros_like(p)
    for kw, err in [(dict(grads=[g[:255]]), ValueError), (dict(grads=[g.half()]), TypeError), (dict(grads=[]), ValueError),
                    (dict(params=[torch.zeros(16, 16, device=gpu).t()], grads=[torch.zeros(16, 16, device=gpu)]), ValueError),
                    (dict(exp_avgs=[m.bfloat16()]), TypeError), (dict(exp_avgs=[b8]), ValueError),
                    (dict(exp_avgs=[b8], exp_avg_sqs=[Blocks8(b8.codes, b8.scales[:1])]), ValueError),
                    (dict(step=step.int()), ValueError), (dict(step=step.cpu()), ValueError), (dict(masters=[m]), ValueError),
                    (dict(params=[p, p], grads=[g, g], exp_avgs=[m, m.clone()], exp_avg_sqs=[v, v.clone()]), ValueError),
                    (dict(params=[p, p.clone()], grads=[g, g], exp_avgs=[m, m], exp_avg_sqs=[v, v.clone()]), ValueError),
                    (dict(exp_avg_sqs=[m]), ValueError),
                    (dict(lr=torch.zeros((), dtype=torch.float64, device=gpu)), ValueError), (dict(seed=-1), ValueError),
                    (dict(max_grad_norm=-1.0), ValueError), (dict(max_grad_norm=1.0, clip=m[0]), ValueError),
                    (dict(params=[p.cpu()]), RuntimeError), (dict(params=[], grads=[], exp_avgs=[], exp_avg_sqs=[]), ValueError)]:
        with pytest.raises(err):
            adamw_step(**{**ok, **kw})
    flat = torch.zeros(600, device=gpu)
    for kw in (dict(params=[flat[:256], flat[255:511]], grads=[g, g], exp_avgs=[m, m.clone()], exp_avg_sqs=[v, v.clone()]),
               dict(params=[flat[:256]], grads=[flat[200:456]])):
        with pytest.raises(RuntimeError, match="overlaps"):
            adamw_step(**{**ok, **kw})
    for kw in (dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(lr=-1.0), dict(weight_decay=float("nan"))):
        with pytest.raises(RuntimeError):
            adamw_step(**ok, **kw)
    assert int(step) == 0
    for kw in (dict(state_bits=4), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(max_grad_norm=-1.0)):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(p)], **kw)
    with pytest.raises(ValueError):
        global_grad_norm([])


def test_neighbours_in_one_buffer(gpu):
    """Everything in one allocation without a gap, one gradient for both parameters: nothing overlaps."""
    n = 301
    flat, g = torch.randn(6 * n, device=gpu), torch.randn(n, device=gpu)
    flat[2 * n:] = 0
    parts = list(flat.split(n))
    before = flat.clone()
    step = torch.zeros((), dtype=torch.int64, device=gpu)
    adamw_step(parts[:2], [g, g], parts[2:4], parts[4:], step, lr=0.1, weight_decay=0.0)
    want = before[:2 * n] - 0.1 * torch.sign(g).repeat(2)
    # |m / sqrt(v)| = 1 in exact arithmetic after one step: eps, some 12 roundings of the update, one each of the two sums
    limit = 0.1 * (16 * 2.0 ** -24 + 1e-8 / float(g.abs().min())) + 2 * 2.0 ** -24 * (float(before.abs().max()) + 0.1)
    assert float((flat[:2 * n] - want).abs().max()) <= limit
