"""What the operators around a per-token fine-tuning step are measured on.

Three operators: ``token_logprobs`` (log-probabilities, entropy and top alternatives of rows of logits, and its
gradient), ``linear_token_logprobs`` (the same from hidden states and the classifier, without the logits) and
``adamw_step`` (AdamW over many tensors, states in 32 or 8 bits, gradients clipped by their global norm).  ``run``
computes them as the library does where ``own`` is true and in elementary torch operations otherwise; ``exact`` in 64
bits."""
from __future__ import annotations

import math

import torch

own = False

IGNORE = -100
BLOCK = 128                     # values that share a scale in the 8-bit states
M32 = 0xFFFFFFFF
K1, K2, K3 = 0x9E3779B9, 0x6A09E667, 0xBB67AE85   # 2^32 / golden ratio, fractions of sqrt 2 and sqrt 3


# ---- cases -------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of one sequence: the sampled token's log-probability and twenty alternatives
        logprobs("logprobs_decode_1", 1, 262208, "bf16", top_k=20),
        # a decode batch whose logits come in fp32, capped and cooled, a tenth of the vocabulary banned
        logprobs("logprobs_decode_48", 48, 262208, "fp32", top_k=5, softcap=30.0, temperature=0.7, banned=True),
        # scoring a block of a packed batch against the tied embedding's vocabulary
        logprobs("logprobs_score_4096", 4096, 262208, "bf16", top_k=8),
        # a policy step: log-probabilities and entropy, and the gradient of both, an odd vocabulary and row count
        logprobs("logprobs_train_2047", 2047, 128257, "bf16", grad=True),
        # a few sequences' last hidden states: bound by reading the classifier
        linear("linear_decode_8", 8, 2560, 262208, "bf16"),
        # one packed row of 8192 tokens scored at the width of the Gemma-3-4B layers
        linear("linear_score_8192", 8192, 2560, 262208, "bf16"),
        # a preference step on a quarter of that, with the gradients of hidden states and classifier
        linear("linear_train_2047", 2047, 2560, 262208, "bf16", grad=True),
        # the fp32 path at a small width
        linear("linear_train_fp32", 300, 640, 32003, "fp32", grad=True),
        # a tiny model's tensors, odd sizes: launch latency
        adamw("adamw_tiny", 24, 60_001, "fp32", 32, clip=True, tiny=True),
        # two decoder layers of the Gemma-3-4B shape: bf16 weights with fp32 masters
        adamw("adamw_layers_master", 22, 188_770_816, "bf16", 32, master=True, clip=True),
        # the same without masters and with 8-bit states
        adamw("adamw_layers_8bit", 22, 188_770_816, "bf16", 8),
        # the tied embedding table of the 262208-word vocabulary at width 2560, one tensor, 8-bit states
        adamw("adamw_embedding_8bit", 1, 671_252_480, "bf16", 8, clip=True),
    ]


def logprobs(name, rows, vocab, dtype, top_k=0, softcap=0.0, temperature=1.0, banned=False, grad=False):
    return dict(name=name, op="logprobs", rows=rows, vocab=vocab, dtype=dtype, top_k=top_k, softcap=softcap,
                temperature=temperature, banned=banned, grad=grad)


def linear(name, rows, width, vocab, dtype, softcap=0.0, temperature=1.0, grad=False):
    return dict(name=name, op="linear", rows=rows, width=width, vocab=vocab, dtype=dtype, softcap=softcap,
                temperature=temperature, grad=grad)


def adamw(name, tensors, total, dtype, bits, master=False, clip=False, tiny=False):
    return dict(name=name, op="adamw", tensors=tensors, total=total, dtype=dtype, bits=bits, master=master, clip=clip, tiny=tiny)


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "linear", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    softcap = rng.choice([0.0, 0.0, 30.0])
    temperature = rng.choice([1.0, 1.0, 0.7])
    grad = rng.random() < 0.5
    if op == "logprobs":
        vocab = rng.choice([_log_uniform(rng, 1000, 262208), 262208])
        rows = _log_uniform(rng, 1, min(4096, (1 << 28) // vocab))
        case = logprobs("", rows, vocab, dtype, 0 if grad else rng.choice([0, 1, 5, 20, 64]), softcap, temperature,
                        not grad and rng.random() < 0.3, grad)
    elif op == "linear":
        vocab = rng.choice([_log_uniform(rng, 1000, 262208), 262208])
        width = 8 * _log_uniform(rng, 8, 320)
        most = int((2 if dtype == "bf16" else 0.5) * 1e12 / (vocab * width))
        rows = _log_uniform(rng, 1, max(2, min(8192, most)))
        case = linear("", rows, width, vocab, dtype, softcap, temperature, grad)
    else:
        tensors = _log_uniform(rng, 1, 60)
        case = adamw("", tensors, _log_uniform(rng, 1000 * tensors, 2e8), dtype, rng.choice([32, 8]),
                     dtype == "bf16" and rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5)
    case.pop("name")
    return case


# ---- inputs ------------------------------------------------------------------------------------------------------
def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _sizes(case):
    """Element counts of a case's tensors: decoder-layer shapes where the total is that of the listed layers, otherwise
    parts of uneven, mostly odd sizes."""
    n, total = case["tensors"], case["total"]
    if n == 22 and total == 188_770_816:
        layer = [4096 * 2560, 2560 * 2048, 10240 * 2560, 10240 * 2560, 2560 * 10240, 2560, 2560, 2560, 2560, 256, 256]
        return layer + layer[:-1] + [total - sum(layer) - sum(layer[:-1])]
    if n == 1:
        return [total]
    weights = [1.0 / (1 + i % 7) ** 2 if not case["tiny"] else 1.0 + i % 5 for i in range(n)]
    part = [max(1, int(total * w / sum(weights))) for w in weights]
    return [p | 1 if i % 2 else p for i, p in enumerate(part)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _dtype(case)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    if case["op"] == "adamw":
        return _prepare_adamw(case, seed, dev, g, randn)
    rows, vocab = case["rows"], case["vocab"]
    targets = torch.randint(0, vocab, (rows,), generator=g, device=dev)
    state = dict(case=case, targets=targets)
    if case["op"] == "logprobs":
        x = randn(rows, vocab)
        x.mul_(3.0)
        x.scatter_add_(1, torch.randint(0, vocab, (rows, 6), generator=g, device=dev), 4.0 + 2.0 * randn(rows, 6))
        if case["banned"]:       # tokens that a sampler has ruled out
            out = torch.rand(vocab, generator=g, device=dev) < 0.1
            out[0] = False
            x.masked_fill_(out, -math.inf)
            targets.masked_fill_(out[targets], 0)
        state["logits"] = x.to(dt)
    else:
        state["e"] = randn(rows, case["width"], dtype=dt)
        state["c"] = randn(vocab, case["width"], dtype=torch.float32).mul_(3.0 / math.sqrt(case["width"])).to(dt)
    if case["grad"]:             # a third of a packed batch's tokens is prompt and carries no label
        drop = torch.rand(rows, generator=g, device=dev) < 0.3
        drop[0] = False
        targets.masked_fill_(drop, IGNORE)
        state["g_logp"], state["g_entropy"] = randn(rows) / rows, 0.01 * randn(rows) / rows
    return state


def _prepare_adamw(case, seed, dev, g, randn):
    sizes = _sizes(case)
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    dt = _dtype(case)
    flat = dict(p=randn(at).mul_(0.02), g=randn(at).mul_(1e-3))
    if case["master"]:
        flat["master"] = flat["p"]
    flat["p"], flat["g"] = flat["p"].to(dt), flat["g"].to(dt)
    if case["bits"] == 32:
        flat["m"], flat["v"] = randn(at).mul_(3e-4), randn(at).mul_(1e-3).square_()
    else:                        # states as an earlier step left them
        for k, width in (("m", 3e-4), ("v", 1e-3)):
            y = randn(at).mul_(width)
            y = (y.abs_() if k == "v" else y).view(-1, BLOCK)
            scale = torch.exp2(torch.ceil(torch.log2(y.abs().amax(1) / 448.0)))
            flat[k] = (y / scale[:, None]).to(torch.float8_e4m3fn).view(-1)
            flat[k + "_scale"] = scale
    views = {k: [t[s:s + n] if not k.endswith("_scale") else t[s // BLOCK:s // BLOCK + -(-n // BLOCK)]
                 for s, n in zip(starts, sizes)] for k, t in flat.items()}
    step = torch.full((), 40, dtype=torch.int64, device=dev)
    return dict(case=case, flat=flat, views=views, step=step, seed=int(seed) & 0x7FFFFFFF)


HYPER = dict(lr=2e-4, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
MAX_NORM = 1.0


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return {"logprobs": _run_logprobs, "linear": _run_linear, "adamw": _run_adamw}[case["op"]](state, case)


def _run_logprobs(state, case):
    cap = case["softcap"] or None
    if own:
        import maester_amd as ma
        x = state["logits"].detach().requires_grad_(case["grad"])
        out = ma.token_logprobs(x, state["targets"], top_k=case["top_k"], ignore_index=IGNORE, softcap=cap,
                                temperature=case["temperature"])
        if case["grad"]:
            dx, = torch.autograd.grad((out.logp, out.entropy), x, (state["g_logp"], state["g_entropy"]))
            return out.logp.detach(), out.entropy.detach(), dx
        return tuple(t for t in out if t is not None)
    x = state["logits"].float()
    logp, entropy, lse, y = _rows_of(x, state["targets"], cap, case["temperature"])
    if case["grad"]:
        d = _rows_gradient(x, y, lse, entropy, state["targets"], cap, case["temperature"], state["g_logp"], state["g_entropy"])
        return logp, entropy, d.to(state["logits"].dtype)
    if not case["top_k"]:
        return logp, entropy
    bits = x.view(torch.int32).to(torch.int64)
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)       # ascending with the value
    key = order * (1 << 31) + ((1 << 31) - 1 - torch.arange(x.shape[1], device=x.device))
    ids = key.topk(case["top_k"], dim=1).indices
    return logp, entropy, ids, y.gather(1, ids) - lse[:, None]


def _rows_of(x, targets, cap, temperature):
    """Log-probability of the target, entropy, log-sum-exp and the capped, tempered rows."""
    y = cap * torch.tanh(x / cap) if cap else x
    y = y / temperature if temperature != 1.0 else y
    m = y.amax(1, keepdim=True)
    e = torch.exp(y - m)
    total = e.sum(1)
    lse = m[:, 0] + torch.log(total)
    entropy = torch.log(total) - (e * (y - m).clamp_min(-1e30)).sum(1) / total
    keep = targets != IGNORE
    logp = y.gather(1, targets.clamp_min(0)[:, None])[:, 0] - lse
    return torch.where(keep, logp, 0.0), torch.where(keep, entropy, 0.0), lse, y


def _rows_gradient(x, y, lse, entropy, targets, cap, temperature, a, b):
    keep = targets != IGNORE
    a, b = torch.where(keep, a, 0.0)[:, None], torch.where(keep, b, 0.0)[:, None]
    logp = (y - lse[:, None]).clamp_min(-1e30)
    d = -torch.exp(logp) * (a + b * (logp + entropy[:, None]))
    d.scatter_add_(1, targets.clamp_min(0)[:, None], a)
    if cap:
        d = d * (1.0 - torch.tanh(x / cap).square())
    return d / temperature


def _run_linear(state, case):
    cap = case["softcap"] or None
    if own:
        import maester_amd as ma
        e, c = (state[k].detach().requires_grad_(case["grad"]) for k in "ec")
        logp, entropy = ma.linear_token_logprobs(e, c, state["targets"], ignore_index=IGNORE, softcap=cap,
                                                 temperature=case["temperature"])
        if case["grad"]:
            de, dc = torch.autograd.grad((logp, entropy), (e, c), (state["g_logp"], state["g_entropy"]))
            return logp.detach(), entropy.detach(), de, dc
        return logp, entropy
    e, c = state["e"].float(), state["c"].float()
    x = e @ c.t()
    logp, entropy, lse, y = _rows_of(x, state["targets"], cap, case["temperature"])
    if not case["grad"]:
        return logp, entropy
    d = _rows_gradient(x, y, lse, entropy, state["targets"], cap, case["temperature"], state["g_logp"], state["g_entropy"])
    return logp, entropy, (d @ c).to(state["e"].dtype), (d.t() @ e).to(state["c"].dtype)


def _run_adamw(state, case):
    v, flat = state["views"], state["flat"]
    if own:
        import maester_amd as ma
        eight = case["bits"] == 8
        m = [ma.Blocks8(*q) for q in zip(v["m"], v["m_scale"])] if eight else v["m"]
        s = [ma.Blocks8(*q) for q in zip(v["v"], v["v_scale"])] if eight else v["v"]
        norm = ma.adamw_step(v["p"], v["g"], m, s, state["step"], **HYPER, max_grad_norm=MAX_NORM if case["clip"] else None,
                             masters=v.get("master"), seed=state["seed"])
        return _adamw_outputs(flat, state["step"], norm)
    state["step"] += 1
    t = state["step"].double()
    norm = clip = None
    if case["clip"]:
        norm = torch.stack([g.double().square().sum() for g in v["g"]]).sum().sqrt().float()
        clip = (MAX_NORM / (norm.double() + 1e-6)).clamp_max(1.0).float()
    b1, b2 = HYPER["betas"]
    base = _mix((t.long() * K1 + state["seed"]) & M32)
    for i in range(len(v["p"])):
        g = v["g"][i].float()
        g = g * clip if case["clip"] else g
        if case["bits"] == 32:
            m, sq = v["m"][i], v["v"][i]
        else:
            m, sq = _spread(v["m"][i], v["m_scale"][i]), _spread(v["v"][i], v["v_scale"][i]).square()
        m = m * b1 + g * (1 - b1)
        sq = sq * b2 + g * g * (1 - b2)
        root = sq.sqrt()
        p = (v["master"] if case["master"] else v["p"])[i]
        step_size, root_bc = (HYPER["lr"] / (1 - b1 ** t)).float(), (1 / torch.sqrt(1 - b2 ** t)).float()
        new = p.float() * (1 - HYPER["lr"] * HYPER["weight_decay"]) - step_size * (m / (root * root_bc + HYPER["eps"]))
        p.copy_(new)
        if case["master"]:
            v["p"][i].copy_(new)
        if case["bits"] == 32:
            v["m"][i].copy_(m)
            v["v"][i].copy_(sq)
        else:
            h = _mix((torch.arange(m.numel(), device=m.device) * K1 + base + i * K3) & M32)
            _pack(m, (h & 0xFFFF) * 16 + 8, v["m"][i], v["m_scale"][i], False)
            _pack(root, (h >> 16) * 16 + 8, v["v"][i], v["v_scale"][i], True)
    return _adamw_outputs(flat, state["step"], norm)


def _adamw_outputs(flat, step, norm):
    """The 8-bit states are torch's float8 values and the scales that multiply them."""
    out = {k: t for k, t in flat.items() if k != "g"}
    return dict(out, step=step, **({} if norm is None else {"norm": norm}))


def _mix(x):
    """32 random-looking bits from 32 bits (int64 tensors of values below 2^32)."""
    x = ((x ^ (x >> 16)) * K2) & M32
    x = ((x ^ (x >> 15)) * K3) & M32
    return x ^ (x >> 16)


def _blocks(x):
    pad = -x.numel() % BLOCK
    return (torch.cat([x, x.new_zeros(pad)]) if pad else x).view(-1, BLOCK)


def _spread(codes, scale):
    x = codes.float()
    return (_blocks(x) * scale[:, None]).view(-1)[:x.numel()]


def _pack(x, r, codes, scale, positive):
    """Rounds x to e4m3 codes stochastically (r: 20 random bits), one power-of-two scale per block."""
    a = _blocks(x.abs())
    top = a.amax(1)
    k = (((top.view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp_min(1)       # exponent field of the scale
    k = torch.where(top == 0, 127, k)
    scale.copy_(torch.where(torch.isfinite(top), (k << 23).view(torch.float32), math.nan))
    y = (a * ((254 - k) << 23).view(torch.float32)[:, None]).view(-1)[:x.numel()]
    normal = ((y.view(torch.int32) + r) >> 20) - 960
    small = ((y * 2.0 ** 29).to(torch.int32) + r) >> 20
    code = torch.where(y >= 2.0 ** -6, normal, small)
    code = torch.maximum(code, (x > 0).long()) if positive else code + 128 * torch.signbit(x)
    codes.view(torch.uint8).copy_(code)


# ---- what one pass cannot do without -----------------------------------------------------------------------------
def work(case):
    elt = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        weights = 8 + elt if case["master"] else 2 * elt
        return {"bytes": n * (weights + state + elt), "flops": 15 * n}
    rows, vocab = case["rows"], case["vocab"]
    if case["op"] == "logprobs":
        n = rows * vocab
        return {"bytes": n * elt * (3 if case["grad"] else 1) + rows * (16 + 12 * case["top_k"]), "flops": n * (18 if case["grad"] else 8)}
    k = case["width"]
    once = (rows + vocab) * k * elt + rows * 16
    return {"bytes": once * (3 if case["grad"] else 1), "flops": rows * vocab * (2 * k * (4 if case["grad"] else 1) + 8)}


# ---- in 64 bits --------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(case, state)
    out, dc = [], 0.0
    rows, step = case["rows"], max(1, (1 << 29) // case["vocab"])
    c = state["c"].double() if case["op"] == "linear" else None
    for r in range(0, rows, step):
        part = slice(r, min(rows, r + step))
        if c is None:
            x = state["logits"][part].double()
        else:
            e = state["e"][part].double()
            x = e @ c.T
        got, d = _exact_rows(case, x, state["targets"][part], *((state[k][part].double() for k in ("g_logp", "g_entropy")) if case["grad"] else (None, None)))
        if case["grad"]:
            got = got[:2] + ([d.to(torch.float32) if d.numel() > 1 << 28 else d] if c is None else [d @ c])
            dc = dc + d.T @ e if c is not None else dc
        out.append(got)
    out = [None if column[0] is None else torch.cat(column) for column in zip(*out)]
    return out + [dc] if case["grad"] and c is not None else out


def _exact_rows(case, x, targets, ga, gb):
    live = targets != IGNORE
    t = torch.where(live, targets, torch.zeros_like(targets))
    cap, temperature = case["softcap"], case["temperature"]
    th = torch.tanh(x / cap) if cap else None
    lp = torch.log_softmax((cap * th if cap else x) / temperature, dim=-1)
    p = lp.exp()
    ent = -torch.nan_to_num(p * lp, nan=0.0).sum(-1)
    picked = lp[torch.arange(len(t), device=t.device), t]
    got = [torch.where(live, picked, torch.zeros_like(picked)), torch.where(live, ent, torch.zeros_like(ent))]
    if case.get("top_k"):
        got += [None, lp.topk(case["top_k"], dim=-1).values]
    if ga is None:
        return got, None
    one = torch.zeros_like(p)
    one[torch.arange(len(t), device=t.device), t] = 1.0
    d = (one - p) * ga[:, None] - p * (lp + ent[:, None]) * gb[:, None]
    d = d * (1 - th * th) if cap else d
    return got, torch.where(live[:, None], d / temperature, torch.zeros_like(d))


def _exact_adamw(case, state):
    views, flat = state["views"], state["flat"]
    t = int(state["step"]) + 1
    (b1, b2), lr = HYPER["betas"], HYPER["lr"]
    norm = math.sqrt(sum(float(g.double().pow(2).sum()) for g in views["g"])) if case["clip"] else None
    factor = min(1.0, MAX_NORM / (norm + 1e-6)) if case["clip"] else 1.0
    eight = case["bits"] == 8
    new = {k: x.clone() if eight and k in ("m", "v") else x.double() for k, x in flat.items()}
    for i, at in enumerate(views["p"]):
        n, start = at.numel(), at.storage_offset()
        part, blocks = slice(start, start + n), slice(start // BLOCK, start // BLOCK + -(-n // BLOCK))
        g = flat["g"][part].double() * factor
        m, v = flat["m"][part].double(), flat["v"][part].double()
        if eight:
            m = m * flat["m_scale"][blocks].double().repeat_interleave(BLOCK)[:n]
            v = (v * flat["v_scale"][blocks].double().repeat_interleave(BLOCK)[:n]) ** 2
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g ** 2
        p = flat["master" if case["master"] else "p"][part].double()
        p = p - lr * (HYPER["weight_decay"] * p + m / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + HYPER["eps"]))
        new["p"][part] = p
        if case["master"]:
            new["master"][part] = p
        if not eight:
            new["m"][part], new["v"][part] = m, v
            continue
        key = _scramble((t * K1 + state["seed"]) % 2 ** 32) + i * K3
        for name, x, low in (("m", m, True), ("v", v.sqrt(), False)):
            h = _scramble((torch.arange(n, device=x.device) * K1 + key) % 2 ** 32)
            u = ((h % 65536 if low else h // 65536).double() + 0.5) / 65536
            del h
            padded = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
            padded[:n] = x.abs()
            top = padded.view(-1, BLOCK).amax(1)
            scale = torch.exp2(torch.ceil(torch.log2(top / 448)))
            scale[top == 0] = 1.0
            y = x.abs() / scale.repeat_interleave(BLOCK)[:n]
            gap = torch.exp2(torch.floor(torch.log2(y.clamp_min(2.0 ** -6))) - 3)      # between neighbouring codes
            y = torch.floor(y / gap + u) * gap
            if not low:
                y = torch.where((x > 0) & (y == 0), 2.0 ** -9, y)
            new[name][part] = torch.copysign(y, x).to(torch.float8_e4m3fn)             # each is a code already
            new[name + "_scale"][blocks] = scale
    new.update({k: new[k].double() for k in ("m", "v")})
    del new["g"]
    new["step"] = None
    return dict(new, **({} if norm is None else {"norm": torch.tensor(norm, dtype=torch.float64)}))


def _scramble(x):
    x = (x ^ (x >> 16)) * K2 % 2 ** 32
    x = (x ^ (x >> 15)) * K3 % 2 ** 32
    return x ^ (x >> 16)
