"""AdamW over many tensors at once, states in 32 or in 8 bits, with the global norm of the gradients.

The step that applies what ``loss.backward()`` left: the reference builds torch's AdamW over the model's parameters
(maester/optimizers.py) and clips the gradients by their global norm in its training loop (train.py).  Here one call does
both in a few launches, without a host synchronisation: ``adamw_step`` on lists of tensors, ``AdamW`` as a
``torch.optim.Optimizer``, ``global_grad_norm`` for the norm alone.

8-bit states (a quarter of the memory, 4.13 instead of 16 bytes moved per element and step): exp_avg and the square root
of exp_avg_sq as ``torch.float8_e4m3fn`` values with one power-of-two scale per 128 consecutive elements, rounded
stochastically from a hash of (seed, step, index of the tensor, element): the same call twice gives the same bits.
"""
from __future__ import annotations

import warnings
from operator import attrgetter
from typing import NamedTuple, Sequence

import numpy as np
import torch

from . import _lib

BLOCK = _lib.MA_ADAMW_BLOCK


class Blocks8(NamedTuple):
    """An 8-bit state of one tensor: ``codes`` ``torch.float8_e4m3fn`` of the tensor's shape, ``scales`` fp32
    ``[ceil(n / 128)]``; element i stands for ``codes[i] * scales[i // 128]`` (exp_avg_sq: for the square of that)."""
    codes: torch.Tensor
    scales: torch.Tensor

    @classmethod
    def zeros_like(cls, p: torch.Tensor) -> "Blocks8":
        return cls(torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn),
                   torch.ones(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device))

    def float(self) -> torch.Tensor:
        """The values that the codes stand for (of exp_avg_sq: its square root)."""
        flat = self.codes.float().view(-1)
        return (flat * self.scales.repeat_interleave(BLOCK)[:flat.numel()]).view(self.codes.shape)


_ACTIVATION = frozenset((torch.bfloat16, torch.float32))
_F32 = frozenset((torch.float32,))
_E4M3 = frozenset((torch.float8_e4m3fn,))
_CODE = {torch.bfloat16: _lib.MA_DTYPE_BF16, torch.float32: _lib.MA_DTYPE_F32}
_dtype, _shape = attrgetter("dtype"), attrgetter("shape")


def _device(tensors, who: str) -> torch.device:
    """The one GPU that all of ``tensors`` are on."""
    _lib.require_gpu(tensors[0], who)
    indices = set(map(torch.Tensor.get_device, tensors))
    if len(indices) > 1:
        raise (RuntimeError if -1 in indices else ValueError)(f"{who}: tensors on several devices; one call takes one GPU's")
    return tensors[0].device


def _addresses(tensors, what: str, shapes: list, dtypes: frozenset, dev: torch.device | None) -> list:
    """Data pointers of ``tensors`` after checking them against the parameters' shapes and device (None: checked already;
    whole lists at a time: a step over hundreds of small tensors is as fast as its host code)."""
    found = set(map(_dtype, tensors))
    if not found <= dtypes:
        raise TypeError(f"{what} must be {' or '.join(sorted(map(str, dtypes)))}, got {', '.join(sorted(map(str, found - dtypes)))}")
    if list(map(_shape, tensors)) != shapes or not all(map(torch.Tensor.is_contiguous, tensors)):
        raise ValueError(f"{what} must be contiguous and of its parameter's shape")
    if dev is not None and set(map(torch.Tensor.get_device, tensors)) != {dev.index}:
        raise ValueError(f"{what} must be on its parameter's device {dev}")
    return list(map(torch.Tensor.data_ptr, tensors))


def _table(n: int, sizes: list, params, grads, **columns) -> np.ndarray:
    """The C array of ``ma_adamw_tensor``: seven addresses, the size, the two dtypes in one word, a word of the library's."""
    none = [0] * n
    names = ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "master")
    codes = [_CODE[p.dtype] | _CODE[g.dtype] << 32 for p, g in zip(params, grads)]
    return np.array([*(columns.get(k, none) for k in names), sizes, codes, none], dtype=np.uint64).T.copy()


def _scalar(t: torch.Tensor, what: str, dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    if t.dtype != dtype or t.numel() != 1 or t.device != dev:
        raise ValueError(f"{what} must be one {dtype} value on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t


def _workspace(count: int, dev: torch.device):
    n = _lib.lib().ma_adamw_workspace_bytes(count)
    return torch.empty(n, dtype=torch.uint8, device=dev), n


def global_grad_norm(grads: Sequence[torch.Tensor], max_norm: float | None = None):
    """2-norm over all elements of ``grads`` (bf16 or fp32, contiguous, one device) as an fp32 scalar on the device, summed
    in fp64; with ``max_norm`` the pair ``(norm, min(1, max_norm / (norm + 1e-6)))``, as ``clip_grad_norm_`` scales by."""
    grads = list(grads)
    if not grads:
        raise ValueError("no gradients")
    _lib.require_plain("global_grad_norm", *grads)
    _lib.refuse_tangents("global_grad_norm", *grads)
    if max_norm is not None and not float(max_norm) >= 0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    dev = _device(grads, "global_grad_norm")
    table = _table(len(grads), list(map(torch.Tensor.numel, grads)), grads, grads,
                   grad=_addresses(grads, "a gradient", list(map(_shape, grads)), _ACTIVATION, dev))
    out = torch.empty(2, dtype=torch.float32, device=dev)
    ws, n = _workspace(len(grads), dev)
    _lib.launch(dev, _lib.lib().ma_grad_norm, table.ctypes.data, len(grads), -1.0 if max_norm is None else float(max_norm),
                out.data_ptr(), out.data_ptr() + 4, ws.data_ptr(), n)
    return out[0] if max_norm is None else (out[0], out[1])


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence, exp_avg_sqs: Sequence,
               step: torch.Tensor, *, lr: float | torch.Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 1e-2, max_grad_norm: float | None = None,
               clip: torch.Tensor | None = None, masters: Sequence[torch.Tensor | None] | None = None,
               seed: int = 0) -> torch.Tensor | None:
    """One AdamW step in place on every tensor of ``params`` (bf16 or fp32, contiguous, all on one device).

    ``grads`` bf16 or fp32 of the same shapes; ``exp_avgs`` / ``exp_avg_sqs`` fp32 tensors, or ``Blocks8`` for 8-bit states
    (all of one kind); ``step`` one int64 on the device, the number of steps so far, incremented by the call; ``lr`` a
    number or one fp32 value on the device (which a captured graph reads anew on every replay).  ``masters``: fp32 weights
    behind bf16 parameters (``None`` entries for parameters without): they are what is updated, the parameter is their
    rounding.  Without a master a bf16 parameter is updated in fp32 and rounded to the nearest bf16 value, which loses
    steps below 2^-9 of the weight.  ``max_grad_norm``: the gradients are scaled by ``min(1, max_grad_norm / (norm + 1e-6))``
    with the global norm of this call's, which is returned as an fp32 scalar on the device; ``clip``: an fp32 factor on the
    device to scale by instead.  A gradient that is not finite makes its element (8-bit states: its block of 128) NaN, or
    all of them through the norm.  ``seed`` picks the random bits of the 8-bit rounding.  All that is written counts as modified
    in place (a backward through a graph that saved it before the step raises)."""
    n = len(params)
    masters = [None] * n if masters is None else masters
    if not len(grads) == len(exp_avgs) == len(exp_avg_sqs) == len(masters) == n:
        raise ValueError("params, grads, exp_avgs, exp_avg_sqs (and masters) must have one entry per parameter")
    if n == 0:
        raise ValueError("no parameters")
    if max_grad_norm is not None and (clip is not None or not float(max_grad_norm) >= 0):
        raise ValueError("max_grad_norm must be >= 0 and cannot be given together with clip")
    if not 0 <= int(seed) < 1 << 32:
        raise ValueError("seed must be in [0, 2^32)")
    kinds = set(map(type, exp_avgs)) | set(map(type, exp_avg_sqs))
    _lib.require_plain_types("adamw_step", kinds.union(map(type, params), map(type, grads), map(type, masters)))
    _lib.refuse_tangents("adamw_step", *params, *grads)
    dev = _device(params, "adamw_step")
    eight = Blocks8 in kinds
    if eight and len(kinds) > 1:
        raise ValueError("exp_avgs and exp_avg_sqs must all be tensors or all Blocks8")
    shapes, sizes = list(map(_shape, params)), list(map(torch.Tensor.numel, params))
    where = _addresses(params, "a parameter", shapes, _ACTIVATION, None)
    columns = dict(param=where, grad=_addresses(grads, "a gradient", shapes, _ACTIVATION, dev))
    for name, states in (("exp_avg", exp_avgs), ("exp_avg_sq", exp_avg_sqs)):
        if eight:
            columns[name] = _addresses([q.codes for q in states], "codes", shapes, _E4M3, dev)
            columns[name + "_scale"] = _addresses([q.scales for q in states], "scales", [(-(-k // BLOCK),) for k in sizes], _F32, dev)
        else:
            columns[name] = _addresses(states, name, shapes, _F32, dev)
    held = [i for i, w in enumerate(masters) if w is not None]
    if held:
        if any(params[i].dtype != torch.bfloat16 for i in held):
            raise ValueError("a master belongs to a bf16 parameter")
        found = iter(_addresses([masters[i] for i in held], "a master", [shapes[i] for i in held], _F32, dev))
        columns["master"] = [0 if w is None else next(found) for w in masters]
    # a tensor that two entries would write is a race
    written = [columns[k] for k in ("param", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "master") if k in columns]
    addresses = [a for column in written for a, k in zip(column, sizes) if k and a]
    if len(set(addresses)) < len(addresses):
        raise ValueError("a parameter, state or master is listed twice")
    table = _table(n, sizes, params, grads, **columns)
    _scalar(step, "step", torch.int64, dev)
    on_device = isinstance(lr, torch.Tensor)
    if on_device:
        _scalar(lr, "lr", torch.float32, dev)
    if clip is not None:
        _scalar(clip, "clip", torch.float32, dev)
    norm = torch.empty((), dtype=torch.float32, device=dev) if max_grad_norm is not None else None
    ws, ws_bytes = _workspace(n, dev)
    _lib.launch(dev, _lib.lib().ma_adamw_step, table.ctypes.data, n, 8 if eight else 32, 0.0 if on_device else float(lr),
                lr.data_ptr() if on_device else None, float(betas[0]), float(betas[1]), float(eps), float(weight_decay),
                -1.0 if max_grad_norm is None else float(max_grad_norm), None if clip is None else clip.data_ptr(),
                None if norm is None else norm.data_ptr(), step.data_ptr(), int(seed), ws.data_ptr(), ws_bytes)
    # the kernels write behind autograd's back: a graph that saved one of these before the step has to raise
    states = [t for q in (*exp_avgs, *exp_avg_sqs) for t in q] if eight else [*exp_avgs, *exp_avg_sqs]
    torch.autograd.graph.increment_version([*params, *states, *(masters[i] for i in held), step])
    return norm


def _check_options(o: dict) -> None:
    """The options of a group, by name: a wrong one would show first in a step, after the states have been made."""
    lr, betas, eps, decay, seed = o["lr"], o["betas"], o["eps"], o["weight_decay"], o["seed"]
    if o["state_bits"] not in (32, 8):
        raise ValueError(f"state_bits must be 32 or 8, got {o['state_bits']}")
    if not isinstance(lr, torch.Tensor) and not float(lr) >= 0:
        raise ValueError(f"lr must be >= 0, got {lr}")
    if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1 and eps >= 0 and decay >= 0):
        raise ValueError(f"betas {betas}, eps {eps} or weight_decay {decay} out of range")
    if not 0 <= int(seed) < 1 << 32:
        raise ValueError(f"seed must be in [0, 2^32), got {seed}")


def _check_params(params: list) -> None:
    """What a step would refuse, before their states take memory."""
    _lib.require_plain("AdamW", *params)
    for p in params:
        if p.dtype not in _ACTIVATION:
            raise TypeError(f"a parameter must be {' or '.join(sorted(map(str, _ACTIVATION)))}, got {p.dtype}")
        if not p.is_contiguous():
            raise ValueError(f"a parameter must be contiguous, got {tuple(p.shape)} with strides {p.stride()}")
    _device(params, "AdamW")


def _check_torchs(group: dict, states: list) -> None:
    """Refuses what ``torch.optim.AdamW`` has not saved, or what its options make another update."""
    if not {"betas", "eps", "weight_decay", "amsgrad"} <= set(group) or any(not {"step", "exp_avg", "exp_avg_sq"} <= set(s) or
                                                                            set(s) - {"step", "exp_avg", "exp_avg_sq", "max_exp_avg_sq"} for s in states):
        raise ValueError("not a state of torch.optim.AdamW: its groups have betas, eps, weight_decay and amsgrad, its parameters step, "
                         "exp_avg and exp_avg_sq")
    for option in ("maximize", "amsgrad"):
        if group.get(option):
            raise ValueError(f"a state saved with {option} cannot be continued: AdamW here has no such option")
    if not group.get("decoupled_weight_decay", True) and group["weight_decay"] != 0:
        raise ValueError("a state whose weight decay is not decoupled (torch.optim.Adam's) cannot be continued")


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW``'s update (same defaults) through ``adamw_step``.

    ``state_bits`` 32 or 8; ``master_weights=True`` keeps fp32 weights behind bf16 parameters; ``max_grad_norm`` clips by the
    global norm over all groups, which ``grad_norm`` then holds as an fp32 scalar on the device.  ``lr`` may be one fp32
    value on the device.  Nothing in ``step()`` waits for the GPU, and it can be captured into a graph once it has run (the
    states exist then).  The step counter is the group's: a parameter without a gradient is left alone in that step but
    shares the others' bias correction.  All parameters on one device, contiguous."""

    def __init__(self, params, lr: float | torch.Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, master_weights: bool = False,
                 max_grad_norm: float | None = None, seed: int = 0):
        if max_grad_norm is not None and not float(max_grad_norm) >= 0:
            raise ValueError(f"max_grad_norm must be >= 0, got {max_grad_norm}")
        options = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                       master_weights=master_weights, seed=seed)
        _check_options(options)
        super().__init__(params, options)
        self.max_grad_norm = max_grad_norm
        self.grad_norm = None

    def add_param_group(self, param_group: dict) -> None:
        _check_options({**self.defaults, **param_group})
        super().add_param_group(param_group)
        try:
            _lib.require_plain("AdamW", *self.param_groups[-1]["params"])
        except TypeError:
            self.param_groups.pop()
            raise

    def _init_state(self, p: torch.Tensor, group: dict) -> dict:
        state = {}
        if group["state_bits"] == 8:
            for k in ("exp_avg", "exp_avg_sq"):
                state[k], state[k + "_scale"] = Blocks8.zeros_like(p)
        else:
            for k in ("exp_avg", "exp_avg_sq"):
                state[k] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if group["master_weights"] and p.dtype == torch.bfloat16:
            state["master"] = p.detach().float()
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work = []
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if params:
                fresh = [p for p in params if not self.state.get(p)]
                if fresh:
                    _check_params(fresh)
                    for p in fresh:
                        self.state[p] = self._init_state(p, group)
                if not isinstance(group.get("step"), torch.Tensor) or group["step"].device != params[0].device:
                    group["step"] = torch.as_tensor(group.get("step", 0), dtype=torch.int64).to(params[0].device)
                work.append((group, params, [p.grad.contiguous() for p in params]))
        if not work:
            return loss
        clip = None
        if self.max_grad_norm is not None and len(work) > 1:
            self.grad_norm, clip = global_grad_norm([g for _, _, grads in work for g in grads], self.max_grad_norm)
        for group, params, grads in work:
            states = [self.state[p] for p in params]
            if group["state_bits"] == 8:
                m, v = ([Blocks8(s[k], s[k + "_scale"]) for s in states] for k in ("exp_avg", "exp_avg_sq"))
            else:
                m, v = ([s[k] for s in states] for k in ("exp_avg", "exp_avg_sq"))
            norm = adamw_step(params, grads, m, v, group["step"], lr=group["lr"], betas=group["betas"], eps=group["eps"],
                              weight_decay=group["weight_decay"], masters=[s.get("master") for s in states], seed=group["seed"],
                              max_grad_norm=self.max_grad_norm if clip is None else None, clip=clip)
            if norm is not None:
                self.grad_norm = norm
        return loss

    @torch.no_grad()
    def load_state_dict(self, state_dict: dict) -> None:
        """Restores the states in the types they were saved in (torch's own would cast them to the parameter's).  A state of
        ``torch.optim.AdamW`` is taken over into 32-bit states; its per-parameter counters become the group's, the largest
        of them (with a warning where they differ).  One with ``maximize``, ``amsgrad`` or a weight decay that is not decoupled,
        or of another optimizer, is refused before anything changes.  Counters and rates that are tensors move to the
        parameters' device.  All tensors are new ones: a graph that captured ``step()`` has to be captured again."""
        saved = state_dict["state"]
        for old in state_dict["param_groups"]:
            if "state_bits" in old:
                _check_options(old)
            else:
                _check_torchs(old, [saved[i] for i in old["params"] if i in saved])
        super().load_state_dict(state_dict)
        for old, group in zip(state_dict["param_groups"], self.param_groups):
            foreign = "state_bits" not in old
            if foreign:
                steps = {int(saved[i]["step"]) for i in old["params"] if i in saved}
                if len(steps) > 1:
                    warnings.warn(f"parameters of one group have taken between {min(steps)} and {max(steps)} steps: all continue with the "
                                  f"bias correction of step {max(steps)}", stacklevel=2)
                group.update(state_bits=32, master_weights=self.defaults["master_weights"], seed=self.defaults["seed"],
                             step=max(steps, default=0))
            for dev in {p.device for p in group["params"]}:          # (one, or none in an empty group)
                if "step" in group:
                    group["step"] = torch.as_tensor(group["step"]).to(dev, torch.int64)
                if isinstance(group["lr"], torch.Tensor):
                    group["lr"] = group["lr"].detach().to(dev, torch.float32)
            for i, p in zip(old["params"], group["params"]):
                if i not in saved:
                    continue
                if not foreign:
                    self.state[p] = {k: t.detach().to(p.device, copy=True) for k, t in saved[i].items()}
                    continue
                self.state[p] = self._init_state(p, group)
                for k in ("exp_avg", "exp_avg_sq"):
                    self.state[p][k].copy_(saved[i][k])
