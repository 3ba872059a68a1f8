"""One AdamW step in IEEE single precision, operation by operation, with the 8-bit states' codes as bit patterns."""
from __future__ import annotations

import numpy as np

F = np.float32
BLOCK = 128


def mix(x: np.ndarray) -> np.ndarray:
    with np.errstate(over="ignore"):
        x = np.asarray(x, dtype=np.uint32)
        x = (x ^ (x >> np.uint32(16))) * np.uint32(0x6A09E667)
        x = (x ^ (x >> np.uint32(15))) * np.uint32(0xBB67AE85)
        return x ^ (x >> np.uint32(16))


def value_of(code: np.ndarray) -> np.ndarray:
    """fp32 values of e4m3 codes (bias 7, no infinities)."""
    c = code.astype(np.int64)
    e, f = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (8 + f) * 2.0 ** (e - 10), f * 2.0 ** -9)
    return np.where(c & 128, -v, v).astype(F)


def spread(code, scale):
    with np.errstate(invalid="ignore"):
        return (value_of(code) * np.repeat(scale, BLOCK)[:len(code)]).astype(F)


def pack(x: np.ndarray, r: np.ndarray, positive: bool):
    """(codes, scales) of x; r: 20 random bits per element."""
    n = len(x)
    mag = np.abs(x)
    padded = np.zeros(-(-n // BLOCK) * BLOCK, dtype=F)
    padded[:n] = mag
    top = padded.reshape(-1, BLOCK).max(1)
    k = np.maximum(((top.view(np.uint32).astype(np.int64) + 0x1FFFFF) >> 23) - 8, 1)
    k = np.where(top == 0, 127, k)
    finite = np.isfinite(top)
    scale = np.where(finite, (k << 23).astype(np.uint32).view(F), F(np.nan)).astype(F)
    with np.errstate(all="ignore"):
        y = mag * np.repeat(((254 - k) << 23).astype(np.uint32).view(F), BLOCK)[:n]
        normal = ((y.view(np.uint32).astype(np.int64) + r) >> 20) - 960
        small = ((y.astype(np.float64) * 2.0 ** 29).astype(np.int64) + r) >> 20
    code = np.where(y >= 2.0 ** -6, normal, small)
    code = np.maximum(code, x > 0) if positive else code | np.where(np.signbit(x), 128, 0)
    return np.where(np.repeat(finite, BLOCK)[:n], code, 0).astype(np.uint8), scale


def step(p, g, m, v, t, ordinal=0, *, lr, betas, eps, weight_decay, clip=1.0, seed=0, scales=None):
    """p, g fp32 arrays; m, v fp32, or e4m3 codes with ``scales = (m's, sqrt v's)``; t: the step's number after counting it.
    Returns (p, m, v) or (p, m codes, sqrt v codes, (scales))."""
    b1, b2 = betas
    if scales is not None:
        m, v = spread(m, scales[0]), spread(v, scales[1])
        v = v * v
    with np.errstate(all="ignore"):
        g = g * F(clip)
        m = m * F(b1) + g * F(1.0 - b1)
        v = v * F(b2) + g * g * F(1.0 - b2)
        root = np.sqrt(v)
        p = p * F(1.0 - lr * weight_decay) - F(lr / (1.0 - b1 ** t)) * (m / (root * F(1.0 / np.sqrt(1.0 - b2 ** t)) + F(eps)))
    if scales is None:
        return p, m, v
    key = mix(np.uint32((t * 0x9E3779B9 + seed) & 0xFFFFFFFF)).astype(np.int64) + ordinal * 0xBB67AE85
    h = mix(((np.arange(len(p), dtype=np.int64) * 0x9E3779B9 + key) & 0xFFFFFFFF).astype(np.uint32)).astype(np.int64)
    mc, ms = pack(m, (h & 0xFFFF) * 16 + 8, False)
    rc, rs = pack(root, (h >> 16) * 16 + 8, True)
    return p, mc, rc, (ms, rs)
