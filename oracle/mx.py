"""64-bit restatement of the microscaled types and of the scored routing (TEST INFRASTRUCTURE ONLY).

MXFP4 blocks (17 bytes: E8M0 scale byte, 32 E2M1 codes, low nibbles first), MXFP6X2 blocks (49 bytes: scale
byte, 32 six-bit E2M3 digits hi, 32 lo; the value is 2^(e - 127) (hi + lo / 16)), and the routing rules of
qmm_moe_route_scored. Written from the formats: codes are found by comparing with every code, not by rounding.
"""
from __future__ import annotations

import math

import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
E2M3 = np.array([m / 8 for m in range(8)] + [2.0 ** (e - 1) * (1 + m / 8) for e in (1, 2, 3) for m in range(8)])


def nearest(t: np.ndarray, grid: np.ndarray) -> np.ndarray:
    """Index of the grid value nearest |t|, ties to the even index (the even mantissa); past the end: the last."""
    a = np.abs(np.asarray(t, dtype=np.float64))
    hi = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
    dl, dh = a - grid[hi - 1], grid[hi] - a
    return np.where((dl < dh) | ((dl == dh) & ((hi - 1) % 2 == 0)), hi - 1, hi)


def scale_byte(block_max: np.ndarray, grid: np.ndarray, least: int) -> np.ndarray:
    """The smallest scale byte at which the largest magnitude does not round past the grid's last value, where the
    grid is continued by its own step; 255 for an infinity or a NaN, `least` (or 0) for a block of zeros."""
    top, step = grid[-1], grid[-1] - grid[-2]
    out = np.empty(block_max.shape, dtype=np.int64)
    for i, v in np.ndenumerate(np.asarray(block_max, dtype=np.float64)):
        if not math.isfinite(v):
            out[i] = 255
            continue
        e = least
        if v > 0:
            e = max(least, math.frexp(v)[1] + 127 - 5)
            # the midpoint after `top` rounds away from it where the last code is odd
            odd = (len(grid) - 1) % 2 == 1
            while v / 2.0 ** (e - 127) > top + step / 2 or (odd and v / 2.0 ** (e - 127) == top + step / 2):
                e += 1
        out[i] = e
    return out


def _blocks(x):
    x = np.asarray(x, dtype=np.float64)
    return x.reshape(x.shape[0], -1, 32)


def to_mxfp4(w) -> np.ndarray:
    """GGML bytes (uint8 [n, k / 32, 17]) of dense rows."""
    b = _blocks(w)
    with np.errstate(invalid="ignore", over="ignore"):
        e = scale_byte(np.where(np.isnan(b).any(-1), np.inf, np.abs(b).max(-1)), E2M1, 0)
    t = np.where((e == 255)[..., None], 0.0, b) / 2.0 ** np.where(e == 255, 0, e - 127)[..., None]
    code = nearest(t, E2M1) + 8 * np.signbit(t)
    code = code.astype(np.uint8)
    return np.concatenate([e[..., None].astype(np.uint8), code[..., :16] | code[..., 16:] << 4], -1)


def from_mxfp4(blocks) -> np.ndarray:
    """f64 values [n, k] of MXFP4 blocks (NaN under scale byte 255)."""
    blocks = np.asarray(blocks, dtype=np.uint8)
    q = np.concatenate([blocks[..., 1:] & 15, blocks[..., 1:] >> 4], -1).astype(np.int64)
    v = E2M1[q & 7] * np.where(q & 8, -1.0, 1.0)
    e = blocks[..., :1].astype(np.int64)
    v = np.where(e == 255, np.nan, v * 2.0 ** (e - 127.0))
    return v.reshape(v.shape[0], -1)


def digits(x):
    """(scale bytes [m, k / 32], hi codes, lo codes [m, k / 32, 32]) of dense rows."""
    b = _blocks(x)
    with np.errstate(invalid="ignore", over="ignore"):
        e = scale_byte(np.where(np.isnan(b).any(-1), np.inf, np.abs(b).max(-1)), E2M3, 4)
    t = np.where((e == 255)[..., None], 0.0, b) / 2.0 ** np.where(e == 255, 0, e - 127)[..., None]
    hi = nearest(t, E2M3)
    rest = 16 * (t - E2M3[hi] * np.where(np.signbit(t), -1, 1))
    lo = nearest(rest, E2M3)
    return e, hi + 32 * np.signbit(t), lo + 32 * np.signbit(rest)


def to_mxfp6x2(x) -> np.ndarray:
    """Bytes (uint8 [m, k / 32, 49]) of dense rows; value j of a digit is bits 6 j .. 6 j + 5 of its 24 bytes."""
    e, hi, lo = digits(x)

    def pack(c):
        bits = (c[..., None] >> np.arange(6)) & 1
        return np.packbits(bits.reshape(*c.shape[:-1], 192).astype(np.uint8), axis=-1, bitorder="little")

    return np.concatenate([e[..., None].astype(np.uint8), pack(hi), pack(lo)], -1)


def digit_values(x) -> np.ndarray:
    """The f64 values a product takes for x: two digits under the block's scale."""
    e, hi, lo = digits(x)

    def val(c):
        return E2M3[c & 31] * np.where(c & 32, -1.0, 1.0)

    v = (val(hi) + val(lo) / 16) * 2.0 ** (np.where(e == 255, 127, e) - 127.0)[..., None]
    return np.where((e == 255)[..., None], np.nan, v).reshape(np.asarray(x).shape)


def product(x, blocks):
    """(x . W^T over the digit values, the sum of the terms' magnitudes), both f64 [m, n]."""
    xv, w = digit_values(x), from_mxfp4(blocks)
    return xv @ w.T, np.abs(xv) @ np.abs(w).T


def route(logits, k, score="softmax", bias=None, groups=1, topk_groups=None, group_top=1, renormalize=True, scale=1.0):
    """Per token: (experts in increasing order, weights), from the rules in 64 bits."""
    logits = np.asarray(logits, dtype=np.float64)
    n = logits.shape[1]
    size = n // groups
    topk_groups = groups if topk_groups is None else topk_groups
    experts, weights = [], []
    for row in logits:
        row = [-math.inf if math.isnan(v) else min(v, float(np.finfo(np.float32).max)) for v in row]
        if score == "softmax":
            m = max(row)
            p = [0.0 if m == -math.inf else math.exp(v - m) for v in row]
            z = math.fsum(p)
            s = [v / z if z > 0 else 0.0 for v in p]
        else:
            s = [0.0 if v < -700 else 1 / (1 + math.exp(-v)) for v in row]
        c = list(s)
        if bias is not None:
            c = [a + float(b) for a, b in zip(s, bias)]
            c = [-1e300 if math.isnan(v) else min(max(v, -1e300), 1e300) for v in c]
        gs = [sum(sorted(c[g * size:(g + 1) * size])[-group_top:]) for g in range(groups)]
        kept = set(sorted(range(groups), key=lambda g: (-gs[g], g))[:topk_groups])
        ids = sorted(sorted((e for e in range(n) if e // size in kept), key=lambda e: (-c[e], e))[:k])
        z = math.fsum(s[e] for e in ids)
        w = [s[e] / z if z > 0 else 0.0 for e in ids] if renormalize else [s[e] for e in ids]
        experts.append(ids)
        weights.append([v * float(np.float32(scale)) for v in w])
    return experts, weights


def lists(experts, weights, n):
    """counts, offsets, pair_token, pair_weight, token_pairs of qmm_moe_route for those selections."""
    pairs = sorted((e, t, w) for t, (ids, ws) in enumerate(zip(experts, weights)) for e, w in zip(ids, ws))
    counts = np.bincount([p[0] for p in pairs], minlength=n)
    place = {(e, t): i for i, (e, t, _) in enumerate(pairs)}
    return (counts, np.concatenate([[0], np.cumsum(counts)]), np.array([p[1] for p in pairs]),
            np.array([p[2] for p in pairs]),
            np.array([place[(e, t)] for t, ids in enumerate(experts) for e in ids]))
