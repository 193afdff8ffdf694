"""The attention layer's operators in 64 bits, from their definitions (include/halo_cuda_attention.h), on numpy arrays.

A cache is a dict: k, v uint8 [page][kv head][slot][dim]; k_scale, v_scale uint8 [page][kv head]; table int32 [seq][max_pages].
Rows: start (n_seq + 1 values) and length (n_seq values)."""
from __future__ import annotations

import math

import numpy as np


def e4m3_values() -> np.ndarray:
    v = np.zeros(256)
    for b in range(256):
        e, m = b >> 3 & 15, b & 7
        x = math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
        v[b] = math.nan if b & 127 == 127 else -x if b & 128 else x
    return v


VALUES = e4m3_values()
POSITIVE = VALUES[:127]  # 0 .. 448, rising


def e4m3_codes(x: np.ndarray) -> np.ndarray:
    """Nearest code, ties to the even one; beyond 448 saturated; NaN stays NaN.  Written from the list of values, not from the format's fields."""
    a = np.minimum(np.abs(np.asarray(x, np.float64)), 448.0)
    hi = np.searchsorted(POSITIVE, a, side="left").clip(0, 126)
    lo = (hi - 1).clip(0)
    up = POSITIVE[hi] - a < a - POSITIVE[lo]
    tie = (POSITIVE[hi] - a == a - POSITIVE[lo]) & (hi % 2 == 0)
    code = np.where(up | tie | (hi == 0), hi, lo)
    code = np.where(POSITIVE[hi] == a, hi, code).astype(np.uint8)
    code = code | np.where(np.signbit(x), 128, 0).astype(np.uint8)
    return np.where(np.isnan(x), np.uint8(127), code).astype(np.uint8)


def scale_of(byte: np.ndarray) -> np.ndarray:
    return np.exp2(np.clip(np.asarray(byte, np.int64), 87, 207) - 127.0)


def need_byte(top: float) -> int:
    e = -40
    while e < 80 and top > math.ldexp(448, e):
        e += 1
    return e + 127


def kv_write(cache: dict, k: np.ndarray, v: np.ndarray, start, length) -> bool:
    """Writes into the cache's arrays; True if a page number was out of range."""
    page_tokens, n_pages, bad = cache["k"].shape[2], cache["k"].shape[0], False
    for i, n in enumerate(length):
        rows = start[i + 1] - start[i]
        first = n - rows
        for index in range(max(first, 0) // page_tokens, -(-n // page_tokens)):
            begin, end = max(first, index * page_tokens), min(n, (index + 1) * page_tokens)
            if begin >= end:
                continue
            p, slot = int(cache["table"][i][index]), begin - index * page_tokens
            if not 0 <= p < n_pages:
                bad = True
                continue
            for name, x in (("k", k), ("v", v)):
                new = np.asarray(x[start[i] + begin - first:start[i] + end - first], np.float64)
                for h in range(new.shape[1]):
                    part = new[:, h]
                    finite = np.abs(part[np.isfinite(part)])
                    b = need_byte(finite.max() if finite.size else 0.0)
                    old = int(np.clip(cache[name + "_scale"][p, h], 87, 207))
                    if slot and old >= b:
                        b = old
                    if slot and old < b:
                        kept = VALUES[cache[name][p, h, :slot]]
                        cache[name][p, h, :slot] = e4m3_codes(kept * 2.0 ** (old - b))
                    cache[name][p, h, slot:slot + end - begin] = e4m3_codes(part * 2.0 ** (127 - b))
                    cache[name + "_scale"][p, h] = b
    return bad


def attention(q: np.ndarray, cache: dict, start, length, scale: float, causal: bool = True, window: int = 0, out: np.ndarray | None = None,
              floor: np.ndarray | None = None):
    """(out, sum of weights * |v|, largest sum of |q_d k_d| * |scale| of a seen token, number of seen tokens); rows of no sequence keep `out`.
    `floor` gets what the smallest weights may be off by.  A kernel holds weight * s_V as fp16 numbers (fp32 operands: as two, the second of the first's
    remainder) scaled so that the row's largest is at least 2^6.  fp16's smallest step is 2^-24, so a rounding is off by at most half a step, 2^-25,
    where the 2^-11 of attention_bound does not cover it: at most 2^-31 of the largest weight * s_V, for each token, times the code it multiplies."""
    n_pages, n_kv, page_tokens, dim = cache["k"].shape
    n_q = q.shape[1]
    g = n_q // n_kv
    y = np.zeros(q.shape) if out is None else np.array(out, np.float64)
    weight, top, count = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    for i, n in enumerate(length):
        lo, hi = start[i], start[i + 1]
        if lo == hi:
            continue
        t = np.arange(n)
        pages = np.asarray(cache["table"][i], np.int64)[t // page_tokens]
        good = (pages >= 0) & (pages < n_pages)
        at = np.where(good, pages, 0)
        pos = n - (hi - lo) + np.arange(hi - lo)
        seen = np.broadcast_to(good[None, :], (hi - lo, n)).copy()
        if causal:
            seen &= t[None, :] <= pos[:, None]
            if window:
                seen &= t[None, :] > pos[:, None] - window
        for h in range(n_kv):
            k = VALUES[cache["k"][at, h, t % page_tokens]] * scale_of(cache["k_scale"][at, h])[:, None]
            v = VALUES[cache["v"][at, h, t % page_tokens]] * scale_of(cache["v_scale"][at, h])[:, None]
            for r in range(hi - lo):
                m = seen[r]
                y[lo + r, h * g:h * g + g] = 0
                if not m.any():
                    continue
                qs = np.asarray(q[lo + r, h * g:h * g + g], np.float64)
                with np.errstate(invalid="ignore"):
                    x = qs @ k[m].T * scale
                    w = np.exp(x - x.max(axis=1, keepdims=True))
                    w /= w.sum(axis=1, keepdims=True)
                    y[lo + r, h * g:h * g + g] = w @ v[m]
                    weight[lo + r, h * g:h * g + g] = w @ np.abs(v[m])
                    if floor is not None:
                        s_v = scale_of(cache["v_scale"][at, h])[m]
                        floor[lo + r, h * g:h * g + g] = 2.0 ** -31 * (w * s_v).max(axis=1)[:, None] * np.abs(v[m] / s_v[:, None]).sum(axis=0)
                    top[lo + r, h * g:h * g + g] = (np.abs(qs) @ np.abs(k[m]).T * abs(scale)).max(axis=1)
                count[lo + r, h * g:h * g + g] = m.sum()
    return y, weight, top, count


def attention_bound(kind: str, dim: int, ref: np.ndarray, weight, top, count) -> np.ndarray:
    """What a kernel may be off by.  u = 2^-24.  A score is a sum of `dim` products in fp32 and two more roundings: off by at most
    (dim + 4) u top in any order, plus the rounding of q to two fp16 terms (2^-22 top) for fp32 operands; with the fp32 subtraction of the maximum and
    exp2 (2 ulp, and the ulp of an argument of up to 2 top log2 e: 4 u top) a weight's relative error is d = (dim + 16) u top + 4 * 2^-24 (+ 2^-22 top).
    16-bit types round the weights to 11 bits (2^-11), fp32 to two fp16 terms (2^-22).  Numerator and denominator are sums of `count` fp32 terms in
    blocks: (count + 32) u each.  Errors of weights enter twice (numerator and denominator).  Last, the output's own rounding: half a step."""
    u = 2.0 ** -24
    d = (dim + 16) * u * top + 4 * u + (2.0 ** -22 * top if kind == "f32" else 0)
    p = {"f32": 2.0 ** -22, "f16": 2.0 ** -11, "bf16": 2.0 ** -11}[kind]
    rel = 2 * d + p + 2 * (count + 32) * u
    step = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[kind]
    tiny = {"f32": 2.0 ** -126, "f16": 2.0 ** -25, "bf16": 2.0 ** -126}[kind]
    return rel[..., None] * weight * (1 + step) + step * np.abs(ref) + tiny


def rope_freqs(rot: int, base: float, scaling: str = "none", factor=1.0, original=0.0, fast=0.0, slow=0.0, pair_factors=None):
    """(radians per position, magnitude), from the definitions."""
    f, magnitude = [], 1.0
    if scaling == "base":
        base = base * factor ** (rot / (rot - 2))
    for j in range(rot // 2):
        w = base ** (-2.0 * j / rot)
        if scaling == "linear":
            w /= factor
        elif scaling == "factors":
            w /= pair_factors[j]
        elif scaling == "ramp":
            pair = lambda turns: rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot - 1)
            r = min(max((j - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            w = w / factor * r + w * (1 - r)
            magnitude = 0.1 * math.log(factor) + 1
        elif scaling == "bands":
            turns = original * w / (2 * math.pi)
            r = min(max((turns - slow) / (fast - slow), 0.0), 1.0)
            w = w / factor * (1 - r) + w * r
        f.append(w)
    return np.array(f), magnitude


def rope(x: np.ndarray, positions, freqs: np.ndarray, magnitude: float, interleaved: bool):
    n = len(freqs)
    y = np.array(x, np.float64)
    a = np.outer(np.asarray(positions, np.float64), freqs)[:, None, :]
    c, s = np.cos(a) * magnitude, np.sin(a) * magnitude
    i, j = (np.arange(0, 2 * n, 2), np.arange(1, 2 * n, 2)) if interleaved else (np.arange(n), np.arange(n, 2 * n))
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    return y
