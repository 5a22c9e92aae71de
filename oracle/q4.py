"""A page pool of 4-bit codes, packed rotated rows and verified drafts, in
float64 NumPy (no counterpart in the reference, which keeps one float cache
and decodes one token per sequence; the rotation is its _rope_norm /
_rope_neox, kernels.py:783-817): each written from its definition."""

from __future__ import annotations

import numpy as np

GROUP = 32


def half(x):
    """float16 of float64 numbers, through float32."""
    with np.errstate(over="ignore", under="ignore"):
        return np.asarray(x, dtype=np.float64).astype(np.float32).astype(np.float16)


def rotate(x, positions, rotary, style, base, scale=1.0):
    """``x [T, H, D]`` with its first ``rotary`` channels turned."""
    x = np.array(x, dtype=np.float64)
    out, half_ = x.copy(), rotary // 2
    for p in range(half_):
        a, b = (2 * p, 2 * p + 1) if style == "norm" else (p, p + half_)
        angle = np.asarray(positions, dtype=np.float64) * (scale * base ** (-2.0 * p / rotary))
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., a] * s + x[..., b] * c
    return out


def encode(x):
    """``(codes [..., D] uint8, steps, least values [..., D / 32] float16)``."""
    x = np.asarray(x, dtype=np.float64)
    g = x.reshape(x.shape[:-1] + (x.shape[-1] // GROUP, GROUP))
    fine = np.isfinite(g).all(-1)
    g = np.where(fine[..., None], g, 0.0)
    least = half(np.clip(g.min(-1), -65504.0, 65504.0))
    step = half(np.clip((g.max(-1) - least.astype(np.float64)) / 15.0, 0.0, 65504.0))
    d, m = step.astype(np.float64)[..., None], least.astype(np.float64)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        codes = np.where(d > 0.0, np.clip(np.rint((g - m) / d), 0.0, 15.0), 0.0)
    codes = np.where(fine[..., None], codes, 0.0)
    least = np.where(fine, least, np.float16(np.nan))
    step = np.where(fine, step, np.float16(0.0))
    return codes.astype(np.uint8).reshape(x.shape), step, least


def decode(codes, step, least):
    """The float32 numbers that codes stand for (one rounding)."""
    g = codes.reshape(codes.shape[:-1] + (codes.shape[-1] // GROUP, GROUP)).astype(np.float64)
    x = g * step.astype(np.float64)[..., None] + least.astype(np.float64)[..., None]
    return x.reshape(codes.shape).astype(np.float32)


def empty_pool(pages, heads, page, dim):
    return (np.zeros((pages, heads, page, dim // 2), np.uint8),
            np.zeros((pages, heads, 2, dim // GROUP, page), np.float16))


def put(pool, slots, x):
    """Rows ``x [T, H, D]`` at pool rows ``slots``; others are not stored."""
    data, scales = pool
    pages, _, page, _ = data.shape
    codes, step, least = encode(x)
    for t, slot in enumerate(slots):
        if 0 <= slot < pages * page:
            at, row = divmod(int(slot), page)
            data[at, :, row] = codes[t, :, 0::2] | (codes[t, :, 1::2] << 4)
            scales[at, :, 0, :, row] = step[t]
            scales[at, :, 1, :, row] = least[t]


def get(pool, slots):
    """float32 ``[T, H, D]`` of pool rows; zeros for a slot outside."""
    data, scales = pool
    pages, heads, page, width = data.shape
    out = np.zeros((len(slots), heads, 2 * width), np.float32)
    for t, slot in enumerate(slots):
        if 0 <= slot < pages * page:
            at, row = divmod(int(slot), page)
            codes = np.stack([data[at, :, row] & 15, data[at, :, row] >> 4], -1)
            out[t] = decode(codes.reshape(heads, -1), scales[at, :, 0, :, row],
                            scales[at, :, 1, :, row])
    return out


def gross(pool, slots):
    """float64 ``|least| + step * code`` of pool rows: what the two parts of a
    number amount to before their sum."""
    data, scales = pool
    out = get((data, np.abs(scales)), slots)
    return out.astype(np.float64)


def attend(q, k, v, prefix, length, count, scale, parts=None):
    """One sequence: ``q [N, Hq, D]`` over its rows ``k, v [R, Hkv, D]``.
    Token i < count whose row ``prefix + i`` lies below ``length`` sees the
    rows up to and with it.  Returns ``(out, weight)``: the result and
    ``sum p parts / sum p`` (``parts``: ``|v|``), which bounds what roundings
    of p do to it."""
    n, hq, d = q.shape
    hkv = k.shape[1]
    out, weight = np.zeros((n, hq, d)), np.zeros((n, hq, d))
    parts = np.abs(v) if parts is None else parts
    prefix = min(max(prefix, 0), length)
    for i in range(n):
        if i >= count or prefix + i >= length:
            continue
        for h in range(hq):
            g = h // (hq // hkv)
            kk, vv = (x[:prefix + i + 1, g].astype(np.float64) for x in (k, v))
            with np.errstate(invalid="ignore", over="ignore"):
                s = (kk @ q[i, h].astype(np.float64)) * scale
                p = np.exp(s - s.max())
                p = p / p.sum()
                out[i, h], weight[i, h] = p @ vv, p @ parts[:prefix + i + 1, g]
    return out, weight


def verify(tokens, target, uniforms, parents=None, draft=None, count=None):
    """One sequence: ``(path, new tokens)`` as lists, from the definition."""
    n, vocab = target.shape
    count = n if count is None else min(max(count, 0), n)
    if count == 0:
        return [], []

    def weights(row):
        with np.errstate(invalid="ignore"):
            row = np.asarray(row, dtype=np.float64)
            return np.where((row > 0.0) & np.isfinite(row), row, 0.0)

    up = [i - 1 if parents is None else int(parents[i]) for i in range(n)]
    u = [float(x) for x in uniforms]
    path, new, at = [0], [], 0
    while True:
        p = weights(target[at])
        q = None if draft is None else weights(draft[at])
        r, z, tried, moved = p, 1.0, 0, False
        for i in range(at + 1, count):
            if up[i] != at:
                continue
            x = int(tokens[i])
            inside = 0 <= x < vocab
            w = r[x] if inside else 0.0
            by = (q[x] if inside else 0.0) if q is not None else 1.0
            if u[i] * by * z < w:
                path.append(i)
                new.append(x)
                at, moved = i, True
                break
            tried += 1
            if q is not None:
                r = np.maximum(r - z * q, 0.0)
                z = r.sum()
            elif inside:
                r = r.copy()
                z -= r[x]
                r[x] = 0.0
        if moved:
            continue
        if not r.sum() > 0.0:
            r = p
        if not r.sum() > 0.0:
            return path, new + [-1]
        sums = np.cumsum(r)
        t = u[0] * sums[-1]
        t = t if t > 0.0 else 0.0
        over = np.flatnonzero((sums > t) & (r > 0.0))
        return path, new + [int(over[0]) if over.size else int(np.flatnonzero(r > 0.0)[-1])]
