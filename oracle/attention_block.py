"""64-bit definitions of the attention block's operators (rotary positions, head norms, prompt and tree
attention, cache compaction), one sequence and one row at a time, in numpy."""
from __future__ import annotations

import math

import numpy as np


def frequencies(rotary_dim, theta, scaling_type="", factor=1.0, original=0, beta_fast=32.0, beta_slow=1.0):
    i = np.arange(0, rotary_dim, 2, dtype=np.float64)
    f = theta ** (-i / rotary_dim)
    if scaling_type == "linear":
        return f / factor, 1.0
    if scaling_type == "ntk":
        return (theta * factor ** (rotary_dim / (rotary_dim - 2))) ** (-i / rotary_dim), 1.0
    if scaling_type == "yarn":
        keep = np.clip((original * f / (2 * math.pi) - beta_slow) / (beta_fast - beta_slow), 0, 1)
        return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def positions(seqstarts, start_pos, total):
    """-> positions [total] and which tokens belong to a sequence."""
    pos, live = np.zeros(total, np.int64), np.zeros(total, bool)
    for b in range(len(start_pos)):
        for t in range(seqstarts[b], min(seqstarts[b + 1], total)):
            pos[t], live[t] = start_pos[b] + t - seqstarts[b], True
    return pos, live


def rotary(x, pos, live, freq, factor, interleaved, weight=None, eps=0.0):
    """x [T, heads, D] -> the same shape in 64 bits."""
    x = x.astype(np.float64)
    y, r = x.copy(), 2 * len(freq)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)
    angle = pos.astype(np.float64)[:, None, None] * freq
    c, s = np.cos(angle) * factor, np.sin(angle) * factor
    out = y.copy()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    out[~live] = x[~live]
    return out


def attend_row(q, k, v, seen, scale, cap, bias):
    """One query [D] against k, v [L, D] -> (o [D], sum p |v| [D], largest sum |q||k| scale, largest |s|): the last
    three bound what the roundings of a kernel can do.  Keys that are not seen are not looked at."""
    zero = np.zeros(v.shape[1])
    if not seen.any():
        return zero, zero, 0.0, 0.0
    k, v = k[seen], v[seen]
    s = k @ q * scale
    if cap:
        s = cap * np.tanh(s / cap)
    if bias is not None:
        s = s + bias[seen]
    p = np.exp(s - s.max())
    p /= p.sum()
    return p @ v, p @ np.abs(v), float((np.abs(k) @ np.abs(q)).max() * scale), float(np.abs(s).max())


def prompt_attention(q, k, v, seqstarts, kvstarts, causal, scale, cap=0.0, slopes=None, prefix=None):
    """-> o, sum p |v|, per-row dot bound, per-row score bound; rows of no sequence stay zero."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    T, Hq, D = q.shape
    G = Hq // k.shape[1]
    o, A = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    dots, tops = np.zeros((T, Hq)), np.zeros((T, Hq))
    for b in range(len(seqstarts) - 1):
        n, L = seqstarts[b + 1] - seqstarts[b], kvstarts[b + 1] - kvstarts[b]
        j = np.arange(L)
        kk, vv = k[kvstarts[b]:kvstarts[b + 1]], v[kvstarts[b]:kvstarts[b + 1]]
        for i in range(n):
            at, t = i + L - n, seqstarts[b] + i
            seen = np.ones(L, bool)
            if causal:
                seen = j <= at
                if prefix is not None:
                    seen |= j < prefix[b]
            for h in range(Hq):
                bias = None if slopes is None else -float(slopes[h]) * np.abs(at - j)
                o[t, h], A[t, h], dots[t, h], tops[t, h] = attend_row(q[t, h], kk[:, h // G], vv[:, h // G], seen, scale,
                                                                      cap, bias)
    return o, A, dots, tops


def cache_rows(cache, layout):
    """A view [rows, layers, 2, heads, D] of the cache."""
    return cache.transpose([(0, 1, 2, 3, 4), (1, 0, 2, 3, 4), (2, 0, 1, 3, 4), (3, 0, 1, 2, 4)][layout])


def tree_attention(q, k, v, cache, layout, layer, seqstarts, cachestarts, start_pos, masks, scale, cap=0.0):
    """As prompt_attention(); stores the new keys and values into `cache`."""
    rows = cache_rows(cache, layout)[:, layer]
    q = q.astype(np.float64)
    T, Hq, D = q.shape
    G = Hq // k.shape[1]
    o, A = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    dots, tops = np.zeros((T, Hq)), np.zeros((T, Hq))
    for b in range(len(start_pos)):
        t0, n, L, c = seqstarts[b], seqstarts[b + 1] - seqstarts[b], start_pos[b], cachestarts[b]
        for i in range(n):
            if c + L + i < rows.shape[0]:
                rows[c + L + i, 0], rows[c + L + i, 1] = k[t0 + i], v[t0 + i]
        kk = np.concatenate([rows[c:c + L, 0], k[t0:t0 + n]]).astype(np.float64)
        vv = np.concatenate([rows[c:c + L, 1], v[t0:t0 + n]]).astype(np.float64)
        for i in range(n):
            bits = int(masks[t0 + i]) & (2 ** 64 - 1)
            seen = np.array([True] * L + [bool(bits >> j & 1) for j in range(n)])
            for h in range(Hq):
                o[t0 + i, h], A[t0 + i, h], dots[t0 + i, h], tops[t0 + i, h] = attend_row(
                    q[t0 + i, h], kk[:, h // G], vv[:, h // G], seen, scale, cap, None)
    return o, A, dots, tops


def compact_cache(cache, layout, cachestarts, start_pos, accept_starts, accept_index):
    rows = cache_rows(cache, layout)
    for b in range(len(start_pos)):
        base = cachestarts[b] + start_pos[b]
        old = rows.copy()
        for i, j in enumerate(accept_index[accept_starts[b]:accept_starts[b + 1]]):
            if j >= 0 and base + j < rows.shape[0] and base + i < rows.shape[0]:
                rows[base + i] = old[base + j]


def attention_tolerance(o, A, dots, tops, unit, unit_p, head_dim, keys, cap=0.0):
    """How far a kernel's result may be from `o`, element by element, from its roundings alone.

    unit: half a step of the output type; unit_p: of the type that the probabilities take for the second product.
    A score is a dot product of head_dim terms (each addition off by 2^-24 of at most sum |q||k|), scaled, capped
    (tanh built of one exponential and one reciprocal, 2^-20 of cap) and shifted in 32 bits (2^-22 of its size covers the
    conversions to base two): e.  exp(s) is then off by a factor 1 + e + 2^-21.  The weighted sum and the sum it is
    divided by each take that, and `keys` additions of 2^-24; the sum of |p v| bounds them all.  An output near nothing
    rounds to the type's smallest step."""
    e = (head_dim + 4) * 2.0 ** -24 * dots + 2.0 ** -22 * tops + 2.0 ** -20 * cap
    rel = unit_p + 2 * (e + 2.0 ** -21) + 2 * min(keys, 2048) * 2.0 ** -24
    return unit * np.abs(o) * (1 + unit) + rel[..., None] * A * (1 + 4 * unit_p) + 2.0 ** -24
