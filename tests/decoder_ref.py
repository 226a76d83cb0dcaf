"""Plain forms, in 64 bits, of the operators around the products of a decoder
layer: the norm, rotary positions, the paged 8-bit cache, attention over it."""
from __future__ import annotations

import math

import numpy as np

LEAST_SCALE = np.float32(2.0 ** -100)


def rms_norm(x, w, r=None, eps=1e-6):
    """(h, y, u): the sum, the norm and its numerator h w."""
    h = x.astype(np.float64) + (0.0 if r is None else r.astype(np.float64))
    u = h * w.astype(np.float64)
    return h, u / np.sqrt((h * h).mean(axis=1, keepdims=True) + eps), u


def rotary(x, pos, table, heads, d, rot, interleaved):
    """(y, size): the result, and |x_a c| + |x_b s| that its rounding goes by."""
    t = x.shape[0]
    x = x.astype(np.float64).reshape(t, heads, d)
    c = table[pos, :rot // 2].astype(np.float64)[:, None]
    s = table[pos, rot // 2:].astype(np.float64)[:, None]
    a = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    b = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    y, size = x.copy(), np.abs(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = abs(x[..., a] * c) + abs(x[..., b] * s)
    size[..., b] = abs(x[..., b] * c) + abs(x[..., a] * s)
    return y.reshape(t, -1), size.reshape(t, -1)


def kv_write(x, codes, scale, table, lens, rows):
    """The rows [t, heads * d] written into codes [pages, heads, page, d] and
    scale [pages, heads] (changed in place), with the f32 operations that the
    codes are defined by."""
    _, heads, page, d = codes.shape
    f32 = np.float32
    x = x.astype(f32).reshape(-1, heads, d)
    at = 0
    for b, (length, n) in enumerate(zip(lens, rows)):
        first = max(length - n, 0)
        mine = x[at + n - (length - first):at + n]
        at += n
        p = first
        while p < length:
            slot, end = p % page, min(length - p + p % page, page)
            new = mine[p - first:p - first + end - slot].transpose(1, 0, 2)      # [heads, tokens, d]
            pid = table[b][p // page]
            p += end - slot
            if not 0 <= pid < codes.shape[0]:
                continue
            for h in range(heads):
                old = scale[pid, h] if slot else f32(0)
                if not np.isfinite(new[h]).all() or np.isnan(old):
                    scale[pid, h] = np.nan
                    codes[pid, h, slot:end] = 0
                    continue
                s = max(old, f32(np.abs(new[h]).max()) * f32(f32(1) / f32(127)), LEAST_SCALE)
                if slot and s > old:
                    q = np.rint(codes[pid, h, :slot].astype(f32) * f32(old / s))
                    codes[pid, h, :slot] = np.clip(q, -127, 127).astype(np.int8)
                codes[pid, h, slot:end] = np.clip(np.rint(new[h] * f32(f32(1) / s)), -127, 127).astype(np.int8)
                scale[pid, h] = s


def kv_read(codes, scale, table, lens, rows):
    """The last rows[b] tokens of each sequence, f64 [t, heads * d]: absent ones
    0, of pages that do not exist NaN."""
    pages, heads, page, d = codes.shape
    out = []
    for b, (length, n) in enumerate(zip(lens, rows)):
        for p in range(length - n, length):
            if p < 0:
                out.append(np.zeros(heads * d))
                continue
            pid = table[b][p // page]
            if not 0 <= pid < pages:
                out.append(np.full(heads * d, np.nan))
                continue
            out.append((codes[pid, :, p % page].astype(np.float64) * scale[pid].astype(np.float64)[:, None]).ravel())
    return np.array(out).reshape(-1, heads * d)


def attention(q, kc, vc, ks, vs, table, lens, rows, *, scale=None, window=0, sinks=0):
    """(out, weight, spread): the result; sum p |v| / sum p, which the rounding
    of the probabilities goes by; and the largest of |score| + sum |q k|, which
    the scores' rounding goes by. kc [pages, heads, page, d], vc [pages, heads,
    d, page]."""
    pages, heads, page, d = kc.shape
    qh = q.shape[1] // d
    q = q.astype(np.float64).reshape(-1, qh, d)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out = np.zeros(q.shape)
    weight = np.zeros(q.shape)
    spread = 0.0
    at = 0
    for b, (length, n) in enumerate(zip(lens, rows)):
        ids = [table[b][i] for i in range(-(-length // page))]
        there = np.array([0 <= i < pages for i in ids], dtype=bool)
        ids = np.array([i if ok else 0 for i, ok in zip(ids, there)], dtype=np.int64)
        for h in range(heads):
            if length == 0:
                continue
            bad = np.where(there, 1.0, np.nan)[:, None, None]
            k = (kc[ids, h].astype(np.float64) * ks[ids, h].astype(np.float64)[:, None, None] * bad).reshape(-1, d)[:length]
            v = (vc[ids, h].astype(np.float64) * vs[ids, h].astype(np.float64)[:, None, None]) * bad
            v = v.transpose(0, 2, 1).reshape(-1, d)[:length]
            mine = slice(h * (qh // heads), (h + 1) * (qh // heads))
            size_k, size_v = abs(k), abs(v)
            for i in range(n):
                p = length - n + i
                if p < 0:
                    continue
                seen = slice(0, p + 1)
                if window:
                    j = np.arange(p + 1)
                    seen = np.flatnonzero((p - j < window) | (j < sinks))
                x = q[at + i, mine] @ k[seen].T * scale
                with np.errstate(invalid="ignore"):
                    e = np.exp(x - x.max(axis=1, keepdims=True))
                    e /= e.sum(axis=1, keepdims=True)
                    top = (abs(q[at + i, mine]) @ size_k[seen].T).max() * scale
                    out[at + i, mine] = e @ v[seen]
                    weight[at + i, mine] = e @ size_v[seen]
                spread = max(spread, 2.0 * top if np.isfinite(top) else 0.0)
        at += n
    return out.reshape(-1, qh * d), weight.reshape(-1, qh * d), spread


def attention_tolerance(f16, out, weight, spread, v_scale):
    """How far a result may be from the 64-bit one. A score x carries an error of
    a few roundings of what it is made of (its products, log2 of the value
    scale), so that a probability is off by the factor 1 + delta; the
    probabilities enter the product as f16 (f32 rows: as three bf16 parts, all
    their 24 bits); the result is rounded once."""
    logs = np.abs(np.log2(v_scale[np.isfinite(v_scale) & (v_scale > 0)])).max() if v_scale.size else 0.0
    delta = 4.0 * 2.0 ** -24 * (1.45 * spread + logs + 16.0) + 2.0 ** -20
    part = 2.0 ** -11 if f16 else 2.0 ** -21
    last = 2.0 ** -11 if f16 else 2.0 ** -23
    return (2.0 * delta + 1.01 * part) * weight + 1.01 * last * np.abs(out) + (2.0 ** -24 if f16 else 1e-38)
