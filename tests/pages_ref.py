"""Plain forms of the operators for many continuations of one prompt: the page
tables, step by step as they are defined, and log probabilities in 64 bits."""
from __future__ import annotations

import numpy as np


def _held(table, lens, b, page, pages):
    """Page numbers of a sequence's cells, None where a cell holds no page."""
    tokens = min(max(int(lens[b]), 0), table.shape[1] * page)
    return [int(x) if 0 <= x < pages else None for x in table[b, :-(-tokens // page)]], tokens


def fork(table, lens, refs, parents, new, wide, page):
    """(table, lens, refs, copies, counts) of the children."""
    pages, n = len(refs), len(parents)
    refs = refs.astype(np.int64)
    out = np.full((n, wide), -1, np.int64)
    out_lens, copies = np.zeros(n, np.int64), np.full((n, 2), -1, np.int64)
    for b in range(len(lens)):
        for x in _held(table, lens, b, page, pages)[0]:
            if x is not None:
                refs[x] -= 1
    kept = np.zeros(n, np.int64)
    for i in range(n):
        mine, had = _held(table, lens, parents[i], page, pages) if 0 <= parents[i] < len(lens) else ([], 0)
        out_lens[i] = min(max(had + int(new[i]), 0), wide * page)
        kept[i] = min(had, out_lens[i])
        for c, x in enumerate(mine[:-(-int(kept[i]) // page)]):
            if x is not None:
                out[i, c] = x
                refs[x] += 1
    free = [x for x in range(pages) if refs[x] == 0]
    writers = {}
    for i in range(n):
        if out_lens[i] > kept[i] and kept[i] % page:
            writers.setdefault(out[i, kept[i] // page], []).append(i)
    keeps = {w[0] for x, w in writers.items() if x >= 0 and refs[x] <= len(w)}
    missing, give_up = 0, []
    for i in range(n):
        cells = list(range(-(-int(kept[i]) // page), -(-int(out_lens[i]) // page)))
        if out_lens[i] > kept[i] and kept[i] % page and i not in keeps:
            cells.insert(0, int(kept[i] // page))
        for c in cells:
            old, to = out[i, c], free.pop(0) if free else -1
            missing += to < 0
            out[i, c] = to
            if old >= 0:
                give_up.append(old)
                if to >= 0:
                    copies[i] = old, to
            if to >= 0:
                refs[to] = 1
    for x in give_up:
        refs[x] -= 1
    return out, out_lens, refs, copies, np.array([len(free), missing])


def compact(table, lens, refs, page):
    """(table, refs, copies, moved, counts)"""
    pages = len(refs)
    used = np.flatnonzero(refs)
    u = len(used)
    src, dst = used[used >= u], np.flatnonzero(refs[:u] == 0)
    moved = np.full(pages, -1, np.int64)
    moved[used] = used
    moved[src] = dst
    new_refs = np.zeros(pages, np.int64)
    new_refs[moved[used]] = refs[used]
    copies = np.full((pages // 2, 2), -1, np.int64)
    copies[:len(src), 0], copies[:len(src), 1] = src, dst
    out = np.full(table.shape, -1, np.int64)
    for b in range(len(lens)):
        for c, x in enumerate(_held(table, lens, b, page, pages)[0]):
            out[b, c] = -1 if x is None else moved[x]
    return out, new_refs, copies, moved, np.array([u, len(src)])


def holders(table, lens, page, pages):
    refs = np.zeros(pages, np.int64)
    for b in range(len(lens)):
        for x in _held(table, lens, b, page, pages)[0]:
            if x is not None:
                refs[x] += 1
    return refs


def log_probs(x, tokens, top):
    """(log_probs, entropy, top_tokens, top_log_probs), f64."""
    x = x.astype(np.float64)
    rows, vocab = x.shape
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(axis=1, keepdims=True)
        none = np.isneginf(m)
        z = x - np.where(none, 0.0, m)
        e = np.exp(z)
        s = e.sum(axis=1, keepdims=True)
        lp = z - np.log(s)
        entropy = np.where(none[:, 0], 0.0, -(np.where(e > 0, lp, 0.0) * e / s).sum(axis=1))
    lp = np.where(none, -np.inf, lp)
    bad = ~np.isfinite(x).all(axis=1) & (np.isnan(x) | np.isposinf(x)).any(axis=1)
    entropy[bad] = np.nan
    lp[bad] = np.nan
    at = np.clip(tokens, 0, vocab - 1)
    given = np.where(tokens < 0, 0.0, np.where(tokens < vocab, np.take_along_axis(lp, at, 1), np.nan))
    order = np.argsort(-np.where(np.isnan(x), 0, x), axis=1, kind="stable")[:, :top]
    best = np.take_along_axis(lp, order, 1)
    order = order.copy()
    order[bad] = -1
    return given, entropy, order, best


def log_probs_tolerance(x, lp, entropy):
    """How far log probabilities and entropies may be off: a logit's distance from
    the reference carries two roundings, a sum those of at most vocab / 256 + 64
    additions and of its terms (a hardware exponential: a few units), their
    logarithm another; a result is rounded once."""
    vocab, u = x.shape[1], 2.0 ** -24
    sums = (vocab / 256 + 64) * u
    size = np.where(np.isfinite(lp), np.abs(lp), 0.0)
    spread = np.log(vocab) + 2.0
    return 2.0 * sums + 4.0 * u * (size + spread), (sums + 8.0 * u) * (2.0 * spread + 4.0)
