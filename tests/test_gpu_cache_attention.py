"""CacheAttention against attention in 64 bits over the dequantized cache: head
sizes, pages and groups, one token and prompts, ragged mixtures, windows and
sinks, sequences that are split and joined, rows that see nothing, pages that
do not exist, NaN and infinite values where the masks hide them, strides,
streams and graphs."""
from __future__ import annotations

import numpy as np
import pytest

import datagen as dg
import decoder_ref as ref
import nnops_amd as na
from gpu_util import dev, host, pitched, announce

pytestmark = pytest.mark.gpu


def _cache(seqs, tokens, heads, page, d, seed=1, spare=2):
    """codes and scales (numpy), pages shuffled, and the table."""
    per = max(1, -(-tokens // page))
    n = seqs * per + spare
    kc, vc = dg.ints(seed, (n, heads, page, d), -127, 127), dg.ints(seed + 1, (n, heads, d, page), -127, 127)
    ks = (0.01 * np.exp(0.5 * dg.normal(seed + 2, (n, heads)))).astype(np.float32)
    vs = (0.02 * np.exp(0.7 * dg.normal(seed + 3, (n, heads)))).astype(np.float32)
    table = np.argsort(dg.unit(seed + 4, n))[:seqs * per].reshape(seqs, per).astype(np.int32)
    return kc, vc, ks, vs, table


def _run(q, cache, lens, rows, *, ragged, window=0, sinks=0, scale=0.0, pad=0, stream=None, workspace=None):
    import torch
    kc, vc, ks, vs, table = cache
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    dq = pitched(q, q.shape[1] + pad)
    out = pitched(np.full(q.shape, 7, q.dtype), q.shape[1] + 2 * pad)
    ins = [na.tensor(dq)] + [na.tensor(dev(x)) for x in (kc, vc, ks, vs, table, np.array(lens, np.int32))]
    ins += [na.tensor(dev(starts))] if ragged else []
    op = na.CacheAttention(window=window, sinks=sinks, scale=scale)
    outs = [na.tensor(out)]
    assert op.validate(ins, outs) == na.OK
    assert op.compute(outs, ins, stream=stream, workspace=workspace) == na.OK
    torch.cuda.synchronize()
    return host(out)


def _check(q, cache, lens, rows, *, window=0, sinks=0, scale=0.0, **kw):
    got = _run(q, cache, lens, rows, window=window, sinks=sinks, scale=scale, **kw).astype(np.float64)
    want, weight, spread = ref.attention(q, *cache, lens, rows, window=window, sinks=sinks,
                                         scale=scale or None)
    tol = ref.attention_tolerance(q.dtype == np.float16, want, weight, spread, cache[3])
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    worst = np.max((abs(got - want) / tol)[ok]) if ok.any() else 0.0
    assert worst <= 1.0, worst
    return got


def _q(seed, t, width, f16):
    return dg.normal(seed, (t, width)).astype(np.float16 if f16 else np.float32)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("d,page,heads,group", [(128, 64, 2, 4), (128, 16, 1, 1), (64, 32, 2, 8), (80, 16, 2, 5),
                                                (96, 128, 1, 16), (256, 64, 1, 2), (16, 256, 3, 1), (112, 64, 2, 7),
                                                (64, 16, 1, 71), (192, 32, 1, 3)])
def test_single_tokens(d, page, heads, group, f16):
    """One query each: lengths of one, around pages and tiles of 64."""
    announce(f"attention d={d} page={page} heads={heads} group={group} f16={f16}")
    lens = [1, 15, 16, 17, 63, 64, 65, 300]
    cache = _cache(len(lens), 300, heads, page, d)
    q = _q(3, len(lens), heads * group * d, f16)
    rows = [1] * len(lens)
    a = _check(q, cache, lens, rows, ragged=False)
    b = _check(q, cache, lens, rows, ragged=True, pad=3)
    assert np.array_equal(a, b)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("d,page,heads,group", [(128, 16, 1, 4), (64, 64, 2, 1), (80, 128, 1, 3), (256, 32, 1, 1)])
def test_prompts(d, page, heads, group, f16):
    """Ragged prompts behind prefixes of different lengths, a sequence without
    rows, a whole prompt, a single token."""
    announce(f"attention prompts d={d} page={page} group={group} f16={f16}")
    lens, rows = [130, 70, 9, 200, 64], [130, 5, 0, 1, 64]
    cache = _cache(len(lens), 200, heads, page, d)
    _check(_q(4, sum(rows), heads * group * d, f16), cache, lens, rows, ragged=True)
    # as many rows each
    _check(_q(5, 5 * 9, heads * group * d, f16), cache, lens, [9] * 5, ragged=False, pad=5)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (64, 0), (100, 70), (100, 200), (300, 5),
                                          (1 << 40, 3), (7, 1 << 40)])
def test_windows(window, sinks, f16):
    announce(f"attention window={window} sinks={sinks} f16={f16}")
    heads, group, d, page = 2, 3, 64, 16
    lens, rows = [400, 1, 333, 90], [1, 1, 70, 90]
    cache = _cache(4, 400, heads, page, d)
    _check(_q(6, sum(rows), heads * group * d, f16), cache, lens, rows, ragged=True, window=window, sinks=sinks)


@pytest.mark.parametrize("tokens,page,group,n", [(5000, 64, 4, 1), (5000, 16, 1, 1), (3001, 128, 8, 3), (2000, 32, 2, 40)])
def test_long(tokens, page, group, n):
    """Long sequences, split over workgroups and joined, beside short ones."""
    announce(f"attention long {tokens} page={page} group={group} n={n}")
    heads, d = 2, 64
    lens = [tokens, n, 900]
    cache = _cache(3, tokens, heads, page, d)
    q = _q(7, 3 * n, heads * group * d, True)
    a = _check(q, cache, lens, [n] * 3, ragged=False)
    b = _check(q, cache, lens, [n] * 3, ragged=True)
    assert np.max(abs(a - b)) <= 2.0 ** -9 * np.max(abs(a))
    _check(q.astype(np.float32), cache, lens, [n] * 3, ragged=True, window=1500, sinks=100)


# Calls with rows enough for the tiles that share their codes: at the mean more
# than 256 rows (tokens x heads of a group) a sequence of ragged calls, 96 of
# others, and 128 full tiles or more, of 256 rows or 128 (by type and head size;
# equal rows also where they fill no more).
TILES = [(128, 64, 16, 9, True), (128, 16, 16, 10, True), (64, 128, 20, 9, True), (80, 32, 16, 11, True),
         (112, 256, 16, 9, True), (16, 16, 20, 9, True), (256, 64, 16, 9, True), (192, 128, 16, 10, True),
         (128, 64, 16, 9, False), (96, 16, 16, 10, False), (64, 64, 16, 9, False), (48, 32, 16, 11, False), (32, 16, 16, 9, False)]


def _mixed(total):
    """Eight sequences, ragged: an empty one, one token, a whole prompt, rows
    behind prefixes that end inside pages and tiles."""
    lens, rows = [130, 70, 9, 200, 64, 33, 600, 1], [33, 70, 0, 40, 64, 33, 12, 1]
    if total > 300:
        rows[0], rows[3], rows[6] = 130, 101, 80
    return lens, rows


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("d,page,heads,group,f16", TILES)
def test_tiles(d, page, heads, group, f16, many):
    announce(f"attention tiles d={d} page={page} heads={heads} group={group} f16={f16} many={many}")
    lens, rows = _mixed(400 if many else 200)
    cache = _cache(len(lens), 600, heads, page, d)
    _check(_q(21, sum(rows), heads * group * d, f16), cache, lens, rows, ragged=True, pad=8 if many else 1)


@pytest.mark.parametrize("n", [13, 34])
@pytest.mark.parametrize("d,page,heads,group,f16", TILES)
def test_tiles_of_equal_rows(d, page, heads, group, f16, n):
    """As many rows each, without starts; more rows than tokens among them."""
    announce(f"attention equal tiles d={d} page={page} heads={heads} group={group} f16={f16} n={n}")
    lens = [34, 12, 0, 64, 65, 300, 511, 513, 40]
    cache = _cache(len(lens), 520, heads, page, d)
    q = _q(22, n * len(lens), heads * group * d, f16)
    got = _check(q, cache, lens, [n] * len(lens), ragged=False)
    assert np.all(got[n:2 * n - 12] == 0) and np.all(got[2 * n:3 * n] == 0)


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (64, 0), (100, 70), (300, 5), (7, 1 << 40)])
@pytest.mark.parametrize("page,f16", [(16, True), (64, True), (128, False), (32, False)])
def test_windows_in_tiles(window, sinks, page, f16):
    announce(f"attention tiles window={window} sinks={sinks} page={page} f16={f16}")
    heads, group, d = 20, 7, 64
    lens, rows = _mixed(400)
    cache = _cache(len(lens), 600, heads, page, d)
    _check(_q(23, sum(rows), heads * group * d, f16), cache, lens, rows, ragged=True, window=window, sinks=sinks)


@pytest.mark.parametrize("page,f16", [(64, True), (16, True), (64, False)])
def test_tiles_that_are_split(page, f16):
    """Few tiles over a long sequence, so many splits that they are joined by a
    workgroup a row; beside one that has a single tile of tokens."""
    announce(f"attention split tiles page={page} f16={f16}")
    heads, group, d, n, tokens = 4, 4, 128, 26, 33000
    cache = _cache(2, tokens, heads, page, d)
    q = _q(24, 2 * n, heads * group * d, f16)
    _check(q, cache, [tokens, 50], [n, n], ragged=False)
    _check(q, cache, [tokens, 50], [n, n], ragged=False, window=20000, sinks=100)
    group = 11
    q = _q(28, 2 * n, heads * group * d, f16)
    _check(q, cache, [tokens, 50], [n, n], ragged=True)


@pytest.mark.parametrize("page,f16", [(64, True), (16, True), (128, False), (32, False)])
def test_hidden_values_do_not_show_in_tiles(page, f16):
    """The same bits whatever lies past the rows' positions or before their
    window; a page that exists nowhere, a NaN scale and a NaN query show in the
    rows and heads that see them alone."""
    announce(f"attention hidden in tiles page={page} f16={f16}")
    heads, group, d, n, seqs = 16, 4, 64, 40, 8
    lens = [4 * page + 7] + [300] * (seqs - 1)
    kc, vc, ks, vs, table = clean = _cache(seqs, 4 * page + 320, heads, page, d)
    q = _q(25, seqs * n, heads * group * d, f16)
    kw = dict(ragged=False)
    want = _check(q, clean, lens, [n] * seqs, **kw)
    table = table.copy()
    for b in range(seqs):
        table[b, -(-lens[b] // page):] = (-5, 1 << 30)[b % 2]
    assert np.array_equal(want, _run(q, (kc, vc, ks, vs, table), lens, [n] * seqs, **kw))
    # the last 7 tokens' page of the first sequence: a NaN in one head
    k2, v2 = ks.copy(), vs.copy()
    k2[table[0, 4], 3] = np.nan
    v2[table[0, 4], 5] = np.nan
    got = _run(q, (kc, vc, k2, v2, table), lens, [n] * seqs, **kw).reshape(-1, heads, group * d).astype(np.float64)
    hit = np.zeros(got.shape, bool)
    hit[n - 7:n, [3, 5]] = True
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], want.reshape(got.shape)[~hit])
    t2 = table.copy()
    t2[1, 299 // page] = 1 << 30
    got = _run(q, (kc, vc, ks, vs, t2), lens, [n] * seqs, **kw)
    first = max(0, 299 // page * page - (300 - n))          # the first row at or past the page
    assert np.isnan(got[n + first:2 * n]).all()
    assert np.array_equal(got[:n + first], want[:n + first]) and np.array_equal(got[2 * n:], want[2 * n:])
    q2 = q.copy()
    q2[n + 3, 5], q2[3 * n, d + 1] = np.nan, np.inf
    got = _run(q2, (kc, vc, ks, vs, table), lens, [n] * seqs, **kw)
    hit = np.zeros(got.shape, bool)
    hit[n + 3, :d], hit[3 * n, d:2 * d] = True, True
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], want[~hit])
    # a window that has moved past the first pages
    kw = dict(ragged=False, window=60)
    want = _run(q, clean, lens, [n] * seqs, **kw)
    past = (300 - n - 60) // page
    k2, v2, t2 = ks.copy(), vs.copy(), table.copy()
    if past:
        k2[table[1, :past]], v2[table[2, :past]], t2[3, 0] = np.nan, np.inf, -1
        assert np.array_equal(want, _run(q, (kc, vc, k2, v2, t2), lens, [n] * seqs, **kw))


# d, page, heads, group, sequences, rows of each, tokens of the longest, window, type, splits
FEW_SPLITS = [(64, 16, 1, 2, 3, 1, 640, 0, True, 3), (128, 64, 2, 4, 2, 2, 700, 0, True, 3), (256, 32, 1, 3, 2, 1, 300, 0, True, 2),
              (128, 128, 1, 16, 8, 8, 1000, 0, True, 4), (80, 16, 2, 8, 32, 2, 1900, 0, True, 8),
              (64, 32, 2, 16, 16, 2, 1500, 1000, True, 5), (64, 64, 1, 4, 2, 1, 300, 0, False, 2),
              (128, 16, 2, 8, 16, 4, 1100, 0, False, 5), (256, 256, 1, 4, 3, 1, 600, 0, False, 3)]


@pytest.mark.parametrize("d,page,heads,group,seqs,n,tokens,window,f16,splits", FEW_SPLITS)
def test_few_splits(d, page, heads, group, seqs, n, tokens, window, f16, splits):
    """Few splits, joined by lanes of a wave; sequences of one split, of none and
    of all beside one another."""
    announce(f"attention few splits d={d} page={page} seqs={seqs} n={n} tokens={tokens} f16={f16}")
    lens = [(tokens, n, 130, 300, tokens - 1, 0, 257, 700)[i % 8] for i in range(seqs)]
    lens = [min(x, tokens) for x in lens]
    cache = _cache(seqs, tokens, heads, page, d)
    q = _q(40, seqs * n, heads * group * d, f16)
    for ragged in (False, True):
        _check(q, cache, lens, [n] * seqs, ragged=ragged, window=window, pad=4 if ragged else 0)


@pytest.mark.parametrize("d,page,heads,group", [(128, 64, 2, 4), (64, 16, 2, 3), (96, 32, 1, 16), (256, 64, 1, 2)])
def test_weights_of_few_rows_hold_22_bits(d, page, heads, group):
    """f16 rows, a few tokens of nearly equal weight: rounding the weights to
    f16 would show (2^-12 of each, of results that cancel), the sum of two f16
    leaves the output's rounding and the scores'."""
    announce(f"attention weights d={d} page={page}")
    lens, rows = [2, 3, 5, 9, 17, 33, 70, 300], [1] * 8
    cache = _cache(8, 300, heads, page, d)
    for size in (0.01, 1.0):
        q = (size * dg.normal(41, (8, heads * group * d))).astype(np.float16)
        got = _run(q, cache, lens, rows, ragged=False).astype(np.float64)
        want, weight, spread = ref.attention(q, *cache, lens, rows)
        # scores: as the other tests have it; weights: two f16, whose smallest step
        # is 2^-30 of a weight that the running maximum stands for (64 there)
        exact = ref.attention_tolerance(False, want, weight, spread, cache[3])
        most = 127.0 * cache[3].max() * max(lens) * 2.0 ** -30
        tol = exact + most + 1.01 * 2.0 ** -11 * abs(want) + 2.0 ** -24
        worst = np.max(abs(got - want) / tol)
        assert worst <= 1.0, (size, worst)


@pytest.mark.parametrize("d,page,heads,group,n,f16", [(128, 64, 2, 4, 1, True), (64, 16, 2, 2, 1, False), (256, 32, 1, 2, 3, True),
                                                      (128, 128, 4, 4, 40, True), (64, 16, 4, 8, 40, True), (64, 64, 4, 8, 40, False),
                                                      (128, 32, 4, 4, 40, False)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 30)])
def test_wide_page_tables(d, page, heads, group, n, f16, window, sinks):
    """A page table with room for far more tokens than any sequence holds, its
    unused entries garbage: the split goes by what the rows look at (each
    sequence its own), the results as ever."""
    announce(f"attention wide table d={d} page={page} group={group} n={n} f16={f16} window={window}")
    lens = [777, 2048, n, 513, 3000]
    kc, vc, ks, vs, table = _cache(len(lens), 3000, heads, page, d)
    wide = np.full((len(lens), 131072 // page), -5, np.int32)
    wide[:, 1::2] = 1 << 30
    for b, length in enumerate(lens):
        wide[b, :-(-length // page)] = table[b, :-(-length // page)]
    q = _q(42, len(lens) * n, heads * group * d, f16)
    for ragged in (False, True):
        _check(q, (kc, vc, ks, vs, wide), lens, [n] * len(lens), ragged=ragged, window=window, sinks=sinks)


@pytest.mark.parametrize("seqs,longest", [(63, 62), (64, 0), (65, 64), (65, 63), (130, 129), (130, 70), (200, 100)])
@pytest.mark.parametrize("f16", [True, False])
def test_splits_of_many_sequences(seqs, longest, f16):
    """More sequences than the 64 that a wave looks at in one step, the longest
    anywhere among them (or one without rows, which does not count)."""
    announce(f"attention splits of {seqs} sequences, longest {longest} f16={f16}")
    heads, group, d, page, tokens = 1, 3, 64, 32, 1500
    lens = 1 + dg.ints(43, (seqs,), 0, 119).astype(np.int64)
    lens[longest], lens[seqs // 3] = tokens, 1300
    kc, vc, ks, vs, table = _cache(seqs, tokens, heads, page, d)
    wide = np.full((seqs, 4 * table.shape[1]), -1, np.int32)
    wide[:, :table.shape[1]] = table
    cache = (kc, vc, ks, vs, wide)
    q = _q(44, 2 * seqs, group * d, f16)
    for ragged in (False, True):
        _check(q, cache, lens, [2] * seqs, ragged=ragged)
    rows = [0 if i == longest else 1 + i % 3 for i in range(seqs)]
    _check(_q(45, sum(rows), group * d, f16), cache, lens, rows, ragged=True)


def test_scales_far_apart():
    """Pages whose value scales differ by powers of ten, pages of zeros, the
    smallest scale; a scale of 0 reads as zeros."""
    heads, d, page, n = 1, 64, 16, 200
    for f16 in (True, False):
        announce(f"attention scales far apart f16={f16}")
        kc, vc, ks, vs, table = _cache(1, n, heads, page, d)
        vs[table[0], 0] = (10.0 ** (np.arange(table.shape[1]) % 7 - 4.0)).astype(np.float32)
        vs[table[0, 2], 0] = ref.LEAST_SCALE
        vs[table[0, 3], 0] = 0
        vc[table[0, 2]] = 0
        ks[table[0, 4], 0] = 0
        cache = (kc, vc, ks, vs, table)
        _check(_q(8, 3, 2 * d, f16), cache, [n], [3], ragged=False)
        # nothing but zeros
        vs[:], vc[:] = ref.LEAST_SCALE, 0
        assert np.all(_run(_q(9, 1, d, f16), cache, [n], [1], ragged=False) == 0)


def test_sharp_and_flat():
    """Scores of hundreds (one token takes all) and of nothing (an average), rows
    far from 1, a scale of the caller's."""
    heads, d, page, n = 2, 128, 64, 500
    cache = _cache(1, n, heads, page, d)
    for f16 in (True, False):
        for size in (60.0, 1e-4, 0.0) if f16 else (60.0, 1e-30, 0.0, 1e30):
            announce(f"attention size {size} f16={f16}")
            q = (size * dg.normal(10, (2, heads * d))).astype(np.float16 if f16 else np.float32)
            _check(q, cache, [n], [2], ragged=False, scale=0.0 if size < 1e20 else 1e-30)
        _check(_q(11, 2, heads * d, f16), cache, [n], [2], ragged=False, scale=0.3)


def test_hidden_values_do_not_show():
    """Pages past a row's position hold NaN scales and any codes; unwritten page
    table entries are garbage; a query that is NaN or infinite shows in its own
    row alone."""
    heads, d, page = 1, 64, 16
    for f16 in (True, False):
        announce(f"attention hidden f16={f16}")
        kc, vc, ks, vs, table = _cache(2, 160, heads, page, d)
        clean = [x.copy() for x in (kc, vc, ks, vs, table)]
        q = _q(12, 40, 2 * d, f16)
        lens, rows = [100, 40], [20, 20]
        want = _check(q, (kc, vc, ks, vs, table), lens, rows, ragged=False)
        # rows at positions 80 .. 99 of the first: its pages of tokens 96 on hold
        # a NaN from row 16 on; past the length the table holds garbage
        ks[table[0, 6]], vs[table[0, 6]] = np.nan, np.nan
        table[0, 7:], table[1, 3:] = -5, 1 << 30
        got = _run(q, (kc, vc, ks, vs, table), lens, rows, ragged=False).astype(np.float64)
        assert np.array_equal(got[:16], want[:16]) and np.array_equal(got[20:], want[20:])
        assert np.isnan(got[16:20]).all()
        # a window that has moved past them
        kc, vc, ks, vs, table = [x.copy() for x in clean]
        want = _run(q, (kc, vc, ks, vs, table), lens, rows, ragged=False, window=30)
        ks[table[0, :3]], vs[table[0, :3]] = np.nan, np.inf
        table[0, 0] = -1
        assert np.array_equal(want, _run(q, (kc, vc, ks, vs, table), lens, rows, ragged=False, window=30))
        q[3, 5], q[25, d + 1] = np.nan, np.inf
        want = _run(_q(12, 40, 2 * d, f16), tuple(clean), lens, rows, ragged=False).astype(np.float64)
        got = _run(q, tuple(clean), lens, rows, ragged=False).astype(np.float64)
        hit = np.zeros_like(got, bool)
        hit[3, :d], hit[25, d:] = True, True
        assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], want[~hit])


def test_rows_that_see_nothing():
    """More rows than tokens, sequences without tokens: zeros; a page number
    outside the cache: NaN in the rows that see it."""
    announce("attention empty rows")
    heads, d, page = 2, 32, 16
    cache = _cache(3, 64, heads, page, d)
    lens, rows = [4, 0, 64], [10, 3, 7]
    for f16 in (True, False):
        q = _q(13, 20, heads * d, f16)
        got = _check(q, cache, lens, rows, ragged=True)
        assert np.all(got[:6] == 0) and np.all(got[10:13] == 0) and np.all(np.any(got[6:10] != 0, axis=1))
        _check(q[:9], cache, [0, 0, 2], [3, 3, 3], ragged=False)
        table = cache[4].copy()
        table[2, 1] = 99999
        got = _check(q, cache[:4] + (table,), lens, rows, ragged=True)
        assert np.isnan(got[13:]).all()


def test_rows_without_a_sequence_stay():
    """Rows past the last start belong to nobody and are left as they are."""
    import torch
    announce("attention rows without a sequence")
    heads, d, page = 1, 32, 16
    cache = _cache(1, 40, heads, page, d)
    q = _q(14, 6, d, True)
    out = torch.full((6, d), 7.0, dtype=torch.float16, device="cuda")
    ins = [na.tensor(dev(x)) for x in (q,) + cache + (np.array([40], np.int32), np.array([1, 4], np.int32))]
    assert na.CacheAttention().compute([na.tensor(out)], ins) == na.OK
    torch.cuda.synchronize()
    want = _run(q[1:4], cache, [40], [3], ragged=False)
    assert np.array_equal(host(out)[1:4], want) and np.all(host(out)[[0, 4, 5]] == 7)


@pytest.mark.parametrize("seqs", [65, 130])
def test_many_sequences(seqs):
    announce(f"attention {seqs} sequences")
    heads, group, d, page = 1, 2, 32, 16
    cache = _cache(seqs, 90, heads, page, d)
    lens = 1 + dg.ints(15, (seqs,), 0, 80).astype(np.int64)
    rows = np.minimum(dg.ints(16, (seqs,), 0, 12), lens)
    _check(_q(17, int(rows.sum()), group * d, True), cache, lens, rows, ragged=True)


def test_cache_past_2_gib():
    import torch
    announce("attention past 2^32 bytes")
    page, heads, d = 128, 8, 128
    n = (1 << 32) // (heads * page * d) + 40
    small = _cache(1, 3 * page, heads, page, d, spare=0)
    kc, vc = (torch.zeros((n,) + x.shape[1:], dtype=torch.int8, device="cuda") for x in small[:2])
    ks, vs = (torch.zeros((n, heads), device="cuda") for _ in range(2))
    places = [n - 1, n // 2 + 1, n - 7]
    for i, at in enumerate(places):
        for big, x in zip((kc, vc, ks, vs), small):
            big[at] = torch.from_numpy(x[i]).cuda()
    table = np.array([[places[i] for i in small[4][0]]], np.int32)
    q = _q(18, 2, heads * 2 * d, True)
    out = torch.zeros((2, heads * 2 * d), dtype=torch.float16, device="cuda")
    op = na.CacheAttention()
    assert op.compute([na.tensor(out)], [na.tensor(dev(q))] + [na.tensor(x) for x in (kc, vc, ks, vs)] +
                      [na.tensor(dev(table)), na.tensor(dev(np.array([370], np.int32)))]) == na.OK
    torch.cuda.synchronize()
    assert np.array_equal(host(out), _run(q, small, [370], [2], ragged=False))


def test_streams_and_workspace():
    """A stream of the caller's, a workspace of the caller's that holds anything,
    the same bits every time; too little workspace is refused."""
    import ctypes
    import torch
    announce("attention stream and workspace")
    heads, d, page, n = 2, 128, 64, 3000
    cache = _cache(1, n, heads, page, d)
    q = _q(19, 1, heads * 4 * d, True)
    want = _run(q, cache, [n], [1], ragged=False)
    side = torch.cuda.Stream()
    ws = torch.full((64 << 20,), 0xFF, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for _ in range(3):
        assert np.array_equal(want, _run(q, cache, [n], [1], ragged=False, stream=side, workspace=ws))
    dq, t = dev(q), [dev(x) for x in cache] + [dev(np.array([n], np.int32))]
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    a = na.CacheAttentionArgs()
    a.q, a.out, a.rows, a.q_heads, a.ld_q, a.ld_out, a.f16 = dq.data_ptr(), out.data_ptr(), 1, 8, 1024, 1024, 1
    c = a.cache
    c.k, c.v, c.k_scale, c.v_scale, c.page_table, c.lengths = (x.data_ptr() for x in t)
    c.pages, c.heads, c.page_tokens, c.head_dim = cache[0].shape
    c.sequences, c.table_pages, c.ld_table = 1, cache[4].shape[1], cache[4].shape[1]
    lib = na.lib()
    need = lib.nnops_hip_cache_attention_workspace_size(ctypes.byref(a))
    assert need > 0
    assert lib.nnops_hip_cache_attention(ctypes.byref(a), ws.data_ptr(), need - 1, None) == na.NOT_INITIALIZED
    assert lib.nnops_hip_cache_attention(ctypes.byref(a), None, 0, None) == na.NOT_INITIALIZED
    torch.cuda.synchronize()
    assert np.all(host(out) == 7)
    assert lib.nnops_hip_cache_attention(ctypes.byref(a), ws.data_ptr(), need, None) == na.OK
    torch.cuda.synchronize()
    assert np.array_equal(host(out), want)


def test_graph_replays():
    """The operators of a step captured into one graph: the norm, the rotation,
    the cache's write and the attention, replayed with other inputs between."""
    import torch
    announce("decoder step under graph replay")
    heads, group, d, page, b = 2, 2, 64, 16, 3
    hq = heads * group
    width = (hq + 2 * heads) * d
    lens = np.array([40, 1, 700], np.int32)
    kc, vc, ks, vs, table = _cache(b, 700, heads, page, d)
    dt, dl = dev(table), dev(lens)
    cache = [dev(x) for x in (kc, vc, ks, vs)]
    keep = [x.clone() for x in cache]
    x = dev(dg.normal(20, (b, width)).astype(np.float16))
    w = dev(np.ones(width, np.float16))
    y = torch.zeros_like(x)
    out = torch.zeros((b, hq * d), dtype=torch.float16, device="cuda")
    pos = dev((lens - 1).astype(np.int32))
    tab = na.rotary_table(1000, d)
    norm, rot, wr, at = na.RmsNorm(), na.Rotary(head_dim=d), na.KvCacheWrite(), na.CacheAttention()
    qk = y[:, :(hq + heads) * d]
    pages = [na.tensor(z) for z in cache]
    where = [na.tensor(dt), na.tensor(dl)]
    ains, aouts = [na.tensor(y[:, :hq * d])] + pages + where, [na.tensor(out)]
    ws = torch.empty(max(1, at.workspace_size(ains, aouts)), dtype=torch.uint8, device="cuda")

    def step(s):
        assert norm.compute([na.tensor(y)], [na.tensor(x), na.tensor(w)], stream=s) == na.OK
        assert rot.compute([na.tensor(qk)], [na.tensor(qk), na.tensor(pos), na.tensor(tab)], stream=s) == na.OK
        assert wr.compute(pages, [na.tensor(y[:, hq * d:(hq + heads) * d]), na.tensor(y[:, (hq + heads) * d:])] + where,
                          stream=s) == na.OK
        assert at.compute(aouts, ains, stream=s, workspace=ws) == na.OK

    def reset():
        for z, k in zip(cache, keep):
            z.copy_(k)

    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        step(s)
    torch.cuda.synchronize()
    reset()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step(s)
    for r in range(4):
        x.copy_(dev(dg.normal(30 + r, (b, width)).astype(np.float16)))
        reset()
        step(None)
        torch.cuda.synchronize()
        want = [host(z).copy() for z in [out] + cache]
        reset()
        out.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, z in zip(want, [out] + cache):
            assert np.array_equal(a, host(z), equal_nan=True), r
