"""PrefixAttention against attention in 64 bits over each sequence's own tokens:
groups of different sizes and prefixes, single tokens and ragged rows, rows inside
what is shared, sequences in no group, prefixes that end inside pages and tiles,
pages that do not exist, NaN, group starts out of order, strides, graphs. Where a
table has little room every sequence is looked at by itself: the tests widen theirs
so that what is shared is read once, and make the call with the narrow one too."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import datagen as dg
import decoder_ref as ref
import nnops_amd as na
from nnops_amd import _lib as L
from gpu_util import announce, dev, host, pitched

pytestmark = pytest.mark.gpu


def _cache(lens, groups, shared, heads, page, d, seed=1, spare=2, wide=0):
    """codes and scales (numpy), and a table whose groups' sequences hold the same
    pages as far as `shared` fills them."""
    per = [-(-n // page) for n in lens]
    n = sum(per) + spare
    kc, vc = dg.ints(seed, (n, heads, page, d), -127, 127), dg.ints(seed + 1, (n, heads, d, page), -127, 127)
    ks = (0.01 * np.exp(0.5 * dg.normal(seed + 2, (n, heads)))).astype(np.float32)
    vs = (0.02 * np.exp(0.7 * dg.normal(seed + 3, (n, heads)))).astype(np.float32)
    order = iter(np.argsort(dg.unit(seed + 4, n)))
    table = np.full((len(lens), max(max(per), 1) + wide), -1, np.int32)
    for i, p in enumerate(per):
        table[i, :p] = [next(order) for _ in range(p)]
    for g, s in enumerate(shared):
        a = groups[g]
        for b in range(a + 1, groups[g + 1]):
            k = max(0, min(s, lens[a], lens[b])) // page
            table[b, :k] = table[a, :k]
    return kc, vc, ks, vs, table


def _plan(heads, group, d, page, columns, rows, sequences, groups, f16, ragged):
    a = L.PrefixAttentionArgs(rows=rows, q_heads=heads * group, f16=int(f16), groups=groups)
    a.cache = L.KvPages(pages=1, heads=heads, page_tokens=page, head_dim=d, sequences=sequences, table_pages=columns,
                        row_starts=16 if ragged else None)
    p = L.PrefixAttentionPlan()
    assert na.lib().nnops_hip_prefix_attention_plan(C.byref(a), C.byref(p)) == na.OK
    return p


def _widened(q, cache, lens, groups, ragged):
    """The table with columns enough that what is shared is read once, which no number
    is where each sequence's rows (nearly) fill tiles, or groups are hardly more than one."""
    kc, table = cache[0], cache[4]
    _, heads, page, d = kc.shape
    columns, seqs, n = table.shape[1], len(lens), len(groups) - 1
    group = q.shape[1] // heads // d

    def plan(columns):
        return _plan(heads, group, d, page, columns, q.shape[0], seqs, n, q.dtype == np.float16, ragged)
    while plan(columns).shared_rows == 0 and columns * seqs < 2 ** 25:
        columns += columns // 4 + 1
    full = q.shape[0] * group > 64 * seqs or not ragged and q.shape[0] // seqs * group % 16 == 0
    assert plan(columns).shared_rows or full or 2 * n > seqs
    return np.pad(table, ((0, 0), (0, columns - table.shape[1])), constant_values=-1)


def _run(q, cache, lens, rows, groups, shared, *, ragged, pad=0, scale=0.0, stream=None, share=True):
    import torch
    kc, vc, ks, vs, table = cache
    if share and len(groups) - 1 in range(1, len(lens)):
        table = _widened(q, cache, lens, groups, ragged)
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    dq = pitched(q, q.shape[1] + pad)
    out = pitched(np.full(q.shape, 7, q.dtype), q.shape[1] + 2 * pad)
    ints = [np.array(x, np.int32) for x in (lens, groups, shared)]
    ins = [na.tensor(dq)] + [na.tensor(dev(x)) for x in [kc, vc, ks, vs, table] + ints]
    ins += [na.tensor(dev(starts))] if ragged else []
    op = na.PrefixAttention(scale=scale)
    outs = [na.tensor(out)]
    assert op.validate(ins, outs) == na.OK
    assert op.compute(outs, ins, stream=stream) == na.OK
    torch.cuda.synchronize()
    return host(out)


def _check(q, cache, lens, rows, groups, shared, *, scale=0.0, **kw):
    want, weight, spread = ref.attention(q, *cache, lens, rows, scale=scale or None)
    tol = ref.attention_tolerance(q.dtype == np.float16, want, weight, spread, cache[3])
    ok = ~np.isnan(want)
    for share in (False, True):
        got = _run(q, cache, lens, rows, groups, shared, scale=scale, share=share, **kw).astype(np.float64)
        assert np.array_equal(np.isnan(got), np.isnan(want)), share
        worst = np.max((abs(got - want) / tol)[ok]) if ok.any() else 0.0
        assert worst <= 1.0, (share, worst)
    return got


def _q(seed, t, width, f16):
    return dg.normal(seed, (t, width)).astype(np.float16 if f16 else np.float32)


SIZES = [(128, 64, 2, 4), (128, 16, 1, 1), (64, 32, 2, 8), (80, 16, 2, 5), (96, 128, 1, 16), (256, 64, 1, 2), (16, 256, 3, 1),
         (112, 64, 2, 7), (64, 16, 1, 71), (192, 32, 1, 3)]


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("d,page,heads,group", SIZES)
def test_single_tokens(d, page, heads, group, f16):
    """Two groups and a sequence in none; prefixes around tiles and pages."""
    announce(f"prefix d={d} page={page} heads={heads} group={group} f16={f16}")
    groups, shared = [1, 5, 8], [300, 130]
    lens = [70, 301, 364, 500, 333, 131, 257, 140]
    cache = _cache(lens, groups, shared, heads, page, d)
    q = _q(3, len(lens), heads * group * d, f16)
    a = _check(q, cache, lens, [1] * 8, groups, shared, ragged=False)
    b = _check(q, cache, lens, [1] * 8, groups, shared, ragged=True, pad=3)
    assert np.array_equal(a, b) or group >= 16             # (rows that nearly fill tiles: one of them by itself)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("d,page,heads,group", [(128, 64, 2, 4), (64, 16, 2, 3), (80, 128, 1, 5), (256, 64, 1, 2), (32, 32, 1, 8)])
def test_ragged_rows(d, page, heads, group, f16):
    """Rows of several tokens, of none, rows that lie inside what is shared (which
    is then not shared so far), a sequence that is a whole prompt."""
    announce(f"prefix ragged d={d} page={page} group={group} f16={f16}")
    groups, shared = [0, 4, 7], [512, 200]
    lens, rows = [600, 520, 513, 700, 200, 290, 256], [3, 1, 0, 80, 0, 33, 1]
    cache = _cache(lens, groups, shared, heads, page, d)
    _check(_q(4, sum(rows), heads * group * d, f16), cache, lens, rows, groups, shared, ragged=True, pad=2)
    # (the prompt's first row sees only itself: nothing is shared)
    rows = [3, 513, 0, 1, 200, 2, 1]
    lens[1] = 513
    _check(_q(5, sum(rows), heads * group * d, f16), cache, lens, rows, groups, shared, ragged=True)
    # the last rows: at the border of what is shared and one before
    lens = [513, 512, 575, 576, 64, 65, 128]
    cache = _cache(lens, groups, shared, heads, page, d)
    _check(_q(6, 7, heads * group * d, f16), cache, lens, [1] * 7, groups, shared, ragged=False)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("d,page,heads,group", [(128, 64, 2, 8), (128, 16, 2, 8), (64, 64, 2, 8), (64, 16, 4, 8), (256, 64, 1, 8),
                                                (96, 128, 1, 8), (192, 32, 1, 8), (256, 128, 2, 5)])
def test_tiles_of_many_rows(d, page, heads, group, f16):
    """Groups with rows enough for tiles of 128 and of 256 rows, several tiles. (The
    choice goes by the table's room: wide ones, of which the sequences fill little.)"""
    announce(f"prefix tiles d={d} page={page} heads={heads} f16={f16}")
    groups, shared = [0, 10], [640]
    lens = [640 + 7 * i + 9 for i in range(10)]
    wide = 2 ** 31 // (10 * heads * group * d * page)
    cache = _cache(lens, groups, shared, heads, page, d, wide=wide)
    columns = cache[4].shape[1]
    tiled = d <= 128 or (f16 and page >= 64)                   # (wider heads: f16, a tile in one page)
    for rows in ([1] * 10, [9, 1, 7, 0, 9, 5, 9, 9, 30, 2], [40] * 10):
        p = _plan(heads, group, d, page, columns, sum(rows), 10, 1, f16, True)
        many = 256 if d <= (128 if f16 else 64) and sum(rows) * group > 128 else 128
        assert p.shared_rows == (many if tiled and sum(rows) * group > 64 else 16)
        _check(_q(7, sum(rows), heads * group * d, f16), cache, lens, rows, groups, shared, ragged=True, pad=4)
        # the same rows in two groups and none, in nine, in as many as there are sequences
        for starts, of in (([0, 4, 9], [640, 500]), ([0, 2, 3, 4, 5, 6, 7, 8, 9, 10], [640] * 9), (list(range(11)), [640] * 10)):
            _check(_q(8, sum(rows), heads * group * d, f16), cache, lens, rows, starts, of, ragged=True)
    _check(_q(9, 20, heads * group * d, f16), cache, lens, [2] * 10, groups, shared, ragged=False)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("d,page,heads,group,members", [(128, 64, 8, 4, 70), (64, 16, 8, 1, 80), (80, 32, 8, 3, 66), (256, 64, 8, 4, 64)])
def test_own_tokens_join_the_parts(d, page, heads, group, members, f16):
    """Batches so large that own tokens are not split: where they are looked at, the
    parts are joined. More than 64 sequences: a kernel finds the plan first."""
    announce(f"prefix joined d={d} page={page} members={members} f16={f16}")
    groups, shared = [1, 41, members - 1], [320, 200]
    lens = [320 + 3 * (i % 20) + 9 for i in range(members)]
    wide = 2 ** 31 // (members * heads * group * d * page)
    cache = _cache(lens, groups, shared, heads, page, d, wide=wide)
    for rows, ragged in (([1] * members, False), ([i % 4 for i in range(members)], True), ([5] * members, True)):
        p = _plan(heads, group, d, page, cache[4].shape[1], sum(rows), members, 2, f16, ragged)
        if p.shared_rows != 16 and p.own_splits == 1 and p.own_rows == 16:
            assert p.join == 0 and p.launches == 2 + (members > 64)
        q = _q(9, sum(rows), heads * group * d, f16)
        a = _check(q, cache, lens, rows, groups, shared, ragged=ragged, pad=2)
        assert np.array_equal(a, _run(q, cache, lens, rows, groups, shared, ragged=ragged).astype(np.float64))


def test_every_way_is_reached():
    """The plans that the tests above are meant for (f16, d 128)."""
    few = _plan(2, 4, 128, 64, 100, 8, 8, 2, True, False)
    assert (few.shared_rows, few.own_rows, few.launches, few.join) == (16, 16, 2, 1)
    alone = _plan(2, 4, 128, 64, 1, 8, 8, 2, True, False)
    assert (alone.shared_rows, alone.own_splits, alone.launches, alone.join, alone.workspace_bytes) == (0, 1, 1, 0, 0)
    alone = _plan(2, 4, 128, 64, 10, 8, 8, 2, True, False)
    assert (alone.shared_rows, alone.launches, alone.join) == (0, 2, 1) and alone.workspace_bytes > 0
    assert _plan(8, 4, 128, 64, 600, 64, 64, 64, True, False).shared_rows == 0         # nothing is read twice
    many = _plan(8, 4, 128, 64, 600, 64, 64, 1, True, False)
    assert (many.shared_rows, many.own_rows, many.own_splits, many.launches, many.join) == (256, 16, 1, 2, 0)
    assert _plan(8, 4, 128, 64, 600, 65, 65, 1, True, False).launches == 3
    tiles = _plan(8, 4, 128, 64, 600, 6400, 64, 1, True, False)
    assert (tiles.shared_rows, tiles.own_rows, tiles.launches, tiles.join) == (256, 256, 3, 1)
    assert _plan(8, 4, 128, 64, 600, 64, 64, 0, True, False).shared_rows == 0


@pytest.mark.parametrize("prefix,page,group,members,n", [(6000, 64, 4, 3, 1), (6000, 16, 1, 2, 1), (5100, 128, 8, 5, 2),
                                                         (3000, 32, 4, 40, 1)])
def test_long_prefixes(prefix, page, group, members, n):
    """Prefixes that are split, own tokens that are split too, one table with room
    for far more."""
    announce(f"prefix long {prefix} page={page} group={group} members={members} n={n}")
    heads, d = 2, 64
    lens = [prefix + n + 13 * i for i in range(members)]
    lens[-1] += 3000
    for f16 in (True, False):
        for wide in (0, 2000):
            cache = _cache(lens, [0, members], [prefix], heads, page, d, wide=wide)
            q = _q(7, members * n, heads * group * d, f16)
            a = _check(q, cache, lens, [n] * members, [0, members], [prefix], ragged=False)
            b = _check(q, cache, lens, [n] * members, [0, members], [prefix], ragged=True)
            assert np.max(abs(a - b)) <= 2.0 ** -9 * np.max(abs(a))


@pytest.mark.parametrize("f16", [True, False])
def test_nothing_shared(f16):
    """No groups, groups of one, of none, prefixes of 0, negative, beyond all
    tokens, shorter than a page; empty sequences; more rows than tokens."""
    announce(f"prefix nothing f16={f16}")
    heads, group, d, page = 2, 4, 64, 32
    lens, rows = [100, 0, 3, 250, 64], [1, 1, 5, 2, 64]
    q = _q(9, sum(rows), heads * group * d, f16)
    for groups, shared in (([0], []), ([0, 1, 2, 3, 4, 5], [64, 0, 2, 10 ** 9, -4]), ([2, 2, 2, 4], [9, 64, 31]),
                           ([0, 0], [50]), ([0, 5], [0])):
        cache = _cache(lens, groups, shared, heads, page, d)
        got = _check(q, cache, lens, rows, groups, shared, ragged=True)
        assert (got[1] == 0).all() and (got[2:4] == 0).all()       # no tokens; rows before the first


def test_group_starts_out_of_order():
    """Nothing out of range is read, and every row is still its own sequence's
    attention: the tables of all agree here."""
    announce("prefix starts")
    heads, group, d, page = 1, 4, 64, 16
    lens = [200, 220, 190, 205, 300, 192]
    cache = _cache(lens, [0, 6], [180], heads, page, d)
    q = _q(11, 6, heads * group * d, True)
    want = _check(q, cache, lens, [1] * 6, [0, 6], [180], ragged=False)
    for groups in ([5, 2, 6], [0, 4, 2, 6], [-9, 3, 99], [0, 2 ** 31 - 1, -2 ** 31], [6, 6, 0], [3, 0, 3]):
        shared = [150] * (len(groups) - 1)
        got = _check(q, cache, lens, [1] * 6, groups, shared, ragged=False)
        assert np.max(abs(got - want)) <= 2.0 ** -9 * np.max(abs(want))
    # more sequences and groups than a wave finds the plan of, past one step of 1024
    lens = [150 + i % 70 for i in range(90)]
    cache = _cache(lens, [0, 90], [140], heads, page, d)
    q = _q(12, 90, heads * group * d, True)
    r = np.random.RandomState(4)
    starts = np.sort(r.randint(0, 91, 80))
    for groups in ([0, 40, 20, 90], [89, 3, 90], list(starts), list(r.permutation(starts)), [7] * 60 + [90, 3, 90],
                   [7] * 1200 + [90, 3, 90]):
        _check(q, cache, lens, [1] * 90, groups, [140] * (len(groups) - 1), ragged=False)
    lens = [50 + i % 70 for i in range(1300)]
    cache = _cache(lens, [0, 1300], [48], heads, page, d)
    q = _q(13, 1300, heads * group * d, True)
    starts = np.sort(r.randint(0, 1301, 1200))
    for groups in (list(starts), list(r.permutation(starts)), [700] * 1150 + [1300, 3, 1300]):
        _check(q, cache, lens, [1] * 1300, groups, [48] * (len(groups) - 1), ragged=False)


def test_a_bad_row_shows_in_itself_only():
    """NaN and infinite queries, in 16-row workgroups and in tiles."""
    announce("prefix bad rows")
    heads, group, d, page, members = 2, 8, 64, 64, 12
    lens = [400 + 7 * i for i in range(members)]
    for wide in (0, 2 ** 31 // (members * heads * group * d * page)):
        cache = _cache(lens, [0, members], [384], heads, page, d, wide=wide)
        q = _q(16, members, heads * group * d, True)
        want = _check(q, cache, lens, [1] * members, [0, members], [384], ragged=False)
        q[3, 5], q[7, 70] = np.nan, np.inf
        got = _run(q, cache, lens, [1] * members, [0, members], [384], ragged=False).astype(np.float64)
        bad = np.zeros(got.shape, bool)
        bad[3, :d], bad[7, d:2 * d] = True, True
        assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], want[~bad])


def test_pitched_tables_and_caches_past_32_bits():
    """A page table that is part of a wider one; pages that lie past 4 GiB."""
    import torch
    announce("prefix pitched tables, large cache")
    heads, group, d, page, pages = 8, 2, 128, 256, 17000
    k = torch.zeros((pages, heads, page, d), dtype=torch.int8, device="cuda")
    v = torch.zeros((pages, heads, d, page), dtype=torch.int8, device="cuda")
    assert k.numel() > 2 ** 32
    lens, groups, shared = [600, 530, 513], [0, 3], [512]
    used = [16999, 16500, 3, 16998, 9]
    table = np.array([[16999, 16500, 3], [16999, 16500, 16998], [16999, 16500, 9]], np.int32)
    small = _cache([1280], [0, 1], [0], heads, page, d, spare=0)
    kc, vc, ks, vs, _ = small
    scales = [torch.zeros((pages, heads), device="cuda") for _ in range(2)]
    for i, p in enumerate(used):
        k[p], v[p] = dev(kc[i]), dev(vc[i])
        scales[0][p], scales[1][p] = dev(ks[i]), dev(vs[i])
    near = np.vectorize(used.index)(table)
    q = _q(17, 3, heads * group * d, True)
    out = torch.empty(q.shape, dtype=torch.float16, device="cuda")
    wide = pitched(np.pad(table, ((0, 0), (0, 20)), constant_values=-1), 31)
    assert _plan(heads, group, d, page, 23, 3, 3, 1, True, False).shared_rows == 16
    ins = [dev(q), k, v, *scales, wide] + [dev(np.array(x, np.int32)) for x in (lens, groups, shared)]
    assert na.PrefixAttention().compute([na.tensor(out)], [na.tensor(x) for x in ins]) == na.OK
    torch.cuda.synchronize()
    want, weight, spread = ref.attention(q, kc, vc, ks, vs, near, lens, [1] * 3)
    assert (abs(host(out) - want) <= ref.attention_tolerance(True, want, weight, spread, vs)).all()
    del k, v


def test_rows_of_no_sequence_are_left_alone():
    announce("prefix rows left")
    heads, group, d, page = 1, 2, 64, 16
    lens, rows = [200, 210], [2, 1]
    for wide in (0, 30000):
        _rows_left(heads, group, d, page, lens, rows, _cache(lens, [0, 2], [190], heads, page, d, wide=wide))


def _rows_left(heads, group, d, page, lens, rows, cache):
    plan = _plan(heads, group, d, page, cache[4].shape[1], 8, 2, 1, True, True)
    assert plan.shared_rows == (16 if cache[4].shape[1] > 30000 else 0)
    q = _q(12, 8, heads * group * d, True)
    import torch
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    starts = dev(np.array([1, 3, 4], np.int32))
    ins = [na.tensor(dev(x)) for x in [q, *cache] + [np.array(x, np.int32) for x in (lens, [0, 2], [190])]]
    assert na.PrefixAttention().compute([na.tensor(out)], ins + [na.tensor(starts)]) == na.OK
    torch.cuda.synchronize()
    got = host(out)
    assert (got[[0, 4, 5, 6, 7]] == 7).all()
    want, weight, spread = ref.attention(q[1:4], *cache, lens, rows)
    tol = ref.attention_tolerance(True, want, weight, spread, cache[3])
    assert (abs(got[1:4] - want) <= tol).all()


@pytest.mark.parametrize("f16", [True, False])
def test_pages_that_do_not_exist_and_nan(f16):
    """A missing page of the prefix shows in the whole group, one of a sequence's
    own only there; NaN scales the same; tokens past a sequence's last do not."""
    announce(f"prefix bad pages f16={f16}")
    heads, group, d, page = 2, 2, 64, 64
    groups, shared = [0, 3, 6], [256, 256]
    lens = [300, 320, 260, 257, 300, 310]
    cache = _cache(lens, groups, shared, heads, page, d, spare=9)
    kc, vc, ks, vs, table = cache
    table[0:3, 2] = 10 ** 6                      # of the first group's prefix
    table[4, 4] = -3                             # of one sequence's own
    ks[table[5, 4], 1] = np.nan                  # one head of one page
    q = _q(13, 6, heads * group * d, f16)
    got = _check(q, cache, lens, [1] * 6, groups, shared, ragged=False)
    assert np.isnan(got[:3]).all() and np.isnan(got[4]).all() and np.isfinite(got[3]).all()
    assert np.isfinite(got[5, :group * d]).all() and np.isnan(got[5, group * d:]).all()
    # behind the last token: whatever it is
    vs[table[3, 4]] = np.float32(0.01)
    vc[table[3, 4], :, :, 1:] = 127
    _check(q, cache, lens, [1] * 6, groups, shared, ragged=False)


def test_scale_and_equal_to_cache_attention():
    """The same numbers as CacheAttention's up to the order of sums."""
    import torch
    announce("prefix against cache attention")
    heads, group, d, page, members = 8, 4, 128, 64, 33
    groups, shared = [0, 20, members], [4096, 1000]
    lens = [4096 + 5 * i + 1 for i in range(20)] + [1001 + 100 * i for i in range(13)]
    cache = _cache(lens, groups, shared, heads, page, d)
    q = _q(14, members, heads * group * d, True)
    got = _run(q, cache, lens, [1] * members, groups, shared, ragged=False, scale=0.05).astype(np.float64)
    out = torch.empty(q.shape, dtype=torch.float16, device="cuda")
    ins = [na.tensor(dev(x)) for x in [q, *cache, np.array(lens, np.int32)]]
    assert na.CacheAttention(scale=0.05).compute([na.tensor(out)], ins) == na.OK
    torch.cuda.synchronize()
    want = host(out).astype(np.float64)
    assert np.linalg.norm(got - want) <= 2.0 ** -10 * np.linalg.norm(want)


def test_graph_streams_and_repeats():
    """A captured call follows lengths and prefixes that change before a replay;
    two streams at once; the same bits every time."""
    import torch
    announce("prefix graph")
    heads, group, d, page, members = 2, 4, 64, 16, 12
    groups, shared = [0, 5, members], [700, 300]
    lens = [701 + 3 * i for i in range(5)] + [301 + 50 * i for i in range(7)]
    cache = _cache([n + 100 for n in lens], groups, shared, heads, page, d, wide=500)
    assert _plan(heads, group, d, page, cache[4].shape[1], members, members, 2, True, False).shared_rows == 16
    q = _q(15, members, heads * group * d, True)
    T = na.tensor
    runs = []
    for _ in range(2):
        out = torch.empty(q.shape, dtype=torch.float16, device="cuda")
        held = [dev(x) for x in [q, *cache] + [np.array(x, np.int32) for x in (lens, groups, shared)]]
        op = na.PrefixAttention()
        ins = [T(x) for x in held]
        ws = torch.empty(op.workspace_size(ins, [T(out)]), dtype=torch.uint8, device="cuda")
        runs.append((torch.cuda.Stream(), op, ins, out, ws, held))
    torch.cuda.synchronize()
    for _ in range(3):
        for s, op, ins, out, ws, _ in runs:
            assert op.compute([T(out)], ins, stream=s, workspace=ws) == na.OK
    torch.cuda.synchronize()
    assert torch.equal(runs[0][3], runs[1][3])
    s, op, ins, out, ws, held = runs[0]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        assert op.compute([T(out)], ins, stream=s, workspace=ws) == na.OK
    for step in range(3):
        held[6].copy_(dev(np.array(lens, np.int32) + 33 * step))
        held[8].copy_(dev(np.array(shared, np.int32) - 100 * step))
        ws.fill_(0xff)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        now = [n + 33 * step for n in lens]
        want, weight, spread = ref.attention(q, *cache, now, [1] * members)
        tol = ref.attention_tolerance(True, want, weight, spread, cache[3])
        assert (abs(host(out) - want) <= tol).all(), step


def test_more_rows_than_2_to_the_23():
    """A call whose rows times heads pass what a launch of a workgroup each would hold:
    sequences from all over it."""
    import torch
    announce("prefix many rows")
    heads, group, d, page, members, n = 8, 16, 16, 64, 1024, 65
    assert members * n * heads * group > 2 ** 23
    groups, shared = [0, members], [640]
    lens = [640 + n + i % 50 for i in range(members)]
    cache = _cache(lens, groups, shared, heads, page, d, wide=188)
    assert _plan(heads, group, d, page, cache[4].shape[1], members * n, members, 1, True, False).shared_rows == 256
    q = _q(18, members * n, heads * group * d, True)
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    ins = [na.tensor(dev(x)) for x in [q, *cache] + [np.array(x, np.int32) for x in (lens, groups, shared)]]
    assert na.PrefixAttention().compute([na.tensor(out)], ins) == na.OK
    torch.cuda.synchronize()
    some = [0, 1, 500, 1009, 1010, 1022, 1023]         # (2^23 / 128 / 65: sequence 1008)
    at = np.concatenate([np.arange(b * n, (b + 1) * n) for b in some])
    of = [*cache[:4], cache[4][some, :12]]
    want, weight, spread = ref.attention(q[at], *of, [lens[b] for b in some], [n] * len(some))
    got = host(out)[at]
    assert (abs(got - want) <= ref.attention_tolerance(True, want, weight, spread, cache[3])).all()


@pytest.mark.parametrize("d,page,heads,group,members,n", [(128, 64, 4, 4, 64, 1), (128, 16, 4, 4, 40, 1), (64, 64, 8, 8, 10, 1),
                                                          (64, 16, 8, 8, 33, 1), (96, 128, 4, 4, 24, 3), (256, 64, 4, 4, 40, 1)])
def test_probabilities_in_tiles_are_as_fine_as_cache_attentions(d, page, heads, group, members, n):
    """Rows that CacheAttention gives workgroups of 16, whose probabilities are two f16:
    in tiles over shared tokens they are as well. Few tokens have most of the weight, so
    that where values cancel one f16 (2^-12 to 2^-11 of each weight) shows beside the
    result's own rounding: in 0.05 to 0.9 % of the results, by numpy."""
    import torch
    announce(f"prefix fine d={d} page={page} heads={heads} members={members} n={n}")
    groups, shared, scale = [0, members], [1280], 2.0 / d ** 0.5
    lens = [1280 + n + 5 * i for i in range(members)]
    wide = 2 ** 31 // (members * n * heads * group * d * page)
    cache = _cache(lens, groups, shared, heads, page, d, wide=wide)
    plan = _plan(heads, group, d, page, cache[4].shape[1], members * n, members, 1, True, False)
    assert plan.shared_rows in (128, 256) and plan.own_rows == 16
    q = _q(19, members * n, heads * group * d, True)
    want, weight, spread = ref.attention(q, *cache, lens, [n] * members, scale=scale)
    # (two f16 hold 22 bits: less than half of 2^-21; the result is rounded once)
    tol = ref.attention_tolerance(False, want, weight, spread, cache[3]) + 1.01 * 2.0 ** -11 * abs(want) + 2.0 ** -24
    out = torch.empty(q.shape, dtype=torch.float16, device="cuda")
    ins = [na.tensor(dev(x)) for x in [q, *cache, np.array(lens, np.int32)]]
    assert na.CacheAttention(scale=scale).compute([na.tensor(out)], ins) == na.OK
    torch.cuda.synchronize()
    assert (abs(host(out) - want) <= tol).all()
    got = _run(q, cache, lens, [n] * members, groups, shared, ragged=False, scale=scale).astype(np.float64)
    assert (abs(got - want) <= tol).all()
