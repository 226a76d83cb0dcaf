"""KvCacheFork, KvCacheCompact and KvCacheCopy against their definitions step by
step: forks, growth, cuts, sequences given up, shared and half-full pages, a cache
that runs out, tables with numbers that are no pages, wide and narrow tables, many
pages, graphs and streams."""
from __future__ import annotations

import numpy as np
import pytest

import nnops_amd as na
import pages_ref as ref
from gpu_util import announce, dev, host, pitched

pytestmark = pytest.mark.gpu


def _tables(r, b, wide, page, pages, *, share=0.5, most=None, junk=0.0):
    """A table whose sequences share first pages, lengths and counts."""
    order = list(r.permutation(pages))
    table, lens = np.full((b, wide), -7, np.int32), np.zeros(b, np.int32)
    for i in range(b):
        lens[i] = r.randint(0, (most or wide * page) + 1)
        held = -(-int(lens[i]) // page)
        k = 0
        if i and r.rand() < share:
            j = r.randint(0, i)
            k = r.randint(0, min(held, int(lens[j]) // page) + 1)
            table[i, :k] = table[j, :k]
        for c in range(k, held):
            if not order:
                lens[i] = c * page
                break
            table[i, c] = order.pop()
    if junk:
        bad = r.rand(b, wide) < junk
        table[bad] = r.choice([-1, -5, pages, pages + 9, 2 ** 31 - 1, -2 ** 31], bad.sum())
    return table, lens, ref.holders(table, lens, page, pages)


def _fork(table, lens, refs, parents, new, wide, page, *, in_place=False, pad=0, stream=None):
    import torch
    n = len(parents)
    i32 = dict(dtype=torch.int32, device="cuda")
    t_in = pitched(table.astype(np.int32), table.shape[1] + pad)
    t_out = torch.full((n, wide + pad), 77, **i32)
    refs_in = dev(refs.astype(np.int32))
    refs_out = refs_in if in_place else torch.empty_like(refs_in)
    outs = [t_out[:, :wide], torch.empty(n, **i32), refs_out, torch.empty((n, 2), **i32), torch.empty(2, **i32)]
    ins = [t_in, dev(lens.astype(np.int32)), refs_in, dev(np.asarray(parents, np.int32)), dev(np.asarray(new, np.int32))]
    op = na.KvCacheFork(page_tokens=page)
    ti, to = [na.tensor(x) for x in ins], [na.tensor(x) for x in outs]
    assert op.validate(ti, to) == na.OK
    assert op.compute(to, ti, stream=stream) == na.OK
    torch.cuda.synchronize()
    assert (host(t_out)[:, wide:] == 77).all()
    return [host(x) for x in outs]


def _check_fork(table, lens, refs, parents, new, wide, page, **kw):
    got = _fork(table, lens, refs, parents, new, wide, page, **kw)
    want = ref.fork(table, lens, refs, parents, new, wide, page)
    for name, g, w in zip(("table", "lengths", "refs", "copies", "counts"), got, want):
        assert np.array_equal(g, w), name
    return got


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("b,n,wide,pages", [(1, 1, 1, 2), (1, 9, 3, 40), (7, 5, 4, 60), (20, 33, 5, 300), (64, 64, 9, 900),
                                            (64, 70, 9, 13000)])
def test_fork(page, b, n, wide, pages):
    """Children with parents of their own, twins, none; growth from nothing to
    whole pages, cuts, and refs in place."""
    announce(f"fork page={page} b={b} n={n} wide={wide} pages={pages}")
    r = np.random.RandomState(1000 * page + b)
    table, lens, refs = _tables(r, b, wide, page, pages)
    parents = np.where(r.rand(n) < 0.15, -1, r.randint(0, b, n))
    new = r.choice([0, 1, 1, 1, 2, page, page + 1, -1, -page, -3 * page, 3 * page], n)
    a = _check_fork(table, lens, refs, parents, new, wide + 2, page, pad=3)
    c = _check_fork(table, lens, refs, parents, new, wide + 2, page, in_place=True)
    for x, y in zip(a, c):
        assert np.array_equal(x, y)
    # what follows from the definition: the counts are the children's
    assert np.array_equal(a[2], ref.holders(a[0], a[1], page, pages))
    assert a[4][0] == (a[2] == 0).sum()


def test_twins_share_all_but_the_page_they_write():
    """Three children of one parent in a page in part full: the first keeps it; of
    a page that somebody else holds too (a count of the caller's), none does."""
    announce("fork twins")
    table, lens = np.array([[4, 2, 9]]), np.array([40])
    refs = np.zeros(12, np.int64)
    refs[[4, 2, 9]] = 1
    t, ln, rf, copies, counts = _check_fork(table, lens, refs, [0, 0, 0], [1, 1, 1], 3, 16)
    assert t.tolist() == [[4, 2, 9], [4, 2, 0], [4, 2, 1]] and ln.tolist() == [41] * 3
    assert copies.tolist() == [[-1, -1], [9, 0], [9, 1]] and rf[9] == 1 and rf[4] == 3
    refs[9] += 1
    t, _, rf, copies, _ = _check_fork(table, lens, refs, [0, 0, 0], [1, 1, 1], 3, 16)
    assert copies.tolist() == [[9, 0], [9, 1], [9, 3]] and rf[9] == 1
    # not all of them write
    refs[9] -= 1
    _, _, rf, copies, _ = _check_fork(table, lens, refs, [0, 0, 0], [1, 0, 1], 3, 16)
    assert copies.tolist() == [[9, 0], [-1, -1], [9, 1]] and rf[9] == 1
    # at a page's end nothing is written into
    _, _, rf, copies, _ = _check_fork(table, np.array([32]), np.bincount([4, 2], minlength=12), [0, 0], [1, 1], 3, 16)
    assert (copies == -1).all() and rf.tolist() == [1, 1, 2, 0, 2] + [0] * 7


def test_fork_given_up_pages_are_free_at_once():
    announce("fork frees")
    table, lens = np.array([[0, 1], [2, 3]]), np.array([32, 32])
    t, _, rf, _, counts = _check_fork(table, lens, np.ones(4, np.int64), [1, -1], [0, 30], 4, 16)
    assert t.tolist() == [[2, 3, -1, -1], [0, 1, -1, -1]] and rf.tolist() == [1] * 4 and counts.tolist() == [0, 0]


@pytest.mark.parametrize("held", [0, 20000])      # (pages that somebody else holds: more than a workgroup counts)
@pytest.mark.parametrize("seed", range(4))
def test_fork_without_pages_enough(seed, held):
    """Cells that get none are -1 and are counted; tables too narrow cut lengths."""
    announce(f"fork short {seed}")
    r = np.random.RandomState(seed)
    table, lens, refs = _tables(r, 12, 6, 16, 40)
    refs[r.rand(40) < 0.5] += 1
    refs = np.concatenate([refs, np.ones(held, np.int64)])
    parents = r.randint(-1, 12, 30)
    got = _check_fork(table, lens, refs, parents, r.randint(-20, 150, 30), 7, 16)
    assert got[4][1] > 0
    _check_fork(table, lens, refs, parents, np.full(30, 2 ** 31 - 1), 3, 16)
    _check_fork(table, lens, refs, parents, np.full(30, -2 ** 31), 3, 16)
    # (what got none is asked for again by the next call)
    more = np.concatenate([got[2], np.zeros(160, np.int64)])
    _check_fork(got[0], got[1], more, np.arange(30), np.full(30, 1), 9, 16)


@pytest.mark.parametrize("pages", [200, 13000])
def test_fork_of_tables_that_hold_no_pages(pages):
    """Page numbers out of range, lengths and parents too: no memory is touched by
    them, and the rest is as defined."""
    announce(f"fork junk {pages}")
    r = np.random.RandomState(5)
    table, lens, refs = _tables(r, 30, 8, 16, pages, junk=0.3)
    lens = lens.astype(np.int64)
    lens[3], lens[4], lens[5] = -9, 2 ** 31 - 1, -2 ** 31
    refs = ref.holders(table, lens, 16, pages)
    parents = r.randint(-3, 33, 50)
    parents[:2] = 2 ** 31 - 1, -2 ** 31
    _check_fork(table, lens, refs, parents, r.randint(-30, 60, 50), 9, 16)


@pytest.mark.parametrize("b,n,wide,out_wide,pages", [
    (3, 4, 700, 1000, 40000),              # rows of several chunks
    (40, 1100, 3, 4, 2500),                # more children than the workgroup has threads
    (2, 3, 2, 2, 70000),                   # more pages than one step looks at
    (20, 30, 3, 4, 12288), (20, 30, 3, 4, 12289), (1024, 1024, 3, 4, 9000), (3, 2, 9000, 9001, 3000),
    (300, 16384, 2, 2, 60000), (16384, 100, 1, 2, 14000), (1025, 3, 1, 1, 1100), (3, 1025, 1, 1, 1100),
    (1500, 7, 2, 3, 4000), (5, 0, 3, 2, 50), (0, 6, 0, 5, 60), (4, 4, 3, 0, 50), (3, 2, 4, 4, 0), (0, 0, 0, 0, 0)])
def test_fork_sizes(b, n, wide, out_wide, pages):
    announce(f"fork sizes {b} {n} {wide} {out_wide} {pages}")
    r = np.random.RandomState(b + n)
    table, lens, refs = _tables(r, b, wide, 16, pages)
    parents = r.randint(-1, b, n) if b else np.full(n, -1)
    _check_fork(table, lens, refs, parents, r.randint(-5, 40, n), out_wide, 16)


def test_fork_free_pages_far_up():
    """The free pages that are needed lie behind 100000 held ones."""
    announce("fork far")
    refs = np.ones(131072, np.int64)
    refs[[5, 65535, 99999, 131070, 131071]] = 0
    t, _, rf, _, counts = _check_fork(np.zeros((0, 0)), np.zeros(0), refs, [-1] * 3, [16, 32, 1], 2, 16)
    assert t.tolist() == [[5, -1], [65535, 99999], [131070, -1]] and counts.tolist() == [1, 0]


# --- compact -----------------------------------------------------------------------

def _check_compact(table, lens, refs, page, *, in_place=False, pad=0):
    import torch
    i32 = dict(dtype=torch.int32, device="cuda")
    pages = len(refs)
    ins = [pitched(table.astype(np.int32), table.shape[1] + pad) if pad else dev(table.astype(np.int32)),
           dev(lens.astype(np.int32)), dev(refs.astype(np.int32))]
    outs = [ins[0] if in_place else torch.empty(table.shape, **i32), ins[2] if in_place else torch.empty(pages, **i32),
            torch.empty((pages // 2, 2), **i32), torch.empty(pages, **i32), torch.empty(2, **i32)]
    op = na.KvCacheCompact(page_tokens=page)
    ti, to = [na.tensor(x) for x in ins], [na.tensor(x) for x in outs]
    assert op.validate(ti, to) == na.OK
    assert op.compute(to, ti) == na.OK
    torch.cuda.synchronize()
    got = [host(x) for x in outs]
    for name, g, w in zip(("table", "refs", "copies", "moved", "counts"), got, ref.compact(table, lens, refs, page)):
        assert np.array_equal(g, w), name
    return got


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("b,wide,page,pages", [(1, 1, 16, 1), (3, 2, 16, 7), (9, 5, 64, 64), (20, 6, 16, 500),
                                               (50, 300, 16, 30000), (3, 3, 256, 9000), (0, 0, 16, 20), (4, 0, 16, 20),
                                               (3, 2, 16, 0), (5, 4, 32, 4096), (5, 4, 32, 8192),
                                               (5, 4, 32, 16384), (5, 4, 32, 16385), (3, 22000, 16, 2000)])
def test_compact(b, wide, page, pages, in_place):
    announce(f"compact {b} {wide} page={page} pages={pages} in_place={in_place}")
    r = np.random.RandomState(pages + b)
    table, lens, refs = _tables(r, b, wide, page, pages)
    held = r.rand(pages) < 0.2                       # held by somebody else
    refs[held] += 1
    _check_compact(table, lens, refs, page, in_place=in_place, pad=5 if wide else 0)


@pytest.mark.parametrize("pages,pattern", [(100, "none"), (100, "all"), (101, "upper"), (4097, "upper"), (4096, "lower"),
                                           (12288, "one block"), (9001, "last"), (8192, "odd"), (2, "upper"), (1, "all"),
                                           (40960, "upper"), (40961, "lower"), (20480, "one block"), (24000, "last"),
                                           (32768, "odd"), (16385, "all"), (30000, "none")])
def test_compact_patterns(pages, pattern):
    """Nothing held, all, only the upper half, a block that ends at the border."""
    announce(f"compact pattern {pages} {pattern}")
    refs = np.zeros(pages, np.int64)
    at = dict(none=slice(0, 0), all=slice(None), upper=slice(pages // 2, None), lower=slice(0, pages // 2),
              odd=slice(1, None, 2), last=slice(pages - 1, None))
    refs[at.get(pattern, slice(4096, 8192))] = 3
    refs[-1:] *= -1                                   # (a count that is not 0 is held)
    got = _check_compact(np.zeros((0, 0)), np.zeros(0), refs, 16)
    again = _check_compact(np.zeros((0, 0)), np.zeros(0), got[1].astype(np.int64), 16)
    assert again[4][1] == 0


@pytest.mark.parametrize("pages", [200, 20000])
def test_compact_of_tables_that_hold_no_pages(pages):
    announce(f"compact junk {pages}")
    r = np.random.RandomState(8)
    table, lens, refs = _tables(r, 30, 8, 16, pages, junk=0.3)
    lens = lens.astype(np.int64)
    lens[3], lens[4] = -9, 2 ** 31 - 1
    refs[r.rand(pages) < 0.1] = 0                       # (tables that say more than the counts)
    _check_compact(table, lens, refs, 16)


# --- copy --------------------------------------------------------------------------

@pytest.mark.parametrize("heads,page,d", [(1, 16, 16), (8, 64, 128), (3, 32, 80), (1, 256, 256), (2, 128, 112), (64, 16, 16),
                                          (300, 16, 16)])
def test_copy(heads, page, d):
    """Pages smaller and larger than a workgroup's piece; pairs that are skipped;
    all other pages as they were."""
    import torch
    announce(f"copy heads={heads} page={page} d={d}")
    r = np.random.RandomState(heads + d)
    pages = 23
    kc = r.randint(-127, 128, (pages, heads, page, d)).astype(np.int8)
    vc = r.randint(-127, 128, (pages, heads, d, page)).astype(np.int8)
    ks, vs = r.rand(pages, heads).astype(np.float32), r.rand(pages, heads).astype(np.float32)
    ks[3, 0] = np.nan
    pairs = np.array([[3, 9], [-1, -1], [0, 22], [3, 1], [5, -1], [-1, 5], [pages, 2], [4, pages], [2 ** 31 - 1, 4],
                      [22, 8], [7, 7], [-2 ** 31, 6]][:11 if heads > 1 else 12], np.int32)
    pairs[9] = 21, 8
    cache = [dev(x) for x in (kc, vc, ks, vs)]
    op, outs, ins = na.KvCacheCopy(), [na.tensor(x) for x in cache], [na.tensor(dev(pairs))]
    assert op.validate(ins, outs) == na.OK
    assert op.compute(outs, ins) == na.OK
    torch.cuda.synchronize()
    for got, was in zip(cache, (kc, vc, ks, vs)):
        want = was.copy()
        for a, b in ((3, 9), (0, 22), (3, 1), (21, 8)):
            want[b] = was[a]
        assert np.array_equal(host(got), want, equal_nan=was.dtype == np.float32)
    assert op.compute(outs, [na.tensor(torch.empty((0, 2), dtype=torch.int32, device="cuda"))]) == na.OK


def test_copy_past_32_bits():
    """A cache of more than 4 GiB a side."""
    import torch
    announce("copy past 32 bits")
    heads, page, d, pages = 8, 256, 256, 8300
    side = heads * page * d
    k = torch.zeros((pages, heads, page, d), dtype=torch.int8, device="cuda")
    v = torch.zeros((pages, heads, d, page), dtype=torch.int8, device="cuda")
    assert k.numel() > 2 ** 32 and side * (pages - 1) > 2 ** 32
    ks, vs = torch.zeros((pages, heads), device="cuda"), torch.zeros((pages, heads), device="cuda")
    k[8299] = 5
    v[8299] = 6
    ks[8299], vs[3] = 0.5, 0.25
    k[3], v[3] = 1, 2
    pairs = dev(np.array([[8299, 1], [3, 8290]], np.int32))
    assert na.KvCacheCopy().compute([na.tensor(x) for x in (k, v, ks, vs)], [na.tensor(pairs)]) == na.OK
    torch.cuda.synchronize()
    assert (k[1] == 5).all() and (v[1] == 6).all() and (ks[1] == 0.5).all()
    assert (k[8290] == 1).all() and (v[8290] == 2).all() and (vs[8290] == 0.25).all()
    assert int(k.sum(dtype=torch.int64)) == 12 * side and int((ks != 0).sum()) == 2 * heads
    del k, v


# --- together ------------------------------------------------------------------------

def _graph_case(stream):
    """Tables that go back and forth between two buffers, as a program's do."""
    import torch
    r = np.random.RandomState(3)
    b, wide, page, pages = 16, 12, 16, 400
    table, lens, refs = _tables(r, b, wide, page, pages, most=100)
    parents = [dev(r.randint(0, b, b).astype(np.int32)) for _ in range(2)]
    new = dev(np.full(b, 3, np.int32))
    t = [dev(table), torch.empty((b, wide), dtype=torch.int32, device="cuda")]
    ln = [dev(lens), torch.empty(b, dtype=torch.int32, device="cuda")]
    rf = dev(refs.astype(np.int32))
    copies, counts = torch.empty((b, 2), dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
    cache = [x.random_(-127, 128) if x.dtype == torch.int8 else x.uniform_() for x in na.kv_cache(pages, 2, page, 32)]
    op, copy = na.KvCacheFork(page_tokens=page), na.KvCacheCopy()
    T = na.tensor
    calls = []
    for i in range(2):
        ins = [T(t[i]), T(ln[i]), T(rf), T(parents[i]), T(new)]
        outs = [T(t[1 - i]), T(ln[1 - i]), T(rf), T(copies), T(counts)]
        calls.append((ins, outs, torch.empty(op.workspace_size(ins, outs), dtype=torch.uint8, device="cuda")))
    state = t + ln + [rf, copies, counts] + cache

    def step():
        for ins, outs, ws in calls:
            assert op.compute(outs, ins, workspace=ws, stream=stream) == na.OK
            assert copy.compute([T(x) for x in cache], [T(copies)], stream=stream) == na.OK
    return step, state


def test_fork_and_copy_in_a_graph():
    import torch
    announce("fork in a graph")
    s = torch.cuda.Stream()
    step, state = _graph_case(s)
    begin = [x.clone() for x in state]
    want = []
    for _ in range(3):
        step()
        torch.cuda.synchronize()
        want.append([x.clone() for x in state])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step()
    for x, y in zip(state, begin):
        x.copy_(y)
    for i in range(3):
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip(state, want[i]):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), i
        torch.empty(1 << 20, device="cuda").zero_()   # eager work between replays


def test_calls_on_two_streams():
    """Each with its workspace and outputs, at once."""
    import torch
    announce("fork on two streams")
    runs = [_graph_case(torch.cuda.Stream()) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for step, _ in runs:
            step()
    torch.cuda.synchronize()
    for x, y in zip(runs[0][1][:7], runs[1][1][:7]):
        assert torch.equal(x, y)


def test_refused_calls_write_nothing():
    import torch
    announce("refused fork")
    t = torch.full((2, 3), 5, dtype=torch.int32, device="cuda")
    two, refs, copies = torch.ones(2, dtype=torch.int32, device="cuda"), torch.ones(9, dtype=torch.int32, device="cuda"), \
        torch.ones((2, 2), dtype=torch.int32, device="cuda")
    op = na.KvCacheFork(page_tokens=16)
    T = na.tensor
    ins = [T(t), T(two), T(refs), T(two), T(two)]
    out = torch.full((2, 3), 5, dtype=torch.int32, device="cuda")
    assert op.compute([T(t), T(two.clone()), T(refs), T(copies), T(two.clone())], ins) == na.INVALID_ARGUMENT
    assert op.compute([T(out), T(two), T(refs), T(copies), T(two.clone())], ins) == na.INVALID_ARGUMENT
    assert na.KvCacheFork(page_tokens=17).compute([T(out), T(two.clone()), T(refs), T(copies), T(two.clone())],
                                                  ins) == na.UNSUPPORTED
    torch.cuda.synchronize()
    assert (t == 5).all() and (out == 5).all() and (refs == 1).all() and (copies == 1).all() and (two == 1).all()
