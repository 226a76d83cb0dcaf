"""The kernel selection of CacheAttention (nnops_hip_cache_attention_plan), on
the host: no call here reaches a kernel launch. The shapes that the GPU tests
run for a kernel's sake have to be that kernel's."""
from __future__ import annotations

import ctypes as C

import pytest

import nnops_amd as na
from nnops_amd import _lib as L
import test_gpu_cache_attention as gpu


def args(rows, seqs, tokens, *, heads=8, group=4, d=128, page=64, f16=True, ragged=False, window=0, sinks=0):
    g = na.CacheAttentionArgs()
    c = g.cache
    per = max(1, -(-tokens // page))
    c.pages, c.heads, c.page_tokens, c.head_dim, c.sequences, c.table_pages = seqs * per, heads, page, d, seqs, per
    g.rows, g.q_heads, g.f16, g.window, g.sinks = rows, heads * group, int(f16), window, sinks
    c.row_starts = 4096 if ragged else None
    return g


def plan(*a, **kw):
    g, p = args(*a, **kw), L.CacheAttentionPlan()
    assert na.lib().nnops_hip_cache_attention_plan(C.byref(g), C.byref(p)) == na.OK
    assert p.workspace_bytes == na.lib().nnops_hip_cache_attention_workspace_size(C.byref(g))
    assert (p.splits > 1) == (p.workspace_bytes > 0) == (p.join > 0)
    return p


def test_refusals():
    f, p = na.lib().nnops_hip_cache_attention_plan, L.CacheAttentionPlan()
    assert f(None, C.byref(p)) == na.INVALID_ARGUMENT
    assert f(C.byref(args(4, 4, 100)), None) == na.INVALID_ARGUMENT
    assert f(C.byref(args(2, 4, 100)), C.byref(p)) == na.INVALID_ARGUMENT
    assert f(C.byref(args(4, 4, 100, page=24)), C.byref(p)) == na.UNSUPPORTED
    assert f(C.byref(args(0, 4, 100)), C.byref(p)) == na.OK and p.tile_rows == 0


def rows_of(d, f16):
    """Rows of a workgroup that shares its tiles, where the rows fill more than 128."""
    return 256 if d <= (128 if f16 else 64) else 128


# --- the GPU tests' shapes ---------------------------------------------------------

@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("d,page,heads,group,f16", gpu.TILES)
def test_tiles_share_their_tokens(d, page, heads, group, f16, many):
    """test_tiles; test_tiles_of_equal_rows, whose rows fill 128 or more."""
    lens, rows = gpu._mixed(400 if many else 200)
    kw = dict(heads=heads, group=group, d=d, page=page, f16=f16)
    one = int(page >= 64)
    p = plan(sum(rows), len(rows), 600, ragged=True, **kw)
    assert (p.tile_rows, p.one_page) == (rows_of(d, f16), one)
    for n in (13, 34):
        p = plan(9 * n, 9, 520, **kw)
        assert (p.tile_rows, p.one_page) == (rows_of(d, f16) if n * group > 128 else 128, one)


@pytest.mark.parametrize("page,f16", [(16, True), (64, True), (128, False), (32, False)])
def test_windows_and_hidden_values_in_tiles(page, f16):
    _, rows = gpu._mixed(400)
    for window, sinks in ((1, 0), (16, 4), (64, 0), (100, 70), (300, 5), (7, 1 << 40)):
        p = plan(sum(rows), len(rows), 600, heads=20, group=7, d=64, page=page, f16=f16, ragged=True, window=window,
                 sinks=sinks)
        assert p.tile_rows == 256 and p.one_page == (page >= 64)
    for window in (0, 60):
        p = plan(8 * 40, 8, 4 * page + 320, heads=16, group=4, d=64, page=page, f16=f16, window=window)
        assert p.tile_rows == 256 and p.one_page == (page >= 64)


@pytest.mark.parametrize("page,f16", [(64, True), (16, True), (64, False)])
def test_tiles_that_are_split(page, f16):
    kw = dict(heads=4, d=128, page=page, f16=f16)
    for rows, tokens, more in ((52, 33000, dict(group=4)), (52, 33000, dict(group=4, window=20000, sinks=100)),
                               (52, 33000, dict(group=11, ragged=True))):
        p = plan(rows, 2, tokens, **kw, **more)
        assert p.tile_rows >= 128 and p.splits > 8 and p.join == 2


def test_long_sequences_are_split_and_joined():
    """test_long: 16 rows a workgroup, joined by a workgroup a row;
    test_few_splits: 2 to 8 splits, joined by lanes of a wave."""
    for tokens, page, group, n in ((5000, 64, 4, 1), (5000, 16, 1, 1), (3001, 128, 8, 3), (2000, 32, 2, 40)):
        p = plan(3 * n, 3, tokens, heads=2, group=group, d=64, page=page)
        assert p.tile_rows == 16 and p.splits > 1 and p.join == 2
    for d, page, heads, group, seqs, n, tokens, window, f16, splits in gpu.FEW_SPLITS:
        for ragged in (False, True):
            p = plan(seqs * n, seqs, tokens, heads=heads, group=group, d=d, page=page, window=window, f16=f16, ragged=ragged)
            assert (p.tile_rows, p.join) == (16, 1) and (2 <= p.splits <= 8 if ragged else p.splits == splits)


def test_many_sequences_are_split():
    """test_splits_of_many_sequences."""
    for seqs in (63, 64, 65, 130, 200):
        for f16 in (True, False):
            for rows, ragged in ((2 * seqs, False), (2 * seqs, True)):
                assert plan(rows, seqs, 6000, heads=1, group=3, d=64, page=32, f16=f16, ragged=ragged).splits > 1


# --- the rules ------------------------------------------------------------------------

def test_rules_of_the_rows():
    """Shared tiles from a mean of more than 96 rows a sequence on (256 where
    they are ragged), where they fill the chip alone or by the tokens they see."""
    assert plan(24, 1, 8000, heads=64, group=4).tile_rows == 16                   # 96 rows
    assert plan(25, 1, 8000, heads=64, group=4).tile_rows == 128
    assert plan(8 * 64, 8, 8000, heads=64, group=4, ragged=True).tile_rows == 16  # a mean of 256
    assert plan(8 * 65, 8, 8000, heads=64, group=4, ragged=True).tile_rows == 256
    # 128 items of 256 rows, or items x tiles x d of 7 2^14 (d <= 64: 7 2^15)
    assert plan(16 * 64, 16, 64).tile_rows == 256 and plan(15 * 64, 15, 64).tile_rows == 16
    for d, least in ((128, 7 << 14), (64, 7 << 15), (96, 7 << 14)):
        tiles = -(-least // (8 * d))
        assert plan(64, 1, 64 * tiles, d=d).tile_rows == 256
        assert plan(64, 1, 64 * (tiles - 1), d=d).tile_rows == 16
    # f32: 9 2^15 for wider heads (128 rows a tile); heads of 64 7 2^14 unless ragged
    for tokens, want in ((64 * (9 << 15) // 1024, 128), (64 * (9 << 15) // 1024 - 64, 16)):
        assert plan(32, 1, tokens, f16=False).tile_rows == want
    assert plan(64, 1, 64 * (7 << 14) // 512, d=64, f16=False).tile_rows == 256
    assert plan(33, 1, 64000, heads=8, group=4).tile_rows == 256 and plan(32, 1, 64000, heads=8, group=4).tile_rows == 128


def test_no_shared_tiles_for_wide_heads():
    for page, f16, want in ((64, True, 128), (16, True, 16), (128, False, 16)):
        assert plan(4096, 1, 4096, d=256, page=page, f16=f16).tile_rows == want


def test_rules_of_the_splits():
    """None where a wave has no more than two tiles without (f16 rows of up to
    128 channels), no fewer than 4 tiles each, no more than fill the chip."""
    assert plan(1, 1, 512).splits == 1 and plan(1, 1, 513).splits == 3
    assert plan(1, 1, 512, f16=False).splits == 2 and plan(1, 1, 512, d=256).splits == 2
    p = plan(1, 1, 126976)
    assert p.splits == 62 and p.split_tokens * 62 >= 126976 and p.join == 2
    assert plan(64, 64, 4096).splits == 1
    p = plan(2, 2, 777)
    assert p.splits == 4 and p.split_tokens == 256 and p.join == 2
    assert plan(2, 2, 700).join == 1                                              # 3 splits: a wave a row
    assert plan(32, 32, 1000, heads=2, group=16).join == 1                        # 4 of 1024 rows
