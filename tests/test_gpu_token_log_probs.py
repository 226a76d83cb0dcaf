"""TokenLogProbs against log probabilities in 64 bits: vocabularies from one token
to rows that are split, ties, masks, rows of nothing, NaN and infinities, strides,
several tokens a row, tokens that are none, graphs and streams."""
from __future__ import annotations

import numpy as np
import pytest

import datagen as dg
import nnops_amd as na
import pages_ref as ref
from gpu_util import announce, dev, host, pitched

pytestmark = pytest.mark.gpu


def _run(x, tokens, top, *, pad=0, stream=None, flat=False):
    import torch
    rows = x.shape[0]
    dx = pitched(x, x.shape[1] + pad) if pad else dev(x)
    dt = dev(tokens[:, 0] if flat else tokens)
    lp = torch.full((rows, tokens.shape[1] + pad), 7.0, device="cuda")
    ins = [na.tensor(dx), na.tensor(dt)]
    outs = [lp[:, 0].contiguous() if flat else lp[:, :tokens.shape[1]], torch.full((rows,), 7.0, device="cuda")]
    if top:
        outs += [torch.full((rows, top + pad), 7, dtype=torch.int32, device="cuda")[:, :top],
                 torch.full((rows, top + pad), 7.0, device="cuda")[:, :top]]
    op = na.TokenLogProbs(top=top)
    to = [na.tensor(t) for t in outs]
    assert op.validate(ins, to) == na.OK
    assert op.compute(to, ins, stream=stream) == na.OK
    torch.cuda.synchronize()
    if pad and not flat:
        assert (host(lp)[:, tokens.shape[1]:] == 7).all()
    got = [host(t) for t in outs]
    return [got[0].reshape(tokens.shape)] + got[1:]


def _near(got, want, tol):
    got, want = got.astype(np.float64), want.astype(np.float64)
    # (a log probability past f32's range rounds to -inf)
    want = np.where(want < -float(np.finfo(np.float32).max) * (1 + 2.0 ** -25), -np.inf, want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isinf(got), np.isinf(want)) and np.array_equal(got[np.isinf(got)], want[np.isinf(want)])
    fine = np.isfinite(want)
    worst = np.max(np.abs(got[fine] - want[fine]) / np.broadcast_to(tol, want.shape)[fine], initial=0.0)
    assert worst <= 1.0, worst


def _check(x, tokens, top, **kw):
    got = _run(x, tokens, top, **kw)
    lp, entropy, best, best_lp = ref.log_probs(x, tokens, top)
    tol_lp, tol_h = ref.log_probs_tolerance(x, lp, entropy)
    _near(got[0], lp, tol_lp)
    _near(got[1], entropy, tol_h)
    if top:
        assert np.array_equal(got[2], best)
        _near(got[3], best_lp, ref.log_probs_tolerance(x, best_lp, entropy)[0])
    return got


def _x(seed, rows, vocab, f16, size=3.0):
    return (size * dg.normal(seed, (rows, vocab))).astype(np.float16 if f16 else np.float32)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 7), (2, 63), (2, 65), (3, 511), (3, 512), (3, 513), (2, 2047),
                                        (2, 2048), (2, 2049), (5, 4100), (1, 100003), (3, 50257), (1030, 77), (1500, 2600),
                                        (1, 1 << 21), (513, 32768), (520, 32769)])
def test_sizes(rows, vocab, f16):
    announce(f"log probs rows={rows} vocab={vocab} f16={f16}")
    x = _x(rows + vocab, rows, vocab, f16)
    tokens = dg.ints(5, (rows, 2), 0, max(0, min(vocab - 1, 100))).astype(np.int32) % vocab
    for top in sorted({0, 1, min(5, vocab), min(32, vocab)}):
        _check(x, tokens, top)
    _check(x, tokens, min(3, vocab), pad=1)
    _check(x, tokens[:, :1], min(3, vocab), flat=True)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("order", ["ascending", "descending", "equal", "two values", "zeros", "steps"])
def test_orders(order, f16):
    """Rows that make the threshold work: sorted either way, all equal, ties across
    tiles, waves and splits, signed zeros."""
    announce(f"log probs order={order} f16={f16}")
    for rows, vocab in ((2, 3000), (2, 40001), (1100, 5000)):
        i = np.arange(vocab)
        x = dict(ascending=i / vocab * 20 - 10, descending=10 - i / vocab * 20, equal=np.full(vocab, 1.5),
                 zeros=np.where(i % 3 == 0, -0.0, 0.0), steps=(i // 700) % 5 * 1.0)
        x["two values"] = np.where(i % 1001 == 17, 2.0, 1.0)
        x = np.tile(x[order], (rows, 1)).astype(np.float16 if f16 else np.float32)
        x[1:] += (np.arange(1, rows) % 3)[:, None].astype(x.dtype)
        _check(x, np.array([[0, vocab - 1]] * rows, np.int32), 20)
        _check(x, np.array([[vocab // 2]] * rows, np.int32), 32)


@pytest.mark.parametrize("f16", [True, False])
def test_crowded_groups(f16):
    """Rows whose large logits lie in the columns of few threads, so that nearly all
    of these reach any threshold; runs of allowed tokens in a masked vocabulary."""
    announce(f"log probs crowded f16={f16}")
    for vocab in (32768, 30000, 131072):
        x = _x(vocab, 4, vocab, f16, 0.5)
        i = np.arange(vocab)
        x[0, i % 4096 < 8 * 160] += 8                    # 10 of 32 groups
        x[1, i % 4096 >= 4096 - 8 * 400] += 8
        x[2, :] = -np.inf
        x[2, 5000:5300] = _x(2, 1, 300, f16)[0]
        x[3, i % 4096 >= 128] = -np.inf                  # one group
        for top in (1, 12, 32):
            _check(x, np.array([[5001]] * 4, np.int32), top)


@pytest.mark.parametrize("f16", [True, False])
def test_masks(f16):
    """-inf and the type's lowest value in most places, in all but one, in all."""
    announce(f"log probs masks f16={f16}")
    low = float(np.finfo(np.float16 if f16 else np.float32).min)
    for vocab in (40, 600, 9000, 70000):
        x = _x(vocab, 9, vocab, f16)
        x[0, 3:] = -np.inf
        x[1, :] = -np.inf
        x[1, vocab - 1] = 2.0
        x[2, :] = -np.inf
        x[3, 5:] = low
        x[4, :] = low
        x[5, ::2] = -np.inf
        x[6, :vocab - 2] = low
        x[7, : vocab // 2] = -np.inf
        x[8, 1:] = -np.inf
        tokens = np.array([[0, 4, vocab - 1]] * 9, np.int32)
        got = _check(x, tokens, 5)
        assert got[1][2] == 0.0 and np.isneginf(got[0][2]).all() and got[2][2].tolist() == [0, 1, 2, 3, 4]
        assert got[0][1, 2] == 0.0 and got[1][1] == 0.0
        _check(x, tokens, 32)
        _check(x, tokens, 0)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("vocab", [40, 1984, 8192, 16384, 32768, 70000])
def test_more_keys_than_rooms(vocab, f16):
    """Rows whose threshold more logits reach than a wave has room for, in many
    workgroups at once: all equal, masked but for a few groups (which leave none),
    one group, runs of equal ones among others. Every row has its own results, with
    sums, counts and alternatives that are the same in all rows alike."""
    announce(f"log probs rooms vocab={vocab} f16={f16}")
    i = np.arange(vocab)
    x = _x(vocab, 6, vocab, f16)
    x[0, :] = 1.5
    x[1, i % 4096 >= 64 * 7] = -np.inf               # 7 of 64 groups
    x[2, 5:] = -np.inf
    x[3, i % 3 != 0] = np.float16(x[3].astype(np.float32).max()) + 1
    x[4, : vocab // 2] = -2.0
    x[4, vocab // 2:] = -3.0
    tokens = np.array([[0, vocab // 2, vocab - 1]] * 6, np.int32)
    rows = np.arange(600 if vocab <= 16384 else 300) % 6
    for top in (5, 8, 32):
        one = _check(x, tokens, top)
        many = _run(x[rows], tokens[rows], top)
        lp, entropy, best, best_lp = ref.log_probs(x, tokens, top)
        tol_lp, tol_h = ref.log_probs_tolerance(x, lp, entropy)
        _near(many[0], lp[rows], np.broadcast_to(tol_lp, lp.shape)[rows])
        _near(many[1], entropy[rows], np.broadcast_to(tol_h, entropy.shape)[rows])
        assert np.array_equal(many[2], best[rows]) and np.array_equal(one[2], best)
        _near(many[3], best_lp[rows], np.broadcast_to(ref.log_probs_tolerance(x, best_lp, entropy)[0], best_lp.shape)[rows])
        for k in range(6):                            # the same row, the same bits
            for got in many:
                assert (got[rows == k] == got[k]).all() or np.isnan(got[k]).any()


@pytest.mark.parametrize("f16", [True, False])
def test_nan_and_infinity(f16):
    """They show in their row, and only there."""
    announce(f"log probs nan f16={f16}")
    for vocab in (33, 3001, 70001):
        x = _x(vocab, 7, vocab, f16)
        x[1, vocab - 1] = np.nan
        x[2, 0] = np.inf
        x[3, :] = np.nan
        x[4, 5], x[4, 6] = np.inf, np.nan
        x[5, 2] = -np.nan
        x[5, 3] = -np.inf
        got = _check(x, np.array([[0, 3]] * 7, np.int32), 4)
        assert (got[2][[1, 2, 3, 4, 5]] == -1).all() and np.isfinite(got[3][[0, 6]]).all()
        _check(x, np.array([[0, 3]] * 7, np.int32), 0)
        _check(x, np.array([[0, 3]] * 7, np.int32), 32)
    x = np.full((1, 200000), np.nan, np.float16 if f16 else np.float32)
    assert (_check(x, np.array([[0]], np.int32), 32)[2] == -1).all()


def test_large_values():
    """f32 logits up to f32's own range, offsets that cancel, f16's range."""
    announce("log probs large")
    for scale in (1e4, 1e10, 1e30, 3e38):
        x = (dg.unit(3, 4 * 5000).reshape(4, 5000) * 2.0 - 1.0) * scale
        _check(x.astype(np.float32), np.array([[0, 77]] * 4, np.int32), 6)
    x = _x(4, 4, 5000, False, 2.0) + np.array([[0.0], [1000.0], [-5000.0], [65000.0]], np.float32)
    _check(x, np.array([[0, 77]] * 4, np.int32), 6)
    x = _x(4, 2, 5000, True, 20000.0)
    _check(x, np.array([[0, 77]] * 2, np.int32), 6)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("vocab", [700, 5000, 70000])
def test_log_probs_far_from_the_largest(vocab, f16):
    """Whole logits: their distance from the largest is exact, so that the difference to
    the sum's logarithm is rounded, and nothing else that counts."""
    announce(f"log probs far vocab={vocab} f16={f16}")
    x = np.clip(np.round(500.0 * dg.normal(vocab, (8, vocab))), -2000, 2000).astype(np.float16 if f16 else np.float32)
    tokens = (np.arange(8 * 400).reshape(8, 400) * 7919 % vocab).astype(np.int32)
    got = _run(x, tokens, 3)
    lp, _, best, best_lp = ref.log_probs(x, tokens, 3)
    # (the logarithm: of a sum of a few terms, with a few of their roundings)
    for a, b in ((got[0], lp), (got[3], best_lp)):
        assert (abs(a - b) <= 1.001 * 2.0 ** -24 * abs(b) + 2.0 ** -20).all()
    assert np.array_equal(got[2], best)


def test_given_tokens():
    """Many a row, none, negative ones (0), ones past the vocabulary (NaN)."""
    import torch
    announce("log probs tokens")
    x = _x(1, 3, 1000, True)
    tokens = dg.ints(2, (3, 700), 0, 127).astype(np.int32)
    tokens[0, :4] = -1, -100, 1000, 2 ** 31 - 1
    got = _check(x, tokens, 2)
    assert got[0][0, :2].tolist() == [0, 0] and np.isnan(got[0][0, 2:4]).all()
    bad = x.copy()
    bad[0, 0] = np.nan
    assert _run(bad, tokens, 0)[0][0, 0] == 0.0
    wide = torch.full((3, 900), 5, dtype=torch.int32, device="cuda")
    wide[:, 100:800] = dev(tokens)
    lp, h = torch.empty((3, 700), device="cuda"), torch.empty(3, device="cuda")
    T = na.tensor
    assert na.TokenLogProbs().compute([T(lp), T(h)], [T(dev(x)), T(wide[:, 100:800])]) == na.OK
    torch.cuda.synchronize()
    assert np.array_equal(host(lp), got[0], equal_nan=True)
    op = na.TokenLogProbs()
    none = torch.empty((3, 0), dtype=torch.int32, device="cuda")
    h = torch.empty(3, device="cuda")
    assert op.compute([T(none.float()), T(h)], [T(dev(x)), T(none)]) == na.OK
    torch.cuda.synchronize()
    assert np.array_equal(host(h), got[1])
    # no rows
    e = torch.empty((0, 5), device="cuda")
    assert op.compute([T(none[:0].float()), T(h[:0])], [T(e), T(none[:0])]) == na.OK


def test_results_do_not_depend_on_the_other_rows():
    """The same row alone (split) and among many (not) within their tolerance, the
    alternatives the same; the same call twice bit for bit."""
    announce("log probs alone")
    x = _x(9, 1200, 9001, True)
    tokens = dg.ints(3, (1200, 1), 0, 100).astype(np.int32)
    a, b = _run(x, tokens, 7), _run(x, tokens, 7)
    for u, v in zip(a, b):
        assert np.array_equal(u, v)
    c = _run(x[:1], tokens[:1], 7)
    assert np.array_equal(a[2][:1], c[2]) and np.max(abs(a[3][:1] - c[3])) < 1e-5 and abs(a[1][0] - c[1][0]) < 1e-4


def test_graph_and_streams():
    import torch
    announce("log probs graph")
    s = torch.cuda.Stream()
    T = na.tensor
    for rows, vocab in ((2, 60001), (1100, 900)):
        x, tokens = dev(_x(2, rows, vocab, True)), dev(np.full((rows, 1), 9, np.int32))
        outs = [torch.empty((rows, 1), device="cuda"), torch.empty(rows, device="cuda"),
                torch.empty((rows, 8), dtype=torch.int32, device="cuda"), torch.empty((rows, 8), device="cuda")]
        op = na.TokenLogProbs(top=8)
        ins, to = [T(x), T(tokens)], [T(o) for o in outs]
        ws = torch.empty(max(16, op.workspace_size(ins, to)), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        assert op.compute(to, ins, stream=s, workspace=ws) == na.OK
        torch.cuda.synchronize()
        want = [o.clone() for o in outs]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            assert op.compute(to, ins, stream=s, workspace=ws) == na.OK
        for _ in range(3):
            for o in outs:
                o.zero_()
            ws.fill_(0xff)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            for o, w in zip(outs, want):
                assert torch.equal(o, w)
