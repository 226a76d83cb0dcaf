"""Rotary and its table against 64 bits: both pairings, parts of a head, odd
head sizes, both types, pitched rows, in place, positions outside the table."""
from __future__ import annotations

import math

import numpy as np
import pytest

import datagen as dg
import decoder_ref as ref
import nnops_amd as na
from gpu_util import dev, host, pitched, announce

pytestmark = pytest.mark.gpu


def _table(most, rot):
    f = 10000.0 ** (-2.0 * np.arange(rot // 2) / rot)
    a = np.arange(most)[:, None] * f
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


def _tol(f16, want, size):
    # two products, a sum, the type
    return 2.0 ** -23 * size + (2.0 ** -11 * abs(want) + 2.0 ** -25 if f16 else 0.0)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 32), (80, 80), (80, 40), (96, 96), (256, 128), (6, 6), (10, 4),
                                   (7, 2), (128, 126)])
def test_shapes(d, rot, interleaved, f16):
    import torch
    announce(f"rotary d={d} rot={rot} interleaved={interleaved} f16={f16}")
    t, heads, most = 37, 5, 5000
    x = dg.normal(d + rot, (t, heads * d)).astype(np.float16 if f16 else np.float32)
    pos = dg.ints(3, (t,), 0, most - 1, np.int32)
    pos[0], pos[1] = 0, most - 1
    table = _table(most, rot)
    want, size = ref.rotary(x, pos, table, heads, d, rot, interleaved)
    op = na.Rotary(head_dim=d, rotary_dim=rot, interleaved=interleaved)
    for pad in (0, 3):
        dx = pitched(x, heads * d + pad)
        y = pitched(np.zeros_like(x), heads * d + 2 * pad)
        ins = [na.tensor(dx), na.tensor(dev(pos)), na.tensor(pitched(table, rot + pad))]
        assert op.validate(ins, [na.tensor(y)]) == na.OK
        assert op.compute([na.tensor(y)], ins) == na.OK
        assert op.compute([na.tensor(dx)], ins) == na.OK          # in place
        torch.cuda.synchronize()
        assert np.all(abs(host(y).astype(np.float64) - want) <= _tol(f16, want, size))
        assert np.array_equal(host(y), host(dx))
        keep = want.reshape(t, heads, d)[..., rot:]
        assert np.array_equal(host(y).reshape(t, heads, d)[..., rot:].astype(np.float64), keep)


def test_packed_projection():
    """The q and k heads of a fused projection's rows in one call; the v heads
    beside them stay."""
    import torch
    announce("rotary in a packed projection")
    t, d, heads = 9, 64, 6
    full = dg.normal(5, (t, (heads + 2) * d)).astype(np.float16)
    pos = np.arange(100, 100 + t, dtype=np.int32)
    table = _table(200, d)
    buf = dev(full)
    x = buf[:, :heads * d]
    op = na.Rotary(head_dim=d)
    assert op.compute([na.tensor(x)], [na.tensor(x), na.tensor(dev(pos)), na.tensor(dev(table))]) == na.OK
    torch.cuda.synchronize()
    want, size = ref.rotary(full[:, :heads * d], pos, table, heads, d, d, False)
    got = host(buf)
    assert np.all(abs(got[:, :heads * d].astype(np.float64) - want) <= _tol(True, want, size))
    assert np.array_equal(got[:, heads * d:], full[:, heads * d:])


def test_positions_outside_the_table():
    import torch
    announce("rotary positions outside")
    d, rot = 32, 16
    x = dg.normal(6, (4, d)).astype(np.float32)
    pos = np.array([-1, 3, 10, 2 ** 31 - 1], dtype=np.int32)
    y = torch.zeros((4, d), device="cuda")
    op = na.Rotary(head_dim=d, rotary_dim=rot)
    assert op.compute([na.tensor(y)], [na.tensor(dev(x)), na.tensor(dev(pos)), na.tensor(dev(_table(10, rot)))]) == na.OK
    torch.cuda.synchronize()
    got = host(y)
    assert np.isnan(got[[0, 2, 3], :rot]).all() and np.array_equal(got[:, rot:], x[:, rot:])
    assert np.isfinite(got[1]).all()


def test_one_token_and_many():
    import torch
    d, heads, most = 128, 40, 64
    table = dev(_table(most, d))
    op = na.Rotary(head_dim=d)
    for t in (1, 3000):
        announce(f"rotary {t} tokens")
        x = dg.normal(7, (t, heads * d)).astype(np.float16)
        pos = (np.arange(t) % most).astype(np.int32)
        y = torch.zeros((t, heads * d), dtype=torch.float16, device="cuda")
        assert op.compute([na.tensor(y)], [na.tensor(dev(x)), na.tensor(dev(pos)), na.tensor(table)]) == na.OK
        torch.cuda.synchronize()
        want, size = ref.rotary(x, pos, host(table), heads, d, d, False)
        assert np.all(abs(host(y).astype(np.float64) - want) <= _tol(True, want, size))


@pytest.mark.parametrize("kw", [dict(), dict(base=500000.0), dict(factor=4.0),
                                dict(factor=8.0, original_context=8192, low_turns=1.0, high_turns=4.0),
                                dict(factor=16.0, original_context=4096, low_turns=1.0, high_turns=32.0,
                                     attention_factor=0.1 * math.log(16.0) + 1.0)])
def test_table(kw):
    """Against angles in 64 bits at positions up to a million: the table's values
    are the cosines and sines rounded once (an angle of 10^6 has 2^-33 left
    after the 2^-53 of its factors)."""
    import torch
    announce(f"rotary table {kw}")
    rot, most = 128, 1 << 20
    got = na.rotary_table(most, rot, **kw)
    torch.cuda.synchronize()
    base, factor, ctx = kw.get("base", 10000.0), kw.get("factor", 1.0), kw.get("original_context", 0)
    f = base ** (-2.0 * np.arange(rot // 2) / rot)
    g = np.ones_like(f)
    if factor != 1.0:
        g = np.zeros_like(f)
        if ctx:
            lo, hi = kw["low_turns"], kw["high_turns"]
            g = np.clip((ctx * f / (2 * math.pi) - lo) / (hi - lo), 0.0, 1.0)
    f = g * f + (1 - g) * f / factor
    rows = np.array([0, 1, 2, 1000, 4097, 65535, 777777, most - 1])
    a = rows[:, None] * f
    m = kw.get("attention_factor", 1.0)
    want = m * np.concatenate([np.cos(a), np.sin(a)], 1)
    assert np.all(abs(host(got[torch.from_numpy(rows).cuda()]) - want) <= m * (2.0 ** -24 + 2.0 ** -30))
