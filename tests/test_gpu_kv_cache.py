"""KvCacheWrite and KvCacheRead: the codes and scales equal, bit for bit, to
the same f32 operations on the CPU; values within half a step of the rows;
ragged rows, partly filled pages, pages whose scale grows, rows that stand for
no token, pages that do not exist, infinities and NaNs, caches past 2^31
bytes."""
from __future__ import annotations

import numpy as np
import pytest

import datagen as dg
import decoder_ref as ref
import nnops_amd as na
from gpu_util import dev, host, pitched, announce

pytestmark = pytest.mark.gpu


class Cache:
    """A device cache and the same on the CPU; pages handed out in a shuffled order."""

    def __init__(self, seqs, tokens, heads, page, d, seed=1, spare=3):
        per = -(-tokens // page)
        n = seqs * per + spare
        self.page, self.heads, self.d = page, heads, d
        self.t = na.kv_cache(n, heads, page, d)
        self.k, self.v = np.zeros((n, heads, page, d), np.int8), np.zeros((n, heads, page, d), np.int8)
        self.ks, self.vs = np.zeros((n, heads), np.float32), np.zeros((n, heads), np.float32)
        order = np.argsort(dg.unit(seed, n))
        self.table = order[:seqs * per].reshape(seqs, per).astype(np.int32)
        self.n = n

    def descs(self):
        return [na.tensor(x) for x in self.t]

    def fill(self, seed):
        """Codes and scales of earlier tokens everywhere."""
        import torch
        self.k[:] = dg.ints(seed, self.k.shape, -127, 127)
        self.v[:] = dg.ints(seed + 1, self.v.shape, -127, 127)
        self.ks[:] = dg.uniform(seed + 2, self.ks.shape, 0.005, 0.03)
        self.vs[:] = dg.uniform(seed + 3, self.vs.shape, 0.005, 0.03)
        for t, x in zip(self.t, (self.k, self.v.transpose(0, 1, 3, 2), self.ks, self.vs)):
            t.copy_(torch.from_numpy(np.ascontiguousarray(x)))

    def write(self, k, v, lens, rows, ragged=True, pad=0, table=None):
        """Both sides; returns nothing, the two are compared by same()."""
        table = self.table if table is None else table
        starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        ins = [na.tensor(pitched(k, k.shape[1] + pad)), na.tensor(pitched(v, v.shape[1] + 2 * pad)),
               na.tensor(dev(table)), na.tensor(dev(np.array(lens, np.int32)))]
        ins += [na.tensor(dev(starts))] if ragged else []
        op = na.KvCacheWrite()
        assert op.validate(ins, self.descs()) == na.OK
        assert op.compute(self.descs(), ins) == na.OK
        ref.kv_write(k, self.k, self.ks, table, lens, rows)
        ref.kv_write(v, self.v, self.vs, table, lens, rows)

    def same(self, lens, table=None):
        """Equal in every slot that holds a token, and in every scale."""
        import torch
        torch.cuda.synchronize()
        table = self.table if table is None else table
        k, v, ks, vs = [host(t) for t in self.t]
        v = v.transpose(0, 1, 3, 2)
        assert np.array_equal(ks, self.ks, equal_nan=True) and np.array_equal(vs, self.vs, equal_nan=True)
        for b, length in enumerate(lens):
            for p in range(-(-length // self.page)):
                pid, n = table[b][p], min(self.page, length - p * self.page)
                if 0 <= pid < self.n:
                    assert np.array_equal(k[pid, :, :n], self.k[pid, :, :n]), (b, p)
                    assert np.array_equal(v[pid, :, :n], self.v[pid, :, :n]), (b, p)

    def read(self, lens, rows, f16, ragged=True, pad=0, table=None):
        import torch
        table = self.table if table is None else table
        starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        width, t = self.heads * self.d, int(sum(rows))
        dt = np.float16 if f16 else np.float32
        k, v = (pitched(np.full((t, width), 9, dt), width + (i + 1) * pad) for i in range(2))
        ins = self.descs() + [na.tensor(dev(table)), na.tensor(dev(np.array(lens, np.int32)))]
        ins += [na.tensor(dev(starts))] if ragged else []
        op = na.KvCacheRead(output_dtype=na.DT_F16 if f16 else na.DT_F32)
        outs = [na.tensor(k), na.tensor(v)]
        assert op.validate(ins, outs) == na.OK
        assert op.compute(outs, ins) == na.OK
        torch.cuda.synchronize()
        for got, codes, scale in ((host(k), self.k, self.ks), (host(v), self.v, self.vs)):
            want = ref.kv_read(codes, scale, table, lens, rows)
            half, least = (2.0 ** -11, 2.0 ** -25) if f16 else (2.0 ** -24, 0.0)
            assert np.array_equal(np.isnan(got), np.isnan(want))
            ok = ~np.isnan(want)
            assert np.all(abs(got[ok].astype(np.float64) - want[ok]) <= (half + 2.0 ** -24) * abs(want[ok]) + least)
        return host(k), host(v)


def _rows(seed, t, width, f16):
    """Rows of different sizes, so that scales grow now and then."""
    x = dg.normal(seed, (t, width)) * np.exp(dg.normal(seed + 50, (t, 1)))
    return x.astype(np.float16 if f16 else np.float32)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("page,d,heads", [(16, 128, 2), (32, 80, 3), (64, 64, 1), (128, 16, 2), (256, 256, 1),
                                          (64, 96, 8)])
def test_prompt_then_tokens(page, d, heads, f16):
    """A ragged prompt (a sequence without rows among it), then chunks and single
    tokens that fill pages and begin new ones."""
    announce(f"cache page={page} d={d} heads={heads} f16={f16}")
    seqs, width = 4, heads * d
    c = Cache(seqs, 3 * page + 40, heads, page, d)
    lens = np.array([page + 1, 3, 0, 2 * page])
    c.write(_rows(1, lens.sum(), width, f16), _rows(2, lens.sum(), width, f16), lens, lens)
    c.same(lens)
    for step, rows in enumerate([(1, 0, 1, 1), (13, 13, 13, 13), (1, 1, 1, 1), (1, 1, 1, 1), (0, 20, 1, 17)]):
        rows = np.array(rows)
        lens = lens + rows
        ragged = len(set(rows)) > 1
        c.write(_rows(10 + step, rows.sum(), width, f16), _rows(30 + step, rows.sum(), width, f16), lens, rows,
                ragged=ragged, pad=step)
        c.same(lens)
    c.read(lens, lens, f16)
    c.read(lens, np.minimum(lens, 5), not f16, pad=3)


def test_values_within_half_a_step():
    """A prompt read back: each value within half a step of its page's scale, and
    the scale no larger than the page's rows need."""
    announce("cache values")
    page, heads, d, n = 32, 2, 64, 100
    c = Cache(1, n, heads, page, d)
    k, v = _rows(3, n, heads * d, False), _rows(4, n, heads * d, False)
    c.write(k, v, [n], [n])
    gk, gv = c.read([n], [n], False)
    for x, got, scale in ((k, gk, c.ks), (v, gv, c.vs)):
        for p in range(-(-n // page)):
            rows = slice(p * page, min(n, (p + 1) * page))
            for h in range(heads):
                cols = slice(h * d, (h + 1) * d)
                s = scale[c.table[0, p], h].astype(np.float64)
                top = abs(x[rows, cols]).max()
                assert abs(s - top / 127) <= 2.0 ** -23 * s
                assert np.all(abs(got[rows, cols] - x[rows, cols].astype(np.float64)) <= (0.5 + 2.0 ** -16) * s)


def test_same_call_twice():
    """Tokens written again at their places change nothing; the same inputs give
    the same bits."""
    announce("cache written twice")
    page, heads, d = 64, 2, 128
    c = Cache(2, 200, heads, page, d)
    c.fill(5)
    lens, rows = [100, 131], [1, 40]
    k, v = _rows(6, 41, heads * d, True), _rows(7, 41, heads * d, True)
    c.write(k, v, lens, rows)
    c.same(lens)
    before = [host(t).copy() for t in c.t]
    c.write(k, v, lens, rows)
    c.same(lens)
    assert all(np.array_equal(a, host(t)) for a, t in zip(before, c.t))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_no_numbers(bad):
    """A row with no number in one head: that head's page says so, also after
    more tokens; the other heads, the other side and the next page do not."""
    announce(f"cache {bad}")
    page, heads, d = 16, 2, 32
    c = Cache(1, 40, heads, page, d)
    k, v = _rows(8, 8, heads * d, False), _rows(9, 8, heads * d, False)
    c.write(k, v, [8], [8])
    k1, v1 = _rows(10, 1, heads * d, False), _rows(11, 1, heads * d, False)
    k1[0, d + 5] = bad
    c.write(k1, v1, [9], [1])
    c.same([9])
    assert np.isnan(c.ks[c.table[0, 0], 1]) and np.isfinite(c.ks[c.table[0, 0], 0])
    c.write(_rows(12, 10, heads * d, False), _rows(13, 10, heads * d, False), [19], [10])
    c.same([19])
    gk, gv = c.read([19], [19], False)
    assert np.isnan(gk[:16, d:]).all() and np.isfinite(gk[:, :d]).all() and np.isfinite(gk[16:]).all()
    assert np.isfinite(gv).all()


def test_pages_of_nothing():
    """Zeros, and values below the smallest scale: a positive scale, codes 0,
    and numbers once there are some."""
    announce("cache zeros")
    page, heads, d = 16, 1, 16
    c = Cache(1, 16, heads, page, d)
    z = np.zeros((3, d), np.float32)
    tiny = np.full((3, d), 1e-38, np.float32)
    c.write(z, tiny, [3], [3])
    c.same([3])
    pid = c.table[0, 0]
    assert c.ks[pid, 0] == ref.LEAST_SCALE and c.vs[pid, 0] == ref.LEAST_SCALE
    c.write(_rows(1, 2, d, False), _rows(2, 2, d, False), [5], [2])
    c.same([5])
    gk, gv = c.read([5], [5], False)
    assert np.all(gk[:3] == 0) and np.all(gv[:3] == 0) and np.any(gk[3:] != 0)


def test_rows_and_pages_that_are_not_there():
    """More rows than tokens (the first read as zeros and are not written), no
    tokens at all, page numbers outside the cache, a length past the table."""
    announce("cache absent rows and pages")
    page, heads, d = 16, 2, 32
    c = Cache(3, 48, heads, page, d)
    c.fill(20)
    table = c.table.copy()
    table[1, 1], table[2, 0] = -1, c.n
    lens, rows = [4, 40, 20], [10, 33, 20]
    k, v = _rows(21, 63, heads * d, True), _rows(22, 63, heads * d, True)
    c.write(k, v, lens, rows, table=table)
    c.same(lens, table=table)
    gk, _ = c.read(lens, rows, True, table=table)
    assert np.all(gk[:6] == 0) and np.isnan(gk[10 + 16 - 7:10 + 32 - 7]).all()
    c.read([0, 1, 16], [5, 0, 2], False, table=c.table)
    gk, _ = c.read([0, 0, 0], [2, 2, 2], False, ragged=False)
    assert np.all(gk == 0)
    # 1000 is past the table's 48 tokens: its end
    starts = dev(np.array([0, 0, 0, 2], np.int32))
    import torch
    k = torch.zeros((2, heads * d), device="cuda")
    v = torch.zeros((2, heads * d), device="cuda")
    ins = c.descs() + [na.tensor(dev(c.table)), na.tensor(dev(np.array([0, 0, 1000], np.int32))), na.tensor(starts)]
    assert na.KvCacheRead(output_dtype=na.DT_F32).compute([na.tensor(k), na.tensor(v)], ins) == na.OK
    torch.cuda.synchronize()
    want = ref.kv_read(c.k, c.ks, c.table[2:], [48], [2])
    assert np.all(abs(host(k) - want) <= 2.0 ** -23 * abs(want))


@pytest.mark.parametrize("seqs", [1, 63, 64, 65, 200])
def test_many_sequences(seqs):
    """The search for a workgroup's sequence over one and several steps of 64."""
    announce(f"cache {seqs} sequences")
    page, heads, d = 16, 1, 16
    c = Cache(seqs, 60, heads, page, d)
    rows = dg.ints(seqs, (seqs,), 0, 40).astype(np.int64)
    rows[::7] = 0
    lens = rows + dg.ints(seqs + 1, (seqs,), 0, 20).astype(np.int64)
    c.fill(9)
    c.write(_rows(1, rows.sum(), d, True), _rows(2, rows.sum(), d, True), lens, rows)
    c.same(lens)
    c.read(lens, lens, True)


def test_cache_past_2_gib():
    """Pages whose bytes begin past 2^31 (and past 2^32) of each side."""
    import torch
    announce("cache past 2^32 bytes")
    page, heads, d = 128, 8, 128
    n = (1 << 32) // (heads * page * d) + 40
    kc, vc = (torch.empty((n,) + s, dtype=torch.int8, device="cuda") for s in ((heads, page, d), (heads, d, page)))
    ks, vs = (torch.zeros((n, heads), device="cuda") for _ in range(2))
    table = np.array([[n - 1, 5, n // 2 + 3]], np.int32)
    t = 300
    x, y = _rows(1, t, heads * d, True), _rows(2, t, heads * d, True)
    cache = [na.tensor(z) for z in (kc, vc, ks, vs)]
    where = [na.tensor(dev(table)), na.tensor(dev(np.array([t], np.int32)))]
    assert na.KvCacheWrite().compute(cache, [na.tensor(dev(x)), na.tensor(dev(y))] + where) == na.OK
    gk, gv = (torch.zeros((t, heads * d), dtype=torch.float16, device="cuda") for _ in range(2))
    assert na.KvCacheRead().compute([na.tensor(gk), na.tensor(gv)], cache + where) == na.OK
    torch.cuda.synchronize()
    k, s = np.zeros((3, heads, page, d), np.int8), np.zeros((3, heads), np.float32)
    for rows, got in ((x, gk), (y, gv)):
        ref.kv_write(rows, k, s, [[0, 1, 2]], [t], [t])
        want = ref.kv_read(k, s, [[0, 1, 2]], [t], [t])
        assert np.all(abs(host(got).astype(np.float64) - want) <= 2.0 ** -11 * 1.01 * abs(want) + 2.0 ** -25)
