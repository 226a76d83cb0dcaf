"""The operators for continuations as they are used together: beams that fork, grow,
are given up and packed over one shared cache, against a cache of its own for each
beam (cloned by torch where a beam forks), and the example that runs them."""
from __future__ import annotations

import os
import sys

import numpy as np
import pytest

import decoder_ref as ref
import nnops_amd as na
import pages_ref
from gpu_util import announce, host

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def _run(op, outs, ins):
    assert op.compute([na.tensor(t) for t in outs], [na.tensor(t) for t in ins]) == na.OK


@pytest.mark.parametrize("page,d,hkv,group,f16", [(16, 64, 2, 4, True), (64, 128, 1, 3, True), (32, 80, 2, 1, False)])
def test_beams_share_a_cache(page, d, hkv, group, f16):
    """Every step: the codes that the tables lead to are those of the beam's own
    cache, bit for bit; PrefixAttention's results those of its own tokens; the page
    counts those of the tables, and no page is lost."""
    import torch
    announce(f"beams page={page} d={d} f16={f16}")
    r = np.random.RandomState(page + d)
    dt = torch.float16 if f16 else torch.float32
    i32 = dict(dtype=torch.int32, device="cuda")
    prompts, beams, wide, pages = 3, 4, 24, 200
    n = prompts * beams
    shared = [150, 37, 3 * page]
    cache = na.kv_cache(pages, hkv, page, d)
    refs, counts, moved = torch.zeros(pages, **i32), torch.empty(2, **i32), torch.empty(pages, **i32)
    fork, copy, compact = na.KvCacheFork(page_tokens=page), na.KvCacheCopy(), na.KvCacheCompact(page_tokens=page)
    write, attend = na.KvCacheWrite(), na.PrefixAttention()
    read = na.KvCacheRead(output_dtype=na.DT_F32)
    state = dict(table=torch.empty((0, wide), **i32), lens=torch.empty(0, **i32))

    def ints(x):
        return torch.tensor(np.asarray(x), **i32)

    def rows(t, heads):
        return torch.tensor(r.randn(t, heads * d) * np.exp(0.5 * r.randn(t, 1)), dtype=dt, device="cuda")

    def step(parents, new):
        m = len(parents)
        table, lens, copies = torch.empty((m, wide), **i32), torch.empty(m, **i32), torch.empty((m, 2), **i32)
        _run(fork, [table, lens, refs, copies, counts], [state["table"], state["lens"], refs, ints(parents), ints(new)])
        _run(copy, cache, [copies])
        state.update(table=table, lens=lens)

    # a cache of its own for each beam: pages i * wide .. and a table that never changes
    own_table = torch.arange(n * wide, **i32).reshape(n, wide)
    own = na.kv_cache(n * wide, hkv, page, d)

    def clone(parents):
        for x in own:
            y = x.reshape(n, wide, *x.shape[1:])
            y.copy_(torch.stack([y[p] if p >= 0 else torch.zeros_like(y[0]) for p in parents]))

    def check(q, starts, lens):
        """Codes and scales by reading both caches whole; attention in 64 bits."""
        m = len(lens)
        total = sum(lens)
        at = ints(np.concatenate([[0], np.cumsum(lens)]))
        got = [torch.empty((total, hkv * d), device="cuda") for _ in range(4)]
        _run(read, got[:2], list(cache) + [state["table"], state["lens"], at])
        _run(read, got[2:], list(own) + [own_table[:m].contiguous(), state["lens"], at])
        torch.cuda.synchronize()
        assert torch.equal(got[0], got[2]) and torch.equal(got[1], got[3])
        o = torch.empty_like(q)
        ins = [q, *cache, state["table"], state["lens"], ints(starts), ints(shared)]
        _run(attend, [o], ins)
        torch.cuda.synchronize()
        table = host(state["table"])
        want, weight, spread = ref.attention(host(q), *[host(x) for x in cache], table, lens, [q.shape[0] // m] * m)
        tol = ref.attention_tolerance(f16, want, weight, spread, host(cache[3]))
        assert (np.abs(host(o) - want) <= tol).all()
        assert np.array_equal(host(refs), pages_ref.holders(table, lens, page, pages))

    # the prompts, each written once; then their beams
    step([-1] * prompts, shared)
    starts = ints(np.concatenate([[0], np.cumsum(shared)]))
    k, v = rows(sum(shared), hkv), rows(sum(shared), hkv)
    _run(write, cache, [k, v, state["table"], state["lens"], starts])
    _run(write, own, [k, v, own_table[:prompts].contiguous(), state["lens"], starts])
    parents = np.repeat(np.arange(prompts), beams)
    lens = np.repeat(shared, beams)
    for i in range(9):
        new = 1 if i < 7 else page + 3
        clone(list(parents))
        step(parents, [new] * n)
        lens = lens[parents] + new if i else lens + new
        assert np.array_equal(host(state["lens"]), lens) and counts.tolist()[1] == 0
        k, v = rows(n * new, hkv), rows(n * new, hkv)
        _run(write, cache, [k, v, state["table"], state["lens"]])
        _run(write, own, [k, v, own_table, state["lens"]])
        check(rows(n * new if new == 1 else n, hkv * group), np.arange(0, n + 1, beams), [int(x) for x in lens])
        # the next beams of a prompt come from any of its own
        parents = np.concatenate([p * beams + np.sort(r.randint(0, beams, beams)) for p in range(prompts)])
        if i == 5:
            copies = torch.empty((pages // 2, 2), **i32)
            _run(compact, [state["table"], refs, copies, moved, counts], [state["table"], state["lens"], refs])
            _run(copy, cache, [copies])
            used = counts.tolist()[0]
            assert (host(refs)[:used] > 0).all() and (host(refs)[used:] == 0).all()
            check(rows(n, hkv * group), np.arange(0, n + 1, beams), [int(x) for x in lens])
    # all given up: every page is free again
    step([-1], [0])
    torch.cuda.synchronize()
    assert (host(refs) == 0).all() and counts.tolist() == [pages, 0]


def test_example_runs():
    """The example's beams: scores that are sums of log probabilities, in descending
    order, the same from call to call; the pages that they hold, packed."""
    import torch
    announce("beam search example")
    import continuations
    args = "--width 256 --heads 8 --kv-heads 2 --head-dim 64 --ffn 512 --vocab 1000 --prompts 2 --beams 3 --prompt 150 --steps 6"
    history, total, beams = continuations.main(args.split())
    again = continuations.main(args.split())
    assert torch.equal(history, again[0]) and torch.equal(total, again[1])
    assert history.shape == (2, 3, 6) and (total[:, :-1] >= total[:, 1:]).all() and (total < 0).all()
    assert len({tuple(h) for h in history[0].tolist()}) == 3
    # every page is held by the beams' tables, and only there
    used = beams.counts.tolist()[0]
    table, lens = host(beams.table), host(beams.lengths)
    assert np.array_equal(host(beams.refs), pages_ref.holders(table, lens, beams.layer.page_tokens, beams.pages))
    assert (host(beams.refs)[:used] > 0).all() and (host(beams.refs)[used:] == 0).all()
