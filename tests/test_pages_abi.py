"""PrefixAttention, KvCacheFork, KvCacheCompact, KvCacheCopy and TokenLogProbs
without a GPU: output descriptors, validate, workspace sizes and refusals at both
C layers. No call here reaches a kernel launch."""
from __future__ import annotations

import ctypes as C

import pytest

import nnops_amd as na
from nnops_amd import _lib as L
from test_abi import desc
from test_decoder_abi import cache, tables, with_

F16, F32, S8, S32 = na.DT_F16, na.DT_F32, na.DT_S8, na.DT_S32
INVALID, UNSUPPORTED = na.INVALID_ARGUMENT, na.UNSUPPORTED


def fork_descs(b=3, p=4, pages=9, n=5, wide=6):
    return ([desc([b, p], S32), desc([b], S32), desc([pages], S32), desc([n], S32), desc([n], S32)],
            [desc([n, wide], S32), desc([n], S32), desc([pages], S32), desc([n, 2], S32), desc([2], S32)])


def compact_descs(b=3, p=4, pages=9):
    return ([desc([b, p], S32), desc([b], S32), desc([pages], S32)],
            [desc([b, p], S32), desc([pages], S32), desc([pages // 2, 2], S32), desc([pages], S32), desc([2], S32)])


# --- descriptors -----------------------------------------------------------------

def test_fork_rules():
    op = na.KvCacheFork(page_tokens=16)
    ins, outs = fork_descs()
    assert op.output_descs(ins) == [([5, 4], S32), ([5], S32), ([9], S32), ([5, 2], S32), ([2], S32)]
    assert op.validate(ins, outs) == na.OK
    assert op.workspace_size(ins, outs) == 0                                      # a cache of few pages
    assert op.workspace_size(*fork_descs(pages=20000)) >= 3 * 4 * 20000 + 12 * 5
    for at, new in ((0, desc([3, 4], F32)), (0, desc([12], S32)), (1, desc([4], S32)), (1, desc([3, 1], S32)),
                    (2, desc([9, 1], S32)), (3, desc([5, 1], S32)), (4, desc([6], S32)), (4, desc([5], F32))):
        assert op.validate(with_(ins, at, new), outs) == INVALID, at
        assert op.workspace_size(with_(ins, at, new), outs) == 0
    for at, new in ((0, desc([4, 6], S32)), (0, desc([5, 6], F32)), (1, desc([4], S32)), (2, desc([8], S32)),
                    (3, desc([5, 3], S32)), (3, desc([4, 2], S32)), (4, desc([1], S32)), (4, desc([2, 1], S32))):
        assert op.validate(ins, with_(outs, at, new)) == INVALID, at
    assert op.validate(ins[:4], outs) == INVALID and op.validate(ins, outs[:4]) == INVALID
    wide = desc([5, 2], S32)
    wide.pitch = 16
    assert op.validate(ins, with_(outs, 3, wide)) == UNSUPPORTED
    for t in (0, 8, 48, 512, -16):
        assert na.KvCacheFork(page_tokens=t).validate(ins, outs) == UNSUPPORTED
    big = fork_descs(n=16385)
    assert op.validate(*big) == na.OK and op.workspace_size(*big) == 0       # (the call says unsupported)


def test_compact_rules():
    op = na.KvCacheCompact(page_tokens=32)
    ins, outs = compact_descs()
    assert op.output_descs(ins) == [([3, 4], S32), ([9], S32), ([4, 2], S32), ([9], S32), ([2], S32)]
    assert op.validate(ins, outs) == na.OK
    assert op.workspace_size(ins, outs) == 0 and op.workspace_size(*compact_descs(pages=20000)) >= 4 * 20000
    for at, new in ((0, desc([3, 5], S32)), (1, desc([8], S32)), (2, desc([5, 2], S32)), (3, desc([4], S32)),
                    (4, desc([3], S32)), (3, desc([9], F32))):
        assert op.validate(ins, with_(outs, at, new)) == INVALID, at
    assert op.validate(with_(ins, 1, desc([2], S32)), outs) == INVALID
    assert op.validate(ins + [desc([3], S32)], outs) == INVALID
    assert na.KvCacheCompact(page_tokens=33).validate(ins, outs) == UNSUPPORTED


def test_copy_rules():
    op, c = na.KvCacheCopy(), cache()
    copies = desc([7, 2], S32)
    assert op.validate([copies], c) == na.OK
    assert op.validate([desc([0, 2], S32)], c) == na.OK
    for bad in (desc([7, 3], S32), desc([14], S32), desc([7, 2], F32)):
        assert op.validate([bad], c) == INVALID
    assert op.validate([copies, copies], c) == INVALID and op.validate([copies], c[:3]) == INVALID
    assert op.validate([copies], with_(c, 1, desc([9, 2, 16, 64], S8))) == INVALID
    assert op.validate([copies], cache(page=24)) == UNSUPPORTED and op.validate([copies], cache(d=40)) == UNSUPPORTED
    wide = desc([7, 2], S32)
    wide.pitch = 12
    assert op.validate([wide], c) == UNSUPPORTED
    with pytest.raises(ValueError):
        op.output_descs([copies])                                                # the caller's


def test_prefix_attention_rules():
    op = na.PrefixAttention()
    q, c = desc([6, 512], F16), cache()
    groups = [desc([3], S32), desc([2], S32)]
    ins = [q] + c + tables() + groups
    assert op.output_descs(ins) == [([6, 512], F16)]
    assert op.validate(ins, [q]) == na.OK
    assert op.validate(ins + [desc([4], S32)], [q]) == na.OK
    assert op.workspace_size(ins, [q]) == 0                                         # little room: nothing is read once
    assert op.validate([q] + c + tables() + [desc([1], S32), desc([0], S32)], [q]) == na.OK
    for g in ([desc([2], S32), desc([2], S32)], [desc([3], F32), desc([2], S32)], [desc([3], S32), desc([2], F32)],
              [desc([3, 1], S32), desc([2], S32)], [desc([3], S32), desc([2, 1], S32)], groups[:1]):
        assert op.validate([q] + c + tables() + g, [q]) == INVALID
    assert op.validate(ins + [desc([5], S32)], [q]) == INVALID                      # row starts of 4 sequences
    assert op.validate(ins, [desc([6, 512], F32)]) == INVALID
    assert op.validate(ins, [desc([5, 512], F16)]) == INVALID
    assert op.validate([desc([7, 512], F16)] + ins[1:], [desc([7, 512], F16)]) == INVALID   # 7 rows of 3 sequences
    assert op.validate([desc([6, 500], F16)] + ins[1:], [desc([6, 500], F16)]) == INVALID
    assert op.validate([desc([6, 512], S8)] + ins[1:], [desc([6, 512], S8)]) == UNSUPPORTED
    assert na.PrefixAttention(scale=-1.0).validate(ins, [q]) == INVALID
    assert na.PrefixAttention(scale=float("nan")).validate(ins, [q]) == INVALID


def test_token_log_probs_rules():
    x, tok = desc([5, 100], F16), desc([5, 3], S32)
    assert na.TokenLogProbs().output_descs([x, tok]) == [([5, 3], F32), ([5], F32)]
    op = na.TokenLogProbs(top=4)
    want = [([5], F32), ([5], F32), ([5, 4], S32), ([5, 4], F32)]
    assert op.output_descs([x, desc([5], S32)]) == want
    outs = [desc(s, d) for s, d in op.output_descs([x, tok])]
    assert op.validate([x, tok], outs) == na.OK
    assert op.workspace_size([x, tok], outs) == 0                                 # one part a row
    wide = [desc([5, 100000], F32), tok]
    assert op.workspace_size(wide, outs) > 0
    for ins in ([x], [x, desc([4, 3], S32)], [x, desc([5, 3], F32)], [desc([500], F16), tok],
                [x, desc([5, 3, 1], S32)], [desc([5, 3], F16), tok]):
        assert op.validate(ins, outs) == INVALID
    for at, new in ((0, desc([5, 3], F16)), (0, desc([5], F32)), (1, desc([5, 1], F32)), (2, desc([5, 4], F32)),
                    (3, desc([5, 5], F32))):
        assert op.validate([x, tok], with_(outs, at, new)) == INVALID
    assert op.validate([x, tok], outs[:2]) == INVALID and na.TokenLogProbs().validate([x, tok], outs) == INVALID
    assert op.validate([desc([5, 100], S8), tok], outs) == UNSUPPORTED
    for vocab, status in ((1 << 21, na.OK), ((1 << 21) + 1, UNSUPPORTED)):
        assert op.validate([desc([5, vocab], F16), tok], outs) == status
    many = na.TokenLogProbs(top=33)
    assert many.validate([x, tok], [desc(s, d) for s, d in many.output_descs([x, tok])]) == UNSUPPORTED
    assert na.TokenLogProbs(top=-1).validate([x, tok], outs[:2]) == INVALID


@pytest.mark.parametrize("rows,vocab,status", [
    (1 << 22, 100, na.OK), ((1 << 22) + 1, 100, UNSUPPORTED), ((1 << 22) - 1, 33000, na.OK), (1 << 22, 33000, UNSUPPORTED),
    (1 << 17, 1 << 21, UNSUPPORTED), ((1 << 17) - 1, 1 << 21, na.OK),
])
def test_token_log_probs_rows(rows, vocab, status):
    """validate says what the call says of rows, and of rows times parts."""
    op, lib = na.TokenLogProbs(), na.lib()
    ins, outs = [desc([rows, vocab], F16), desc([rows], S32)], [desc([rows], F32), desc([rows], F32)]
    assert op.validate(ins, outs) == status
    a = probs_args(rows=rows, vocab=vocab, ld_logits=vocab, top=0, logits=None)
    assert lib.nnops_hip_token_log_probs(C.byref(a), None, 0, None) == (INVALID if status == na.OK else status)


# --- the launch boundary: refusals before any launch -------------------------------

BASE = 1 << 20                 # addresses that nothing is read from: 1 MB apart


def args(cls, **kw):
    a = cls()
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def fork_args(**kw):
    at = {n: BASE * (i + 1) for i, n in enumerate(("page_table", "lengths", "refs", "parents", "new_tokens", "new_table",
                                                   "new_lengths", "new_refs", "copies", "counts"))}
    at.update(sequences=3, table_pages=4, ld_table=4, pages=9, page_tokens=16, children=5, new_table_pages=6,
              ld_new_table=6)
    at.update(kw)
    return args(L.KvForkArgs, **at)


def compact_args(**kw):
    at = {n: BASE * (i + 1) for i, n in enumerate(("page_table", "lengths", "refs", "new_table", "new_refs", "copies",
                                                   "moved", "counts"))}
    at.update(sequences=3, table_pages=4, ld_table=4, pages=9, page_tokens=16, ld_new_table=4)
    at.update(kw)
    return args(L.KvCompactArgs, **at)


@pytest.mark.parametrize("kw,status", [
    (dict(sequences=-1), INVALID), (dict(children=-1), INVALID), (dict(pages=-1), INVALID), (dict(table_pages=-1), INVALID),
    (dict(new_table_pages=-2), INVALID), (dict(page_tokens=24), UNSUPPORTED), (dict(children=16385), UNSUPPORTED),
    (dict(sequences=16385), UNSUPPORTED), (dict(pages=1 << 30), UNSUPPORTED), (dict(table_pages=1 << 28), UNSUPPORTED),
    (dict(ld_table=3), INVALID), (dict(ld_new_table=5), INVALID), (dict(counts=None), INVALID), (dict(refs=None), INVALID),
    (dict(lengths=None), INVALID), (dict(parents=None), INVALID), (dict(new_table=None), INVALID),
    (dict(new_table=BASE), INVALID),                          # children over their parents
    (dict(new_table=BASE + 44), INVALID),
    (dict(new_lengths=2 * BASE), INVALID), (dict(copies=10 * BASE - 4), INVALID), (dict(new_refs=3 * BASE + 4), INVALID),
    (dict(new_refs=4 * BASE), INVALID),
    (dict(children=16384, new_table_pages=1 << 16, ld_new_table=1 << 16), UNSUPPORTED),    # 2^30 cells
])
def test_fork_call_refusals(kw, status):
    lib, a = na.lib(), fork_args(**kw)
    assert lib.nnops_hip_kv_cache_fork(C.byref(a), C.c_void_p(99 * BASE), 1 << 20, None) == status


def test_fork_workspace():
    lib, a = na.lib(), fork_args(new_refs=3 * BASE, pages=20000)   # counts in place: not refused
    need = lib.nnops_hip_kv_cache_fork_workspace_size(C.byref(a))
    assert need > 0
    for at, size in ((None, need), (99 * BASE, need - 1), (99 * BASE + 8, need)):
        assert lib.nnops_hip_kv_cache_fork(C.byref(a), C.c_void_p(at), size, None) == na.NOT_INITIALIZED
    assert lib.nnops_hip_kv_cache_fork(None, None, 0, None) == INVALID
    assert lib.nnops_hip_kv_cache_fork_workspace_size(None) == 0


@pytest.mark.parametrize("kw,status", [
    (dict(sequences=-1), INVALID), (dict(pages=-1), INVALID), (dict(page_tokens=0), UNSUPPORTED),
    (dict(pages=1 << 30), UNSUPPORTED), (dict(ld_table=3), INVALID), (dict(ld_new_table=3), INVALID),
    (dict(counts=None), INVALID), (dict(copies=None), INVALID), (dict(moved=None), INVALID), (dict(page_table=None), INVALID),
    (dict(new_table=BASE, ld_new_table=5), INVALID),          # in place at another pitch
    (dict(new_table=BASE + 4), INVALID), (dict(new_refs=3 * BASE + 4), INVALID), (dict(moved=3 * BASE), INVALID),
    (dict(new_refs=7 * BASE), INVALID), (dict(counts=6 * BASE + 4), INVALID),
])
def test_compact_call_refusals(kw, status):
    lib, a = na.lib(), compact_args(**kw)
    assert lib.nnops_hip_kv_cache_compact(C.byref(a), C.c_void_p(99 * BASE), 1 << 20, None) == status


def test_compact_workspace():
    lib, a = na.lib(), compact_args(new_table=BASE, new_refs=3 * BASE, pages=20000)
    need = lib.nnops_hip_kv_cache_compact_workspace_size(C.byref(a))
    for at, size in ((None, need), (99 * BASE, need - 1), (99 * BASE + 4, need)):
        assert lib.nnops_hip_kv_cache_compact(C.byref(a), C.c_void_p(at), size, None) == na.NOT_INITIALIZED


@pytest.mark.parametrize("sequences,status", [(0, na.NOT_INITIALIZED), (1, na.NOT_INITIALIZED), (2, INVALID)])
def test_compact_in_place_pitch(sequences, status):
    """A table of one row, or of none, has no pitch that could differ."""
    lib, a = na.lib(), compact_args(sequences=sequences, new_table=BASE, ld_new_table=7, pages=20000)
    assert lib.nnops_hip_kv_cache_compact(C.byref(a), None, 0, None) == status


def copy_args(**kw):
    at = dict(k=BASE, v=2 * BASE, k_scale=3 * BASE, v_scale=4 * BASE, copies=5 * BASE, pages=9, heads=2, page_tokens=16,
              head_dim=64, count=3)
    at.update(kw)
    return args(L.KvCopyArgs, **at)


@pytest.mark.parametrize("kw,status", [
    (dict(count=-1), INVALID), (dict(pages=-1), INVALID), (dict(heads=-1), INVALID), (dict(page_tokens=24), UNSUPPORTED),
    (dict(head_dim=40), UNSUPPORTED), (dict(head_dim=272), UNSUPPORTED), (dict(heads=1 << 17), UNSUPPORTED),
    (dict(k=None), INVALID), (dict(v=2 * BASE + 8), INVALID), (dict(k_scale=None), INVALID), (dict(copies=None), INVALID),
    (dict(count=0, copies=None), na.OK), (dict(pages=0, k=None), na.OK), (dict(heads=0), na.OK),
])
def test_copy_call_refusals(kw, status):
    a = copy_args(**kw)
    assert na.lib().nnops_hip_kv_cache_copy(C.byref(a), None) == status


def prefix_args(**kw):
    c = args(L.KvPages, k=BASE, v=2 * BASE, k_scale=3 * BASE, v_scale=4 * BASE, pages=9, heads=2, page_tokens=16,
             head_dim=64, page_table=5 * BASE, sequences=3, table_pages=4, ld_table=4, lengths=6 * BASE)
    for k in list(kw):
        if hasattr(c, k):
            setattr(c, k, kw.pop(k))
    at = dict(cache=c, q=7 * BASE, out=8 * BASE, rows=6, q_heads=8, ld_q=512, ld_out=512, f16=1, groups=2,
              group_starts=9 * BASE, shared=10 * BASE)
    at.update(kw)
    return args(L.PrefixAttentionArgs, **at)


@pytest.mark.parametrize("kw,status", [
    (dict(groups=-1), INVALID), (dict(groups=1 << 25), UNSUPPORTED), (dict(rows=-1), INVALID), (dict(q_heads=7), INVALID),
    (dict(q_heads=0), INVALID), (dict(scale=-1.0), INVALID), (dict(scale=float("nan")), INVALID),
    (dict(group_starts=None), INVALID), (dict(shared=None), INVALID), (dict(q=None), INVALID), (dict(ld_out=511), INVALID),
    (dict(page_tokens=24), UNSUPPORTED), (dict(head_dim=24), UNSUPPORTED), (dict(rows=7), INVALID), (dict(pages=0), INVALID),
    (dict(k=BASE + 8), INVALID), (dict(lengths=None), INVALID), (dict(ld_table=3), INVALID), (dict(rows=0), na.OK),
    (dict(sequences=0), INVALID),
])
def test_prefix_call_refusals(kw, status):
    lib, a = na.lib(), prefix_args(**kw)
    assert lib.nnops_hip_prefix_attention(C.byref(a), C.c_void_p(99 * BASE), 1 << 40, None) == status


def test_prefix_workspace():
    lib, a = na.lib(), prefix_args()
    assert lib.nnops_hip_prefix_attention_workspace_size(C.byref(a)) == 0      # a table of so little room
    a = prefix_args(table_pages=16000, ld_table=16000)
    need = lib.nnops_hip_prefix_attention_workspace_size(C.byref(a))
    assert need >= 2 * 6 * 8 * 66 * 4                         # a part of the prefix's and one of its own for every row
    for at, size in ((None, need), (99 * BASE, need - 1), (99 * BASE + 8, need)):
        assert lib.nnops_hip_prefix_attention(C.byref(a), C.c_void_p(at), size, None) == na.NOT_INITIALIZED
    a.rows = 7
    assert lib.nnops_hip_prefix_attention_workspace_size(C.byref(a)) == 0


def probs_args(**kw):
    at = dict(logits=BASE, rows=5, vocab=100, ld_logits=100, f16=1, top=4, tokens=2 * BASE, per_row=3, ld_tokens=3,
              log_probs=3 * BASE, ld_log_probs=3, entropy=4 * BASE, top_tokens=5 * BASE, top_log_probs=6 * BASE,
              ld_top_tokens=4, ld_top_log_probs=4)
    at.update(kw)
    return args(L.TokenLogProbsArgs, **at)


@pytest.mark.parametrize("kw,status", [
    (dict(rows=-1), INVALID), (dict(vocab=-1), INVALID), (dict(per_row=-1), INVALID), (dict(top=-1), INVALID),
    (dict(top=101), INVALID), (dict(top=33), UNSUPPORTED), (dict(vocab=0, top=0), INVALID), (dict(rows=1 << 23), UNSUPPORTED),
    (dict(vocab=(1 << 21) + 1, ld_logits=1 << 22), UNSUPPORTED), (dict(ld_logits=99), INVALID), (dict(logits=None), INVALID), (dict(entropy=None), INVALID), (dict(tokens=None), INVALID),
    (dict(log_probs=None), INVALID), (dict(ld_tokens=2), INVALID), (dict(top_tokens=None), INVALID),
    (dict(ld_top_log_probs=3), INVALID), (dict(rows=0), na.OK),
    (dict(rows=1 << 22, vocab=33000, ld_logits=33000), UNSUPPORTED),                       # threads past 2^32
])
def test_probs_call_refusals(kw, status):
    a = probs_args(**kw)
    assert na.lib().nnops_hip_token_log_probs(C.byref(a), None, 0, None) == status


def test_probs_workspace():
    lib, a = na.lib(), probs_args(vocab=100000, ld_logits=100000)
    need = lib.nnops_hip_token_log_probs_workspace_size(C.byref(a))
    assert need > 0
    for at, size in ((None, need), (99 * BASE, need - 1), (99 * BASE + 8, need)):
        assert lib.nnops_hip_token_log_probs(C.byref(a), C.c_void_p(at), size, None) == na.NOT_INITIALIZED


def test_other_backends_are_refused():
    x, tok = desc([5, 100], F16), desc([5], S32)
    for cls, kw, ins, outs in ((na.KvCacheFork, dict(page_tokens=16), *fork_descs()),
                               (na.KvCacheCompact, dict(page_tokens=16), *compact_descs()),
                               (na.TokenLogProbs, {}, [x, tok], [desc([5], F32), desc([5], F32)])):
        for t in ins + outs:
            t.data = 16
        assert cls(**kw, backend=na.BACKEND_CPU).compute(outs, ins, workspace=16, stream=1) == UNSUPPORTED
