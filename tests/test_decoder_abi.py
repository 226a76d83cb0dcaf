"""RmsNorm, Rotary, KvCacheWrite, KvCacheRead and CacheAttention without a GPU:
output descriptors, validate, workspace sizes and refusals at both C layers. No
call here reaches a kernel launch."""
from __future__ import annotations

import ctypes as C

import pytest

import nnops_amd as na
from nnops_amd import _lib as L
from test_abi import desc

F16, F32, S8, S32 = na.DT_F16, na.DT_F32, na.DT_S8, na.DT_S32


def cache(pages=9, heads=2, page=16, d=64):
    return [desc([pages, heads, page, d], S8), desc([pages, heads, d, page], S8), desc([pages, heads], F32),
            desc([pages, heads], F32)]


def tables(seqs=3, per=4, starts=False):
    t = [desc([seqs, per], S32), desc([seqs], S32)]
    return t + [desc([seqs + 1], S32)] if starts else t


def with_(descs, at, new):
    return descs[:at] + [new] + descs[at + 1:]


# --- descriptors ---------------------------------------------------------------

def test_rms_norm_descriptors():
    x, w = desc([2, 5, 64], F16), desc([64], F16)
    op = na.RmsNorm(output_dtype=S8)
    assert op.output_descs([x, w]) == [([2, 5, 64], S8), ([10], F32)]
    assert op.output_descs([x, w, x]) == [([2, 5, 64], S8), ([10], F32), ([2, 5, 64], F16)]
    assert na.RmsNorm().output_descs([x, w, x]) == [([2, 5, 64], F16), ([2, 5, 64], F16)]
    assert op.output_desc([x, w]) == ([2, 5, 64], S8)
    assert op.validate([x, w], [desc([2, 5, 64], S8), desc([10], F32)]) == na.OK
    assert op.workspace_size([x, w], [desc([2, 5, 64], S8), desc([10], F32)]) == 0


@pytest.mark.parametrize("ins,outs,status", [
    ([([4, 8], F16)], [([4, 8], F16)], na.INVALID_ARGUMENT),                                  # no weight
    ([([4, 8], F16), ([7], F16)], [([4, 8], F16)], na.INVALID_ARGUMENT),                      # weight's size
    ([([4, 8], F16), ([8], F32)], [([4, 8], F16)], na.INVALID_ARGUMENT),                      # weight's type
    ([([4, 8], F32), ([8], F32)], [([4, 8], F16)], na.UNSUPPORTED),                           # f32 to f16
    ([([4, 8], S8), ([8], S8)], [([4, 8], F16)], na.UNSUPPORTED),
    ([([4, 8], F16), ([8], F16)], [([4, 9], F16)], na.INVALID_ARGUMENT),
    ([([4, 8], F16), ([8], F16)], [([4, 8], F16), ([4, 8], F16)], na.INVALID_ARGUMENT),       # a sum of nothing
    ([([4, 8], F16), ([8], F16), ([4, 8], F16)], [([4, 8], F16)], na.INVALID_ARGUMENT),       # no sum
    ([([4, 8], F16), ([8], F16), ([1, 8], F16)], [([4, 8], F16), ([4, 8], F16)], na.INVALID_ARGUMENT),
    ([([4, 8], F16), ([8], F16), ([4, 8], F32)], [([4, 8], F16), ([4, 8], F16)], na.INVALID_ARGUMENT),
    ([([], F16), ([8], F16)], [([], F16)], na.INVALID_ARGUMENT),
])
def test_rms_norm_refusals(ins, outs, status):
    assert na.RmsNorm().validate([desc(*d) for d in ins], [desc(*d) for d in outs]) == status


def test_rms_norm_s8_refusals():
    op = na.RmsNorm(output_dtype=S8)
    x, w, y = desc([4, 8], F16), desc([8], F16), desc([4, 8], S8)
    assert op.validate([x, w], [y]) == na.INVALID_ARGUMENT                     # no scales
    assert op.validate([x, w], [y, desc([3], F32)]) == na.INVALID_ARGUMENT
    assert op.validate([x, w], [y, desc([4], F16)]) == na.INVALID_ARGUMENT
    assert na.RmsNorm(epsilon=-1.0).validate([x, w], [x]) == na.INVALID_ARGUMENT
    assert na.RmsNorm(epsilon=float("nan")).validate([x, w], [x]) == na.INVALID_ARGUMENT
    assert na.RmsNorm(output_dtype=na.DT_U8).validate([x, w], [desc([4, 8], na.DT_U8)]) == na.UNSUPPORTED


def test_rotary_rules():
    op = na.Rotary(head_dim=16, rotary_dim=8)
    x, pos, tab = desc([5, 48], F16), desc([5], S32), desc([100, 8], F32)
    assert op.output_descs([x, pos, tab]) == [([5, 48], F16)]
    assert op.validate([x, pos, tab], [x]) == na.OK
    for ins, status in (([x, pos], na.INVALID_ARGUMENT), ([desc([5, 40], F16), pos, tab], na.INVALID_ARGUMENT),
                        ([desc([5, 3, 16], F16), pos, tab], na.INVALID_ARGUMENT),
                        ([x, desc([4], S32), tab], na.INVALID_ARGUMENT), ([x, desc([5], F32), tab], na.INVALID_ARGUMENT),
                        ([x, pos, desc([100, 16], F32)], na.INVALID_ARGUMENT),
                        ([x, pos, desc([0, 8], F32)], na.INVALID_ARGUMENT),
                        ([x, pos, desc([100, 8], F16)], na.INVALID_ARGUMENT),
                        ([desc([5, 48], S8), pos, tab], na.UNSUPPORTED)):
        assert op.validate(ins, [ins[0]]) == status
    assert op.validate([x, pos, tab], [desc([5, 48], F32)]) == na.INVALID_ARGUMENT
    for kw in (dict(head_dim=0), dict(head_dim=16, rotary_dim=7), dict(head_dim=16, rotary_dim=18),
               dict(head_dim=15), dict(head_dim=16, rotary_dim=-2)):
        assert na.Rotary(**kw).validate([x, pos, tab], [x]) == na.INVALID_ARGUMENT


def test_kv_cache_rules():
    wr, rd = na.KvCacheWrite(), na.KvCacheRead(output_dtype=F16)
    rows, c = desc([6, 128], F16), cache()
    assert wr.validate([rows, rows] + tables(), c) == na.OK
    assert wr.validate([rows, rows] + tables(starts=True), c) == na.OK
    assert rd.validate(c + tables(), [rows, rows]) == na.OK
    bad = [(0, desc([9, 2, 16], S8)), (0, desc([9, 2, 16, 64], F16)), (1, desc([9, 2, 16, 64], S8)),
           (1, desc([8, 2, 64, 16], S8)), (2, desc([9, 3], F32)), (2, desc([9, 2], F16)), (3, desc([2, 9], F32))]
    for at, new in bad:
        assert wr.validate([rows, rows] + tables(), with_(c, at, new)) == na.INVALID_ARGUMENT
        assert rd.validate(with_(c, at, new) + tables(), [rows, rows]) == na.INVALID_ARGUMENT
    for t in ([desc([3, 4], S32)], [desc([3, 4], S32), desc([4], S32)], [desc([3, 4], F32), desc([3], S32)],
              tables() + [desc([3], S32)], tables(starts=True) + [desc([4], S32)]):
        assert wr.validate([rows, rows] + t, c) == na.INVALID_ARGUMENT
    assert wr.validate([desc([6, 64], F16), desc([6, 64], F16)] + tables(), c) == na.INVALID_ARGUMENT
    assert wr.validate([rows, desc([5, 128], F16)] + tables(), c) == na.INVALID_ARGUMENT
    assert wr.validate([rows, desc([6, 128], F32)] + tables(), c) == na.INVALID_ARGUMENT
    assert wr.validate([desc([6, 128], S8), desc([6, 128], S8)] + tables(), c) == na.UNSUPPORTED
    assert rd.validate(c + tables(), [desc([6, 128], F32)] * 2) == na.INVALID_ARGUMENT       # not output_dtype
    pitched = cache()
    pitched[0].pitch = 80
    assert wr.validate([rows, rows] + tables(), pitched) == na.UNSUPPORTED                   # a cache is dense
    with pytest.raises(ValueError):
        wr.output_descs([rows, rows] + tables())                                             # the caller's


def test_cache_attention_rules():
    op = na.CacheAttention(window=5, sinks=1)
    q, c = desc([6, 512], F16), cache()
    assert op.output_descs([q] + c + tables()) == [([6, 512], F16)]
    assert op.validate([q] + c + tables(), [q]) == na.OK
    assert op.validate([q] + c + tables(starts=True), [q]) == na.OK
    assert op.validate([desc([6, 192], F16)] + c + tables(), [desc([6, 192], F16)]) == na.INVALID_ARGUMENT
    assert op.validate([q] + c + tables(), [desc([6, 512], F32)]) == na.INVALID_ARGUMENT
    assert op.validate([q] + c + tables(), [desc([5, 512], F16)]) == na.INVALID_ARGUMENT
    assert op.validate([desc([6, 512], S8)] + c + tables(), [desc([6, 512], S8)]) == na.UNSUPPORTED
    assert op.validate([q] + c, [q]) == na.INVALID_ARGUMENT
    for kw in (dict(window=-1), dict(sinks=-1), dict(scale=-1.0), dict(scale=float("nan"))):
        assert na.CacheAttention(**kw).validate([q] + c + tables(), [q]) == na.INVALID_ARGUMENT


def test_cache_attention_workspace():
    """None for short tables; partial results of the rows for long ones, no more
    for a window than the window needs."""
    q, c = desc([1, 1024], F16), cache(pages=4000, heads=2, d=128)
    assert na.CacheAttention().workspace_size([q] + c + tables(1, 4), [q]) == 0
    full = na.CacheAttention().workspace_size([q] + c + tables(1, 3000), [q])
    assert full > 0 and full % (8 * 130 * 4) == 0
    assert na.CacheAttention(window=512).workspace_size([q] + c + tables(1, 3000), [q]) < full
    assert na.CacheAttention().workspace_size([q] + c, [q]) == 0                             # refused: nothing


def test_compute_refusals():
    """compute() says what validate() says, and refuses views without memory,
    row pitches that are no whole elements, and backends without kernels."""
    def at(d, data=4096):
        d.data = data
        return d
    x, w, y = at(desc([4, 8], F16)), at(desc([8], F16)), at(desc([4, 8], F16))
    assert na.RmsNorm(backend=na.BACKEND_CPU).compute([y], [x, w], stream=0, workspace=0) == na.UNSUPPORTED
    assert na.RmsNorm().compute([y], [x], stream=0, workspace=0) == na.INVALID_ARGUMENT
    assert na.RmsNorm().compute([y], [desc([4, 8], F16), w], stream=0, workspace=0) == na.INVALID_ARGUMENT
    odd = at(desc([4, 8], F16))
    odd.pitch = 19
    assert na.RmsNorm().compute([y], [odd, w], stream=0, workspace=0) == na.INVALID_ARGUMENT
    odd.pitch = 14                                                       # less than a row
    assert na.RmsNorm().compute([y], [odd, w], stream=0, workspace=0) == na.INVALID_ARGUMENT
    rows, c, t = at(desc([6, 128], F16)), [at(d) for d in cache()], [at(d) for d in tables()]
    q = at(desc([6, 512], F16))
    assert na.KvCacheWrite(backend=na.BACKEND_CPU).compute(c, [rows, rows] + t, stream=0, workspace=0) == na.UNSUPPORTED
    assert na.KvCacheRead(backend=na.BACKEND_CPU).compute([rows, rows], c + t, stream=0, workspace=0) == na.UNSUPPORTED
    assert na.CacheAttention(backend=na.BACKEND_CPU).compute([q], [q] + c + t, stream=0, workspace=0) == na.UNSUPPORTED
    # page and head sizes that no kernel takes
    for page, d, status in ((24, 64, na.UNSUPPORTED), (512, 64, na.UNSUPPORTED), (16, 72, na.UNSUPPORTED),
                            (16, 272, na.UNSUPPORTED), (16, 8, na.UNSUPPORTED)):
        c2 = [at(x) for x in cache(page=page, d=d)]
        r2 = at(desc([6, 2 * d], F16))
        assert na.KvCacheWrite().compute(c2, [r2, r2] + t, stream=0, workspace=0) == status
        assert na.CacheAttention().compute([r2], [r2] + c2 + t, stream=0, workspace=0) == status
    # rows that do not divide among the sequences
    r7 = at(desc([7, 128], F16))
    assert na.KvCacheWrite().compute(c, [r7, r7] + t, stream=0, workspace=0) == na.INVALID_ARGUMENT
    # codes that are not 16-byte aligned
    c3 = [at(cache()[0], 4104)] + c[1:]
    assert na.KvCacheWrite().compute(c3, [rows, rows] + t, stream=0, workspace=0) == na.INVALID_ARGUMENT
    # a workspace that is asked for and not given
    long = [at(d) for d in tables(3, 3000)]
    assert na.CacheAttention().compute([q], [q] + [at(d) for d in cache(pages=9000)] + long, stream=0,
                                       workspace=0) == na.NOT_INITIALIZED


@pytest.mark.parametrize("rows,seqs", [(1, 3), (2, 3), (4, 3), (7, 3), (1, 64), (5, 2)])
def test_rows_that_do_not_divide(rows, seqs):
    """Without row starts every sequence has as many rows: fewer rows than
    sequences, or rows that do not divide among them, are refused by validate(),
    by compute() and by the query of the workspace, which returns."""
    c, r, q = cache(pages=9000), desc([rows, 128], F16), desc([rows, 512], F16)
    for d in c + [r, q]:
        d.data = 4096
    for per in (4, 3000):                                                # (a long table: splits, so a workspace)
        t, with_starts = tables(seqs, per), tables(seqs, per, starts=True)
        for d in t + with_starts:
            d.data = 4096
        for op, outs, ins in ((na.CacheAttention(), [q], [q] + c), (na.KvCacheWrite(), c, [r, r]),
                              (na.KvCacheRead(), [r, r], c)):
            assert op.validate(ins + t, outs) == na.INVALID_ARGUMENT
            assert op.workspace_size(ins + t, outs) == 0
            assert op.compute(outs, ins + t, stream=0, workspace=0) == na.INVALID_ARGUMENT
            assert op.compute(outs, ins + t, stream=0) == na.INVALID_ARGUMENT        # (asks for the size)
            assert op.validate(ins + with_starts, outs) == na.OK
        assert (na.CacheAttention().workspace_size([q] + c + with_starts, [q]) > 0) == (per == 3000)


def test_rows_of_no_sequence():
    c, r, q = cache(), desc([2, 128], F16), desc([2, 512], F16)
    for t in (tables(0), tables(0, starts=True)):
        for op, outs, ins in ((na.CacheAttention(), [q], [q] + c), (na.KvCacheWrite(), c, [r, r]),
                              (na.KvCacheRead(), [r, r], c)):
            assert op.validate(ins + t, outs) == na.INVALID_ARGUMENT
            assert op.workspace_size(ins + t, outs) == 0


# --- the C ABI below -------------------------------------------------------------

def test_abi_rms_norm():
    f = na.lib().nnops_hip_rms_norm
    g = na.RmsNormArgs()
    assert f(None, None) == na.INVALID_ARGUMENT
    assert f(C.byref(g), None) == na.OK                                  # no rows
    g.rows, g.cols, g.in_f16, g.out_kind = 2, 8, 1, na.OUT_F16
    assert f(C.byref(g), None) == na.INVALID_ARGUMENT                    # no data
    g.x = g.weight = g.y = 4096
    g.ld_x, g.ld_y = 8, 7
    assert f(C.byref(g), None) == na.INVALID_ARGUMENT
    g.ld_y, g.out_kind = 8, na.OUT_F32
    assert f(C.byref(g), None) == na.UNSUPPORTED
    g.out_kind = na.OUT_S8
    assert f(C.byref(g), None) == na.INVALID_ARGUMENT                    # no scales
    g.out_kind, g.residual = na.OUT_F16, 4096
    assert f(C.byref(g), None) == na.INVALID_ARGUMENT                    # no sum
    g.sum, g.ld_sum, g.ld_residual = 4096, 8, 4
    assert f(C.byref(g), None) == na.INVALID_ARGUMENT
    g.ld_residual, g.epsilon = 8, -1.0
    assert f(C.byref(g), None) == na.INVALID_ARGUMENT
    g.epsilon, g.rows = 0.0, 1 << 40
    assert f(C.byref(g), None) == na.UNSUPPORTED


def test_abi_rms_norm_in_place():
    """An output over an input needs the input's row pitch; codes lie over
    neither, and the two outputs not over one another. (No call here is let
    through: each names one refusal.)"""
    f = na.lib().nnops_hip_rms_norm
    X, R, Y, S = 1 << 20, 2 << 20, 3 << 20, 4 << 20

    def args(**kw):
        g = na.RmsNormArgs()
        g.rows, g.cols, g.in_f16, g.out_kind, g.weight = 2, 8, 1, na.OUT_F16, 4096
        g.x, g.residual, g.y, g.sum = X, R, Y, S
        g.ld_x = g.ld_residual = g.ld_y = g.ld_sum = 16
        for k, v in kw.items():
            setattr(g, k, v)
        return g
    for kw in (dict(sum=X, ld_sum=8), dict(sum=R, ld_sum=24), dict(y=X, ld_y=8), dict(y=R, ld_y=24), dict(y=S),
               dict(sum=X, y=X), dict(y=X, out_kind=na.OUT_S8, scale=4096), dict(y=R, out_kind=na.OUT_S8, scale=4096)):
        assert f(C.byref(args(**kw)), None) == na.INVALID_ARGUMENT, kw


def test_abi_rotary():
    f = na.lib().nnops_hip_rotary
    g = na.RotaryArgs()
    assert f(None, None) == na.INVALID_ARGUMENT
    g.tokens, g.heads, g.head_dim, g.rotary_dim, g.max_pos = 2, 1, 8, 8, 4
    g.x, g.y, g.positions, g.table = 4096, 8192, 4096, 4096
    g.ld_x = g.ld_y = g.ld_table = 8
    for field, value, status in (("rotary_dim", 7, 1), ("rotary_dim", 10, 1), ("head_dim", 0, 1), ("max_pos", 0, 1),
                                 ("ld_x", 7, 1), ("ld_y", 7, 1), ("ld_table", 7, 1), ("table", None, 1),
                                 ("positions", None, 1), ("tokens", -1, 1), ("tokens", 0, 0), ("heads", 1 << 21, 2)):
        old = getattr(g, field)
        setattr(g, field, value)
        assert f(C.byref(g), None) == status, field
        setattr(g, field, old)
    g.y, g.ld_y = 4096, 9                                                # in place, another pitch
    assert f(C.byref(g), None) == na.INVALID_ARGUMENT
    f, t = na.lib().nnops_hip_rotary_table, na.RotaryTableArgs()
    t.table, t.max_pos, t.rotary_dim, t.ld_table, t.base, t.factor, t.attention_factor = 4096, 4, 8, 8, 1e4, 1.0, 1.0
    for field, value in (("rotary_dim", 7), ("base", 0.0), ("factor", 0.0), ("factor", -2.0), ("ld_table", 7),
                         ("attention_factor", 0.0), ("table", None), ("original_context", -1.0),
                         ("original_context", 5.0)):                     # low_turns = high_turns
        old = getattr(t, field)
        setattr(t, field, value)
        assert f(C.byref(t), None) == na.INVALID_ARGUMENT, field
        setattr(t, field, old)
    t.max_pos = 0
    assert f(C.byref(t), None) == na.OK


def _pages(c):
    c.k, c.v, c.k_scale, c.v_scale, c.page_table, c.lengths = (4096,) * 6
    c.pages, c.heads, c.page_tokens, c.head_dim = 4, 2, 16, 32
    c.sequences, c.table_pages, c.ld_table = 2, 3, 3


CACHE_REFUSALS = [("page_tokens", 48, 2), ("page_tokens", 8, 2), ("head_dim", 40, 2), ("head_dim", 512, 2), ("k", 4104, 1),
                  ("v", None, 1), ("k_scale", None, 1), ("page_table", None, 1), ("lengths", None, 1), ("ld_table", 2, 1),
                  ("sequences", 0, 1), ("sequences", 3, 1), ("pages", -1, 1), ("heads", -1, 1), ("table_pages", -1, 1),
                  ("table_pages", 1 << 40, 2), ("heads", 1 << 20, 2), ("pages", 1 << 40, 2)]


def test_abi_kv_cache():
    lib = na.lib()
    for f in (lib.nnops_hip_kv_cache_write, lib.nnops_hip_kv_cache_read):
        assert f(None, None) == na.INVALID_ARGUMENT
        g = na.KvRowsArgs()
        _pages(g.cache)
        assert f(C.byref(g), None) == na.OK                              # no rows
        g.rows, g.ld_k, g.ld_v, g.k_rows, g.v_rows, g.f16 = 4, 64, 64, 4096, 4096, 1
        for field, value, status in CACHE_REFUSALS:
            old = getattr(g.cache, field)
            setattr(g.cache, field, value)
            assert f(C.byref(g), None) == status, field
            setattr(g.cache, field, old)
        for field, value, status in (("ld_k", 63, 1), ("ld_v", 63, 1), ("k_rows", None, 1), ("rows", -1, 1),
                                     ("rows", 1 << 40, 2), ("rows", 5, 1)):
            old = getattr(g, field)
            setattr(g, field, value)
            assert f(C.byref(g), None) == status, field
            setattr(g, field, old)


def test_abi_cache_attention():
    lib = na.lib()
    f = lib.nnops_hip_cache_attention
    assert f(None, None, 0, None) == na.INVALID_ARGUMENT
    assert lib.nnops_hip_cache_attention_workspace_size(None) == 0
    g = na.CacheAttentionArgs()
    _pages(g.cache)
    g.q_heads = 8
    assert f(C.byref(g), None, 0, None) == na.OK                         # no rows
    g.rows, g.ld_q, g.ld_out, g.q, g.out, g.f16 = 4, 256, 256, 4096, 4096, 1
    for field, value, status in CACHE_REFUSALS + [("pages", 0, 1)]:
        old = getattr(g.cache, field)
        setattr(g.cache, field, value)
        assert f(C.byref(g), None, 0, None) == status, field
        setattr(g.cache, field, old)
    for field, value, status in (("ld_q", 255, 1), ("ld_out", 255, 1), ("q", None, 1), ("out", None, 1), ("q_heads", 7, 1),
                                 ("q_heads", 0, 1), ("q_heads", -2, 1), ("window", -1, 1), ("sinks", -1, 1),
                                 ("scale", -1.0, 1), ("scale", float("nan"), 1), ("rows", 1 << 40, 2)):
        old = getattr(g, field)
        setattr(g, field, value)
        assert f(C.byref(g), None, 0, None) == status, field
        setattr(g, field, old)


def test_output_descs_room():
    ins = (L.Tensor * 2)(desc([2, 4], F16), desc([4], F16))
    outs = (L.Tensor * 2)()
    op = na.RmsNorm(output_dtype=S8)
    assert L.lib().nnops_op_output_descs(op._h, ins, 2, outs, 1) == -na.INVALID_ARGUMENT
    assert L.lib().nnops_op_output_descs(op._h, ins, 2, outs, 2) == 2
    assert L.lib().nnops_op_output_descs(None, ins, 2, outs, 2) == -na.INVALID_ARGUMENT


def test_abi_workspace_size_of_refused_calls():
    """The query takes any argument that the call itself would refuse: 0, and it returns."""
    lib = na.lib()
    g = na.CacheAttentionArgs()
    c = g.cache
    c.pages, c.heads, c.page_tokens, c.head_dim, c.sequences, c.table_pages = 4000, 2, 16, 64, 3, 3000
    g.rows, g.q_heads, g.f16 = 6, 8, 1                                   # (no pointers: they play no part)
    f = lib.nnops_hip_cache_attention_workspace_size
    need = f(C.byref(g))
    assert need > 0
    for obj, field, values in ((g, "rows", (0, -1, 1, 2, 7, 1 << 40)), (g, "q_heads", (0, -2, 7, 1 << 20)),
                               (g, "window", (-1,)), (g, "sinks", (-1,)), (g, "scale", (-1.0, float("nan"))),
                               (c, "heads", (0, -1, 3, 1 << 20)), (c, "page_tokens", (0, -16, 24, 1 << 40)),
                               (c, "head_dim", (0, 8, 72, 1 << 40)), (c, "sequences", (0, -1, 4, 64, 1 << 40)),
                               (c, "table_pages", (-1, 1 << 40, (1 << 63) - 1)), (c, "pages", (-1, 0, 1 << 40))):
        old = getattr(obj, field)
        for value in values:
            setattr(obj, field, value)
            assert f(C.byref(g)) == 0, (field, value)
        setattr(obj, field, old)
    assert f(C.byref(g)) == need


# --- tensor(): views as descriptors ----------------------------------------------

def test_tensor_of_views():
    """A view whose rows are evenly spaced has their step as its pitch, whatever
    its rank; any other is refused, not read as a dense one."""
    import torch
    x = torch.zeros((4, 10, 64), dtype=torch.float16)
    for view, pitch in ((x, 128), (x[:, :, :32], 128), (x[1:, :, 8:24], 128), (x[:, 3], 1280), (x[:, 3, :16], 1280),
                        (x[:, :1], 1280), (x[2:3, :4], 128), (x[1, 2:3, 5:9], 128), (x[:, ::2], 256), (x[1], 128),
                        (x[1, 2], 0), (x[1, 2, :7], 0), (x[1:2, 4, :], 1280), (x[:, :, :1][:, :, 0:1], 128)):
        t = na.tensor(view)
        assert t.pitch == pitch and [t.dims[i] for i in range(t.rank)] == list(view.shape), view.stride()
        assert t.data == view.data_ptr()
    one = torch.zeros((5, 1)).t()                                        # strides (1, 1): a dense row
    assert na.tensor(one).pitch == 20
    assert na.tensor(torch.zeros((1, 4, 8)).transpose(0, 1)).pitch == 32  # [4, 1, 8], strides (8, 32, 1)
    assert na.tensor(torch.zeros((0, 8))).pitch == 0
    lengths = torch.zeros((6, 2), dtype=torch.int32)
    cache = torch.zeros((9, 4, 16, 32), dtype=torch.int8)
    for view in (x[:, :5], x[::2, :5], x[:, 2:4, :8], x[1, 2, ::2], lengths[:, 0], lengths.t()[1], cache[:, :2],
                 cache[:, :, :8], torch.zeros(8).expand(3, 8), torch.zeros((1, 8)).expand(4, 8),
                 torch.zeros(20).as_strided((3, 8), (6, 1))):
        with pytest.raises((ValueError, AssertionError)):
            na.tensor(view)
    with pytest.raises(AssertionError):
        na.tensor(x.transpose(1, 2))


def test_rotary_table_out():
    """What the table is written to has to hold it: type, shape, rows."""
    import torch
    for out in (torch.zeros((4, 8), dtype=torch.float16), torch.zeros((3, 8)), torch.zeros((4, 6)), torch.zeros(32),
                torch.zeros((8, 4)).t(), torch.zeros((1, 8)).expand(4, 8), torch.zeros((4, 16))[:, ::2]):
        with pytest.raises(ValueError):
            na.rotary_table(4, 8, out=out, stream=0)
    assert na.rotary_table(0, 8, out=torch.zeros((0, 8)), stream=0).shape == (0, 8)
