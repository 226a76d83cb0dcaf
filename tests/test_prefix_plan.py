"""The kernel selection of PrefixAttention (nnops_hip_prefix_attention_plan) at the
limits of its launches, on the host: what the plan, the workspace query and the call
say of a size is the same, and what the launches over shared tokens cannot hold is
left to CacheAttention's. No call here reaches a kernel launch."""
from __future__ import annotations

import ctypes as C

import pytest

import nnops_amd as na
from nnops_amd import _lib as L

BASE = 1 << 20                 # addresses that nothing is read from


def args(heads, group, d, page, columns, rows, sequences, groups, f16=True, ragged=False):
    width = heads * group * d
    a = L.PrefixAttentionArgs(q=7 * BASE, out=8 * BASE, rows=rows, q_heads=heads * group, ld_q=width, ld_out=width,
                              f16=int(f16), groups=groups, group_starts=9 * BASE, shared=10 * BASE)
    a.cache = L.KvPages(k=BASE, v=2 * BASE, k_scale=3 * BASE, v_scale=4 * BASE, pages=9, heads=heads, page_tokens=page,
                        head_dim=d, page_table=5 * BASE, sequences=sequences, table_pages=columns, ld_table=columns,
                        lengths=6 * BASE, row_starts=11 * BASE if ragged else None)
    return a


def whole(a):
    """CacheAttention's arguments for the same call."""
    return L.CacheAttentionArgs(cache=a.cache, q=a.q, out=a.out, rows=a.rows, q_heads=a.q_heads, ld_q=a.ld_q,
                                ld_out=a.ld_out, f16=a.f16)


def plan(a):
    p = L.PrefixAttentionPlan()
    return na.lib().nnops_hip_prefix_attention_plan(C.byref(a), C.byref(p)), p


# heads, group, d, page, columns, rows, sequences, groups, f16, ragged, shared rows of a workgroup
SIZES = [
    (8, 16, 128, 64, 2000, 1024 * 70, 1024, 1, True, False, 256),
    (8, 4, 128, 64, 130, 4096 * 97, 4096, 1, True, True, 256),
    (8, 16, 16, 64, 200, 1024 * 65, 1024, 1, True, False, 256),
    # either side of the workgroups that a join can have
    (8, 16, 256, 64, 4000, 1024 * 250, 1024, 1, True, False, 128),
    (8, 16, 256, 64, 4000, 1024 * 257, 1024, 1, True, False, 0),
    # a sequence's workgroup each
    (64, 4, 16, 64, 400, 1 << 15, 1 << 15, 1 << 12, True, False, 16),
]


@pytest.mark.parametrize("heads,group,d,page,columns,rows,sequences,groups,f16,ragged,shared", SIZES)
def test_plan_query_and_call_agree(heads, group, d, page, columns, rows, sequences, groups, f16, ragged, shared):
    lib, a = na.lib(), args(heads, group, d, page, columns, rows, sequences, groups, f16, ragged)
    rc, p = plan(a)
    assert (rc, p.shared_rows) == (na.OK, shared)
    assert lib.nnops_hip_prefix_attention_workspace_size(C.byref(a)) == p.workspace_bytes
    if p.workspace_bytes:
        # the sizes are taken: it is the workspace that there is too little of
        call = lib.nnops_hip_prefix_attention
        assert call(C.byref(a), None, 0, None) == na.NOT_INITIALIZED
        assert call(C.byref(a), C.c_void_p(99 * BASE), p.workspace_bytes - 1, None) == na.NOT_INITIALIZED
    if shared == 0:
        w, q = whole(a), L.CacheAttentionPlan()
        assert lib.nnops_hip_cache_attention_plan(C.byref(w), C.byref(q)) == na.OK
        assert (p.own_rows, p.own_splits, p.workspace_bytes) == (q.tile_rows, q.splits, q.workspace_bytes)


@pytest.mark.parametrize("heads,group,d,page,columns,rows,sequences,groups", [
    (64, 4, 16, 64, 400, 1 << 16, 1 << 16, 1 << 13), (64, 1, 256, 64, 64, 1 << 16, 1 << 16, 1), (16, 1, 64, 16, 9, 1 << 18, 1 << 18, 0),
])
def test_sizes_that_no_launch_holds(heads, group, d, page, columns, rows, sequences, groups):
    """2^22 workgroups: plans and calls refuse them alike, and no workspace is asked for."""
    lib, a = na.lib(), args(heads, group, d, page, columns, rows, sequences, groups)
    w, q = whole(a), L.CacheAttentionPlan()
    assert plan(a)[0] == na.UNSUPPORTED and lib.nnops_hip_prefix_attention_workspace_size(C.byref(a)) == 0
    assert lib.nnops_hip_prefix_attention(C.byref(a), C.c_void_p(99 * BASE), 1 << 50, None) == na.UNSUPPORTED
    assert lib.nnops_hip_cache_attention_plan(C.byref(w), C.byref(q)) == na.UNSUPPORTED
    assert lib.nnops_hip_cache_attention_workspace_size(C.byref(w)) == 0
    assert lib.nnops_hip_cache_attention(C.byref(w), C.c_void_p(99 * BASE), 1 << 50, None) == na.UNSUPPORTED
    # one sequence fewer
    a = args(heads, group, d, page, columns, rows - 1, sequences - 1, groups)
    assert plan(a)[0] == na.OK
