"""Calls without a stream argument run on torch's current stream: the default
one, a stream made current, and the default again."""
from __future__ import annotations

import numpy as np
import pytest

import oracle
import datagen as dg
import nnops_amd as na
from nnops_amd import ops
from gpu_util import dev, host, announce

pytestmark = pytest.mark.gpu


def test_current_stream():
    import torch
    announce("current stream")
    M, K, N = 3, 256, 64
    a, w = dg.act_s8(1, (M, K)), dg.ints(2, (N, K), -127, 127)
    da, dw = dev(a), dev(w)
    want = oracle.gemm_i8(a, w, trans_b=True)
    side = torch.cuda.Stream()
    for stream in (torch.cuda.default_stream(), side, torch.cuda.default_stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            assert (ops._stream_ptr(None) or 0) == stream.cuda_stream
            c = torch.zeros((M, N), dtype=torch.int32, device="cuda")
            na.gemm_i8(da, dw, c, trans_b=True)
            stream.synchronize()
        assert np.array_equal(host(c), want)
    assert (ops._stream_ptr(side) or 0) == side.cuda_stream


def test_current_stream_without_the_private_name(monkeypatch):
    """A torch whose raw stream lookup has another name: the Stream object's
    handle."""
    import torch
    announce("current stream, public names only")
    monkeypatch.setattr(ops, "_RAW_STREAM", None)
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream")
    side = torch.cuda.Stream()
    for stream in (side, torch.cuda.default_stream()):
        with torch.cuda.stream(stream):
            assert (ops._stream_ptr(None) or 0) == stream.cuda_stream


def _gemms():
    """f16 products with a workspace: the direct call and the operator, and the
    result that both leave in c."""
    import torch
    M, K, N = 8, 4096, 512
    a, w = dev(dg.normal(1, (M, K)).astype(np.float16)), dev(dg.normal(2, (N, K)).astype(np.float16))
    c = torch.zeros((M, N), dtype=torch.float16, device="cuda")
    lin, ins, outs = na.Linear(output_dtype=na.DT_F16), [na.tensor(a), na.tensor(w)], [na.tensor(c)]
    assert lin.workspace_size(ins, outs) > 0

    def both(stream):
        na.gemm_fp(a, w, c, stream=stream)
        first = c.clone() if stream is None else None
        assert lin.compute(outs, ins, stream=stream) == na.OK
        return first
    return both, c


def test_workspace_without_entering_the_stream(monkeypatch):
    """A named stream (an object, a handle, the default one's 0) costs a call no
    more than an allocation: torch's stream context, as long as a small call, is
    not entered."""
    import torch
    announce("workspace of a named stream")
    both, c = _gemms()
    both(None)
    torch.cuda.synchronize()
    want = host(c).copy()

    def entered(*_):
        raise AssertionError("the stream was entered")
    side = torch.cuda.Stream()
    monkeypatch.setattr(torch.cuda, "stream", entered)
    monkeypatch.setattr(torch.cuda, "set_stream", entered)
    for stream in (side, side.cuda_stream, torch.cuda.current_stream(), 0):
        c.zero_()
        torch.cuda.synchronize()
        both(stream)
        torch.cuda.synchronize()
        assert np.array_equal(host(c), want)


def test_workspace_belongs_to_its_stream():
    """Freed, it goes to that stream's next allocation, not to another stream's."""
    import torch
    announce("workspace and the allocator")
    n, side = 3 << 20, torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        used = torch.cuda.memory_allocated()
        at = ops._workspace(n, "cuda", stream).data_ptr()
        assert torch.cuda.memory_allocated() == used
        other = torch.empty(n, dtype=torch.uint8, device="cuda")
        assert other.data_ptr() != at
        with torch.cuda.stream(side):
            again = torch.empty(n, dtype=torch.uint8, device="cuda")
        assert again.data_ptr() == at
        del other, again
    assert ops._workspace(0, "cuda", side) is None


def test_workspace_of_a_captured_call():
    """Calls that name the capturing stream and bring no workspace, replayed."""
    import torch
    announce("captured calls with workspaces of their own")
    both, c = _gemms()
    side = torch.cuda.Stream()
    both(side)
    torch.cuda.synchronize()
    want = host(c).copy()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        both(side)
    for _ in range(3):
        c.zero_()
        keep = [torch.full((1 << 20,), 77, dtype=torch.uint8, device="cuda") for _ in range(8)]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(c), want)
        del keep
