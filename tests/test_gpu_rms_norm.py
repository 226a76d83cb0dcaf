"""RmsNorm against the norm in 64 bits: widths of every kernel (a wave per row,
a workgroup per row, rows read twice), odd widths and pitches, both types, the
residual, the s8 form and what it does with rows of nothing, infinities and
NaNs."""
from __future__ import annotations

import numpy as np
import pytest

import datagen as dg
import decoder_ref as ref
import nnops_amd as na
from gpu_util import dev, host, pitched, announce

pytestmark = pytest.mark.gpu

# one row-wave, two chunks, a workgroup, its two chunks, 8 and 16 waves, the wide form
WIDTHS = [1, 7, 64, 500, 512, 513, 1024, 1536, 2047, 4096, 5001, 8192, 11008, 16384, 16385, 40000]


def _data(rows, cols, f16, seed=1):
    t = np.float16 if f16 else np.float32
    big = np.where(dg.uniform(seed + 9, (cols,), 0, 1) < 0.01, 20.0, 1.0)
    x = (dg.normal(seed, (rows, cols)) * big).astype(t)
    r = dg.normal(seed + 1, (rows, cols)).astype(t)
    w = (1 + 0.2 * dg.normal(seed + 2, (cols,))).astype(t)
    return x, r, w


def _run(x, r, w, out, *, eps=1e-6, pad=0):
    """(y, scale, sum) as numpy; every buffer pitched by `pad` more elements."""
    import torch
    f16 = x.dtype == np.float16
    dt = na.DT_F16 if f16 else na.DT_F32
    rows, cols = x.shape
    dx = pitched(x, cols + pad)
    ins = [na.tensor(dx), na.tensor(dev(w))]
    y = pitched(np.full((rows, cols), 3, np.int8 if out == "s8" else x.dtype), cols + pad)
    outs = [na.tensor(y)]
    scale = total = None
    if out == "s8":
        scale = torch.full((rows,), 5.0, device="cuda")
        outs.append(na.tensor(scale))
    if r is not None:
        ins.append(na.tensor(pitched(r, cols + pad)))
        total = pitched(np.full((rows, cols), 3, x.dtype), cols + pad)
        outs.append(na.tensor(total))
    op = na.RmsNorm(epsilon=eps, output_dtype=na.DT_S8 if out == "s8" else dt)
    assert op.validate(ins, outs) == na.OK
    assert op.compute(outs, ins) == na.OK
    torch.cuda.synchronize()
    return host(y), None if scale is None else host(scale), None if total is None else host(total)


def _check(x, r, w, out, y, scale, total, eps=1e-6):
    f16 = x.dtype == np.float16
    half = 2.0 ** -11 if f16 else 2.0 ** -24      # one rounding to the type, and f16's smallest step
    least = 2.0 ** -25 if f16 else 0.0
    h, want, u = ref.rms_norm(x, w, r, eps)
    if r is not None:
        # the f32 sum, rounded to the type
        assert np.all(abs(total - h) <= (half + 2.0 ** -24) * abs(h) + least)
    # rstd: the f32 sum of squares by chunks and a tree, a square root, a division
    rel = 2.0 ** -19
    if out != "s8":
        assert np.all(abs(y.astype(np.float64) - want) <= (half + rel) * abs(want) + least)
        return
    a = abs(u).max(axis=1, keepdims=True)
    step = want_scale = a / np.sqrt((h * h).mean(axis=1, keepdims=True) + eps) / 127
    assert np.all(abs(scale[:, None] - want_scale) <= rel * want_scale)
    assert y.min() >= -127
    # half a step; u, 1 / a and the product each rounded once in f32
    assert np.all(abs(y.astype(np.float64) * step - want) <= (0.5 + 127 * 2.0 ** -21) * step)
    assert np.all(abs(y.astype(np.int64)).max(axis=1) == 127)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("cols", WIDTHS)
def test_widths(cols, f16):
    rows = 3 if cols > 2048 else 9
    for residual in (True, False):
        for out in ("s8", "fp"):
            announce(f"norm {rows}x{cols} f16={f16} residual={residual} {out}")
            x, r, w = _data(rows, cols, f16)
            r = r if residual else None
            _check(x, r, w, out, *_run(x, r, w, out))


@pytest.mark.parametrize("cols,pad", [(4096, 1), (640, 24), (16385, 3), (33, 7)])
def test_pitches(cols, pad):
    """Rows that begin anywhere: the chunks' loads are unaligned."""
    x, r, w = _data(5, cols, True)
    for out in ("s8", "fp"):
        announce(f"norm pitch {cols}+{pad} {out}")
        _check(x, r, w, out, *_run(x, r, w, out, pad=pad))


@pytest.mark.parametrize("cols", [300, 4096, 20000])
def test_sum_over_an_input(cols):
    """sum in x's buffer, in the residual's, and y in x's."""
    import torch
    announce(f"norm in place {cols}")
    x, r, w = _data(4, cols, True)
    want_y, _, want_sum = _run(x, r, w, "fp")
    dw = dev(w)
    op = na.RmsNorm(output_dtype=na.DT_F16)
    for over in ("x", "r"):
        dx, dr, y = dev(x), dev(r), torch.zeros((4, cols), dtype=torch.float16, device="cuda")
        total = dx if over == "x" else dr
        assert op.compute([na.tensor(y), na.tensor(total)], [na.tensor(dx), na.tensor(dw), na.tensor(dr)]) == na.OK
        torch.cuda.synchronize()
        assert np.array_equal(host(y), want_y) and np.array_equal(host(total), want_sum)
    dx, dr = dev(x), dev(r)
    assert op.compute([na.tensor(dx), na.tensor(dr)], [na.tensor(dx), na.tensor(dw), na.tensor(dr)]) == na.OK
    torch.cuda.synchronize()
    assert np.array_equal(host(dx), want_y) and np.array_equal(host(dr), want_sum)


@pytest.mark.parametrize("cols", [40, 4096, 20000])
@pytest.mark.parametrize("f16", [True, False])
def test_rows_of_nothing_and_of_no_number(cols, f16):
    announce(f"norm special rows {cols} f16={f16}")
    x, _, w = _data(5, cols, f16)
    x[0] = 0
    x[1, cols // 2] = np.inf
    x[2, cols - 1] = np.nan
    x[3] = 0
    x[3, 0] = 1e-7                                     # one value far below epsilon
    y, scale, _ = _run(x, None, w, "s8")
    assert np.all(y[0] == 0) and scale[0] == 0
    assert np.all(y[1] == 0) and np.isnan(scale[1])
    assert np.all(y[2] == 0) and np.isnan(scale[2])
    assert abs(y[3, 0]) == 127 and np.all(y[3, 1:] == 0) and 0 < scale[3] < 1
    _check(x[4:], None, w, "s8", y[4:], scale[4:], None)
    y, _, _ = _run(x, None, w, "fp")
    assert np.all(y[0] == 0) and np.isnan(y[2]).any() and np.isfinite(y[[0, 3, 4]]).all()


def test_feeds_the_int8_product():
    """The codes and scales as Linear's per-token activation."""
    import torch
    announce("norm -> int8 Linear")
    rows, cols, n = 5, 512, 96
    x, r, w = _data(rows, cols, True)
    wq = dg.ints(7, (n, cols), -127, 127)
    sw = dg.uniform(8, (n,), 0.001, 0.002)
    q = torch.empty((rows, cols), dtype=torch.int8, device="cuda")
    s = torch.empty(rows, device="cuda")
    h = torch.empty((rows, cols), dtype=torch.float16, device="cuda")
    op = na.RmsNorm(output_dtype=na.DT_S8)
    assert op.compute([na.tensor(q), na.tensor(s), na.tensor(h)],
                      [na.tensor(dev(x)), na.tensor(dev(w)), na.tensor(dev(r))]) == na.OK
    y = torch.empty((rows, n), dtype=torch.float32, device="cuda")
    lin = na.Linear(output_dtype=na.DT_F32)
    assert lin.compute([na.tensor(y)], [na.tensor(q, scale_data=s, granularity=1),
                                        na.tensor(dev(wq), scale_data=dev(sw), granularity=2)]) == na.OK
    torch.cuda.synchronize()
    exact = host(q).astype(np.float64) @ wq.T.astype(np.float64)
    want = exact * host(s).astype(np.float64)[:, None] * sw.astype(np.float64)[None]
    assert np.all(abs(host(y) - want) <= 2.0 ** -22 * abs(want))


def test_many_rows_and_empty():
    import torch
    announce("norm 70000 rows, and none")
    x, r, w = _data(7, 24, True)
    big = np.tile(x, (10000, 1))
    y, scale, _ = _run(big, None, w, "s8")
    one, s1, _ = _run(x, None, w, "s8")
    assert np.array_equal(y, np.tile(one, (10000, 1))) and np.array_equal(scale, np.tile(s1, 10000))
    e = torch.empty((0, 24), dtype=torch.float16, device="cuda")
    assert na.RmsNorm().compute([na.tensor(e)], [na.tensor(e), na.tensor(dev(w))]) == na.OK


@pytest.mark.parametrize("cols", [40, 600, 4096, 16384, 20000])
@pytest.mark.parametrize("f16", [True, False])
def test_epsilon_of_zero(cols, f16):
    """Rows of zeros (with a residual: x and -x) are zeros, their scale 0; the
    rows beside them are what the formula says without an epsilon."""
    announce(f"norm epsilon 0 {cols} f16={f16}")
    x, r, w = _data(4, cols, f16)
    r[1], x[2], r[2] = -x[1], 0, 0
    for residual in (True, False):
        for out in ("s8", "fp"):
            y, scale, total = _run(x, r if residual else None, w, out, eps=0.0)
            zero = [1, 2] if residual else [2]
            rest = [i for i in range(4) if i not in zero]
            assert np.all(y[zero] == 0) and (scale is None or np.all(scale[zero] == 0))
            _check(x[rest], r[rest] if residual else None, w, out, y[rest], None if scale is None else scale[rest],
                   None if total is None else total[rest], eps=0.0)


@pytest.mark.parametrize("cols", [40, 600, 1100, 4096, 5001, 8192, 16384, 20000])
def test_f32_rows_whose_squares_leave_the_range(cols):
    """f32 rows of 1e20 and 1e36, whose squares are infinite, and, without an
    epsilon, of 1e-25 and 1e-41, whose squares are 0: what the formula says, as
    for the ordinary row beside them; with an epsilon small rows stay small."""
    announce(f"norm f32 range {cols}")
    x, r, w = _data(6, cols, False)
    size = np.array([1e20, 1.0, 1e36, 1e-25, 1e-41, 3e17])[:, None]
    x, r = (x * size).astype(np.float32), (r * size).astype(np.float32)
    for residual in (r, None):
        for out in ("s8", "fp"):
            _check(x, residual, w, out, *_run(x, residual, w, out, eps=0.0), eps=0.0)
            rows = slice(0, 4) if out == "fp" else slice(0, 3)           # (u below 2^-119 has codes 0)
            part = None if residual is None else r[rows]
            _check(x[rows], part, w, out, *_run(x[rows], part, w, out))
    # an infinity or a NaN in such a row still shows
    x[0, cols // 3], x[2, cols - 1] = np.inf, np.nan
    y, scale, _ = _run(x, None, w, "s8", eps=0.0)
    assert np.all(y[[0, 2]] == 0) and np.isnan(scale[[0, 2]]).all() and np.isfinite(scale[[1, 3, 4, 5]]).all()
    y, _, _ = _run(x, None, w, "fp", eps=0.0)
    assert np.isnan(y[0, cols // 3]) and np.isnan(y[2]).all() and np.isfinite(y[[1, 3, 4, 5]]).all()


def test_more_wide_rows_than_a_launch_holds():
    """2^22 + 3 rows of 16385, a workgroup of 1024 threads each, in place: all
    alike but for a few at the ends of the launches."""
    import torch
    rows, cols = (1 << 22) + 3, 16385
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < rows * cols * 2 + (24 << 30):
        pytest.skip("needs half of the card's memory")
    announce(f"norm {rows}x{cols}")
    x, _, w = _data(2, cols, True)
    want = dev(_run(x, None, w, "fp")[0])
    big = torch.empty((rows, cols), dtype=torch.float16, device="cuda")
    big[:] = dev(x[0])
    odd = torch.tensor([1, (1 << 20) - 1, 1 << 20, (1 << 22) - 1, 1 << 22, rows - 1], device="cuda")
    big[odd] = dev(x[1])
    assert na.RmsNorm().compute([na.tensor(big)], [na.tensor(big), na.tensor(dev(w))]) == na.OK
    torch.cuda.synchronize()
    assert torch.equal(big[odd], want[1:].expand(len(odd), cols))
    big[odd] = want[0]
    for r0 in range(0, rows, 1 << 18):
        part = big[r0:r0 + (1 << 18)]
        assert torch.equal(part, want[:1].expand(len(part), cols)), r0
    del big, part
    torch.cuda.empty_cache()


def test_wide_rows_of_the_second_launch():
    """2^20 + 2 rows of 16385 with residual and codes: every pointer moves on."""
    import torch
    rows, cols = (1 << 20) + 2, 16385
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < rows * cols * 5 + (24 << 30):
        pytest.skip("needs half of the card's memory")
    announce(f"norm {rows}x{cols} residual, codes")
    x, r, w = _data(2, cols, True)
    want_y, want_scale, want_sum = (dev(z) for z in _run(x, r, w, "s8"))
    bx, br = (torch.empty((rows, cols), dtype=torch.float16, device="cuda") for _ in range(2))
    bx[:], br[:] = dev(x[0]), dev(r[0])
    odd = torch.tensor([1, (1 << 20) - 1, 1 << 20], device="cuda")
    bx[odd], br[odd] = dev(x[1]), dev(r[1])
    y, scale = torch.empty((rows, cols), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    op = na.RmsNorm(output_dtype=na.DT_S8)
    assert op.compute([na.tensor(y), na.tensor(scale), na.tensor(bx)],
                      [na.tensor(bx), na.tensor(dev(w)), na.tensor(br)]) == na.OK
    torch.cuda.synchronize()
    for got, want in ((y, want_y), (scale, want_scale), (bx, want_sum)):
        shape = (len(odd),) + got.shape[1:]
        assert torch.equal(got[odd], want[1:].expand(shape))
        got[odd] = want[0]
        for r0 in range(0, rows, 1 << 18):
            part = got[r0:r0 + (1 << 18)]
            assert torch.equal(part, want[:1].expand(part.shape)), r0
    del bx, br, y, got, part
    torch.cuda.empty_cache()


@pytest.mark.parametrize("cols,rows", [(500, 9000), (1000, 8200), (1100, 2500), (4096, 2100), (5001, 2100), (8192, 1100),
                                       (16384, 600)])
def test_rows_past_the_workgroups(cols, rows):
    """More rows than the launch has units (of 1, 4, 8 and 16 waves): each takes
    several, the next one's loads in flight; then the same in place."""
    import torch
    for f16 in (True, False) if cols < 8192 else (True,):
        announce(f"norm rows in turn {rows}x{cols} f16={f16}")
        x, r, w = _data(rows, cols, f16)
        want = {}
        for out in ("s8", "fp"):
            want[out] = _run(x, r, w, out)
            _check(x, r, w, out, *want[out])
        _check(x, None, w, "s8", *_run(x, None, w, "s8"))
        # sum over x and over the residual, y over the other
        op = na.RmsNorm(output_dtype=na.DT_F16 if f16 else na.DT_F32)
        dw = dev(w)
        for over in ("x", "r"):
            dx, dr = dev(x), dev(r)
            total, y = (dx, dr) if over == "x" else (dr, dx)
            assert op.compute([na.tensor(y), na.tensor(total)], [na.tensor(dx), na.tensor(dw), na.tensor(dr)]) == na.OK
            torch.cuda.synchronize()
            assert np.array_equal(host(y), want["fp"][0]) and np.array_equal(host(total), want["fp"][2])
        op8 = na.RmsNorm(output_dtype=na.DT_S8)
        dx, codes, scale = dev(x), torch.zeros((rows, cols), dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
        assert op8.compute([na.tensor(codes), na.tensor(scale), na.tensor(dx)],
                           [na.tensor(dx), na.tensor(dw), na.tensor(dev(r))]) == na.OK
        torch.cuda.synchronize()
        for got, want8 in zip((codes, scale, dx), want["s8"]):
            assert np.array_equal(host(got), want8)
