"""The decoder layer of examples/decoder_layer.py: prompts and then single
tokens through all its operators, each step against its plain form in 64 bits
over the step's own inputs."""
from __future__ import annotations

import importlib.util
import os

import numpy as np
import pytest

import decoder_ref as ref
import nnops_amd as na
from gpu_util import host, announce

pytestmark = pytest.mark.gpu


def _example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decoder_layer.py")
    spec = importlib.util.spec_from_file_location("decoder_layer", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _dense(weight, k):
    """A Q4_1 weight's values."""
    return host(na.q4_1_dequantize(weight._keep[-1], k)).astype(np.float64)


def _close(got, want, size, rel):
    """|got - want| within rel of size: the sum of the products' sizes where the
    products' operands are rounded, plus the result's own rounding to f16."""
    got = got.astype(np.float64)
    tol = rel * size + 1.01 * 2.0 ** -11 * abs(want) + 2.0 ** -24
    assert np.max(abs(got - want) / tol) <= 1.0, np.max(abs(got - want) / tol)


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_prompts_then_tokens(window, sinks):
    import torch
    announce(f"decoder layer window={window}")
    width, heads, kv, d, ffn, page = 256, 8, 2, 64, 512, 16
    layer = _example().DecoderLayer(width, heads, kv, d, ffn, page_tokens=page, pages=64, max_tokens=256,
                                    window=window, sinks=sinks)
    lens = np.array([70, 1, 33, 128])
    per = 10
    table = torch.randperm(64, generator=torch.Generator().manual_seed(3))[:4 * per].reshape(4, per).int().cuda()
    gen = torch.Generator().manual_seed(4)
    o, up, down = _dense(layer.o, heads * d), _dense(layer.up, width), _dense(layer.down, ffn)
    rot = host(layer.table)
    kc, vc = (host(z).copy() for z in layer.cache[:2])
    ks, vs = (host(z).copy() for z in layer.cache[2:])
    for step in range(4):
        rows = lens if step == 0 else np.ones(4, int)
        starts = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda")
        pos = np.concatenate([np.arange(n - r, n) for n, r in zip(lens, rows)]).astype(np.int32)
        x = torch.randn((int(rows.sum()), width), generator=gen).half().cuda()
        out = layer(x, torch.from_numpy(pos).cuda(), starts if step % 2 == 0 else None,
                    torch.tensor(lens, dtype=torch.int32, device="cuda"), table)
        torch.cuda.synchronize()
        s = {k: host(z) for k, z in layer.steps.items()}
        xs, tab = host(x), host(table)
        # the norm's codes: within half a step, the scale's and the factor's f32 roundings beside it
        _, norm, _ = ref.rms_norm(xs, host(layer.norm1))
        scale = s["scale"].astype(np.float64)[:, None]
        assert np.max(abs(s["codes"] * scale - norm) / scale) <= 0.5 + 127 * 2.0 ** -20
        # q, k, v: the product of codes is exact; then f32 roundings, f16, and the rotation's of q and k
        plain = (s["codes"].astype(np.float64) @ host(layer.qkv).astype(np.float64).T) * scale
        plain *= host(layer.qkv_scale).astype(np.float64)
        n_qk = (heads + kv) * d
        turned, size = ref.rotary(plain[:, :n_qk], pos, rot, heads + kv, d, d, False)
        _close(s["qkv"][:, :n_qk], turned, size, 1.01 * 2.0 ** -11)
        _close(s["qkv"][:, n_qk:], plain[:, n_qk:], abs(plain[:, n_qk:]), 2.0 ** -22)
        # the cache: its codes are defined to the bit
        k, v = s["qkv"][:, heads * d:n_qk], s["qkv"][:, n_qk:]
        ref.kv_write(k, kc, ks, tab, lens, rows)
        vt = vc.transpose(0, 1, 3, 2).copy()
        ref.kv_write(v, vt, vs, tab, lens, rows)
        vc = vt.transpose(0, 1, 3, 2).copy()
        for got, want in zip(layer.cache, (kc, vc, ks, vs)):
            assert np.array_equal(host(got), want)
        want, weight, spread = ref.attention(s["qkv"][:, :heads * d], kc, vc, ks, vs, tab, lens, rows, window=window,
                                             sinks=sinks)
        tol = ref.attention_tolerance(True, want, weight, spread, vs[vs > 0])
        assert np.all(abs(s["o"] - want) <= tol)
        # Q4_1 products: weights as f16 (2^-11 of each) and f32 sums
        f16 = lambda a: a.astype(np.float64)
        _close(s["y"], f16(s["o"]) @ o.T, abs(f16(s["o"])) @ abs(o).T, 1.1 * 2.0 ** -11)
        total, normed, _ = ref.rms_norm(s["y"], host(layer.norm2), xs)
        # (the norm is of the sum before its rounding, or after it: 2^-11 either way)
        _close(s["normed"], normed, abs(normed), 2.02 * 2.0 ** -11)
        both = f16(s["normed"]) @ up.T
        size = abs(f16(s["normed"])) @ abs(up).T * 1.1 * 2.0 ** -11
        gate, val = both[:, :ffn], both[:, ffn:]
        silu = gate / (1 + np.exp(-gate))
        hidden = silu * val
        # |silu'| <= 1.1; the gated product's own rounding to f16
        err = 1.1 * size[:, :ffn] * abs(val) + (abs(silu) + 1.1 * size[:, :ffn]) * size[:, ffn:] + 2.0 ** -11 * abs(hidden)
        want = hidden @ down.T
        size = err @ abs(down).T + 1.2 * 2.0 ** -11 * (abs(hidden) @ abs(down).T)
        tol = size + 2.02 * 2.0 ** -11 * (abs(total) + abs(want)) + 2.0 ** -20
        assert np.all(abs(host(out) - (total + want)) <= tol)
        lens = lens + 1
