"""A decoder layer over a paged 8-bit cache, from the framework's operators:

    norm to s8 codes -> s8 Linear (q, k, v) -> rotary positions of q and k in
    place -> cache write -> attention over the cache -> Q4_1 Linear
    norm of (x + that) -> gated Q4_1 Linear -> Q4_1 Linear added to the sum

A call takes any mixture of prompts, chunks of prompts and single tokens: the
rows of sequence b are x[starts[b] : starts[b + 1]], the last tokens of its
lengths[b].

    python examples/decoder_layer.py [--width 4096 --heads 32 --kv-heads 8 ...]
"""
from __future__ import annotations

import argparse
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

import nnops_amd as na


def q4_1(w):
    """A Q4_1 weight of a float one [N, K]."""
    return na.tensor(na.q4_1_quantize(w), dtype=na.DT_Q4_1, shape=list(w.shape))


class DecoderLayer:
    def __init__(self, width, heads, kv_heads, head_dim, ffn, *, page_tokens=64, pages=256, max_tokens=8192,
                 window=0, sinks=0, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(n, k):
            return torch.randn((n, k), generator=g, device="cuda", dtype=torch.float32) / k ** 0.5

        self.width, self.heads, self.kv_heads, self.head_dim, self.ffn = width, heads, kv_heads, head_dim, ffn
        self.page_tokens, self.per = page_tokens, -(-max_tokens // page_tokens)
        n = (heads + 2 * kv_heads) * head_dim
        w = weight(n, width)
        self.qkv_scale = w.abs().amax(1) / 127.0
        self.qkv = torch.round(w / self.qkv_scale[:, None]).to(torch.int8)
        self.o, self.up = q4_1(weight(width, heads * head_dim)), q4_1(weight(2 * ffn, width))
        self.down = q4_1(weight(width, ffn))
        self.norm1 = 1.0 + 0.1 * torch.randn(width, generator=g, device="cuda", dtype=torch.float32)
        self.norm1, self.norm2 = self.norm1.half(), torch.ones(width, device="cuda", dtype=torch.float16)
        self.table = na.rotary_table(max_tokens, head_dim)
        self.cache = na.kv_cache(pages, kv_heads, page_tokens, head_dim)
        self.to_codes, self.to_f16 = na.RmsNorm(output_dtype=na.DT_S8), na.RmsNorm()
        self.linear = na.Linear(output_dtype=na.DT_F16)
        self.gated = na.Linear(output_dtype=na.DT_F16, gated=True, gate_activation=na.EP_SILU)
        self.linear_add = na.Linear(output_dtype=na.DT_F16, add_to=True)
        self.rotary = na.Rotary(head_dim=head_dim)
        self.write, self.attention = na.KvCacheWrite(), na.CacheAttention(window=window, sinks=sinks)
        self.prefix_attention = na.PrefixAttention()

    def __call__(self, x, positions, starts, lengths, page_table, groups=None):
        """x f16 [T, width]; positions s32 [T]; starts s32 [B + 1], or None where
        every sequence has as many rows; lengths s32 [B] with these rows;
        page_table s32 [B, pages of a sequence]; groups: (s32 [G + 1], s32 [G])
        where sequences share first tokens (without a window). Returns the layer's
        output."""
        t, d, hq, hk = x.shape[0], self.head_dim, self.heads, self.kv_heads
        new = dict(device=x.device, dtype=torch.float16)
        codes, scale = torch.empty_like(x, dtype=torch.int8), torch.empty(t, device=x.device)
        qkv = torch.empty((t, (hq + 2 * hk) * d), **new)
        q, qk = qkv[:, :hq * d], qkv[:, :(hq + hk) * d]
        k, v = qkv[:, hq * d:(hq + hk) * d], qkv[:, (hq + hk) * d:]
        o, y, total, normed = (torch.empty((t, w), **new) for w in (hq * d, self.width, self.width, self.width))
        hidden = torch.empty((t, self.ffn), **new)
        T = na.tensor
        where = [T(page_table), T(lengths)]
        ends = [] if starts is None else [T(starts)]
        pages = [T(z) for z in self.cache]

        def run(op, outs, ins):
            rc = op.compute(outs, ins)
            if rc != na.OK:
                raise RuntimeError(f"{type(op).__name__}: status {rc}")

        run(self.to_codes, [T(codes), T(scale)], [T(x), T(self.norm1)])
        run(self.linear, [T(qkv)], [T(codes, scale_data=scale, granularity=1),
                                    T(self.qkv, scale_data=self.qkv_scale, granularity=1)])
        run(self.rotary, [T(qk)], [T(qk), T(positions), T(self.table)])
        run(self.write, pages, [T(k), T(v)] + where + ends)
        if groups is None:
            run(self.attention, [T(o)], [T(q)] + pages + where + ends)
        else:
            run(self.prefix_attention, [T(o)], [T(q)] + pages + where + [T(g) for g in groups] + ends)
        run(self.linear, [T(y)], [T(o), self.o])
        run(self.to_f16, [T(normed), T(total)], [T(y), T(self.norm2), T(x)])
        run(self.gated, [T(hidden)], [T(normed), self.up])
        run(self.linear_add, [T(total)], [T(hidden), self.down])
        self.steps = dict(codes=codes, scale=scale, qkv=qkv, o=o, y=y, normed=normed)
        return total


def main():
    a = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("width", 4096), ("heads", 32), ("kv-heads", 8), ("head-dim", 128), ("ffn", 14336),
                        ("sequences", 16), ("prompt", 512), ("steps", 32)):
        a.add_argument("--" + name, type=int, default=value)
    a = a.parse_args()
    lens = [max(1, a.prompt - 17 * b) for b in range(a.sequences)]       # ragged prompts
    per = -(-(a.prompt + a.steps) // 64)
    layer = DecoderLayer(a.width, a.heads, a.kv_heads, a.head_dim, a.ffn, pages=a.sequences * per,
                         max_tokens=a.prompt + a.steps)
    table = torch.randperm(a.sequences * per, device="cuda").reshape(a.sequences, per).int()
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0] + lens, device="cuda").cumsum(0).int()
    pos = torch.cat([torch.arange(n) for n in lens]).int().cuda()
    x = torch.randn((sum(lens), a.width), device="cuda").half()

    def timed(label, rows, f):
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        y = f()
        torch.cuda.synchronize()
        print(f"{label}: {rows} rows, {(time.perf_counter() - t0) * 1e3:.3f} ms")
        return y

    layer(x, pos, starts, length, table)         # (loads the kernels; writes what the next call writes again)
    y = timed("prompts", sum(lens), lambda: layer(x, pos, starts, length, table))
    y = y[(starts[1:] - 1).long()].contiguous()

    def decode():
        z = y
        for _ in range(a.steps):
            pos = length.clone()
            length.add_(1)
            z = layer(z, pos, None, length, table)
        return z

    z = timed(f"{a.steps} tokens each", a.steps * a.sequences, decode)
    assert torch.isfinite(z.float()).all()


if __name__ == "__main__":
    main()
