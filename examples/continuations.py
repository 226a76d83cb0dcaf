"""Beam search over a decoder layer and a paged 8-bit cache: every prompt's beams
share the prompt's pages, a step scores all of them and keeps the best.

    layer (PrefixAttention reads a prompt once for its beams) -> norm -> s8 Linear
    -> TokenLogProbs: each beam's best candidates -> the best beams of each prompt
    -> KvCacheFork: their tables; KvCacheCopy: the pages that two would write into

    python examples/continuations.py [--prompts 2 --beams 8 --prompt 2000 --steps 32 ...]
"""
from __future__ import annotations

import argparse
import time

import torch

import decoder_layer
import nnops_amd as na


def run(op, outs, ins):
    rc = op.compute([na.tensor(t) for t in outs], [na.tensor(t) for t in ins])
    if rc != na.OK:
        raise RuntimeError(f"{type(op).__name__}: status {rc}")


class Beams:
    """`beams` continuations of each of `prompts` prompts over one layer."""

    def __init__(self, layer, vocab, prompts, beams, pages, *, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.layer, self.vocab, self.prompts, self.beams, self.pages = layer, vocab, prompts, beams, pages
        self.embedding = torch.randn((vocab, layer.width), generator=g, device="cuda").half()
        w = torch.randn((vocab, layer.width), generator=g, device="cuda") / layer.width ** 0.5
        self.scale = w.abs().amax(1) / 127.0
        self.head = torch.round(w / self.scale[:, None]).to(torch.int8)
        self.norm = torch.ones(layer.width, device="cuda", dtype=torch.float16)
        self.linear, self.codes = na.Linear(output_dtype=na.DT_F16), na.RmsNorm(output_dtype=na.DT_S8)
        self.log_probs = na.TokenLogProbs(top=beams)
        self.fork, self.copy = na.KvCacheFork(page_tokens=layer.page_tokens), na.KvCacheCopy()
        self.compact = na.KvCacheCompact(page_tokens=layer.page_tokens)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.refs, self.counts = torch.zeros(pages, **i32), torch.empty(2, **i32)
        self.moved = torch.empty(pages, **i32)
        self.table, self.lengths = torch.empty((0, layer.per), **i32), torch.empty(0, **i32)

    def continue_from(self, parents, new_tokens):
        """The next batch: its tables, and the pages copied that it will write into."""
        n = parents.shape[0]
        table, lengths, copies = (torch.empty(s, dtype=torch.int32, device="cuda") for s in ((n, self.layer.per), n, (n, 2)))
        run(self.fork, [table, lengths, self.refs, copies, self.counts],
            [self.table, self.lengths, self.refs, parents, new_tokens])
        run(self.copy, self.layer.cache, [copies])
        self.table, self.lengths = table, lengths

    def pack(self):
        """The pages in use at the lowest numbers."""
        copies = torch.empty((self.pages // 2, 2), dtype=torch.int32, device="cuda")
        run(self.compact, [self.table, self.refs, copies, self.moved, self.counts], [self.table, self.lengths, self.refs])
        run(self.copy, self.layer.cache, [copies])

    def score(self, x):
        """Each row's best candidates: tokens and log probabilities."""
        t = x.shape[0]
        codes, scale = torch.empty_like(x, dtype=torch.int8), torch.empty(t, device="cuda")
        logits = torch.empty((t, self.vocab), dtype=torch.float16, device="cuda")
        run(self.codes, [codes, scale], [x, self.norm])
        rc = self.linear.compute([na.tensor(logits)], [na.tensor(codes, scale_data=scale, granularity=1),
                                                       na.tensor(self.head, scale_data=self.scale, granularity=1)])
        if rc != na.OK:
            raise RuntimeError(f"Linear: status {rc}")
        none = torch.empty((t, 0), dtype=torch.int32, device="cuda")
        tokens = torch.empty((t, self.beams), dtype=torch.int32, device="cuda")
        best, entropy = torch.empty((t, self.beams), device="cuda"), torch.empty(t, device="cuda")
        run(self.log_probs, [torch.empty((t, 0), device="cuda"), entropy, tokens, best], [logits, none])
        return tokens, best

    def __call__(self, prompts, steps):
        """prompts: lists of tokens. Returns tokens [prompts, beams, steps] and their
        log probabilities [prompts, beams]."""
        p, b = self.prompts, self.beams
        i32 = dict(dtype=torch.int32, device="cuda")
        size = torch.tensor([len(t) for t in prompts], **i32)
        self.continue_from(torch.full((p,), -1, **i32), size)
        starts = torch.cat([size.new_zeros(1), size.cumsum(0).int()])
        flat = torch.cat([torch.as_tensor(t) for t in prompts]).long().cuda()
        pos = torch.cat([torch.arange(len(t)) for t in prompts]).int().cuda()
        x = self.layer(self.embedding[flat], pos, starts, self.lengths, self.table)
        tokens, total = self.score(x[(starts[1:] - 1).long()].contiguous())
        # every prompt's first beams are its best first tokens
        history, parent = tokens.reshape(p, b, 1), torch.arange(p, **i32).repeat_interleave(b)
        tokens, total = tokens.reshape(-1), total.reshape(p, b)
        one, groups = torch.ones(p * b, **i32), torch.arange(0, p * b + 1, b, **i32)
        for _ in range(steps - 1):
            self.continue_from(parent, one)
            x = self.layer(self.embedding[tokens.long()], self.lengths - 1, None, self.lengths, self.table, (groups, size))
            candidates, best = self.score(x)
            # of the beams' candidates the best b of each prompt (the first, of equal ones)
            all_of = (total[:, :, None] + best.reshape(p, b, b)).reshape(p, b * b)
            total, at = torch.sort(all_of, dim=1, descending=True, stable=True)
            total, at = total[:, :b].contiguous(), at[:, :b]
            tokens = candidates.reshape(p, b * b).gather(1, at)
            history = torch.cat([history.gather(1, (at // b)[..., None].expand(-1, -1, history.shape[2])), tokens[..., None]], 2)
            parent = (torch.arange(p, device="cuda")[:, None] * b + at // b).reshape(-1).int()
            tokens = tokens.reshape(-1).int()
        return history, total


def main(argv=None):
    a = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("width", 4096), ("heads", 32), ("kv-heads", 8), ("head-dim", 128), ("ffn", 14336),
                        ("vocab", 32000), ("prompts", 2), ("beams", 8), ("prompt", 2000), ("steps", 32)):
        a.add_argument("--" + name, type=int, default=value)
    a = a.parse_args(argv)
    per = -(-(a.prompt + a.steps) // 64)
    pages = a.prompts * (per + a.beams * (2 + a.steps // 32)) + 8
    layer = decoder_layer.DecoderLayer(a.width, a.heads, a.kv_heads, a.head_dim, a.ffn, pages=pages,
                                       max_tokens=a.prompt + a.steps)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, a.vocab, (max(1, a.prompt - 17 * i),), generator=g).tolist() for i in range(a.prompts)]
    for label in ("first", "again"):
        beams = Beams(layer, a.vocab, a.prompts, a.beams, pages)
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        history, total = beams(prompts, a.steps)
        torch.cuda.synchronize()
        print(f"{label}: {a.steps} steps of {a.prompts} x {a.beams} beams, {(time.perf_counter() - t0) * 1e3:.2f} ms")
    beams.pack()
    print(f"pages: {beams.counts.tolist()[0]} of {pages} in use; best: {total[:, 0].tolist()}")
    return history, total, beams


if __name__ == "__main__":
    main()
