"""The operators for many continuations of one prompt over the paged 8-bit
cache, and the calls that they are measured on.

  fork      KvCacheFork and KvCacheCopy: the next batch's page tables (children
            share their parents' pages, grow, or are given up), and the pages
            that two would write copied;
  compact   KvCacheCompact and KvCacheCopy: the pages in use moved to the lowest
            numbers;
  attn      PrefixAttention: attention for groups of sequences whose first
            tokens lie in the same pages, read once for a group;
  logprobs  TokenLogProbs: log probabilities of given tokens, the entropy, and
            the most probable alternatives.

Every kind has its plain form here (`own` false): elementary torch operations
in 32 bits, rounded once at the end.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
MOST_FLOPS = 6.9e10
MOST_BYTES = 2.6e8
MOST_SCORES = 1.5e9         # bytes of the plain form's padded scores
MOST_HELD = 6.0e8           # bytes of a cache


def listed():
    return [
        # a step of parallel sampling: 64 continuations, each grows by a token,
        # some are given up and others taken twice
        dict(name="fork_step", kind="fork", b=64, n=64, ctx=1500, fan=16, new=1, mixed=False, hkv=8, d=128, page=64,
             spare=0.3),
        # a busy server: many short sequences in small pages, prompts that come
        # in, sequences that end, some cut back
        dict(name="fork_many", kind="fork", b=500, n=517, ctx=1300, fan=7, new=300, mixed=True, hkv=2, d=64, page=16,
             spare=0.6),
        # a small cache packed after a few sequences have ended: latency
        dict(name="compact_small", kind="compact", b=9, ctx=333, fan=3, hkv=4, d=80, page=16, spare=0.4),
        # a large cache packed after a peak of load
        dict(name="compact_large", kind="compact", b=64, ctx=3800, fan=4, hkv=8, d=128, page=64, spare=0.9),
        # four samples of a short prompt: latency
        dict(name="attn_few", kind="attn", groups=1, fan=4, shared=1900, own=90, n=1, mixed=False, hq=32, hkv=8, d=128,
             page=64, dtype="f16"),
        # a serving batch behind one long system prompt
        dict(name="attn_batch", kind="attn", groups=1, fan=64, shared=32768, own=400, n=1, mixed=False, hq=32, hkv=8,
             d=128, page=64, dtype="f16"),
        # several prompts of different lengths, a few beams each, rows of
        # several tokens and of none, in f32 and small pages
        dict(name="attn_groups_f32", kind="attn", groups=5, fan=9, shared=4100, own=300, n=3, mixed=True, hq=16, hkv=4,
             d=64, page=16, dtype="f32"),
        # questions of many tokens about one document
        dict(name="attn_questions", kind="attn", groups=1, fan=12, shared=8000, own=200, n=97, mixed=True, hq=32,
             hkv=8, d=128, page=128, dtype="f16"),
        # the scores of one token of one user, with alternatives: latency
        dict(name="logprobs_one", kind="logprobs", t=1, v=131072, n=1, top=8, dtype="f16"),
        # a beam step: every beam's best candidates
        dict(name="logprobs_beams", kind="logprobs", t=64, v=151000, n=1, top=20, dtype="f16"),
        # a prompt scored, the probabilities alone, an odd vocabulary in f32
        dict(name="logprobs_score", kind="logprobs", t=1025, v=50001, n=1, top=0, dtype="f32"),
        # long texts scored with alternatives at each place
        dict(name="logprobs_long", kind="logprobs", t=4096, v=32000, n=3, top=5, dtype="f16"),
    ]


# --- drawn cases -------------------------------------------------------------

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("fork", "compact", "attn", "attn", "attn", "logprobs", "logprobs"))
    heads = dict(hkv=rng.choice((1, 2, 4, 8, 8)), d=rng.choice((64, 80, 96, 128, 128, 256)),
                 page=rng.choice((16, 32, 64, 128)))
    while True:
        if kind in ("fork", "compact"):
            b = _log_int(rng, 1, 400)
            c = dict(kind=kind, b=b, ctx=_log_int(rng, 1, 8000), fan=rng.randint(1, max(1, min(b, 32))),
                     spare=rng.choice((0.1, 0.5, 1.0)), **heads)
            if kind == "fork":
                c.update(n=_log_int(rng, 1, 500), new=rng.choice((0, 1, 1, 1, 5, _log_int(rng, 1, 900))),
                         mixed=rng.random() < 0.4)
            if _cells(c) * c["page"] * 2 * c["hkv"] * c["d"] * (1.1 + c["spare"]) > MOST_HELD:
                continue
        elif kind == "attn":
            c = dict(kind=kind, groups=rng.choice((1, 1, 1, 2, 5)), fan=_log_int(rng, 1, 64),
                     shared=_log_int(rng, 1, 40000), own=_log_int(rng, 1, 1500),
                     n=rng.choice((1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 200))), mixed=rng.random() < 0.3,
                     hq=heads["hkv"] * rng.choice((1, 4, 4, 7, 8)), **heads,
                     dtype=rng.choice(("f16", "f16", "f32")))
            lens, rows, members, shared = _sequences(c)
            most = max(max(members) * max(rows) * max(shared) * c["groups"],
                       len(lens) * max(rows) * max(x - s for x, s in zip(lens, _of_members(shared, members))))
            held = sum(shared) + sum(lens) - sum(s * m for s, m in zip(shared, members))
            if 4 * most * c["hq"] > MOST_SCORES or 2 * held * c["hkv"] * c["d"] > MOST_HELD:
                continue
        else:
            c = dict(kind=kind, t=_log_int(rng, 1, 5000), v=rng.choice((_log_int(rng, 32, 262144), 32000, 128000)),
                     n=rng.choice((1, 1, 1, 4)), top=rng.choice((0, 1, 5, 20, 32)),
                     dtype=rng.choice(("f16", "f16", "f32")))
        w = work(c)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return c


# --- sequences and their pages ------------------------------------------------

def _cut(case, tokens):
    """The part of the first tokens that fills whole pages."""
    return tokens // case["page"] * case["page"]


def _of_members(per_group, members):
    return [x for x, m in zip(per_group, members) for _ in range(m)]


def _share(i):
    """A fraction in 0.15 .. 1, another for each i; the first is 1."""
    return 0.15 + 0.85 * ((1.0 - 0.618034 * i) % 1.0) if i else 1.0


def _page_lengths(case):
    """Lengths of the sequences of a fork or compact case, and the tokens that
    each shares with the first of its `fan` sequences."""
    lens = [max(1, int(case["ctx"] * _share(i))) for i in range(case["b"])]
    same = [min(lens[i], lens[i - i % case["fan"]]) * 2 // 3 if i % case["fan"] else 0 for i in range(case["b"])]
    return lens, [_cut(case, s) for s in same]


def _cells(case):
    lens, same = _page_lengths(case)
    cells = sum(-(-x // case["page"]) - s // case["page"] for x, s in zip(lens, same))
    if case["kind"] == "fork":
        cells += -(-case["n"] * case["new"] // case["page"])
    return cells


def _sequences(case):
    """Of an attn case: the tokens of each sequence, how many of them are this
    call's rows, the sequences of each group and the tokens that these share."""
    g, fan = case["groups"], case["fan"]
    members = [max(1, fan - 2 * i) for i in range(g)]
    shared = [_cut(case, max(1, int(case["shared"] * _share(i)))) for i in range(g)]
    lens, rows = [], []
    for i, s in enumerate(_of_members(shared, members)):
        n = case["n"]
        if case["mixed"]:
            n = 0 if i % 6 == 5 else 1 if i % 3 == 1 else max(1, n - 2 * i)
        lens.append(s + max(n, 1, int(case["own"] * _share(i))))
        rows.append(n)
    return lens, rows, members, shared


def _table(lens, same, first, page, spare, r):
    """A page table of shuffled pages, the holders of each page, and its
    columns. Sequence i has the first same[i] tokens in first[i]'s pages."""
    per = [-(-x // page) for x in lens]
    fresh = sum(p - s // page for p, s in zip(per, same))
    pages = int(fresh * (1.0 + spare)) + 3
    order = r.permutation(pages).astype(np.int32)
    table = np.full((len(lens), max(per)), -1, dtype=np.int32)
    at = 0
    for i, p in enumerate(per):
        k = same[i] // page
        table[i, :k] = table[first[i], :k]
        table[i, k:p] = order[at:at + p - k]
        at += p - k
    refs = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
    return table, refs


# --- inputs --------------------------------------------------------------------

def _dtype(case):
    return torch.float16 if case["dtype"] == "f16" else torch.float32


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _codes(g, *shape):
    return torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)


def _ints(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(DEV)


def _cache(case, g, pages):
    page, hkv, d = case["page"], case["hkv"], case["d"]
    return dict(kc=_codes(g, pages, hkv, page, d), vc=_codes(g, pages, hkv, d, page),
                ks=0.014 * torch.exp(0.2 * _normal(g, pages, hkv)), vs=0.014 * torch.exp(0.2 * _normal(g, pages, hkv)))


def _inputs(case, seed):
    g, kind = _gen(seed), case["kind"]
    r = np.random.RandomState(int(seed) % (1 << 32))
    if kind == "logprobs":
        t, v = case["t"], case["v"]
        x = _normal(g, t, v).mul_(2.5 * torch.exp(0.4 * _normal(g, t, 1)))
        tokens = torch.randint(0, v, (t, case["n"]), generator=g, device=DEV, dtype=torch.int32)
        return dict(x=x.to(_dtype(case)), tokens=tokens)
    if kind == "attn":
        lens, rows, members, shared = _sequences(case)
        starts = np.cumsum([0] + members)
        first = np.repeat(starts[:-1], members)
        same = _of_members(shared, members)
        same = [s if i != f else 0 for i, (s, f) in enumerate(zip(same, first))]
        table, refs = _table(lens, same, first, case["page"], 0.1, r)
        s = _cache(case, g, len(refs))
        t, hq, d = sum(rows), case["hq"], case["d"]
        # scores of a few units: some heads look at few tokens, some at many
        sharp = torch.exp(0.5 * _normal(g, hq)).repeat_interleave(d)
        packed = _normal(g, t, (hq + 2 * case["hkv"]) * d)
        packed[:, :hq * d] *= sharp
        s.update(q=packed.to(_dtype(case))[:, :hq * d], table=_ints(table), lens=_ints(lens),
                 rows=_ints(np.cumsum([0] + rows)), groups=_ints(starts), shared=_ints(shared))
        return s
    lens, same = _page_lengths(case)
    first = [i - i % case["fan"] for i in range(len(lens))]
    table, refs = _table(lens, same, first, case["page"], case["spare"], r)
    b = len(lens)
    s = dict(lens=_ints(lens), refs=_ints(refs))
    if kind == "fork":
        n = case["n"]
        parents = r.randint(0, b, n)                       # some twice or more, some not at all
        new = np.full(n, case["new"])
        if case["mixed"]:
            parents = np.where(r.rand(n) < 0.6, np.arange(n) % b, parents)
            parents = np.where(r.rand(n) < 0.1, -1, parents)     # a new sequence, or none
            new = np.where(r.rand(n) < 0.7, 1, r.randint(-3, max(1, case["new"]) + 1, n))
        s.update(parents=_ints(parents), new=_ints(new))
        most = max(lens) + max(0, int(new.max()))
        s["wide"] = -(-most // case["page"])
    s["table"] = _ints(table)
    s.update(_cache(case, g, len(refs)))
    return s


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=dict(case))
    kind = case["kind"]
    i32 = dict(dtype=torch.int32, device=DEV)
    f32 = dict(dtype=torch.float32, device=DEV)
    if kind == "logprobs":
        t, n, top = case["t"], case["n"], case["top"]
        out = dict(logprobs=torch.empty((t, n), **f32), entropy=torch.empty(t, **f32))
        if top:
            out.update(top_tokens=torch.empty((t, top), **i32), top_logprobs=torch.empty((t, top), **f32))
    elif kind == "attn":
        out = dict(o=torch.empty(s["q"].shape, dtype=s["q"].dtype, device=DEV))
        s["at"] = _places(case)
    else:
        pages = s["refs"].shape[0]
        out = dict(refs=torch.empty(pages, **i32), counts=torch.empty(2, **i32), kc=s["kc"], vc=s["vc"], ks=s["ks"],
                   vs=s["vs"])
        if kind == "fork":
            n = case["n"]
            out.update(table=torch.empty((n, s["wide"]), **i32), lens=torch.empty(n, **i32),
                       copies=torch.empty((n, 2), **i32))
        else:
            out.update(table=torch.empty_like(s["table"]), copies=torch.empty((pages // 2, 2), **i32),
                       moved=torch.empty(pages, **i32))
    s["out"] = out
    if own:
        # the operators, the tensors' descriptors and the workspace, as a
        # program makes them once per layer
        s["calls"] = _calls(s)
    return s


def _calls(s):
    import nnops_amd as na
    case, out = s["case"], s["out"]
    kind, t = case["kind"], na.tensor
    if kind == "logprobs":
        names = ["logprobs", "entropy"] + (["top_tokens", "top_logprobs"] if case["top"] else [])
        return [_call(na.TokenLogProbs(top=case["top"]), [t(out[x]) for x in names], [t(s["x"]), t(s["tokens"])])]
    pages = [t(s["kc"]), t(s["vc"]), t(s["ks"]), t(s["vs"])]
    if kind == "attn":
        ins = [t(s["q"])] + pages + [t(s["table"]), t(s["lens"]), t(s["groups"]), t(s["shared"])]
        return [_call(na.PrefixAttention(), [t(out["o"])], ins + ([t(s["rows"])] if case["mixed"] else []))]
    copy = _call(na.KvCacheCopy(), pages, [t(out["copies"])])
    held = [t(s["table"]), t(s["lens"]), t(s["refs"])]
    if kind == "fork":
        return [_call(na.KvCacheFork(page_tokens=case["page"]),
                      [t(out[x]) for x in ("table", "lens", "refs", "copies", "counts")],
                      held + [t(s["parents"]), t(s["new"])]), copy]
    return [_call(na.KvCacheCompact(page_tokens=case["page"]),
                  [t(out[x]) for x in ("table", "refs", "copies", "moved", "counts")], held), copy]


def _call(op, outs, ins):
    size = op.workspace_size(ins, outs)
    return op, outs, ins, torch.empty(size, dtype=torch.uint8, device=DEV) if size else None


def run(state):
    if not own:
        return _PLAIN[state["case"]["kind"]](state)
    for op, outs, ins, ws in state["calls"]:
        rc = op.compute(outs, ins, workspace=ws)
        if rc:
            raise RuntimeError(f"compute failed: status {rc}")
    return state["out"]


# --- the plain forms -----------------------------------------------------------

def _held(table, lens, page):
    """Which cells of a page table hold a page of their sequence."""
    return torch.arange(table.shape[1], device=DEV) < ((lens.long() + page - 1) // page)[:, None]


def _count(pages, ids, which):
    """How often each page is among ids[which] (the others count at one past the last)."""
    at = torch.where(which, ids.long(), pages).reshape(-1)
    return torch.zeros(pages + 1, dtype=torch.int64, device=DEV).index_add_(0, at, torch.ones_like(at))


def _in_order(pages, which):
    """The numbers of the pages where `which` holds, ascending, -1 behind them."""
    rank = torch.where(which, which.long().cumsum(0) - 1, pages)
    out = torch.full((pages + 1,), -1, dtype=torch.int64, device=DEV)
    out.scatter_(0, rank, torch.arange(pages, device=DEV))
    out[pages] = -1
    return out


def _copy_pages(s, copies):
    at = copies[copies[:, 0] >= 0].long()
    for x in ("kc", "vc", "ks", "vs"):
        s[x][at[:, 1]] = s[x][at[:, 0]]


def _plain_fork(s):
    page, pages, n, wide = s["case"]["page"], s["refs"].shape[0], s["case"]["n"], s["wide"]
    table, lens, parents = s["table"].long(), s["lens"].long(), s["parents"].long()
    held = _held(table, lens, page)
    child = parents >= 0
    had = torch.where(child, lens[parents.clamp_min(0)], 0)
    will = (had + s["new"].long()).clamp(0, wide * page)
    kept = torch.minimum(had, will)
    cell = torch.arange(wide, device=DEV)
    mine = table[parents.clamp_min(0)]
    mine = torch.nn.functional.pad(mine, (0, max(0, wide - mine.shape[1])), value=-1)[:, :wide]
    shares = cell < ((kept + page - 1) // page)[:, None]
    refs = s["refs"].long() - _count(pages, table, held)[:pages] + _count(pages, mine, shares)[:pages]
    free = refs == 0
    # the page that a child would write into behind the tokens that it keeps
    writes = (will > kept) & (kept % page != 0)
    tail = torch.where(writes, torch.gather(mine, 1, (kept // page).clamp_max(wide - 1)[:, None])[:, 0], pages)
    writers = _count(pages, tail, writes)
    i = torch.arange(n, device=DEV)
    first = torch.full((pages + 1,), n, device=DEV).scatter_reduce_(0, tail, i, "amin")
    alone = torch.nn.functional.pad(refs, (0, 1))[tail] <= writers[tail]
    copied = writes & ~(alone & (first[tail] == i))
    need = (cell < ((will + page - 1) // page)[:, None]) & ~shares
    need |= copied[:, None] & (cell == (kept // page)[:, None])
    at = need.reshape(-1).long().cumsum(0).reshape(n, wide) - 1
    got = torch.where(need, _in_order(pages, free)[at.clamp(0, pages)], -1)
    out = torch.where(need, got, torch.where(shares, mine, -1))
    refs = refs - _count(pages, tail, copied)[:pages] + _count(pages, got, got >= 0)[:pages]
    to = torch.gather(out, 1, (kept // page).clamp_max(wide - 1)[:, None])[:, 0]
    copies = torch.where((copied & (to >= 0))[:, None], torch.stack([tail, to], 1), -1)
    _copy_pages(s, copies)
    counts = torch.stack([(refs == 0).sum(), (need & (got < 0)).sum()])
    i32 = torch.int32
    return dict(table=out.to(i32), lens=will.to(i32), refs=refs.to(i32), copies=copies.to(i32), counts=counts.to(i32),
                kc=s["kc"], vc=s["vc"], ks=s["ks"], vs=s["vs"])


def _plain_compact(s):
    page, pages = s["case"]["page"], s["refs"].shape[0]
    table, refs = s["table"].long(), s["refs"].long()
    used = refs != 0
    total = used.sum()
    number = torch.arange(pages, device=DEV)
    move, room = used & (number >= total), ~used & (number < total)
    src, dst = _in_order(pages, move)[:pages // 2], _in_order(pages, room)[:pages // 2]
    copies = torch.stack([src, dst], 1)
    rank = move.long().cumsum(0) - 1
    moved = torch.where(move, _in_order(pages, room)[rank.clamp_min(0)], torch.where(used, number, -1))
    held = _held(table, s["lens"], page)
    new = torch.where(held, moved[table.clamp(0, pages - 1)], -1)
    back = torch.zeros(pages + 1, dtype=torch.int64, device=DEV)
    back.scatter_(0, torch.where(used, moved, pages), refs)
    _copy_pages(s, copies)
    counts = torch.stack([total, move.sum()])
    i32 = torch.int32
    return dict(table=new.to(i32), refs=back[:pages].to(i32), copies=copies.to(i32), moved=moved.to(i32),
                counts=counts.to(i32), kc=s["kc"], vc=s["vc"], ks=s["ks"], vs=s["vs"])


def _places(case):
    """Where the rows, prefixes and own tokens of an attn case lie in padded tensors."""
    lens, rows, members, shared = _sequences(case)
    b, most = len(lens), max(max(rows), 1)
    group = _of_members(range(len(members)), members)
    place = [i for m in members for i in range(m)]
    first = np.cumsum([0] + members)
    starts = np.cumsum([0] + rows)
    padded = np.full((b, most), -1)
    flat = np.zeros(sum(rows), dtype=np.int64)
    for i, n in enumerate(rows):
        padded[i, :n] = np.arange(starts[i], starts[i + 1])
        flat[starts[i]:starts[i + 1]] = i * most + np.arange(n)
    long = lambda x: torch.tensor(np.asarray(x), dtype=torch.int64, device=DEV)  # noqa: E731
    own_most = max(x - s for x, s in zip(lens, _of_members(shared, members)))
    return dict(group=long(group), place=long(place), first=long(first[:-1]), padded=long(padded), flat=long(flat),
                shared=long(shared), skip=long(_of_members(shared, members)), most=most, members=max(members),
                prefix=max(shared), tail=-(-own_most // case["page"]) * case["page"])


def _plain_attn(s):
    case, at = s["case"], s["at"]
    page, hq, hkv, d = case["page"], case["hq"], case["hkv"], case["d"]
    b, most, fan = s["lens"].shape[0], at["most"], at["members"]
    rep, groups = hq // hkv, at["shared"].shape[0]

    def values(codes, scale, ids, transposed):
        """[.., hkv, d, tokens] of the pages ids [.., pages]."""
        x = codes[ids].float() * scale[ids][..., None, None]
        x = x if transposed else x.transpose(3, 4)
        return x.permute(0, 2, 3, 1, 4).reshape(ids.shape[0], hkv, d, ids.shape[1] * page).contiguous()

    q = s["q"].float().reshape(-1, hkv, rep, d)
    q = q[at["padded"].clamp_min(0)] * (at["padded"] >= 0)[..., None, None, None] * (1.0 / math.sqrt(d))
    # a group's rows side by side, over its prefix
    qg = torch.zeros((groups, fan, most, hkv, rep, d), device=DEV)
    qg[at["group"], at["place"]] = q
    qg = qg.permute(0, 3, 1, 2, 4, 5).reshape(groups, hkv, -1, d)
    ids = s["table"].long()[at["first"]][:, :at["prefix"] // page].clamp_min(0)
    x = torch.matmul(qg, values(s["kc"], s["ks"], ids, False))
    x.masked_fill_(torch.arange(x.shape[-1], device=DEV) >= at["shared"][:, None, None, None], -math.inf)
    # a sequence's rows over its own tokens
    cells = at["skip"][:, None] // page + torch.arange(at["tail"] // page, device=DEV)
    own_ids = torch.gather(s["table"].long(), 1, cells.clamp_max(s["table"].shape[1] - 1)).clamp_min(0)
    y = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(b, hkv, most * rep, d), values(s["kc"], s["ks"], own_ids, False))
    n = (s["rows"][1:] - s["rows"][:-1]).long()
    pos = (s["lens"].long() - n)[:, None] + torch.arange(most, device=DEV)
    token = at["skip"][:, None] + torch.arange(at["tail"], device=DEV)
    unseen = token[:, None] > pos[:, :, None]
    y.reshape(b, hkv, most, rep, -1).masked_fill_(unseen[:, None, :, None], -math.inf)

    def by_sequence(z):
        z = z.reshape(groups, hkv, fan, most * rep, -1).permute(0, 2, 1, 3, 4)
        return z[at["group"], at["place"]]

    top = y.amax(-1, keepdim=True)
    if x.shape[-1]:
        top = torch.maximum(top, by_sequence(x.amax(-1, keepdim=True)))
    y = y.sub_(top).exp_()
    total = y.sum(-1, keepdim=True)
    o = torch.matmul(y, values(s["vc"], s["vs"], own_ids, True).transpose(2, 3).contiguous())
    if x.shape[-1]:
        high = torch.zeros((groups, fan, hkv, most * rep, 1), device=DEV)
        high[at["group"], at["place"]] = top
        x = x.sub_(high.permute(0, 2, 1, 3, 4).reshape(groups, hkv, -1, 1)).exp_()
        total = total + by_sequence(x.sum(-1, keepdim=True))
        o = o + by_sequence(torch.matmul(x, values(s["vc"], s["vs"], ids, True).transpose(2, 3).contiguous()))
    o = (o / total).reshape(b, hkv, most, rep, d).permute(0, 2, 1, 3, 4).reshape(b * most, hq * d)
    return dict(o=o[at["flat"]].to(s["q"].dtype))


def _plain_logprobs(s):
    top = s["case"]["top"]
    x = s["x"].float()
    high = x.amax(dim=1, keepdim=True)
    z = x - high
    e = z.exp()
    total = e.sum(dim=1, keepdim=True)
    log = total.log()
    out = dict(logprobs=torch.gather(z, 1, s["tokens"].long()) - log,
               entropy=(log - (e * z).sum(dim=1, keepdim=True) / total)[:, 0])
    if top:
        # by value, and equal ones by index: both in one whole number
        bits = (x + 0.0).view(torch.int32)
        rank = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() * (1 << 32) - torch.arange(x.shape[1], device=DEV)
        tokens = torch.topk(rank, top, dim=1)[1]
        out.update(top_tokens=tokens.to(torch.int32), top_logprobs=torch.gather(z, 1, tokens) - log)
    return out


_PLAIN = dict(fork=_plain_fork, compact=_plain_compact, attn=_plain_attn, logprobs=_plain_logprobs)


# --- what a call cannot do without, and what it should give ---------------------

def _copied(case):
    """About the pages that a fork copies: one for each child beyond the first of a parent."""
    if case["new"] == 0:
        return 0
    b, n = case["b"], case["n"]
    parents = b * (1.0 - (1.0 - 1.0 / b) ** n) if not case["mixed"] else n * 0.7
    return max(0.0, n - parents) * (1.0 - 1.0 / case["page"])


def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        t, v, e = case["t"], case["v"], 2 if case["dtype"] == "f16" else 4
        return {"bytes": t * v * e + t * (8 * case["n"] + 4 + 8 * case["top"]), "flops": 6.0 * t * v}
    if kind == "attn":
        e = 2 if case["dtype"] == "f16" else 4
        lens, rows, members, shared = _sequences(case)
        skip = _of_members(shared, members)
        keys = sum(shared) + sum(x - s for x, s in zip(lens, skip) if x > s)
        pairs = sum(n * (x - n) + n * (n + 1) // 2 for x, n in zip(lens, rows))
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        return {"bytes": 2 * hkv * d * keys + 8 * hkv * (keys // case["page"] + 1) + 2 * sum(rows) * hq * d * e,
                "flops": 4.0 * pairs * hq * d}
    lens, same = _page_lengths(case)
    page = case["page"]
    cells = sum(-(-x // page) for x in lens)
    per_page = 2 * page * case["hkv"] * case["d"] + 8 * case["hkv"]
    fresh = sum(-(-x // page) - s // page for x, s in zip(lens, same))
    pages = int(fresh * (1.0 + case["spare"])) + 3
    if kind == "fork":
        moved = _copied(case)
        out = case["n"] * (max(lens) + case["new"] + page - 1) // page
    else:
        moved = fresh * (1.0 - fresh / pages)
        out = case["b"] * -(-max(lens) // page) + 2 * pages
    return {"bytes": 4.0 * (cells + out + 2 * pages) + 2.0 * moved * per_page, "flops": float(cells + out + 4 * pages)}


def exact(case, seed):
    kind, f64 = case["kind"], torch.float64
    if kind in ("fork", "compact"):
        # whole numbers, and copies of the scales: nothing is rounded
        return None
    s = _inputs(case, seed)
    if kind == "logprobs":
        lp, entropy, best = [], [], []
        for i in range(0, case["t"], 256):
            x = s["x"][i:i + 256].to(f64)
            p = torch.log_softmax(x, dim=1)
            lp.append(p.gather(1, s["tokens"][i:i + 256].long()))
            entropy.append(-(p.exp() * p).sum(dim=1))
            if case["top"]:
                best.append(torch.sort(p, dim=1, descending=True)[0][:, :case["top"]])
        out = dict(logprobs=torch.cat(lp), entropy=torch.cat(entropy))
        if case["top"]:
            out.update(top_tokens=None, top_logprobs=torch.cat(best))
        return out
    lens, rows, _, _ = _sequences(case)
    page, hq, hkv, d = case["page"], case["hq"], case["hkv"], case["d"]
    o = torch.zeros((sum(rows), hq, d), dtype=f64, device=DEV)
    q = s["q"].to(f64).reshape(-1, hq, d)
    at = 0
    for i, (length, n) in enumerate(zip(lens, rows)):
        if n == 0:
            continue
        ids = s["table"][i, :-(-length // page)].long()
        for h in range(hkv):
            k = (s["kc"][ids, h].to(f64) * s["ks"][ids, h].to(f64)[:, None, None]).reshape(-1, d)[:length]
            v = s["vc"][ids, h].to(f64) * s["vs"][ids, h].to(f64)[:, None, None]
            v = v.transpose(1, 2).reshape(-1, d)[:length]
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            x = (q[at:at + n, heads].reshape(-1, d) @ k.T / math.sqrt(d)).reshape(n, -1, length)
            last = length - n + torch.arange(n, device=DEV)
            x.masked_fill_((torch.arange(length, device=DEV) > last[:, None])[:, None], -math.inf)
            o[at:at + n, heads] = (torch.softmax(x, dim=2).reshape(-1, length) @ v).reshape(n, -1, d)
        at += n
    return dict(o=o.reshape(-1, hq * d))


if __name__ == "__main__":
    _rng = random.Random(1)
    for _c in listed() + [draw(_rng) for _ in range(12)]:
        _w = work(_c)
        print(_c, "%.3g bytes, %.3g flops" % (_w["bytes"], _w["flops"]))
