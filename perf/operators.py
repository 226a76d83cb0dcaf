"""The operators around the int8 products of a decoder layer, and the calls
that they are measured on.

  norm    RmsNorm: the residual's addition, the root-mean-square norm, and the
          result in f16 / f32 or as s8 codes with one scale per token;
  rotary  rotary positions over the heads of a packed q|k buffer;
  cache   KvCacheWrite and KvCacheRead: new keys and values quantized into the
          pages of an 8-bit cache (one scale per page and head), and the
          sequences read back;
  attn    CacheAttention: causal attention over that cache, for single tokens,
          prompts and ragged mixtures of both, with an optional sliding window
          and first tokens that stay visible.

Every kind has its plain form here (`own` false): elementary torch operations
in 32 bits, rounded once at the end.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
TINY = 2.0 ** -100          # the smallest scale of a page
MOST_FLOPS = 1.3e11
MOST_BYTES = 2.6e8
MOST_PAIRS = 1.0e9          # entries of the plain form's padded score matrix


def listed():
    return [
        # a decode batch between two int8 layers of a 4096-wide model: the
        # residual added, the norm's rows as codes with a scale per token
        dict(name="norm_decode_s8", kind="norm", rows=8, c=4096, residual=True, out="s8", dtype="f16"),
        # the same over a long prefill
        dict(name="norm_prefill_s8", kind="norm", rows=4096, c=4096, residual=True, out="s8", dtype="f16"),
        # a final norm over a ragged prompt, a width that is not a multiple of
        # anything, the output left in f16
        dict(name="norm_odd_f16", kind="norm", rows=777, c=5001, residual=False, out="fp", dtype="f16"),
        # one step of a serving batch: q and k heads of the fused projection
        dict(name="rotary_decode", kind="rotary", t=32, heads=40, d=128, rot=128, interleaved=False, most=32768,
             dtype="f16"),
        # a prompt of a model that rotates half of each head in adjacent pairs, in f32
        dict(name="rotary_prefill_part", kind="rotary", t=2049, heads=40, d=128, rot=64, interleaved=True, most=8192,
             dtype="f32"),
        # a step of a serving batch: a token appended to each sequence (its page
        # requantized where its scale grows), and the sequences handed on in f16
        dict(name="cache_append_read", kind="cache", b=32, ctx=1000, n=1, mixed=False, hkv=8, d=128, page=64,
             dtype="f16"),
        # a prompt written in one go behind a short prefix, and read back
        dict(name="cache_prompt_read", kind="cache", b=1, ctx=4107, n=4096, mixed=False, hkv=8, d=128, page=16,
             dtype="f16"),
        # one token of one user over a short context: latency
        dict(name="attn_decode_one", kind="attn", b=1, ctx=777, n=1, mixed=False, hq=32, hkv=8, d=128, page=64,
             window=0, sinks=0, dtype="f16"),
        # a serving batch of contexts of many lengths
        dict(name="attn_decode_batch", kind="attn", b=64, ctx=4096, n=1, mixed=False, hq=32, hkv=8, d=128, page=64,
             window=0, sinks=0, dtype="f16"),
        # one token over a very long context
        dict(name="attn_decode_long", kind="attn", b=1, ctx=126976, n=1, mixed=False, hq=32, hkv=8, d=128, page=128,
             window=0, sinks=0, dtype="f16"),
        # a prompt
        dict(name="attn_prefill", kind="attn", b=1, ctx=4096, n=4096, mixed=False, hq=32, hkv=8, d=128, page=64,
             window=0, sinks=0, dtype="f16"),
        # chunks of prompts and single tokens in one call, with a sliding window
        # and four first tokens that stay visible, in f32
        dict(name="attn_mixed_window", kind="attn", b=7, ctx=2500, n=301, mixed=True, hq=16, hkv=4, d=64, page=16,
             window=1024, sinks=4, dtype="f32"),
    ]


# --- drawn cases -------------------------------------------------------------

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "rotary", "cache", "cache", "attn", "attn", "attn", "attn"))
    dtype = rng.choice(("f16", "f16", "f32"))
    while True:
        if kind == "norm":
            c = dict(kind=kind, rows=_log_int(rng, 1, 4096),
                     c=rng.choice((1024, 4096, 11008, 14336, _log_int(rng, 1, 16384), _log_int(rng, 64, 16384))),
                     residual=rng.random() < 0.7, out=rng.choice(("s8", "s8", "fp")), dtype=dtype)
        elif kind == "rotary":
            d = rng.choice((64, 80, 96, 128, 256))
            c = dict(kind=kind, t=_log_int(rng, 1, 4096), heads=rng.choice((1, 5, 12, 40, 64)), d=d,
                     rot=rng.choice((d, d, d // 2)), interleaved=rng.random() < 0.4,
                     most=rng.choice((4096, 32768, 131072)), dtype=dtype)
        else:
            c = dict(kind=kind, b=_log_int(rng, 1, 64), ctx=_log_int(rng, 1, 40000),
                     n=rng.choice((1, 1, 1, rng.randint(2, 8), _log_int(rng, 16, 2048))), mixed=False)
            c["n"] = min(c["n"], c["ctx"])
            c["mixed"] = c["b"] > 1 and rng.random() < 0.3
            hkv = rng.choice((1, 2, 4, 8, 8, 8))
            if kind == "attn":
                c.update(hq=hkv * rng.choice((1, 4, 4, 7, 8)))
            c.update(hkv=hkv, d=rng.choice((64, 80, 96, 128, 128, 128, 256)), page=rng.choice((16, 32, 64, 128)))
            if kind == "attn":
                w = rng.random() < 0.35
                c.update(window=_log_int(rng, 1, 4096) if w else 0, sinks=rng.choice((0, 4, 17)) if w else 0)
            c["dtype"] = dtype
        w = work(c)
        pairs = c["b"] * c["hq"] * c["n"] * c["ctx"] if kind == "attn" else 0
        held = c["b"] * c["ctx"] * c["hkv"] * c["d"] if kind in ("attn", "cache") else 0
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS and pairs <= MOST_PAIRS and 2 * held <= MOST_BYTES:
            return c


# --- inputs ------------------------------------------------------------------

def _dtype(case):
    return torch.float16 if case["dtype"] == "f16" else torch.float32


def _lengths(case):
    """Tokens that each sequence holds, and how many of them are this call's
    rows. The first sequence is the longest; in a mixed call every second
    sequence brings a single token, and one in five none."""
    lens, rows = [], []
    for i in range(case["b"]):
        length = max(1, int(case["ctx"] * (0.15 + 0.85 * ((1.0 - 0.618034 * i) % 1.0)))) if i else case["ctx"]
        n = case["n"]
        if case["mixed"]:
            n = 0 if i % 5 == 4 else 1 if i % 2 else max(1, n - 3 * i)
        n = min(n, length) if case["mixed"] else n
        lens.append(max(length, n))
        rows.append(n)
    return lens, rows


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)


def _cache(case, g, lens):
    """A cache of shuffled pages that holds codes of earlier tokens, and its page table."""
    page, hkv, d = case["page"], case["hkv"], case["d"]
    per = [-(-n // page) for n in lens]
    most = max(per)
    total = sum(per) + 3
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros((len(lens), most), dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = order[at:at + n]
        at += n
    kc = _normal(g, total, hkv, page, d).mul_(36.0).round_().clamp_(-127, 127).to(torch.int8)
    vc = _normal(g, total, hkv, d, page).mul_(36.0).round_().clamp_(-127, 127).to(torch.int8)
    ks = 0.028 * torch.exp(0.2 * _normal(g, total, hkv))
    vs = 0.028 * torch.exp(0.2 * _normal(g, total, hkv))
    return dict(kc=kc, vc=vc, ks=ks, vs=vs, table=table)


def _inputs(case, seed):
    g, kind, dt = _gen(seed), case["kind"], _dtype(case)
    if kind == "norm":
        rows, c = case["rows"], case["c"]
        # rows of different sizes, a few channels far larger than the others
        big = 1.0 + 20.0 * (torch.rand(c, generator=g, device=DEV) < 0.002).float()
        s = dict(x=(_normal(g, rows, c) * torch.exp(0.5 * _normal(g, rows, 1)) * big).to(dt),
                 w=(1.0 + 0.2 * _normal(g, c)).to(dt))
        if case["residual"]:
            s["r"] = (_normal(g, rows, c) * big).to(dt)
        return s
    if kind == "rotary":
        t, heads, d, rot = case["t"], case["heads"], case["d"], case["rot"]
        # q and k heads lie before the v heads of the fused projection's rows
        packed = _normal(g, t, (heads + 8) * d).to(dt)
        pos = torch.randint(0, case["most"], (t,), generator=g, device=DEV, dtype=torch.int32)
        freq = 10000.0 ** (-2.0 * torch.arange(rot // 2, device=DEV, dtype=torch.float64) / rot)
        angle = torch.arange(case["most"], device=DEV, dtype=torch.float64)[:, None] * freq
        return dict(x=packed[:, :heads * d], pos=pos, table=torch.cat([angle.cos(), angle.sin()], 1).float())
    lens, rows = _lengths(case)
    s = _cache(case, g, lens)
    t, hkv, d = sum(rows), case["hkv"], case["d"]
    hq = case.get("hq", hkv)
    packed = _normal(g, t, (hq + 2 * hkv) * d).to(dt)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s["starts"] = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32, device=DEV)
    if kind == "attn":
        # scores of a few units: some heads look at few tokens, some at many
        sharp = torch.exp(0.5 * _normal(g, hq)).repeat_interleave(d)
        s["q"] = (packed[:, :hq * d].float() * sharp).to(dt)
    else:
        s["k"], s["v"] = packed[:, hq * d:(hq + hkv) * d], packed[:, (hq + hkv) * d:]
    return s


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=dict(case))
    kind, dt = case["kind"], _dtype(case)
    if kind == "norm":
        rows, c = case["rows"], case["c"]
        out = dict(y=torch.empty((rows, c), dtype=dt, device=DEV))
        if case["residual"]:
            out["sum"] = torch.empty((rows, c), dtype=dt, device=DEV)
    elif kind == "rotary":
        out = dict(y=torch.empty((case["t"], case["heads"] * case["d"]), dtype=dt, device=DEV))
    elif kind == "cache":
        lens, _ = _lengths(case)
        at = (sum(lens), case["hkv"] * case["d"])
        s["all"] = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
        out = dict(k=torch.empty(at, dtype=dt, device=DEV), v=torch.empty(at, dtype=dt, device=DEV),
                   k_scale=s["ks"], v_scale=s["vs"])
    else:
        out = dict(o=torch.empty(s["q"].shape, dtype=dt, device=DEV))
    s["out"] = out
    if own:
        # the operators, the tensors' descriptors and the workspace, as a
        # program makes them once per layer
        s["calls"] = _calls(s)
    return s


def _calls(s):
    import nnops_amd as na
    case, out = s["case"], s["out"]
    kind, dt = case["kind"], na.DT_F16 if case["dtype"] == "f16" else na.DT_F32
    t = na.tensor
    if kind == "norm":
        x, w, r = t(s["x"]), t(s["w"]), [t(s["r"])] if "r" in s else []
        h = [t(out["sum"])] if "r" in s else []
        if case["out"] == "fp":
            return [_call(na.RmsNorm(epsilon=EPS, output_dtype=dt), [t(out["y"])] + h, [x, w] + r)]
        # the codes and scales, and the values that they stand for
        s["codes"] = torch.empty((case["rows"], case["c"]), dtype=torch.int8, device=DEV)
        s["scale"] = torch.empty(case["rows"], dtype=torch.float32, device=DEV)
        s["zero"] = torch.zeros(case["rows"], dtype=torch.int8, device=DEV)
        q, sc = t(s["codes"]), t(s["scale"])
        return [_call(na.RmsNorm(epsilon=EPS, output_dtype=na.DT_S8), [q, sc] + h, [x, w] + r),
                _call(na.DequantizeLinear(axis=0, output_dtype=dt), [t(out["y"])], [q, sc, t(s["zero"])])]
    if kind == "rotary":
        op = na.Rotary(head_dim=case["d"], rotary_dim=case["rot"], interleaved=case["interleaved"])
        return [_call(op, [t(out["y"])], [t(s["x"]), t(s["pos"]), t(s["table"])])]
    pages = [t(s["kc"]), t(s["vc"]), t(s["ks"]), t(s["vs"])]
    where = [t(s["table"]), t(s["lens"])]
    starts = [t(s["starts"])] if case["mixed"] else []     # else: as many rows for each sequence
    if kind == "cache":
        return [_call(na.KvCacheWrite(), pages, [t(s["k"]), t(s["v"])] + where + starts),
                _call(na.KvCacheRead(output_dtype=dt), [t(out["k"]), t(out["v"])], pages + where + [t(s["all"])])]
    op = na.CacheAttention(window=case["window"], sinks=case["sinks"])
    return [_call(op, [t(out["o"])], [t(s["q"])] + pages + where + starts)]


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


# --- the plain forms ---------------------------------------------------------

def _plain_norm(s):
    case, dt = s["case"], s["x"].dtype
    h = s["x"].float()
    if case["residual"]:
        h = h + s["r"].float()
    rstd = torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS)
    u = h * s["w"].float()
    if case["out"] == "s8":
        # the codes do not depend on rstd: u's largest magnitude is 127 steps
        a = u.abs().amax(dim=1, keepdim=True)
        inv = torch.where(a >= 2.0 ** -119, (1.0 / a) * 127.0, torch.zeros_like(a))
        y = (torch.round(u * inv).clamp(-127, 127) * (a * rstd * (1.0 / 127.0))).to(dt)
    else:
        y = (u * rstd).to(dt)
    return dict(y=y, sum=h.to(dt)) if case["residual"] else dict(y=y)


def _plain_rotary(s):
    case = s["case"]
    t, heads, d, rot = case["t"], case["heads"], case["d"], case["rot"]
    x = s["x"].reshape(t, heads, d).float()
    row = s["table"][s["pos"].long()][:, None]
    cos, sin = row[..., :rot // 2], row[..., rot // 2:]
    y = x.clone()
    a = x[..., 0:rot:2] if case["interleaved"] else x[..., :rot // 2]
    b = x[..., 1:rot:2] if case["interleaved"] else x[..., rot // 2:rot]
    u, v = a * cos - b * sin, b * cos + a * sin
    if case["interleaved"]:
        y[..., 0:rot:2], y[..., 1:rot:2] = u, v
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = u, v
    return dict(y=y.reshape(t, heads * d).to(s["x"].dtype))


def _touched(case, s):
    """Per sequence the pages that its new rows fall in (a page given twice
    stands for one that is not there), and each slot's position."""
    page = case["page"]
    lens, rows = _lengths(case)
    most = max((n - 1) // page - (n - m) // page + 1 if m else 1 for n, m in zip(lens, rows))
    ln = s["lens"].long()
    first = ln - (s["starts"][1:] - s["starts"][:-1]).long()
    at = (first // page)[:, None] + torch.arange(most, device=DEV)
    at = torch.minimum(at, ((ln - 1) // page)[:, None])
    ids = torch.gather(s["table"].long(), 1, at)
    return ids, at[..., None] * page + torch.arange(page, device=DEV), first, ln


def _plain_write(case, x, starts, ids, pos, first, length, codes, scale):
    """Codes [pages, hkv, page, d] of a cache and their scales, updated in place."""
    hkv, d = case["hkv"], case["d"]
    new = (pos >= first[:, None, None]) & (pos < length[:, None, None])
    old = pos < first[:, None, None]
    row = (starts[:-1].long()[:, None, None] + pos - first[:, None, None]).clamp(0, x.shape[0] - 1)
    v = x.float().reshape(-1, hkv, d)[row].transpose(2, 3)           # [b, pages, hkv, page, d]
    v = torch.where(new[:, :, None, :, None], v, torch.zeros_like(v))
    before = scale[ids]
    held = torch.where(old.any(dim=2)[..., None], before, torch.zeros_like(before))
    s = torch.maximum(held, v.abs().amax(dim=(3, 4)) * (1.0 / 127.0)).clamp_min(TINY)
    was = codes[ids].float()
    ratio = (held / s)[..., None, None]
    got = torch.where(new[:, :, None, :, None], torch.round(v * (1.0 / s)[..., None, None]),
                      torch.where(old[:, :, None, :, None], torch.round(was * ratio), was))
    any_new = new.any(dim=2)[..., None]
    codes[ids] = torch.where(any_new[..., None, None], got, was).clamp(-127, 127).to(torch.int8)
    scale[ids] = torch.where(any_new, s, before)


def _plain_cache(s):
    case, dt = s["case"], s["k"].dtype
    ids, pos, first, length = _touched(case, s)
    if s["k"].shape[0]:
        _plain_write(case, s["k"], s["starts"], ids, pos, first, length, s["kc"], s["ks"])
        _plain_write(case, s["v"], s["starts"], ids, pos, first, length, s["vc"].transpose(2, 3), s["vs"])
    n = s["out"]["k"].shape[0]
    at = torch.arange(n, device=DEV)
    b = torch.searchsorted(s["all"][1:].long(), at, right=True)
    p = at - s["all"].long()[b]
    page, slot = s["table"][b, p // case["page"]].long(), p % case["page"]
    k = s["kc"][page, :, slot].float() * s["ks"][page][..., None]
    v = s["vc"][page, :, :, slot].float() * s["vs"][page][..., None]
    return dict(k=k.reshape(n, -1).to(dt), v=v.reshape(n, -1).to(dt), k_scale=s["ks"], v_scale=s["vs"])


def _plain_attn(s):
    case = s["case"]
    b, hq, hkv, d = case["b"], case["hq"], case["hkv"], case["d"]
    lens, rows = _lengths(case)
    most, t = max(rows), s["q"].shape[0]
    length, first_row = s["lens"].long(), s["starts"][:-1].long()
    n = (s["starts"][1:] - s["starts"][:-1]).long()
    i = torch.arange(most, device=DEV)
    row = (first_row[:, None] + i).clamp_max(t - 1)                   # [b, most]
    q = s["q"].float().reshape(t, hkv, hq // hkv, d)[row]              # [b, most, hkv, g, d]
    q = (q * (1.0 / math.sqrt(d))).permute(0, 2, 3, 1, 4).reshape(b * hkv, hq // hkv * most, d)
    ids = s["table"].long()
    keys = ids.shape[1] * case["page"]
    k = s["kc"][ids].float() * s["ks"][ids][..., None, None]           # [b, pages, hkv, page, d]
    k = k.permute(0, 2, 4, 1, 3).reshape(b * hkv, d, keys)
    v = s["vc"][ids].float() * s["vs"][ids][..., None, None]           # [b, pages, hkv, d, page]
    v = v.permute(0, 2, 1, 4, 3).reshape(b * hkv, keys, d)
    at = (length - n)[:, None, None] + i[None, :, None]                # a query's position
    j = torch.arange(keys, device=DEV)
    seen = (j <= at) & (j < length[:, None, None])
    if case["window"]:
        seen &= (at - j < case["window"]) | (j < case["sinks"])
    x = torch.matmul(q, k).reshape(b, hkv, hq // hkv, most, keys)
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(dim=-1, keepdim=True).clamp_min(-1e30)
    x = x.sub_(top).exp_()
    total = x.sum(dim=-1, keepdim=True).reshape(b * hkv, -1, 1).clamp_min(1e-38)
    o = torch.matmul(x.reshape(b * hkv, -1, keys), v) / total
    o = o.reshape(b, hkv, hq // hkv, most, d).permute(0, 3, 1, 2, 4).reshape(b * most, hq * d)
    # the padded rows are left out
    seq = torch.searchsorted(s["starts"][1:].long(), torch.arange(t, device=DEV), right=True)
    return dict(o=o[seq * most + torch.arange(t, device=DEV) - first_row[seq]].to(s["q"].dtype))


_PLAIN = dict(norm=_plain_norm, rotary=_plain_rotary, cache=_plain_cache, attn=_plain_attn)


# --- what a call cannot do without, and what it should give -------------------

def _seen(case):
    """(query, key) pairs that the masks leave, and the keys that some query of a sequence sees."""
    lens, rows = _lengths(case)
    w, sinks, pairs, keys = case["window"], case["sinks"], 0, 0
    for length, n in zip(lens, rows):
        lo = length - n
        if not n:
            continue
        if not w:
            pairs += n * lo + n * (n + 1) // 2
            keys += length
            continue
        for p in range(lo, length):
            pairs += min(p + 1, w) + min(sinks, max(0, p + 1 - w))
        begin = max(0, lo - w + 1)
        keys += length - begin + min(sinks, begin)
    return pairs, keys


def work(case):
    kind, e = case["kind"], 2 if case["dtype"] == "f16" else 4
    if kind == "norm":
        rows, c = case["rows"], case["c"]
        n = rows * c * e * (4 if case["residual"] else 2) + c * e
        return {"bytes": n + (4 * rows if case["out"] == "s8" else 0), "flops": 8.0 * rows * c}
    if kind == "rotary":
        n = case["t"] * case["heads"]
        return {"bytes": 2 * n * case["d"] * e + case["t"] * (4 + 4 * case["rot"]), "flops": 3.0 * n * case["rot"]}
    lens, rows = _lengths(case)
    hkv, d, page = case["hkv"], case["d"], case["page"]
    if kind == "cache":
        n, t = sum(lens), sum(rows)
        scales = 8 * hkv * sum(-(-x // page) for x in lens)
        # new rows in, their codes out; codes in, values out
        return {"bytes": 2 * hkv * d * (t * (e + 1) + n * (1 + e)) + 2 * scales, "flops": 2.0 * hkv * d * (2 * t + n)}
    pairs, keys = _seen(case)
    t = sum(rows)
    return {"bytes": 2 * hkv * d * keys + 8 * hkv * (keys // page + case["b"]) + 2 * t * case["hq"] * d * e,
            "flops": 4.0 * pairs * case["hq"] * d}


def exact(case, seed):
    s, kind, f64 = _inputs(case, seed), case["kind"], torch.float64
    if kind == "norm":
        h = s["x"].to(f64) + (s["r"].to(f64) if case["residual"] else 0.0)
        y = h / torch.sqrt((h ** 2).sum(1, keepdim=True) / case["c"] + EPS) * s["w"].to(f64)
        if case["out"] == "s8":
            step = y.abs().max(dim=1, keepdim=True).values / 127
            y = torch.where(step > 0, torch.round(y / step) * step, torch.zeros_like(y))
        return dict(y=y, sum=h) if case["residual"] else dict(y=y)
    if kind == "rotary":
        t, heads, d, half = case["t"], case["heads"], case["d"], case["rot"] // 2
        y = s["x"].to(f64).reshape(t, heads, d).clone()
        angle = s["pos"].to(f64)[:, None] * 10000.0 ** (-torch.arange(half, device=DEV, dtype=f64) / half)
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        if case["interleaved"]:
            z = torch.view_as_complex(y[..., :2 * half].reshape(t, heads, half, 2)) * turn
            y[..., :2 * half] = torch.view_as_real(z).reshape(t, heads, 2 * half)
        else:
            z = torch.complex(y[..., :half], y[..., half:2 * half]) * turn
            y[..., :half], y[..., half:2 * half] = z.real, z.imag
        return dict(y=y.reshape(t, heads * d))
    lens, rows = _lengths(case)
    page, hkv, d = case["page"], case["hkv"], case["d"]
    table = s["table"].tolist()
    start = [sum(rows[:i]) for i in range(len(rows))]
    if kind == "cache":
        back = []
        scales = []
        for x, codes, scale in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"].transpose(2, 3), s["vs"])):
            x = x.to(f64).reshape(-1, hkv, d)
            value = codes.to(f64) * scale.to(f64)[..., None, None]       # [pages, hkv, page, d]
            scale = scale.to(f64).clone()
            for i, (length, n) in enumerate(zip(lens, rows)):
                p = length - n
                while p < length:
                    pid, a, z = table[i][p // page], p % page, min(page, p % page + length - p)
                    xs = x[start[i] + p - (length - n):][:z - a].transpose(0, 1)     # [hkv, tokens, d]
                    step = (xs.abs().amax(dim=(1, 2)) / 127).clamp_min(TINY)
                    grown = torch.maximum(step, scale[pid]) if a else step
                    if a:
                        q = torch.round(codes[pid, :, :a].to(f64) * (scale[pid] / grown)[:, None, None])
                        value[pid, :, :a] = q * grown[:, None, None]
                    value[pid, :, a:z] = torch.round(xs / grown[:, None, None]) * grown[:, None, None]
                    scale[pid] = grown
                    p += z - a
            flat = [value[table[i][:-(-n // page)]].transpose(1, 2).reshape(-1, hkv * d)[:n] for i, n in enumerate(lens)]
            back.append(torch.cat(flat))
            scales.append(scale)
        return dict(k=back[0], v=back[1], k_scale=scales[0], v_scale=scales[1])
    g, out = case["hq"] // hkv, torch.zeros(s["q"].shape, dtype=f64, device=DEV)
    for i, (length, n) in enumerate(zip(lens, rows)):
        if not n:
            continue
        ids = table[i][:-(-length // page)]
        at = torch.arange(length - n, length, device=DEV)[:, None]
        j = torch.arange(length, device=DEV)
        hide = j > at
        if case["window"]:
            hide = hide | ((j <= at - case["window"]) & (j >= case["sinks"]))
        for h in range(hkv):
            k = (s["kc"][ids, h].to(f64) * s["ks"][ids, h].to(f64)[:, None, None]).reshape(-1, d)[:length]
            v = (s["vc"][ids, h].to(f64) * s["vs"][ids, h].to(f64)[:, None, None]).transpose(1, 2).reshape(-1, d)[:length]
            for m in range(h * g, h * g + g):
                q = s["q"][start[i]:start[i] + n, m * d:(m + 1) * d].to(f64)
                x = (q @ k.t().contiguous() / math.sqrt(d)).masked_fill(hide, -math.inf)
                out[start[i]:start[i] + n, m * d:(m + 1) * d] = torch.softmax(x, dim=-1) @ v
    return dict(o=out)
