"""Cases for the paged-cache operators of a serving step: the append that rotates queries and keys
on the way (`paged_append_rope`), attention of any number of query tokens per sequence over the
paged cache (`paged_attention`), and single-token attention for requests that share a long prefix
(`paged_shared_prefix_attention`).

`own` selects between the plain torch form of each operator (fp32, rounded once) and the calls a
program makes of `llmik_cuda`. Heads have 128 channels, caches are fp16 or INT8 with one fp16 scale
per token, as everywhere in the package.
"""
import math
import os
import random
import sys

import torch

own = False

D = 128
_lib = None


def _own():
    global _lib
    if _lib is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "llm-inference-kernels_b200"))
        import llmik_cuda
        _lib = llmik_cuda
    return _lib


# ---------------------------------------------------------------------- cases

def _append(name, tokens, heads, kv_heads, block, kv, sections, rot, interleaved, padding):
    return dict(name=name, op="append", tokens=tokens, heads=heads, kv_heads=kv_heads, block=block, kv=kv,
                sections=sections, rot=rot, interleaved=interleaved, padding=padding)


def _attend(name, kv, heads, kv_heads, seqs, q_lo, q_hi, ctx_lo, ctx_hi, block, causal=True, softcap=0.0, window=0,
            alibi=False, prefix=0, docs=0, salt=1):
    return dict(name=name, op="attention", kv=kv, heads=heads, kv_heads=kv_heads, seqs=seqs, q_lo=q_lo, q_hi=q_hi,
                ctx_lo=ctx_lo, ctx_hi=ctx_hi, block=block, causal=causal, softcap=softcap, window=window, alibi=alibi,
                prefix=prefix, docs=docs, salt=salt)


def _shared(name, kv, heads, kv_heads, seqs, groups, prefix, own_lo, own_hi, block, softcap=0.0, alibi=False, salt=1):
    return dict(name=name, op="shared", kv=kv, heads=heads, kv_heads=kv_heads, seqs=seqs, groups=groups, prefix=prefix,
                own_lo=own_lo, own_hi=own_hi, block=block, softcap=softcap, alibi=alibi, salt=salt)


def listed():
    return [
        # one new token of each of 8 requests, the append of a decode step: latency alone
        _append("append, 8 tokens", 8, 32, 8, 16, "fp16", "", 128, False, 0),
        # a prompt with images: time, height and width positions, a section of frequencies each
        _append("append, 8192 tokens, 3 axes", 8192, 32, 8, 64, "fp16", "16,24,24", 128, False, 0),
        # a padded batch of prompt chunks into an INT8 cache, half of each head rotated in
        # neighbouring pairs; the fp16 view of the cache that a prompt step reads comes with it
        _append("append, 2047 tokens, INT8", 2047, 32, 8, 32, "int8", "", 64, True, 37),
        # the decode step of 8 requests of 4096 positions for a model that caps its scores
        _attend("decode, 8 x 4096, capped", "fp16", 32, 8, 8, 1, 1, 4096, 4096, 16, softcap=50.0),
        # 64 requests of different ages, distance bias, INT8 cache
        _attend("decode, 64 ragged, bias, INT8", "int8", 32, 8, 64, 1, 1, 300, 8192, 32, alibi=True, salt=2),
        # one long prompt
        _attend("prompt of 8192", "fp16", 32, 8, 1, 8192, 8192, 8192, 8192, 64),
        # chunks of prompts behind what is cached already, among them single tokens; sliding
        # window and capped scores; INT8 cache
        _attend("chunks, window, capped, INT8", "int8", 32, 8, 7, 1, 1500, 40, 6000, 16, softcap=30.0, window=1024,
                salt=3),
        # packed documents behind a common preamble that every token sees, one query head per KV head
        _attend("documents, prefix", "fp16", 16, 16, 3, 900, 4001, 900, 4001, 128, prefix=300, docs=700, salt=4),
        # 16 requests with the same system prompt, just started
        _shared("16 share 2048", "fp16", 32, 8, 16, 1, 2048, 1, 130, 16),
        # 64 requests on one long document
        _shared("64 share 32768", "fp16", 32, 8, 64, 1, 32768, 1, 1024, 64, salt=2),
        # three documents, 100 requests on them in unequal parts, larger groups of heads, INT8
        _shared("100 on 3 documents, INT8", "int8", 64, 8, 100, 3, 8000, 20, 700, 32, softcap=50.0, salt=3),
    ]


def _span(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "shared"])
    kv = rng.choice(["fp16", "int8"])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    heads = kv_heads * group
    block = rng.choice([16, 32, 48, 64, 128, 256])
    salt = rng.randrange(1 << 20)
    if op == "append":
        kv_heads, heads = min(kv_heads, 8), min(heads, 32) // min(kv_heads, 8) * min(kv_heads, 8)
        rot = 2 * rng.choice([64, 64, 32, 48, 11])
        sections = ""
        if rng.random() < 0.4:
            a = rng.randrange(1, rot // 2 - 1)
            b = rng.randrange(1, rot // 2 - a)
            sections = "%d,%d,%d" % (a, b, rot // 2 - a - b) if rng.random() < 0.7 else "%d,%d" % (a, rot // 2 - a)
        tokens = _span(rng, 1, 8000)
        case = _append("", tokens, heads, kv_heads, block, kv, sections, rot, rng.random() < 0.4,
                       rng.randrange(0, max(1, tokens // 8)))
    elif op == "attention":
        q_hi = 1 if rng.random() < 0.3 else _span(rng, 2, 4000)
        q_lo = max(1, _span(rng, 1, q_hi))
        ctx_hi = max(q_hi, _span(rng, 1, 8192))
        ctx_lo = _span(rng, 1, ctx_hi)
        # the plain form holds scores of [seqs, heads, q_hi, ctx_hi]: below the largest listed case's
        most = int(min(1 << 30, 32 * 8192 * 8192) // (heads * q_hi * ctx_hi))
        most = max(1, min(most, 64, (64 * 8192 * 8) // (ctx_hi * kv_heads)))
        heads_ok = heads if heads * q_hi * ctx_hi <= 32 * 8192 * 4096 else kv_heads
        case = _attend("", kv, heads_ok, kv_heads, _span(rng, 1, most), q_lo, q_hi, ctx_lo, ctx_hi, block,
                       causal=rng.random() < 0.8, softcap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                       window=rng.choice([0, 0, _span(rng, 16, 4096)]), alibi=rng.random() < 0.3,
                       prefix=rng.choice([0, 0, _span(rng, 1, 1000)]),
                       docs=rng.choice([0, 0, _span(rng, 50, 2000)]), salt=salt)
    else:
        kv_heads = min(kv_heads, 8)
        heads = kv_heads * group
        seqs = _span(rng, 1, 64)
        groups = min(seqs, rng.choice([1, 1, 2, 5]))
        case = _shared("", kv, heads, kv_heads, seqs, groups, _span(rng, 1, 8192), rng.randrange(0, 20),
                       20 + _span(rng, 1, 1000), block, softcap=rng.choice([0.0, 30.0]), alibi=rng.random() < 0.3,
                       salt=salt)
    del case["name"]
    return case


def _lengths(rng, n, lo, hi):
    """n lengths between lo and hi, spread over their logarithm, the last one hi."""
    return [max(lo, min(hi, _span(rng, max(lo, 1), max(hi, 1)))) if hi > lo > 0 else rng.randint(lo, hi)
            for _ in range(n - 1)] + [hi]


def _shape(case):
    """The lengths of a case's sequences: they belong to the case, not to the seed."""
    rng = random.Random(case["salt"])
    if case["op"] == "attention":
        nq = _lengths(rng, case["seqs"], case["q_lo"], case["q_hi"])
        ctx = [max(a, b) for a, b in zip(nq, _lengths(rng, case["seqs"], case["ctx_lo"], case["ctx_hi"]))]
        pre = [min(c, rng.randint(0, 2 * case["prefix"])) for c in ctx]
        return nq, ctx, pre
    suffix = _lengths(rng, case["seqs"], case["own_lo"], case["own_hi"])
    cuts = sorted(rng.sample(range(1, case["seqs"]), case["groups"] - 1))
    sizes = [b - a for a, b in zip([0] + cuts, cuts + [case["seqs"]])]
    prefix = [case["prefix"]] + [rng.randint(1, case["prefix"]) for _ in range(case["groups"] - 1)]
    return sizes, prefix, suffix


def _doc_starts(case, n, ctx):
    """The first key that each of a sequence's last n positions sees: its document's start."""
    rng = random.Random(case["salt"] + ctx)
    starts, at = [], 0
    while at < ctx:
        size = max(1, int(case["docs"] * (0.5 + rng.random())))
        starts += [at] * min(size, ctx - at)
        at += size
    return starts[ctx - n:]


# --------------------------------------------------------------------- inputs

def _pages(case, lens, extra, g):
    """Block tables over a scrambled pool for sequences of the given lengths."""
    bs = case["block"]
    need = [-(-n // bs) for n in lens]
    pool = torch.randperm(sum(need) + extra, device="cuda", generator=g).to(torch.int32)
    width = max(1, max(need))
    at = torch.tensor([0] + need, device="cuda").cumsum(0)[:-1]
    col = torch.arange(width, device="cuda")
    idx = at[:, None] + col
    live = col < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(live, pool[idx.clamp(max=len(pool) - 1)], torch.zeros_like(idx, dtype=torch.int32))
    return table.to(torch.int32).contiguous(), sum(need) + extra


def _cache(case, blocks, g):
    """A K (or V) cache of random contents and its per-token scales."""
    shape = (blocks, case["kv_heads"], case["block"], D)
    if case["kv"] == "fp16":
        return torch.randn(shape, device="cuda", generator=g, dtype=torch.float16), None
    codes = torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int8)
    scale = (torch.rand(shape[:3], device="cuda", generator=g) * 0.5 + 0.75) * (1.7 / 127)
    return codes, scale.half()


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _offsets(sizes):
    return _int32([0] + torch.tensor(sizes).cumsum(0).tolist())


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h, hk = case["heads"], case["kv_heads"]
    st = dict(case=case, scale=1 / math.sqrt(D))
    if case["op"] == "append":
        n, bs, rot = case["tokens"], case["block"], case["rot"]
        # one fused projection, as a model leaves it; q, k and v are views of it
        qkv = torch.randn(n, h + 2 * hk, D, device="cuda", generator=g, dtype=torch.float16)
        st["q"], st["k"], st["v"] = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
        sec = [int(x) for x in case["sections"].split(",")] if case["sections"] else None
        st["sections"] = sec
        axes = len(sec) if sec else 1
        pos = torch.randint(0, 120000, (axes, n), device="cuda", generator=g)
        st["positions"] = pos if sec else pos[0]
        st["inv_freq"] = (10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)).float()
        axis = [a for a, m in enumerate(sec or [rot // 2]) for _ in range(m)]
        st["axis"] = torch.tensor(axis, device="cuda")
        blocks = -(-(n + 1) // bs)
        slots = torch.randperm(blocks * bs, device="cuda", generator=g)[:n + 1]
        st["guard"] = slots[n:]                                     # a row that no token is written to
        slots = slots[:n].clone()
        if case["padding"]:
            slots[n - case["padding"]:] = -1
        st["slots"] = slots
        dt = torch.float16 if case["kv"] == "fp16" else torch.int8
        for x in "kv":
            st[x + "_cache"] = torch.zeros(blocks, hk, bs, D, dtype=dt, device="cuda")
            st[x + "_scale"] = None if case["kv"] == "fp16" else torch.ones(blocks, hk, bs, dtype=torch.float16,
                                                                          device="cuda")
        return st
    slopes = 2.0 ** (-8.0 * torch.arange(1, h + 1, device="cuda", dtype=torch.float32) / h)
    st["slopes"] = slopes if case["alibi"] else None
    # capped scores are capped because they grow: a wider spread of scores there
    spread = 4.0 if case["softcap"] else 1.0
    if case["op"] == "attention":
        nq, ctx, pre = _shape(case)
        st["tables"], blocks = _pages(case, ctx, 2, g)
        st["ctx"], st["cu"] = _int32(ctx), _offsets(nq)
        st["max_q"], st["max_ctx"] = max(nq), max(ctx)
        st["pre"] = _int32(pre) if case["prefix"] else None
        st["first"] = None
        if case["docs"]:
            st["first"] = _int32([f for n, c in zip(nq, ctx) for f in _doc_starts(case, n, c)])
        rows = sum(nq)
    else:
        sizes, prefix, suffix = _shape(case)
        tables, blocks = _pages(case, prefix + suffix, 2, g)
        st["prefix_tables"] = tables[:len(prefix), :-(-max(prefix) // case["block"])].contiguous()
        st["tables"] = tables[len(prefix):, :max(1, -(-max(suffix) // case["block"]))].contiguous()
        st["prefix"], st["ctx"], st["cu"] = _int32(prefix), _int32(suffix), _offsets(sizes)
        st["max_prefix"], st["max_ctx"], st["max_q"] = max(prefix), max(suffix), max(sizes)
        rows = case["seqs"]
    st["q"] = (torch.randn(rows, h, D, device="cuda", generator=g) * spread).half()
    st["k_cache"], st["k_scale"] = _cache(case, blocks, g)
    st["v_cache"], st["v_scale"] = _cache(case, blocks, g)
    return st


# ---------------------------------------------------------------- plain forms

def _rows(cache, scale, tables, length):
    """fp32 rows [seqs, length, kv_heads, D] of the first `length` positions that the tables name."""
    bs = cache.shape[2]
    pos = torch.arange(length, device=cache.device)
    blk = tables.long()[:, (pos // bs).clamp(max=tables.shape[1] - 1)]
    x = cache[blk, :, pos % bs].float()
    return x if scale is None else x * scale[blk, :, pos % bs].float()[..., None]


def _scores(case, q, k, scale, q_pos, k_pos, slopes):
    """fp32 scores [seqs, kv_heads, group, queries, keys]."""
    b, n = q.shape[:2]
    q = q.view(b, n, case["kv_heads"], -1, D).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q, k.permute(0, 2, 3, 1)[:, :, None]) * scale
    if case["softcap"]:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    if slopes is not None:
        far = (q_pos[..., None] - k_pos).abs().float()
        s = s - slopes.view(1, case["kv_heads"], -1, 1, 1) * far[:, None, None]
    return s


def _plain_attention(st):
    case, q = st["case"], st["q"]
    cu, ctx = st["cu"].long(), st["ctx"].long()
    nq = cu[1:] - cu[:-1]
    i = torch.arange(st["max_q"], device=q.device)
    row = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)
    k = _rows(st["k_cache"], st["k_scale"], st["tables"], st["max_ctx"])
    v = _rows(st["v_cache"], st["v_scale"], st["tables"], st["max_ctx"])
    j = torch.arange(st["max_ctx"], device=q.device)
    p = (ctx - nq)[:, None] + i                                            # a query's position
    seen = j <= (p if case["causal"] else torch.full_like(p, st["max_ctx"]))[..., None]
    if case["window"]:
        seen = seen & (j > (p - case["window"])[..., None])
    if st["pre"] is not None:
        seen = seen | (j < st["pre"].long()[:, None, None])
    if st["first"] is not None:
        seen = seen & (j >= st["first"].long()[row][..., None])
    seen = (seen & (j < ctx[:, None, None]))[:, None, None]
    s = _scores(case, q[row].float(), k, st["scale"], p, j, st["slopes"])
    s = s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = s.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    o = torch.matmul(e, v.permute(0, 2, 1, 3)[:, :, None])
    o = o / e.sum(-1, keepdim=True).clamp(min=1e-37)
    o = o.permute(0, 3, 1, 2, 4).reshape(len(nq), st["max_q"], -1, D)
    t = torch.arange(q.shape[0], device=q.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    return o[b, t - cu[b]].half()


def _plain_shared(st):
    case, q = st["case"], st["q"]
    cu, prefix, ctx = st["cu"].long(), st["prefix"].long(), st["ctx"].long()
    t = torch.arange(q.shape[0], device=q.device)
    grp = torch.searchsorted(cu, t, right=True) - 1
    i = t - cu[grp]
    row = (cu[:-1, None] + torch.arange(st["max_q"], device=q.device)).clamp(max=q.shape[0] - 1)
    pos = prefix[grp] + ctx - 1
    kp = _rows(st["k_cache"], st["k_scale"], st["prefix_tables"], st["max_prefix"])
    vp = _rows(st["v_cache"], st["v_scale"], st["prefix_tables"], st["max_prefix"])
    ks = _rows(st["k_cache"], st["k_scale"], st["tables"], st["max_ctx"])
    vs = _rows(st["v_cache"], st["v_scale"], st["tables"], st["max_ctx"])
    jp = torch.arange(st["max_prefix"], device=q.device)
    js = torch.arange(st["max_ctx"], device=q.device)
    # [groups, kv_heads, group, queries, prefix] -> one row per request
    sp = _scores(case, q[row].float(), kp, st["scale"], pos[row], jp, st["slopes"])
    sp = sp.masked_fill_(~(jp < prefix[:, None])[:, None, None, None], -math.inf)
    ss = _scores(case, q[:, None].float(), ks, st["scale"], (ctx - 1)[:, None], js, st["slopes"])
    ss = ss.masked_fill_(~(js < ctx[:, None])[:, None, None, None], -math.inf)[:, :, :, 0]
    top = torch.maximum(sp.amax(-1)[grp, :, :, i], ss.amax(-1))
    top_of_row = top[row].permute(0, 2, 3, 1)                               # [groups, kv_heads, group, queries]
    ep = sp.sub_(top_of_row[..., None]).exp_()
    es = ss.sub_(top[..., None]).exp_()
    op = torch.matmul(ep, vp.permute(0, 2, 1, 3)[:, :, None])[grp, :, :, i]
    own_part = torch.matmul(es, vs.permute(0, 2, 1, 3))
    total = ep.sum(-1)[grp, :, :, i] + es.sum(-1)
    return ((op + own_part) / total[..., None]).reshape(q.shape).half()


def _plain_rotate(st, x):
    case, r = st["case"], st["case"]["rot"] // 2
    pos = st["positions"] if st["sections"] else st["positions"][None]
    angle = pos[st["axis"]].double().T * st["inv_freq"].double()             # [tokens, rot / 2]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = x.float()
    y = x.clone()
    if case["interleaved"]:
        a, b = x[..., 0:2 * r:2], x[..., 1:2 * r:2]
        y[..., 0:2 * r:2], y[..., 1:2 * r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :r], x[..., r:2 * r]
        y[..., :r], y[..., r:2 * r] = a * cos - b * sin, b * cos + a * sin
    return y.half()


def _plain_store(st, which, x):
    """Writes x [tokens, kv_heads, D] into its slots; tokens without one change nothing."""
    cache, scale, slots = st[which + "_cache"], st[which + "_scale"], st["slots"]
    bs = cache.shape[2]
    keep = slots >= 0
    at = torch.where(keep, slots, st["guard"])
    blk, off = at // bs, at % bs
    if scale is not None:
        f = x.float()
        sc = (f.abs().amax(-1) / 127).clamp(min=1e-8)
        x = (f / sc[..., None]).round().clamp(-127, 127).to(torch.int8)
        scale[blk, :, off] = torch.where(keep[:, None], sc.half(), scale[blk, :, off])
    cache[blk, :, off] = torch.where(keep[:, None, None], x, cache[blk, :, off])


def _plain_append(st):
    q = _plain_rotate(st, st["q"])
    _plain_store(st, "k", _plain_rotate(st, st["k"]))
    _plain_store(st, "v", st["v"])
    if st["k_scale"] is None:
        return q, st["k_cache"], st["v_cache"]
    return (q, (st["k_cache"].float() * st["k_scale"].float()[..., None]).half(),
            (st["v_cache"].float() * st["v_scale"].float()[..., None]).half())


# ------------------------------------------------------------------------ run

def run(st):
    op = st["case"]["op"]
    if not own:
        return {"append": _plain_append, "attention": _plain_attention, "shared": _plain_shared}[op](st)
    L = _own()
    case = st["case"]
    if op == "append":
        q = L.paged_append_rope(st["q"], st["k"], st["v"], st["positions"], st["inv_freq"], st["slots"],
                                st["k_cache"], st["v_cache"], k_scale=st["k_scale"], v_scale=st["v_scale"],
                                sections=st["sections"], interleaved=case["interleaved"])
        if st["k_scale"] is None:
            return q, st["k_cache"], st["v_cache"]
        return (q,) + tuple(L.dequantize_int8(st["k_cache"], st["k_scale"], st["v_cache"], st["v_scale"]))
    if op == "attention":
        return L.paged_attention(st["q"], st["k_cache"], st["v_cache"], st["tables"], st["ctx"], st["cu"],
                                 st["scale"], k_scale=st["k_scale"], v_scale=st["v_scale"], causal=case["causal"],
                                 window=case["window"], softcap=case["softcap"], alibi_slopes=st["slopes"],
                                 prefix_lens=st["pre"], first_keys=st["first"])
    return L.paged_shared_prefix_attention(st["q"], st["k_cache"], st["v_cache"], st["prefix_tables"], st["prefix"],
                                           st["cu"], st["tables"], st["ctx"], st["scale"], k_scale=st["k_scale"],
                                           v_scale=st["v_scale"], softcap=case["softcap"], alibi_slopes=st["slopes"])


# ----------------------------------------------------------------------- work

def _seen(case, n, ctx, pre, first):
    """How many keys each of a sequence's n queries sees, and how many keys any of them sees."""
    p = torch.arange(ctx - n, ctx)
    hi = p if case["causal"] else torch.full_like(p, ctx - 1)
    lo = (p - case["window"] + 1).clamp(min=0) if case["window"] else torch.zeros_like(p)
    lo = torch.maximum(lo, first)
    main = (hi - lo + 1).clamp(min=0)
    far = (torch.minimum(torch.full_like(p, pre), lo) - first).clamp(min=0) if pre else torch.zeros_like(p)
    ahead = (pre - torch.maximum(torch.maximum(hi + 1, first), lo)).clamp(min=0) if pre else torch.zeros_like(p)
    top = max(int(hi.max()) + 1, pre)
    return int((main + far + ahead).sum()), max(0, min(ctx, top) - (0 if pre else int(lo.min())))


def work(case):
    h, hk = case["heads"], case["kv_heads"]
    row = 2 * D * 2 if case["kv"] == "fp16" else 2 * (D + 2)                 # K and V of one position and head
    if case["op"] == "append":
        n = case["tokens"]
        axes = len(case["sections"].split(",")) if case["sections"] else 1
        moved = n * (2 * h + 2 * hk) * D * 2 + (n - case["padding"]) * hk * row + n * 8 * (1 + axes)
        if case["kv"] != "fp16":                                             # the fp16 view of all rows
            slots = -(-(n + 1) // case["block"]) * case["block"]
            moved += slots * hk * (row + 2 * D * 2)
        return {"bytes": moved, "flops": n * (h + hk) * case["rot"] * 3}
    if case["op"] == "attention":
        nq, ctx, pre = _shape(case)
        pairs = keys = 0
        for n, c, f in zip(nq, ctx, pre):
            first = torch.tensor(_doc_starts(case, n, c)) if case["docs"] else torch.zeros(n, dtype=torch.int64)
            a, b = _seen(case, n, c, f if case["prefix"] else 0, first)
            pairs, keys = pairs + a, keys + b
        return {"bytes": sum(nq) * h * D * 4 + keys * hk * row, "flops": 4 * D * h * pairs}
    sizes, prefix, suffix = _shape(case)
    pairs = sum(a * b for a, b in zip(sizes, prefix)) + sum(suffix)
    return {"bytes": case["seqs"] * h * D * 4 + (sum(prefix) + sum(suffix)) * hk * row, "flops": 4 * D * h * pairs}


# ---------------------------------------------------------------------- exact

def _exact_rows(cache, scale, blocks, length):
    """One sequence's rows [kv_heads, length, D] in 64 bits."""
    n = -(-length // cache.shape[2]) if length else 0
    x = cache[blocks[:n].long()].double()
    if scale is not None:
        x = x * scale[blocks[:n].long()].double().unsqueeze(-1)
    return x.transpose(0, 1).reshape(cache.shape[1], -1, D)[:, :length]


def _exact_head(case, q, k, v, scale, dist, hidden, slope):
    """softmax(scores) v of one query head, q [n, D], k and v [m, D]; rows that see nothing are zero."""
    s = (q @ k.T) * scale
    if case["softcap"]:
        s = torch.tanh(s / case["softcap"]) * case["softcap"]
    if slope is not None:
        s = s - float(slope) * dist.double()
    s = s.masked_fill(hidden, -math.inf)
    w = torch.nan_to_num(torch.softmax(s, dim=-1), nan=0.0)
    return w @ v


def _exact_attention(st):
    case, q = st["case"], st["q"].double()
    out = torch.zeros_like(q)
    group = case["heads"] // case["kv_heads"]
    cu, ctx = st["cu"].tolist(), st["ctx"].tolist()
    pre = st["pre"].tolist() if st["pre"] is not None else [0] * len(ctx)
    for b, c in enumerate(ctx):
        lo, hi = cu[b], cu[b + 1]
        k = _exact_rows(st["k_cache"], st["k_scale"], st["tables"][b], c)
        v = _exact_rows(st["v_cache"], st["v_scale"], st["tables"][b], c)
        for at in range(lo, hi, 2048):                                       # bounded scores
            to = min(hi, at + 2048)
            p = torch.arange(at, to, device=q.device)[:, None] - hi + c
            j = torch.arange(c, device=q.device)[None]
            hidden = torch.zeros(to - at, c, dtype=torch.bool, device=q.device)
            if case["causal"]:
                hidden |= j > p
            if case["window"]:
                hidden |= j <= p - case["window"]
            hidden &= j >= pre[b]
            if st["first"] is not None:
                hidden |= j < st["first"][at:to, None]
            for h in range(case["heads"]):
                out[at:to, h] = _exact_head(case, q[at:to, h], k[h // group], v[h // group], st["scale"],
                                            (p - j).abs(), hidden,
                                            None if st["slopes"] is None else st["slopes"][h])
    return out


def _exact_shared(st):
    case, q = st["case"], st["q"].double()
    out = torch.zeros_like(q)
    group = case["heads"] // case["kv_heads"]
    cu, prefix, ctx = st["cu"].tolist(), st["prefix"].tolist(), st["ctx"].tolist()
    for g, m in enumerate(prefix):
        kp = _exact_rows(st["k_cache"], st["k_scale"], st["prefix_tables"][g], m)
        vp = _exact_rows(st["v_cache"], st["v_scale"], st["prefix_tables"][g], m)
        for b in range(cu[g], cu[g + 1]):
            n = m + ctx[b]
            k = torch.cat([kp, _exact_rows(st["k_cache"], st["k_scale"], st["tables"][b], ctx[b])], dim=1)
            v = torch.cat([vp, _exact_rows(st["v_cache"], st["v_scale"], st["tables"][b], ctx[b])], dim=1)
            s = torch.einsum("hgd,hnd->hgn", q[b].view(-1, group, D), k) * st["scale"]
            if case["softcap"]:
                s = torch.tanh(s / case["softcap"]) * case["softcap"]
            if st["slopes"] is not None:
                far = (n - 1) - torch.arange(n, device=q.device, dtype=torch.float64)
                s = s - st["slopes"].double().view(-1, group, 1) * far
            out[b] = torch.einsum("hgn,hnd->hgd", torch.softmax(s, dim=-1), v).reshape(-1, D)
    return out


def _exact_append(st):
    case, r = st["case"], st["case"]["rot"] // 2
    pos = st["positions"].reshape(-1, case["tokens"]).double()
    angle = torch.stack([pos[a] * st["inv_freq"][f].double() for f, a in enumerate(st["axis"].tolist())], dim=-1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def rotate(x):
        x = x.double()
        z = x[..., :2 * r].unflatten(-1, (r, 2) if case["interleaved"] else (2, r))
        z = torch.complex(z[..., 0], z[..., 1]) if case["interleaved"] else torch.complex(z[..., 0, :], z[..., 1, :])
        z = torch.view_as_real(z * turn)
        z = z if case["interleaved"] else z.transpose(-1, -2)
        return torch.cat([z.flatten(-2), x[..., 2 * r:]], dim=-1)

    got, bs = [rotate(st["q"])], case["block"]
    for which, x in (("k", rotate(st["k"])), ("v", st["v"].double())):
        cache = st[which + "_cache"].double()
        if case["kv"] != "fp16":
            x = x.half().double()                                            # a cache row is made of fp16 values
            step = (x.abs().amax(-1, keepdim=True) / 127).clamp(min=1e-8)
            x = torch.round(x / step).clamp(-127, 127) * step.half().double()
        live = (st["slots"] >= 0).nonzero()[:, 0]
        at = st["slots"][live]
        cache[at // bs, :, at % bs] = x[live]
        got.append(cache)
    return tuple(got)


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "shared": _exact_shared}[case["op"]](st)
