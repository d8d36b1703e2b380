"""The paged K/V cache as cases that can be timed and whose outputs can be compared: writing new tokens into pages,
reading sequences back, and attention of new tokens over their sequence's pages.

Packed, ragged batches: sequence b's new tokens are the rows start[b] .. start[b + 1] - 1 of k, v and q, at the positions
ctx[b], ctx[b] + 1, ...; position j of sequence b lies in row j % page of page table[b, j // page]. Pages hold int8 rows
with one fp32 scale per (token, head), or bf16 rows. Kinds:

  append   the new tokens' K and V written into their pages
  read     the first length[b] tokens of every sequence as dense (B, heads, T, D) tensors, zeros behind them
  attn     every new token attends its sequence's cached tokens and the new ones from row_begin on up to itself

The dims are those of the package's decoders: 32 / 8 heads of 128, the hybrid stack's 16 / 4 heads of 256, and the 16 / 4
heads of 64 of the attention tests.
"""
import math

import torch

own = False

DEV = "cuda"
BF = torch.bfloat16


def listed():
    return [
        # a token for each of 64 running sequences: one launch, latency
        dict(name="append_64x1", kind="append", seqs=64, new=1, ctx=48, kv=8, d=128, page=16, int8=True),
        # the chunks of 8 states of different lengths, a prefill step of about 4000 tokens
        dict(name="append_8x900", kind="append", seqs=8, new=900, ctx=150, kv=8, d=128, page=64, int8=True),
        # one short state of 256-wide heads handed to an operator that takes dense tensors
        dict(name="read_1x333", kind="read", seqs=1, ctx=333, kv=4, d=256, page=16, int8=True, out="float32"),
        # eight long states read back in bf16
        dict(name="read_8x4096", kind="read", seqs=8, ctx=4096, kv=8, d=128, page=64, int8=True, out="bfloat16"),
        # one token over one short state: latency
        dict(name="token_1x700", kind="attn", seqs=1, new=1, ctx=700, rows=0, heads=16, kv=4, d=256, page=16, int8=True),
        # a token for each of 64 sequences of different lengths
        dict(name="token_64x4096", kind="attn", seqs=64, new=1, ctx=4096, rows=0, heads=32, kv=8, d=128, page=64, int8=True),
        # a token for each of 8 long states: bound by reading them
        dict(name="token_8x32768", kind="attn", seqs=8, new=1, ctx=32768, rows=0, heads=32, kv=8, d=128, page=128, int8=True),
        # the same with unquantized pages
        dict(name="token_bf16_16x8000", kind="attn", seqs=16, new=1, ctx=8000, rows=0, heads=32, kv=8, d=128, page=64,
             int8=False),
        # a long chunk appended to a long state: bound by the matrix cores
        dict(name="chunk_2048_32768", kind="attn", seqs=1, new=2048, ctx=32768, rows=0, heads=32, kv=8, d=128, page=64,
             int8=True),
        # ragged chunks over ragged states of 256-wide heads
        dict(name="chunk_4x900_256", kind="attn", seqs=4, new=900, ctx=6000, rows=0, heads=16, kv=4, d=256, page=32, int8=True),
        # option rows: 8 requests of 32 options of up to 16 tokens over their own states, an option sees its own tokens only
        dict(name="options_8x512", kind="attn", seqs=8, new=512, ctx=2048, rows=16, heads=32, kv=8, d=128, page=64, int8=True),
        # chunks over unquantized pages, heads of 64
        dict(name="chunk_bf16_3x700", kind="attn", seqs=3, new=700, ctx=3000, rows=0, heads=16, kv=4, d=64, page=16, int8=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _drawn(rng):
    kind = rng.choice(["append", "read", "attn", "attn", "attn"])
    heads, kv, d = rng.choice([(32, 8, 128), (32, 8, 128), (16, 4, 256), (16, 4, 64), (28, 4, 128), (8, 8, 64)])
    c = dict(kind=kind, kv=kv, d=d, page=rng.choice([16, 32, 64, 128]), int8=rng.random() < 0.75)
    if kind == "append":
        return dict(c, seqs=_log(rng, 1, 128), new=_log(rng, 1, 1500), ctx=_log(rng, 1, 300))
    if kind == "read":
        return dict(c, seqs=_log(rng, 1, 32), ctx=_log(rng, 20, 9000), out=rng.choice(["bfloat16", "bfloat16", "float32"]))
    c = dict(c, heads=heads, rows=0)
    form = rng.choice(["token", "tokens", "chunk", "rows"])
    if form == "token":
        return dict(c, seqs=_log(rng, 1, 128), new=1, ctx=_log(rng, 30, 32768))
    if form == "tokens":
        return dict(c, seqs=_log(rng, 1, 32), new=rng.randrange(2, 33), ctx=_log(rng, 30, 16000))
    if form == "chunk":
        return dict(c, seqs=_log(rng, 1, 8), new=_log(rng, 40, 2500), ctx=_log(rng, 1, 20000))
    return dict(c, seqs=_log(rng, 1, 8), new=_log(rng, 40, 1500), ctx=_log(rng, 100, 8000), rows=_log(rng, 1, 40))


def draw(rng):
    most = [max(work(c)[k] for c in listed()) for k in ("bytes", "flops")]
    scores = max(_scores(c) for c in listed())
    while True:
        c = _drawn(rng)
        w = work(c)
        if w["bytes"] <= most[0] and w["flops"] <= most[1] and _scores(c) <= scores:
            return c


def _ragged(n, most, least):
    """n lengths from `least` up to `most`: the first and the longest is `most`, the others spread below it."""
    return [most if i == 0 else max(least, round(most * (0.35 + 0.65 * ((i * 37) % n) / n))) for i in range(n)]


def _lengths(c):
    """(new tokens, cached tokens) of every sequence. A decode step has one new token for each; the last of several
    ragged chunks starts an empty state."""
    n = c["seqs"]
    new = _ragged(n, c["new"], 1) if c.get("new", 1) > 1 else [c.get("new", 0)] * n
    ctx = _ragged(n, c["ctx"], 1)[::-1]
    if n > 1 and c.get("new", 1) > 1:
        ctx[0 if ctx[0] != c["ctx"] else 1] = 0
    return new, ctx


def _own_pairs(n, rows):
    """Pairs (query, key) among n new tokens: causal, in rows of `rows` tokens each (0: one row)."""
    if not rows:
        return n * (n + 1) // 2
    full, rest = divmod(n, rows)
    return full * rows * (rows + 1) // 2 + rest * (rest + 1) // 2


def _scores(c):
    """Scores that the padded plain form holds at once."""
    return c["seqs"] * c["heads"] * c["new"] * (c["ctx"] + c["new"]) if c["kind"] == "attn" else 0


def work(case):
    c = case
    new, ctx = _lengths(c)
    kv, d = c["kv"], c["d"]
    row = kv * (d + 4) if c["int8"] else kv * d * 2  # one token's K or V in the pages
    if c["kind"] == "append":
        return {"bytes": sum(new) * 2 * (kv * d * 2 + row), "flops": sum(new) * 2 * kv * d * 4}
    if c["kind"] == "read":
        size = 4 if c["out"] == "float32" else 2
        return {"bytes": sum(ctx) * 2 * row + c["seqs"] * max(ctx) * 2 * kv * d * size, "flops": sum(ctx) * 2 * kv * d}
    pairs = sum(n * t + _own_pairs(n, c["rows"]) for n, t in zip(new, ctx))
    return {"bytes": sum(ctx) * 2 * row + sum(new) * 2 * (kv + c["heads"]) * d * 2, "flops": 4 * c["heads"] * d * pairs}


def _quantized(x):
    """int8 rows and fp32 scales of x (..., D): scale = max(max |x|, 1e-8) / 127, q = round(x / scale), fp32 quotients (a
    Python number as divisor would be turned into a product with its reciprocal)."""
    xf = x.float()
    s = xf.abs().amax(-1, keepdim=True).clamp_min(1e-8) / xf.new_full((), 127.0)
    return torch.round(xf / s).clamp_(-127, 127).to(torch.int8), s[..., 0]


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    new, ctx = _lengths(c)
    B, kv, d, ps = c["seqs"], c["kv"], c["d"], c["page"]
    per = [-(-(t + n) // ps) for n, t in zip(new, ctx)]
    cols = max(max(per), 1)
    pages = sum(per) + 3  # some of the pool is free
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    held = torch.arange(cols, device=DEV)[None] < torch.tensor(per, device=DEV)[:, None]
    first = torch.tensor([sum(per[:b]) for b in range(B)], device=DEV)[:, None] + torch.arange(cols, device=DEV)[None]
    table = torch.where(held, order[first.clamp_max(pages - 1)], -1).to(torch.int32).contiguous()
    start = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEV)
    N = sum(new)

    def rows(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(BF)

    common = rows(kv, d).float()  # the direction that every query shares with its sequence's first key
    s = dict(c, B=B, N=N, start=start, ctx=torch.tensor(ctx, dtype=torch.int32, device=DEV), table=table, max_new=max(new),
             max_ctx=max(ctx), k=rows(pages, kv, ps, d), v=rows(pages, kv, ps, d) * 0.5, k_scale=None, v_scale=None)
    # a sequence's first token draws much of the attention and has a small value, as in trained models
    sinks = table[:, 0].clamp_min(0).long()
    s["k"][sinks, :, 0] = (1.2 * common).to(BF)
    s["v"][sinks, :, 0] *= 0.05
    if c["int8"]:
        (s["k"], s["k_scale"]), (s["v"], s["v_scale"]) = _quantized(s["k"]), _quantized(s["v"])
    if c["kind"] != "read":
        # the new tokens' projections in one buffer, as a fused projection writes them
        hq = c.get("heads", 0)
        qkv = rows(N, (hq + 2 * kv) * d)
        q, k, v = qkv.split([hq * d, kv * d, kv * d], 1)
        s.update(k_new=k.view(N, kv, d), v_new=v.view(N, kv, d))
        if hq:
            q.view(N, kv, hq // kv, d).add_((0.5 * common[:, None]).to(BF))
            s.update(q=q.view(N, hq, d), scale=d ** -0.5, row_begin=None)
            if c["rows"]:
                local = torch.cat([torch.arange(n, device=DEV) for n in new])
                s["row_begin"] = (local // c["rows"] * c["rows"]).to(torch.int32)
    return s


def _tokens(s):
    """(sequence, index within its new tokens) of every packed row."""
    n = torch.arange(s["N"], device=DEV)
    seq = torch.searchsorted(s["start"].long(), n, right=True) - 1
    return seq, n - s["start"].long()[seq]


def _values(rows, scale):
    return rows.float() if scale is None else rows * scale[..., None]


def _write(pages, scales, x, page, row):
    if scales is None:
        pages[page, :, row] = x
        return
    q, sc = _quantized(x)
    pages[page, :, row] = q
    scales[page, :, row] = sc


def _plain_append(s):
    seq, i = _tokens(s)
    pos = s["ctx"].long()[seq] + i
    page, row = s["table"].long()[seq, pos // s["page"]], pos % s["page"]
    _write(s["k"], s["k_scale"], s["k_new"], page, row)
    _write(s["v"], s["v_scale"], s["v_new"], page, row)


def _cached(s, T):
    """The first T positions of every sequence, (B, T, heads, D) fp32 K and V, zeros where it has none."""
    j = torch.arange(T, device=DEV)
    there = j[None] < s["ctx"][:, None]
    page = s["table"].long()[:, j // s["page"]].clamp_min(0)
    row = (j % s["page"])[None].expand_as(page)

    def side(p, sc):
        y = _values(p[page, :, row], None if sc is None else sc[page, :, row])
        return torch.where(there[:, :, None, None], y, 0.0)

    return side(s["k"], s["k_scale"]), side(s["v"], s["v_scale"]), there


def _plain_read(s):
    k, v, _ = _cached(s, s["max_ctx"])
    to = torch.float32 if s["out"] == "float32" else BF
    return {"k": k.transpose(1, 2).to(to).contiguous(), "v": v.transpose(1, 2).to(to).contiguous()}


def _plain_attn(s):
    B, n, T, hq, kv, d = s["B"], s["max_new"], s["max_ctx"], s["heads"], s["kv"], s["d"]
    rep = hq // kv
    kc, vc, there = _cached(s, T)
    i = torch.arange(n, device=DEV)
    at = (s["start"].long()[:-1, None] + i).clamp_max(s["N"] - 1)  # (B, n) packed rows, repeated past a sequence's end
    real = i[None] < (s["start"][1:] - s["start"][:-1])[:, None]
    k = torch.cat([kc, s["k_new"][at].float()], 1).permute(0, 2, 3, 1).contiguous()  # (B, kv, d, T + n)
    v = torch.cat([vc, s["v_new"][at].float()], 1).transpose(1, 2).contiguous()
    q = s["q"][at].float().view(B, n, kv, rep, d).permute(0, 2, 1, 3, 4).reshape(B, kv, n * rep, d)
    begin = s["row_begin"][at] if s["row_begin"] is not None else torch.zeros(B, n, dtype=torch.int32, device=DEV)
    mine = real[:, None] & (i[None, None] <= i[None, :, None]) & (i[None, None] >= begin[:, :, None])  # (B, query, key)
    seen = torch.cat([there[:, None].expand(B, n, T), mine], 2)[:, None, :, None]
    p = torch.matmul(q, k).view(B, kv, n, rep, T + n).mul_(s["scale"]).masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True).clamp_min(-3e38)
    p = p.sub_(top).exp_()
    o = torch.matmul(p.view(B, kv, n * rep, T + n), v).view(B, kv, n, rep, d)
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3, 4).reshape(B, n, hq, d)
    seq, local = _tokens(s)
    return o[seq, local].to(BF)


def run(state):
    s = state
    if own:
        from opendecider_amd import PagedKVCache, kernels
        cache = PagedKVCache.from_tensors(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if s["kind"] == "append":
            kernels.page_append(s["k_new"], s["v_new"], cache, s["table"], s["start"], s["ctx"])
        elif s["kind"] == "read":
            k, v = kernels.page_read(cache, s["table"], s["ctx"], s["max_ctx"], dtype=getattr(torch, s["out"]))
            return {"k": k, "v": v}
        else:
            return kernels.paged_attn(s["q"], s["k_new"], s["v_new"], cache, s["table"], s["start"], s["ctx"], s["scale"],
                                      row_begin=s["row_begin"], max_new=s["max_new"], max_ctx=s["max_ctx"])
    elif s["kind"] == "append":
        _plain_append(s)
    elif s["kind"] == "read":
        return _plain_read(s)
    else:
        return _plain_attn(s)
    # the pages after the write, as the values that they stand for
    return {"k": s["k"] if s["k_scale"] is None else s["k"] * s["k_scale"][..., None],
            "v": s["v"] if s["v_scale"] is None else s["v"] * s["v_scale"][..., None]}


def exact(case, seed):
    c, s = case, prepare(case, seed)
    new, ctx = _lengths(c)
    ps, table, start = c["page"], s["table"].tolist(), s["start"].tolist()
    k64, v64 = ((p.double() if sc is None else p.double() * sc.double()[..., None])
                for p, sc in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))

    def sequence(pages, b, n):  # the first n tokens of sequence b, (heads, n, D)
        at = table[b][:-(-n // ps)]
        return pages[at].transpose(0, 1).reshape(c["kv"], -1, c["d"])[:, :n] if n else pages.new_zeros(c["kv"], 0, c["d"])

    if c["kind"] == "append":
        for b in range(c["seqs"]):
            for pages, x in ((k64, s["k_new"]), (v64, s["v_new"])):
                x = x[start[b]:start[b + 1]].double()
                if c["int8"]:  # the stored scale and the quotient that is rounded are fp32 numbers by definition
                    scale = (x.abs().amax(-1, keepdim=True).clamp_min(1e-8) / 127).float().double()
                    x = (x / scale).float().double().round().clamp(-127, 127) * scale
                pos = torch.arange(ctx[b], ctx[b] + new[b], device=DEV)
                pages[torch.tensor(table[b], device=DEV)[pos // ps], :, pos % ps] = x
        return {"k": k64, "v": v64}
    if c["kind"] == "read":
        out = {n: torch.zeros(c["seqs"], c["kv"], max(ctx), c["d"], dtype=torch.float64, device=DEV) for n in "kv"}
        for b in range(c["seqs"]):
            out["k"][b, :, :ctx[b]], out["v"][b, :, :ctx[b]] = sequence(k64, b, ctx[b]), sequence(v64, b, ctx[b])
        return out
    out = torch.zeros(s["N"], c["heads"], c["d"], dtype=torch.float64, device=DEV)
    rep = c["heads"] // c["kv"]
    for b in range(c["seqs"]):
        a, e, n, t = start[b], start[b + 1], new[b], ctx[b]
        i = torch.arange(n, device=DEV)
        first = torch.zeros_like(i) if s["row_begin"] is None else s["row_begin"][a:e].long()
        hidden = (i[None] > i[:, None]) | (i[None] < first[:, None])
        hidden = torch.cat([hidden.new_zeros(n, t), hidden], 1)
        keys = torch.cat([sequence(k64, b, t), s["k_new"][a:e].double().transpose(0, 1)], 1)
        vals = torch.cat([sequence(v64, b, t), s["v_new"][a:e].double().transpose(0, 1)], 1)
        for h in range(c["heads"]):
            y = (s["q"][a:e, h].double() @ keys[h // rep].T * s["scale"]).masked_fill(hidden, -math.inf)
            out[a:e, h] = torch.softmax(y, -1) @ vals[h // rep]
    return out
