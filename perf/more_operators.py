"""Serving in 4 bits as cases that can be timed and whose outputs can be compared: projections with 4-bit weights, the write of
new tokens into pages with the q/k norm and the rotation on the way, and attention over pages of 4 bits.

Formats. Weights (N, K) in blocks of 32 along a row: w = (u - 8) d with u in 0..15 and one fp16 d a block; a block's 16 bytes
hold values 0-15 in their low halves, 16-31 in the high ones. Pages of 4 bits hold token rows of D values in blocks of 32:
value (u - 8) d with one bf16 d a block; four bytes hold 8 values, the even ones 0, 2, 4, 6 in the halves of the first two bytes
(low half first), the odd ones in those of the last two. A row x is written as: m the value of the largest |x| of the block (the
first of several), d = bf16(m / -8), u = floor(x / d + 8.5) within 0..15; a block below 2^-100 is d = 0, u = 8. Pages may also
hold int8 rows with one fp32 scale, or bf16 rows.

Batches are packed and ragged: sequence b's new tokens are the rows start[b] .. start[b + 1] - 1, at the positions ctx[b],
ctx[b] + 1, ...; position j of sequence b lies in row j % page of page table[b, j // page]. Kinds:

  write   per token, RMSNorm of every q and k head and the rotation of its first `rot` dims, the new K and V into their pages
          (the rounding steps of the package's qk_norm_rope: each elementwise product in bf16); then the sequences read back
  attn    every new token attends its sequence's cached tokens, 4 bits each, and the new ones from row_begin on up to itself
  linear  y = x W^T (+ residual) with 4-bit W, x and y in bf16

The dims are those of the package's decoders: 32 / 8 heads of 128, the hybrid stack's 16 / 4 heads of 256 with 64 rotated dims
and zero-centred norms, the 16 / 4 heads of 64 of the attention tests; hidden 4096, MLP 12288, vocabulary 151936.
"""
import math

import torch

own = False

DEV = "cuda"
BF = torch.bfloat16
EPS = 1e-6
ORDER = [0, 2, 4, 6, 1, 3, 5, 7]  # the values of 8 in the order of their four bits


def listed():
    return [
        # a token for each of 64 running sequences: latency
        dict(name="write_64x1", kind="write", seqs=64, new=1, ctx=48, heads=32, kv=8, d=128, rot=128, offset=False, page=16,
             bits=4),
        # the chunks of 8 states of different lengths, a prefill step of about 4000 tokens
        dict(name="write_8x900", kind="write", seqs=8, new=900, ctx=150, heads=32, kv=8, d=128, rot=128, offset=False, page=64,
             bits=4),
        # the same step of the hybrid stack's attention layers (partial rotation, zero-centred norms) into int8 pages
        dict(name="write_4x700_256", kind="write", seqs=4, new=700, ctx=333, heads=16, kv=4, d=256, rot=64, offset=True, page=32,
             bits=8),
        # one token over one short state: latency
        dict(name="token_1x700", kind="attn", seqs=1, new=1, ctx=700, rows=0, heads=16, kv=4, d=256, page=16),
        # a token for each of 64 sequences of different lengths
        dict(name="token_64x4096", kind="attn", seqs=64, new=1, ctx=4096, rows=0, heads=32, kv=8, d=128, page=64),
        # a token for each of 8 long states: bound by reading them
        dict(name="token_8x32768", kind="attn", seqs=8, new=1, ctx=32768, rows=0, heads=32, kv=8, d=128, page=128),
        # a long chunk appended to a long state: bound by the matrix cores
        dict(name="chunk_2048_16384", kind="attn", seqs=1, new=2048, ctx=16384, rows=0, heads=32, kv=8, d=128, page=64),
        # option rows: 8 requests of 32 options of up to 16 tokens over their own states, an option sees its own tokens only
        dict(name="options_8x512", kind="attn", seqs=8, new=512, ctx=2048, rows=16, heads=32, kv=8, d=128, page=64),
        # the output projection of one token, added to the residual: latency
        dict(name="linear_1_4096x4096", kind="linear", m=1, n=4096, k=4096, residual=True),
        # gate and up projections of 24 sequences' tokens
        dict(name="linear_24_24576x4096", kind="linear", m=24, n=24576, k=4096, residual=False),
        # one token's logits over the vocabulary
        dict(name="linear_1_151936x4096", kind="linear", m=1, n=151936, k=4096, residual=False),
        # the down projection of a prefill step
        dict(name="linear_2000_4096x12288", kind="linear", m=2000, n=4096, k=12288, residual=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _drawn(rng):
    kind = rng.choice(["write", "attn", "attn", "attn", "linear", "linear"])
    if kind == "linear":
        m = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 65, 3000)])
        return dict(kind=kind, m=m, n=_log(rng, 200, 60000 if m < 65 else 16000), k=32 * _log(rng, 8, 400),
                    residual=rng.random() < 0.5)
    heads, kv, d, rot, offset = rng.choice([(32, 8, 128, 128, False), (32, 8, 128, 128, False), (16, 4, 256, 64, True),
                                            (16, 4, 64, 64, False), (28, 4, 128, 128, False), (8, 8, 64, 64, False)])
    c = dict(kind=kind, heads=heads, kv=kv, d=d, page=rng.choice([16, 32, 64, 128]))
    if kind == "write":
        return dict(c, seqs=_log(rng, 1, 128), new=_log(rng, 1, 1200), ctx=_log(rng, 1, 300), rot=rot, offset=offset,
                    bits=rng.choice([4, 4, 8, 16]))
    c["rows"] = 0
    form = rng.choice(["token", "token", "tokens", "chunk", "rows"])
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
    new = _ragged(n, c["new"], 1) if c["new"] > 1 else [1] * n
    ctx = _ragged(n, c["ctx"], 1)[::-1]
    if n > 1 and c["new"] > 1:
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


def _row_bytes(c):
    """One token's K or V in the pages."""
    d = c["d"]
    return c["kv"] * {4: d // 2 + d // 16, 8: d + 4, 16: 2 * d}[c.get("bits", 4)]


def work(case):
    c = case
    if c["kind"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": n * k // 32 * 18 + 2 * m * k + 2 * m * n * (2 if c["residual"] else 1), "flops": 2 * m * n * k}
    new, ctx = _lengths(c)
    hq, kv, d, row = c["heads"], c["kv"], c["d"], _row_bytes(c)
    if c["kind"] == "write":  # the projection in, q and k out, the new rows of K and V, and both read back as bf16
        T = max(t + n for t, n in zip(new, ctx))
        back = (sum(new) + sum(ctx)) * 2 * row + c["seqs"] * T * 2 * kv * d * 2
        return {"bytes": sum(new) * ((hq + 2 * kv) * d * 2 + (hq + kv) * d * 2 + 2 * row) + back,
                "flops": sum(new) * (hq + kv) * d * 8 + (sum(new) + sum(ctx)) * 2 * kv * d}
    pairs = sum(n * t + _own_pairs(n, c["rows"]) for n, t in zip(new, ctx))
    return {"bytes": sum(ctx) * 2 * row + sum(new) * 2 * (kv + hq) * d * 2, "flops": 4 * hq * d * pairs}


# ---------------------------------------------------------------------------------------------- formats, plain
def _q8(x):
    """int8 rows and fp32 scales of x (..., D): scale = max(max |x|, 1e-8) / 127, q = round(x / scale), fp32 quotients (a
    Python number as divisor would be turned into a product with its reciprocal)."""
    xf = x.float()
    s = xf.abs().amax(-1, keepdim=True).clamp_min(1e-8) / xf.new_full((), 127.0)
    return torch.round(xf / s).clamp_(-127, 127).to(torch.int8), s[..., 0]


def _q4(x):
    """uint8 rows (..., D / 2) and bf16 scales (..., D / 32) of bf16 x (..., D); quotients in 64 bits, next to borders."""
    g = x.float().unflatten(-1, (-1, 32))
    m = g.gather(-1, g.abs().argmax(-1, keepdim=True))
    d = torch.where(m.abs() < 2.0 ** -100, 0.0, m / -8.0).to(BF)
    inv = torch.where(d == 0, 0.0, 1.0).double()
    u = torch.floor(g.double() * inv / torch.where(d == 0, 1.0, d.double()) + 8.5).clamp_(0, 15).to(torch.uint8).flatten(-2)
    u = u.unflatten(-1, (-1, 8))[..., ORDER].flatten(-2)
    return u[..., 0::2] | (u[..., 1::2] << 4), d[..., 0]


def _values(rows, scale):
    """The fp32 values that page rows stand for."""
    if scale is None:
        return rows.float()
    if rows.dtype == torch.int8:
        return rows * scale[..., None]
    u = torch.stack([rows & 15, rows >> 4], -1).flatten(-2).unflatten(-1, (-1, 8))
    u = u.unflatten(-1, (2, 4)).transpose(-1, -2).flatten(-3)  # even and odd ones side by side
    return ((u.float() - 8.0).unflatten(-1, (-1, 32)) * scale.float()[..., None]).flatten(-2)


def _weights(qs, d):
    """fp32 (N, K) of 4-bit weights."""
    u = qs.unflatten(-1, (-1, 16))
    return ((torch.cat([u & 15, u >> 4], -1).float() - 8.0) * d.float()[..., None]).flatten(-2)


# ---------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rows(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(BF)

    return _prepare_linear(case, g, rows) if case["kind"] == "linear" else _prepare_pages(case, g, rows)


def _prepare_linear(c, g, rows):
    m, n, k = c["m"], c["n"], c["k"]
    qs, d = torch.empty(n, k // 2, dtype=torch.uint8, device=DEV), torch.empty(n, k // 32, dtype=torch.float16, device=DEV)
    step = max(1, (1 << 26) // k)
    for a in range(0, n, step):
        w = 0.02 * torch.randn(min(step, n - a), k // 32, 32, generator=g, device=DEV)
        big = w.gather(-1, w.abs().argmax(-1, keepdim=True)) / -8.0
        u = torch.floor(w / big + 8.5).clamp_(0, 15).to(torch.uint8)
        qs[a:a + step], d[a:a + step] = (u[..., :16] | (u[..., 16:] << 4)).flatten(-2), big[..., 0].to(torch.float16)
    x = rows(m, k)
    x[:, ::97] *= 8.0  # a few large channels, as the activations of trained models have
    return dict(c, x=x, qs=qs, d=d, res=rows(m, n) if c["residual"] else None)


def _prepare_pages(c, g, rows):
    new, ctx = _lengths(c)
    B, hq, kv, d, ps, bits = c["seqs"], c["heads"], c["kv"], c["d"], c["page"], c.get("bits", 4)
    per = [-(-(t + n) // ps) for n, t in zip(new, ctx)]
    cols, pages = max(per), sum(per) + 3  # some of the pool is free
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    held = torch.arange(cols, device=DEV)[None] < torch.tensor(per, device=DEV)[:, None]
    first = torch.tensor([sum(per[:b]) for b in range(B)], device=DEV)[:, None] + torch.arange(cols, device=DEV)[None]
    table = torch.where(held, order[first.clamp_max(pages - 1)], -1).to(torch.int32).contiguous()
    start = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEV)
    N = sum(new)
    common = rows(kv, d).float()  # the direction that every query shares with its sequence's first key
    k, v = rows(pages, kv, ps, d), rows(pages, kv, ps, d) * 0.5
    # a sequence's first token draws much of the attention and has a small value, as in trained models
    sinks = table[:, 0].long()
    k[sinks, :, 0] = (1.2 * common).to(BF)
    v[sinks, :, 0] *= 0.05
    ks = vs = None
    if bits < 16:
        (k, ks), (v, vs) = (_q4(k), _q4(v)) if bits == 4 else (_q8(k), _q8(v))
    qkv = rows(N, (hq + 2 * kv) * d)  # the new tokens' projections in one buffer, as a fused projection writes them
    s = dict(c, B=B, N=N, start=start, ctx=torch.tensor(ctx, dtype=torch.int32, device=DEV), table=table, max_new=max(new),
             max_ctx=max(ctx), k=k, v=v, k_scale=ks, v_scale=vs, qkv=qkv)
    if c["kind"] == "write":
        T = max(t + n for t, n in zip(new, ctx))
        angle = torch.arange(T, device=DEV).double()[:, None] / 1e6 ** (torch.arange(0, c["rot"], 2, device=DEV).double() / c["rot"])
        weight = [(0.1 * rows(d).float() + (0.0 if c["offset"] else 1.0)).to(BF) for _ in range(2)]
        pos = torch.cat([torch.arange(t, t + n, dtype=torch.int32, device=DEV) for n, t in zip(new, ctx)])
        return dict(s, T=T, end=s["ctx"] + start[1:] - start[:-1], cos=angle.cos().to(BF), sin=angle.sin().to(BF), qw=weight[0],
                    kw=weight[1], pos=pos, out=torch.empty(N, (hq + kv) * d, dtype=BF, device=DEV))
    qkv[:, :hq * d].view(N, kv, hq // kv, d).add_((0.5 * common[:, None]).to(BF))
    q, k_new, v_new = qkv.split([hq * d, kv * d, kv * d], 1)
    s.update(q=q.view(N, hq, d), k_new=k_new.view(N, kv, d), v_new=v_new.view(N, kv, d), scale=d ** -0.5, row_begin=None)
    if c["rows"]:
        local = torch.cat([torch.arange(n, device=DEV) for n in new])
        s["row_begin"] = (local // c["rows"] * c["rows"]).to(torch.int32)
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _tokens(s):
    """(sequence, index within its new tokens) of every packed row."""
    n = torch.arange(s["N"], device=DEV)
    seq = torch.searchsorted(s["start"].long(), n, right=True) - 1
    return seq, n - s["start"].long()[seq]


def _normed(x, w, offset):
    """RMSNorm of bf16 heads (..., D) as the decoder's bf16 modules round it."""
    xd = x.double()
    r = (1.0 / torch.sqrt((xd * xd).mean(-1, keepdim=True) + float(torch.tensor(EPS)))).float()
    if offset:
        return ((x.float() * r) * (1.0 + w.float())).to(BF)
    return w * (x.float() * r).to(BF)


def _rotated(n, cos, sin, rot):
    a, b, rest = n.split([rot // 2, rot // 2, n.shape[-1] - rot], -1)
    return torch.cat([a * cos + (-b) * sin, b * cos + a * sin, rest], -1)


def _plain_write(s):
    hq, kv, d, N = s["heads"], s["kv"], s["d"], s["N"]
    q, k, v = (x.view(N, -1, d) for x in s["qkv"].split([hq * d, kv * d, kv * d], 1))
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    q, k = (_rotated(_normed(x, w, s["offset"]), cos, sin, s["rot"]) for x, w in ((q, s["qw"]), (k, s["kw"])))
    seq, i = _tokens(s)
    at = s["ctx"].long()[seq] + i
    page, row = s["table"].long()[seq, at // s["page"]], at % s["page"]
    for x, pages, scales in ((k, s["k"], s["k_scale"]), (v, s["v"], s["v_scale"])):
        if scales is None:
            pages[page, :, row] = x
        else:
            pages[page, :, row], scales[page, :, row] = (_q4 if s["bits"] == 4 else _q8)(x)
    out = {"qk": torch.cat([q, k], 1).flatten(1)}
    out["k"], out["v"], _ = _cached(s, s["T"], s["end"])
    return {n: x if n == "qk" else x.transpose(1, 2).to(BF).contiguous() for n, x in out.items()}


def _cached(s, T, length):
    """The first T positions of every sequence, (B, T, heads, D) fp32 K and V, zeros where it has none."""
    j = torch.arange(T, device=DEV)
    there = j[None] < length[:, None]
    page = s["table"].long()[:, j // s["page"]].clamp_min(0)
    row = (j % s["page"])[None].expand_as(page)

    def side(p, sc):
        y = _values(p[page, :, row], None if sc is None else sc[page, :, row])
        return torch.where(there[:, :, None, None], y, 0.0)

    return side(s["k"], s["k_scale"]), side(s["v"], s["v_scale"]), there


def _plain_attn(s):
    B, n, T, hq, kv, d = s["B"], s["max_new"], s["max_ctx"], s["heads"], s["kv"], s["d"]
    rep = hq // kv
    kc, vc, there = _cached(s, T, s["ctx"])
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


def _plain_linear(s):
    y = s["x"].float() @ _weights(s["qs"], s["d"]).T
    return (y if s["res"] is None else y + s["res"].float()).to(BF)


def run(state):
    s = state
    if not own:
        return {"write": _plain_write, "attn": _plain_attn, "linear": _plain_linear}[s["kind"]](s)
    from opendecider_amd import PagedKVCache, kernels
    if s["kind"] == "linear":
        return kernels.q4_linear(s["x"], s["qs"], s["d"], residual=s["res"])
    if "cache" not in s:  # the program's handle on its pools
        s["cache"] = PagedKVCache.from_tensors(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if s["kind"] == "write":
        kernels.qk_norm_rope_page_append(s["qkv"], s["heads"], s["kv"], s["d"], s["qw"], s["kw"], s["cos"], s["sin"], s["pos"],
                                         EPS, s["cache"], s["table"], s["start"], s["ctx"], rot_dim=s["rot"],
                                         offset=s["offset"], out=s["out"])
        k, v = kernels.page_read(s["cache"], s["table"], s["end"], s["T"])
        return {"qk": s["out"], "k": k, "v": v}
    return kernels.paged_attn(s["q"], s["k_new"], s["v_new"], s["cache"], s["table"], s["start"], s["ctx"], s["scale"],
                              row_begin=s["row_begin"], max_new=s["max_new"], max_ctx=s["max_ctx"])


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_rows(pages, scales):
    """The float64 values of whole pools."""
    if scales is None:
        return pages.double()
    if pages.dtype == torch.int8:
        return pages.double() * scales.double()[..., None]
    y = torch.empty(*pages.shape[:-1], 2 * pages.shape[-1], dtype=torch.float64, device=DEV)
    for byte in range(4):
        for half, part in enumerate((pages[..., byte::4] % 16, pages[..., byte::4] // 16)):
            y[..., ORDER[2 * byte + half]::8] = part.double() - 8
    return y * scales.double().repeat_interleave(32, -1)


def _exact_written(x, bits):
    """What bf16 rows x (n, heads, D) stand for once written, float64."""
    x = x.double()
    if bits == 16:
        return x
    if bits == 8:  # the stored scale and the quotient that is rounded are fp32 numbers by definition
        scale = (x.abs().amax(-1, keepdim=True).clamp_min(1e-8) / 127).float().double()
        return (x / scale).float().double().round().clamp(-127, 127) * scale
    y = torch.zeros_like(x)
    for a in range(0, x.shape[-1], 32):
        b = x[..., a:a + 32]
        size = b.abs().amax(-1, keepdim=True)
        lead = b.abs() == size
        m = (b * (lead & (lead.cumsum(-1) == 1))).sum(-1, keepdim=True)
        d = (m / -8).to(BF).double()
        u = (b / torch.where(size < 2.0 ** -100, torch.ones_like(d), d) + 8.5).floor().clamp(0, 15)
        y[..., a:a + 32] = torch.where(size < 2.0 ** -100, torch.zeros_like(b), (u - 8) * d)
    return y


def _exact_head(x, w, c, cos, sin):
    """One head's rows (n, D) float64, normed and rotated: each product of bf16 numbers rounded to bf16, by definition."""
    def bf(y):
        return y.float().to(BF).double()

    r = (1 / ((x ** 2).mean(1, keepdim=True) + float(torch.tensor(EPS))).sqrt()).float().double()
    xr = (x * r).float().double()
    n = bf(xr * (1 + w).float().double()) if c["offset"] else bf(w * bf(xr))
    h = c["rot"] // 2
    a, b = n[:, :h].clone(), n[:, h:2 * h].clone()
    n[:, :h], n[:, h:2 * h] = bf(bf(a * cos) - bf(b * sin)), bf(bf(b * cos) + bf(a * sin))
    return n


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "linear":
        y = torch.empty(c["m"], c["n"], dtype=torch.float64, device=DEV)
        for a in range(0, c["n"], 8192):
            u = s["qs"][a:a + 8192].view(-1, c["k"] // 32, 16)
            w = torch.empty(u.shape[0], c["k"] // 32, 32, dtype=torch.float64, device=DEV)
            w[..., :16], w[..., 16:] = (u % 16).double() - 8, (u // 16).double() - 8
            w *= s["d"][a:a + 8192].double()[..., None]
            y[:, a:a + 8192] = s["x"].double() @ w.view(u.shape[0], c["k"]).T
        return y if s["res"] is None else y + s["res"].double()
    new, ctx = _lengths(c)
    B, hq, kv, d, ps, table, start = c["seqs"], c["heads"], c["kv"], c["d"], c["page"], s["table"].tolist(), s["start"].tolist()
    k64, v64 = _exact_rows(s["k"], s["k_scale"]), _exact_rows(s["v"], s["v_scale"])

    def sequence(pages, b, n):  # the first n tokens of sequence b, (heads, n, D)
        at = table[b][:-(-n // ps)]
        return pages[at].transpose(0, 1).reshape(kv, -1, d)[:, :n] if n else pages.new_zeros(kv, 0, d)

    if c["kind"] == "write":
        cos, sin = (s[n].double()[s["pos"].long()] for n in ("cos", "sin"))
        qk = torch.empty(s["N"], hq + kv, d, dtype=torch.float64, device=DEV)
        for h in range(hq + kv):
            qk[:, h] = _exact_head(s["qkv"][:, h * d:(h + 1) * d].double(), (s["qw"] if h < hq else s["kw"]).double(), c, cos, sin)
        v = s["qkv"][:, (hq + kv) * d:].reshape(s["N"], kv, d)
        out = {"qk": qk.flatten(1)}
        for name, pages, x in (("k", k64, qk[:, hq:]), ("v", v64, v)):
            dense = torch.zeros(B, kv, s["T"], d, dtype=torch.float64, device=DEV)
            x = _exact_written(x, c["bits"])
            for b in range(B):
                dense[b, :, :ctx[b]] = sequence(pages, b, ctx[b])
                dense[b, :, ctx[b]:ctx[b] + new[b]] = x[start[b]:start[b + 1]].transpose(0, 1)
            out[name] = dense
        return out
    out = torch.zeros(s["N"], hq, d, dtype=torch.float64, device=DEV)
    rep = hq // kv
    for b in range(B):
        a, e, n, t = start[b], start[b + 1], new[b], ctx[b]
        i = torch.arange(n, device=DEV)
        first = torch.zeros_like(i) if s["row_begin"] is None else s["row_begin"][a:e].long()
        hidden = (i[None] > i[:, None]) | (i[None] < first[:, None])
        hidden = torch.cat([hidden.new_zeros(n, t), hidden], 1)
        keys = torch.cat([sequence(k64, b, t), s["k_new"][a:e].double().transpose(0, 1)], 1)
        vals = torch.cat([sequence(v64, b, t), s["v_new"][a:e].double().transpose(0, 1)], 1)
        for h in range(hq):
            y = (s["q"][a:e, h].double() @ keys[h // rep].T * s["scale"]).masked_fill(hidden, -math.inf)
            out[a:e, h] = torch.softmax(y, -1) @ vals[h // rep]
    return out
