"""The paged K/V cache in 4 bits on the GPU against its float64 restatement (oracle/paged.py): the bytes written, with and without
the q/k norm and rotation on the way, the values read back, and attention, at the sizes, masks and layouts of
test_gpu_paged.py, whose batches and bounds these are.

Bounds of the attention: those of test_gpu_paged.py without the int8 values' rounding, since a 4-bit value is exact in fp16 (3
significant bits by 8): the scores' error e is that of fp32 sums, 2^-24 (D + 8) S, plus what frames lose: a value below fp16's
normal numbers in a frame whose largest is at least 2^10 moves by 2^-25 at most, 2^-35 of the largest, so a score by 2^-35 D
S_max, S_max = scale max|q| sum over d of the largest |k| of the 64 keys that share a frame, taken from the pages below.
"""
import math

import pytest
import torch

import test_gpu_paged as tp
from oracle import decoder as od
from oracle import paged as op

pytestmark = pytest.mark.gpu

DEV, BF = tp.DEV, tp.BF
gpu, cache_of, run_attn, SHAPES, MANY = tp.gpu, tp.cache_of, tp.run_attn, tp.SHAPES, tp.MANY


def make(*a, int8=None, **kw):
    """A batch of test_gpu_paged over 4-bit pages (int8 True, False: over those)."""
    if int8 is not None:
        return tp.make(*a, int8=int8, **kw)
    c = tp.make(*a, int8=False, **kw)
    packed = [op.pack4(x) for x in c["pages"]]
    c["pages"], c["scales"] = [q for q, _ in packed], [s for _, s in packed]
    return c


def check_attn(c, out, lse, own=True):
    ref, rl, mean, size, total = op.attention(c["q"], c["k"] if own else None, c["v"] if own else None, (*c["pages"], *c["scales"]),
                                              c["table"], c["start"], c["ctx"], c["scale"], c["row_begin"])
    out, lse = out.double().cpu(), lse.double().cpu()
    live = ~rl.isnan()
    D, T = c["q"].shape[2], int(c["ctx"].clamp_min(0).max()) + c["q"].shape[0]
    largest = op.values(c["pages"][0], c["scales"][0]).nan_to_num(posinf=0, neginf=0).abs().amax()
    e = 2.0 ** -24 * (D + 8) * size + 2.0 ** -35 * c["scale"] * c["q"].double().nan_to_num(posinf=0, neginf=0).abs().sum(-1) * largest
    bound = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2 * e[..., None] + 2.0 ** -22 * (T + 16)) * 1.02 * mean + 2.0 ** -31 * total[..., None]
    bad = (out - ref).abs() > bound
    assert not bad[live].any(), f"{int(bad[live].sum())} of {int(live.sum()) * D}: worst {((out - ref).abs() / bound.clamp_min(1e-300))[live].max()}"
    assert not out[live].isnan().any()
    none = live & (rl == -math.inf)
    assert (out[none] == 0).all() and (lse[none] == -math.inf).all()
    some = live & ~none
    lb = e + 2.0 ** -20 * (1 + rl.abs() + size)
    assert ((lse - rl).abs() <= lb)[some].all(), f"lse off by {((lse - rl).abs() / lb)[some].max()} of its bound"


def as_many(c, form):
    """The same batch as the library takes it for a large one: rows of no sequence, a table with room for many tokens, or both
    (then the pages go through the image)."""
    if form in ("table", "image"):
        page = c["pages"][0].shape[2]
        wide = torch.full((c["table"].shape[0], (2 ** 20 if form == "table" else 2 ** 16) // page), -1, dtype=torch.int32)
        wide[:, :c["table"].shape[1]] = c["table"]
        c["table"] = wide
    return c


def padded(form):
    return {} if form in ("few", "table") else dict(pad=1100)


FORMS = ["few", "rows", "table", "image"]


@pytest.mark.parametrize("d,heads,kv", [(64, 4, 4), (128, 8, 2), (256, 4, 1), (128, 7, 1)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention(gpu_lib, shape, d, heads, kv):
    new, ctx = SHAPES[shape]
    c = make(shape, new, ctx, heads, kv, d, page=[16, 64, 32][shape % 3])
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("d,heads,kv", [(64, 4, 4), (128, 8, 2), (256, 8, 4), (256, 4, 1)])
@pytest.mark.parametrize("seqs", [1, 3, 90])
def test_tokens_of_many_sequences(gpu_lib, seqs, d, heads, kv):
    """One token a sequence, from few (the cached tokens in many parts) to more workgroups than CUs."""
    g = torch.Generator().manual_seed(seqs)
    ctx = torch.randint(0, 2600 if seqs < 10 else 300, (seqs,), generator=g).tolist()
    ctx[-1] = 2600 if seqs < 10 else 300
    c = tp.make(70 + seqs, [1] * seqs, ctx, heads, kv, d, page=32, int8=False)
    shape = c["pages"][0].shape[:3]  # any bytes are rows of 4 bits
    c["pages"] = [torch.randint(0, 256, (*shape, d // 2), generator=g, dtype=torch.uint8) for _ in range(2)]
    c["scales"] = [(torch.randn(*shape, d // 32, generator=g) / 4).to(BF) for _ in range(2)]
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("d,heads,kv", [(64, 4, 4), (128, 8, 2), (256, 4, 1), (128, 7, 1)])
@pytest.mark.parametrize("form", FORMS[1:])
@pytest.mark.parametrize("shape", range(len(MANY)))
def test_many_slots(gpu_lib, shape, form, d, heads, kv):
    new, ctx = MANY[shape]
    c = as_many(make(shape, new, ctx, heads, kv, d, page=[16, 64, 32][shape % 3], **padded(form)), form)
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,ctx,rows", [([24, 40, 1], [50, 0, 129], 8), ([150, 90], [33, 64], 30)])
def test_option_rows(gpu_lib, new, ctx, rows, d, form):
    c = as_many(make(7, new, ctx, 8, 2, d, page=32, rows=rows, **padded(form)), form)
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("new,ctx", [([3, 1], [0, 40]), ([100, 60], [0, 90]), ([1, 1, 1], [0, 700, -5])])
def test_cached_tokens_only(gpu_lib, new, ctx, form):
    c = as_many(make(3, new, ctx, **padded(form)), form)
    check_attn(c, *run_attn(c, own=False), own=False)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,ctx", [([1, 1, 1, 1], [700, 90, 40, 33]), ([40, 1, 100], [200, 90, 33])])
def test_no_pages_and_short_tables(gpu_lib, new, ctx, d, form):
    c = make(11, new, ctx, d=d, **padded(form))
    n, cols = c["pages"][0].shape[0], c["table"].shape[1]
    c["table"][0, 1], c["table"][0, 3], c["table"][1, 0], c["table"][-1, 0], c["table"][-1, 1] = -1, n, 2 ** 31 - 1, -7, n + 5
    c = as_many(c, form)
    check_attn(c, *run_attn(c))
    if form in ("few", "rows"):
        c["ctx"][1] = 10 ** 6
        c["table"] = c["table"][:, :4].contiguous()
        check_attn(c, *run_attn(c))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,ctx", [([2, 1], [30, 40]), ([100], [70])])
def test_what_is_masked_does_not_matter(gpu_lib, new, ctx, d, form):
    """NaN and infinite scales in the pages past the cached tokens, NaN in pad rows: bit for bit the same."""
    c = as_many(make(4, new, ctx, d=d, rows=1, **padded(form)), form)
    c["q"], c["k"], c["v"] = (torch.cat([x, x[:5]]) for x in (c["q"], c["k"], c["v"]))
    c["row_begin"] = torch.cat([c["row_begin"], c["row_begin"][:5]])
    want, wl = run_attn(c)
    used = torch.zeros(c["pages"][0].shape[0], 16, dtype=torch.bool)
    for b, t in enumerate(ctx):
        for j in range(t):
            used[c["table"][b, j // 16], j % 16] = True
    for i in range(2):
        c["scales"][i] = torch.where(used[:, None, :, None], c["scales"][i].float(), float("nan") if i else float("inf")).to(BF)
        c["pages"][i] = torch.where(used[:, None, :, None], c["pages"][i], 255)
    N = sum(new)
    c["k"][N:], c["v"][N:], c["q"][N:] = float("nan"), float("inf"), float("nan")
    got, gl = run_attn(c)
    assert torch.equal(got[:N], want[:N]) and torch.equal(gl[:N], wl[:N])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_blocks_that_are_not_finite(gpu_lib, d, bad, form):
    """A key's block of that kind makes its scores NaN: every output that sees the key. A value's makes its 32 columns NaN, no
    others."""
    c = as_many(make(21, [3, 40], [70, 30], 4, 2, d, **padded(form)), form)
    N = 43
    clean, _ = run_attn(c)
    at = lambda b, pos: (int(c["table"][b, pos // 16]), pos % 16)
    p, r = at(1, 5)
    keep = c["scales"][1][p, 1, r].clone()
    c["scales"][1][p, 1, r, 1] = bad  # sequence 1, head group 1, columns 32 .. 63
    out, _ = run_attn(c)
    hit = torch.zeros(out.shape, dtype=torch.bool)
    hit[3:N, 2:, 32:64] = True
    live = torch.zeros(out.shape[0], dtype=torch.bool)
    live[:N] = True
    out, clean = out.cpu(), clean.cpu()
    assert out[hit].isnan().all() and torch.equal(out[live][~hit[live]], clean[live][~hit[live]])
    c["scales"][1][p, 1, r] = keep
    p, r = at(0, 69)
    c["scales"][0][p, 0, r, -1] = bad  # sequence 0, head group 0
    out = run_attn(c)[0].cpu()
    hit = torch.zeros(out.shape, dtype=torch.bool)
    hit[:3, :2] = True
    assert out[hit].isnan().all() and torch.equal(out[live][~hit[live]], clean[live][~hit[live]])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("k_exp,v_exp", [(-100, 60), (60, -100), (0, -20), (20, 100)])
def test_sizes_of_the_rows(gpu_lib, d, k_exp, v_exp, form):
    """Scales far from 1 in the pages, queries that bring the scores back to their usual size."""
    for new, ctx in (([1, 1], [600, 90]), ([40], [300])):
        c = as_many(make(8, new, ctx, 4, 1, d, **padded(form)), form)
        c["scales"][0] = (c["scales"][0].float() * 2.0 ** k_exp).to(BF)
        c["scales"][1] = (c["scales"][1].float() * 2.0 ** v_exp).to(BF)
        c["q"] = (c["q"].float() * 2.0 ** -k_exp).to(BF)
        c["k"] = (c["k"].float() * 2.0 ** k_exp).to(BF)
        c["v"] = (c["v"].float() * 2.0 ** v_exp).to(BF)
        check_attn(c, *run_attn(c))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_sizes_within_a_row(gpu_lib, d, form):
    """Blocks of one row 2^20 apart, and rows 2^40 apart."""
    for new, ctx in (([1, 2], [200, 90]), ([40], [130])):
        c = make(9, new, ctx, 4, 2, d, **padded(form))
        g = torch.Generator().manual_seed(1)
        for i, spread in enumerate((0, 20)):  # K's blocks near each other: the scores are what their largest ones make
            e = torch.randint(-10, 11, c["scales"][i].shape, generator=g).float() + torch.randint(-spread, spread + 1,
                                                                                              (*c["scales"][i].shape[:3], 1), generator=g)
            c["scales"][i] = (c["scales"][i].float() * torch.exp2(e if i else e / 4)).to(BF)
        c = as_many(c, form)
        check_attn(c, *run_attn(c))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("new,ctx", [([1, 1], [1000, 64]), ([64, 90], [400, 10])])
def test_sharp_scores(gpu_lib, new, ctx, form):
    c = as_many(make(9, new, ctx, mag=12.0, **padded(form)), form)
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("new", [[1, 1, 1], [3, 60, 1]])
def test_bounds_do_not_change_what_is_computed(gpu_lib, new):
    c = make(10, new, [300, 1100, 17])
    for mn in (1, max(new), None):
        for mc in (0, 64, 1100, 10 ** 6, None):
            check_attn(c, *run_attn(c, max_new=mn, max_ctx=mc))


@pytest.mark.parametrize("d,heads,kv,pad", [(256, 4, 1, 6000), (128, 8, 1, 24000), (64, 8, 1, 24000)])
def test_image_of_some(gpu_lib, d, heads, kv, pad):
    """max_ctx below one state's length: the others go through the image, that one as it is."""
    from opendecider_amd import kernels
    c = make(15, [70, 40, 30], [500, 3000, 1024], heads, kv, d, page=64, pad=pad)
    dev = torch.device(DEV, torch.cuda.current_device())
    assert kernels.paged_attn_workspace_floats(3, pad + 140, heads, kv, d, pad + 140, 1024, dev, "int4") > 3 * kv * 1024 * d
    check_attn(c, *run_attn(c, max_ctx=1024))


@pytest.mark.parametrize("new,ctx,pad", [([1] * 5, [2500, 3, 900, 0, 64], 0), ([50, 3], [900, 64], 0), ([300, 3], [900, 64], 0),
                                         ([8, 3, 5], [9, 900, 64], 0)])
def test_same_calls_same_bits_and_order(gpu_lib, new, ctx, pad):
    c = make(13, new, ctx, pad=pad)
    kw = dict(max_new=max(new), max_ctx=max(ctx))
    a, al = run_attn(c, **kw)
    b, bl = run_attn(c, **kw)
    assert torch.equal(a, b) and torch.equal(al, bl)
    perm = list(range(len(new)))[::-1]
    s = [int(x) for x in c["start"]]
    rows = torch.cat([torch.arange(s[p], s[p + 1]) for p in perm])
    d = dict(c, table=c["table"][perm].contiguous(), ctx=c["ctx"][perm].contiguous(), q=c["q"][rows], k=c["k"][rows], v=c["v"][rows],
             start=torch.tensor([sum(new[p] for p in perm[:i]) for i in range(len(new) + 1)], dtype=torch.int32))
    o, ol = run_attn(d, **kw)
    assert torch.equal(o, a[rows.to(DEV)]) and torch.equal(ol, al[rows.to(DEV)])


def test_rows_of_no_sequence_stay(gpu_lib):
    for new in ([3, 2], [80, 70]):
        c = make(2, new, [20, 50], pad=9)
        out = torch.full(c["q"].shape, 7.0, dtype=BF, device=DEV)
        c["start"] = c["start"] + 2
        got, lse = run_attn(c, out=out)
        N = sum(new)
        assert got is out and (out[:2] == 7).all() and (out[2 + N:] == 7).all()
        check_attn(c, out, lse)


@pytest.mark.parametrize("new,pad", [(1, 0), (70, 1100), (70, 6000)])
def test_a_pool_past_32_bits(gpu_lib, new, pad):
    """Pages behind the first 2^32 values of the pool: bit for bit what the same pages do in a small one."""
    from opendecider_amd import PagedKVCache, kernels
    c = make(18, [new, new], [900, 333], 8, 2, page=64, pad=pad)
    want, wl = run_attn(c)
    n, kv, page, half = c["pages"][0].shape
    total = 2 ** 31 // (kv * page * half) + n
    big = [torch.zeros(total, *x.shape[1:], dtype=x.dtype, device=DEV) for x in (*c["pages"], *c["scales"])]
    for x, y in zip(big, (*c["pages"], *c["scales"])):
        x[-n:] = gpu(y)
    cache = PagedKVCache.from_tensors(*big)
    table = torch.where(c["table"] >= 0, c["table"] + (total - n), -1).to(torch.int32)
    got, gl = run_attn(dict(c, table=table), cache=cache)
    N = 2 * new
    assert torch.equal(got[:N], want[:N]) and torch.equal(gl[:N], wl[:N])
    args, small = (gpu(c["start"]), gpu(c["ctx"])), cache_of(c)
    kernels.page_append(gpu(c["k"]), gpu(c["v"]), cache, gpu(table), *args)
    kernels.page_append(gpu(c["k"]), gpu(c["v"]), small, gpu(c["table"]), *args)
    assert torch.equal(cache.k[-n:], small.k) and torch.equal(cache.v_scale[-n:], small.v_scale) and not cache.k[:-n].any()
    for x, y in zip(kernels.page_read(cache, gpu(table), args[1], 900), kernels.page_read(small, gpu(c["table"]), args[1], 900)):
        assert torch.equal(x, y)


# ------------------------------------------------------------------------------------------------ append, read
def same_pools(cache, pools):
    for got, want in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), pools):
        if got is not None:
            got = got.cpu()
            if got.is_floating_point():  # a NaN scale is any NaN
                assert torch.equal(got.isnan(), want.isnan())
                got, want = got.nan_to_num(7.0), want.nan_to_num(7.0)
            assert torch.equal(got, want)


def appended(c, k):
    new = [op.append(c["pages"][i], c["scales"][i], x, c["table"], c["start"], c["ctx"]) for i, x in enumerate((k, c["v"]))]
    return new[0][0], new[1][0], new[0][1], new[1][1]


@pytest.mark.parametrize("d,kv", [(64, 1), (64, 5), (128, 2), (128, 8), (256, 3)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_append(gpu_lib, shape, d, kv):
    from opendecider_amd import kernels
    new, ctx = SHAPES[shape]
    c = make(20 + shape, new, ctx, kv, kv, d, page=[16, 32, 64][shape % 3], pad=3)
    c["k"][0] = 0.0
    cache = cache_of(c)
    kernels.page_append(gpu(c["k"]), gpu(c["v"]), cache, gpu(c["table"]), gpu(c["start"]), gpu(c["ctx"]))
    same_pools(cache, appended(c, c["k"]))


def test_append_odd_blocks(gpu_lib):
    """Ties, values half way between codes, the smallest and largest blocks, infinities and NaN."""
    from opendecider_amd import kernels
    from test_int4_pages import odd_blocks
    x = odd_blocks()
    c = make(31, [12], [3], 1, 1, 64)
    c["k"], c["v"] = x[:, None].clone(), x.flip(1)[:, None].contiguous()
    cache = cache_of(c)
    kernels.page_append(gpu(c["k"]), gpu(c["v"]), cache, gpu(c["table"]), gpu(c["start"]), gpu(c["ctx"]))
    same_pools(cache, appended(c, c["k"]))


@pytest.mark.parametrize("seed", range(4))
def test_append_every_pair_of_significands(gpu_lib, seed):
    """A block's largest value of every significand beside values of every significand in each of the eight octaves below it."""
    from opendecider_amd import kernels
    m = (128 + torch.arange(128))[seed::4].float()
    x = torch.zeros(32 * 8 * 5, 32)
    others = ((128 + torch.arange(128)).float()[None] * 2.0 ** -torch.arange(8)[:, None].float())  # (8, 128)
    rows = []
    for v in m.tolist():
        for o in others:
            keep = o[o <= v]
            for a in range(0, len(keep), 31):
                r = torch.zeros(32)
                r[0] = v * (-1) ** a
                r[1:1 + len(keep[a:a + 31])] = keep[a:a + 31]
                rows.append(r)
    x = torch.stack(rows)
    x = torch.cat([x, x.new_zeros(-len(x) % 2, 32)]).view(-1, 1, 64).to(BF)
    c = make(32, [x.shape[0]], [0], 1, 1, 64)
    c["k"], c["v"] = x, -x
    cache = cache_of(c)
    kernels.page_append(gpu(c["k"]), gpu(c["v"]), cache, gpu(c["table"]), gpu(c["start"]), gpu(c["ctx"]))
    same_pools(cache, appended(c, c["k"]))


@pytest.mark.parametrize("d,kv", [(64, 3), (128, 2), (256, 1)])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_read(gpu_lib, dtype, d, kv):
    from opendecider_amd import kernels
    c = make(40, [0] * 6, [33, 0, 1, 64, 700, -4], kv, kv, d)
    c["table"][4, 2], c["table"][3, 0] = -1, c["pages"][0].shape[0]
    for T in (0, 1, 40, 800):
        got = kernels.page_read(cache_of(c), gpu(c["table"]), gpu(c["ctx"]), T, dtype=dtype)
        for i in range(2):
            rows, sc, valid = op.read(c["pages"][i], c["scales"][i], c["table"], c["ctx"], T)
            want = (op.values(rows, sc) * valid[:, None, :, None]).to(dtype)
            assert torch.equal(got[i].cpu(), want)
            assert not got[i].cpu()[~valid[:, None].expand(-1, kv, -1)].view(torch.int16 if dtype == BF else torch.int32).any()


# ------------------------------------------------------------------------ the norm and rotation on the way
def rope_case(seed, new, ctx, hq, hk, d, rot, offset, int8=None, pad=3, cols=0):
    """A batch with a projection buffer [q; k; v; `cols` more columns], norm weights, rotary tables and positions."""
    c = make(seed, new, ctx, hk, hk, d, page=32, int8=int8, pad=pad, spare=3)
    g = torch.Generator().manual_seed(seed + 1)
    N = sum(new) + pad
    cfg = od.DecoderConfig(n_heads=hq, n_kv_heads=hk, head_dim=d, rot_dim=0 if rot == d else rot, norm_offset=offset)
    c["qkv"] = torch.randn(N, (hq + 2 * hk) * d + cols, generator=g).to(BF)
    c["cos"], c["sin"] = od.rope_tables(cfg, 1200)
    c["qw"], c["kw"] = ((0.0 if offset else 1.0) + 0.1 * torch.randn(d, generator=g) for _ in range(2))
    c["qw"], c["kw"] = c["qw"].to(BF), c["kw"].to(BF)
    c["pos"] = torch.randint(0, 1200, (N,), generator=g).to(torch.int32)
    w = (hq + hk) * d
    ref = od.qk_norm_rope(c["qkv"][:, :w + hk * d], cfg, c["qw"], c["kw"], c["cos"], c["sin"], c["pos"].long())
    c["want"], c["k"], c["v"] = ref[:, :w], ref[:, hq * d:w].reshape(N, hk, d), ref[:, w:].reshape(N, hk, d)
    c["args"] = (hq, hk, d)
    c["kw_args"] = dict(rot_dim=rot, offset=offset)
    return c


def rope_call(c, cache, qkv, out=None, pos=None):
    from opendecider_amd import kernels
    return kernels.qk_norm_rope_page_append(qkv, *c["args"], gpu(c["qw"]), gpu(c["kw"]), gpu(c["cos"]), gpu(c["sin"]),
                                            gpu(c["pos"]) if pos is None else pos, 1e-6, cache, gpu(c["table"]), gpu(c["start"]),
                                            gpu(c["ctx"]), out=out, **c["kw_args"])


HEADS = [(4, 2, 128, 128, False), (7, 1, 128, 32, False), (2, 2, 256, 64, True), (3, 3, 256, 256, False), (5, 5, 64, 64, True),
         (8, 2, 64, 16, False), (0, 3, 128, 128, True)]


@pytest.mark.parametrize("hq,hk,d,rot,offset", HEADS)
@pytest.mark.parametrize("int8", [None, True, False])
@pytest.mark.parametrize("new,ctx", [([1], [0]), ([1] * 9, [15, 16, 17, 31, 32, 33, 0, 64, 1]), ([0, 70, 0, 33, 1, 0], [3, 5, 9, 0, 64, 7])])
def test_norm_rope_append(gpu_lib, new, ctx, int8, hq, hk, d, rot, offset):
    """Bit for bit the oracle's norm and rotation, and what page_append writes of them; in place and not."""
    c = rope_case(60, new, ctx, hq, hk, d, rot, offset, int8)
    pools = appended(c, c["k"])
    cache, qkv = cache_of(c), gpu(c["qkv"])
    out = torch.full(c["want"].shape, 9.0, dtype=BF, device=DEV)
    assert rope_call(c, cache, qkv, out) is out
    assert torch.equal(out.cpu(), c["want"]) and torch.equal(qkv.cpu(), c["qkv"])
    same_pools(cache, pools)
    cache = cache_of(c)
    assert rope_call(c, cache, qkv) is qkv
    assert torch.equal(qkv[:, :out.shape[1]].cpu(), c["want"])
    assert torch.equal(qkv[:, out.shape[1]:].cpu(), c["qkv"][:, out.shape[1]:])
    same_pools(cache, pools)


@pytest.mark.parametrize("int8", [None, True, False])
def test_norm_rope_append_many_sequences(gpu_lib, int8):
    """More sequences than one level of the search takes, runs of empty ones, tokens without a page, padding around."""
    g = torch.Generator().manual_seed(1)
    new = torch.randint(0, 3, (300,), generator=g).tolist()
    new[100:180] = [0] * 80
    c = rope_case(61, new, torch.randint(0, 40, (300,), generator=g).tolist(), 3, 1, 64, 64, False, int8, pad=6)
    c["start"] = c["start"] + 4
    c["table"][5], c["table"][7] = -1, c["pages"][0].shape[0]
    c["ctx"][9], c["ctx"][11] = -3, 10 ** 6
    c["start"][-1] = 10 ** 6  # the last sequence reaches outside the rows: it has no tokens
    cache = cache_of(c)
    out = rope_call(c, cache, gpu(c["qkv"]))
    assert torch.equal(out[:, :c["want"].shape[1]].cpu(), c["want"])
    same_pools(cache, appended(c, c["k"]))


def test_norm_rope_append_strides(gpu_lib):
    """Rows at odd addresses and of odd widths, gated projections' further columns, an output of any strides."""
    c = rope_case(62, [5, 40], [9, 70], 4, 2, 128, 128, False, cols=24)
    N, W = c["qkv"].shape
    w = c["want"].shape[1]
    pools = appended(c, c["k"])
    for lead in (0, 1):
        for extra in (0, 3, 8):
            buf = torch.zeros(N * (W + extra) + 8, dtype=BF, device=DEV)[lead:]
            x = buf[:N * (W + extra)].view(N, W + extra)[:, :W]
            x.copy_(gpu(c["qkv"]))
            for size in (w, w + 5, w + 8):
                out = torch.full((N, size), 3.0, dtype=BF, device=DEV)
                cache = cache_of(c)
                rope_call(c, cache, x, out[:, size - w:])
                assert torch.equal(out[:, size - w:].cpu(), c["want"]) and (out[:, :size - w] == 3).all()
                same_pools(cache, pools)
            assert torch.equal(x.cpu(), c["qkv"])
            cache = cache_of(c)
            rope_call(c, cache, x)
            assert torch.equal(x[:, :w].cpu(), c["want"]) and torch.equal(x[:, w:].cpu(), c["qkv"][:, w:])
            same_pools(cache, pools)


def test_norm_rope_append_past_the_tables(gpu_lib):
    """A position outside the rotary tables: that row's rotated heads are NaN, in the pages too, and nothing else changes."""
    c = rope_case(63, [3, 2], [0, 20], 2, 1, 64, 64, False, pad=0)
    pos = c["pos"].clone()
    pos[1], pos[4] = 1200, -1
    cache = cache_of(c)
    out = rope_call(c, cache, gpu(c["qkv"]), pos=gpu(pos)).cpu()[:, :192]
    odd = torch.tensor([False, True, False, False, True])
    assert out[odd].isnan().all() and torch.equal(out[~odd], c["want"][~odd])
    k = c["k"].clone()
    k[odd] = float("nan")
    same_pools(cache, appended(c, k))


def test_norm_rope_append_refusals(gpu_lib):
    from opendecider_amd import PagedKVCache, kernels
    c = rope_case(64, [3], [4], 4, 2, 64, 64, False, pad=0)
    a = dict(qkv=gpu(c["qkv"]), hq=4, hk=2, D=64, qw=gpu(c["qw"]), kw=gpu(c["kw"]), cos=gpu(c["cos"]), sin=gpu(c["sin"]),
             pos=gpu(c["pos"]), cache=cache_of(c), table=gpu(c["table"]), start=gpu(c["start"]), ctx=gpu(c["ctx"]), rot=64, out=None)

    def call(**bad):
        b = dict(a, **bad)
        return kernels.qk_norm_rope_page_append(b["qkv"], b["hq"], b["hk"], b["D"], b["qw"], b["kw"], b["cos"], b["sin"], b["pos"], 1e-6,
                                                b["cache"], b["table"], b["start"], b["ctx"], rot_dim=b["rot"], out=b["out"])

    call()
    for bad in (dict(qkv=a["qkv"].float()), dict(qw=a["qw"].float()), dict(cos=a["cos"].float()), dict(table=a["table"].long()),
                dict(ctx=a["ctx"].long())):
        with pytest.raises(TypeError):
            call(**bad)
    for bad in (dict(qkv=a["qkv"][:, :500]), dict(hq=5), dict(hk=1), dict(D=128), dict(rot=32), dict(rot=16), dict(qw=a["qw"][:32]),
                dict(pos=a["pos"].long()), dict(pos=a["pos"][:2]), dict(start=a["start"][:1]), dict(table=a["table"][:0]),
                dict(out=torch.empty(3, 300, dtype=BF, device=DEV)), dict(out=torch.empty(3, 384, device=DEV)),
                dict(cache=PagedKVCache(2, 2, 128, 16, DEV, "int4")), dict(qkv=a["qkv"].t().contiguous().t()),
                dict(cos=a["cos"][:, :16]), dict(qkv=a["qkv"][:1].expand(3, -1))):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(qkv=c["qkv"]), dict(pos=c["pos"]), dict(cos=c["cos"])):
        with pytest.raises((RuntimeError, ValueError)):
            call(**bad)


def test_nothing_to_do(gpu_lib):
    from opendecider_amd import PagedKVCache, kernels
    e = lambda *s, dt=BF: torch.empty(*s, dtype=dt, device=DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    cache = PagedKVCache(0, 2, 64, 16, DEV, quantized="int4")
    assert kernels.paged_attn(e(0, 4, 64), e(0, 2, 64), e(0, 2, 64), cache, e(1, 0, dt=torch.int32), i32(0, 0), i32(0), 0.1).shape == (0, 4, 64)
    kernels.page_append(e(3, 2, 64), e(3, 2, 64), cache, e(0, 0, dt=torch.int32), i32(0), e(0, dt=torch.int32))
    k, v = kernels.page_read(cache, e(2, 0, dt=torch.int32), i32(5, 0), 7)
    assert k.shape == (2, 2, 7, 64) and not k.any() and not v.any()
    q, x = torch.randn(3, 4, 64, device=DEV).to(BF), torch.randn(3, 2, 64, device=DEV).to(BF)
    o = kernels.paged_attn(q, x, x, cache, e(1, 0, dt=torch.int32), i32(0, 3), i32(9), 0.1)
    assert torch.equal(o[0], x[0].repeat_interleave(2, 0))
    w, t = torch.ones(64, device=DEV).to(BF), torch.ones(4, 32, device=DEV).to(BF)
    for N, B in ((0, 1), (3, 0), (3, 1)):  # no rows; no sequences; no pages: the rows are normed and rotated all the same
        qkv = torch.randn(N, 8 * 64, device=DEV).to(BF)
        before = qkv.clone()
        kernels.qk_norm_rope_page_append(qkv, 4, 2, 64, w, w, t, t, torch.zeros(N, dtype=torch.int32, device=DEV), 1e-6, cache,
                                         e(B, 0, dt=torch.int32), torch.arange(B + 1, dtype=torch.int32, device=DEV) * N, torch.zeros(B, dtype=torch.int32, device=DEV))
        kernels.qk_norm_rope(before, 4, 2, 64, w, w, t, t, torch.zeros(N, dtype=torch.int32, device=DEV), 1e-6)
        assert torch.equal(qkv, before)


@pytest.mark.parametrize("quantized", ["int4", "int8", False])
@pytest.mark.parametrize("N,cols", [(3, 0), (200, 0), (200, 3)])
def test_no_pages_at_all(gpu_lib, N, cols, quantized):
    """A pool without pages, tables without columns: the tokens see each other, few slots and many."""
    from opendecider_amd import PagedKVCache, kernels
    cache = PagedKVCache(0, 2, 64, 16, DEV, quantized=quantized)
    x = torch.randn(N, 2, 64, generator=torch.Generator().manual_seed(N)).to(BF)
    q = torch.zeros(N, 4, 64, dtype=BF, device=DEV)
    out = torch.full((N, 4, 64), 5.0, dtype=BF, device=DEV)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    table = torch.zeros(1, cols, dtype=torch.int32, device=DEV)
    kernels.paged_attn(q, gpu(x), gpu(x), cache, table, i32(0, N), i32(9), 0.1, out=out)
    mean = x.double().cumsum(0) / torch.arange(1, N + 1)[:, None, None]
    size = x.double().abs().cumsum(0) / torch.arange(1, N + 1)[:, None, None]
    bound = 2.0 ** -8 * mean.abs() + (2.0 ** -8 + 2.0 ** -22 * (N + 16)) * size  # the output's rounding, the probabilities'
    assert ((out.double().cpu() - mean.repeat_interleave(2, 1)).abs() <= bound.repeat_interleave(2, 1)).all()


def test_read_refusals(gpu_lib):
    from opendecider_amd import PagedKVCache, kernels
    cache = PagedKVCache(2, 2, 128, 16, DEV, quantized="int4")
    tab, n = torch.zeros(1, 2, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    for dt in (torch.int8, torch.uint8, torch.float16):
        with pytest.raises(TypeError):
            kernels.page_read(cache, tab, n, 4, dtype=dt)


# ------------------------------------------------------------------------------------------------ together
def test_a_graph_of_a_step(gpu_lib):
    """A decode step (norm, rotate and write; attend; read; advance the lengths) captured once and replayed: every replay equals
    the eager step."""
    from opendecider_amd import kernels
    c = rope_case(50, [1, 1, 1], [30, 100, 0], 4, 2, 128, 128, False, pad=0)
    used = set(c["table"].flatten().tolist())
    table = torch.full((3, c["table"].shape[1] + 1), -1, dtype=torch.int32)
    table[:, :-1] = c["table"]
    free = [p for p in range(c["pages"][0].shape[0]) if p not in used]
    for b in range(3):
        table[b, int((c["table"][b] >= 0).sum())] = free[b]
    c["table"] = table
    tab, start, one, w = gpu(table), gpu(c["start"]), torch.ones(3, dtype=torch.int32, device=DEV), 6 * 128
    qkv, tables = gpu(c["qkv"]), [gpu(c[x]) for x in ("qw", "kw", "cos", "sin")]

    def step(cache, ctx):
        x = qkv.clone()
        kernels.qk_norm_rope_page_append(x, 4, 2, 128, *tables, ctx, 1e-6, cache, tab, start, ctx)
        q, k, v = (y.view(3, -1, 128) for y in x.split([512, 256, 256], 1))
        o = kernels.paged_attn(q, k, v, cache, tab, start, ctx, 128 ** -0.5, max_new=1, max_ctx=200)
        ctx.add_(one)
        return o, *kernels.page_read(cache, tab, ctx, 128)

    eager, ectx = cache_of(c), gpu(c["ctx"])
    cap, cctx = cache_of(c), gpu(c["ctx"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache_of(c), gpu(c["ctx"]))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cap, cctx)
    for r in range(5):
        qkv.copy_(torch.randn(qkv.shape, generator=torch.Generator().manual_seed(r)).to(BF))
        want = step(eager, ectx)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), r
        assert torch.equal(cap.k, eager.k) and torch.equal(cap.v_scale, eager.v_scale) and torch.equal(cctx, ectx)


def test_a_graph_of_a_long_chunk(gpu_lib):
    """The image, the tiles and the merge of splits captured, replayed with new contents between eager calls."""
    from opendecider_amd import kernels
    c = make(19, [70, 40, 30], [500, 3000, 1024], 4, 1, 256, page=64, pad=6000)
    cache, meta = cache_of(c), (gpu(c["table"]), gpu(c["start"]), gpu(c["ctx"]), c["scale"])
    q, k, v = gpu(c["q"]), gpu(c["k"]), gpu(c["v"])
    out = torch.zeros_like(q)
    call = lambda o: kernels.paged_attn(q, k, v, cache, *meta, max_ctx=3000, out=o)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(torch.zeros_like(q))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(out)
    for seed in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)))
        cache.v_scale.mul_(1.5)
        meta[2].copy_(torch.tensor([500 - seed, 3000 - 700 * seed, 1024 - 64 * seed]))
        graph.replay()
        want = call(torch.zeros_like(q))
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.isfinite(out.float()).all() and out[:140].any(2).all()


def test_on_another_stream(gpu_lib):
    for new in ([50, 2], [1, 1]):
        c = make(51, new, [300, 20])
        want, _ = run_attn(c)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got, _ = run_attn(c)
        side.synchronize()
        assert torch.equal(got, want)


def check_calls(calls):
    for (q, k, v, pages, table, start, ctx, scale), kw, out in calls:
        cpu = lambda x: None if x is None else x.cpu()
        c = dict(q=q.cpu(), k=k.cpu(), v=v.cpu(), pages=[cpu(pages[0]), cpu(pages[1])], scales=[cpu(pages[2]), cpu(pages[3])],
                 table=table.cpu(), start=start.cpu(), ctx=ctx.cpu(), scale=scale, row_begin=cpu(kw["row_begin"]))
        lse = op.attention(c["q"], c["k"], c["v"], (*c["pages"], *c["scales"]), c["table"], c["start"], c["ctx"], scale, c["row_begin"])[1]
        check_attn(c, out, lse)


def test_decoder_over_4_bit_pages(gpu_lib, monkeypatch):
    """States in 4 bits grow in chunks of any length, end, and score their options. Every attention call is right for its own
    inputs; layer 0's pages hold what pack_int4 makes of the keys and values of the bf16 states for the same tokens."""
    from opendecider_amd import kernels, pack_int4, unpack_int4
    from opendecider_amd.decoder import DecoderConfig, random_decoder
    dec = random_decoder(DecoderConfig(**tp.CFG), seed=1, max_pos=512)
    g = torch.Generator().manual_seed(2)
    tok = lambda n: torch.randint(0, 300, (n,), generator=g).to(DEV)
    states, dense = (dec.new_paged_states(3, n_pages=15, max_tokens=400, page=32, quantized=x) for x in ("int4", False))
    calls = tp.recorded(monkeypatch, "paged_attn")
    for counts in ([70, 0, 5], [1, 1, 1], [0, 40, 300]):
        ids = tok(sum(counts))
        h = dec.extend(ids, counts, states)
        assert h.shape == (sum(counts), 256) and torch.isfinite(h.float()).all()
        n = len(calls)
        dec.extend(ids, counts, dense)
        del calls[n:]
    ids = torch.randint(0, 300, (3, 4, 5), generator=g).to(DEV)
    lp = dec.score_paged(ids, states)
    assert lp.shape == (3, 5) and torch.allclose(lp.exp().sum(1), torch.ones(3, device=DEV), atol=1e-5)
    check_calls(calls)
    for x, y in zip(states.read(0, torch.float32), dense.read(0)):
        assert torch.equal(x.cpu(), unpack_int4(*pack_int4(y.cpu())) + 0.0)
    with pytest.raises(MemoryError):
        dec.extend(tok(50), [50, 0, 0], states)
    states.release(2)
    dec.extend(tok(80), [50, 0, 30], states)
    assert states.lengths == [121, 41, 30] and torch.isfinite(dec.score_paged(ids, states)).all()
