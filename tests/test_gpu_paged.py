"""The paged K/V cache on the GPU against its float64 restatement (oracle/paged.py): writing, reading back and attention at
the sizes, masks and layouts where they can go wrong, their refusals, and graphs.

Bounds of the attention. With seen keys j, probabilities p_j and A_d = sum_j p_j |v_jd|, an output differs from the float64
one by
  * its own rounding to bf16, 2^-8 |o|;
  * the probabilities' rounding for the P.V product, at most 2^-8 A (bf16; 2^-11 where they are fp16), and where int8
    values are scaled in fp16 theirs, 2^-11 A;
  * the scores' error e, which moves every p_j by at most a factor exp(+-2 e): 2 e A. e is at most 2^-11 S (int8 rows scaled in
    fp16; none for the others) + 2^-24 (D + 8) S (fp32 sums), S = max_j scale sum_d |q_d k_jd|;
  * the fp32 sums over T keys and exp2 / log2 of a few ulps: 2^-22 (T + 16) A is far above them;
  * numbers too small for their format. Probabilities are held relative to a maximum of at least 1, so their sum is at least
    1; one that is lost (below 2^-126 in fp32 and bf16; half a subnormal step in fp16, 2^-25, is 2^-32 of the maximum where
    fp16 probabilities are kept 2^7 above it) costs at most 2^-32 |v_jd|, and an int8 value below fp16's subnormals in a frame
    whose largest scale is above 2^7 at most 2^-32 of that scale: 2^-31 sum_j max_d |v_jd| together.
An LSE differs by e and a few fp32 ulps of it and of the max.
"""
import math

import pytest
import torch

from oracle import paged as op

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF = torch.bfloat16


def make(seed, new, ctx, heads=8, kv=2, d=128, page=16, int8=True, rows=0, pad=0, spare=2, mag=1.0):
    """A packed ragged batch: CPU tensors of the pages, the table, the tokens (pad rows behind the last sequence)."""
    g = torch.Generator().manual_seed(seed)
    B = len(new)
    per = [-(-(max(t, 0) + n) // page) for n, t in zip(new, ctx)]
    cols = max(per + [1]) + 1
    n_pages = sum(per) + spare
    order = torch.randperm(n_pages, generator=g)
    table = torch.full((B, cols), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    N = sum(new) + pad
    c = dict(table=table, start=torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32),
             ctx=torch.tensor(ctx, dtype=torch.int32), scale=d ** -0.5, row_begin=None)
    c["q"] = (torch.randn(N, heads, d, generator=g) * mag).to(BF)
    c["k"], c["v"] = (torch.randn(N, kv, d, generator=g).to(BF) for _ in range(2))
    c["pages"] = []
    for _ in range(2):
        x = torch.randn(n_pages, kv, page, d, generator=g).to(BF)
        # rows of very different sizes: scales over several powers of two
        x = x * torch.exp2(torch.randint(-3, 4, (n_pages, kv, page, 1), generator=g).float()).to(BF)
        c["pages"].append(x)
    c["scales"] = [None, None]
    if int8:
        from oracle.quant import quantize_rows
        qs = [quantize_rows(x) for x in c["pages"]]
        c["pages"], c["scales"] = [a for a, _ in qs], [s[..., 0].contiguous() for _, s in qs]
    if rows:
        local = torch.cat([torch.arange(n) for n in new] + [torch.zeros(pad, dtype=torch.long)])
        c["row_begin"] = (local // rows * rows).to(torch.int32)
    return c


def gpu(x):
    return None if x is None else x.to(DEV)


def cache_of(c):
    from opendecider_amd import PagedKVCache
    return PagedKVCache.from_tensors(*(gpu(x) for x in c["pages"]), *(gpu(x) for x in c["scales"]))


def run_attn(c, cache=None, own=True, **kw):
    from opendecider_amd import kernels
    return kernels.paged_attn(gpu(c["q"]), gpu(c["k"]) if own else None, gpu(c["v"]) if own else None,
                              cache_of(c) if cache is None else cache, gpu(c["table"]), gpu(c["start"]), gpu(c["ctx"]),
                              c["scale"], row_begin=gpu(c["row_begin"]), return_lse=True, **kw)


def check_attn(c, out, lse, own=True, rows=None):
    ref, rl, mean, size, total = op.attention(c["q"], c["k"] if own else None, c["v"] if own else None, (*c["pages"], *c["scales"]),
                                       c["table"], c["start"], c["ctx"], c["scale"], c["row_begin"])
    out, lse = out.double().cpu(), lse.double().cpu()
    live = ~rl.isnan()
    D, T = c["q"].shape[2], int(c["ctx"].clamp_min(0).max()) + c["q"].shape[0]
    e = (2.0 ** -11 if c["scales"][0] is not None else 0.0) * size + 2.0 ** -24 * (D + 8) * size
    bound = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -11 + 2 * e[..., None] + 2.0 ** -22 * (T + 16)) * 1.02 * mean + \
        2.0 ** -31 * total[..., None]
    bad = (out - ref).abs() > bound
    assert not bad[live].any(), f"{int(bad[live].sum())} of {int(live.sum()) * D}: worst {((out - ref).abs() / bound.clamp_min(1e-300))[live].max()}"
    assert not out[live].isnan().any()
    none = live & (rl == -math.inf)
    assert (out[none] == 0).all() and (lse[none] == -math.inf).all()
    some = live & ~none
    lb = e + 2.0 ** -20 * (1 + rl.abs() + size)
    assert ((lse - rl).abs() <= lb)[some].all(), f"lse off by {((lse - rl).abs() / lb)[some].max()} of its bound"


SHAPES = [  # new tokens, cached tokens
    ([1], [0]), ([1], [1]), ([1, 1, 1], [15, 16, 17]), ([1, 1], [700, 3]), ([2, 0, 3], [5, 9, 0]), ([0, 4, 0, 1, 0], [3, 0, 40, 64, 7]),
    ([5], [63]), ([33, 64, 7], [64, 65, 130]), ([130], [200]), ([70, 1, 150], [0, 300, 31]), ([300], [0]),
]


@pytest.mark.parametrize("d,heads,kv", [(64, 4, 4), (128, 8, 2), (256, 4, 1), (128, 7, 1)])
@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention(gpu_lib, shape, int8, d, heads, kv):
    new, ctx = SHAPES[shape]
    c = make(shape, new, ctx, heads, kv, d, page=[16, 64, 32][shape % 3], int8=int8)
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,ctx,rows", [([24, 40, 1], [50, 0, 129], 8), ([37], [70], 5), ([150, 90], [33, 64], 30), ([260], [10], 100)])
def test_option_rows(gpu_lib, new, ctx, rows, d, int8):
    c = make(7, new, ctx, 8, 2, d, page=32, int8=int8, rows=rows)
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("new,ctx", [([3, 1], [0, 40]), ([100, 60], [0, 90]), ([1, 1, 1], [0, 700, -5])])
@pytest.mark.parametrize("int8", [True, False])
def test_cached_tokens_only(gpu_lib, new, ctx, int8):
    """Without k and v the tokens see the cache only: those of an empty state see nothing."""
    c = make(3, new, ctx, int8=int8)
    check_attn(c, *run_attn(c, own=False), own=False)


@pytest.mark.parametrize("new", [[6, 4], [90, 70]])
def test_any_row_begin(gpu_lib, new):
    """row_begin in any order: negative ones are 0, one past the token leaves it the cache (and of an empty state nothing)."""
    c = make(5, new, [0, 45])
    g = torch.Generator().manual_seed(1)
    c["row_begin"] = torch.randint(-3, max(new) + 5, (sum(new),), generator=g).to(torch.int32)
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("new,ctx", [([1, 1, 1, 1], [700, 90, 40, 33]), ([40, 1, 100], [200, 90, 33])])
@pytest.mark.parametrize("int8", [True, False])
def test_no_pages_and_short_tables(gpu_lib, new, ctx, int8):
    """Entries outside the pool hold no keys; cached tokens past the table's end do not exist."""
    c = make(11, new, ctx, int8=int8)
    n = c["pages"][0].shape[0]
    c["table"][0, 1], c["table"][0, 3], c["table"][1, 0], c["table"][-1, 0], c["table"][-1, 1] = -1, n, 2 ** 31 - 1, -7, n + 5
    check_attn(c, *run_attn(c))
    c["ctx"][1] = 10 ** 6
    c["table"] = c["table"][:, :4].contiguous()
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("new", [[3, 2], [80, 70]])
def test_rows_of_no_sequence_stay(gpu_lib, new):
    c = make(2, new, [20, 50], pad=9)
    out = torch.full(c["q"].shape, 7.0, dtype=BF, device=DEV)
    c["start"] = c["start"] + 2  # two rows ahead of the first sequence, seven behind the last
    got, lse = run_attn(c, out=out)
    assert got is out
    N = sum(new)
    assert (out[:2] == 7).all() and (out[2 + N:] == 7).all()
    check_attn(c, out, lse)


@pytest.mark.parametrize("new,ctx", [([2, 1], [30, 40]), ([100], [70])])
@pytest.mark.parametrize("int8", [True, False])
def test_what_is_masked_does_not_matter(gpu_lib, new, ctx, int8):
    """NaN and infinities where no token looks: rows of the pages past the cached tokens, other pages, tokens of other
    rows or later ones, pad rows."""
    c = make(4, new, ctx, int8=int8, pad=5, rows=1)
    want, wl = run_attn(c)
    used = torch.zeros(c["pages"][0].shape[0], 16, dtype=torch.bool)
    for b, t in enumerate(ctx):
        for j in range(t):
            used[c["table"][b, j // 16], j % 16] = True
    for i in range(2):
        bad = float("nan") if i else float("inf")
        if int8:
            c["scales"][i] = torch.where(used[:, None], c["scales"][i], bad)
        else:
            c["pages"][i] = torch.where(used[:, None, :, None], c["pages"][i], bad)
    N = sum(new)
    c["k"][N:], c["v"][N:], c["q"][N:] = float("nan"), float("inf"), float("nan")
    got, gl = run_attn(c)
    assert torch.equal(got[:N], want[:N]) and torch.equal(gl[:N], wl[:N])
    # each token sees itself only (rows of one): a bad one changes its own outputs and no others
    c["k"][1, 0], c["v"][1, 0] = float("nan"), float("inf")
    got, gl = run_attn(c)
    keep = torch.arange(c["q"].shape[0]) != 1
    keep[N:] = False
    assert torch.equal(got[keep.to(DEV)], want[keep.to(DEV)])
    assert got[1].isnan()[: c["q"].shape[1] // 2].all() and not got[1].isnan()[c["q"].shape[1] // 2:].any()
    # causal: a later token's NaN and infinities change no earlier token
    c["row_begin"] = None
    c["k"][1, 0], c["v"][1, 0] = 0.5, 0.5
    want, _ = run_attn(c)
    late = N // 2 if len(new) == 1 else new[0] - 1
    c["k"][late], c["v"][late, :, ::2], c["v"][late, :, 1::2] = float("nan"), float("inf"), float("nan")
    got, _ = run_attn(c)
    assert torch.equal(got[:late], want[:late])


def test_infinite_values_are_seen(gpu_lib):
    """An infinite value that a token does see arrives, also where other tokens of its tile do not see it."""
    c = make(6, [70], [20], heads=2, kv=1, d=64, int8=False)
    c["v"][30, 0, 5] = float("inf")
    out, _ = run_attn(c)
    assert torch.isfinite(out[:30].float()).all() and (out[30:, :, 5] == float("inf")).all()
    rest = torch.cat([out[30:, :, :5], out[30:, :, 6:]], 2)
    assert torch.isfinite(rest.float()).all()


@pytest.mark.parametrize("new,ctx", [([1, 1], [600, 90]), ([90], [300])])
@pytest.mark.parametrize("k_exp,v_exp", [(-100, 60), (60, -100), (0, -20), (20, 100)])
def test_sizes_of_the_rows(gpu_lib, new, ctx, k_exp, v_exp):
    """Scales far from 1 in the pages, queries that bring the scores back to their usual size."""
    c = make(8, new, ctx, heads=4, kv=1)
    c["scales"][0] = c["scales"][0] * 2.0 ** k_exp
    c["scales"][1] = c["scales"][1] * 2.0 ** v_exp
    c["q"] = (c["q"].float() * 2.0 ** -k_exp).to(BF)
    c["k"] = (c["k"].float() * 2.0 ** k_exp).to(BF)
    c["v"] = (c["v"].float() * 2.0 ** v_exp).to(BF)
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("new,ctx", [([1, 1], [1000, 64]), ([64, 90], [400, 10])])
@pytest.mark.parametrize("int8", [True, False])
def test_sharp_scores(gpu_lib, new, ctx, int8):
    c = make(9, new, ctx, int8=int8, mag=12.0)
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("new", [[1, 1, 1], [3, 60, 1]])
def test_bounds_do_not_change_what_is_computed(gpu_lib, new):
    """max_new and max_ctx size the work; wrong ones still give the right result."""
    c = make(10, new, [300, 1100, 17])
    for mn in (1, max(new), None):
        for mc in (0, 64, 1100, 10 ** 6, None):
            check_attn(c, *run_attn(c, max_new=mn, max_ctx=mc))


def test_strides_and_alignment(gpu_lib):
    """Views of a fused projection, heads before tokens, rows at odd addresses, an output of any strides."""
    from opendecider_amd import kernels
    c = make(12, [40, 3], [20, 90])
    want, wl = run_attn(c)
    N, Hq, D = c["q"].shape
    cache, meta = cache_of(c), (gpu(c["table"]), gpu(c["start"]), gpu(c["ctx"]), c["scale"])
    fused = torch.cat([c[x].reshape(N, -1) for x in "qkv"], 1).to(DEV)
    q, k, v = fused.split([Hq * D, 2 * D, 2 * D], 1)
    assert torch.equal(kernels.paged_attn(q.view(N, Hq, D), k.view(N, 2, D), v.view(N, 2, D), cache, *meta), want)
    qt = gpu(c["q"]).transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(N * 2 * D + 1, dtype=BF, device=DEV)[1:].view(N, 2, D).copy_(gpu(c["k"]))
    vs = gpu(c["v"]).repeat_interleave(2, 2)[:, :, ::2]
    wide = torch.full((N, Hq, D + 8), 3.0, dtype=BF, device=DEV)
    out = kernels.paged_attn(qt, odd, vs, cache, *meta, out=wide[..., :D])
    assert torch.equal(out, want) and (wide[..., D:] == 3).all()
    odd_out = torch.zeros(N, Hq, D + 1, dtype=BF, device=DEV)[..., 1:]
    assert torch.equal(kernels.paged_attn(qt, odd, vs, cache, *meta, out=odd_out), want) and torch.equal(odd_out, want)
    table = torch.full((2, c["table"].shape[1] + 3), -1, dtype=torch.int32)
    table[:, :-3] = c["table"]
    assert torch.equal(kernels.paged_attn(qt, odd, vs, cache, table.to(DEV)[:, :-3], *meta[1:]), want)


@pytest.mark.parametrize("new,ctx", [([1] * 5, [2500, 3, 900, 0, 64]), ([50, 3], [900, 64])])
def test_same_calls_same_bits_and_order(gpu_lib, new, ctx):
    """The result does not change from call to call, nor with where a sequence stands in the batch."""
    c = make(13, new, ctx)
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


# ------------------------------------------------------------------------ the same, by the kernel for many slots
MANY = [([20], [0]), ([9, 17, 3], [70, 0, 300]), ([33, 64, 7], [64, 65, 130]), ([130], [200]), ([70, 1, 150], [0, 300, 31]),
        ([300], [0]), ([1, 1], [700, 3]), ([0, 12, 0], [9, 500, 0])]


@pytest.fixture(params=["rows", "table"])
def tiled(request, monkeypatch):
    """Small calls that the library takes for large ones, by rows of no sequence or by a table with room for 2^20 tokens."""
    small = make

    def large(*a, **kw):
        c = small(*a, **dict(kw, pad=kw.get("pad", 0) + (1100 if request.param == "rows" else 0)))
        if request.param == "table":
            wide = torch.full((c["table"].shape[0], 2 ** 20 // c["pages"][0].shape[2]), -1, dtype=torch.int32)
            wide[:, :c["table"].shape[1]] = c["table"]
            c["table"] = wide
        return c

    monkeypatch.setitem(globals(), "make", large)
    return request.param


@pytest.mark.parametrize("d,heads,kv", [(64, 4, 4), (128, 8, 2), (256, 4, 1), (128, 7, 1)])
@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("shape", range(len(MANY)))
def test_many_slots(gpu_lib, tiled, shape, int8, d, heads, kv):
    new, ctx = MANY[shape]
    c = make(shape, new, ctx, heads, kv, d, page=[16, 64, 32][shape % 3], int8=int8)
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new,ctx,rows", [([24, 40, 1], [50, 0, 129], 8), ([150, 90], [33, 64], 30), ([260], [10], 100)])
def test_many_slots_option_rows(gpu_lib, tiled, new, ctx, rows, d, int8):
    test_option_rows(gpu_lib, new, ctx, rows, d, int8)


@pytest.mark.parametrize("int8", [True, False])
def test_many_slots_masks(gpu_lib, tiled, int8):
    test_cached_tokens_only(gpu_lib, [100, 60], [0, 90], int8)
    test_no_pages_and_short_tables(gpu_lib, [40, 1, 100], [200, 90, 33], int8)
    test_what_is_masked_does_not_matter(gpu_lib, [100], [70], int8)
    test_sharp_scores(gpu_lib, [64, 90], [400, 10], int8)


def test_many_slots_values(gpu_lib, tiled):
    c = make(6, [70], [20], heads=2, kv=1, d=64, int8=False)
    c["v"][30, 0, 5] = float("inf")
    out, _ = run_attn(c)
    assert torch.isfinite(out[:30].float()).all() and (out[30:70, :, 5] == float("inf")).all()
    assert torch.isfinite(torch.cat([out[30:70, :, :5], out[30:70, :, 6:]], 2).float()).all()
    for k_exp, v_exp in [(-100, 60), (60, -100), (0, -20), (20, 100)]:
        test_sizes_of_the_rows(gpu_lib, [90], [300], k_exp, v_exp)
    test_bounds_do_not_change_what_is_computed(gpu_lib, [3, 60, 1])


@pytest.fixture
def imaged(monkeypatch):
    """Small calls with the bounds of large ones: their int8 pages go through the image (rows of no sequence, a table with room
    for 2^16 tokens)."""
    small = make

    def large(*a, **kw):
        c = small(*a, **dict(kw, pad=kw.get("pad", 0) + 1100))
        B, (_, kv, page, d) = c["table"].shape[0], c["pages"][0].shape
        wide = torch.full((B, 2 ** 16 // page), -1, dtype=torch.int32)
        wide[:, :c["table"].shape[1]] = c["table"]
        c["table"] = wide
        if c["scales"][0] is not None:
            from opendecider_amd import kernels
            N, heads, _ = c["q"].shape
            dev = torch.device(DEV, torch.cuda.current_device())
            assert kernels.paged_attn_workspace_floats(B, N, heads, kv, d, N, 2 ** 16, dev) > B * kv * 2 ** 16 * d
        return c

    monkeypatch.setitem(globals(), "make", large)


@pytest.mark.parametrize("d,heads,kv", [(64, 4, 4), (128, 8, 2), (256, 4, 1), (128, 7, 1)])
@pytest.mark.parametrize("shape", range(len(MANY)))
def test_image(gpu_lib, imaged, shape, d, heads, kv):
    new, ctx = MANY[shape]
    c = make(shape, new, ctx, heads, kv, d, page=[16, 64, 32][shape % 3])
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_image_option_rows(gpu_lib, imaged, d):
    test_option_rows(gpu_lib, [150, 90], [33, 64], 30, d, True)


def test_image_masks_and_values(gpu_lib, imaged):
    test_cached_tokens_only(gpu_lib, [100, 60], [0, 90], True)
    c = make(11, [40, 1, 100], [200, 90, 33])
    n = c["pages"][0].shape[0]
    c["table"][0, 1], c["table"][0, 3], c["table"][1, 0], c["table"][2, 0], c["table"][2, 1] = -1, n, 2 ** 31 - 1, -7, n + 5
    check_attn(c, *run_attn(c))
    test_what_is_masked_does_not_matter(gpu_lib, [100], [70], True)
    test_sharp_scores(gpu_lib, [64, 90], [400, 10], True)
    for k_exp, v_exp in [(-100, 60), (60, -100), (0, -20), (20, 100)]:
        test_sizes_of_the_rows(gpu_lib, [90], [300], k_exp, v_exp)


@pytest.mark.parametrize("d,heads,kv,pad", [(256, 4, 1, 6000), (128, 8, 1, 24000)])
def test_image_of_some(gpu_lib, d, heads, kv, pad):
    """max_ctx below one state's length: the others go through the image, that one as it is."""
    c = make(15, [70, 40, 30], [500, 3000, 1024], heads, kv, d, page=64, pad=pad)
    from opendecider_amd import kernels
    dev = torch.device(DEV, torch.cuda.current_device())
    assert kernels.paged_attn_workspace_floats(3, pad + 140, heads, kv, d, pad + 140, 1024, dev) > 3 * kv * 1024 * d
    check_attn(c, *run_attn(c, max_ctx=1024))


def test_many_slots_same_bits(gpu_lib):
    test_same_calls_same_bits_and_order(gpu_lib, [300, 3], [900, 64])
    test_same_calls_same_bits_and_order(gpu_lib, [8, 3, 5], [9, 900, 64])  # two columns of 16


@pytest.mark.parametrize("new", [[7, 8, 3], [60, 2]])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_infinite_values_of_new_tokens(gpu_lib, new, d):
    """Each later token sees an infinite value, and nothing else is infinite: bit for bit the rest of the outputs."""
    c = make(14, new, [40, 0, 9][:len(new)], heads=4, kv=1, d=d)
    want, _ = run_attn(c)
    c["v"][2, 0, 5], c["v"][new[0], 0, d - 1] = float("inf"), float("-inf")
    out, _ = run_attn(c)
    hit = torch.zeros(out.shape, dtype=torch.bool)
    hit[2:new[0], :, 5] = True
    hit[new[0]:new[0] + new[1], :, d - 1] = True
    hit = hit.to(DEV)
    assert torch.equal(out[~hit], want[~hit])
    assert (out[2:new[0], :, 5] == float("inf")).all() and (out[new[0]:new[0] + new[1], :, d - 1] == float("-inf")).all()


@pytest.mark.parametrize("new,pad", [(2, 0), (60, 0), (60, 6000)])
def test_one_table_row_for_all(gpu_lib, new, pad):
    """An expanded table: every sequence reads the same pages."""
    from opendecider_amd import kernels
    c = make(16, [new] * 3, [500, 300, 500], 8, 2, pad=pad, page=32)
    row = gpu(c["table"][:1])
    c["table"] = c["table"][:1].repeat(3, 1)
    want, wl = run_attn(c)
    cache = cache_of(c)
    got, gl = kernels.paged_attn(gpu(c["q"]), gpu(c["k"]), gpu(c["v"]), cache, row.expand(3, -1), gpu(c["start"]), gpu(c["ctx"]),
                                 c["scale"], return_lse=True)
    N = 3 * new
    assert torch.equal(got[:N], want[:N]) and torch.equal(gl[:N], wl[:N])
    for x, y in zip(kernels.page_read(cache, row.expand(3, -1), gpu(c["ctx"]), 500),
                    kernels.page_read(cache, gpu(c["table"]), gpu(c["ctx"]), 500)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("int8", [True, False])
def test_many_sequences(gpu_lib, int8):
    """More sequences than are put in order by their lengths."""
    new = [(37 * b) % 50 for b in range(70)]
    c = make(17, new, [(61 * b) % 300 for b in range(70)], 8, 2, int8=int8, page=32)
    check_attn(c, *run_attn(c, max_new=max(new), max_ctx=300))


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("new,pad", [(1, 0), (70, 1100), (70, 6000)])
def test_a_pool_past_32_bits(gpu_lib, int8, new, pad):
    """Pages behind the first 2^31 values of the pool: bit for bit what the same pages do in a small one."""
    from opendecider_amd import PagedKVCache, kernels
    c = make(18, [new, new], [900, 333], 8, 2, page=64, int8=int8, pad=pad)
    want, wl = run_attn(c)
    n, kv, page, d = c["pages"][0].shape
    total = 2 ** 31 // (kv * page * d) + n
    big = []
    for x in (*c["pages"], *c["scales"]):
        big.append(None if x is None else torch.zeros(total, *x.shape[1:], dtype=x.dtype, device=DEV))
        if x is not None:
            big[-1][-n:] = gpu(x)
    cache = PagedKVCache.from_tensors(*big)
    table = torch.where(c["table"] >= 0, c["table"] + (total - n), -1).to(torch.int32)
    got, gl = run_attn(dict(c, table=table), cache=cache)
    N = 2 * new
    assert torch.equal(got[:N], want[:N]) and torch.equal(gl[:N], wl[:N])
    args = gpu(c["start"]), gpu(c["ctx"])
    small = cache_of(c)
    kernels.page_append(gpu(c["k"]), gpu(c["v"]), cache, gpu(table), *args)
    kernels.page_append(gpu(c["k"]), gpu(c["v"]), small, gpu(c["table"]), *args)
    assert torch.equal(cache.k[-n:], small.k) and torch.equal(cache.v[-n:], small.v) and not cache.k[:-n].any()
    for x, y in zip(kernels.page_read(cache, gpu(table), args[1], 900), kernels.page_read(small, gpu(c["table"]), args[1], 900)):
        assert torch.equal(x, y)


# ------------------------------------------------------------------------------------------------ append, read
@pytest.mark.parametrize("d,kv", [(64, 1), (64, 5), (128, 2), (128, 8), (256, 3)])
@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_append(gpu_lib, shape, int8, d, kv):
    from opendecider_amd import kernels
    new, ctx = SHAPES[shape]
    c = make(20 + shape, new, ctx, kv, kv, d, page=[16, 32, 64][shape % 3], int8=int8, pad=3)
    c["k"][0] = 0.0
    cache = cache_of(c)
    kernels.page_append(gpu(c["k"]), gpu(c["v"]), cache, gpu(c["table"]), gpu(c["start"]), gpu(c["ctx"]))
    for i, (x, got, gs) in enumerate(((c["k"], cache.k, cache.k_scale), (c["v"], cache.v, cache.v_scale))):
        want, ws = op.append(c["pages"][i], c["scales"][i], x, c["table"], c["start"], c["ctx"])
        assert torch.equal(got.cpu(), want)
        assert ws is None or torch.equal(gs.cpu(), ws)


def test_append_many_sequences(gpu_lib):
    """More sequences than one level of the search takes, runs of empty ones, tokens without a page, padding around."""
    from opendecider_amd import kernels
    g = torch.Generator().manual_seed(1)
    new = torch.randint(0, 3, (300,), generator=g).tolist()
    new[100:180] = [0] * 80
    ctx = torch.randint(0, 40, (300,), generator=g).tolist()
    c = make(30, new, ctx, 1, 1, 64, pad=6)
    c["start"] = c["start"] + 4
    c["table"][5], c["table"][7] = -1, c["pages"][0].shape[0]
    c["ctx"][9], c["ctx"][11] = -3, 10 ** 6
    cache = cache_of(c)
    kernels.page_append(gpu(c["k"]), gpu(c["v"]), cache, gpu(c["table"]), gpu(c["start"]), gpu(c["ctx"]))
    want, ws = op.append(c["pages"][0], c["scales"][0], c["k"], c["table"], c["start"], c["ctx"])
    assert torch.equal(cache.k.cpu(), want) and torch.equal(cache.k_scale.cpu(), ws)
    check_attn(c, *run_attn(c))


def test_append_takes_what_the_quantizer_takes(gpu_lib):
    """NaN and infinite rows, zeros and subnormals: the bytes of the rectangular cache's append."""
    from opendecider_amd import Int8KVCache, kernels
    c = make(31, [6], [0], 2, 2, 128)
    c["k"][0, 0, 3], c["k"][1], c["k"][2, 1, 0], c["k"][3], c["k"][4] = float("nan"), float("inf"), -float("inf"), 0.0, 1e-39
    cache, flat = cache_of(c), Int8KVCache(1, 2, 128, 6, DEV)
    kernels.page_append(gpu(c["k"]), gpu(c["v"]), cache, gpu(c["table"]), gpu(c["start"]), gpu(c["ctx"]))
    flat.append(gpu(c["k"]).transpose(0, 1)[None])
    k, v = kernels.page_read(cache, gpu(c["table"]), torch.tensor([6], dtype=torch.int32, device=DEV), 6, dtype=torch.int8)
    assert torch.equal(k.q, flat.q) and torch.equal(k.scale[..., 0].nan_to_num(7.0), flat.scale.nan_to_num(7.0))


@pytest.mark.parametrize("d,kv", [(64, 3), (128, 2), (256, 1)])
@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("dtype", [BF, torch.float32, torch.int8])
def test_read(gpu_lib, dtype, int8, d, kv):
    from opendecider_amd import kernels
    if dtype == torch.int8 and not int8:
        pytest.skip("bf16 pages hold no int8 rows")
    c = make(40, [0] * 6, [33, 0, 1, 64, 700, -4], kv, kv, d, int8=int8)
    c["table"][4, 2], c["table"][3, 0] = -1, c["pages"][0].shape[0]
    for T in (0, 1, 40, 800):
        got = kernels.page_read(cache_of(c), gpu(c["table"]), gpu(c["ctx"]), T, dtype=dtype)
        for i in range(2):
            rows, sc, _ = op.read(c["pages"][i], c["scales"][i], c["table"], c["ctx"], T)
            if dtype == torch.int8:
                assert torch.equal(got[i].q.cpu(), rows) and torch.equal(got[i].scale[..., 0].cpu(), sc)
            else:
                want = (rows.float() * sc[..., None] if int8 else rows.float()).to(dtype)
                assert torch.equal(got[i].cpu(), want)


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("int8", [True, False])
def test_a_graph_of_the_three(gpu_lib, int8):
    """A decode step (attend, append, advance the lengths) captured once and replayed: every replay equals the eager step."""
    from opendecider_amd import kernels
    c = make(50, [1, 1, 1], [30, 100, 0], int8=int8, spare=12)
    used, cols = int((c["table"] >= 0).sum()), c["table"].shape[1] + 1
    table = torch.full((3, cols), -1, dtype=torch.int32)
    table[:, :-1] = c["table"]
    free = [p for p in range(c["pages"][0].shape[0]) if p not in set(c["table"].flatten().tolist())]
    for b in range(3):  # a page more for each
        table[b, int((c["table"][b] >= 0).sum())] = free[b]
    assert used and len(free) >= 3
    tab, start, one = gpu(table), gpu(c["start"]), torch.ones(3, dtype=torch.int32, device=DEV)
    q, k, v = gpu(c["q"]), gpu(c["k"]), gpu(c["v"])

    def step(cache, ctx):
        o = kernels.paged_attn(q, k, v, cache, tab, start, ctx, c["scale"], max_new=1, max_ctx=200)
        kernels.page_append(k, v, cache, tab, start, ctx)
        kd, vd = kernels.page_read(cache, tab, ctx, 128)
        ctx.add_(one)
        return o, kd, vd

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
        for x, s in ((q, 1.0), (k, 1.0), (v, 1.0)):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(r)).to(BF))
        want = step(eager, ectx)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), r
        assert torch.equal(cap.k, eager.k) and torch.equal(cctx, ectx)


def test_on_another_stream(gpu_lib):
    c = make(51, [50, 2], [300, 20])
    want, _ = run_attn(c)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got, _ = run_attn(c)
    side.synchronize()
    assert torch.equal(got, want)


def test_a_graph_of_a_long_chunk(gpu_lib):
    """The image, the tiles and the merge of splits captured on a stream of their own, replayed with new contents between eager
    calls on another stream."""
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
        g = torch.Generator().manual_seed(seed)
        q.copy_(torch.randn(q.shape, generator=g))
        cache.v_scale.mul_(1.5)
        meta[2].copy_(torch.tensor([500 - seed, 3000 - 700 * seed, 1024 - 64 * seed]))
        graph.replay()
        want = call(torch.zeros_like(q))
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.isfinite(out.float()).all() and out[:140].any(2).all()


# ------------------------------------------------------------------------------------------------ in the decoder
CFG = dict(hidden=256, ffn=512, n_heads=8, n_kv_heads=2, head_dim=64, n_layers=2, vocab=300)


def recorded(monkeypatch, name):
    """Every call of a kernels function with its arguments and result, tensors copied."""
    from opendecider_amd import kernels
    calls, fn = [], getattr(kernels, name)
    keep = lambda x: x.clone() if isinstance(x, torch.Tensor) else x

    def wrap(*a, **kw):
        held = [keep(x) for x in a], {k: keep(v) for k, v in kw.items()}
        if name == "paged_attn":
            c = a[3]
            held[0][3] = [keep(x) for x in (c.k, c.v, c.k_scale, c.v_scale)]
        res = fn(*a, **kw)
        calls.append((*held, keep(res)))
        return res

    monkeypatch.setattr(kernels, name, wrap)
    return calls


def check_calls(calls):
    for (q, k, v, pages, table, start, ctx, scale), kw, out in calls:
        cpu = lambda x: None if x is None else x.cpu()
        c = dict(q=q.cpu(), k=k.cpu(), v=v.cpu(), pages=[cpu(pages[0]), cpu(pages[1])], scales=[cpu(pages[2]), cpu(pages[3])],
                 table=table.cpu(), start=start.cpu(), ctx=ctx.cpu(), scale=scale, row_begin=cpu(kw["row_begin"]))
        _, lse, _, _, _ = op.attention(c["q"], c["k"], c["v"], (*c["pages"], *c["scales"]), c["table"], c["start"], c["ctx"], scale,
                                       c["row_begin"])
        check_attn(c, out, lse)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("gated", [False, True])
def test_decoder_over_pages(gpu_lib, monkeypatch, quantized, gated):
    """Ragged states grow in chunks of any length, end, and score their options. Layer 0's inputs to the attention and the bytes
    in its pages equal the rectangular path's for the same tokens at the same positions; every attention call is right for
    its own inputs (the rest of a layer is the rectangular path's code); a state that another one's end made room for works."""
    from opendecider_amd import kernels
    from opendecider_amd.decoder import DecoderConfig, random_decoder
    dec = random_decoder(DecoderConfig(gated=gated, **CFG), seed=1, max_pos=512)
    g = torch.Generator().manual_seed(2)
    tok = lambda n: torch.randint(0, 300, (n,), generator=g).to(DEV)
    states = dec.new_paged_states(3, n_pages=15, max_tokens=400, page=32, quantized=quantized)
    calls = recorded(monkeypatch, "paged_attn")
    parts = [[tok(70), tok(0), tok(5)], [tok(1), tok(1), tok(1)], [tok(0), tok(40), tok(300)]]
    for part in parts:
        h = dec.extend(torch.cat(part), [p.numel() for p in part], states)
        assert h.shape == (sum(p.numel() for p in part), 256) and torch.isfinite(h.float()).all()
    assert states.lengths == [71, 41, 306] and states.ctx.tolist() == [71, 41, 306]
    ids = torch.randint(0, 300, (3, 4, 5), generator=g).to(DEV)
    before = states[1].k.clone()
    lp = dec.score_paged(ids, states)
    assert lp.shape == (3, 5) and torch.allclose(lp.exp().sum(1), torch.ones(3, device=DEV), atol=1e-5)
    assert torch.equal(states[1].k, before)
    check_calls(calls)
    # layer 0 against the rectangular path, state by state
    old = recorded(monkeypatch, "branched_attn")
    for b in range(3):
        whole = torch.cat([p[b] for p in parts])
        flat = dec.new_state_caches(1, 400)
        dec.prefill(whole[None], flat)
        T = whole.numel()
        if quantized:
            k, v = kernels.page_read(states[0], states.table, states.ctx, 306, dtype=torch.int8)
            for x, c in ((k, flat[0][0]), (v, flat[0][1])):
                assert torch.equal(x.q[b, :, :T], c.q[0, :, :T]) and torch.equal(x.scale[b, :, :T, 0], c.scale[0, :, :T])
        old.clear()
        dec.score(ids[b:b + 1], flat)
        (q, k, v), score0 = old[0][0][:3], calls[-2][0]
        for want, got in ((q, score0[0]), (k, score0[1]), (v, score0[2])):
            assert torch.equal(want.transpose(1, 2).reshape(20, -1, 64), got[20 * b:20 * b + 20])
    # no room: nothing changes; after a state's end there is
    with pytest.raises(MemoryError):
        dec.extend(tok(50), [50, 0, 0], states)
    assert states.lengths == [71, 41, 306]
    states.release(2)
    dec.extend(tok(80), [50, 0, 30], states)
    assert states.lengths == [121, 41, 30] and torch.isfinite(dec.score_paged(ids, states)).all()
    del calls[:-4]
    check_calls(calls)
    for bad in (lambda: dec.extend(tok(3), [1, 1, 2], states), lambda: dec.extend(tok(500), [500, 0, 0], states),
                lambda: dec.score_paged(ids[:2], states)):
        with pytest.raises(ValueError):
            bad()


def test_captured_scoring_follows_the_states(gpu_lib, monkeypatch):
    """One graph of a scoring pass over paged states, replayed as they grow, end and start anew: bit for bit the eager calls
    with the graph's hint of the lengths (by which the keys are split, and so summed)."""
    from opendecider_amd import kernels
    from opendecider_amd.decoder import DecoderConfig, random_decoder
    dec = random_decoder(DecoderConfig(**CFG), seed=3, max_pos=512)
    g = torch.Generator().manual_seed(4)
    tok = lambda n: torch.randint(0, 300, (n,), generator=g).to(DEV)
    states = dec.new_paged_states(2, n_pages=20, max_tokens=448, page=32)
    ids = tok(2 * 3 * 4).view(2, 3, 4)
    dec.extend(tok(40), [33, 7], states)
    dec.score_paged(ids, states)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lp = dec.score_paged(ids, states)
    for counts in ([0, 0], [1, 200], [90, 1], None, [60, 0]):
        if counts is None:
            states.release(0)
        else:
            dec.extend(tok(sum(counts)), counts, states)
        ids.copy_(tok(24).view(2, 3, 4))
        graph.replay()
        got = lp.clone()
        with monkeypatch.context() as m:
            fn = kernels.paged_attn
            m.setattr(kernels, "paged_attn", lambda *a, max_ctx, **kw: fn(*a, max_ctx=33, **kw))
            want = dec.score_paged(ids, states)
        assert torch.equal(got, want) and torch.isfinite(got).all()
        graph.replay()
        assert torch.equal(lp, got)
    small = dec.new_paged_states(2, n_pages=4, max_tokens=512, page=32)  # its table holds more than the rotary tables
    dec.score_paged(ids, small)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(ValueError):
        dec.score_paged(ids, small)


def test_hybrid_has_no_paged_states(gpu_lib):
    from opendecider_amd.decoder import DecoderConfig, random_decoder
    dec = random_decoder(DecoderConfig(hidden=256, ffn=512, n_heads=4, n_kv_heads=2, head_dim=64, n_layers=2, vocab=50,
                                       full_attention_interval=2, lin_k_heads=2, lin_v_heads=2), max_pos=64)
    with pytest.raises(ValueError):
        dec.new_paged_states(1, 2, 32)


def test_states_of_another_decoder(gpu_lib):
    from opendecider_amd import PagedStates
    from opendecider_amd.decoder import DecoderConfig, random_decoder
    hybrid = random_decoder(DecoderConfig(hidden=256, ffn=512, n_heads=4, n_kv_heads=2, head_dim=64, n_layers=2, vocab=50,
                                          full_attention_interval=2, lin_k_heads=2, lin_v_heads=2), max_pos=64)
    dec = random_decoder(DecoderConfig(**CFG), max_pos=64)
    ids = torch.zeros(1, dtype=torch.int64, device=DEV)
    for d, states in ((hybrid, PagedStates(2, 1, 2, 64, 2, 32, 16)), (dec, PagedStates(3, 1, 2, 64, 2, 32, 16)),
                      (dec, PagedStates(2, 0, 2, 64, 2, 32, 16)), (dec, dec.new_state_caches(1, 32))):
        with pytest.raises(ValueError):
            d.extend(ids, [1], states)
        with pytest.raises(ValueError):
            d.score_paged(ids.view(1, 1, 1), states)
    narrow = PagedStates(2, 1, 4, 64, 2, 32, 16)  # of other heads: refused by the kernels, and nothing is counted
    with pytest.raises(ValueError):
        dec.extend(ids, [1], narrow)
    assert narrow.lengths == [0]


def test_refusals(gpu_lib):
    from opendecider_amd import PagedKVCache, kernels
    c = make(52, [4, 3], [20, 5])
    cache = cache_of(c)
    q, k, v = gpu(c["q"]), gpu(c["k"]), gpu(c["v"])
    tab, start, ctx, sc = gpu(c["table"]), gpu(c["start"]), gpu(c["ctx"]), c["scale"]
    with pytest.raises(RuntimeError):
        kernels.paged_attn(c["q"], k, v, cache, tab, start, ctx, sc)
    with pytest.raises(RuntimeError):
        kernels.page_append(k, v, cache, c["table"], start, ctx)
    for bad in (dict(q=q.float()), dict(k=k.half()), dict(tab=tab.long()), dict(start=start.long()), dict(ctx=ctx.long())):
        a = dict(dict(q=q, k=k, v=v, tab=tab, start=start, ctx=ctx), **bad)
        with pytest.raises(TypeError):
            kernels.paged_attn(a["q"], a["k"], a["v"], cache, a["tab"], a["start"], a["ctx"], sc)
    for bad in (dict(k=k[:, :1]), dict(k=None), dict(v=v[:3]), dict(q=q[:, :7]), dict(tab=tab[:1]), dict(start=start[:2]),
                dict(ctx=ctx[:1]), dict(sc=0.0), dict(sc=float("nan")), dict(sc=-1.0), dict(rb=torch.zeros(3, dtype=torch.int32, device=DEV)),
                dict(rb=torch.zeros(7, device=DEV)), dict(out=torch.empty(7, 8, 64, dtype=BF, device=DEV)), dict(q=q[..., :64]),
                dict(tab=tab.t().contiguous().t())):
        a = dict(dict(q=q, k=k, v=v, tab=tab, start=start, ctx=ctx, sc=sc, rb=None, out=None), **bad)
        with pytest.raises(ValueError):
            kernels.paged_attn(a["q"], a["k"], a["v"], cache, a["tab"], a["start"], a["ctx"], a["sc"], row_begin=a["rb"], out=a["out"])
    with pytest.raises(TypeError):
        kernels.page_append(k.float(), v, cache, tab, start, ctx)
    with pytest.raises(ValueError):
        kernels.page_append(k, v[:, :, :64], cache, tab, start, ctx)
    with pytest.raises(ValueError):
        kernels.page_read(cache, tab, ctx, -1)
    for dt in (torch.float16, torch.int32):
        with pytest.raises(TypeError):
            kernels.page_read(cache, tab, ctx, 4, dtype=dt)
    with pytest.raises(TypeError):
        kernels.page_read(PagedKVCache(2, 2, 128, 16, DEV, quantized=False), tab, ctx, 4, dtype=torch.int8)


def test_nothing_to_do(gpu_lib):
    """No tokens, no sequences, no pages."""
    from opendecider_amd import PagedKVCache, kernels
    cache = PagedKVCache(0, 2, 64, 16, DEV)
    e = lambda *s, dt=BF: torch.empty(*s, dtype=dt, device=DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    assert kernels.paged_attn(e(0, 4, 64), e(0, 2, 64), e(0, 2, 64), cache, e(1, 0, dt=torch.int32), i32(0, 0), i32(0), 0.1).shape == (0, 4, 64)
    kernels.page_append(e(3, 2, 64), e(3, 2, 64), cache, e(0, 0, dt=torch.int32), i32(0), e(0, dt=torch.int32))
    k, v = kernels.page_read(cache, e(2, 0, dt=torch.int32), i32(5, 0), 7)
    assert k.shape == (2, 2, 7, 64) and not k.any() and not v.any()
    q, x = torch.randn(3, 4, 64, device=DEV).to(BF), torch.randn(3, 2, 64, device=DEV).to(BF)
    o = kernels.paged_attn(q, x, x, cache, e(1, 0, dt=torch.int32), i32(0, 3), i32(9), 0.1)
    assert torch.equal(o[0], x[0].repeat_interleave(2, 0))
