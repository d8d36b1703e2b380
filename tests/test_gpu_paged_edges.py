"""The paged K/V cache at the edges of its range, on the GPU against its float64 restatement: values and scales that are not
finite, sizes near the ends of the formats, offsets outside the packed rows. Batches, bounds and checks are
test_gpu_paged.py's; every case runs through each kernel that it can reach."""
import math

import pytest
import torch

import paged_exact
from oracle import paged as op
from oracle.quant import quantize_rows
from test_gpu_paged import BF, DEV, check_attn, gpu, make, run_attn

pytestmark = pytest.mark.gpu

HEADS = [(64, 4, 4), (128, 8, 2), (256, 4, 1)]  # head dim, query heads, K/V heads


def through(path, seed, new, ctx, heads, kv, d, of=make, **kw):
    """A batch that the library takes by the kernels of `path`: "stream" (small calls), "tiles" (rows of no sequence make the
    call a large one), "image" (and a table with room for 2^16 tokens)."""
    page = kw.get("page", 16)
    c = of(seed, new, ctx, heads, kv, d, **dict(kw, pad=0 if path == "stream" else 1100))
    if path == "image":
        wide = torch.full((len(new), 2 ** 16 // page), -1, dtype=torch.int32)
        wide[:, :c["table"].shape[1]] = c["table"]
        c["table"] = wide
    return c


def place(c, b, pos):
    """(page, row) of a cached position."""
    page = c["pages"][0].shape[2]
    return int(c["table"][b, pos // page]), pos % page


# ------------------------------------------------------------------------------------------------ not finite
@pytest.mark.parametrize("d,heads,kv", HEADS)
@pytest.mark.parametrize("path", ["stream", "tiles"])
def test_infinite_values_in_bf16_pages(gpu_lib, path, d, heads, kv):
    """A cached infinity arrives at every token of its sequence in its column, both signs and NaN as NaN, and every other
    output keeps its bits."""
    c = through(path, 60, [1, 2, 1], [40, 2500, 70], heads, kv, d, int8=False)
    at = [place(c, 0, 3), place(c, 0, 39), place(c, 1, 1200), place(c, 1, 2499)]
    for page, row in at:  # of ordinary weight: no score is far below the others
        c["pages"][0][page, 0, row] = 0
    want, wl = run_attn(c)
    inf, rep = float("inf"), heads // kv
    c["pages"][1][at[0][0], 0, at[0][1], 5] = inf
    c["pages"][1][at[1][0], 0, at[1][1], d - 1] = -inf
    c["pages"][1][at[2][0], 0, at[2][1], 0] = -inf
    c["pages"][1][at[2][0], 0, at[2][1], 17] = inf
    c["pages"][1][at[3][0], 0, at[3][1], 17] = -inf
    c["pages"][1][at[3][0], 0, at[3][1], 18] = float("nan")
    got, gl = run_attn(c)
    assert torch.equal(gl[:4], wl[:4])
    hit = torch.zeros(4, heads, d, dtype=torch.bool)
    hit[0, :rep, [5, d - 1]] = True
    hit[1:3, :rep, [0, 17, 18]] = True
    assert torch.equal(got[:4].cpu()[~hit], want[:4].cpu()[~hit])
    assert (got[0, :rep, 5] == inf).all() and (got[0, :rep, d - 1] == -inf).all()
    assert (got[1:3, :rep, 0] == -inf).all() and got[1:3, :rep, 17:19].isnan().all()


@pytest.mark.parametrize("d,heads,kv", HEADS)
@pytest.mark.parametrize("path", ["stream", "tiles", "image"])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_scales_that_are_not_finite(gpu_lib, bad, path, d, heads, kv):
    """An int8 row with such a scale counts as NaN: K's in the whole outputs and the LSE of the tokens that see it, V's in the
    outputs. Other heads and sequences keep their bits."""
    c = through(path, 61, [1, 2, 1], [40, 700, 70], heads, kv, d)
    want, wl = run_attn(c)
    rep = heads // kv
    for i, b, pos in ((0, 0, 9), (1, 1, 650)):
        page, row = place(c, b, pos)
        c["scales"][i][page, 0, row] = bad
    got, gl = run_attn(c)
    assert got[:3, :rep].isnan().all() and gl[0, :rep].isnan().all()
    assert torch.equal(gl[1:4], wl[1:4]) and torch.equal(got[3], want[3])
    assert torch.equal(got[:3, rep:], want[:3, rep:]) and torch.equal(gl[0, rep:], wl[0, rep:])


# ------------------------------------------------------------------------------------------------ small numbers
@pytest.mark.parametrize("d,heads,kv", HEADS)
@pytest.mark.parametrize("path", ["stream", "tiles", "image"])
@pytest.mark.parametrize("q_exp,k_exp", [(-66, -66), (-126, 0), (-100, None)])
def test_small_queries_and_keys(gpu_lib, q_exp, k_exp, path, d, heads, kv):
    """Scores that vanish: the mean of the values, also where a block's last keys are none. k_exp None: keys of zeros, with the
    scale that the append gives them."""
    c = through(path, 62, [1, 3], [300, 70], heads, kv, d)
    c["q"] = (c["q"].float() * 2.0 ** q_exp).to(BF)
    if k_exp is None:
        c["pages"][0].zero_()
        c["scales"][0].fill_(1e-8 / 127)
        c["k"].zero_()
    else:
        c["scales"][0] = c["scales"][0] * 2.0 ** k_exp
        c["k"] = (c["k"].float() * 2.0 ** k_exp).to(BF)
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("d,heads,kv", HEADS)
@pytest.mark.parametrize("path", ["tiles", "image"])
@pytest.mark.parametrize("own", [False, True])
def test_small_values(gpu_lib, own, path, d, heads, kv):
    """int8 values around 2^-120, whose frames' reciprocals no fp32 number holds. The outputs are partly subnormal: half of
    their step, 2^-134, more than the relative bounds."""
    c = through(path, 63, [1, 40], [300, 130], heads, kv, d)
    c["scales"][1] = c["scales"][1] * 2.0 ** -120
    c["v"] = (c["v"].float() * 2.0 ** -120).to(BF)
    assert c["scales"][1].max() < 2.0 ** -121
    out, lse = run_attn(c, own=own)
    live = 41
    ref, rl, mean, size, total = op.attention(c["q"][:live], c["k"][:live] if own else None, c["v"][:live] if own else None,
                                              (*c["pages"], *c["scales"]), c["table"], c["start"], c["ctx"], c["scale"])
    e = (2.0 ** -11 + 2.0 ** -24 * (d + 8)) * size
    bound = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -11 + 2 * e[..., None] + 2.0 ** -22 * 400) * 1.02 * mean + \
        2.0 ** -31 * total[..., None] + 2.0 ** -134
    out = out[:live].double().cpu()
    assert ((out - ref).abs() <= bound).all(), ((out - ref).abs() / bound).max()
    assert ((lse[:live].double().cpu() - rl).abs() <= e + 2.0 ** -20 * (1 + rl.abs() + size)).all()


# ------------------------------------------------------------------------------------------------ every key
@pytest.mark.parametrize("d,heads,kv", [*HEADS, (128, 7, 1)])
@pytest.mark.parametrize("path", ["stream", "tiles", "image"])
@pytest.mark.parametrize("shape", range(len(paged_exact.SHAPES)))
def test_every_key_counts(gpu_lib, shape, path, d, heads, kv):
    """Narrow bounds (paged_exact.py) at the borders of tiles and blocks, for the bounds that the call knows and for a max_ctx that
    leaves the last split all keys but the first 64."""
    new, ctx = paged_exact.SHAPES[shape]
    c = through(path, shape, new, ctx, heads, kv, d, of=paged_exact.batch, page=[16, 64, 32][shape % 3])
    for own in (True, False):
        paged_exact.check(c, *run_attn(c, own=own), path == "stream", own)
    if path != "image":
        paged_exact.check(c, *run_attn(c, max_ctx=64), path == "stream")


@pytest.mark.parametrize("d,heads,kv", HEADS)
@pytest.mark.parametrize("path", ["stream", "tiles", "image"])
def test_every_key_counts_in_option_rows(gpu_lib, path, d, heads, kv):
    c = through(path, 67, [24, 40, 1], [63, 65, 128], heads, kv, d, of=paged_exact.batch, rows=8, page=32)
    paged_exact.check(c, *run_attn(c), path == "stream")


# ------------------------------------------------------------------------------------------------ offsets
@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("pad", [0, 1100])
def test_sequences_outside_the_packed_rows(gpu_lib, pad, int8):
    """A sequence that begins before the first packed row, or ends behind the last one, has no tokens: nothing of it is
    written, and its rows stay as they were."""
    from opendecider_amd import kernels
    from test_gpu_paged import cache_of
    c = make(64, [5, 4, 6], [20, 3, 40], int8=int8, pad=pad)
    N = c["q"].shape[0]
    for first, last in ((-3, N), (0, N + 5), (-1, N + 1), (-(2 ** 31), 2 ** 31 - 1)):
        c["start"] = torch.tensor([first, 5, 9, last], dtype=torch.int32)
        cache = cache_of(c)
        kernels.page_append(gpu(c["k"]), gpu(c["v"]), cache, gpu(c["table"]), gpu(c["start"]), gpu(c["ctx"]))
        for i, (x, got, gs) in enumerate(((c["k"], cache.k, cache.k_scale), (c["v"], cache.v, cache.v_scale))):
            want, ws = op.append(c["pages"][i], c["scales"][i], x, c["table"], c["start"], c["ctx"])
            assert torch.equal(got.cpu(), want), (first, last)
            assert ws is None or torch.equal(gs.cpu(), ws)
        out = torch.full(c["q"].shape, 7.0, dtype=BF, device=DEV)
        _, lse = run_attn(c, out=out)
        check_attn(c, out, lse)
        if first < 0:
            assert (out[:5] == 7).all()
        if last > N:
            assert (out[9:] == 7).all()


# ------------------------------------------------------------------------------------------------ many
@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("bounds", [{}, dict(max_new=1, max_ctx=1)])
def test_many_states_without_bounds(gpu_lib, bounds, int8):
    """20000 states of a token each, for bounds that ask for more slot tiles than a launch holds. Queries of 0: the token's value,
    or half of it beside a cached token of zeros."""
    from opendecider_amd import PagedKVCache, kernels
    B, heads, d = 20000, 8, 128
    cache = PagedKVCache(1, 1, d, 16, DEV, quantized=int8)
    i32 = lambda x: x.to(torch.int32).to(DEV)
    v = torch.randn(B, 1, d, generator=torch.Generator().manual_seed(65)).to(BF).to(DEV)
    ctx = torch.arange(B) % 2
    out = kernels.paged_attn(torch.zeros(B, heads, d, dtype=BF, device=DEV), v, v, cache, i32(torch.zeros(B, 1)), i32(torch.arange(B + 1)),
                             i32(ctx), d ** -0.5, **bounds)
    want = torch.where(ctx.to(DEV).bool()[:, None, None], v / 2, v).expand(B, heads, d)
    assert torch.equal(out, want)


# ------------------------------------------------------------------------------------------------ states
def test_states_do_not_change_in_a_capture(gpu_lib, monkeypatch):
    """What changes the host's lengths and free pages is refused while a graph is captured, with nothing changed."""
    from opendecider_amd import PagedStates
    s = PagedStates(1, 2, 1, 64, n_pages=4, max_tokens=64, page=16)
    s.reserve([20, 3])
    s.advance([20, 3])
    held = lambda: (list(s.lengths), [list(p) for p in s.pages], list(s.free), s.table.tolist(), s.ctx.tolist())
    before = held()
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        for step in (lambda: s.reserve([1, 20]), lambda: s.advance([1, 1]), lambda: s.release(0)):
            with pytest.raises(RuntimeError):
                step()
    assert held() == before
    s.reserve([1, 20])
    s.release(0)
    assert s.lengths == [0, 3] and s.ctx.tolist() == [0, 3]


@pytest.mark.parametrize("quantized", [True, False])
def test_states_read(gpu_lib, quantized):
    """PagedStates.read: every layer's own pages through the common table, as long as the longest state."""
    from opendecider_amd import PagedStates, kernels
    s = PagedStates(2, 3, 2, 64, n_pages=9, max_tokens=64, page=16, quantized=quantized)
    counts = [20, 0, 33]
    x = torch.randn(4, 53, 2, 64, generator=torch.Generator().manual_seed(66)).to(BF)
    s.reserve(counts)
    start = torch.tensor([0, 20, 20, 53], dtype=torch.int32)
    for li in range(2):
        kernels.page_append(gpu(x[2 * li]), gpu(x[2 * li + 1]), s[li], s.table, gpu(start), s.ctx)
    s.advance(counts)
    for li in range(2):
        for dtype in (BF, torch.float32):
            for side, got in enumerate(s.read(li, dtype=dtype)):
                want = torch.zeros(3, 2, 33, 64, dtype=dtype)
                for b in (0, 2):
                    rows = x[2 * li + side][start[b]:start[b + 1]].transpose(0, 1)
                    if quantized:
                        q, sc = quantize_rows(rows)
                        rows = q.float() * sc
                    want[b, :, :counts[b]] = rows.to(dtype)
                assert torch.equal(got.cpu(), want)
    none = PagedStates(1, 0, 2, 64, n_pages=1, max_tokens=16, page=16, quantized=quantized)
    assert [t.shape for t in none.read(0)] == [(0, 2, 0, 64)] * 2
