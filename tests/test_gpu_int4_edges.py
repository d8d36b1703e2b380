"""Attention over pages at the ends of what values may be, on the GPU against its float64 restatement: 4-bit pages whose first
values are zeros and whose others are the smallest numbers, and values up to the largest finite ones, in 4-bit pages, in the others
where they share the kernels, and among the new tokens. Batches, bounds and checks are test_gpu_int4_pages.py's and
test_gpu_paged.py's; the forms send them through each kernel that they can reach."""
import pytest
import torch

import test_gpu_int4_pages as t4
import test_gpu_paged as tp
from oracle import paged as op

pytestmark = pytest.mark.gpu

BF, FORMS = t4.BF, t4.FORMS
MOST = torch.finfo(BF).max


def zero_values(c, first):
    """The values' scales of every sequence's first positions become 0."""
    page = c["pages"][0].shape[2]
    for row in c["table"].tolist():
        for pos in range(first):
            if row[pos // page] >= 0:
                c["scales"][1][row[pos // page], :, pos % page] = 0


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("exp", [-126, -128, -133])
@pytest.mark.parametrize("own", [False, True])
def test_no_values_before_the_smallest(gpu_lib, own, exp, d, form):
    """A sequence's first block of 64 keys has values of zero, the others some of the smallest scales that bf16 holds. The outputs
    are partly subnormal: half of bf16's step, 2^-134, more than the relative bounds, and as much for fp32's: 2^-149 for each of the
    less than 2^10 keys' products and for the sums'."""
    for new, ctx in (([1, 1], [600, 90]), ([40], [300])):
        c = t4.as_many(t4.make(31, new, ctx, 4, 1, d, **t4.padded(form)), form)
        c["scales"][1].fill_(2.0 ** exp)
        c["v"] = (c["v"].float() * 2.0 ** -120).to(BF)
        zero_values(c, 64)
        n = sum(new)
        out, lse = t4.run_attn(c, own=own)
        ref, rl, mean, size, total = op.attention(c["q"][:n], c["k"][:n] if own else None, c["v"][:n] if own else None,
                                                  (*c["pages"], *c["scales"]), c["table"], c["start"], c["ctx"], c["scale"])
        e = 2.0 ** -24 * (d + 8) * size + 2.0 ** -30 * size
        bound = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2 * e[..., None] + 2.0 ** -22 * 700) * 1.02 * mean + 2.0 ** -31 * total[..., None] + \
            2.0 ** -133
        out = out[:n].double().cpu()
        assert ((out - ref).abs() <= bound).all(), ((out - ref).abs() / bound).max()


LARGE = [(122, 125), (0, 125), (122, 0), (113, 113)]  # 2^ of the cached values' size over the usual one, and the new ones'


def enlarged(c, cached, new):
    i = 0 if c["scales"][1] is None else 1
    side = (c["pages"], c["scales"])[i]
    side[1] = (side[1].double() * 2.0 ** cached).clamp(-MOST, MOST).to(side[1].dtype)
    c["v"] = (c["v"].double() * 2.0 ** new).clamp(-MOST, MOST).to(BF)
    return c


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cached,new", LARGE)
def test_values_up_to_the_largest(gpu_lib, cached, new, d, form):
    """Averages of finite values are finite, whatever their size."""
    for n, ctx, rows in (([1, 1], [600, 90], 0), ([40], [300], 0), ([30, 3], [130, 0], 8)):
        c = enlarged(t4.as_many(t4.make(32, n, ctx, 4, 1, d, rows=rows, **t4.padded(form)), form), cached, new)
        t4.check_attn(c, *t4.run_attn(c))
        t4.check_attn(c, *t4.run_attn(c, own=False), own=False)


@pytest.mark.parametrize("d,heads,kv", [(64, 8, 8), (128, 8, 1), (256, 4, 1)])
def test_large_values_of_many_splits(gpu_lib, d, heads, kv):
    """The merge of as many parts as a call is split into, each of them near the largest number."""
    c = enlarged(t4.make(33, [1], [9000], heads, kv, d, page=64), 122, 122)
    g = torch.Generator().manual_seed(5)
    c["scales"][1] = (2.0 ** 124 * (1 + torch.rand(c["scales"][1].shape, generator=g) * 0.5)).to(BF)
    c["pages"][1].fill_(0xFF)  # every value 7 times its scale: far past half of the largest number
    c["q"] = c["q"] * 0.0  # a plain average of them all
    c["v"] = torch.full(c["v"].shape, 2.0 ** 127).to(BF)
    t4.check_attn(c, *t4.run_attn(c))


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("form", ["rows", "image"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cached,new", LARGE)
def test_values_up_to_the_largest_in_other_pages(gpu_lib, cached, new, d, form, int8):
    """Chunks and option rows over int8 and bf16 pages."""
    for n, ctx, rows in (([40], [300], 0), ([30, 3], [130, 0], 8)):
        c = enlarged(t4.as_many(tp.make(34, n, ctx, 4, 1, d, int8=int8, rows=rows, **t4.padded(form)), form), cached, new)
        tp.check_attn(c, *t4.run_attn(c))


def small_and(c, exp):
    """New values around 2^-100 in every column, those of every third one times 2^exp; the cached ones as they are."""
    e = torch.full((c["v"].shape[2],), -100.0)
    e[::3] = exp
    c["v"] = (c["v"].double() * torch.exp2(e.double())).clamp(-MOST, MOST).to(BF)
    return c


@pytest.mark.parametrize("int8,form", [*((None, f) for f in FORMS), *((q, f) for q in (True, False) for f in ("rows", "image"))])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_small_values_beside_large_and_infinite_ones(gpu_lib, d, form, int8):
    """A column's large or infinite values change nothing in the others, whatever their size. (Few slots over int8 and bf16 pages
    sum as they are.)"""
    for n, ctx, rows in (([1, 1], [600, 0], 0), ([40], [300], 0), ([30, 3], [0, 130], 8)):
        c = t4.as_many(t4.make(35, n, ctx, 4, 1, d, int8=int8, rows=rows, **t4.padded(form)), form)
        v, live = c["v"], sum(n)
        plain = t4.run_attn(small_and(c, -100))
        for exp in (0, 125, None):
            c["v"] = v
            small_and(c, exp or 0)
            if exp is None:
                c["v"][:, :, ::3] = float("inf")
            out, lse = t4.run_attn(c)
            others = torch.arange(d) % 3 != 0
            assert torch.equal(out[:live, :, others], plain[0][:live, :, others]) and torch.equal(lse[:live], plain[1][:live]), exp
            if exp is None:
                assert (out[:live, :, ::3] == float("inf")).all()
            else:
                (t4.check_attn if int8 is None else tp.check_attn)(c, out, lse)
