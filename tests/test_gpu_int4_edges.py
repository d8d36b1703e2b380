"""Attention over 4-bit pages at the ends of what values may be, on the GPU against its float64 restatement: first values that are
zeros and others that are the smallest numbers. Batches and checks are test_gpu_int4_pages.py's; the forms send them through each
kernel that they can reach."""
import pytest
import torch

import test_gpu_int4_pages as t4
from oracle import paged as op

pytestmark = pytest.mark.gpu

BF, FORMS = t4.BF, t4.FORMS


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
