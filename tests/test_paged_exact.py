"""The narrow check of the paged attention (paged_exact.py) on the CPU: it takes the float64 result as bf16, and none of the
mistakes that the kernels' tails could make."""
import pytest
import torch

from oracle import paged as op
from paged_exact import BF, SHAPES, batch, check


def result(c, own=True):
    new = (c["k"], c["v"]) if own else (None, None)
    return op.attention(c["q"], *new, (*c["pages"], *c["scales"]), c["table"], c["start"], c["ctx"], c["scale"])


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("own", [True, False])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_check_sees_a_key_and_a_percent(shape, own, d):
    new, ctx = SHAPES[shape]
    c = batch(shape, new, ctx, 4, 2, d, spare=1)
    right = result(c, own)
    wrong = {
        "one key less": result(dict(c, ctx=(c["ctx"] - 1).clamp_min(0)), own),
        "one key more": result(dict(c, ctx=c["ctx"] + 1), own),
        "values 1% off": result(dict(c, scales=[c["scales"][0], c["scales"][1] * 1.01]), own),
    }
    if max(ctx) > 64:  # the last key of the first block of 64, and the first of the second, are not there
        cut = dict(c, scales=[c["scales"][0], c["scales"][1].clone()])
        b = ctx.index(max(ctx))
        for pos in (63, 64):
            cut["scales"][1][int(c["table"][b, pos // 16]), :, pos % 16] = 0
        wrong["no values at a block's border"] = result(cut, own)
    for stream in (True, False):
        check(c, right[0].to(BF), right[1].float(), stream, own, against=right)
        for name, (out, lse, *_) in wrong.items():
            with pytest.raises(AssertionError):
                check(c, out.to(BF), right[1].float(), stream, own, against=right)
            if name.startswith("one"):
                with pytest.raises(AssertionError):
                    check(c, right[0].to(BF), lse.float(), stream, own, against=right)
