"""The narrow check of the attention over 4-bit pages (int4_exact.py) on the CPU: its batches are what it says, and it takes the
float64 result as bf16, and none of the mistakes that the kernels could make."""
import pytest
import torch

from int4_exact import SHAPES, batch, check, pack
from oracle import paged as op

BF = torch.bfloat16


def result(c, own=True):
    new = (c["k"], c["v"]) if own else (None, None)
    return op.attention(c["q"], *new, (*c["pages"], *c["scales"]), c["table"], c["start"], c["ctx"], c["scale"])


def test_packed_codes():
    u = torch.randint(0, 16, (3, 64), generator=torch.Generator().manual_seed(0))
    assert torch.equal(op.values4(pack(u), torch.ones(3, 2)), u.double() - 8)


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("own", [True, False])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_check_sees_a_key_and_a_percent(shape, own, d):
    new, ctx = SHAPES[shape]
    c = batch(shape, new, ctx, 4, 2, d, spare=1)
    right = result(c, own)
    vs = c["scales"][1].double()
    wrong = {
        "one key less": result(dict(c, ctx=(c["ctx"] - 1).clamp_min(0)), own),
        "one key more": result(dict(c, ctx=c["ctx"] + 1), own),
        "values 1% off": result(dict(c, scales=[c["scales"][0], vs * 1.01]), own),
    }
    for block in (0, d // 32 - 1):  # of one head's columns
        off = vs.clone()
        off[:, (block + shape) % 2, :, block] *= 1.01
        wrong[f"block {block} 1% off"] = result(dict(c, scales=[c["scales"][0], off]), own)
    off = vs.clone()
    off[:, :, ::2], off[:, :, 1::2] = vs[:, :, 1::2], vs[:, :, ::2]
    wrong["scales of the keys beside"] = result(dict(c, scales=[c["scales"][0], off]), own)
    off = torch.cat([vs[..., 1:], vs[..., :1]], -1)
    wrong["scales of the blocks beside"] = result(dict(c, scales=[c["scales"][0], off]), own)
    if max(ctx) > 64:  # the last key of the first block of 64, and the first of the second, are not there
        cut = vs.clone()
        b = ctx.index(max(ctx))
        for pos in (63, 64):
            cut[int(c["table"][b, pos // 16]), :, pos % 16] = 0
        wrong["no values at a block's border"] = result(dict(c, scales=[c["scales"][0], cut]), own)
    for stream in (True, False):
        check(c, right[0].to(BF), right[1].float(), stream, own, against=right)
        for name, (out, lse, *_) in wrong.items():
            try:
                check(c, out.to(BF), right[1].float(), stream, own, against=right)
            except AssertionError:
                pass
            else:
                pytest.fail(f"{name} passes (streaming: {stream})")
            if name.startswith("one"):
                with pytest.raises(AssertionError):
                    check(c, right[0].to(BF), lse.float(), stream, own, against=right)
