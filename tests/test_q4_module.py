"""Q4Linear as a module, on the CPU: casts and moves of a model, and (on the GPU) activations and residuals of other types."""
import pytest
import torch
import torch.nn as nn

from opendecider_amd import Q4Linear, quantize_q4_

BF = torch.bfloat16


def net(seed=0):
    torch.manual_seed(seed)
    return quantize_q4_(nn.Sequential(nn.Linear(100, 64), nn.LayerNorm(64), nn.Sequential(nn.Linear(64, 8, bias=False))))


CASTS = {"to bf16": lambda m: m.to(BF), "float": lambda m: m.float(), "half": lambda m: m.half(), "double": lambda m: m.double(),
         "bfloat16, then half": lambda m: m.bfloat16().half(), "to cpu bf16": lambda m: m.to("cpu", BF),
         "the module itself": lambda m: (m[0].to(BF), m[2][0].float())}


@pytest.mark.parametrize("cast", CASTS)
def test_casts_leave_the_format(cast):
    """Scales and bias keep their types and bits whatever the model is cast to; other modules follow."""
    m = net()
    want = {k: v.clone() for k, v in m.state_dict().items() if not k.startswith("1.")}
    assert want["0.d"].dtype == torch.float16 and want["0.bias"].dtype == BF and "2.0.bias" not in want
    assert not torch.equal(want["0.d"].to(BF).to(torch.float16), want["0.d"])  # a cast would lose bits
    CASTS[cast](m)
    got = m.state_dict()
    for k, v in want.items():
        assert got[k].dtype == v.dtype and torch.equal(got[k], v), k
    if cast != "the module itself":
        assert m[1].weight.dtype != torch.float32 or cast == "float"
    assert torch.equal(m[0].weight, Q4Linear(want["0.qs"], want["0.d"], in_features=100).weight)


def test_moves_reach_every_buffer():
    m = net().to("meta", BF)
    assert {(b.device.type, b.dtype) for b in m[0].buffers()} == {("meta", torch.uint8), ("meta", torch.float16), ("meta", BF)}


@pytest.mark.gpu
def test_cast_models_run(gpu_lib):
    """A model that is cast after it was quantized, inputs and residuals of other types: the bf16 call's outputs."""
    torch.manual_seed(1)
    for M in (3, 50):
        x, r = torch.randn(M, 100).to(BF).cuda(), torch.randn(M, 64).to(BF).cuda()
        x[x.abs() < 2.0 ** -10] = 0  # the others are the same numbers in fp16
        m = net()[0].cuda()
        want, added = m(x), m(x, r)
        for dtype in (BF, torch.float32, torch.float16):
            c = net()[0].cuda().to(dtype)
            assert torch.equal(c(x), want)
            y = c(x.to(dtype), r.float())
            assert y.dtype == dtype and torch.equal(y, added.to(dtype))
