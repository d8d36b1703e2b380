"""Linears with 4-bit weights on the GPU against float64 products of the same weights, at the sizes, strides and values where
they can go wrong.

Bounds. With the weights w (exact in float64) and A = sum_k |x_k w_k|, an output differs from the float64 one by
  * its own rounding to bf16, 2^-8 |y|;
  * the fp32 sums. A block's 32 products are summed as x (128 + u) beside -136 x, in fp32: 64 terms of at most 143 |x| for |u - 8|
    >= 0 of the true ones, at most 64 * 143 * 2^-24 sum |x| |d| over the block, then 2^-24 (K / 32 + 40) A for the blocks' sum,
    the waves' and the epilogue's (up to 32 rows);
  * the weights' rounding to fp16, 2^-11 A, with fp32 sums of K terms, 2^-24 (K + 40) A, and what fp16 frames of x lose, 2^-39 of the
    row's largest value a term (more rows).
"""
import math

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF = torch.bfloat16
FEW = 32  # rows of x up to which the weights are streamed


def weights(N, K, seed=0, mag=0.02):
    """Packed values and scales of random weights, and the float64 weights that they stand for."""
    g = torch.Generator().manual_seed(seed)
    u = torch.randint(0, 16, (N, K // 32, 32), generator=g)
    d = (torch.randn(N, K // 32, generator=g) * mag / 4).to(torch.float16)
    qs = (u[..., :16] | (u[..., 16:] << 4)).to(torch.uint8).view(N, K // 2)
    return qs, d, ((u.double() - 8) * d.double()[..., None]).view(N, K)


def rows(M, N, seed=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, N, generator=g)
    x[:, ::7] *= 10.0
    return x.to(BF)


def check(y, x, w, d, bias=None, residual=None):
    M, K = x.shape
    x, y = x.double(), y.double().cpu()
    ref, A = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        ref, A = ref + bias.double(), A + bias.double().abs()
    if residual is not None:
        ref, A = ref + residual.double(), A + residual.double().abs()
    sums = x.abs().unflatten(-1, (-1, 32)).sum(-1) @ d.double().abs().T
    if M <= FEW:
        err = 64 * 143 * 2.0 ** -24 * sums + 2.0 ** -24 * (K / 32 + 40) * A
    else:
        err = (2.0 ** -11 + 2.0 ** -24 * (K + 40)) * A + 2.0 ** -39 * x.abs().amax(1, keepdim=True) * w.abs().sum(1)
    bound = 2.0 ** -8 * ref.abs() + 1.01 * err
    bad = ~((y - ref).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}: worst {((y - ref).abs() / bound.clamp_min(1e-300)).max()}"


SIZES = [(1, 1, 32), (1, 16, 128), (1, 17, 160), (2, 100, 1024), (3, 250, 96), (5, 1000, 4096), (16, 40, 64), (17, 300, 736), (31, 65, 2048),
         (32, 512, 512), (33, 512, 512), (33, 1, 32), (40, 257, 96), (64, 300, 1056), (129, 511, 160), (200, 33, 4096), (257, 640, 1024),
         (513, 1030, 288), (1, 4096, 12288), (24, 1536, 4096), (300, 200, 12288)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear(gpu_lib, M, N, K):
    from opendecider_amd import kernels
    qs, d, w = weights(N, K)
    x = rows(M, K)
    check(kernels.q4_linear(x.to(DEV), qs.to(DEV), d.to(DEV)), x, w, d)


@pytest.mark.parametrize("M,N,K", [(1, 9000, 160), (16, 9001, 2080), (7, 60000, 96), (1, 60001, 1056), (12, 60001, 1056), (20, 9000, 288),
                                   (32, 9001, 2080), (29, 17000, 2080), (18, 30007, 160), (24, 40000, 544), (30, 60001, 1056), (40, 30000, 224)])
def test_many_rows_of_weights(gpu_lib, M, N, K):
    test_linear(gpu_lib, M, N, K)


@pytest.mark.parametrize("M,N,K", [(1, 50, 96), (20, 100, 544), (70, 131, 1056)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [False, True])
def test_epilogue(gpu_lib, M, N, K, bias, residual):
    from opendecider_amd import kernels
    qs, d, w = weights(N, K, 2)
    x, b, r = rows(M, K), rows(1, N, 3)[0], rows(M, N, 4)
    b, r = (b if bias else None), (r if residual else None)
    gpu = lambda t: None if t is None else t.to(DEV)
    y = kernels.q4_linear(gpu(x), gpu(qs), gpu(d), gpu(b), gpu(r))
    check(y, x, w, d, b, r)
    if residual:  # in place on the residual
        h = gpu(r)
        assert kernels.q4_linear(gpu(x), gpu(qs), gpu(d), gpu(b), h, out=h) is h and torch.equal(h, y)


@pytest.mark.parametrize("M", [1, 7, 32, 33, 90])
def test_every_value_and_place(gpu_lib, M):
    """Weights that are one value in one place of a block, the rest 0 (u = 8), and x that names the place: each product alone."""
    from opendecider_amd import kernels
    N, K = 16, 32 * 32
    u = torch.full((N, 32, 32), 8)
    for n in range(N):
        for b in range(32):
            u[n, b, (b + n) % 32] = n  # block b: value n at place (b + n) % 32
    d = torch.full((N, 32), 0.5).to(torch.float16) * (torch.arange(32) + 1)[None].to(torch.float16)
    qs = (u[..., :16] | (u[..., 16:] << 4)).to(torch.uint8).view(N, K // 2)
    x = torch.zeros(M, 32, 32)
    for m in range(M):
        x[m, m % 32] = torch.arange(1, 33).float() * (1 + m // 32)  # one block of x, another number in each place
    want = torch.einsum("mbk,nbk->mn", x.double(), (u.double() - 8) * d.double()[..., None])
    got = kernels.q4_linear(x.view(M, K).to(BF).to(DEV), qs.to(DEV), d.to(DEV)).double().cpu()
    assert torch.equal(got, want.to(BF).double())


@pytest.mark.parametrize("lead", [(), (0,), (2, 0), (3, 1), (2, 20)])
def test_leading_dims(gpu_lib, lead):
    """A vector, no rows, several leading dims; an output and a residual of that shape, which may be one tensor."""
    from opendecider_amd import kernels
    N, K = 70, 160
    M = math.prod(lead)
    qs, d, w = weights(N, K, 12)
    x, r = rows(M, K, 13), rows(M, N, 14)
    y = kernels.q4_linear(x.view(*lead, K).to(DEV), qs.to(DEV), d.to(DEV), residual=r.view(*lead, N).to(DEV))
    assert y.shape == (*lead, N) and y.dtype == BF
    if M:
        check(y.view(M, N), x, w, d, residual=r)
    both = r.view(*lead, N).to(DEV)
    assert kernels.q4_linear(x.view(*lead, K).to(DEV), qs.to(DEV), d.to(DEV), residual=both, out=both) is both
    assert torch.equal(both, y)


@pytest.mark.parametrize("M", [3, 50])
def test_strides(gpu_lib, M):
    from opendecider_amd import kernels
    N, K = 100, 352
    qs, d, w = weights(N, K, 5)
    x, r = rows(M, K), rows(M, N, 6)
    want = kernels.q4_linear(x.to(DEV), qs.to(DEV), d.to(DEV), residual=r.to(DEV))
    wide = lambda t, left, right: torch.nn.functional.pad(t.to(DEV), (left, right))
    for left, right in ((0, 8), (8, 16), (1, 0), (0, 3)):
        xs, rs = wide(x, left, right)[:, left:left + K], wide(r, left, right)[:, left:left + N]
        buf = torch.full((M, N + left + right), 3.0, dtype=BF, device=DEV)
        out = buf[:, left:left + N]
        assert kernels.q4_linear(xs, qs.to(DEV), d.to(DEV), residual=rs, out=out) is out
        assert torch.equal(out, want) and (buf[:, :left] == 3).all() and (buf[:, left + N:] == 3).all()
    q2, d2 = wide(qs, 16, 16)[:, 16:16 + K // 2], wide(d, 1, 2)[:, 1:1 + K // 32]
    assert torch.equal(kernels.q4_linear(x.to(DEV), q2, d2, residual=r.to(DEV)), want)
    q3 = wide(qs, 1, 0)[:, 1:]
    assert torch.equal(kernels.q4_linear(x.to(DEV).t().contiguous().t(), q3, d.to(DEV), residual=r.to(DEV)), want)
    assert torch.equal(kernels.q4_linear(x.to(DEV).view(1, M, K), qs.to(DEV), d.to(DEV), residual=r.to(DEV).view(1, M, N)), want[None])
    one = kernels.q4_linear(x[0].to(DEV), qs.to(DEV), d.to(DEV))
    assert one.shape == (N,) and torch.equal(one, kernels.q4_linear(x[:1].to(DEV), qs.to(DEV), d.to(DEV))[0])
    out3 = torch.zeros(2, M, N, dtype=BF, device=DEV).transpose(0, 1)  # (M, 2, N), rows that are no matrix
    x3 = torch.stack([x, x.flip(0)], 1).to(DEV)
    assert torch.equal(kernels.q4_linear(x3, qs.to(DEV), d.to(DEV), out=out3), kernels.q4_linear(x3, qs.to(DEV), d.to(DEV)))


@pytest.mark.parametrize("M", [5, 60])
def test_rows_do_not_mix(gpu_lib, M):
    """A row with NaN or an infinity is NaN; the others are what they were, bit for bit. So is the memory around the rows."""
    from opendecider_amd import kernels
    N, K = 70, 416
    qs, d, w = weights(N, K, 7)
    x = rows(M, K)
    want = kernels.q4_linear(x.to(DEV), qs.to(DEV), d.to(DEV))
    buf = torch.full((M, K + 64), math.nan, dtype=BF, device=DEV)
    buf[:, :K] = x.to(DEV)
    assert torch.equal(kernels.q4_linear(buf[:, :K], qs.to(DEV), d.to(DEV)), want)
    for bad in (math.nan, math.inf, -math.inf):
        x[2, 100] = bad
        got = kernels.q4_linear(x.to(DEV), qs.to(DEV), d.to(DEV))
        assert got[2].isnan().all() and torch.equal(got[:2], want[:2]) and torch.equal(got[3:], want[3:])


@pytest.mark.parametrize("M", [4, 64])
@pytest.mark.parametrize("exp", [-110, -30, 40, 110])
def test_sizes_of_x(gpu_lib, M, exp):
    from opendecider_amd import kernels
    qs, d, w = weights(80, 288, 8)
    x = (rows(M, 288).float() * 2.0 ** (exp - 8 + torch.arange(M)[:, None] % 3 * 4)).to(BF)
    y = kernels.q4_linear(x.to(DEV), qs.to(DEV), d.to(DEV))
    keep = (x.double() @ w.T).abs().amax(1) < 1e38
    tiny = 2.0 ** -126 * 300  # fp32's own range
    yc = y[keep.to(DEV)].double().cpu()
    xk = x[keep]
    if exp > -100:
        check(yc, xk, w, d) if (M <= FEW) == (len(xk) <= FEW) else None
    else:
        assert ((yc - xk.double() @ w.T).abs() <= 2.0 ** -7 * (xk.double().abs() @ w.abs().T) + tiny).all()


@pytest.mark.parametrize("M", [2, 40])
def test_zeros_and_extreme_scales(gpu_lib, M):
    from opendecider_amd import kernels
    qs, d, w = weights(64, 256, 9)
    d[::3] = 0.0
    d[1::3] = d[1::3].sign() * 2.0 ** -24  # fp16's smallest
    d[5] = 8188.0  # -8 d is fp16's largest but one
    u = torch.cat([qs.view(64, 8, 16) & 15, qs.view(64, 8, 16) >> 4], -1).double() - 8
    w = (u * d.double()[..., None]).view(64, 256)
    x = rows(M, 256)
    y = kernels.q4_linear(x.to(DEV), qs.to(DEV), d.to(DEV))
    check(y, x, w, d)
    assert not y[:, ::3].any()


def test_refusals(gpu_lib):
    from opendecider_amd import kernels
    qs, d, _ = weights(20, 64)
    x = rows(3, 64)
    g = lambda t: t.to(DEV)
    for a in ((g(x).float(), g(qs), g(d)), (g(x), g(qs).to(torch.int8), g(d)), (g(x), g(qs), g(d).to(BF)), (g(x), g(qs), g(d), g(x).float())):
        with pytest.raises(TypeError):
            kernels.q4_linear(*a)
    for a in ((g(x)[:, :32], g(qs), g(d)), (g(x), g(qs)[:, :31], g(d)), (g(x), g(qs), g(d)[:, :1]), (g(x), g(qs)[:0], g(d)[:0]),
              (g(x)[:, :24], g(qs)[:, :12], g(d)[:, :1]), (g(x), g(qs), g(d), g(x)[0]), (g(x), g(qs), g(d), None, g(x)),
              (g(x), g(qs), g(d), None, None, g(x))):
        with pytest.raises(ValueError):
            kernels.q4_linear(*a)
    for a in ((x, g(qs), g(d)), (g(x), qs, g(d)), (g(x), g(qs), g(d), None, rows(3, 20))):
        with pytest.raises((RuntimeError, ValueError)):
            kernels.q4_linear(*a)
    assert kernels.q4_linear(g(x)[:0], g(qs), g(d)).shape == (0, 20)


def test_same_calls_same_bits_and_streams(gpu_lib):
    from opendecider_amd import kernels
    for M, N, K in ((1, 500, 4096), (32, 500, 4096), (100, 300, 8192)):
        qs, d, _ = weights(N, K)
        x, qs, d = rows(M, K).to(DEV), qs.to(DEV), d.to(DEV)
        a = kernels.q4_linear(x, qs, d)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            b = kernels.q4_linear(x, qs, d)
        side.synchronize()
        assert torch.equal(a, b) and torch.equal(a, kernels.q4_linear(x, qs, d))


@pytest.mark.parametrize("M", [1, 100])
def test_graph(gpu_lib, M):
    from opendecider_amd import kernels
    qs, d, _ = weights(300, 4096)
    x, qs, d = rows(M, 4096).to(DEV), qs.to(DEV), d.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.q4_linear(x, qs, d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kernels.q4_linear(x, qs, d)
    for seed in range(4):
        x.copy_(rows(M, 4096, seed))
        want = kernels.q4_linear(x, qs, d)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_module(gpu_lib):
    """Q4Linear: the weights of its Q4Table, padded inputs, other activation types; quantize_q4_ over a model."""
    from opendecider_amd import Q4Linear, Q4Table, quantize_q4_
    torch.manual_seed(0)
    lin = nn.Linear(100, 60).to(DEV, BF)
    m = Q4Linear.from_linear(lin)
    w = Q4Table(torch.nn.functional.pad(lin.weight.data, (0, 28)))
    assert torch.equal(m.qs, w.qs) and torch.equal(m.d, w.d) and torch.equal(m.weight, w.weight[:, :100])
    u = torch.cat([m.qs.view(60, 4, 16) & 15, m.qs.view(60, 4, 16) >> 4], -1).double().cpu() - 8
    exact = (u * m.d.double().cpu()[..., None]).view(60, 128)
    for M in (3, 50):
        x, r = rows(M, 100), rows(M, 60, 3)
        check(m(x.to(DEV)), torch.nn.functional.pad(x, (0, 28)), exact, m.d.cpu(), lin.bias.data.cpu())
        check(m(x.to(DEV), r.to(DEV)), torch.nn.functional.pad(x, (0, 28)), exact, m.d.cpu(), lin.bias.data.cpu(), r)
        y = m(x.float().to(DEV))
        assert y.dtype == torch.float32 and torch.equal(y, m(x.to(DEV)).float())
    net = nn.Sequential(nn.Linear(64, 32), nn.Sequential(nn.Linear(32, 32), nn.ReLU()), nn.Linear(32, 8)).to(DEV, BF)
    quantize_q4_(net, skip=("2",))
    assert [type(x).__name__ for x in (net[0], net[1][0], net[2])] == ["Q4Linear", "Q4Linear", "Linear"]
    assert net(rows(2, 64).to(DEV)).shape == (2, 8)
    t = Q4Table(torch.randn(50, 64))
    assert torch.equal(Q4Linear.from_table(t).qs, t.qs)
    with pytest.raises(ValueError):
        m(rows(2, 128).to(DEV))
    with pytest.raises(RuntimeError):
        m(rows(2, 100))
    with pytest.raises(ValueError):
        Q4Linear(m.qs, m.d, in_features=96)
    with pytest.raises(ValueError):
        Q4Linear(m.qs, m.d[:, :2])


def test_a_layer_in_4_bits(gpu_lib):
    """An attention layer of a decode step and of a chunk, over 4-bit weights and a 4-bit cache: projection, norm and rotation with the
    write into pages, attention, output projection with the residual. Each step is right for the inputs it is given."""
    import test_gpu_int4_pages as tg
    from opendecider_amd import kernels
    from oracle import decoder as od
    from oracle import paged as op
    H, hq, hk, D = 256, 4, 2, 64
    for new, ctx in (([1, 1, 1], [40, 0, 17]), ([30, 1, 20], [64, 5, 0])):
        c = tg.rope_case(70, new, ctx, hq, hk, D, D, False, pad=0)
        N = sum(new)
        wqkv, wo = weights((hq + 2 * hk) * D, H, 11), weights(H, hq * D, 12)
        h = rows(N, H)
        qkv = kernels.q4_linear(h.to(DEV), wqkv[0].to(DEV), wqkv[1].to(DEV))
        check(qkv, h, wqkv[2], wqkv[1])
        cfg = od.DecoderConfig(n_heads=hq, n_kv_heads=hk, head_dim=D)
        ref = od.qk_norm_rope(qkv.cpu(), cfg, c["qw"], c["kw"], c["cos"], c["sin"], c["pos"].long())
        c["k"], c["v"] = (ref[:, a * D:b * D].reshape(N, b - a, D) for a, b in ((hq, hq + hk), (hq + hk, hq + 2 * hk)))
        cache = tg.cache_of(c)
        tg.rope_call(c, cache, qkv)
        assert torch.equal(qkv.cpu(), ref)
        tg.same_pools(cache, tg.appended(c, c["k"]))
        q, k, v = (qkv[:, a * D:b * D].view(N, b - a, D) for a, b in ((0, hq), (hq, hq + hk), (hq + hk, hq + 2 * hk)))
        o, lse = kernels.paged_attn(q, k, v, cache, c["table"].to(DEV), c["start"].to(DEV), c["ctx"].to(DEV), D ** -0.5, return_lse=True)
        c.update(q=q.cpu(), scale=D ** -0.5)
        tg.check_attn(c, o, lse)
        y = kernels.q4_linear(o.reshape(N, hq * D), wo[0].to(DEV), wo[1].to(DEV), residual=h.to(DEV))
        check(y, o.reshape(N, hq * D).cpu(), wo[2], wo[1], residual=h)
