"""4-bit pages on the CPU: the format against its restatement, what a cache of it checks, and the C ABI's refusals."""
import math

import pytest
import torch

from oracle import paged as op

BF = torch.bfloat16


def rows(seed, *shape):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-20, 20, (*shape[:-1], 1), generator=g).float())).to(BF)


def same(a, b):
    return torch.equal(a.view(torch.int16) if a.dtype == BF else a, b.view(torch.int16) if b.dtype == BF else b)


def odd_blocks():
    """Ties of the largest magnitude, values half way between two codes, zeros, the smallest blocks, infinities and NaN."""
    x = torch.zeros(12, 64, dtype=BF)
    x[0, 5], x[0, 9] = 3.0, -3.0
    x[1, 5], x[1, 9] = -3.0, 3.0
    x[2, :32] = torch.arange(-16, 16).to(BF) / 2 + 0.25  # d = -(-7.75) / 8
    x[3, :16] = (torch.arange(16) - 8).to(BF) + 0.5  # half way: d = 0.9375
    x[4, :17] = torch.arange(-8, 9).to(BF) * 0.5  # m = -4, d = 0.5: all on codes, the last past them
    x[5, :16], x[5, 20] = (torch.arange(16) - 8).to(BF) * 0.5 + 0.25, -4.0  # half way between codes of 0.5
    x[6, 3], x[6, 40] = 2.0 ** -100, 2.0 ** -101
    x[7, 3], x[7, 40] = -2.0 ** -133, 2.0 ** -99
    x[8, 3], x[8, 40] = math.inf, -math.inf
    x[9, 3], x[9, 4], x[9, 40] = math.nan, 1.0, 3e38
    x[10, 31], x[10, 32] = 3.3e38, -3.3e38
    x[11] = -1.0
    return x


@pytest.mark.parametrize("x", [rows(1, 3, 5, 64), rows(2, 40, 128), rows(3, 2, 256), odd_blocks()], ids=["64", "128", "256", "odd"])
def test_pack_is_the_format(x):
    from opendecider_amd import pack_int4, unpack_int4
    q, d = pack_int4(x)
    wq, wd = op.pack4(x)
    assert same(q, wq) and torch.equal(d.isnan(), wd.isnan()) and same(d.nan_to_num(), wd.nan_to_num())
    y, want = unpack_int4(q, d), op.values4(q, d)
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num().double(), want.nan_to_num())
    # off by half a step, or by a whole one at the end that 4 bits do not reach (u = 16 would be 8 d)
    err = (y.double() - x.double()).abs().unflatten(-1, (-1, 32))
    step = d.double().abs()[..., None]
    # (a block below 2^-100 is zero)
    assert (err <= torch.where(step == 0, 2.0 ** -100, step))[~d.isnan()].all()


@pytest.mark.parametrize("seed", range(4))
def test_every_quotient_of_bf16_numbers(seed):
    """x / d is half way between two codes or at least 1 / 1020 away from it: for a largest value of every significand."""
    m = 128 + torch.arange(128, dtype=torch.float64)[seed::4]
    x = 128 + torch.arange(128, dtype=torch.float64)
    for e in range(0, 8):
        t = (x[None] * 2.0 ** -e) / m[:, None] * 8 + 0.5
        away = (t - t.round()).abs()
        assert ((away == 0) | (away >= 1 / 1020))[t <= 8.5].all()


def test_round_trip_of_what_pages_hold():
    """Values that came from 4 bits come back exactly (their largest is -8 d)."""
    from opendecider_amd import pack_int4, unpack_int4
    y = unpack_int4(*pack_int4(rows(7, 50, 128)))
    assert torch.equal(unpack_int4(*pack_int4(y.to(BF))), y)


def test_pack_refusals():
    from opendecider_amd import pack_int4
    with pytest.raises(TypeError):
        pack_int4(torch.zeros(2, 64))
    with pytest.raises(ValueError):
        pack_int4(torch.zeros(2, 48, dtype=BF))


def test_cache_checks():
    from opendecider_amd import PagedKVCache, PagedStates
    c = PagedKVCache(3, 2, 128, 32, "cpu", quantized="int4")
    assert c.k.shape == (3, 2, 32, 64) and c.k_scale.shape == (3, 2, 32, 4) and c.head_dim == 128 and c.page == 32 and c.quantized
    assert c.nbytes() == 2 * 3 * 2 * 32 * (64 + 8)
    assert PagedKVCache(3, 2, 128, 32, "cpu", quantized="int8").k.dtype == torch.int8
    d = PagedKVCache.from_tensors(c.k, c.v, c.k_scale, c.v_scale)
    assert d.format == c.format and d.k is c.k
    with pytest.raises(ValueError):
        PagedKVCache(3, 2, 128, 32, "cpu", quantized="int5")
    for D in (32, 96, 512):
        with pytest.raises(ValueError):
            PagedKVCache(3, 2, D, 32, "cpu", quantized="int4")
    with pytest.raises(ValueError):
        PagedKVCache(3, 2, 128, 24, "cpu", quantized="int4")
    s = c.k_scale
    for ks, vs in ((None, None), (s, None), (s.float(), s.float()), (s[:, :, :, :2], s[:, :, :, :2]), (s, s[:2])):
        with pytest.raises(TypeError):
            PagedKVCache.from_tensors(c.k, c.v, ks, vs)
    with pytest.raises(ValueError):
        PagedKVCache.from_tensors(c.k, c.v, s.transpose(0, 1).contiguous().transpose(0, 1), s)
    with pytest.raises(ValueError):
        PagedKVCache.from_tensors(c.k.transpose(0, 1).contiguous().transpose(0, 1), c.v, s, s)
    states = PagedStates(2, 3, 2, 64, 10, 64, 16, device="cpu", quantized="int4")
    states.reserve([20, 0, 5])
    states.advance([20, 0, 5])
    assert states.lengths == [20, 0, 5] and states[1].k.shape == (10, 2, 16, 32)


def test_abi_refusals():
    """Codes of the entry points for what they do not take; nothing is launched."""
    import ctypes

    from opendecider_amd import _lib
    L = _lib.lib()
    P, odd = ctypes.c_void_p(64), ctypes.c_void_p(72)
    NULL, SHAPE, ALIGN, UNSUP = -1, -2, -3, -4

    def append(fmt=2, ks=P, vs=P, pages=4, page=16, D=128, k=P):
        return L.od_page_append_ex(k, 256, 128, P, 256, 128, fmt, P, ks, P, vs, pages, page, P, 4, 4, P, P, 1, 2, 2, D, None)

    assert append(fmt=3) == UNSUP and append(fmt=-1) == UNSUP and append(D=32) == UNSUP and append(page=24) == UNSUP
    assert append(ks=None) == NULL and append(ks=None, vs=None) == NULL and append(fmt=1, ks=None, vs=None) == NULL
    assert append(k=None) == NULL and append(ks=odd) == ALIGN and append(pages=-1) == SHAPE

    def read(form, fmt=2, out=P):
        return L.od_page_read_ex(fmt, P, P, P, P, 4, 16, P, 4, 4, P, 1, 8, 2, 128, form, out, P, P, P, None)

    assert read(2) == UNSUP and read(3) == UNSUP and read(0, out=None) == NULL and read(0, fmt=7) == UNSUP

    def attn(fmt=2, scale=0.1, ks=P, B=1, Hq=4):
        return L.od_paged_attn_ex(P, 512, 128, P, 256, 128, P, 256, 128, fmt, P, ks, P, P, 4, 16, P, 4, 4, P, P, None, P, 512, 128,
                                  None, B, 2, Hq, 2, 128, 1, 8, scale, None, 0, None)

    assert attn(fmt=9) == UNSUP and attn(scale=0.0) == UNSUP and attn(ks=None) == NULL and attn(ks=odd) == ALIGN
    assert attn(B=70000) == SHAPE and attn(Hq=5) == UNSUP
    n = ctypes.c_int64(0)
    assert L.od_paged_attn_ws_ex(1, 1, 4, 2, 128, 1, 8, 5, ctypes.byref(n)) == UNSUP
    assert L.od_paged_attn_ws_ex(1, 1, 4, 2, 128, 1, 8, 2, None) == NULL

    def rope(ld=768, ldo=512, D=128, rot=128, zc=0, fmt=2, out=P, qw=P, start=P, hq=2, qkv=P):
        return L.od_qk_norm_rope_page_append(qkv, ld, out, ldo, hq, rot, zc, qw, P, P, P, 16, P, 1e-6, fmt, P, P, P, P, 4, 16, P, 4,
                                             4, start, P, 1, 2, 2, D, None)

    assert rope(ld=760) == SHAPE and rope(ldo=500) == SHAPE and rope(hq=-1) == SHAPE and rope(rot=64) == UNSUP and rope(zc=2) == UNSUP
    assert rope(fmt=4) == UNSUP and rope(D=96) == UNSUP and rope(out=None) == NULL and rope(qw=None) == NULL and rope(start=None) == NULL
    assert rope(ld=772) == ALIGN and rope(qkv=odd) == ALIGN and rope(out=odd) == ALIGN and rope(qw=odd) == ALIGN

    def linear(M=4, N=64, K=128, ldx=128, ldq=64, ldd=4, ldo=64, x=P, qs=P, d=P, out=P, ws=None, nws=0, res=None, ldr=64):
        return L.od_q4_linear(x, ldx, qs, ldq, d, ldd, None, res, ldr, out, ldo, M, N, K, ws, nws, None)

    for bad in (dict(M=-1), dict(N=0), dict(K=0), dict(K=100), dict(ldx=120), dict(ldq=48), dict(ldd=3), dict(ldo=60), dict(res=P, ldr=60),
                dict(M=1 << 23), dict(ldx=1 << 22), dict(M=40, ws=P, nws=3)):
        assert linear(**bad) == SHAPE, bad
    for bad in (dict(x=None), dict(qs=None), dict(d=None), dict(out=None), dict(M=40)):
        assert linear(**bad) == NULL, bad
    for bad in (dict(x=odd), dict(qs=odd), dict(ldx=132), dict(ldq=72), dict(d=ctypes.c_void_p(65)), dict(M=40, ws=odd, nws=1 << 30)):
        assert linear(**bad) == ALIGN, bad
    assert linear(M=0, x=None) == 0
    assert L.od_q4_linear_ws(4, 64, 100, ctypes.byref(n)) == SHAPE and L.od_q4_linear_ws(4, 64, 128, None) == NULL
    assert L.od_q4_linear_ws(32, 64, 128, ctypes.byref(n)) == 0 and n.value == 0
    assert L.od_q4_linear_ws(33, 64, 128, ctypes.byref(n)) == 0 and n.value >= 33 * 128 // 2
