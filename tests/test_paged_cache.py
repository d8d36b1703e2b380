"""The paged K/V cache without a GPU: its restatement against brute force, the pages' bookkeeping, and the refusals of the
C ABI (host checks before any launch)."""
import ctypes
import math
import os

import pytest
import torch

from oracle import paged as op

OK, NULL, SHAPE, ALIGN, UNSUP = 0, -1, -2, -3, -4
P = 0x10000  # never dereferenced: every call below is refused or has nothing to do


@pytest.fixture(scope="module")
def L():
    from opendecider_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from opendecider_amd.build import build
        build()
    return _lib.lib()


def test_oracle_attention_against_loops():
    """Scalar loops from the definition: each key's place looked up, seen or not, one softmax."""
    g = torch.Generator().manual_seed(0)
    kp, vp = torch.randn(5, 2, 16, 8, generator=g), torch.randn(5, 2, 16, 8, generator=g)
    table = torch.tensor([[3, 1, -1], [4, 9, 0]], dtype=torch.int32)
    start, ctx = [0, 3, 5], [20, 40]
    q, k, v = (torch.randn(5, h, 8, generator=g) for h in (4, 2, 2))
    begin = torch.tensor([0, 1, 1, -2, 5], dtype=torch.int32)
    out, lse, *_ = op.attention(q, k, v, (kp, vp, None, None), table, start, ctx, 0.3, begin)
    for b in range(2):
        for n in range(start[b], start[b + 1]):
            i = n - start[b]
            for h in range(4):
                keys = []
                for j in range(ctx[b]):
                    col = j // 16
                    pg = int(table[b, col]) if col < 3 else -1
                    if 0 <= pg < 5:
                        keys.append((kp[pg, h // 2, j % 16], vp[pg, h // 2, j % 16]))
                keys += [(k[start[b] + j, h // 2], v[start[b] + j, h // 2]) for j in range(max(int(begin[n]), 0), i + 1)]
                e = [math.exp(0.3 * float((a.double() * q[n, h].double()).sum())) for a, _ in keys]
                want = sum(w * x.double() for w, (_, x) in zip(e, keys)) / sum(e)
                assert torch.allclose(out[n, h], want, atol=1e-12) and abs(float(lse[n, h]) - math.log(sum(e))) < 1e-12


def test_oracle_append_then_read():
    g = torch.Generator().manual_seed(1)
    table = torch.tensor([[2, 0], [1, -1]], dtype=torch.int32)
    x = torch.randn(23, 3, 64, generator=g).to(torch.bfloat16)
    pages, _ = op.append(torch.zeros(3, 3, 16, 64, dtype=torch.bfloat16), None, x, table, [0, 20, 23], [0, 15])
    rows, _, valid = op.read(pages, None, table, [20, 18], 20)
    assert torch.equal(rows[0].transpose(0, 1), x[:20]) and valid[0].all()
    assert torch.equal(rows[1, :, 15], x[20]) and not valid[1, 16:].any() and not rows[1, :, 16:].any()


def test_states_take_and_return_pages():
    from opendecider_amd import PagedStates
    s = PagedStates(2, 3, 2, 64, n_pages=6, max_tokens=100, page=16, device="cpu")
    assert len(s) == 2 and s.cols == 7 and s.batch == 3
    s.reserve([20, 0, 16])
    assert [len(p) for p in s.pages] == [2, 0, 1] and (s.table >= 0).sum() == 3
    s.advance([20, 0, 16])
    assert s.lengths == [20, 0, 16] and s.ctx.tolist() == [20, 0, 16]
    s.reserve([12, 0, 0])  # fits the page that is there
    assert len(s.free) == 3
    before = s.table.clone()
    with pytest.raises(MemoryError):
        s.reserve([0, 33, 17])
    assert len(s.free) == 3 and torch.equal(s.table, before)
    with pytest.raises(ValueError):
        s.reserve([93, 0, 0])
    with pytest.raises(ValueError):
        s.reserve([1, 1])
    with pytest.raises(ValueError):
        s.reserve([1, -1, 0])
    with pytest.raises(ValueError):
        s.advance([0, 1, 0])
    held = set(s.pages[0])
    s.release(0)
    assert s.lengths[0] == 0 and (s.table[0] == -1).all() and held <= set(s.free) and s.ctx.tolist()[0] == 0
    s.reserve([0, 48, 16])
    used = [p for ps in s.pages for p in ps]
    assert len(used) == len(set(used)) == 5


def test_cache_refusals():
    from opendecider_amd import PagedKVCache
    z = lambda *s, dt=torch.int8: torch.zeros(*s, dtype=dt)
    k, sc = z(2, 1, 16, 64), z(2, 1, 16, dt=torch.float32)
    PagedKVCache.from_tensors(k, k, sc, sc)
    for bad in ((k, k), (k, k, sc, sc.double()), (k, k, sc, None), (k, k, sc, z(2, 1, 8, dt=torch.float32)),
                (k.float(), k.float()), (k.bfloat16(), k.bfloat16(), sc, sc)):
        with pytest.raises(TypeError):
            PagedKVCache.from_tensors(*bad)
    for bad in ((k, z(2, 1, 16, 128), sc, sc), (k[:, :, :8], k[:, :, :8], sc[:, :, :8], sc[:, :, :8]),
                (z(2, 1, 48, 64), z(2, 1, 48, 64), *[z(2, 1, 48, dt=torch.float32)] * 2),
                (z(2, 1, 16, 96), z(2, 1, 16, 96), sc, sc), (k, k.bfloat16(), sc, sc)):
        with pytest.raises(ValueError):
            PagedKVCache.from_tensors(*bad)


def test_abi_refusals(L):
    def append(k=P, skt=128, kp=P, ks=P, vs=P, n=4, page=16, ld=3, cols=3, start=P, B=2, N=5, H=2, D=64):
        return L.od_page_append(k, skt, 64, P, 128, 64, kp, ks, P, vs, n, page, P, ld, cols, start, P, B, N, H, D, None)
    assert append(D=96) == UNSUP and append(page=24) == UNSUP and append(page=8) == UNSUP
    assert append(ld=2) == SHAPE and append(B=-1) == SHAPE and append(H=0) == SHAPE and append(n=-1) == SHAPE
    assert append(cols=1 << 29, ld=1 << 29) == SHAPE  # positions past 31 bits
    assert append(ks=None) == NULL and append(kp=None) == NULL and append(k=None) == NULL and append(start=None) == NULL
    assert append(skt=4) == ALIGN and append(k=P + 8) == ALIGN and append(kp=P + 4) == ALIGN
    assert append(N=0) == OK and append(B=0) == OK and append(n=0, kp=None) == OK

    def read(kp=P, ks=P, vs=P, page=16, length=P, T=4, form=0, ko=P, kso=None, D=64):
        return L.od_page_read(kp, ks, P, vs, 4, page, P, 3, 3, length, 2, T, 2, D, form, ko, kso, P, kso, None)
    assert read(form=3) == UNSUP and read(form=2, ks=None, vs=None) == UNSUP and read(form=2) == NULL and read(T=-1) == SHAPE
    assert read(length=None) == NULL and read(ko=None) == NULL and read(ko=P + 8) == ALIGN and read(D=32) == UNSUP
    assert read(T=0) == OK

    def attn(q=P, sq=256, k=P, v=P, ks=P, page=16, out=P, so=256, N=5, Hq=4, H=2, D=64, mn=5, mc=9, scale=0.1, start=P, ws=0):
        return L.od_paged_attn(q, sq, 64, k, 128, 64, v, 128, 64, P, ks, P, ks, 4, page, P, 3, 3, start, P, None, out, so, 64, None,
                               2, N, Hq, H, D, mn, mc, scale, None, ws, None)
    assert attn(Hq=3) == UNSUP and attn(D=80) == UNSUP and attn(page=17) == UNSUP and attn(Hq=0) == SHAPE
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        assert attn(scale=bad) == UNSUP
    assert attn(q=None) == NULL and attn(out=None) == NULL and attn(k=None) == NULL and attn(v=None) == NULL
    assert attn(start=None) == NULL and attn(mn=-1) == SHAPE and attn(mc=-1) == SHAPE
    assert attn(sq=68) == ALIGN and attn(so=4) == ALIGN and attn(out=P + 2) == ALIGN
    assert attn(N=0) == OK
    n = ctypes.c_int64(-1)
    assert L.od_paged_attn_ws(2, 0, 4, 2, 64, 1, 1000, ctypes.byref(n)) == OK and n.value == 0
    assert L.od_paged_attn_ws(2, 5, 4, 3, 64, 1, 1000, ctypes.byref(n)) == UNSUP
    assert L.od_paged_attn_ws(2, -1, 4, 2, 64, 1, 1000, ctypes.byref(n)) == SHAPE
    assert L.od_paged_attn_ws(2, 5, 4, 2, 64, 1, 1000, None) == NULL


def test_no_cpu_path():
    from opendecider_amd import PagedKVCache, kernels
    c = PagedKVCache(2, 1, 64, 16, "cpu")
    x, i = torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        kernels.page_append(x, x, c, i[None], i, i[:1])
    with pytest.raises(RuntimeError):
        kernels.page_read(c, i[None], i[:1], 4)
    with pytest.raises(RuntimeError):
        kernels.paged_attn(x, x, x, c, i[None], i, i[:1], 0.1)


def test_workspace_of_any_hint():
    """The lengths are hints: past any call's own size they ask for no more (what a split holds stays countable), and a call
    with more slots of a KV head than an int counts is refused."""
    import ctypes
    from opendecider_amd._lib import lib

    def ws(*sizes, want=0):
        n = ctypes.c_int64(-1)
        assert (lib().od_paged_attn_ws(*sizes, ctypes.byref(n)) == 0) == (want == 0)
        return n.value
    for n, rep in ((1, 1), (8, 4), (700, 4), (4096, 8)):
        most = ws(2, n, 8 * rep, 8, 128, n, 1 << 30)
        for new, ctx in ((1 << 40, 1 << 30), (n, 1 << 31), (1 << 62, (1 << 62) + 1)):
            assert ws(2, n, 8 * rep, 8, 128, new, ctx) == most
        assert most % (n * 8 * rep * 129) == 0 and most <= 128 * n * 8 * rep * 129
    ws(1, 1 << 29, 64, 1, 128, 1, 100, want="refused")


def test_cache_on_one_device():
    from opendecider_amd import PagedKVCache
    k, sc = torch.zeros(2, 1, 16, 64, dtype=torch.int8), torch.zeros(2, 1, 16)
    for bad in ((k, k.to("meta"), sc, sc), (k, k, sc, sc.to("meta"))):
        with pytest.raises(ValueError):
            PagedKVCache.from_tensors(*bad)


def test_workspace_by_page_type():
    """bf16 pages have no image; a workspace for either type is the larger one."""
    import ctypes
    from opendecider_amd._lib import lib
    n = [ctypes.c_int64(-1) for _ in range(3)]
    sizes = (1, 2048, 32, 8, 128, 2048, 32768)
    assert lib().od_paged_attn_ws_of(*sizes, 1, ctypes.byref(n[0])) == lib().od_paged_attn_ws_of(*sizes, 0, ctypes.byref(n[1])) == 0
    assert lib().od_paged_attn_ws(*sizes, ctypes.byref(n[2])) == 0
    assert n[0].value >= 32768 * 8 * 128 > n[1].value and n[2].value == max(n[0].value, n[1].value)
    assert lib().od_paged_attn_ws_of(*sizes, 1, None) == NULL
