"""Batches of the paged attention over 4-bit pages whose rounding errors are few, and a check that one key too many or too few, or
a block's scale 1% off, does not pass (paged_exact.py has the same over int8 pages).

The scales are powers of two within 2^8 of each other, other ones for every 32 values of every key: a value is exact in any of the
kernels' formats (3 significant bits by a power of two, in fp16 in a frame), and so are the queries (8 bits). Keys are small against
sqrt(D), so every key has a share of the output that counts. Every other block of 32 columns has values of mostly one sign, whose
sums are near A below: there an error of the scales shows; in the others, whose sums are smaller, an error of a key. With p_j the
probabilities, A_c and A_n the sums of p_j |v_jd| over the cached and the new keys and A = A_c + A_n, what is left of an output's
error is
  * its own rounding to bf16, 2^-8 |o|;
  * the rounding of the probabilities for the product with the values: 2^-11 A_c (fp16), and for the new keys 2^-16 A_n where they go
    in as bf16 high and low parts (the streaming kernels), else 2^-8 A_n (bf16);
  * the scores' fp32 sums, e <= 2^-24 (D + 8) S with S = max_j scale sum_d |q_d k_jd|, twice over all p_j: 2 e A;
  * fp32 sums over T keys, exp2 and log2, 2^-22 (T + 16) A."""
import math

import torch

from oracle import paged as op
from paged_exact import SHAPES
from test_gpu_paged import BF, make

__all__ = ["SHAPES", "batch", "check"]


def batch(seed, new, ctx, heads, kv, d, **kw):
    """test_gpu_paged.make's batch with 4-bit pages: K's small, V's blocks differing by row and rising from block to block of 64
    positions."""
    c = make(seed, new, ctx, heads, kv, d, int8=False, **kw)
    g = torch.Generator().manual_seed(seed)
    n, _, page, _ = c["pages"][0].shape
    u = [torch.randint(0, 16, (n, kv, page, d // 32, 32), generator=g) for _ in range(2)]
    near = (torch.arange(kv)[:, None, None, None] + torch.arange(d // 32)[:, None] + seed) % 2 == 0
    u[1] = torch.where(near, u[1].clamp_min(9), u[1])
    c["pages"] = [pack(x.flatten(-2)) for x in u]
    exps = [torch.randint(-6, -3, (n, kv, page, d // 32), generator=g).float() for _ in range(2)]
    for b, row in enumerate(c["table"].tolist()):
        for col, p in enumerate(row):
            if p >= 0:
                exps[1][p] += min(col * page // 64, 3)
    c["scales"] = [torch.exp2(e).to(BF) for e in exps]
    c["k"] = (c["k"].float() * 0.3).to(BF)
    return c


def pack(u):
    """Codes (..., D) as the bytes (..., D / 2) of 4-bit rows: value 2 i of 8 at bit 4 i of a word, value 2 i + 1 at bit 16 + 4 i."""
    w = u.unflatten(-1, (-1, 8))
    q = torch.stack([w[..., i] | w[..., i + 2] << 4 for i in (0, 4, 1, 5)], -1)
    return q.to(torch.uint8).flatten(-2)


def check(c, out, lse, stream, own=True, against=None):
    """out and lse as the kernels (stream: the streaming ones) give them for c. against: what op.attention gives for c."""
    new = (c["k"], c["v"]) if own else (None, None)
    args = (*c["pages"], *c["scales"]), c["table"], c["start"], c["ctx"], c["scale"]
    ref, rl, mean, size, _ = against or op.attention(c["q"], *new, *args, c["row_begin"])
    old = mean
    if own:  # the cached keys' part of the mean: their own softmax's by its share of the whole
        _, ol, om, _, _ = op.attention(c["q"], None, None, *args)
        old = om * torch.exp(ol - rl).nan_to_num(0.0)[..., None]
    out, lse = out.double().cpu(), lse.double().cpu()
    live = ~rl.isnan() & (rl > -math.inf)
    D, T = c["q"].shape[2], int((c["ctx"].clamp_min(0) + c["start"][1:] - c["start"][:-1]).max())
    e = 2.0 ** -24 * (D + 8) * size
    p = 2.0 ** -11 * old + (2.0 ** -16 if stream else 2.0 ** -8) * (mean - old).clamp_min(0)
    bound = 2.0 ** -8 * ref.abs() + 1.02 * (p + (2 * e[..., None] + 2.0 ** -22 * (T + 16)) * mean)
    bad = ~((out - ref).abs() <= bound)
    assert not bad[live].any(), f"{int(bad[live].sum())} of {int(live.sum()) * D}: worst {((out - ref).abs() / bound)[live].max()}"
    lb = e + 2.0 ** -20 * (1 + rl.abs() + size)
    assert ((lse - rl).abs() <= lb)[live].all(), f"lse off by {((lse - rl).abs() / lb)[live].max()} of its bound"
