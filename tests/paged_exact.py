"""Batches of the paged attention over int8 pages whose rounding errors are few, and a check that one key too many or too few,
or a value scale 1% off, does not pass.

The scales are powers of two within 2^8 of each other: an int8 row is then exact in any of the kernels' formats (7 bits times
a power of two, in bf16 or in fp16 in a frame), and so are the queries (8 bits). Keys are small against sqrt(D), so every key
has a share of the output that counts. With p_j the probabilities, A_c and A_n the sums of p_j |v_jd| over the cached and the
new keys and A = A_c + A_n, what is left of an output's error is
  * its own rounding to bf16, 2^-8 |o|;
  * the rounding of the probabilities for the product with the values: 2^-16 A where they go in as bf16 high and low parts
    (the streaming kernels: two half steps of 2^-8, one of the other's remainder); else 2^-11 A_c (fp16) and 2^-8 A_n (bf16)
  * the scores' fp32 sums, e <= 2^-24 (D + 8) S with S = max_j scale sum_d |q_d k_jd|, twice over all p_j: 2 e A;
  * fp32 sums over T keys, exp2 and log2, 2^-22 (T + 16) A."""
import math

import torch

from oracle import paged as op
from test_gpu_paged import BF, make

SHAPES = [  # new tokens, cached tokens: the borders of tiles of 16, 32 and 64 keys, and of the splits' last ones
    ([5], [63]), ([33, 64, 7], [64, 65, 130]), ([130], [200]), ([1, 1, 1], [1, 15, 129]), ([3, 1], [32, 33]), ([70, 2], [127, 0]),
    ([1], [700]),
]


def batch(seed, new, ctx, heads, kv, d, **kw):
    """test_gpu_paged.make's batch with int8 pages of uniform values under power-of-two scales: K's are small, V's differ from
    row to row and rise from block to block of 64 positions."""
    c = make(seed, new, ctx, heads, kv, d, **kw)
    g = torch.Generator().manual_seed(seed)
    n, _, page, _ = c["pages"][0].shape
    c["pages"] = [torch.randint(-127, 128, (n, kv, page, d), generator=g).to(torch.int8) for _ in range(2)]
    exps = torch.randint(-7, -5, (n, kv, page), generator=g).float()
    for b, row in enumerate(c["table"].tolist()):
        for col, p in enumerate(row):
            if p >= 0:
                exps[p] += min(col * page // 64, 3)
    c["scales"] = [torch.full((n, kv, page), 2.0 ** -8), torch.exp2(exps)]
    c["k"] = (c["k"].float() * 0.3).to(BF)
    return c


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
    p = 2.0 ** -16 * mean if stream else 2.0 ** -11 * old + 2.0 ** -8 * (mean - old).clamp_min(0)
    bound = 2.0 ** -8 * ref.abs() + 1.02 * (p + (2 * e[..., None] + 2.0 ** -22 * (T + 16)) * mean)
    bad = ~((out - ref).abs() <= bound)
    assert not bad[live].any(), f"{int(bad[live].sum())} of {int(live.sum()) * D}: worst {((out - ref).abs() / bound)[live].max()}"
    lb = e + 2.0 ** -20 * (1 + rl.abs() + size)
    assert ((lse - rl).abs() <= lb)[live].all(), f"lse off by {((lse - rl).abs() / lb)[live].max()} of its bound"
