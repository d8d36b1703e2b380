"""The paged K/V cache restated in float64 on the CPU: where a token's row lies, what is written, what is read back, and
attention of packed, ragged new tokens over their sequence's pages."""
from __future__ import annotations

import math

import torch

from .quant import quantize_rows


def pack4(x):
    """bf16 rows (..., D) as 4-bit pages hold them: bytes (..., D / 2) and bf16 scales (..., D / 32). Value by value: per 32, m the
    first of the largest magnitude, d = m / -8, u = floor(x / d + 8.5) within 0..15, in float64 (where x / d + 8.5 of bf16 numbers is
    never on the wrong side of an integer); value 2 i of 8 at bit 4 i of a little-endian word, value 2 i + 1 at bit 16 + 4 i."""
    rows = x.double().reshape(-1, x.shape[-1])
    q = torch.zeros(rows.shape[0], x.shape[-1] // 2, dtype=torch.uint8)
    s = torch.zeros(rows.shape[0], x.shape[-1] // 32, dtype=torch.float64)
    for r, row in enumerate(rows.tolist()):
        for a in range(0, len(row), 32):
            block = row[a:a + 32]
            if all(math.isfinite(v) for v in block):
                m = max(block, key=abs)
                d = 0.0 if abs(m) < 2.0 ** -100 else m / -8.0
                u = [8 if d == 0 else min(15, max(0, math.floor(v / d + 8.5))) for v in block]
            else:
                d, u = math.nan, [8 if math.isfinite(v) else 0 for v in block]
            s[r, a // 32] = d
            for w in range(4):
                word = sum(u[8 * w + i] << (16 * (i % 2) + 4 * (i // 2)) for i in range(8))
                q[r, a // 2 + 4 * w:a // 2 + 4 * w + 4] = torch.tensor(list(word.to_bytes(4, "little")), dtype=torch.uint8)
    return q.view(*x.shape[:-1], -1), s.to(torch.bfloat16).view(*x.shape[:-1], -1)


def values4(q, s):
    """The float64 values (..., D) of 4-bit rows: (u - 8) d, NaN where d is not finite."""
    y = torch.empty(*q.shape[:-1], 2 * q.shape[-1], dtype=torch.float64)
    for i in range(8):  # value i of every word: byte 2 (i % 2) + i / 4, its half i / 2 % 2
        byte = q[..., 2 * (i % 2) + i // 4::4].long()
        y[..., i::8] = ((byte >> 4 * (i // 2 % 2)) & 15).double() - 8
    d = s.double()
    return y * d.masked_fill(~d.isfinite(), math.nan).repeat_interleave(32, -1)


def values(rows, scales):
    """The float64 values of rows (..., D) of any pages."""
    if rows.dtype == torch.uint8:
        return values4(rows, scales)
    return rows.double() if scales is None else rows.double() * scales.double()[..., None]


def place(table, n_pages: int, page: int, b: int, pos: int):
    """(page, row) of position pos of sequence b, or None where there is no page."""
    col = pos // page
    if pos < 0 or col >= table.shape[1]:
        return None
    p = int(table[b, col])
    return (p, pos % page) if 0 <= p < n_pages else None


def sequences(start, N: int):
    """(b, first packed row, end) of every sequence."""
    s = [int(x) for x in start]
    return [(b, s[b], s[b + 1]) for b in range(len(s) - 1) if 0 <= s[b] <= s[b + 1] <= N]


def append(pages, scales, x, table, start, ctx):
    """pages (n_pages, H, page, D) (and fp32 scales (n_pages, H, page) or None; or 4 bits, as pack4 gives them) after the rows
    x (N, H, D) are written: new tensors."""
    pages, scales = pages.clone(), None if scales is None else scales.clone()
    n_pages, _, page, _ = pages.shape
    for b, a, e in sequences(start, x.shape[0]):
        for i in range(e - a):
            at = place(table, n_pages, page, b, max(int(ctx[b]), 0) + i)
            if at is None:
                continue
            if scales is None:
                pages[at[0], :, at[1]] = x[a + i]
            elif pages.dtype == torch.uint8:
                pages[at[0], :, at[1]], scales[at[0], :, at[1]] = pack4(x[a + i])
            else:
                q, s = quantize_rows(x[a + i])
                pages[at[0], :, at[1]], scales[at[0], :, at[1]] = q, s[..., 0]
    return pages, scales


def read(pages, scales, table, length, T: int):
    """(rows (B, H, T, D), scales (B, H, T) or None, valid (B, T)): the stored rows of every sequence, zeros where none is (4-bit
    rows keep their own widths)."""
    n_pages, H, page, D = pages.shape
    B = len(length)
    rows = torch.zeros(B, H, T, D, dtype=pages.dtype)
    sc = None if scales is None else torch.zeros(B, H, T, *scales.shape[3:], dtype=scales.dtype)
    valid = torch.zeros(B, T, dtype=torch.bool)
    for b in range(B):
        for j in range(min(T, max(int(length[b]), 0))):
            at = place(table, n_pages, page, b, j)
            if at is not None:
                rows[b, :, j], valid[b, j] = pages[at[0], :, at[1]], True
                if sc is not None:
                    sc[b, :, j] = scales[at[0], :, at[1]]
    return rows, sc, valid


def attention(q, k, v, pages, table, start, ctx, scale: float, row_begin=None):
    """q (N, Hq, D), k / v (N, H, D) or None, pages = (k, v, k_scale, v_scale). Returns float64 tensors: out (N, Hq, D),
    lse (N, Hq), and what error bounds need: the probability-weighted mean of |v| (N, Hq, D), the largest scale * sum
    |q_d k_d| over the seen keys and the sum of their largest |v_d| (N, Hq). Rows of no sequence are NaN. Only keys that a token sees enter its sums."""
    N, Hq, D = q.shape
    H = pages[0].shape[1]
    rep = Hq // H
    out, mean = (torch.full((N, Hq, D), math.nan, dtype=torch.float64) for _ in range(2))
    lse, size, total = (torch.full((N, Hq), math.nan, dtype=torch.float64) for _ in range(3))
    for b, a, e in sequences(start, N):
        n = e - a
        if n == 0:
            continue
        t = min(max(int(ctx[b]), 0), table.shape[1] * pages[0].shape[2])
        kr, ks, valid = read(pages[0], pages[2], table[b:b + 1], [t], t)
        vr, vs, _ = read(pages[1], pages[3], table[b:b + 1], [t], t)
        kc, vc = (values(r[0], None if x is None else x[0]) for r, x in ((kr, ks), (vr, vs)))
        seen = valid.expand(n, t)
        if k is not None:
            i = torch.arange(n)
            first = torch.zeros(n, dtype=torch.long) if row_begin is None else row_begin[a:e].long().clamp_min(0)
            seen = torch.cat([seen, (i[None] <= i[:, None]) & (i[None] >= first[:, None])], 1)
            kc = torch.cat([kc, k[a:e].double().transpose(0, 1)], 1)
            vc = torch.cat([vc, v[a:e].double().transpose(0, 1)], 1)
        for h in range(Hq):
            qh, kh, vh = q[a:e, h].double(), kc[h // rep], vc[h // rep]
            for i in range(n):  # row by row over its own keys, so that nothing masked can enter
                at = seen[i].nonzero()[:, 0]
                if at.numel() == 0:
                    out[a + i, h], mean[a + i, h], lse[a + i, h], size[a + i, h], total[a + i, h] = 0, 0, -math.inf, 0, 0
                    continue
                y = (kh[at] @ qh[i]) * scale
                p = torch.softmax(y, 0)
                out[a + i, h], mean[a + i, h] = p @ vh[at], p @ vh[at].abs()
                lse[a + i, h] = torch.logsumexp(y, 0)
                size[a + i, h] = (kh[at].abs() @ qh[i].abs()).max() * scale
                total[a + i, h] = vh[at].abs().amax(1).sum()
    return out, lse, mean, size, total
