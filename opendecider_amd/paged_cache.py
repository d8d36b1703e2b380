"""A paged K/V cache: states of different lengths that grow and end on their own, in one pool of pages.

Int8KVCache holds every state of a batch at one common length in a rectangle of its own; here a state is a row of page
numbers, so a batch may be ragged in what it holds and in what it adds, and memory is taken page by page. (Tables of a caller's
own may name a page in several sequences, for reading; PagedStates gives each state pages of its own.) The operators over it (kernels.page_append, page_read, paged_attn) take a batch's new
tokens packed, sequence after sequence, with the offsets `start`.
"""
from __future__ import annotations

import torch

from . import kernels


class PagedKVCache:
    """One layer's K and V in pages: k and v int8 (n_pages, Hkv, page, D) with k_scale and v_scale fp32 (n_pages, Hkv,
    page), the bytes and scales of Int8KVCache (quantized True or "int8"); with quantized=False bf16 pages without scales; with
    quantized="int4" 4 bits a value, uint8 (n_pages, Hkv, page, D / 2) with bf16 scales (n_pages, Hkv, page, D / 32), one per 32
    values (pack_int4, unpack_int4). page is a power of two of at least 16, D 64, 128 or 256."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "format", "head_dim")

    def __init__(self, n_pages: int, n_heads: int, head_dim: int, page: int = 64, device="cuda",
                 quantized: bool | str = True):
        quantized = quantized if isinstance(quantized, str) else bool(quantized)
        if quantized not in kernels.PAGE_FORMATS:
            raise ValueError(f"PagedKVCache: quantized must be True, False, 'int8' or 'int4', got {quantized!r}")
        if head_dim not in (64, 128, 256):  # (half of an odd one would be the width of another)
            raise ValueError(f"PagedKVCache: head_dim must be 64, 128 or 256, got {head_dim}")
        dtype, width, scales = {0: (torch.bfloat16, head_dim, None), 1: (torch.int8, head_dim, ((), torch.float32)),
                                2: (torch.uint8, head_dim // 2, ((head_dim // 32,), torch.bfloat16))}[kernels.PAGE_FORMATS[quantized]]
        k, v = (torch.zeros(n_pages, n_heads, page, width, dtype=dtype, device=device) for _ in range(2))
        ks, vs = (torch.zeros(n_pages, n_heads, page, *scales[0], dtype=scales[1], device=device) if scales else None
                  for _ in range(2))
        self._set(k, v, ks, vs)

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                     v_scale: torch.Tensor | None = None) -> "PagedKVCache":
        """A cache over existing contiguous pools: int8 with fp32 scales, uint8 (4 bits) with bf16 scales, or bf16 without."""
        c = cls.__new__(cls)
        c._set(k, v, k_scale, v_scale)
        return c

    def _set(self, k, v, ks, vs) -> None:
        shape = k.shape
        if k.dim() != 4 or v.shape != shape or v.dtype != k.dtype:
            raise ValueError("PagedKVCache: k and v must be (n_pages, Hkv, page, D) of one type")
        if k.dtype == torch.int8:
            if ks is None or vs is None or ks.dtype != torch.float32 or vs.dtype != torch.float32 or \
                    ks.shape != shape[:3] or vs.shape != shape[:3]:
                raise TypeError("PagedKVCache: int8 pages need fp32 scales (n_pages, Hkv, page)")
            if not (ks.is_contiguous() and vs.is_contiguous()):
                raise ValueError("PagedKVCache: the scales must be contiguous")
        elif k.dtype == torch.uint8:
            if ks is None or vs is None or ks.dtype != torch.bfloat16 or vs.dtype != torch.bfloat16 or \
                    ks.shape != (*shape[:3], shape[3] // 16) or vs.shape != ks.shape:
                raise TypeError("PagedKVCache: 4-bit pages (n_pages, Hkv, page, D / 2) need bf16 scales (n_pages, Hkv, page, D / 32)")
            if not (ks.is_contiguous() and vs.is_contiguous()):
                raise ValueError("PagedKVCache: the scales must be contiguous")
        elif k.dtype != torch.bfloat16:
            raise TypeError(f"PagedKVCache: pages are int8, uint8 (4 bits) or bfloat16, got {k.dtype}")
        elif ks is not None or vs is not None:
            raise TypeError("PagedKVCache: bf16 pages have no scales")
        if any(x is not None and x.device != k.device for x in (v, ks, vs)):
            raise ValueError("PagedKVCache: the pages and scales must be on one device")
        if not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("PagedKVCache: the pages must be contiguous")
        if shape[2] < 16 or shape[2] & (shape[2] - 1):
            raise ValueError(f"PagedKVCache: the page size must be a power of two of at least 16, got {shape[2]}")
        four = k.dtype == torch.uint8
        head_dim = shape[3] * (2 if four else 1)
        if head_dim not in (64, 128, 256):
            raise ValueError(f"PagedKVCache: head_dim must be 64, 128 or 256, got {head_dim}")
        self.k, self.v, self.k_scale, self.v_scale, self.head_dim = k, v, ks, vs, head_dim
        self.format = kernels.PAGE_FORMATS["int4" if four else ks is not None]  # OD_PAGE_*

    @property
    def page(self) -> int:
        return self.k.shape[2]

    @property
    def quantized(self) -> bool:
        return self.k_scale is not None

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None)


_ORDER = (0, 2, 4, 6, 1, 3, 5, 7)  # the values of 8 in the order of their four bits


def pack_int4(x: torch.Tensor):
    """bf16 values (..., D), D a multiple of 32, as a 4-bit cache holds them: uint8 (..., D / 2) and bf16 scales (..., D / 32), the
    bytes of kernels.page_append. Per 32 values: m the one of the largest magnitude (the first of several), d = m / -8,
    u = floor(x / d + 8.5) within 0..15 for (u - 8) d; a block below 2^-100 is d = 0, u = 8; with an infinity or NaN d is NaN."""
    if x.dtype != torch.bfloat16:
        raise TypeError(f"pack_int4: expected bfloat16, got {x.dtype}")
    if x.shape[-1] % 32:
        raise ValueError(f"pack_int4: blocks of 32 values, got {x.shape[-1]}")
    g = x.double().unflatten(-1, (-1, 32))
    size = g.abs().nan_to_num(nan=float("inf"), posinf=float("inf"))
    m = g.gather(-1, size.argmax(-1, keepdim=True))
    odd = size.amax(-1, keepdim=True).isinf()
    none = m.abs() < 2.0 ** -100
    d = (m / -8.0).masked_fill(none, 0.0)
    u = torch.floor(g / d.masked_fill(none | odd, 1.0) + 8.5).clamp_(0, 15).masked_fill(none, 8.0)
    u = torch.where(odd, torch.where(g.isfinite(), 8.0, 0.0), u).to(torch.uint8).flatten(-2)
    u = u.unflatten(-1, (-1, 8))[..., _ORDER].flatten(-2)
    return u[..., 0::2] | (u[..., 1::2] << 4), d.masked_fill(odd, float("nan"))[..., 0].to(torch.bfloat16)


def unpack_int4(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """The fp32 values (..., D) of a 4-bit cache's bytes (..., D / 2) and scales (..., D / 32), each exact."""
    u = torch.stack([q & 15, q >> 4], -1).flatten(-2).unflatten(-1, (-1, 2, 4)).transpose(-1, -2).flatten(-3)
    return ((u.float() - 8.0).unflatten(-1, (-1, 32)) * scale.float()[..., None]).flatten(-2)


class PagedStates:
    """Every layer's pages of `batch` states: one pool of n_pages pages per layer, one table (batch, max_tokens / page) for
    all layers on the device (-1: no page), the states' lengths on the host (`lengths`) and on the device (`ctx`). Indexing
    and iteration give the layers' PagedKVCache. reserve -> write (every layer) -> advance appends tokens; these steps, and
    release, change the host's side too and are refused while a graph is captured."""

    def __init__(self, n_layers: int, batch: int, n_heads: int, head_dim: int, n_pages: int, max_tokens: int, page: int = 64,
                 device="cuda", quantized: bool | str = True):
        self.layers = [PagedKVCache(n_pages, n_heads, head_dim, page, device, quantized) for _ in range(n_layers)]
        self.page = page
        self.pages: list[list[int]] = [[] for _ in range(batch)]  # each state's pages, in order
        self.free = list(range(n_pages - 1, -1, -1))
        self.lengths = [0] * batch
        self.cols = -(-max_tokens // page)
        self.table = torch.full((batch, self.cols), -1, dtype=torch.int32, device=device)
        self.ctx = torch.zeros(batch, dtype=torch.int32, device=device)

    def __len__(self) -> int:
        return len(self.layers)

    def __getitem__(self, li) -> PagedKVCache:
        return self.layers[li]

    def __iter__(self):
        return iter(self.layers)

    @property
    def batch(self) -> int:
        return len(self.lengths)

    def reserve(self, counts) -> None:
        """Pages for counts[b] more tokens of every state b. MemoryError (nothing taken) where the pool has too few."""
        self._not_captured("reserve")
        counts = [int(n) for n in counts]
        if len(counts) != self.batch or min(counts, default=0) < 0:
            raise ValueError("PagedStates: one count of new tokens per state")
        need = [max(0, -(-(t + n) // self.page) - len(p)) for t, n, p in zip(self.lengths, counts, self.pages)]
        longest = max((t + n for t, n in zip(self.lengths, counts)), default=0)
        if longest > self.cols * self.page:
            raise ValueError(f"PagedStates: {longest} tokens exceed the table's {self.cols * self.page}")
        if sum(need) > len(self.free):
            raise MemoryError(f"PagedStates: {sum(need)} pages wanted, {len(self.free)} free")
        for b, n in enumerate(need):
            if n:
                got = [self.free.pop() for _ in range(n)]
                at = len(self.pages[b])
                self.pages[b] += got
                self._put(self.table[b, at:at + n], got)

    def advance(self, counts) -> None:
        """Counts the tokens that every layer has written since reserve."""
        self._not_captured("advance")
        counts = [int(n) for n in counts]
        if len(counts) != self.batch or min(counts, default=0) < 0:
            raise ValueError("PagedStates: one count of new tokens per state")
        lengths = [t + n for t, n in zip(self.lengths, counts)]
        if any(t > len(p) * self.page for t, p in zip(lengths, self.pages)):
            raise ValueError("PagedStates: advance past the reserved pages")
        self.lengths = lengths
        self._write_ctx()

    def release(self, b: int) -> None:
        """State b ends: its pages go back to the pool and it is empty."""
        self._not_captured("release")
        self.free += self.pages[b][::-1]
        self.pages[b] = []
        self.table[b].fill_(-1)
        self.lengths[b] = 0
        self._write_ctx()

    def _not_captured(self, name: str) -> None:
        if self.ctx.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"PagedStates.{name} cannot be captured: a replay would write the lengths and pages of the capture "
                               "again, whatever the states have come to since")

    def _write_ctx(self) -> None:
        self._put(self.ctx, self.lengths)

    @staticmethod
    def _put(out: torch.Tensor, values: list) -> None:
        if out.is_cuda:
            kernels.fill_i32(values, out)
        else:
            out.copy_(torch.tensor(values, dtype=torch.int32))

    def read(self, li: int, dtype=torch.bfloat16):
        """Layer li's cached K and V as dense (batch, Hkv, T, D), T the longest state (kernels.page_read)."""
        return kernels.page_read(self.layers[li], self.table, self.ctx, max(self.lengths, default=0), dtype=dtype)
