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
    page), the bytes and scales of Int8KVCache, or with quantized=False bf16 pages without scales. page is a power of two
    of at least 16, D 64, 128 or 256."""

    __slots__ = ("k", "v", "k_scale", "v_scale")

    def __init__(self, n_pages: int, n_heads: int, head_dim: int, page: int = 64, device="cuda", quantized: bool = True):
        dtype = torch.int8 if quantized else torch.bfloat16
        k, v = (torch.zeros(n_pages, n_heads, page, head_dim, dtype=dtype, device=device) for _ in range(2))
        ks, vs = (torch.zeros(n_pages, n_heads, page, dtype=torch.float32, device=device) if quantized else None
                  for _ in range(2))
        self._set(k, v, ks, vs)

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                     v_scale: torch.Tensor | None = None) -> "PagedKVCache":
        """A cache over existing contiguous pools: int8 with fp32 scales, or bf16 without."""
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
        elif k.dtype != torch.bfloat16:
            raise TypeError(f"PagedKVCache: pages are int8 or bfloat16, got {k.dtype}")
        elif ks is not None or vs is not None:
            raise TypeError("PagedKVCache: bf16 pages have no scales")
        if any(x is not None and x.device != k.device for x in (v, ks, vs)):
            raise ValueError("PagedKVCache: the pages and scales must be on one device")
        if not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("PagedKVCache: the pages must be contiguous")
        if shape[2] < 16 or shape[2] & (shape[2] - 1):
            raise ValueError(f"PagedKVCache: the page size must be a power of two of at least 16, got {shape[2]}")
        if shape[3] not in (64, 128, 256):
            raise ValueError(f"PagedKVCache: head_dim must be 64, 128 or 256, got {shape[3]}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, ks, vs

    @property
    def page(self) -> int:
        return self.k.shape[2]

    @property
    def quantized(self) -> bool:
        return self.k_scale is not None

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None)


class PagedStates:
    """Every layer's pages of `batch` states: one pool of n_pages pages per layer, one table (batch, max_tokens / page) for
    all layers on the device (-1: no page), the states' lengths on the host (`lengths`) and on the device (`ctx`). Indexing
    and iteration give the layers' PagedKVCache. reserve -> write (every layer) -> advance appends tokens; these steps, and
    release, change the host's side too and are refused while a graph is captured."""

    def __init__(self, n_layers: int, batch: int, n_heads: int, head_dim: int, n_pages: int, max_tokens: int, page: int = 64,
                 device="cuda", quantized: bool = True):
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
