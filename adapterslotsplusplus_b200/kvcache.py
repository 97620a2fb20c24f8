"""A paged key/value cache held in 4 bits, and the attention that reads it.

KvCache4 keeps K and V of every token as 4-bit codes with one (scale, zero)
pair per token and kv head (layout and format: wp_kv4_append in
include/wp_api.h): D + 8 bytes per token and kv head instead of 4 D. Pages are
handed out by the caller, who keeps the page table; all index tensors live on
the device, so a step is graph-capturable.

One step of a batch (sequence b brings cu[b + 1] - cu[b] new tokens, lens[b]
is its length with those included):

    cache.append(k, v, table, lens, cu)               # the new tokens' K and V
    out = cache.attention(q, table, lens, cu, max_q)  # each sees all before it

With one token per sequence cu is left out. A later chunk of a prompt reads
its context back with `read` and runs WarpPipeEngine.prompt_attention on it.
"""

from __future__ import annotations

import math
from typing import Dict, Optional, Tuple

import torch

from . import _lib
from .engine import WarpPipeEngine, _DTYPES, _empty_rows, _index, _packed_rows, _stream_ptr


class KvCache4:
    TILE = 16

    def __init__(self, engine: WarpPipeEngine, num_pages: Optional[int] = None, kv_heads: Optional[int] = None,
                 head_dim: Optional[int] = None, page_size: int = 64, dtype=torch.bfloat16,
                 pages: Optional[torch.Tensor] = None):
        """A cache of num_pages pages of page_size tokens (a multiple of 16),
        head_dim 64 or 128; or one over existing `pages` (uint8 [num_pages,
        kv_heads, page_size / 16, 16 * head_dim + 128], contiguous, CUDA)."""
        self.engine = engine
        self._lib = _lib.load()
        if dtype not in _DTYPES:
            raise RuntimeError(f"KvCache4: dtype must be fp16 or bf16, got {dtype}")
        if pages is None:
            if not num_pages or not kv_heads or head_dim not in (64, 128) or page_size < 1 or page_size % self.TILE:
                raise RuntimeError("KvCache4: num_pages and kv_heads must be positive, head_dim 64 or 128, page_size "
                                   "a multiple of 16")
            pages = torch.zeros(num_pages, kv_heads, page_size // self.TILE, self._lib.wp_kv4_tile_bytes(head_dim),
                                dtype=torch.uint8, device=engine.device)
        if (pages.dtype != torch.uint8 or pages.dim() != 4 or pages.get_device() != engine.device.index
                or not pages.is_contiguous()):
            raise RuntimeError(f"KvCache4: pages must be a contiguous 4-d uint8 tensor on {engine.device}")
        if pages.size(3) not in (16 * 64 + 128, 16 * 128 + 128):
            raise RuntimeError("KvCache4: pages.size(3) must be 16 * head_dim + 128 with head_dim 64 or 128")
        self.pages = pages
        self.dtype = dtype
        self.num_pages, self.kv_heads = int(pages.size(0)), int(pages.size(1))
        self.page_size = int(pages.size(2)) * self.TILE
        self.head_dim = (int(pages.size(3)) - 128) // 16
        self._code = _DTYPES[dtype]
        self._work_bytes: Dict[Tuple[int, int], int] = {}  # (heads, max_q) -> attention's workspace

    def _place(self, table, lens, cu, tokens: int, what: str) -> Tuple:
        dev = self.engine.device
        table = _index(table, f"{what}: table", 2, dev)
        lens = _index(lens, f"{what}: lens", 1, dev)
        n = lens.numel()
        if table.size(0) != n:
            raise RuntimeError(f"{what}: table and lens must have one row per sequence")
        if cu is None:
            if tokens != n:
                raise RuntimeError(f"{what}: without cu every sequence has one token")
        else:
            cu = _index(cu, f"{what}: cu", 1, dev)
            if cu.numel() != n + 1:
                raise RuntimeError(f"{what}: cu must have one entry more than there are sequences")
        return table, lens, cu, n

    def _rows(self, t: torch.Tensor, heads: int, what: str) -> torch.Tensor:
        shape = t.shape
        if len(shape) != 3 or (heads and shape[1] != heads) or shape[2] != self.head_dim:
            raise RuntimeError(f"{what} must be [tokens, {heads or 'heads'}, {self.head_dim}]")
        if t.dtype != self.dtype:
            raise RuntimeError(f"{what} must be of the cache's dtype {self.dtype}, got {t.dtype}")
        return _packed_rows(t, what, self.engine.device)

    def append(self, k: torch.Tensor, v: torch.Tensor, table, lens, cu=None) -> None:
        """Stores k and v [tokens, kv_heads, head_dim] as the last tokens of
        their sequences. table [sequences, pages] page numbers, lens
        [sequences] lengths with these tokens included, cu [sequences + 1]
        offsets of each sequence's tokens (None: one each); int32."""
        k, v = self._rows(k, self.kv_heads, "append: k"), self._rows(v, self.kv_heads, "append: v")
        tokens = k.size(0)
        if v.size(0) != tokens:
            raise RuntimeError("append: k and v must have the same number of tokens")
        table, lens, cu, n = self._place(table, lens, cu, tokens, "append")
        ks, vs = k.stride(), v.stride()
        _lib.check(self._lib.wp_kv4_append(
            self.engine.handle, self.pages.data_ptr(), self.num_pages, self.page_size, k.data_ptr(), ks[0], ks[1],
            v.data_ptr(), vs[0], vs[1], table.data_ptr(), table.size(1), lens.data_ptr(),
            None if cu is None else cu.data_ptr(), n, tokens, self.kv_heads, self.head_dim, self._code,
            _stream_ptr(self.pages.device)), self.engine.handle)

    def read(self, table, lens, cu=None, tokens: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """The values that the last cu[b + 1] - cu[b] tokens of each sequence
        stand for, as packed k and v [tokens, kv_heads, head_dim]; tokens:
        their total, the length of the packed tensors (needed with cu). Rows
        past the last sequence's, where tokens is more, are not written."""
        if tokens is None:
            if cu is not None:
                raise RuntimeError("read: tokens (the total, cu[-1]) is needed with cu")
            tokens = int(lens.numel())
        tokens = int(tokens)
        table, lens, cu, n = self._place(table, lens, cu, tokens, "read")
        dev = self.pages.device
        k = torch.empty((tokens, self.kv_heads, self.head_dim), dtype=self.dtype, device=dev)
        v = torch.empty_like(k)
        _lib.check(self._lib.wp_kv4_read(
            self.engine.handle, k.data_ptr(), v.data_ptr(), self.pages.data_ptr(), self.num_pages, self.page_size,
            table.data_ptr(), table.size(1), lens.data_ptr(), None if cu is None else cu.data_ptr(), n, tokens,
            self.kv_heads, self.head_dim, self._code, _stream_ptr(dev)), self.engine.handle)
        return k, v

    def attention(self, q: torch.Tensor, table, lens, cu=None, max_q: int = 1, scale: Optional[float] = None,
                  return_lse: bool = False):
        """Causal attention of each sequence's last tokens over its cached
        ones: query i of n sees the positions < lens[b] - (n - 1 - i). q
        [tokens, heads, head_dim], heads a multiple of kv_heads; scale defaults
        to head_dim ** -0.5; max_q, the most query tokens of one sequence,
        chooses the kernel only. Returns out like q (contiguous), and the
        softmax's log denominators [tokens, heads] in fp32 with return_lse. A
        row that sees nothing is 0 (lse -inf); rows outside every sequence's
        offsets are not written."""
        q = self._rows(q, 0, "attention: q")
        tokens, heads, _ = q.shape
        if heads == 0 or heads % self.kv_heads:
            raise RuntimeError(f"attention: q has {heads} heads, not a multiple of the cache's {self.kv_heads}")
        table, lens, cu, n = self._place(table, lens, cu, tokens, "attention")
        h, dev, max_q = self.engine.handle, q.device, int(max_q)
        out = _empty_rows(q)
        lse = torch.empty(tokens, heads, dtype=torch.float32, device=dev) if return_lse else None
        size = self._work_bytes.get((heads, max_q))
        if size is None:
            size = self._work_bytes[heads, max_q] = max(
                self._lib.wp_kv4_attention_workspace(h, heads, self.kv_heads, self.head_dim, max_q, self._code), 0)
        # from the caching allocator, so that calls on several streams never share it
        work = torch.empty(size, dtype=torch.uint8, device=dev)
        qs = q.stride()
        _lib.check(self._lib.wp_kv4_attention(
            h, out.data_ptr(), None if lse is None else lse.data_ptr(), q.data_ptr(), qs[0], qs[1], self.pages.data_ptr(),
            self.num_pages, self.page_size, table.data_ptr(), table.size(1), lens.data_ptr(),
            None if cu is None else cu.data_ptr(), n, max_q, tokens, heads, self.kv_heads, self.head_dim,
            1.0 / math.sqrt(self.head_dim) if scale is None else float(scale), self._code, work.data_ptr(), size,
            _stream_ptr(dev)), h)
        return (out, lse) if return_lse else out
