"""The key/value cache held in 4 or in 8 bits: pools of pages (`KVCache`, `KVCache8`), the description of whose tokens the rows of a
call are (`KVRows`), and the tables of which page belongs to which sequence (`KVPages`).  Pools are written, read and attended over by
`ops.cache_write`, `ops.cache_read` and `ops.cache_attention`; tables follow the lengths that requests ask for with `ops.cache_pages`,
and `ops.cache_slots` tells where the rows of a step go."""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib


class KVRows(NamedTuple):
    """Whose tokens the rows of a call are.  Dense tensors are [rows, heads, head_dim], the newest tokens of the sequences
    packed one behind the other: sequence b owns rows starts[b] to starts[b + 1] (`starts` None: equally many each), and the
    last of them is its token lens[b] - 1.  Token j of sequence b is on page table[b, j // page].  A call may have fewer rows than the
    offsets name: those it has are the same tokens as in a call with all of them.

    All three are int32 tensors on the cache's device and are read when the kernels run: nothing here is copied to the host,
    and a call recorded in a graph follows them; they must not change while it runs.  A table entry outside the pool (-1) is a page
    that is not there."""
    table: torch.Tensor
    lens: torch.Tensor
    starts: Optional[torch.Tensor] = None


class _Pool:
    @property
    def device(self):
        return self.k_codes.device

    def rows(self, table, lens, starts=None) -> KVRows:
        """KVRows of lists or tensors of any integer type, on this cache's device."""
        def as_ints(t, name):
            if t is None:
                return None
            t = torch.as_tensor(t)
            if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
                if t.numel():                                       # (an empty list makes a float tensor)
                    raise TypeError(f"{name} must be integers, not {t.dtype}")
            elif t.dtype not in (torch.int32, torch.int16, torch.int8, torch.uint8):
                t = t.to(torch.int64).clamp(-(1 << 31), (1 << 31) - 1)      # a larger one stays large: no page, no row
            return t.to(self.device, torch.int32).contiguous()
        return KVRows(as_ints(table, "table"), as_ints(lens, "lens"), as_ints(starts, "starts"))


class KVCache(_Pool):
    """A pool of `pages` pages of `page` tokens for `heads` key/value heads of `head_dim` channels, in groups of `group`
    channels with an fp16 scale and minimum each: 4 + 32 / group bits a value.

    page: 16, 32, 64, 128 or 256 tokens; head_dim: 64, 128 or 256; group: 32, 64 or 128, at most head_dim.  Which
    page belongs to which sequence is the caller's business (`KVRows.table`, or a `KVPages` that keeps it)."""

    def __init__(self, pages: int, heads: int, head_dim: int, page: int = 64, group: int = 32, device="cuda"):
        self.pages, self.page, self.heads, self.head_dim, self.group = int(pages), int(page), int(heads), int(head_dim), int(group)
        d = _lib.CbkCache(pages=self.pages, page=self.page, heads=self.heads, head_dim=self.head_dim, group=self.group)
        codes = _lib.lib().cbk_cache_code_bytes(ctypes.byref(d))
        meta = _lib.lib().cbk_cache_meta_bytes(ctypes.byref(d))
        if not codes:
            raise ValueError(f"no cache of {pages} pages of {page} tokens, {heads} heads of {head_dim} channels in groups of {group}: "
                             "pages >= 1; page 16, 32, 64, 128 or 256; head_dim 64, 128 or 256; group 32, 64 or 128, at most head_dim")
        self.k_codes, self.v_codes = (torch.zeros(codes, dtype=torch.uint8, device=device) for _ in range(2))
        self.k_meta, self.v_meta = (torch.zeros(meta, dtype=torch.uint8, device=device) for _ in range(2))

    def native(self):
        return (self.k_codes, self.v_codes, self.k_meta, self.v_meta, self.pages, self.page, self.heads, self.head_dim, self.group)

    def nbytes(self) -> int:
        return 2 * (self.k_codes.numel() + self.k_meta.numel())


class KVCache8(_Pool):
    """The same pool in 8 bits: e4m3 codes, and for each `block` consecutive tokens of a head a power of two that scales its keys and one
    that scales its values: 8 + 32 / (block * head_dim) bits a value.  A block's scale grows with the largest magnitude written to it; the codes
    of its older tokens follow (a move of the exponent).  With its first token a block begins anew: what it held behind the rows of that call is lost.

    page: 16, 32, 64, 128 or 256 tokens; head_dim: 64, 128 or 256; block: 16, 32, 64, 128 or 256 tokens, at most page."""

    def __init__(self, pages: int, heads: int, head_dim: int, page: int = 64, block: int = 16, device="cuda"):
        self.pages, self.page, self.heads, self.head_dim, self.block = int(pages), int(page), int(heads), int(head_dim), int(block)
        d = _lib.CbkCache8(pages=self.pages, page=self.page, heads=self.heads, head_dim=self.head_dim, block=self.block)
        codes = _lib.lib().cbk_cache_eight_code_bytes(ctypes.byref(d))
        if not codes:
            raise ValueError(f"no cache of {pages} pages of {page} tokens, {heads} heads of {head_dim} channels in blocks of {block} tokens: "
                             "pages >= 1; page 16, 32, 64, 128 or 256; head_dim 64, 128 or 256; block 16, 32, 64, 128 or 256, at most page")
        self.k_codes, self.v_codes = (torch.zeros(codes, dtype=torch.uint8, device=device) for _ in range(2))
        self.scales = torch.zeros(_lib.lib().cbk_cache_eight_scale_bytes(ctypes.byref(d)), dtype=torch.uint8, device=device)

    def native(self):
        return (self.k_codes, self.v_codes, self.scales, self.pages, self.page, self.heads, self.head_dim, self.block)

    def nbytes(self) -> int:
        return 2 * self.k_codes.numel() + self.scales.numel()


class KVPages:
    """Which of a pool's `pages` pages belong to which of `seqs` sequences of up to `max_len` tokens, on the device: `table` [seqs,
    ceil(max_len / page)] (-1: no page), `lens` [seqs], and the pages that belong to nobody as a stack, free[:count].  All int32; they
    are written by `ops.cache_pages` only.  One set of tables serves every layer's pool of the same number of pages and tokens a page."""

    def __init__(self, pages: int, seqs: int, max_len: int, page: int = 64, device="cuda"):
        self.pages, self.page, self.seqs, self.max_len = int(pages), int(page), int(seqs), int(max_len)
        if self.page not in (16, 32, 64, 128, 256) or not 1 <= self.pages < 1 << 31 or not 1 <= self.seqs < 1 << 24 or not 1 <= self.max_len <= 1 << 30:
            raise ValueError(f"no tables for {seqs} sequences of {max_len} tokens on {pages} pages of {page}: pages, seqs and max_len are at "
                             "least 1, page is 16, 32, 64, 128 or 256")
        self.table = torch.full((self.seqs, -(-self.max_len // self.page)), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(self.seqs, dtype=torch.int32, device=device)
        self.free = torch.arange(self.pages - 1, -1, -1, dtype=torch.int32, device=device)      # handed out from the end: 0, 1, 2 ...
        self.count = torch.full((1,), self.pages, dtype=torch.int32, device=device)

    @property
    def device(self):
        return self.table.device

    def native(self):
        return (self.table, self.lens, self.free, self.count, self.pages, self.page)
