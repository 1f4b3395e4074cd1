"""The key/value cache held in 4 bits: a pool of pages (`KVCache`) and the description of whose tokens the rows of a
call are (`KVRows`).  Written, read and attended over by `ops.cache_write`, `ops.cache_read` and `ops.cache_attention`."""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib


class KVRows(NamedTuple):
    """Whose tokens the rows of a call are.  Dense tensors are [rows, heads, head_dim], the newest tokens of the sequences
    packed one behind the other: sequence b owns rows starts[b] to starts[b + 1] (`starts` None: equally many each), and the
    last of them is its token lens[b] - 1.  Token j of sequence b is on page table[b, j // page].

    All three are int32 tensors on the cache's device and are read when the kernels run: nothing here is copied to the host,
    and a call recorded in a graph follows them; they must not change while it runs.  A table entry outside the pool (-1) is a page
    that is not there."""
    table: torch.Tensor
    lens: torch.Tensor
    starts: Optional[torch.Tensor] = None


class KVCache:
    """A pool of `pages` pages of `page` tokens for `heads` key/value heads of `head_dim` channels, in groups of `group`
    channels with an fp16 scale and minimum each: 4 + 32 / group bits a value.

    page: 16, 32, 64, 128 or 256 tokens; head_dim: 64, 128 or 256; group: 32, 64 or 128, at most head_dim.  Which
    page belongs to which sequence is the caller's business (`KVRows.table`)."""

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

    @property
    def device(self):
        return self.k_codes.device

    def native(self):
        return (self.k_codes, self.v_codes, self.k_meta, self.v_meta, self.pages, self.page, self.heads, self.head_dim, self.group)

    def nbytes(self) -> int:
        return 2 * (self.k_codes.numel() + self.k_meta.numel())

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
