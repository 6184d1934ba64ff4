"""The pages of a paged cache, dealt to sequences on the GPU (csrc/page_pool.hip; no reference counterpart: the reference
quantizes weights only).

`KVCache4` is a pool of pages, and which of them a sequence has stands in a block table.  A `PagePool` keeps that table: from
the tokens that each sequence is to hold it takes pages and gives them back, and says where the new tokens' rows, positions
and places in the cache are.  Nothing is read on the host, so its calls may be captured in a hipGraph like the cache's.

    pool = PagePool(pages=4096, seqs=64, width=512, page_size=64)
    rows = pool.extend(new, tokens=tokens)                    # room for new[b] more tokens of each sequence
    cache.append(k, v, pool.table, rows.held, rows.offsets)
    out = cache.attend(q, pool.table, pool.lengths, rows.offsets)
    pool.resize(lengths)                                      # fewer where drafts were rejected; 0: the sequence has ended

The pages that no sequence has are a stack.  The table's entries that are too many go back first, those of all sequences in
order, the last one first, each on the stack's top; then those that are missing are taken from the top, sequence by sequence.
A step that is taken back so leaves its pages to the next one in the same order.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

import _hip


class Rows(NamedTuple):
    """The packed rows of a call's new tokens: sequence b's are ``offsets[b]`` to ``offsets[b + 1] - 1`` [B + 1], at the
    positions from ``held[b]`` on [B]; each row's position [tokens] (all int32) and its place in the cache [tokens] (int64:
    page times page_size, plus its place in the page; -1 without a page).  Rows behind the last sequence's have position 0 and
    no place, those past the 2^30 tokens that a sequence may hold position 2^30 and none."""
    offsets: torch.Tensor
    held: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor


class PagePool:
    """``pages`` pages of ``page_size`` tokens for ``seqs`` sequences of at most ``width`` pages.

    The state, on the device, all int32: ``table`` [seqs, width] (-1: no page), ``lengths`` [seqs] (tokens held), ``owned``
    [seqs] (pages, the first entries of the row), ``missing`` [seqs] (pages that the last call had none left for), ``free``
    [pages] and ``left`` [1] (the stack, and its height).  It is written by the calls alone, in the order of the stream that they
    are made on.  Tokens past a sequence's last entry count in its length and have no place; a page that it gets
    later holds nothing of them, so a sequence with pages missing is taken back (`resize`) to what it has pages for, or those
    tokens are appended again."""

    def __init__(self, pages: int, seqs: int, width: int, *, page_size: int = 64, device: torch.device | str = "cuda"):
        if not (0 <= pages < 1 << 31 and 0 <= seqs <= 1 << 24 and 0 <= width and seqs * width < 1 << 31 and width < 1 << 31 and
                1 <= page_size <= 1 << 20):
            raise ValueError(f"no pool of {pages} pages of {page_size} tokens for {seqs} sequences of {width} pages")
        self.page_size, self.width = page_size, width
        whole = dict(dtype=torch.int32, device=device)
        self.table = torch.full((seqs, width), -1, **whole)
        _hip.require_device(self.table)
        self.device = self.table.device
        self.lengths, self.owned, self.missing = (torch.zeros(seqs, **whole) for _ in range(3))
        self.free = torch.arange(pages - 1, -1, -1, **whole)  # page 0 is on top
        self.left = torch.full((1,), pages, **whole)
        size = int(_hip.lib().gptq2d_page_pool_workspace(seqs))
        self._work = torch.empty(size, dtype=torch.uint8, device=device)
        self._bind()

    def _bind(self):
        """The state as the C entry takes it."""
        (seqs, width), pages = self.table.shape, self.free.numel()
        self._state = (self.table.data_ptr(), seqs, width, width, self.page_size, pages, self.owned.data_ptr(),
                       self.lengths.data_ptr(), self.missing.data_ptr(), self.free.data_ptr(), self.left.data_ptr())
        self._scratch = (self._work.data_ptr(), self._work.numel())

    def __setstate__(self, state):  # a copy has tensors of its own
        self.__dict__.update(state)
        self._bind()

    def _request(self, t, name):
        if t.dtype is not torch.int32 or t.shape != self.lengths.shape or t.device != self.device or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 [{self.lengths.numel()}] on the pool's device")
        return t.data_ptr()

    def resize(self, lengths: torch.Tensor) -> None:
        """Pages for ``lengths[b]`` tokens of sequence b (int32; below 0 counts as 0, at most 2^30), no more and no fewer."""
        _hip.launch("page_pool", self.device, *self._state, self._request(lengths, "lengths"), False, 0, None, None, None, None,
              *self._scratch)

    def extend(self, new: torch.Tensor, *, tokens: int) -> Rows:
        """Pages for ``new[b]`` more tokens of sequence b (int32; below 0 counts as 0), and their rows.  ``tokens``: rows in all,
        at least the sum of ``new`` (which is not read on the host); more where a batch is padded."""
        if not 0 <= tokens < 1 << 31:
            raise ValueError("tokens must be a number of rows below 2^31")
        device, seqs = self.device, self.lengths.size(0)
        rows = Rows(torch.empty(seqs + 1, dtype=torch.int32, device=device), torch.empty(seqs, dtype=torch.int32, device=device),
                    torch.empty(tokens, dtype=torch.int32, device=device), torch.empty(tokens, dtype=torch.int64, device=device))
        _hip.launch("page_pool", self.device, *self._state, self._request(new, "new"), True, tokens, *(t.data_ptr() for t in rows),
              *self._scratch)
        return rows


def row_positions(held: torch.Tensor, offsets: torch.Tensor, tokens: int) -> torch.Tensor:
    """Positions [tokens] (int32) of packed rows whose sequence b, rows ``offsets[b]`` to ``offsets[b + 1] - 1`` (int32 [B + 1]),
    follows ``held[b]`` tokens (int32 [B]); 0 for rows that no sequence has."""
    _hip.require_device(held)
    if held.dtype is not torch.int32 or held.dim() != 1 or not held.is_contiguous():
        raise ValueError("held must be a contiguous int32 [B]")
    if offsets.dtype is not torch.int32 or offsets.shape != (held.numel() + 1,) or offsets.device != held.device or \
            not offsets.is_contiguous():
        raise ValueError(f"offsets must be a contiguous int32 [{held.numel() + 1}] on held's device")
    if not 0 <= tokens < 1 << 31:
        raise ValueError("tokens must be a number of rows below 2^31")
    positions = torch.empty(tokens, dtype=torch.int32, device=held.device)
    _hip.launch("row_positions", held.device, held.data_ptr(), offsets.data_ptr(), held.numel(), tokens, positions.data_ptr())
    return positions
