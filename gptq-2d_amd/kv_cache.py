"""A paged cache of keys and values in 4 bits, and attention over it, on the GPU (csrc/kv_append.hip,
csrc/kv_attend.hip; no reference counterpart: the reference quantizes weights only).

A token's key or value vector x of one head is held as 4-bit codes with a scale and a zero of 16 bits each, the affine
quantizer's form (quantizer_int.py:63-83) with the extremes of the vector itself:

    s = bf16((max x - min x) / 15), 1 where that is 0;   z = bf16(min x);   c = clamp(round((x - z) / s), 0, 15)

in fp32, standing for c s + z: 4.5 bits an element at a head size of 64, 4.25 at 128.

The cache is a pool of pages; which pages a sequence has is in a block table the caller keeps, as the number of tokens
that it holds.  Everything a call needs to know of the sequences is read on the GPU: no call synchronises with the host,
and all of them may be captured in a hipGraph (table, lengths and offsets may change between replays).

    cache = KVCache4(pages=4096, kv_heads=8, head_dim=128, page_size=64)
    cache.append(k, v, table, held, offsets)              # new tokens to positions held[b], held[b] + 1, ...
    out = cache.attend(q, table, held + new, offsets)     # causal attention of the new tokens over all that is held
"""

from __future__ import annotations

import math

import torch

import _hip

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class KVCache4:
    """Pages of `page_size` tokens (a multiple of 32, at most 4096) of `kv_heads` heads of `head_dim` (1 to 256)
    elements.

    The methods take ``table`` [B, W] (int32: the pages of each sequence, in order; an entry outside the pool holds no
    token), ``lengths`` [B] (int32) and ``offsets`` [B + 1] (int32: sequence b's rows among the packed tokens of the call are
    ``offsets[b]`` to ``offsets[b + 1] - 1``; None: one token a sequence), all on the cache's device.  Rows before
    ``offsets[0]`` and from ``offsets[B]`` on, as a padded batch has them, are no sequence's: they are not appended, and
    are zeros where they are read or attended.  A page that tokens are appended to belongs to one sequence; full pages may
    be shared between sequences."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, *, page_size: int = 64,
                 device: torch.device | str = "cuda"):
        words = int(_hip.lib().gptq2d_kv_page_words(kv_heads, head_dim, page_size))
        if words < 0 or pages < 0:
            raise ValueError(f"no 4-bit cache of {pages} pages of {page_size} tokens, {kv_heads} heads of {head_dim}: "
                             "a page holds a multiple of 32 tokens, at most 4096, a head 1 to 256 elements")
        self.kv_heads, self.head_dim, self.page_size = kv_heads, head_dim, page_size
        self.pages = torch.empty(pages, words, dtype=torch.int32, device=device)
        _hip.require_device(self.pages)
        self.device = self.pages.device
        lib = _hip.lib()
        self._append, self._read, self._attend = lib.gptq2d_kv_append, lib.gptq2d_kv_read, lib.gptq2d_kv_attend
        self._workspace = lib.gptq2d_kv_attend_workspace
        self._cache = (self.pages.data_ptr(), pages, kv_heads, head_dim, page_size)

    # Arguments of the sequences, as the C entries take them.
    def _sequences(self, table, lengths, offsets, tokens):
        seqs, width = table.shape
        if not (table.dtype is lengths.dtype is torch.int32):
            raise ValueError("table and lengths must be int32")
        if lengths.shape != (seqs,) or not lengths.is_contiguous() or (width > 1 and table.stride(1) != 1):
            raise ValueError("lengths must be a contiguous [B], table a [B, W] with contiguous rows")
        if table.device != self.device or lengths.device != self.device:
            raise ValueError("table and lengths must be on the cache's device")
        if width * self.page_size >= 1 << 29:
            raise ValueError("a sequence's pages must hold fewer than 2^29 tokens")
        at = None
        if offsets is not None:
            if offsets.dtype is not torch.int32 or offsets.shape != (seqs + 1,) or not offsets.is_contiguous() or \
                    offsets.device != self.device:
                raise ValueError("offsets must be a contiguous int32 [B + 1] on the cache's device")
            at = offsets.data_ptr()
        elif tokens != seqs:
            raise ValueError(f"{tokens} tokens for {seqs} sequences need offsets")
        return table.data_ptr(), seqs, width, table.stride(0), lengths.data_ptr(), at, tokens

    def _rows(self, x, name, heads):
        if x.dim() != 3 or x.size(1) != heads or x.size(2) != self.head_dim:
            raise ValueError(f"{name} must be [tokens, {heads}, {self.head_dim}], got {tuple(x.shape)}")
        if x.device != self.device:
            raise ValueError(f"{name} must be on the cache's device")
        return x if x.stride(2) == 1 or self.head_dim == 1 else x.contiguous()

    def _call(self, fn, name, *args):
        device = self.device
        if torch.cuda.current_device() == device.index:
            rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
        else:
            with torch.cuda.device(device):
                rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
        if rc:
            raise _hip.GPTQ2DError(f"gptq2d_kv_{name} failed with code {rc}")

    @torch.no_grad()
    def append(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
               offsets: torch.Tensor | None = None) -> None:
        """Put keys and values [tokens, kv_heads, head_dim] (fp32, bf16 or fp16) into the cache: sequence b's at positions
        ``lengths[b]``, ``lengths[b] + 1``, ... (``lengths``: the tokens held before).  Tokens past the table's last
        page are dropped."""
        k, v = self._rows(k, "k", self.kv_heads), self._rows(v, "v", self.kv_heads)
        kind = _TYPES.get(k.dtype)
        if kind is None or v.dtype is not k.dtype or k.shape != v.shape:
            raise ValueError("k and v must share their shape and be float32, bfloat16 or float16")
        self._call(self._append, "append", *self._cache, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                   v.stride(0), v.stride(1), kind, *self._sequences(table, lengths, offsets, k.size(0)))

    @torch.no_grad()
    def read(self, table: torch.Tensor, lengths: torch.Tensor, offsets: torch.Tensor | None = None, *,
             tokens: int | None = None, dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
        """The values [tokens, kv_heads, head_dim] that the last tokens of each sequence are held as, keys and values:
        sequence b's rows are its positions up to ``lengths[b] - 1``.  ``tokens``: rows in all (``offsets[B]``, which is
        not read on the host; without offsets one a sequence).  Rows without a token in the cache are zeros, as are rows that no
        sequence has."""
        if tokens is None:
            if offsets is not None:
                raise ValueError("read needs the number of tokens where offsets are given")
            tokens = table.size(0)
        kind = _TYPES.get(dtype)
        if kind is None:
            raise ValueError("read gives float32, bfloat16 or float16")
        k = torch.empty(tokens, self.kv_heads, self.head_dim, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        self._call(self._read, "read", *self._cache, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                   v.stride(1), kind, *self._sequences(table, lengths, offsets, tokens))
        return k, v

    @torch.no_grad()
    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, offsets: torch.Tensor | None = None, *,
               scale: float | None = None, window: int | None = None, return_lse: bool = False):
        """Causal attention of q [tokens, heads, head_dim] (fp32, bf16 or fp16; heads a multiple of kv_heads, consecutive
        ones sharing a kv head) over the cache. The queries of a sequence are its last tokens: of its T, number i is at
        position ``lengths[b] - T + i`` and sees the positions up to its own, with ``window`` only the last `window` of
        them. ``scale`` defaults to head_dim^-1/2. A query that sees nothing, or is no sequence's, gives zeros. Each
        head's query counts to 22 bits an element (all that bf16 and fp16 have), or to 2^-31 of its largest where that is
        coarser. ``return_lse``: the logarithm of the softmax's denominator [tokens, heads] too (-inf where a query sees
        nothing)."""
        if q.dim() != 3 or q.size(1) % self.kv_heads or q.size(1) == 0:
            raise ValueError(f"q must be [tokens, heads, {self.head_dim}], heads a multiple of {self.kv_heads}")
        tokens, heads, dim = q.shape
        q = self._rows(q, "q", heads)
        kind = _TYPES.get(q.dtype)
        if kind is None:
            raise ValueError("q must be float32, bfloat16 or float16")
        if window is not None and not 1 <= window < 1 << 30:
            raise ValueError("a window holds at least one token, and fewer than 2^30")
        where = self._sequences(table, lengths, offsets, tokens)
        group, window = heads // self.kv_heads, window or 0
        out = torch.empty(tokens, heads, dim, dtype=q.dtype, device=self.device)
        lse = torch.empty(tokens, heads, dtype=torch.float32, device=self.device) if return_lse else None
        size = self._workspace(tokens, where[1], self.kv_heads, group, dim, where[2] * self.page_size, window)
        if size < 0:
            raise ValueError(f"attention of {tokens} tokens over {where[1]} sequences is too large")
        work = torch.empty(size, dtype=torch.uint8, device=self.device) if size else None
        self._call(self._attend, "attend", *self._cache, q.data_ptr(), q.stride(0), q.stride(1), group, kind, *where,
                   math.pow(dim, -0.5) if scale is None else scale, window, out.data_ptr(), out.stride(0), out.stride(1),
                   None if lse is None else lse.data_ptr(), None if work is None else work.data_ptr(), size)
        return (out, lse) if return_lse else out
