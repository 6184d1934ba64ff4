"""Products with a packed INT layer, and the low-rank adapters of many requests beside it, on the GPU
(csrc/packed_linear.hip; no reference counterpart: the reference returns dequantized weights).

``packing.pack_int`` turns a quantized layer W [m, n] into words of codes; ``packed_linear`` multiplies activations by the
layer straight from them:

    y = x W^T + bias,   W[i, k] = (u[i, k] + qmin - zero_point[i, k / group]) * scale[i, k / group]

and, for requests that each bring an adapter (A, B) of their own to the shared layer, adds to every token the product with
its own: scaling (x A^T) B^T.  Codes enter the products exactly; an activation to 22 bits (all that bf16 and fp16 have), or
to 2^-39 of its token's largest finite element where that is coarser: what lies below is dropped, which a sum in 32 bits
shows only where that element's weight is 0.  Sums are in 32 bits; results are rounded once, to the activations' type.
"""

from __future__ import annotations

import functools
from typing import NamedTuple

import torch

import _hip
import packing

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
BITS = (2, 3, 4, 8)  # code widths that the kernels multiply


class Adapters(NamedTuple):
    """Low-rank adapters of one layer: `a` [count, rank, n], `b` [count, m, rank] and `scaling` [count] (float32, or None for
    1).  Adapters of a lower rank are padded with zeros."""
    a: torch.Tensor
    b: torch.Tensor
    scaling: torch.Tensor | None = None


@functools.lru_cache(maxsize=None)
def _bits(qmin, qmax) -> int:
    bits = packing.int_code_bits(qmin, qmax)
    if bits not in BITS:
        raise ValueError(f"packed_linear multiplies codes of {BITS} bits: [{qmin}, {qmax}] takes {bits}")
    return bits


def _groups(t, name, m, groups, device):
    """(pointer, row stride, group stride) of a scale or zero point: one number, one a row, or one a row and group."""
    if t.dtype is not torch.float32 or t.device != device:
        raise ValueError(f"{name} must be float32 on the activations' device")
    if t.dim() == 0:
        return t.data_ptr(), 0, 0
    shape = t.shape if t.dim() > 1 else (*t.shape, 1)
    if len(shape) != 2 or shape[0] not in (1, m) or shape[1] not in (1, groups):
        raise ValueError(f"{name} must broadcast to [{m}, {groups}] (rows, groups), got {tuple(t.shape)}")
    return (t.data_ptr(), t.stride(0) if shape[0] > 1 else 0, t.stride(1) if t.dim() > 1 and shape[1] > 1 else 0)


@torch.no_grad()
def packed_linear(x: torch.Tensor, words: torch.Tensor, scale: torch.Tensor, zero_point: torch.Tensor | None = None, *,
                  qmin: float, qmax: float, group: int | None = None, bias: torch.Tensor | None = None,
                  adapters: Adapters | tuple | None = None, index: torch.Tensor | None = None) -> torch.Tensor:
    """x [*, n] (float32, bfloat16 or float16) times the packed layer: y [*, m] in x's type.

    ``words`` [m, row_words] are the codes of ``packing.pack_int`` with the bounds ``qmin``, ``qmax`` (2, 3, 4 or 8 bits a
    code).  ``scale`` and ``zero_point`` (None: 0) are float32: one number, one a row ([m] or [m, 1]), or with ``group`` (a
    multiple of 32 columns) one a row and group ([m, ceil(n / group)]).  ``bias`` [m] in x's type.

    ``adapters``: an `Adapters` (or (a, b, scaling)) in x's type, and ``index`` (int32, a number a token: x's shape without
    its last axis) says which one a token has; a token whose index is not in 0 .. count - 1 has none."""
    kind = _TYPES.get(x.dtype)
    if kind is None or x.dim() == 0:
        raise ValueError("x must be a float32, bfloat16 or float16 [*, n] tensor")
    device = x.device
    if not x.is_cuda:
        raise _hip.GPTQ2DError("packed_linear needs GPU tensors")
    n = x.size(-1)
    bits = _bits(qmin, qmax)
    if words.dtype is not torch.int32 or words.dim() != 2 or words.device != device or \
            (words.stride(1) != 1 and words.size(1) > 1):
        raise ValueError("words must be int32 [m, row_words] on x's device, with contiguous rows")
    m, row_words = words.shape
    if n == 0 or m == 0 or row_words * 32 < n * bits:
        raise ValueError(f"{row_words} words a row do not hold {n} codes of {bits} bits")
    if group is not None and (group < 32 or group % 32):
        raise ValueError("a group has a multiple of 32 columns")
    groups = -(-n // group) if group else 1
    s, s_row, s_col = _groups(scale, "scale", m, groups, device)
    z, z_row, z_col = (None, 0, 0) if zero_point is None else _groups(zero_point, "zero_point", m, groups, device)
    rows = x if x.dim() == 2 else x.reshape(-1, n)
    if rows.stride(1) != 1 and n > 1:
        rows = rows.contiguous()
    tokens = rows.size(0)
    if bias is not None and (bias.shape != (m,) or bias.dtype is not x.dtype or bias.device != device or
                             not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous [{m}] in x's type on its device")
    a_ptr = b_ptr = scaling_ptr = index_ptr = None
    count = rank = 0
    if (adapters is None) != (index is None):
        raise ValueError("adapters need an index and an index adapters")
    if adapters is not None:
        a, b, scaling = adapters if len(adapters) == 3 else (*adapters, None)
        if a.dim() != 3 or b.dim() != 3 or a.size(2) != n or b.size(1) != m or a.size(0) != b.size(0) or \
                a.size(1) != b.size(2):
            raise ValueError(f"adapters must be a [count, rank, {n}] and b [count, {m}, rank], got {tuple(a.shape)}, "
                             f"{tuple(b.shape)}")
        if not (a.dtype is b.dtype is x.dtype) or a.device != device or b.device != device or \
                not a.is_contiguous() or not b.is_contiguous():
            raise ValueError("adapters must be contiguous, in x's type and on its device")
        count, rank = a.size(0), a.size(1)
        if rank > 4096:
            raise ValueError("adapters have a rank of at most 4096")
        if scaling is not None:
            if scaling.shape != (count,) or scaling.dtype is not torch.float32 or scaling.device != device or \
                    not scaling.is_contiguous():
                raise ValueError(f"scaling must be a contiguous float32 [{count}] on x's device")
            scaling_ptr = scaling.data_ptr()
        if index.dtype is not torch.int32 or index.shape != x.shape[:-1] or index.device != device or \
                not index.is_contiguous():
            raise ValueError(f"index must be a contiguous int32 {tuple(x.shape[:-1])} on x's device")
        if count and rank:
            a_ptr, b_ptr, index_ptr = a.data_ptr(), b.data_ptr(), index.data_ptr()
        else:
            count = rank = 0
    y = torch.empty(*x.shape[:-1], m, dtype=x.dtype, device=device)
    lib = _hip.lib()
    size = lib.gptq2d_packed_linear_workspace(tokens, m, n, bits, group or 0, kind, count, rank)
    if size < 0:
        raise ValueError(f"packed_linear of {tokens} tokens, a [{m}, {n}] layer and {count} adapters of rank {rank} is "
                         "too large")
    work = torch.empty(size, dtype=torch.uint8, device=device)
    args = (rows.data_ptr(), rows.stride(0), kind, tokens, words.data_ptr(), m, n,
            words.stride(0) if m > 1 else row_words, bits, s, s_row, s_col, z, z_row, z_col, qmin, group or 0,
            None if bias is None else bias.data_ptr(), a_ptr, b_ptr, scaling_ptr, index_ptr, count, rank, y.data_ptr(), m,
            work.data_ptr(), size)
    if torch.cuda.current_device() == device.index:
        rc = lib.gptq2d_packed_linear(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = lib.gptq2d_packed_linear(*args, torch.cuda.current_stream(device).cuda_stream)
    if rc:
        raise _hip.GPTQ2DError(f"gptq2d_packed_linear failed with code {rc}")
    return y
