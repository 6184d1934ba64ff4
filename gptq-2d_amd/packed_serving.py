"""Serving from what the framework quantizes: an attention block whose projections are packed INT layers, with the requests'
own adapters beside them, over a cache of keys and values in 4 bits (no reference counterpart: the reference returns
dequantized weights).

    results = {r.name: r for r in model_driver.quantize_model(model, collector)}
    layers = [PackedLayer.from_result(results[name], bias=...) for name in ("q", "k", "v", "o")]
    cache = KVCache4(pages, kv_heads, head_dim)
    block = PackedAttention(*layers, cache, heads=heads, rotary=Rotary(head_dim))
    y = block(x, table, held, offsets)              # prompts: the sequences' new tokens, packed one after the other
    y = block(x, table, held)                       # a decode step: one token a sequence
    y = block(x, table, held, offsets, tree=tree)   # a step of drafted tokens

No call synchronises with the host, so a decode step may be captured in a hipGraph and replayed while `held` and `table`
change (a `page_pool.PagePool` changes them on the GPU too).  ``python packed_serving.py`` quantizes a small block, serves ragged
prompts and steps of drafted tokens from it and prints how far the outputs are from those of the dequantized weights.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Mapping

import torch

from drafts import DraftTree
from kv_cache import KVCache4
from packed_linear import Adapters, packed_linear
from page_pool import PagePool, row_positions
from rotary import Rotary


def _by_group(t, m, n, group, what) -> torch.Tensor:
    """t, broadcastable to the weight [m, n], as one number a row and group: float32 [m, groups], or [m, 1]."""
    t = torch.as_tensor(t, dtype=torch.float32)
    if t.dim() == 0 or t.size(-1) == 1:
        return t.expand(m, 1).contiguous()
    full = t.expand(m, n)
    size = group or n
    each = full[:, ::size]
    if not torch.equal(full, each.repeat_interleave(size, 1)[:, :n]):
        raise ValueError(f"{what} is not one number a row" + (f" and {group} columns" if group else "; say the group"))
    return each.contiguous()


@dataclass
class PackedLayer:
    """A linear layer as `packing.pack_int` packed it: the arguments of `packed_linear`."""
    words: torch.Tensor
    scale: torch.Tensor
    zero_point: torch.Tensor | None = None
    qmin: float = -8
    qmax: float = 7
    group: int | None = None
    bias: torch.Tensor | None = None
    columns: int | None = None  # of the weight; None: whatever is multiplied by it

    @classmethod
    def from_result(cls, result, *, qmin: float | None = None, qmax: float | None = None, group: int | None = None,
                    bias: torch.Tensor | None = None) -> PackedLayer:
        """Of a `model_driver.LayerResult` with packed codes, whose range it has.  ``group``: columns that share a scale and zero
        point, where the quantizer's are not one a row (its scale then is a map of every entry, [m, n]).  ``qmin`` and
        ``qmax`` only for a result that was made without a range; where it has one they must be that."""
        if result.words is None:
            raise ValueError(f"layer {result.name} has no packed codes")
        own = (getattr(result, "qmin", None), getattr(result, "qmax", None))
        bounds = tuple(o if v is None else v for v, o in zip((qmin, qmax), own))
        if None in bounds or any(o is not None and o != v for v, o in zip(bounds, own)):
            raise ValueError(f"layer {result.name} was packed with the code range {own}, asked for {(qmin, qmax)}")
        m, n = result.shape
        scale, zero = (None if t is None else _by_group(t, m, n, group, f"layer {result.name}: {what}").to(result.words.device)
                       for t, what in ((result.scale, "scale"), (result.zero_point, "zero point")))
        return cls(result.words, scale, zero, *bounds, group, bias, n)

    def __call__(self, x: torch.Tensor, adapters: Adapters | None = None, index: torch.Tensor | None = None) -> torch.Tensor:
        if self.columns is not None and x.size(-1) != self.columns:
            raise ValueError(f"the layer has {self.columns} columns, x {x.size(-1)}")
        return packed_linear(x, self.words, self.scale, self.zero_point, qmin=self.qmin, qmax=self.qmax, group=self.group,
                             bias=self.bias, adapters=adapters, index=None if adapters is None else index)


class PackedAttention:
    """Query, key, value and output projections over one `KVCache4`; `heads` query heads, a multiple of the cache's.  ``rotary``:
    queries and keys are rotated by their positions; the cache holds rotated keys."""

    def __init__(self, q: PackedLayer, k: PackedLayer, v: PackedLayer, out: PackedLayer, cache: KVCache4, *, heads: int,
                 window: int | None = None, rotary: Rotary | None = None):
        dim, kv = cache.head_dim, cache.kv_heads
        if heads % kv:
            raise ValueError(f"{heads} query heads are no multiple of the cache's {kv}")
        for name, layer, rows in (("q", q, heads * dim), ("k", k, kv * dim), ("v", v, kv * dim)):
            if layer.words.size(0) != rows:
                raise ValueError(f"{name} has {layer.words.size(0)} rows, its heads take {rows}")
        if out.columns not in (None, heads * dim):
            raise ValueError(f"out has {out.columns} columns, the heads give {heads * dim}")
        if window is not None and not 1 <= window < 1 << 30:
            raise ValueError("a window holds at least one token, and fewer than 2^30")
        if rotary is not None and (rotary.dim != dim or rotary.device != cache.device):
            raise ValueError(f"the rotation is of {rotary.dim} elements on {rotary.device}, the cache's heads are {dim} on {cache.device}")
        self.q, self.k, self.v, self.out, self.cache, self.heads, self.window = q, k, v, out, cache, heads, window
        self.rotary = rotary

    def __call__(self, x: torch.Tensor, table: torch.Tensor, held: torch.Tensor, offsets: torch.Tensor | None = None, *,
                 adapters: Mapping[str, Adapters] | None = None, index: torch.Tensor | None = None,
                 positions: torch.Tensor | None = None, tree: DraftTree | None = None) -> torch.Tensor:
        """x [tokens, n]: the sequences' new tokens (``offsets`` [B + 1] says which are whose; None: one each), that follow
        the ``held`` [B] tokens of the cache and are appended to it; the pages are there already (``table``).  ``adapters``:
        by layer ("q", "k", "v", "out"), and ``index`` [tokens] says which one a token has.  ``tree``: the new tokens are the
        nodes of this tree, made with the same ``held`` and ``offsets``.  ``positions`` [tokens] of the rotation (int32 or int64):
        the tree's, or those that follow what is held, where they are not given."""
        of, dim = adapters or {}, self.cache.head_dim
        if tree is not None:  # what attention would refuse, before the cache has the tokens
            self.cache._fits(tree, offsets, table.size(0), x.size(0), self.window)
        q = self.q(x, of.get("q"), index).unflatten(-1, (self.heads, dim))
        k = self.k(x, of.get("k"), index).unflatten(-1, (self.cache.kv_heads, dim))
        v = self.v(x, of.get("v"), index).unflatten(-1, (self.cache.kv_heads, dim))
        if self.rotary is not None:
            if positions is None:
                positions = tree.positions if tree is not None else held if offsets is None else \
                    row_positions(held, offsets, x.size(0))
            q, k = self.rotary(q, k, positions=positions)
        elif positions is not None:
            raise ValueError("positions are of a rotation, which the block has not")
        self.cache.append(k, v, table, held, offsets)
        lengths = held + 1 if offsets is None else held + (offsets[1:] - offsets[:-1])
        o = self.cache.attend(q, table, lengths, offsets, window=self.window, tree=tree)
        return self.out(o.flatten(-2), of.get("out"), index)


def main() -> None:
    import model_driver

    torch.manual_seed(0)
    dev, n, heads, kv, dim, page = "cuda", 512, 8, 2, 64, 64
    model = torch.nn.ModuleDict({name: torch.nn.Linear(n if name != "o" else heads * dim, rows, bias=False) for name, rows in
                                 (("q", heads * dim), ("k", kv * dim), ("v", kv * dim), ("o", n))}).to(dev)
    sample = torch.randn(2048, n, device=dev)
    with model_driver.HessianCollector(model, output_side=False) as collector, torch.no_grad():
        for layer in model.values():
            layer(sample)
    packed = {r.name: PackedLayer.from_result(r) for r in model_driver.quantize_model(model, collector)}
    prompts, steps, drafts = torch.tensor([5, 64, 200, 1]), 5, 4
    seqs, ends = len(prompts), (prompts + 2 * steps).tolist()
    cache, rotary = KVCache4(24, kv, dim, page_size=page), Rotary(dim)
    pool = PagePool(24, seqs, 8, page_size=page)
    block = PackedAttention(packed["q"], packed["k"], packed["v"], packed["o"], cache, heads=heads, rotary=rotary)
    # each sequence's tokens, and after them the one that is always wrong
    x = [torch.randn(end + 2, n, device=dev) for end in ends]
    rows = pool.extend(prompts.to(dev, torch.int32), tokens=int(prompts.sum()))
    got = [list(y) for y in block(torch.cat([v[:p] for v, p in zip(x, prompts)]).bfloat16(), pool.table, rows.held, rows.offsets,
                                  positions=rows.positions).split(prompts.tolist())]
    # Steps of four nodes: the next token, a wrong guess and the right one of what follows it, and a wrong one of what follows that.
    # A token's name is its place in the sequence, and the model chooses the next place after every right token.
    parents = torch.tensor([-1, 0, 0, 2], dtype=torch.int32, device=dev).repeat(seqs)
    right = torch.tensor([True, False, True, False], device=dev).repeat(seqs)
    last = torch.tensor(ends, device=dev).repeat_interleave(drafts) + 1
    for step in range(steps):
        rows = pool.extend(torch.full((seqs,), drafts, dtype=torch.int32, device=dev), tokens=seqs * drafts)
        tree = DraftTree(parents, rows.offsets, rows.held, nodes=drafts)
        place = torch.where(right, tree.positions, last)
        inputs = torch.stack([x[i // drafts][p] for i, p in enumerate(place.tolist())])
        y = block(inputs.bfloat16(), pool.table, rows.held, rows.offsets, tree=tree)
        accepted = tree.accept(place, torch.where(right, place + 1, -1))
        cache.keep(pool.table, pool.lengths, rows.offsets, accepted.path, accepted.counts)
        pool.resize(rows.held + accepted.counts)
        for b, (way, count) in enumerate(zip(accepted.path.tolist(), accepted.counts.tolist())):
            got[b] += [y[b * drafts + node] for node in way[:count]]
    assert pool.lengths.tolist() == ends
    worst = 0.
    with torch.no_grad():
        for b, end in enumerate(ends):
            q, k, v = (model[name](x[b][:end]).unflatten(-1, (-1, dim)) for name in "qkv")
            q, k = rotary(q, k, positions=torch.arange(end, device=dev))
            q, k, v = q.transpose(0, 1), *(t.transpose(0, 1).repeat_interleave(heads // kv, 0) for t in (k, v))
            seen = torch.ones(end, end, dtype=torch.bool, device=dev).tril()
            p = torch.softmax((torch.bmm(q, k.transpose(1, 2).contiguous()) * dim ** -0.5).masked_fill(~seen, -torch.inf), -1)
            want = model["o"](torch.bmm(p, v.contiguous()).transpose(0, 1).flatten(1))
            worst = max(worst, float((torch.stack(got[b]).float() - want).norm() / want.norm()))
    print(f"{seqs} sequences, prompts of {prompts.tolist()} tokens and {steps} steps of {drafts} drafted ones: within {worst:.2%} of "
          f"the dequantized weights with an unquantized cache")


if __name__ == "__main__":
    main()
