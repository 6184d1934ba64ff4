"""Serving from what the framework quantizes: an attention block whose projections are packed INT layers, with the requests'
own adapters beside them, over a cache of keys and values in 4 bits (no reference counterpart: the reference returns
dequantized weights).

    results = {r.name: r for r in model_driver.quantize_model(model, collector)}
    layers = [PackedLayer.from_result(results[name], bias=...) for name in ("q", "k", "v", "o")]
    cache = KVCache4(pages, kv_heads, head_dim)
    block = PackedAttention(*layers, cache, heads=heads)
    y = block(x, table, held, offsets)       # prompts: the sequences' new tokens, packed one after the other
    y = block(x, table, held)                # a decode step: one token a sequence

No call synchronises with the host, so a decode step may be captured in a hipGraph and replayed while `held` and `table`
change.  ``python packed_serving.py`` quantizes a small block, serves ragged prompts and decode steps from it and prints how
far the outputs are from those of the dequantized weights.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Mapping

import torch

from kv_cache import KVCache4
from packed_linear import Adapters, packed_linear


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
    """Query, key, value and output projections over one `KVCache4`; `heads` query heads, a multiple of the cache's."""

    def __init__(self, q: PackedLayer, k: PackedLayer, v: PackedLayer, out: PackedLayer, cache: KVCache4, *, heads: int,
                 window: int | None = None):
        dim, kv = cache.head_dim, cache.kv_heads
        if heads % kv:
            raise ValueError(f"{heads} query heads are no multiple of the cache's {kv}")
        for name, layer, rows in (("q", q, heads * dim), ("k", k, kv * dim), ("v", v, kv * dim)):
            if layer.words.size(0) != rows:
                raise ValueError(f"{name} has {layer.words.size(0)} rows, its heads take {rows}")
        if out.columns not in (None, heads * dim):
            raise ValueError(f"out has {out.columns} columns, the heads give {heads * dim}")
        self.q, self.k, self.v, self.out, self.cache, self.heads, self.window = q, k, v, out, cache, heads, window

    def __call__(self, x: torch.Tensor, table: torch.Tensor, held: torch.Tensor, offsets: torch.Tensor | None = None, *,
                 adapters: Mapping[str, Adapters] | None = None, index: torch.Tensor | None = None) -> torch.Tensor:
        """x [tokens, n]: the sequences' new tokens (``offsets`` [B + 1] says which are whose; None: one each), that follow
        the ``held`` [B] tokens of the cache and are appended to it; the pages are there already (``table``).  ``adapters``:
        by layer ("q", "k", "v", "out"), and ``index`` [tokens] says which one a token has."""
        of, dim = adapters or {}, self.cache.head_dim
        q = self.q(x, of.get("q"), index).unflatten(-1, (self.heads, dim))
        k = self.k(x, of.get("k"), index).unflatten(-1, (self.cache.kv_heads, dim))
        v = self.v(x, of.get("v"), index).unflatten(-1, (self.cache.kv_heads, dim))
        self.cache.append(k, v, table, held, offsets)
        lengths = held + 1 if offsets is None else held + (offsets[1:] - offsets[:-1])
        o = self.cache.attend(q, table, lengths, offsets, window=self.window)
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
    prompts, steps = torch.tensor([5, 64, 200, 1]), 8
    seqs, width = len(prompts), int((prompts.max() + steps + page - 1) // page)
    block = PackedAttention(packed["q"], packed["k"], packed["v"], packed["o"], KVCache4(seqs * width, kv, dim, page_size=page),
                            heads=heads)
    table = torch.randperm(seqs * width).to(dev, torch.int32).view(seqs, width)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), prompts.cumsum(0)]).to(dev, torch.int32)
    held = torch.zeros(seqs, dtype=torch.int32, device=dev)
    xs = [torch.randn(int(t) + steps, n, device=dev) for t in prompts]
    got = [block(torch.cat([x[:-steps] for x in xs]).bfloat16(), table, held, offsets)]
    held += prompts.to(dev, torch.int32)
    for step in range(steps):
        got.append(block(torch.stack([x[len(x) - steps + step] for x in xs]).bfloat16(), table, held))
        held += 1
    worst = 0.
    with torch.no_grad():
        for b, x in enumerate(xs):
            q, k, v = (model[name](x).unflatten(-1, (-1, dim)).transpose(0, 1) for name in "qkv")
            k, v = (t.repeat_interleave(heads // kv, 0) for t in (k, v))
            seen = torch.ones(len(x), len(x), dtype=torch.bool, device=dev).tril()
            p = torch.softmax((torch.bmm(q, k.transpose(1, 2).contiguous()) * dim ** -0.5).masked_fill(~seen, -torch.inf), -1)
            want = model["o"](torch.bmm(p, v.contiguous()).transpose(0, 1).flatten(1))
            mine = torch.cat([got[0][int(offsets[b]):int(offsets[b + 1])]] + [g[b:b + 1] for g in got[1:]])
            worst = max(worst, float((mine.float() - want).norm() / want.norm()))
    print(f"{seqs} sequences, prompts of {prompts.tolist()} tokens and {steps} decode steps: within {worst:.2%} of the "
          f"dequantized weights with an unquantized cache")


if __name__ == "__main__":
    main()
