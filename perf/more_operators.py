"""Timing cases of a decode step with drafted tokens on the 4-bit cache: rotary positions, the pages dealt to sequences on
the GPU, attention of a tree of drafted tokens, and their acceptance.

A case is a dict of plain values.  ``listed()`` are the fixed ones, ``draw(rng)`` gives more of the same ranges,
``prepare(case, seed)`` makes what a program holds before the call, ``run(state)`` is one pass (``own`` false: the plain
form, elementary torch in 32 bits, angles in 64; true: the framework's calls), ``work(case)`` the bytes and operations that
pass cannot do without, and ``exact(case, seed)`` the same outputs from the definitions in 64 bits.

Kinds of cases:

* ``rotary``: queries and keys rotated by their positions; with ``train`` their gradients too;
* ``pages``: the sequences' lengths after acceptance give pages back, the next tokens take some; the new tokens' offsets,
  positions and places in the cache;
* ``tree``: attention of a tree of drafted tokens over what its sequence holds and the nodes' own ancestors;
* ``drafts``: the drafted tokens appended, the accepted ones found and kept; gives the values then held.
"""

from __future__ import annotations

import functools
import math
import pathlib
import random
import sys

import torch

own = False

DEV = "cuda"
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_CONTEXT = 8192  # tokens that scaled frequencies were made for
_VOCABULARY = 32000


@functools.lru_cache(maxsize=None)
def _package():
    """The framework's modules, of the tree worked in."""
    path = str(pathlib.Path.cwd() / "gptq-2d_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import drafts
    import kv_cache
    import page_pool
    import rotary
    return rotary, page_pool, drafts, kv_cache


def _rotary(name, tokens, hq, hkv, dim, rotated, interleaved, scaling, far, dtype, train):
    return {"name": name, "kind": "rotary", "tokens": tokens, "hq": hq, "hkv": hkv, "dim": dim, "rotated": rotated,
            "interleaved": interleaved, "scaling": scaling, "far": far, "dtype": dtype, "train": train}


def _pages(name, seqs, new_lo, new_hi, len_lo, len_hi, drop, page):
    return {"name": name, "kind": "pages", "seqs": seqs, "new_lo": new_lo, "new_hi": new_hi, "len_lo": len_lo,
            "len_hi": len_hi, "drop": drop, "page": page}


def _nodes(name, kind, seqs, new_lo, new_hi, len_lo, len_hi, hq, hkv, dim, dtype, window=0, page=64):
    return {"name": name, "kind": kind, "seqs": seqs, "new_lo": new_lo, "new_hi": new_hi, "len_lo": len_lo,
            "len_hi": len_hi, "hq": hq, "hkv": hkv, "dim": dim, "dtype": dtype, "window": window, "page": page}


def listed():
    return [
        # a decode step of 64 sequences: all latency
        _rotary("rotary-64x40x128", 64, 32, 8, 128, 128, False, "", 131072, "bf16", False),
        # ragged: odd sizes, interleaved pairs of part of the head, fp32, far positions of scaled frequencies
        _rotary("rotary-1001x15x80-part-f32", 1001, 12, 3, 80, 44, True, "yarn", 1000000, "f32", False),
        # training: forward and backward over 16384 tokens
        _rotary("rotary-16384x40x128-train", 16384, 32, 8, 128, 128, False, "", 8192, "bf16", True),
        # a decode step: the last step's drafts accepted, eight nodes each for the next
        _pages("pages-64x8", 64, 8, 8, 100, 8000, 5, 64),
        # prompts come in beside sequences that have ended
        _pages("pages-600-prompts", 600, 0, 500, 0, 3000, 2500, 32),
        # a small tree on one short sequence
        _nodes("tree-1x7-of-1000", "tree", 1, 7, 7, 1000, 1000, 32, 8, 128, "bf16"),
        # a decode step of 64 ragged sequences, eight nodes each
        _nodes("tree-64x8-of-8000", "tree", 64, 8, 8, 300, 8000, 32, 8, 128, "bf16"),
        # long contexts with larger trees
        _nodes("tree-4x32-of-131072", "tree", 4, 32, 32, 130000, 131000, 64, 8, 128, "bf16", page=128),
        # a head size that fills no tile, fp32, a window, sequences with one node or nothing held
        _nodes("tree-9x60-dim80-window-f32", "tree", 9, 1, 60, 0, 2000, 12, 3, 80, "f32", window=300, page=32),
        # one sequence's few drafts
        _nodes("drafts-1x7", "drafts", 1, 7, 7, 1000, 1000, 0, 8, 128, "bf16"),
        # a decode step of 64 sequences
        _nodes("drafts-64x24", "drafts", 64, 24, 24, 100, 8000, 0, 8, 128, "bf16"),
        # large trees of different sizes, over several blocks and pages
        _nodes("drafts-17x300-f16", "drafts", 17, 1, 300, 0, 4000, 0, 4, 80, "f16", page=32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "pages", "tree", "tree", "tree", "drafts"])
    if kind == "rotary":
        dim = rng.choice([64, 80, 96, 128, 128, 256, rng.randint(2, 256)])
        rotated = dim // 2 * 2 if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2)
        hkv = rng.randint(1, 8)
        hq = hkv * rng.choice([1, 2, 4, 5, 8])
        train = rng.random() < 0.4
        c = _rotary("", _log(rng, 1, 16384 * 40 * 128 // ((hq + hkv) * dim) if (hq + hkv) * dim > 5120 else 16384), hq, hkv,
                    dim, rotated, rng.random() < 0.5, rng.choice(["", "linear", "ntk", "bands", "yarn"]),
                    _log(rng, 100, 1000000), rng.choice(["bf16", "f16"] if train else ["bf16", "f16", "f32"]), train)
    elif kind == "pages":
        seqs = _log(rng, 1, 600)
        new = _log(rng, 1, 500)
        hi = _log(rng, 1, 8000)
        c = _pages("", seqs, rng.choice([0, 1, new]), new, rng.choice([0, hi // 3]), hi, rng.randint(0, hi),
                   32 * rng.randint(1, 4))
    elif kind == "tree":
        hkv, ratio = rng.randint(1, 8), rng.choice([1, 2, 4, 5, 8])
        dim, dtype = rng.choice([64, 80, 96, 128, 128, 256]), rng.choice(["bf16", "bf16", "f16", "f32"])
        new = _log(rng, 1, 64)
        seqs = _log(rng, 1, max(1, 64 * 8 // new))
        hi = _log(rng, 16, min(65536, 200000 // seqs))
        window = rng.choice([0, 0, 0, _log(rng, 64, 4000)])
        c = _nodes("", kind, seqs, rng.choice([1, new]), new, rng.choice([0, hi // 3, hi]), hi, hkv * ratio, hkv, dim, dtype,
                   window, 32 * rng.randint(1, 4))
    else:
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, max(2, min(300, 5000 // seqs)))
        c = _nodes("", kind, seqs, rng.choice([1, new]), new, 0, _log(rng, 1, 4000), 0, rng.randint(1, 8),
                   rng.choice([64, 80, 128, 128, 256]), rng.choice(["bf16", "f16", "f32"]), page=32 * rng.randint(1, 4))
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ inputs

def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(1000003 * int(seed) + salt)


def _randn(shape, seed, salt):
    return torch.randn(shape, generator=_gen(seed, salt), device=DEV)


def _rand(shape, seed, salt):
    return torch.rand(shape, generator=_gen(seed, salt), device=DEV)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _spread(count, lo, hi, turn=0):
    """`count` whole numbers spread over [lo, hi] without an order (golden-ratio steps)."""
    return [lo + int((hi - lo + 1) * ((0.37 + 0.6180339887498949 * (i + turn)) % 1.0)) for i in range(count)]


def _starts(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _frequencies(case):
    """(radians a position of each pair, factor on the rotated part), in 64 bits on the host."""
    r, base, kind, factor = case["rotated"], 10000., case["scaling"], 8.
    if kind == "ntk" and r > 2:
        base *= factor ** (r / (r - 2))
    f = [base ** (-2 * i / r) for i in range(r // 2)]
    if kind == "linear":
        f = [x / factor for x in f]
    if kind == "bands":  # low frequencies divided, high ones kept, those between in proportion
        low, high, out = 1., 4., []
        for x in f:
            turns = _CONTEXT * x / (2 * math.pi)
            part = min(max((turns - low) / (high - low), 0.), 1.)
            out.append((1 - part) * x / factor + part * x)
        f = out
    if kind == "yarn":
        at = lambda turns: r * math.log(_CONTEXT / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(at(32.)), 0), min(math.ceil(at(1.)), r - 1)
        ramp = [min(max((i - low) / max(high - low, 0.001), 0.), 1.) for i in range(r // 2)]
        return [x / factor * t + x * (1 - t) for x, t in zip(f, ramp)], 0.1 * math.log(factor) + 1
    return f, 1.


def _rotary_inputs(case, seed):
    t, dim, dtype = case["tokens"], case["dim"], _DTYPES[case["dtype"]]
    # queries, keys and values side by side, as one projection gives them
    x = _randn((t, case["hq"] + 2 * case["hkv"], dim), seed, 1).to(dtype)
    q, k = x[:, :case["hq"]], x[:, case["hq"]:case["hq"] + case["hkv"]]
    first = int(torch.randint(0, max(1, case["far"] - t), (1,), generator=torch.Generator().manual_seed(int(seed))))
    if case["train"] or t > 256:  # a long sequence's, or a decode step's of many
        positions = (torch.arange(t, device=DEV) + first).to(torch.int32)
    else:
        positions = torch.randint(0, case["far"], (t,), generator=_gen(seed, 2), device=DEV).to(torch.int32)
    s = {"q": q, "k": k, "positions": positions}
    if case["train"]:
        s["q"], s["k"] = (v.detach().clone().requires_grad_() for v in (q, k))
        s["gq"], s["gk"] = (_randn(v.shape, seed, i).to(dtype) for i, v in ((3, q), (4, k)))
    if own:
        rotary, *_ = _package()
        scaling = {"": None, "linear": rotary.Linear(8.), "ntk": rotary.Ntk(8.), "bands": rotary.Bands(8., _CONTEXT),
                   "yarn": rotary.Yarn(8., _CONTEXT)}[case["scaling"]]
        s["rotary"] = rotary.Rotary(dim, rotated=case["rotated"], interleaved=case["interleaved"], scaling=scaling, device=DEV)
    else:
        f, s["amplitude"] = _frequencies(case)
        s["frequencies"] = torch.tensor(f, dtype=torch.float64, device=DEV)
    return s


def _page_sizes(case, seed=0):
    """Tokens held before the pass, tokens of them that stay, and new ones, of each sequence."""
    stay = _spread(case["seqs"], case["len_lo"], case["len_hi"])
    # some keep nothing, most drop a few
    drops = _spread(case["seqs"], 0, case["drop"], 5)
    held = [(h + d, 0 if case["drop"] > 100 and i % 3 == 0 else h) for i, (h, d) in enumerate(zip(stay, drops))]
    new = _spread(case["seqs"], case["new_lo"], case["new_hi"], 11)
    rng = random.Random(int(seed))
    rng.shuffle(held)
    rng.shuffle(new)
    return [b for b, _ in held], [h for _, h in held], new


def _pool_sizes(case):
    """Pages of the pool and of a sequence at most, enough for every order of the sequences' sizes."""
    before, stay, new = _page_sizes(case)
    up = lambda n: -(-n // case["page"])
    return (max(sum(up(b) for b in before), sum(up(h) + up(n) for h, n in zip(stay, new))) + 10,
            max(up(max(before)), up(max(stay) + max(new)), 1))


def _pages_inputs(case, seed):
    before, stay, new = _page_sizes(case, seed)
    page, seqs = case["page"], case["seqs"]
    count, width = _pool_sizes(case)
    s = {"stay": _int32(stay), "new": _int32(new), "tokens": sum(new), "seqs": seqs, "width": width, "page": page}
    if own:
        _, page_pool, *_ = _package()
        s["pool"] = page_pool.PagePool(count, seqs, width, page_size=page, device=DEV)
        s["pool"].resize(_int32(before))
    else:
        s["table"] = torch.full((seqs, width), -1, dtype=torch.int32, device=DEV)
        s["owned"] = torch.zeros(seqs, dtype=torch.int32, device=DEV)
        s["free"] = torch.arange(count - 1, -1, -1, dtype=torch.int32, device=DEV)
        s["count"] = torch.full((1,), count, dtype=torch.int32, device=DEV)
        _plain_resize(s, _int32(before))
    (_own_pages if own else _plain_pages)(s)  # a pass starts from where the last step left the pool
    return s


def _sizes(case):
    """(nodes, tokens held before them) of each sequence."""
    return _spread(case["seqs"], case["new_lo"], case["new_hi"], 3), _spread(case["seqs"], case["len_lo"], case["len_hi"])


def _kv(case, seed, rows, salt):
    """Keys or values [rows, hkv, dim]: normal, with a spread and a mean per channel."""
    hkv, dim = case["hkv"], case["dim"]
    x = _randn((rows, hkv, dim), seed, salt)
    x.mul_(_randn((hkv, dim), seed, salt + 1).mul_(0.4).exp_()).add_(_randn((hkv, dim), seed, salt + 2).mul_(0.5))
    return x.to(_DTYPES[case["dtype"]])


def _padded_positions(starts, counts):
    """Row of each (sequence, position) among packed rows, 0 where a sequence has none, and whether it has one."""
    at = torch.arange(max(max(counts), 1), device=DEV)
    has = at < _int32(counts)[:, None]
    return torch.where(has, _int32(starts[:-1])[:, None] + at, 0), has


def _trees(new, seed):
    """Parents of the nodes (a random earlier node of the tree; -1: the first), drafted tokens, and those that the model
    chose after each: usually that of a child."""
    starts = _starts(new)
    index = torch.cat([torch.arange(n, device=DEV) for n in new])
    parents = ((index * _rand(index.shape, seed, 60)).floor().clamp(max=index - 1)).to(torch.int32)
    drafted = torch.randint(0, _VOCABULARY, index.shape, generator=_gen(seed, 61), device=DEV)
    base = torch.repeat_interleave(_int32(starts[:-1]).long(), _int32(new).long())
    child = torch.full_like(index, -1)
    child.scatter_reduce_(0, (base + parents)[parents >= 0], (base + index)[parents >= 0], "amax")  # the last one
    chosen = torch.randint(0, _VOCABULARY, index.shape, generator=_gen(seed, 62), device=DEV)
    follows = (child >= 0) & (_rand(index.shape, seed, 63) < 0.9)
    return parents, drafted, torch.where(follows, drafted[child.clamp(min=0)], chosen)


def _quantized(x):
    """Codes packed two a byte, scale and zero of x [..., dim]: what a plain program keeps of keys or values in 4 bits."""
    x = x.float()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((hi - lo) / torch.full((1,), 15., device=DEV)).to(torch.bfloat16)
    scale = torch.where(scale == 0, 1., scale).to(torch.bfloat16)
    zero = lo.to(torch.bfloat16)
    codes = ((x - zero.float()) / scale.float()).round().clamp(0, 15).to(torch.uint8)
    return codes[..., 0::2] | codes[..., 1::2] << 4, scale, zero


def _values(q):
    """The values that _quantized's answer stands for, in 32 bits."""
    codes, scale, zero = q
    return torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).float() * scale.float() + zero.float()


def _cache_inputs(case, seed):
    new, held = _sizes(case)
    page = case["page"]
    blocks = [-(-(h + n) // page) for h, n in zip(held, new)]
    order = torch.randperm(max(1, sum(blocks)), generator=_gen(seed, 20), device=DEV).to(torch.int32)
    at, has = _padded_positions(_starts(blocks), blocks)
    s = {"table": torch.where(has, order[at], 0).to(torch.int32).contiguous(), "held": _int32(held),
         "lengths": _int32([h + n for h, n in zip(held, new)]), "offsets": _int32(_starts(new)), "tokens": sum(new),
         "pages": max(1, sum(blocks)), "nodes": max(new), "new": _int32(new), "dtype": case["dtype"]}
    s["parents"], s["drafted"], s["chosen"] = _trees(new, seed)
    if own:
        *_, kv_cache = _package()
        s["cache"] = kv_cache.KVCache4(s["pages"], case["hkv"], case["dim"], page_size=page, device=DEV)
    else:
        s["at"], s["has"] = _padded_positions(_starts(new), new)
        # rows back: the place of each packed row among the padded ones
        s["flat"] = torch.nonzero(s["has"].flatten()).flatten()
    return s, new, held


def _tree_inputs(case, seed):
    s, new, held = _cache_inputs(case, seed)
    after = [h + n for h, n in zip(held, new)]
    k, v = _kv(case, seed, sum(after), 30), _kv(case, seed, sum(after), 40)
    q = _randn((s["tokens"], case["hq"], case["dim"]), seed, 50).to(_DTYPES[case["dtype"]])
    s.update(q=q, scale=case["dim"] ** -0.5)
    s["window"] = max(case["window"], max(new)) if case["window"] else None
    if own:  # a cache filled by appending, and the tree that all layers share
        _, _, drafts, _ = _package()
        s["cache"].append(k, v, s["table"], torch.zeros_like(s["lengths"]), _int32(_starts(after)))
        s["tree"] = drafts.DraftTree(s["parents"], s["offsets"], s["held"], nodes=s["nodes"])
    else:  # the same in a plain padded cache, and the mask
        at, has = _padded_positions(_starts(after), after)
        for name, x in (("k", k), ("v", v)):
            s[name] = [torch.where(has.view(*has.shape, 1, 1), p[at], torch.zeros((), dtype=p.dtype, device=DEV))
                       for p in _quantized(x)]
        line, depth = _lines(s)
        key = torch.arange(at.size(1), device=DEV)
        rel = key - s["held"][:, None]  # [B, S]: the key's node
        seen = torch.gather(line, 2, rel.clamp(0, line.size(2) - 1)[:, None].expand(-1, line.size(1), -1))
        seen = torch.where((rel < 0)[:, None], True, seen & (rel < s["new"][:, None])[:, None])
        if s["window"]:  # ancestors are always inside
            seen = seen & ((rel >= 0)[:, None] | (key > (s["held"][:, None] + depth)[:, :, None] - s["window"]))
        s["seen"] = seen & s["has"][:, :, None]
    return s


def _drafts_inputs(case, seed):
    s, new, held = _cache_inputs(case, seed)
    s["k"], s["v"] = _kv(case, seed, s["tokens"], 30), _kv(case, seed, s["tokens"], 40)
    return s


_INPUTS = {"rotary": _rotary_inputs, "pages": _pages_inputs, "tree": _tree_inputs, "drafts": _drafts_inputs}


def prepare(case, seed):
    return {"kind": case["kind"], "case": case, **_INPUTS[case["kind"]](case, seed)}


# ------------------------------------------------------------------------------------------------ one pass

def _rotated(x, cos, sin, rotated, interleaved):
    """x [tokens, heads, dim] in 32 bits, its first `rotated` elements by the angles [tokens, 1, rotated / 2]."""
    a, rest = x[..., :rotated].float(), x[..., rotated:].float()
    if interleaved:
        one, two = a[..., 0::2], a[..., 1::2]
    else:
        one, two = a[..., :rotated // 2], a[..., rotated // 2:]
    y1, y2 = one * cos - two * sin, two * cos + one * sin
    y = torch.stack([y1, y2], -1).flatten(-2) if interleaved else torch.cat([y1, y2], -1)
    return torch.cat([y, rest], -1).to(x.dtype)


def _plain_rotary(s):
    c = s["case"]
    angle = (s["positions"].double()[:, None] * s["frequencies"])[:, None]
    cos, sin = ((f(angle) * s["amplitude"]).float() for f in (torch.cos, torch.sin))
    out = [_rotated(x, cos, sin, c["rotated"], c["interleaved"]) for x in (s["q"], s["k"])]
    if c["train"]:
        return [*(o.detach() for o in out), *torch.autograd.grad(out, (s["q"], s["k"]), (s["gq"], s["gk"]))]
    return out


def _plain_resize(s, lengths):
    """Pages of sequences that need fewer go back on the stack, the next ones' on top; then, sequence by sequence, those that
    need more take from its top."""
    want = ((lengths + (s["page"] - 1)) // s["page"]).clamp(max=s["width"])[:, None]
    had = s["owned"][:, None]
    p = torch.arange(s["width"], device=DEV)
    give, take = ((p >= want) & (p < had)).flatten(), ((p >= had) & (p < want)).flatten()
    table = s["table"].flatten()
    rank = give.flip(0).cumsum(0).flip(0) - 1  # the last page first
    free = s["free"].scatter(0, (s["count"] + rank)[give], table[give])
    top = s["count"] + give.sum()
    at = top - take.cumsum(0)
    got = take & (at >= 0)
    table = torch.where(give, -1, table)
    table = torch.where(got, free[at.clamp(0, free.numel() - 1)], table)
    s["table"], s["free"] = table.view(-1, s["width"]).to(torch.int32), free
    s["owned"] = (torch.minimum(s["owned"], want[:, 0]) + got.view(-1, s["width"]).sum(1)).to(torch.int32)
    s["count"] = (top - got.sum()).to(torch.int32)


def _plain_pages(s):
    _plain_resize(s, s["stay"])
    lengths = s["stay"] + s["new"]
    _plain_resize(s, lengths)
    ends = s["new"].cumsum(0)
    offsets = torch.nn.functional.pad(ends, (1, 0)).to(torch.int32)
    row = torch.arange(s["tokens"], device=DEV)
    owner = torch.searchsorted(ends, row, right=True)
    positions = s["stay"][owner] + row - offsets[owner]
    page = positions // s["page"]
    entry = s["table"][owner, page.clamp(max=s["width"] - 1)].long()
    slots = torch.where((page < s["width"]) & (entry >= 0), entry * s["page"] + positions % s["page"], -1)
    return {"table": s["table"], "owned": s["owned"], "left": s["count"], "lengths": lengths, "offsets": offsets,
            "positions": positions.to(torch.int32), "slots": slots}


def _own_pages(s):
    pool = s["pool"]
    pool.resize(s["stay"])
    rows = pool.extend(s["new"], tokens=s["tokens"])
    return {"table": pool.table, "owned": pool.owned, "left": pool.left, "lengths": pool.lengths, "offsets": rows.offsets,
            "positions": rows.positions, "slots": rows.slots}


def _lines(s):
    """Which nodes each node comes from, itself among them, [B, nodes, nodes], and how many are before it."""
    n = s["at"].size(1)
    parents = torch.where(s["has"], s["parents"][s["at"]], -1).long()
    line = torch.zeros(*s["at"].shape, n, dtype=torch.bool, device=DEV)
    at = torch.arange(n, device=DEV).expand_as(parents)
    depth = torch.full_like(parents, -1)
    for _ in range(n):
        there = at >= 0
        line |= there[:, :, None] & (torch.arange(n, device=DEV) == at[:, :, None])
        depth += there
        at = torch.where(there, torch.gather(parents, 1, at.clamp(min=0)), -1)
    return line, depth


def _plain_tree(s):
    c = s["case"]
    hq, hkv, dim, t = c["hq"], c["hkv"], c["dim"], s["at"].size(1)
    k, v = _values(s["k"]).permute(0, 2, 3, 1), _values(s["v"]).permute(0, 2, 1, 3)  # [B, hkv, dim, S], [B, hkv, S, dim]
    q = s["q"].float()[s["at"]].view(-1, t, hkv, hq // hkv, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = (q @ k).view(*q.shape[:2], hq // hkv, t, -1) * s["scale"]  # [B, hkv, group, t, S]
    seen = s["seen"][:, None, None]
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(scores - top), 0.)
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, 1.)
    o = p.flatten(2, 3) @ v
    o = o.view(*o.shape[:2], hq // hkv, t, dim).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [B, t, hq, dim]
    return o.flatten(0, 1)[s["flat"]].to(s["q"].dtype)


def _plain_drafts(s):
    n = s["at"].size(1)
    parents = torch.where(s["has"], s["parents"][s["at"]], -2).long()  # -2: no node
    depth, at = torch.zeros_like(parents), parents
    for _ in range(n):
        depth += at >= 0
        at = torch.where(at >= 0, torch.gather(parents, 1, at.clamp(min=0)), -1)
    positions = (s["held"][:, None] + depth).flatten()[s["flat"]].to(torch.int32)
    drafted, chosen = s["drafted"][s["at"]], s["chosen"][s["at"]]
    node = torch.arange(n, device=DEV)
    at, going = torch.zeros_like(parents[:, :1]), s["has"][:, :1]
    path, count, last = [], torch.zeros_like(parents[:, 0]), torch.full_like(parents[:, 0], -1)
    for _ in range(n):
        path.append(torch.where(going, at, -1))
        count += going[:, 0]
        picked = torch.gather(chosen, 1, at)
        last = torch.where(going, picked, last[:, None])[:, 0]
        match = (parents == at) & (drafted == picked)
        child = torch.where(match, node, n).amin(1, keepdim=True)
        going = going & (child < n)
        at = torch.where(going, child, at)
    path = torch.cat(path, 1)
    # the accepted nodes' entries first; what follows them stays
    from_node = torch.where(path >= 0, path, node)
    rows = torch.gather(s["at"], 1, from_node).flatten()[s["flat"]]
    k, v = (_values([p[rows] for p in _quantized(s[name])]) for name in ("k", "v"))
    return {"positions": positions, "path": path.to(torch.int32), "counts": count.to(torch.int32), "next": last, "k": k, "v": v}


def _own_drafts(s):
    _, _, drafts, _ = _package()
    tree = drafts.DraftTree(s["parents"], s["offsets"], s["held"], nodes=s["nodes"])
    s["cache"].append(s["k"], s["v"], s["table"], s["held"], s["offsets"])
    accepted = tree.accept(s["drafted"], s["chosen"])
    s["cache"].keep(s["table"], s["lengths"], s["offsets"], accepted.path, accepted.counts)
    k, v = s["cache"].read(s["table"], s["lengths"], s["offsets"], tokens=s["tokens"], dtype=torch.float32)
    return {"positions": tree.positions, "path": accepted.path, "counts": accepted.counts, "next": accepted.next, "k": k, "v": v}


def _own_rotary(s):
    out = s["rotary"](s["q"], s["k"], positions=s["positions"])
    if s["case"]["train"]:
        return [*(o.detach() for o in out), *torch.autograd.grad(out, (s["q"], s["k"]), (s["gq"], s["gk"]))]
    return list(out)


def _own_tree(s):
    return s["cache"].attend(s["q"], s["table"], s["lengths"], s["offsets"], scale=s["scale"], window=s["window"], tree=s["tree"])


_PLAIN = {"rotary": _plain_rotary, "pages": _plain_pages, "tree": _plain_tree, "drafts": _plain_drafts}
_OWN = {"rotary": _own_rotary, "pages": _own_pages, "tree": _own_tree, "drafts": _own_drafts}


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


# ------------------------------------------------------------------------------------------------ work and 64 bits

def work(case):
    if case["kind"] == "rotary":
        moved = case["tokens"] * (case["hq"] + case["hkv"]) * case["dim"] * (2 if case["train"] else 1)
        return {"bytes": 2 * moved * _BYTES[case["dtype"]] + 4 * case["tokens"],
                "flops": 3 * moved * case["rotated"] // case["dim"]}
    if case["kind"] == "pages":
        before, stay, new = _page_sizes(case)
        up = lambda t: -(-t // case["page"])
        moved = sum(up(h + n) - up(h) for h, n in zip(stay, new))
        return {"bytes": 2 * 16 * moved + 12 * sum(new) + 40 * case["seqs"], "flops": 8 * sum(new) + 8 * moved}
    size, (new, held) = _BYTES[case["dtype"]], _sizes(case)
    hkv, dim = case["hkv"], case["dim"]
    if case["kind"] == "drafts":  # read, written in 4 bits with scale and zero, and the values then held given
        return {"bytes": sum(new) * (2 * hkv * (dim * size + dim // 2 + 4 + dim * 4) + 24) + 4 * case["seqs"] * max(new),
                "flops": 8 * sum(new) * hkv * dim}
    window = max(case["window"], max(new)) if case["window"] else 1 << 40
    keys = sum(min(h, window - 1) + n for h, n in zip(held, new))
    # a random tree: half of its nodes are no ancestors at least, and the work counts none of them
    pairs = sum(n * min(h, window - 1) + 2 * n for h, n in zip(held, new))
    return {"bytes": 2 * keys * hkv * (dim // 2 + 4) + 2 * sum(new) * case["hq"] * dim * size,
            "flops": 4 * pairs * case["hq"] * dim}


def _exact_rotary(case, seed):
    t, rotated = case["tokens"], case["rotated"]
    s = _rotary_inputs(case, seed)
    f, amplitude = _frequencies(case)
    angle = s["positions"].to(torch.float64)[:, None] * torch.tensor(f, dtype=torch.float64, device=DEV)
    turn = torch.polar(torch.full_like(angle, amplitude), angle)[:, None]
    half = rotated // 2

    def turned(x, by):
        x = x.detach().to(torch.float64)
        y = x.clone()
        first = slice(0, rotated, 2) if case["interleaved"] else slice(0, half)
        second = slice(1, rotated, 2) if case["interleaved"] else slice(half, rotated)
        z = torch.complex(x[..., first], x[..., second]) * by
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = [turned(s["q"], turn), turned(s["k"], turn)]
    if case["train"]:
        out += [turned(s["gq"], turn.conj()), turned(s["gk"], turn.conj())]
    return out


def _exact_pages(case, seed):
    before, stay, new = _page_sizes(case, seed)
    page = case["page"]
    count, width = _pool_sizes(case)
    stack = list(range(count - 1, -1, -1))
    table = [[] for _ in before]

    def resize(lengths):
        want = [min(-(-n // page), width) for n in lengths]
        for mine, w in reversed(list(zip(table, want))):
            while len(mine) > w:
                stack.append(mine.pop())
        for mine, w in zip(table, want):
            while len(mine) < w and stack:
                mine.append(stack.pop())

    after = [h + n for h, n in zip(stay, new)]
    for lengths in (before, stay, after, stay, after):  # the preparation's pass, and this one
        resize(lengths)
    positions = [h + i for h, n in zip(stay, new) for i in range(n)]
    slots = [mine[(h + i) // page] * page + (h + i) % page if (h + i) // page < len(mine) else -1
             for mine, h, n in zip(table, stay, new) for i in range(n)]
    return {"table": _int32([mine + [-1] * (width - len(mine)) for mine in table]), "owned": _int32([len(m) for m in table]),
            "left": _int32([len(stack)]), "lengths": _int32(after), "offsets": _int32(_starts(new)),
            "positions": _int32(positions), "slots": torch.tensor(slots, dtype=torch.int64, device=DEV)}


def _fp32(x):
    """x rounded to 32 bits, in 64: where the operator's definition has a number of 32 bits."""
    return x.to(torch.float32).to(torch.float64)


def _exact_values(x):
    """Values held in 4 bits for x [..., dim], from the definition: scale and zero rounded to bf16, the quotients to 32
    bits (of 64-bit differences and quotients of 32-bit numbers that is the correctly rounded one)."""
    x = x.to(torch.float64)
    low = x.min(dim=-1, keepdim=True).values
    scale = _fp32(_fp32(x.max(dim=-1, keepdim=True).values - low) / 15).to(torch.float32).to(torch.bfloat16).to(torch.float64)
    scale[scale == 0] = 1
    zero = low.to(torch.float32).to(torch.bfloat16).to(torch.float64)
    return torch.clamp(torch.round(_fp32(_fp32(x - zero) / scale)), 0, 15) * scale + zero


def _ancestors(parents):
    """Lists of the nodes that each node comes from, the nearest first, itself before them."""
    lines = []
    for i, p in enumerate(parents):
        lines.append([i] + (lines[p] if p >= 0 else []))
    return lines


def _exact_drafts(case, seed):
    new, held = _sizes(case)
    parents, drafted, chosen = (t.tolist() for t in _trees(new, seed))
    positions, path, rows, last = [], [], [], []
    at = 0
    for n, h in zip(new, held):
        mine = parents[at:at + n]
        positions += [h + len(line) - 1 for line in _ancestors(mine)]
        node, way = 0, [0]
        while True:
            child = next((c for c in range(n) if mine[c] == node and drafted[at + c] == chosen[at + node]), None)
            if child is None:
                break
            node = child
            way.append(node)
        last.append(chosen[at + node])
        rows += [at + (way[i] if i < len(way) else i) for i in range(n)]
        path.append(way)
        at += n
    rows = torch.tensor(rows, device=DEV)
    return {"positions": _int32(positions), "path": _int32([w + [-1] * (max(new) - len(w)) for w in path]),
            "counts": _int32([len(w) for w in path]), "next": torch.tensor(last, device=DEV),
            "k": _exact_values(_kv(case, seed, sum(new), 30))[rows], "v": _exact_values(_kv(case, seed, sum(new), 40))[rows]}


def _exact_tree(case, seed):
    new, held = _sizes(case)
    after = [h + n for h, n in zip(held, new)]
    k, v = _kv(case, seed, sum(after), 30), _kv(case, seed, sum(after), 40)
    q = _randn((sum(new), case["hq"], case["dim"]), seed, 50).to(_DTYPES[case["dtype"]]).to(torch.float64)
    parents = _trees(new, seed)[0].tolist()
    window = max(case["window"], max(new)) if case["window"] else 0
    out, group = torch.zeros_like(q), case["hq"] // case["hkv"]
    q0 = k0 = 0
    for n, h in zip(new, held):
        kk, vv = _exact_values(k[k0:k0 + h + n]), _exact_values(v[k0:k0 + h + n])
        hidden = torch.ones(n, h + n, dtype=torch.bool)
        for i, line in enumerate(_ancestors(parents[q0:q0 + n])):
            position = h + len(line) - 1
            hidden[i, max(0, position + 1 - window) if window else 0:h] = False
            hidden[i, [h + j for j in line]] = False
        hidden = hidden.to(DEV)
        for head in range(case["hq"]):
            z = torch.matmul(q[q0:q0 + n, head], kk[:, head // group].t().contiguous()) * case["dim"] ** -0.5
            weight = torch.softmax(z.masked_fill_(hidden, -math.inf), dim=-1)
            out[q0:q0 + n, head] = torch.matmul(weight, vv[:, head // group].contiguous())
        q0, k0 = q0 + n, k0 + h + n
    return out


def exact(case, seed):
    if case["kind"] == "rotary":
        return _exact_rotary(case, seed)
    if case["kind"] == "pages":
        return _exact_pages(case, seed)
    return _exact_drafts(case, seed) if case["kind"] == "drafts" else _exact_tree(case, seed)
