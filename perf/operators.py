"""Timing cases of what serves a quantized model: products with packed INT layers beside the low-rank adapters of many
requests, and attention over a paged cache of keys and values in 4 bits, with the append that fills it.

A case is a dict of plain values.  ``listed()`` are the fixed ones, ``draw(rng)`` gives more of the same ranges,
``prepare(case, seed)`` makes what a program holds before the call, ``run(state)`` is one pass (``own`` false: the plain
form, elementary torch in 32 bits; true: the framework's calls), ``work(case)`` the bytes and operations that pass cannot
do without, and ``exact(case, seed)`` the same outputs from the definitions in 64 bits.

Kinds of cases:

* ``linear``: y = x W^T with W [m, n] held as packed INT codes, plus each token's own adapter, scaling (x A^T) B^T;
* ``append``: new keys and values of several sequences into the cache; gives the values that are then held for them;
* ``attend``: causal attention of the last tokens of several sequences over all that their caches hold.
"""

from __future__ import annotations

import functools
import math
import pathlib
import sys

import torch

own = False

DEV = "cuda"
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


@functools.lru_cache(maxsize=None)
def _package():
    """The framework's modules, of the tree worked in."""
    path = str(pathlib.Path.cwd() / "gptq-2d_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import kv_cache
    import packed_linear
    return packed_linear, kv_cache


def _spread(count, lo, hi):
    """`count` whole numbers spread over [lo, hi] without an order (golden-ratio steps)."""
    return [lo + int((hi - lo + 1) * ((0.37 + 0.6180339887498949 * i) % 1.0)) for i in range(count)]


def _linear(name, tokens, m, n, bits, group, zero, dtype, adapters, rank):
    return {"name": name, "kind": "linear", "tokens": tokens, "m": m, "n": n, "bits": bits, "group": group, "zero": zero,
            "dtype": dtype, "adapters": adapters, "rank": rank}


def _cache(name, kind, seqs, new_lo, new_hi, len_lo, len_hi, hq, hkv, dim, dtype, window=0, page=64):
    return {"name": name, "kind": kind, "seqs": seqs, "new_lo": new_lo, "new_hi": new_hi, "len_lo": len_lo,
            "len_hi": len_hi, "hq": hq, "hkv": hkv, "dim": dim, "dtype": dtype, "window": window, "page": page}


def listed():
    return [
        # one token of one request through a square INT4 projection: all latency
        _linear("linear-1x4096x4096-int4", 1, 4096, 4096, 4, 0, False, "bf16", 4, 16),
        # a decode batch, every request with an adapter of its own, an MLP projection in asymmetric INT4 groups
        _linear("linear-16x14336x4096-g128", 16, 14336, 4096, 4, 128, True, "f16", 16, 16),
        # ragged: odd sizes, 3-bit codes, fp32 activations, an odd rank, some tokens without an adapter
        _linear("linear-67x3000x4095-int3-f32", 67, 3000, 4095, 3, 0, False, "f32", 5, 9),
        # a decode batch through the largest down projection, a scale per 1 x 32 row
        _linear("linear-32x8192x28672-rows32", 32, 8192, 28672, 4, 32, False, "bf16", 8, 32),
        # prompts of four requests at once: the matrix cores are the bound
        _linear("linear-2048x8192x8192-g128", 2048, 8192, 8192, 4, 128, True, "bf16", 4, 64),
        # a decode step of 64 sequences
        _cache("append-64x1", "append", 64, 1, 1, 100, 4000, 0, 8, 128, "bf16"),
        # two prompts that begin and end inside a page
        _cache("append-2x4000", "append", 2, 3500, 4500, 0, 77, 0, 8, 128, "f16"),
        # one token of one short sequence
        _cache("attend-1x1000", "attend", 1, 1, 1, 1000, 1000, 32, 8, 128, "bf16"),
        # a decode step of 64 ragged sequences
        _cache("attend-64x8000", "attend", 64, 1, 1, 300, 8000, 32, 8, 128, "bf16"),
        # a decode step of four long contexts
        _cache("attend-4x131072", "attend", 4, 1, 1, 130000, 131072, 64, 8, 128, "bf16", page=128),
        # a few tokens each (checked guesses), fp32, a head size that fills no tile, a window, sequences without a token
        _cache("attend-9x5-dim80-window", "attend", 9, 5, 5, 0, 2000, 12, 3, 80, "f32", window=300, page=32),
        # a prompt's last piece over what came before it
        _cache("attend-2048-of-8192", "attend", 1, 2048, 2048, 8192, 8192, 32, 8, 128, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    odd = lambda v, to: v if rng.random() < 0.5 else max(to, v // to * to)  # half of the sizes are whatever came up
    kind = rng.choice(["linear", "linear", "linear", "append", "attend", "attend", "attend"])
    if kind == "linear":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        tokens = _log(rng, 1, 300 if dtype == "f32" else 2048)
        adapters = rng.choice([0, 1, 3, 8, 20, 32])
        c = _linear("", tokens, odd(_log(rng, 200, 8192), 32), odd(_log(rng, 200, 8192), 32), rng.choice([2, 3, 4, 4, 4, 8]),
                    rng.choice([0, 0, 32, 64, 128]), rng.random() < 0.5, dtype, adapters, _log(rng, 4, 64) if adapters else 0)
    elif kind == "append":
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, max(2, 8000 // seqs))
        c = _cache("", kind, seqs, max(1, new // 2), new, 0, _log(rng, 1, 4000), 0, rng.randint(1, 8),
                   rng.choice([64, 80, 128, 128, 256]), rng.choice(["bf16", "f16", "f32"]), page=32 * rng.randint(1, 4))
    else:
        hkv, ratio = rng.randint(1, 8), rng.choice([1, 2, 4, 5, 8])
        dim, dtype = rng.choice([64, 96, 128, 128, 256]), rng.choice(["bf16", "bf16", "f16", "f32"])
        new = rng.choice([1, 1, 1, _log(rng, 2, 8), _log(rng, 8, 512)])
        seqs = _log(rng, 1, 64) if new < 9 else rng.randint(1, 2)
        most = min(65536, 250000 // seqs) if new < 9 else 4096
        hi = max(new, _log(rng, 16, most))
        c = _cache("", kind, seqs, new, new, rng.choice([0, hi // 3, hi]), hi, hkv * ratio, hkv, dim, dtype,
                   rng.choice([0, 0, 0, _log(rng, 8, 4000)]), 32 * rng.randint(1, 4))
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ inputs

def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(1000003 * int(seed) + salt)


def _randn(shape, seed, salt):
    return torch.randn(shape, generator=_gen(seed, salt), device=DEV)


def _pack_words(codes, bits):
    """Codes [m, n] as little-endian bit fields in int32 words [m, ceil(n bits / 32)]."""
    m, n = codes.shape
    per = 32 // math.gcd(32, bits)  # codes that fill whole words
    pad = torch.nn.functional.pad(codes, (0, -n % per)).to(torch.int64).view(m, -1, per)
    out = []
    for word in range(per * bits // 32):
        acc = torch.zeros(pad.shape[:2], dtype=torch.int64, device=DEV)
        for i in range(per):
            at = i * bits - 32 * word
            if -bits < at < 32:
                acc |= (pad[:, :, i] << at if at >= 0 else pad[:, :, i] >> -at) & 0xffffffff
        out.append(acc)
    words = torch.stack(out, dim=2).view(m, -1)[:, :-(-n * bits // 32)]
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32).contiguous()


def _linear_inputs(case, seed):
    t, m, n, bits, r = (case[k] for k in ("tokens", "m", "n", "bits", "rank"))
    dtype, half = _DTYPES[case["dtype"]], 1 << (bits - 1)
    groups = -(-n // case["group"]) if case["group"] else 1
    # normal weights over the code range of an abs-max scale
    codes = (_randn((m, n), seed, 1).mul_(half / 3.2).round_().clamp_(-half, half - 1) + half).to(torch.uint8)
    s = {"words": _pack_words(codes, bits), "qmin": -half, "qmax": half - 1}
    del codes
    s["scale"] = _randn((m, groups), seed, 2).mul_(0.15).exp_().mul_(0.02 * 3.2 / half).to(torch.bfloat16).float()
    s["zero"] = _randn((m, groups), seed, 3).mul_(half / 6).round_().clamp_(-half, half - 1) if case["zero"] else None
    x = _randn((t, n), seed, 4)
    x[:, ::97] *= 12.  # a few large channels, as activations have them
    s["x"] = x.to(dtype)
    s["adapters"] = s["index"] = None
    if case["adapters"]:
        a = case["adapters"]
        s["adapters"] = (_randn((a, r, n), seed, 5).mul_(n ** -0.5).to(dtype), _randn((a, m, r), seed, 6).mul_(0.02).to(dtype),
                         torch.rand(a, generator=_gen(seed, 7), device=DEV) + 0.5)
        # short batches: a request a token; long ones: requests one after the other; a tenth of them without an adapter
        which = torch.randint(0, 10 * a, (max(a, 1),), generator=_gen(seed, 8), device=DEV)
        which = torch.where(which < a, -1, which % a).to(torch.int32)
        s["index"] = which[torch.arange(t, device=DEV) * which.numel() // max(t, which.numel())].contiguous()
    return s


def _sizes(case):
    """(new tokens, tokens held after them) of each sequence."""
    new = _spread(case["seqs"], case["new_lo"], case["new_hi"])
    held = _spread(case["seqs"], case["len_lo"], case["len_hi"])
    if case["kind"] == "append":
        held = [h + t for h, t in zip(held, new)]
    return new, held


def _kv(case, seed, rows, salt):
    """Keys or values [rows, hkv, dim]: normal, with a spread and a mean per channel."""
    hkv, dim = case["hkv"], case["dim"]
    x = _randn((rows, hkv, dim), seed, salt)
    x.mul_(_randn((hkv, dim), seed, salt + 1).mul_(0.4).exp_()).add_(_randn((hkv, dim), seed, salt + 2).mul_(0.5))
    return x.to(_DTYPES[case["dtype"]])


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _padded_positions(starts, counts):
    """Row of each (sequence, position) among packed rows, 0 where a sequence has none, and whether it has one."""
    at = torch.arange(max(max(counts), 1), device=DEV)
    has = at < _int32(counts)[:, None]
    return torch.where(has, _int32(starts[:-1])[:, None] + at, 0), has


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
    blocks = [-(-h // page) for h in held]
    width = max(max(blocks), 1)
    order = torch.randperm(max(1, sum(blocks)), generator=_gen(seed, 20), device=DEV).to(torch.int32)
    at, has = _padded_positions(_starts(blocks), blocks)
    s = {"table": torch.where(has, order[at], 0).to(torch.int32).contiguous(), "lengths": _int32(held), "width": width,
         "offsets": None if case["new_hi"] == 1 else _int32(_starts(new)), "tokens": sum(new),
         "pages": max(1, sum(blocks)), "dtype": case["dtype"]}
    return s, new, held


def _append_inputs(case, seed):
    s, new, held = _cache_inputs(case, seed)
    s["k"], s["v"] = _kv(case, seed, s["tokens"], 30), _kv(case, seed, s["tokens"], 40)
    s["before"] = _int32([h - t for h, t in zip(held, new)])
    if own:
        _, kv_cache = _package()
        s["cache"] = kv_cache.KVCache4(s["pages"], case["hkv"], case["dim"], page_size=case["page"], device=DEV)
    return s


def _attend_inputs(case, seed):
    s, new, held = _cache_inputs(case, seed)
    k, v = _kv(case, seed, sum(held), 30), _kv(case, seed, sum(held), 40)
    q = _randn((s["tokens"], case["hq"], case["dim"]), seed, 50).to(_DTYPES[case["dtype"]])
    s.update(q=q, scale=case["dim"] ** -0.5, window=case["window"] or None)
    if own:  # a cache that was filled by appending, as a program has it
        _, kv_cache = _package()
        s["cache"] = kv_cache.KVCache4(s["pages"], case["hkv"], case["dim"], page_size=case["page"], device=DEV)
        s["cache"].append(k, v, s["table"], torch.zeros_like(s["lengths"]), _int32(_starts(held)))
    else:  # the same in a plain padded cache
        at, has = _padded_positions(_starts(held), held)
        for name, x in (("k", k), ("v", v)):
            parts = _quantized(x) if sum(held) else _quantized(torch.zeros_like(_kv(case, seed, 1, 30)))
            s[name] = [torch.where(has.view(*has.shape, 1, 1), p[at], torch.zeros((), dtype=p.dtype, device=DEV)) for p in parts]
        s["new"] = max(new)
        s["at"], s["has"] = _padded_positions(_starts(new), new)
        s["news"] = _int32(new)
    return s


_INPUTS = {"linear": _linear_inputs, "append": _append_inputs, "attend": _attend_inputs}


def prepare(case, seed):
    return {"kind": case["kind"], "case": case, **_INPUTS[case["kind"]](case, seed)}


# ------------------------------------------------------------------------------------------------ one pass

def _plain_linear(s):
    c = s["case"]
    bits, n = c["bits"], c["n"]
    bit = torch.arange(n, device=DEV) * bits
    word, shift = bit // 32, bit % 32
    if 32 % bits == 0:
        codes = s["words"][:, word] >> shift & (1 << bits) - 1
    else:  # fields that cross words: both words as one 64-bit number
        wide = s["words"].to(torch.int64) & 0xffffffff
        wide = torch.nn.functional.pad(wide, (0, 1))
        codes = (wide[:, word] | wide[:, word + 1] << 32) >> shift & (1 << bits) - 1
    group = torch.arange(n, device=DEV) // (c["group"] or n)
    off = float(s["qmin"]) if s["zero"] is None else s["qmin"] - s["zero"][:, group]
    weights = (codes.float() + off) * s["scale"][:, group]
    x = s["x"].float()
    y = x @ weights.t()
    if s["adapters"] is not None:  # every token through every adapter, all but its own masked
        a, b, scaling = (v.float() for v in s["adapters"])
        count, rank = a.shape[:2]
        inner = (x @ a.flatten(0, 1).t()).view(-1, count, rank) * scaling[:, None]
        inner = torch.where((s["index"][:, None] == torch.arange(count, device=DEV))[:, :, None], inner, 0.)
        y += inner.flatten(1) @ b.permute(0, 2, 1).flatten(0, 1)
    return y.to(s["x"].dtype)


def _plain_append(s):
    return {"k": _values(_quantized(s["k"])), "v": _values(_quantized(s["v"]))}


def _plain_attend(s):
    c = s["case"]
    hq, hkv, dim, t = c["hq"], c["hkv"], c["dim"], s["new"]
    k, v = _values(s["k"]).permute(0, 2, 3, 1), _values(s["v"]).permute(0, 2, 1, 3)  # [B, hkv, dim, S], [B, hkv, S, dim]
    q = s["q"].float()[s["at"]].view(-1, t, hkv, hq // hkv, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = (q @ k).view(*q.shape[:2], hq // hkv, t, -1) * s["scale"]  # [B, hkv, group, t, S]
    position = (s["lengths"] - s["news"])[:, None] + torch.arange(t, device=DEV)  # [B, t]
    key = torch.arange(k.size(-1), device=DEV)
    seen = key <= position[:, :, None]
    if s["window"]:
        seen = seen & (key > position[:, :, None] - s["window"])
    seen = seen[:, None, None]
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(scores - top), 0.)
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, 1.)
    o = p.flatten(2, 3) @ v
    o = o.view(*o.shape[:2], hq // hkv, t, dim).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [B, t, hq, dim]
    return o[s["has"]].to(s["q"].dtype)


def run(state):
    s = state
    if not own:
        return {"linear": _plain_linear, "append": _plain_append, "attend": _plain_attend}[s["kind"]](s)
    packed_linear, _ = _package()
    if s["kind"] == "linear":
        return packed_linear.packed_linear(s["x"], s["words"], s["scale"], s["zero"], qmin=s["qmin"], qmax=s["qmax"],
                                           group=s["case"]["group"] or None, adapters=s["adapters"], index=s["index"])
    if s["kind"] == "append":
        s["cache"].append(s["k"], s["v"], s["table"], s["before"], s["offsets"])
        k, v = s["cache"].read(s["table"], s["lengths"], s["offsets"], tokens=s["tokens"], dtype=torch.float32)
        return {"k": k, "v": v}
    return s["cache"].attend(s["q"], s["table"], s["lengths"], s["offsets"], scale=s["scale"], window=s["window"])


# ------------------------------------------------------------------------------------------------ work and 64 bits

def _visible(case):
    """Sum over the queries of the keys that they see, and over the sequences of the keys that any query sees."""
    pairs = keys = 0
    for t, h in zip(*_sizes(case)):
        lowest = h
        for p in range(max(0, h - t), h):
            first = max(0, p + 1 - case["window"]) if case["window"] else 0
            pairs += p + 1 - first
            lowest = min(lowest, first)
        keys += h - lowest
    return pairs, keys


def work(case):
    size = _BYTES[case["dtype"]]
    if case["kind"] == "linear":
        t, m, n, r = (case[k] for k in ("tokens", "m", "n", "rank"))
        groups = -(-n // case["group"]) if case["group"] else 1
        used = min(t, case["adapters"])
        return {"bytes": m * (-(-n * case["bits"] // 32)) * 4 + m * groups * (8 if case["zero"] else 4)
                + size * (t * n + t * m + used * r * (n + m)) + (4 * t if case["adapters"] else 0),
                "flops": 2 * t * m * n + 2 * t * r * (n + m)}
    new, held = _sizes(case)
    hkv, dim = case["hkv"], case["dim"]
    if case["kind"] == "append":  # read, written in 4 bits with scale and zero, and the held values given
        return {"bytes": 2 * sum(new) * hkv * (dim * size + dim // 2 + 4 + dim * 4), "flops": 8 * sum(new) * hkv * dim}
    pairs, keys = _visible(case)
    return {"bytes": 2 * keys * hkv * (dim // 2 + 4) + 2 * sum(new) * case["hq"] * dim * size,
            "flops": 4 * pairs * case["hq"] * dim}


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


def exact(case, seed):
    if case["kind"] == "linear":
        s = _linear_inputs(case, seed)
        m, n, bits = case["m"], case["n"], case["bits"]
        y = torch.empty(case["tokens"], m, dtype=torch.float64, device=DEV)
        x = s["x"].to(torch.float64)
        step = 1024
        for r0 in range(0, m, step):  # rows of W by bits: code = sum of its bits' weights
            words = s["words"][r0:r0 + step]
            w = torch.zeros(words.size(0), n, dtype=torch.float64, device=DEV)
            for b in range(bits):
                at = torch.arange(n, device=DEV) * bits + b
                w += torch.bitwise_and(torch.bitwise_right_shift(words[:, at // 32], at % 32), 1).to(torch.float64) * 2 ** b
            w += s["qmin"]
            size = case["group"] or n
            for g in range(s["scale"].size(1)):
                part = w[:, g * size:(g + 1) * size]
                if s["zero"] is not None:
                    part -= s["zero"][r0:r0 + step, g:g + 1].to(torch.float64)
                part *= s["scale"][r0:r0 + step, g:g + 1].to(torch.float64)
            y[:, r0:r0 + step] = torch.matmul(x, w.t().contiguous())
        if s["adapters"] is not None:
            for k in range(case["adapters"]):
                rows = torch.nonzero(s["index"] == k).flatten()
                if rows.numel():
                    a, b = (v[k].to(torch.float64) for v in s["adapters"][:2])
                    y[rows] += s["adapters"][2][k].to(torch.float64) * torch.matmul(torch.matmul(x[rows], a.t().contiguous()), b.t().contiguous())
        return y
    new, held = _sizes(case)
    if case["kind"] == "append":
        rows = sum(new)
        return {"k": _exact_values(_kv(case, seed, rows, 30)), "v": _exact_values(_kv(case, seed, rows, 40))}
    rows, group = sum(held), case["hq"] // case["hkv"]
    k, v = _kv(case, seed, rows, 30), _kv(case, seed, rows, 40)
    q = _randn((sum(new), case["hq"], case["dim"]), seed, 50).to(_DTYPES[case["dtype"]]).to(torch.float64)
    out = torch.zeros_like(q)
    q0 = k0 = 0
    for t, h in zip(new, held):
        kk, vv = _exact_values(k[k0:k0 + h]), _exact_values(v[k0:k0 + h])
        place = torch.arange(h - t, h, device=DEV)[:, None]
        keys = torch.arange(h, device=DEV)[None, :]
        hidden = keys > place
        if case["window"]:
            hidden = hidden | (keys <= place - case["window"])
        for head in range(case["hq"]):
            if not h:
                break
            z = torch.matmul(q[q0:q0 + t, head], kk[:, head // group].t().contiguous()) * case["dim"] ** -0.5
            z.masked_fill_(hidden, -math.inf)
            weight = torch.nan_to_num(torch.softmax(z, dim=-1), nan=0.)  # a query before the first token sees none
            out[q0:q0 + t, head] = torch.matmul(weight, vv[:, head // group].contiguous())
        q0, k0 = q0 + t, k0 + h
    return out
