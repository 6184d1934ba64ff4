"""GPU tests of the attention block over packed layers and the 4-bit cache (packed_serving.py) against 64 bits on the CPU.

Tolerance, from the parts' own: fp32 projections are within 2^-20 of their terms' absolute sum; a score is then off by at
most that times |k| and the scale, a weight by exp of twice that, attention by that times the largest |v| and its own 2^-17 of it
(fp32 results), the output by what the projection's |W| makes of it and 2^-20 of its terms.  Keys and values are those
the cache holds, read back; they are compared with the quantizer's formula of the projections, where a code may differ by
one step."""

import functools
import math

import pytest
import torch

import model_driver as MD
import packed_serving
from kv_cache import KVCache4
from packed_linear import Adapters
from packed_serving import PackedAttention, PackedLayer
import packing
import quantizer_int as QI

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make_layer(m, n, g, group=None):
    scale = 0.02 + 0.02 * torch.rand(m, -(-n // group) if group else 1, generator=g)
    wide = scale.repeat_interleave(group, 1)[:, :n] if group else scale
    flat = torch.randint(-8, 8, (m, n), generator=g).float()
    words = packing.pack_int(flat.to(DEV), torch.ones(m, 1, device=DEV), qmin=-8, qmax=7)
    return PackedLayer(words, scale.to(DEV), None, -8, 7, group), flat.double() * wide.double()


class Block:
    def __init__(self, heads=6, kv=2, dim=40, n=96, seqs=4, width=5, group=32, window=None, seed=0):
        g = self.g = torch.Generator().manual_seed(seed)
        self.heads, self.kv, self.dim, self.n, self.window = heads, kv, dim, n, window
        parts = [make_layer(rows, cols, g, group) for rows, cols in
                 ((heads * dim, n), (kv * dim, n), (kv * dim, n), (n, heads * dim))]
        self.w = [w for _, w in parts]
        self.cache = KVCache4(seqs * width, kv, dim, page_size=32)
        self.block = PackedAttention(*(layer for layer, _ in parts), self.cache, heads=heads, window=window)
        self.table = torch.randperm(seqs * width, generator=g).to(torch.int32).view(seqs, width).to(DEV)

    def adapters(self, count, rank, dtype=torch.float32):
        of = {}
        for name, w in zip(("q", "k", "v", "out"), self.w):
            of[name] = Adapters((torch.randn(count, rank, w.size(1), generator=self.g) * w.size(1) ** -0.5).to(DEV, dtype),
                                (0.3 * torch.randn(count, w.size(0), rank, generator=self.g)).to(DEV, dtype), None)
        return of


def project(w, x, adapters=None, index=None):
    y, slack = x @ w.t(), 2.0 ** -20 * (x.abs() @ w.abs().t())
    if adapters is not None:
        a, b = adapters.a.double().cpu(), adapters.b.double().cpu()
        for t in range(x.size(0)):
            e = int(index[t])
            if e >= 0:
                y[t] += b[e] @ (a[e] @ x[t])
                slack[t] += 2.0 ** -19 * (b[e].abs() @ (a[e].abs() @ x[t].abs()))
    return y, slack


@pytest.mark.parametrize("window", [None, 20])
@pytest.mark.parametrize("with_adapters", [False, True])
def test_prompts_and_decode_steps(with_adapters, window):
    """Ragged prompts (one of them nothing), a second piece of them, then decode steps; each against 64 bits."""
    s = Block(window=window)
    adapters = s.adapters(3, 5) if with_adapters else None
    held = torch.zeros(4, dtype=torch.int32, device=DEV)
    for counts in ([40, 0, 1, 100], [3, 50, 0, 7], None, None):
        new = counts or [1] * 4
        offsets = torch.tensor([0] + new).cumsum(0).to(torch.int32)
        x = torch.randn(sum(new), s.n, generator=s.g)
        index = torch.randint(-1, 3, (sum(new),), generator=s.g).to(torch.int32)
        y = s.block(x.to(DEV), s.table, held, offsets.to(DEV) if counts else None, adapters=adapters, index=index.to(DEV))
        held += torch.tensor(new, dtype=torch.int32, device=DEV)
        total = int(held.sum())
        starts = torch.cat([torch.zeros(1, dtype=torch.int64), held.cpu().cumsum(0)])
        k, v = (t.double().cpu() for t in s.cache.read(s.table, held, starts.to(DEV, torch.int32), tokens=total))
        of = adapters or {}
        q, dq = project(s.w[0], x.double(), of.get("q"), index)
        made = {"k": project(s.w[1], x.double(), of.get("k"), index)[0], "v": project(s.w[2], x.double(), of.get("v"), index)[0]}
        o, do = torch.zeros(sum(new), s.heads * s.dim, dtype=torch.float64), torch.zeros(sum(new), s.heads * s.dim, dtype=torch.float64)
        r = 0
        for b, t in enumerate(new):
            first, h = int(starts[b]), int(held[b])
            for i in range(t):
                p = h - t + i
                for name, all_of in (("k", k), ("v", v)):
                    mine = made[name][r].view(s.kv, s.dim)
                    step = (mine.max(1, keepdim=True).values - mine.min(1, keepdim=True).values) / 15
                    # half a step, a step where it differs, and the 16-bit zero and scale: 2^-8 of min and of 15 steps
                    assert bool(((all_of[first + p] - mine).abs() <= 1.6 * step + 2.0 ** -8 * mine.abs().amax(1, keepdim=True)).all())
                lo = max(0, p - window + 1) if window else 0
                kk = k[first + lo:first + p + 1].repeat_interleave(s.heads // s.kv, 1)
                vv = v[first + lo:first + p + 1].repeat_interleave(s.heads // s.kv, 1)
                qq, dd = q[r].view(s.heads, s.dim), dq[r].view(s.heads, s.dim)
                z = (qq[None] * kk).sum(-1) / math.sqrt(s.dim)  # [keys, heads]
                ds = ((dd[None] * kk.abs()).sum(-1) / math.sqrt(s.dim)).max(0).values
                o[r] = (torch.softmax(z, 0)[:, :, None] * vv).sum(0).flatten()
                do[r] = ((torch.expm1(2 * ds) + 2.0 ** -17) * vv.abs().amax((0, 2)))[:, None].expand(s.heads, s.dim).flatten()
                r += 1
        want, slack = project(s.w[3], o, of.get("out"), index)
        slack = slack + do @ s.w[3].abs().t()
        if with_adapters:
            a, b = of["out"].a.double().cpu().abs(), of["out"].b.double().cpu().abs()
            for t in range(sum(new)):
                if int(index[t]) >= 0:
                    slack[t] += b[int(index[t])] @ (a[int(index[t])] @ do[t])
        assert bool(((y.double().cpu() - want).abs() <= slack + 2.0 ** -23 * want.abs()).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decode_step_in_a_graph(dtype):
    """A captured decode step, replayed while the held tokens grow, equals the eager one."""
    s, eager = Block(seed=3), Block(seed=3)
    of = s.adapters(2, 8, dtype)
    offsets = torch.tensor([0, 30, 31, 95, 100], dtype=torch.int32, device=DEV)
    x = torch.randn(100, s.n, generator=s.g).to(DEV, dtype)
    held = torch.zeros(4, dtype=torch.int32, device=DEV)
    for b in (s, eager):
        b.block(x, b.table, held, offsets)
    held += offsets[1:] - offsets[:-1]
    now, step = held.clone(), torch.zeros(4, s.n, dtype=dtype, device=DEV)
    index = torch.tensor([0, 1, -1, 1], dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.block(step, s.table, now, adapters=of, index=index)  # what it appends is overwritten by the first replay
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s.block(step, s.table, now, adapters=of, index=index)
    for i in range(6):
        new = torch.randn(4, s.n, generator=s.g).to(DEV, dtype)
        step.copy_(new)
        now.copy_(held)
        graph.replay()
        want = eager.block(new, eager.table, held, adapters=of, index=index)
        torch.cuda.synchronize()
        assert torch.equal(out, want), f"replay {i}"
        held += 1


def test_refusals():
    s = Block()
    b = s.block
    with pytest.raises(ValueError):
        PackedAttention(b.q, b.k, b.v, b.out, s.cache, heads=5)
    with pytest.raises(ValueError):
        PackedAttention(b.q, b.q, b.v, b.out, s.cache, heads=6)
    with pytest.raises(ValueError):
        PackedAttention(b.q, b.k, b.v, b.out, s.cache, heads=8)

    class Empty:
        name, words = "layer", None

    with pytest.raises(ValueError):
        PackedLayer.from_result(Empty())


def test_example(capsys):
    """Quantizing a block and serving from it: 4-bit weights are the reference's too, so what is left is the 4-bit cache's
    rounding (a step of range / 15, range about 4.6 sigma of 64 elements: 0.09 sigma a value, and the scores') and bf16's."""
    packed_serving.main()
    said = capsys.readouterr().out
    assert float(said.split("within ")[1].split("%")[0]) < 20.


def affine_spec(weight, qmin, qmax, group=None, zero=False):
    """An affine quantizer with a scale (and zero point) a row or group, its maps of every entry where there are groups."""
    m, n = weight.shape
    size = group or n
    columns = torch.arange(n, device=weight.device) // size
    parts = [weight[:, k:k + size] for k in range(0, n, size)]
    if zero:
        lo = torch.stack([p.amin(1) for p in parts], 1)
        scale = ((torch.stack([p.amax(1) for p in parts], 1) - lo) / (qmax - qmin)).to(torch.bfloat16).to(weight.dtype)
        zp = (qmin - lo / scale).round()
    else:
        scale = (torch.stack([p.abs().amax(1) for p in parts], 1) / ((qmax - qmin) / 2)).to(torch.bfloat16).to(weight.dtype)
        zp = torch.zeros_like(scale)
    s, z = scale[:, columns].contiguous(), zp[:, columns].contiguous()
    return MD.QuantSpec(functools.partial(QI.affine_quantizer_hip, qmin=qmin, qmax=qmax), (s, z),
                        pack_scale=s if group else scale, pack_zero=(z if group else zp) if zero else None, qmin=qmin, qmax=qmax)


@pytest.mark.parametrize("bounds,group,zero", [((-7, 7), None, False), ((0, 15), None, True), ((-128, 127), None, False),
                                               ((-2, 1), None, False), ((0, 15), 32, True), ((-8, 7), 64, False)])
def test_layers_of_other_ranges_and_groups(bounds, group, zero):
    """A layer that quantize_model packs comes through from_result with the range it was packed with, rows or groups."""
    g = torch.Generator().manual_seed(1)
    lin = torch.nn.Linear(160, 96, bias=False).to(DEV)
    x = torch.randn(70, 160, generator=g).to(DEV)
    model = torch.nn.Sequential(lin)
    with MD.HessianCollector(model, output_side=False) as col, torch.no_grad():
        model(x)
    res, = MD.quantize_model(model, col, make_quantizer=lambda w: affine_spec(w, *bounds, group, zero))
    assert (res.qmin, res.qmax) == bounds
    layer = PackedLayer.from_result(res, group=group)
    want, slack = x.double().cpu() @ lin.weight.detach().double().cpu().t(), 0.
    # 2^-20 of the terms, whose codes and zero points are up to a range's width each
    slack = 2.0 ** -20 * 3 * (x.double().abs().cpu() @ (res.scale.double().cpu().expand(96, 160) * (bounds[1] - bounds[0])).t())
    assert bool(((layer(x).double().cpu() - want).abs() <= slack + 2.0 ** -23 * want.abs()).all())
    PackedLayer.from_result(res, qmin=bounds[0], qmax=bounds[1], group=group)
    with pytest.raises(ValueError):  # another range than the codes'
        PackedLayer.from_result(res, qmin=bounds[0] - 1, qmax=bounds[1], group=group)
    if group:
        with pytest.raises(ValueError):  # scales that differ within a row
            PackedLayer.from_result(res)
    res.qmin = res.qmax = None
    with pytest.raises(ValueError):  # no range at all
        PackedLayer.from_result(res, group=group)
    assert PackedLayer.from_result(res, qmin=bounds[0], qmax=bounds[1], group=group).qmax == bounds[1]


def test_inputs_of_another_width_are_refused():
    """Rows of words may be longer than the codes that a product takes: a layer of a quantized model knows its width."""
    lin = torch.nn.Linear(160, 96, bias=False).to(DEV)
    with MD.HessianCollector(torch.nn.Sequential(lin), output_side=False) as col, torch.no_grad():
        lin(torch.randn(40, 160, device=DEV))
    layer = PackedLayer.from_result(MD.quantize_model(None, col)[0])
    assert layer(torch.ones(3, 160, device=DEV)).shape == (3, 96)
    for n in (96, 159, 161):
        with pytest.raises(ValueError):
            layer(torch.ones(3, n, device=DEV))
    s = Block()
    b = s.block
    with pytest.raises(ValueError):
        PackedAttention(b.q, b.k, b.v, layer, s.cache, heads=6)
