"""GPU tests of an attention block that serves drafted tokens: rotary positions, pages dealt on the GPU, trees, acceptance and
what is kept, run together as a program does, against 64 bits on the CPU.

Tolerance as test_packed_serving_gpu's (fp32): projections are within 2^-20 of their terms' absolute sum, and a rotation adds
2^-21 of what it turns to that; keys and values are those that the cache holds, read back, and are compared with the
quantizer's formula of the projections, where a code may differ by one step."""

import math
import random

import pytest
import torch

from drafts import DraftTree
from kv_cache import KVCache4
from packed_serving import PackedAttention
from page_pool import PagePool
from rotary import Bands, Rotary, rotary_frequencies
from test_drafts_gpu import lines, random_tree, walk
from test_packed_serving_gpu import Block, project

pytestmark = pytest.mark.gpu
DEV = "cuda"


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def turned(x, position, f):
    """x [heads, dim] rotated in 64 bits, halves."""
    t = position * torch.tensor(f, dtype=torch.float64)
    c, s, half = torch.cos(t), torch.sin(t), len(f)
    y = x.clone()
    y[:, :half], y[:, half:2 * half] = x[:, :half] * c - x[:, half:2 * half] * s, x[:, half:2 * half] * c + x[:, :half] * s
    return y


class Served(Block):
    def __init__(self, window=None, pages=40, width=6):
        super().__init__(window=window)
        self.rotary = Rotary(self.dim, rotated=24, scaling=Bands(4., 64))
        self.f = rotary_frequencies(24, scaling=Bands(4., 64))[0]
        self.cache = KVCache4(pages, self.kv, self.dim, page_size=32)
        self.cache.pages.fill_(-1)
        self.pool = PagePool(pages, 4, width, page_size=32)
        self.block = PackedAttention(self.block.q, self.block.k, self.block.v, self.block.out, self.cache, heads=self.heads,
                                     window=window, rotary=self.rotary)

    def held_now(self):
        """Keys and values of every sequence, as the cache holds them."""
        lengths = self.pool.lengths.tolist()
        ends = torch.tensor([0] + lengths).cumsum(0).to(torch.int32)
        k, v = self.cache.read(self.pool.table, self.pool.lengths, ends.to(DEV), tokens=sum(lengths))
        return [(k[a:b].double().cpu(), v[a:b].double().cpu()) for a, b in zip(ends[:-1].tolist(), ends[1:].tolist())]

    def check(self, y, x, seen):
        """Outputs y of rows x; `seen`: of each row its sequence's keys and values, its position, and the places that it sees."""
        q, dq = project(self.w[0], x.double())
        out, slack = torch.zeros(len(x), self.heads * self.dim, dtype=torch.float64), torch.zeros(len(x), self.heads * self.dim, dtype=torch.float64)
        for r, ((k, v), position, places) in enumerate(seen):
            qq = turned(q[r].view(self.heads, self.dim), position, self.f)
            size = q[r].view(self.heads, self.dim).abs().amax(1, keepdim=True)
            dd = 2 * dq[r].view(self.heads, self.dim).amax(1, keepdim=True) + 2.0 ** -20 * size  # a pair's two, and the turn's own
            kk, vv = (t[places].repeat_interleave(self.heads // self.kv, 1) for t in (k, v))
            z = (qq[None] * kk).sum(-1) / math.sqrt(self.dim)
            ds = ((dd[None] * kk.abs()).sum(-1) / math.sqrt(self.dim)).max(0).values
            out[r] = (torch.softmax(z, 0)[:, :, None] * vv).sum(0).flatten()
            slack[r] = ((torch.expm1(2 * ds) + 2.0 ** -17) * vv.abs().amax((0, 2)))[:, None].expand(self.heads, self.dim).flatten()
        want, own = project(self.w[3], out)
        assert bool(((y.double().cpu() - want).abs() <= own + slack @ self.w[3].abs().t() + 2.0 ** -23 * want.abs()).all())

    def check_held(self, held, x, position):
        """That held keys and values [kv, dim] of input x at a position are the quantizer's of its projections."""
        for got, w, turn in ((held[0], self.w[1], True), (held[1], self.w[2], False)):
            mine = (x.double() @ w.t()).view(self.kv, self.dim)
            mine = turned(mine, position, self.f) if turn else mine
            step = (mine.amax(1, keepdim=True) - mine.amin(1, keepdim=True)) / 15
            assert bool(((got - mine).abs() <= 1.6 * step + 2.0 ** -8 * mine.abs().amax(1, keepdim=True)).all())


@pytest.mark.parametrize("window", [None, 40])
def test_prompts_then_trees(window):
    s, rng = Served(window), random.Random(4)
    prompts, tokens = [40, 0, 1, 100], [[], [], [], []]  # inputs of the tokens that each sequence holds
    x = torch.randn(sum(prompts), s.n, generator=s.g)
    rows = s.pool.extend(int32(prompts), tokens=len(x))
    y = s.block(x.to(DEV), s.pool.table, rows.held, rows.offsets)
    assert torch.equal(y, s.block(x.to(DEV), s.pool.table, rows.held, rows.offsets, positions=rows.positions))
    kv = s.held_now()
    s.check(y, x, [(kv[b], i, list(range(max(0, i + 1 - window) if window else 0, i + 1))) for b, n in enumerate(prompts) for i in range(n)])
    for b, part in enumerate(x.split(prompts)):
        tokens[b] += list(part)
    for step in range(4):
        counts = [[7, 1, 30, 5], [1, 12, 3, 33], [0, 2, 9, 4], [6, 6, 6, 6]][step]
        trees = [random_tree(n, rng, "near") for n in counts]
        x = torch.randn(sum(counts), s.n, generator=s.g)
        rows = s.pool.extend(int32(counts), tokens=len(x))
        assert not bool(s.pool.missing.any())
        tree = DraftTree(int32([p for t in trees for p in t]), rows.offsets, rows.held, nodes=33)
        y = s.block(x.to(DEV), s.pool.table, rows.held, rows.offsets, tree=tree)
        kv, seen = s.held_now(), []
        for b, t in enumerate(trees):
            held = len(tokens[b])
            for line in lines(t):
                at = held + len(line) - 1
                seen.append((kv[b], at, list(range(max(0, at + 1 - window) if window else 0, held)) + [held + j for j in line]))
        s.check(y, x, seen)
        drafted = [[rng.randint(0, 1) for _ in t] for t in trees]
        chosen = [[rng.randint(0, 1) for _ in t] for t in trees]
        accepted = tree.accept(int32([d for t in drafted for d in t]), int32([c for t in chosen for c in t]))
        s.cache.keep(s.pool.table, s.pool.lengths, rows.offsets, accepted.path, accepted.counts)
        s.pool.resize(rows.held + accepted.counts)
        for b, part in enumerate(x.split(counts)):
            if counts[b]:
                tokens[b] += [part[j] for j in walk(trees[b], drafted[b], chosen[b])]
        assert s.pool.lengths.tolist() == [len(t) for t in tokens]
        for (k, v), mine in zip(s.held_now(), tokens):
            for i, row in enumerate(mine):
                s.check_held((k[i], v[i]), row, i)
    x = torch.randn(4, s.n, generator=s.g)  # and a step of one token each
    rows = s.pool.extend(int32([1] * 4), tokens=4)
    y = s.block(x.to(DEV), s.pool.table, rows.held)
    kv = s.held_now()
    s.check(y, x, [(kv[b], len(t), list(range(max(0, len(t) + 1 - window) if window else 0, len(t) + 1))) for b, t in enumerate(tokens)])


def test_a_step_in_a_graph():
    """Pages, tree, block, acceptance, keeping and giving back in one graph, replayed; equal to the same steps made eagerly."""
    s, eager = Served(), Served()
    x = torch.randn(50, s.n, generator=s.g).to(DEV)
    for e in (s, eager):
        rows = e.pool.extend(int32([20, 0, 29, 1]), tokens=50)
        e.block(x, e.pool.table, rows.held, rows.offsets)
    counts = int32([5] * 4)
    step, parents = torch.zeros(20, s.n, device=DEV), int32([-1] * 20)
    drafted, chosen = int32([0] * 20), int32([0] * 20)

    def run(e):
        rows = e.pool.extend(counts, tokens=20)
        tree = DraftTree(parents, rows.offsets, rows.held, nodes=5)
        y = e.block(step, e.pool.table, rows.held, rows.offsets, tree=tree)
        accepted = tree.accept(drafted, chosen)
        e.cache.keep(e.pool.table, e.pool.lengths, rows.offsets, accepted.path, accepted.counts)
        e.pool.resize(rows.held + accepted.counts)
        return y, accepted.next

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, after = run(s)
    rng = random.Random(7)
    for turn in range(5):
        step.copy_(torch.randn(20, s.n, generator=s.g))
        parents.copy_(int32([p for _ in range(4) for p in random_tree(5, rng, "near")]))
        drafted.copy_(int32([rng.randint(0, 1) for _ in range(20)]))
        chosen.copy_(int32([rng.randint(0, 1) for _ in range(20)]))
        graph.replay()
        want, want_after = run(eager)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(after, want_after), f"replay {turn}"
        assert torch.equal(s.pool.lengths, eager.pool.lengths) and torch.equal(s.pool.table, eager.pool.table)


def test_refusals():
    s = Served()
    b = s.block
    with pytest.raises(ValueError):
        PackedAttention(b.q, b.k, b.v, b.out, s.cache, heads=s.heads, rotary=Rotary(s.dim + 8))
    plain = PackedAttention(b.q, b.k, b.v, b.out, s.cache, heads=s.heads)
    with pytest.raises(ValueError):
        plain(torch.zeros(4, s.n, device=DEV), s.pool.table, int32([0] * 4), positions=int32([0] * 4))
