"""GPU tests of trees of drafted tokens (drafts.py over csrc/drafts.hip; KVCache4's attend with a tree, over csrc/kv_tree.hip, and
keep) against their definitions on the CPU.

Ancestors, positions, acceptance and what keep leaves in the cache are whole numbers or copies: equal.  Attention's tolerance
is that of test_kv_cache_gpu (the same roundings; the mask changes which terms are summed)."""

import math
import random

import pytest
import torch

import _hip
from drafts import DraftTree
from kv_cache import KVCache4
from test_kv_cache_gpu import DEV, TYPES, Sequences, check, held_values, starts

pytestmark = pytest.mark.gpu


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def random_tree(n, rng, shape):
    """Parents: a chain, a star, random earlier nodes, near ones, several roots."""
    if shape == "chain":
        return [i - 1 for i in range(n)]
    if shape == "star":
        return [-1] + [0] * (n - 1) if n else []
    if shape == "near":
        return [-1 if i == 0 else rng.randint(max(0, i - 4), i - 1) for i in range(n)]
    return [-1 if i == 0 or (shape == "roots" and rng.random() < 0.2) else rng.randint(0, i - 1) for i in range(n)]


SHAPES = ["chain", "star", "near", "random", "roots"]


def lines(parents):
    """Each node's way from itself back to where it begins."""
    out = []
    for i, p in enumerate(parents):
        out.append([i] + (out[p] if 0 <= p < i else []))
    return out


def as_words(line, words):
    bits = [0] * words
    for j in line:
        bits[j // 32] |= 1 << j % 32
    return [b - (1 << 32) if b >= 1 << 31 else b for b in bits]


def walk(parents, drafted, chosen):
    path = [0]
    while True:
        child = next((c for c in range(len(parents)) if parents[c] == path[-1] and c > path[-1] and
                      drafted[c] == chosen[path[-1]]), None)
        if child is None:
            return path
        path.append(child)


@pytest.mark.parametrize("counts,nodes", [([1], 1), ([5, 0, 7, 1], 7), ([31, 32, 33, 64, 65], 65), ([512, 3, 511], 512),
                                          ([0, 0], 4), ([i % 9 for i in range(100)], 40)])
def test_trees_and_acceptance(counts, nodes):
    print(f"trees of {counts[:6]} nodes", flush=True)
    rng = random.Random(sum(counts))
    for turn, shape in enumerate(SHAPES):
        parents = [random_tree(n, rng, shape) for n in counts]
        if turn == 3 and len(counts) > 2:  # what is no earlier node is none
            parents = [[p if rng.random() < 0.9 else rng.choice([-7, i, i + 1, 600]) for i, p in enumerate(t)] for t in parents]
        held = [rng.randint(0, 10 ** 6) for _ in counts]
        flat = [p for t in parents for p in t]
        for before, after in ((0, 0), (3, 2)):  # a padded batch
            offsets = starts(counts) + before
            tree = DraftTree(int32([0] * before + flat + [1] * after), offsets, int32(held), nodes=nodes)
            words = -(-nodes // 32)
            want = [as_words(line, words) for t in parents for line in lines(t)]
            none = [[0] * words]
            assert tree.ancestors.tolist() == none * before + want + none * after
            at = [h + len(line) - 1 for t, h in zip(parents, held) for line in lines(t)]
            assert tree.positions.tolist() == [0] * before + at + [0] * after
            for kind in (torch.int32, torch.int64):
                big = 0 if kind is torch.int32 else 1 << 40
                drafted = [[rng.randint(0, 2) + big for _ in t] for t in parents]
                chosen = [[rng.randint(0, 2) + big for _ in t] for t in parents]
                pad = lambda rows: torch.tensor([0] * before + [v for t in rows for v in t] + [0] * after, dtype=kind, device=DEV)
                got = tree.accept(pad(drafted), pad(chosen))
                ways = [walk(p, d, c) if p else [] for p, d, c in zip(parents, drafted, chosen)]
                assert got.path.tolist() == [w + [-1] * (nodes - len(w)) for w in ways]
                assert got.counts.tolist() == [len(w) for w in ways]
                assert got.next.dtype is kind and got.next.tolist() == [c[w[-1]] if w else -1 for w, c in zip(ways, chosen)]


def test_more_nodes_than_said_stay_within():
    """A sequence with more nodes than `nodes`: those past it see what was held, and are not accepted."""
    tree = DraftTree(int32([-1, 0, 1, 2, 3, -1, 0]), int32([0, 5, 7]), int32([9, 4]), nodes=3)
    assert tree.ancestors.flatten().tolist() == [1, 3, 7, 0, 0, 1, 3] and tree.positions.tolist() == [9, 10, 11, 9, 9, 4, 5]
    got = tree.accept(int32([0] * 7), int32([0] * 7))
    assert got.path.tolist() == [[0, 1, 2], [0, 1, -1]] and got.counts.tolist() == [3, 2]


class Trees(Sequences):
    """Sequences whose last tokens are the nodes of trees."""

    def __init__(self, before, counts, *args, shape="random", nodes=None, **kw):
        super().__init__([h + n for h, n in zip(before, counts)], *args, **kw)
        rng = random.Random(len(counts) + sum(counts))
        self.before, self.counts = before, counts
        self.parents = [random_tree(n, rng, shape) for n in counts]
        self.offsets = starts(counts)
        self.tree = DraftTree(int32([p for t in self.parents for p in t]), self.offsets, int32(before),
                              nodes=nodes or max(max(counts), 1))

    def reference(self, q, scale, window=None):
        kv, vv = held_values(self.k), held_values(self.v)
        group = q.size(1) // self.hkv
        out, lse, r = torch.zeros(q.shape, dtype=torch.float64), torch.full(q.shape[:2], -math.inf, dtype=torch.float64), 0
        for b, (h, n) in enumerate(zip(self.before, self.counts)):
            for line in lines(self.parents[b]):
                first = max(0, h + len(line) - window) if window else 0
                at = self.starts[b] + torch.tensor(list(range(first, h)) + [h + j for j in line])
                kk, vw = (t[at].repeat_interleave(group, 1) for t in (kv, vv))
                z = torch.einsum("hd,nhd->hn", q[r].double(), kk) * scale
                lse[r] = torch.logsumexp(z, -1)
                out[r] = torch.einsum("hn,nhd->hd", torch.softmax(z, -1), vw)
                r += 1
        return out, lse

    def check(self, heads, window=None, scale=None, tree=None):
        q = torch.randn(sum(self.counts), heads, self.dim, generator=self.g).to(self.dtype)
        scale = self.dim ** -0.5 if scale is None else scale
        out, lse = self.cache.attend(q.to(DEV), self.dev_table, self.lengths(), self.offsets, scale=scale, window=window,
                                     return_lse=True, tree=tree or self.tree)
        want, want_lse = self.reference(q, scale, window)
        check(out, want, float(held_values(self.v).abs().max()) if self.v.numel() else 0., self.dtype)
        assert bool(((lse.cpu().double() - want_lse).abs() <= 3e-5 * (1 + want_lse.abs())).all())
        return out


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,hkv,group,page", [(128, 2, 4, 64), (64, 1, 8, 32), (80, 3, 4, 96), (256, 1, 2, 32), (33, 2, 1, 32),
                                                (192, 1, 5, 64)])
def test_attention(dtype, dim, hkv, group, page):
    """Few columns and many, nothing held, blocks that the nodes begin and end inside, sequences without a node."""
    print(f"tree {dtype} dim {dim} heads {hkv} x {group} page {page}", flush=True)
    for before, counts in (([5, 0, 31, 32, 100, 63, 200], [3, 4, 1, 2, 0, 2, 6]), ([70], [1]), ([0, 257, 30], [40, 33, 65]),
                           ([90, 40], [150, 17])):
        s = Trees(before, counts, hkv, dim, TYPES[dtype], page, seed=dim + len(counts))
        s.check(hkv * group)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("window", [None, 64, 1000])
def test_shapes_and_windows(shape, window):
    s = Trees([300, 10, 64, 0], [60, 5, 33, 64], 2, 64, torch.float32, 32, seed=4, shape=shape)
    s.check(8, window)
    s = Trees([150, 20, 90], [7, 3, 1], 2, 64, torch.float32, 32, seed=5, shape=shape)
    s.check(4, window)


@pytest.mark.parametrize("counts", [[3], [20], [60], [4, 9]])
def test_long_ones_are_split(counts):
    s = Trees([7000 + 100 * i for i in range(len(counts))], counts, 1, 128, torch.float16, 64, seed=6)
    s.check(4)
    s.check(4, window=4000)


def test_a_chain_is_causal_attention():
    """A chain's nodes see what the causal mask shows: within twice the tolerance of each other."""
    s = Trees([77, 0, 500], [9, 3, 30], 2, 128, torch.bfloat16, 64, seed=7, shape="chain")
    q = torch.randn(42, 8, 128, generator=s.g).bfloat16().to(DEV)
    a = s.cache.attend(q, s.dev_table, s.lengths(), s.offsets)
    b = s.cache.attend(q, s.dev_table, s.lengths(), s.offsets, tree=s.tree)
    allowed = 2 * (2. ** -8 * a.float().abs() * 1.02 + 2. ** -11 * float(held_values(s.v).abs().max()))
    assert bool(((a.float() - b.float()).abs() <= allowed).all())


def test_two_calls_give_the_same_bits():
    s = Trees([3000, 4100], [16, 30], 2, 128, torch.bfloat16, 64, seed=8)
    q = torch.randn(46, 8, 128, generator=s.g).bfloat16().to(DEV)
    a, b = (s.cache.attend(q, s.dev_table, s.lengths(), s.offsets, tree=s.tree) for _ in range(2))
    assert torch.equal(a, b)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("group", [1, 8])
def test_nodes_that_are_no_numbers_reach_their_own_line_only(bad, group):
    """Keys and values of one node that are no numbers: its descendants and itself are none, the others as without it."""
    before, counts = [50, 40], [20, 12]
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(122, 2, 64, generator=g) for _ in range(2))
    clean = Trees(before, counts, 2, 64, torch.float32, 32, seed=9, shape="near", k=k.clone(), v=v.clone())
    k[50 + 7], v[50 + 7] = bad, bad  # node 7 of the first tree
    dirty = Trees(before, counts, 2, 64, torch.float32, 32, seed=9, shape="near", k=k, v=v)
    q = torch.randn(32, 2 * group, 64, generator=g).to(DEV)
    a, b = (s.cache.attend(q, s.dev_table, s.lengths(), s.offsets, tree=s.tree) for s in (clean, dirty))
    under = torch.tensor([7 in line for line in lines(clean.parents[0])] + [False] * 12)
    assert torch.equal(a.cpu()[~under], b.cpu()[~under])
    assert not bool(b.cpu()[under].isfinite().any())


def test_padded_batches_and_missing_pages():
    """Rows of no sequence are zeros; what a page that is none held is seen by nobody."""
    s = Trees([40, 100], [6, 9], 2, 64, torch.float32, 32, seed=10)
    q = torch.randn(20, 4, 64, generator=s.g)
    offsets = s.offsets + 2
    parents = torch.zeros(20, dtype=torch.int32, device=DEV)
    parents[2:17] = s.tree.parents
    tree = DraftTree(parents, offsets, int32(s.before), nodes=9)
    out, lse = s.cache.attend(q.to(DEV), s.dev_table, s.lengths(), offsets, tree=tree, return_lse=True)
    want, _ = s.reference(q[2:17], 64 ** -0.5)
    check(out[2:17], want, float(held_values(s.v).abs().max()), torch.float32)
    for rows in (slice(0, 2), slice(17, 20)):
        assert not bool(out[rows].any()) and bool((lse[rows] == -math.inf).all())
    table = s.dev_table.clone()
    table[1, 1] = -1  # positions 32 to 63 of the second sequence
    out = s.cache.attend(q[2:17].to(DEV), table, s.lengths(), s.offsets, tree=s.tree)
    kv, vv = held_values(s.k), held_values(s.v)
    for i, line in enumerate(lines(s.parents[1])):
        at = s.starts[1] + torch.tensor(list(range(32)) + list(range(64, 100)) + [100 + j for j in line])
        z = torch.einsum("hd,nhd->hn", q[8 + i].double(), kv[at].repeat_interleave(2, 1)) / 8
        want = torch.einsum("hn,nhd->hd", torch.softmax(z, -1), vv[at].repeat_interleave(2, 1))
        check(out[6 + i], want, float(vv.abs().max()), torch.float32)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,hkv,page", [(128, 2, 32), (64, 1, 64), (80, 3, 96), (256, 1, 32), (192, 2, 64), (1, 2, 32)])
def test_keep(dtype, dim, hkv, page):
    """Accepted nodes over block and page ends; what was held, and the places behind the kept ones, stay."""
    print(f"keep {dtype} dim {dim} heads {hkv} page {page}", flush=True)
    before, counts = [5, 0, 31, 100, 64, 9, 40], [7, 40, 3, 130, 33, 0, 1]
    s = Sequences([h + n for h, n in zip(before, counts)], hkv, dim, TYPES[dtype], page, seed=dim)
    rng = random.Random(dim)
    total = sum(s.held)
    k, v = (t.double() for t in s.cache.read(s.dev_table, s.lengths(), starts(s.held), tokens=total))
    paths = [sorted(rng.sample(range(n), rng.randint(min(n, 1), n))) for n in counts]
    paths[4] = [0, 1, 2, 32]  # the first ones are in their place
    width = max(map(len, paths)) + 2
    path = int32([p + [-1] * (width - len(p)) for p in paths])
    s.cache.keep(s.dev_table, s.lengths(), starts(counts), path, int32([len(p) for p in paths]))
    rows = list(range(total))
    for b, p in enumerate(paths):
        at = s.starts[b] + before[b]
        rows[at:at + len(p)] = [at + j for j in p]
    rows = torch.tensor(rows, device=DEV)
    k2, v2 = (t.double() for t in s.cache.read(s.dev_table, s.lengths(), starts(s.held), tokens=total))
    assert torch.equal(k2, k[rows]) and torch.equal(v2, v[rows])


def test_keep_of_paths_that_are_none():
    """A path ends where it does not ascend among the nodes; counts past the path, below 0, of more nodes than there are."""
    before, counts = [10, 10, 10, 10, 10, 30], [6, 6, 6, 6, 6, 6]
    s = Sequences([16] * 5 + [36], 1, 64, torch.float32, 32, seed=2)
    k, v = s.cache.read(s.dev_table, s.lengths(), starts(s.held), tokens=116)
    path = int32([[2, 3, 3, 5], [1, 5, 6, 7], [-1, 2, 3, 4], [3, 4, 5, -1], [1, 2, 3, 4], [1, 3, 4, 5]])
    s.cache.keep(s.dev_table, s.lengths(), starts(counts), path, int32([4, 4, 4, 9, -2, 4]))
    rows = list(range(116))
    for b, p in enumerate([[2, 3], [1, 5], [], [3, 4, 5], [], [1, 3, 4, 5]]):
        at = s.starts[b] + before[b]
        rows[at:at + len(p)] = [at + j for j in p]
    k2, v2 = s.cache.read(s.dev_table, s.lengths(), starts(s.held), tokens=116)
    assert torch.equal(k2, k[torch.tensor(rows, device=DEV)]) and torch.equal(v2, v[torch.tensor(rows, device=DEV)])
    # pages that are none: nothing moves from there or to there
    table = s.dev_table.clone()
    table[5, 1] = -1
    s.cache.keep(table, s.lengths(), starts(counts), path, int32([0, 0, 0, 0, 0, 4]))
    rows = list(range(116))
    at = s.starts[5] + 30
    rows[at] = at + 1  # positions 30 and 31 are in the first page; node 3's position 33 is not
    k3, v3 = s.cache.read(s.dev_table, s.lengths(), starts(s.held), tokens=116)
    assert torch.equal(k3, k2[torch.tensor(rows, device=DEV)]) and torch.equal(v3, v2[torch.tensor(rows, device=DEV)])


def test_captured():
    """A step of trees in a graph, replayed with other trees, tokens and lengths."""
    before, counts, dim = [20, 45, 0], [5, 8, 2], 64
    width = 4
    cache = KVCache4(12, 2, dim, page_size=32)
    cache.pages.fill_(-1)
    table = torch.randperm(12, generator=torch.Generator().manual_seed(1)).to(DEV, torch.int32).view(3, width)
    g = torch.Generator().manual_seed(3)
    draw = lambda *shape: torch.randn(*shape, generator=g)
    old_k, old_v = draw(65, 2, dim), draw(65, 2, dim)
    held, offsets = int32(before), starts(counts)
    cache.append(old_k.to(DEV), old_v.to(DEV), table, torch.zeros_like(held), starts(before))
    q, k, v = (torch.zeros(15, h, dim, device=DEV) for h in (4, 2, 2))
    parents, drafted, chosen = int32([-1] * 15), int32([0] * 15), int32([0] * 15)
    lengths = held + (offsets[1:] - offsets[:-1])

    def step():
        tree = DraftTree(parents, offsets, held, nodes=8)
        cache.append(k, v, table, held, offsets)
        out = cache.attend(q, table, lengths, offsets, tree=tree)
        accepted = tree.accept(drafted, chosen)
        cache.keep(table, lengths, offsets, accepted.path, accepted.counts)
        return out, accepted

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, accepted = step()
    rng = random.Random(2)
    for _ in range(4):
        trees = [random_tree(n, rng, "near") for n in counts]
        for t, x in ((q, draw(15, 4, dim)), (k, draw(15, 2, dim)), (v, draw(15, 2, dim))):
            t.copy_(x)
        parents.copy_(int32([p for t in trees for p in t]))
        drafted.copy_(int32([rng.randint(0, 1) for _ in range(15)]))
        chosen.copy_(int32([rng.randint(0, 1) for _ in range(15)]))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in cache.read(table, lengths, starts([25, 53, 2]), tokens=80)]
        got = [out.clone(), accepted.path.clone(), accepted.counts.clone(), accepted.next.clone()]
        out_eager, eager = step()
        assert torch.equal(got[0], out_eager) and all(torch.equal(a, b) for a, b in zip(got[1:], eager))
        assert all(torch.equal(a, b) for a, b in zip(kept, cache.read(table, lengths, starts([25, 53, 2]), tokens=80)))


def test_refusals():
    p, o, h = int32([-1, 0, 0]), int32([0, 3]), int32([5])
    for bad in (dict(nodes=0), dict(nodes=513)):
        with pytest.raises(ValueError):
            DraftTree(p, o, h, **bad)
    for args in ((p.long(), o, h), (p, int32([0]), h), (p, o, h.long()), (p.view(1, 3), o, h), (p, o.cpu(), h), (int32([0] * 6)[::2], o, h)):
        with pytest.raises(ValueError):
            DraftTree(*args, nodes=3)
    with pytest.raises(_hip.GPTQ2DError):
        DraftTree(p.cpu(), o.cpu(), h.cpu(), nodes=3)
    tree = DraftTree(p, o, h, nodes=3)
    for d, c in ((p.float(), p.float()), (p, p.long()), (p[:2], p), (p, p[:2]), (p.cpu(), p.cpu())):
        with pytest.raises(ValueError):
            tree.accept(d, c)
    cache = KVCache4(2, 1, 32)
    table, lengths, q = int32([[0]]), int32([8]), torch.zeros(3, 2, 32, device=DEV)
    for kw in (dict(window=2), dict(offsets=None), dict(tree=DraftTree(int32([-1, 0]), int32([0, 2]), h, nodes=2)),
               dict(tree=DraftTree(p, int32([0, 2, 3]), int32([5, 5]), nodes=3))):
        args = dict(offsets=o, tree=tree, window=None) | kw
        with pytest.raises(ValueError):
            cache.attend(q, table, lengths, **args)
    path, counts = int32([[0, 1]]), int32([2])
    for args in ((table, lengths, None, path, counts), (table, lengths, o, path.long(), counts), (table, lengths, o, path[0], counts),
                 (table, lengths, o, path, int32([1, 1])), (table, lengths, o, path, counts.cpu()),
                 (table, lengths.long(), o, path, counts)):
        with pytest.raises(ValueError):
            cache.keep(*args)
