"""GPU tests of attention with trees (KVCache4.attend with a tree) in the kernel that most of its calls take, csrc/kv_tree.hip's
shared_kernel: the cases of test_kv_cache_gpu where numbers are far apart, no numbers, or nothing, with the mask given as a tree.

A call takes that kernel when it has 1024 blocks of keys or more by its table's width, so tables are widened with entries that
are no page; chains of nodes see what causal attention shows, so Sequences.reference is the definition.

Tolerance: test_kv_cache_gpu's, and for bf16, whose scores and sums of values are good to some 17 bits of their terms, 2^-16 of a
score's terms as a change of its weight."""

import math
import random

import pytest
import torch

from drafts import DraftTree
from test_drafts_gpu import Trees, int32, lines, random_tree
from test_kv_cache_gpu import DEV, OF_VALUES, OWN, TYPES, Sequences, check, held_values, poison, starts

pytestmark = pytest.mark.gpu


def widened(s, blocks=1100):
    """The table of s with room for `blocks` blocks of 32 tokens."""
    width = blocks * 32 // s.page
    none = torch.full((len(s.held), width - s.table.size(1)), -7, dtype=torch.int32)
    return torch.cat([s.table, none], 1).to(DEV)


def chains(new, held, offsets=None, tokens=None):
    """Trees that are chains: node i follows node i - 1."""
    offsets = starts(new) if offsets is None else offsets
    before = int(offsets[0])
    flat = [0] * before + [i - 1 for n in new for i in range(n)]
    flat += [0] * ((len(flat) if tokens is None else tokens) - len(flat))
    return DraftTree(int32(flat), offsets, int32([h - n for h, n in zip(held, new)]), nodes=max([*new, 1]))


def attend(s, q, new, **kw):
    return s.cache.attend(q.to(DEV), widened(s), s.lengths(), starts(new), tree=chains(new, s.held), **kw)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,hkv,group,page", [(128, 2, 4, 64), (64, 1, 8, 32), (80, 3, 4, 96), (256, 1, 2, 32), (33, 2, 1, 32),
                                                (192, 1, 5, 64)])
def test_trees(dtype, dim, hkv, group, page):
    print(f"shared kernel {dtype} dim {dim} heads {hkv} x {group} page {page}", flush=True)
    for before, counts in (([5, 0, 31, 32, 100, 63, 200], [3, 4, 1, 2, 0, 2, 6]), ([70], [1]), ([0, 257, 30], [40, 33, 20]),
                           ([400, 290], [30, 17])):
        s = Trees(before, counts, hkv, dim, TYPES[dtype], page, seed=dim + len(counts), shape="near")
        s.dev_table = widened(s)
        s.check(hkv * group)
        s.check(hkv * group, window=max(64, s.tree.nodes))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_many_short_sequences(dtype):
    """As many tiles as leave each sequence one chunk."""
    rng = random.Random(5)
    counts = [rng.randint(0, 3) for _ in range(400)]
    s = Trees([rng.randint(0, 70) for _ in counts], counts, 8, 64, TYPES[dtype], 32, seed=5)
    s.check(8)
    s.check(32)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("new", [1, 5, 60])
@pytest.mark.parametrize("dim", [64, 128, 200])
def test_queries_of_very_different_size(dim, new, dtype):
    """Heads and tokens whose queries differ by up to 2^42 (2^20 in fp16), in one workgroup's columns: the ordinary ones are as exact
    as they are alone, the large ones give the value of the key that wins where it wins by more than its sums are off."""
    g = torch.Generator().manual_seed(dim + new)
    f16, plain = dtype == "f16", dtype == "bf16"
    k = torch.randn(300, 2, dim, generator=g) * (256. if f16 else 1.)
    s = Sequences([300], 2, dim, TYPES[dtype], 32, k=k, seed=new)
    size = torch.tensor([0., 0., 0., 12., 20.] if f16 else [0., 0., 0., 20., 28., 34., 42.])
    size = size[torch.randint(0, len(size), (new, 8), generator=g)]
    q = (torch.randn(new, 8, dim, generator=g).clamp(-3.9, 3.9) * 2. ** (size - (8 if f16 else 0))[:, :, None]).to(TYPES[dtype])
    scale = dim ** -0.5
    want, _ = s.reference(q, [new], scale, None)
    got = attend(s, q, [new]).cpu()
    most = float(held_values(s.v).abs().max())
    check(got[size == 0], want[size == 0], most, TYPES[dtype])
    keys, looked = held_values(s.k).repeat_interleave(4, 1), 0
    for i, h in (size > 0).nonzero().tolist():
        z = keys[:300 - new + i + 1, h] @ q[i, h].double() * scale
        terms = float((2 * keys[:300 - new + i + 1, h].abs().amax(1) * q[i, h].double().abs().sum() * scale).max())
        margin = max(40., 1e-4 * float(z.abs().max()), 2 * 2. ** -16 * terms if plain else 0.)
        if z.numel() > 1 and float(z.topk(2).values.diff().neg()) > margin:
            check(got[i, h], want[i, h], most, TYPES[dtype])
            looked += 1
    assert looked or new < 60


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("new", [1, 6, 60])
@pytest.mark.parametrize("what", ["zeros", "some zeros", "constants", "constant keys"])
def test_vectors_without_a_spread(what, new, dtype):
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(new)
    k, v = torch.randn(333, 2, 96, generator=g), torch.randn(333, 2, 96, generator=g)
    if what == "zeros":
        v[:, 1] = 0.
    elif what == "some zeros":
        v *= 2. ** -10
        v[::2] = 0.
    elif what == "constants":
        v = (torch.randn(333, 2, 1, generator=g) * 2. ** -10).expand(333, 2, 96).contiguous()
    else:
        k = (torch.randn(333, 2, 1, generator=g) * 2. ** -4).expand(333, 2, 96).contiguous()
    s = Sequences([333], 2, 96, dt, 32, k=k, v=v)
    q = torch.randn(new, 6, 96, generator=g).to(dt)
    want, _ = s.reference(q, [new], 96 ** -0.5, None)
    got = attend(s, q, [new]).cpu()
    for head in range(2):  # each against its own largest value
        check(got[:, 3 * head:3 * head + 3], want[:, 3 * head:3 * head + 3], float(held_values(s.v)[:, head].abs().max()), dt)
    if what == "zeros":
        assert not got[:, 3:].any()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 6, 60])
@pytest.mark.parametrize("what", ["unlikely", "hidden", "falling", "rising"])
def test_values_of_very_different_size(what, new, dim, dtype):
    """Values 2^30 times larger than the others (2^20 in fp16): every query against what its own weights make of the values' sizes."""
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(new + dim)
    up, base = (2. ** 20, 2. ** -8) if dtype == "f16" else (2. ** 30, 1.)
    k, v = torch.randn(400, 2, dim, generator=g), torch.randn(400, 2, dim, generator=g) * base
    q = torch.randn(new, 4, dim, generator=g)
    window = None
    if what == "unlikely":  # a score 100 below the others' middle
        far = torch.arange(400) % 37 == 5
        q[:, :, 0] = dim ** 0.5
        k[far, :, 0] = -100.
        v[far] *= up
    elif what == "hidden":
        window = max(30, new)
        v[400 - new - 25:400 - new - 22] *= up
        v[400 - new // 3 - 1] *= up
    else:
        size = torch.linspace(0, 1, 400) if what == "rising" else torch.linspace(1, 0, 400)
        v *= (up ** size).view(-1, 1, 1)
        k[:, :, 0] = -(up ** size).log().view(-1, 1) * 1.2  # large values get small weights
        q[:, :, 0] = dim ** 0.5
    s = Sequences([400], 2, dim, dt, 32, k=k, v=v)
    q = q.to(dt)
    want, _ = s.reference(q, [new], dim ** -0.5, window)
    got = attend(s, q, [new], window=window).cpu()
    sizes, kv = held_values(s.v).abs().amax(-1), held_values(s.k)
    for i in range(new):
        last = 400 - new + i
        first = max(0, last - window + 1) if window else 0
        keys = kv[first:last + 1].repeat_interleave(2, 1)
        z = torch.einsum("hd,nhd->hn", q[i].double(), keys) * dim ** -0.5
        weight = torch.softmax(z, -1) * sizes[first:last + 1].repeat_interleave(2, 1).t()
        # a weight is off by its score's rounding, up to 100 here in fp32 sums: 100 x 2^-24 x sqrt(dim) x 2 <= 2e-4 of it;
        # bf16: 2^-16 of the terms, at most twice the key's largest element times the query's absolute sum
        of = torch.full_like(z, max(OF_VALUES[dt], 2e-4))
        if dt is torch.bfloat16:
            of = of + 2. ** -16 * 2 * keys.abs().amax(-1).t() * q[i].double().abs().sum(-1, keepdim=True) * dim ** -0.5
        allowed = want[i].abs() * OWN[dt] * 1.01 + torch.finfo(dt).tiny + (of * weight).sum(-1)[:, None]
        if dt is torch.float16:
            allowed = allowed + 2. ** -25  # its subnormal numbers' half step
        off = ((got[i].double() - want[i]).abs() / allowed).max()
        assert bool(off <= 1), f"query {i}: {float(off):.3g} of what is allowed"


@pytest.mark.parametrize("new", [1, 5, 60])
@pytest.mark.parametrize("sign", [-1., 1.])
def test_scores_all_far_from_zero(new, sign):
    """A reference that is far below or above 0 from the first block on, and rises over the keys."""
    g = torch.Generator().manual_seed(new)
    k = torch.randn(500, 1, 64, generator=g)
    k[:, :, 0] = sign * torch.linspace(20, 60, 500).view(-1, 1)
    s = Sequences([500], 1, 64, torch.float32, 32, k=k, seed=3)
    q = torch.randn(new, 2, 64, generator=g)
    q[:, :, 0] = 16.
    want, _ = s.reference(q, [new], 0.125, None)
    got = attend(s, q, [new])
    # scores of up to 120 as fp32 sums: 120 x 2^-24 x 8 x 2 = 1.2e-4 of a weight
    allowed = want.abs() * OWN[torch.float32] * 1.01 + 2e-4 * float(held_values(s.v).abs().max())
    assert bool(((got.cpu().double() - want).abs() <= allowed).all())


@pytest.mark.parametrize("dtype", list(TYPES))
def test_what_is_no_number(dtype):
    """A NaN query, and NaN or infinite keys and values of one node and behind the last token, where others do not look."""
    dt = TYPES[dtype]
    for bad in (math.nan, math.inf):
        g = torch.Generator().manual_seed(9)
        k, v = (torch.randn(122, 2, 64, generator=g) for _ in range(2))
        clean = Trees([50, 40], [20, 12], 2, 64, dt, 32, seed=9, shape="near", k=k.clone(), v=v.clone())
        k[50 + 7], v[50 + 7] = bad, bad
        dirty = Trees([50, 40], [20, 12], 2, 64, dt, 32, seed=9, shape="near", k=k, v=v)
        q = torch.randn(32, 4, 64, generator=g).to(dt)
        a, b = (s.cache.attend(q.to(DEV), widened(s), s.lengths(), s.offsets, tree=s.tree).cpu() for s in (clean, dirty))
        under = torch.tensor([7 in line for line in lines(clean.parents[0])] + [False] * 12)
        assert torch.equal(a[~under], b[~under]) and not bool(b[under].isfinite().any())
        q[3, 1], q[30, 0, 5] = bad, bad
        c = clean.cache.attend(q.to(DEV), widened(clean), clean.lengths(), clean.offsets, tree=clean.tree).cpu()
        mine = torch.zeros(32, 4, dtype=torch.bool)
        mine[3, 1] = mine[30, 0] = True
        assert not bool(c[mine].isfinite().any())
        # the others share a workgroup's exponent, which is that of finite elements: as without them
        assert torch.equal(c[~mine], a[~mine])


@pytest.mark.parametrize("before,after", [(0, 1), (0, 200), (7, 0), (70, 45), (300, 33)])
@pytest.mark.parametrize("new", [[1, 1, 1], [1, 0, 5], [40, 50, 2], [0, 0, 0], []])
def test_rows_that_no_sequence_has(new, before, after):
    held = [100, 3000, 40][:len(new)]
    s = Sequences(held or [40], 2, 80, torch.bfloat16, 32, seed=before + after)
    table, lengths = widened(s)[:len(new)], s.lengths()[:len(new)]
    tokens = before + sum(new) + after
    own = torch.zeros(tokens, dtype=torch.bool)
    own[before:before + sum(new)] = True
    q = torch.randn(tokens, 6, 80, generator=s.g).bfloat16().to(DEV)
    tree = chains(new, held, starts(new) + before, tokens)
    poison((q.shape, q.dtype), (q.shape[:2], torch.float32))
    got, lse = s.cache.attend(q, table, lengths, starts(new) + before, return_lse=True, tree=tree)
    assert not got[~own.to(DEV)].any() and bool((lse[~own.to(DEV)] == -math.inf).all())
    if sum(new):
        want, want_lse = s.reference(q.cpu()[own], new, 80 ** -0.5, None)
        check(got.cpu()[own], want, float(held_values(s.v).abs().max()), torch.bfloat16)
        assert float((lse.cpu()[own].double() - want_lse).abs().max()) < 1e-3


def test_other_trees_in_a_graph():
    """A captured call of 200 rows, replayed with other sequences and trees among them."""
    s = Sequences([90, 300, 65], 2, 64, torch.float16, 32, seed=3)
    q = torch.randn(200, 4, 64, generator=s.g).half().to(DEV)
    lengths, offsets, table = s.lengths(), starts([30, 100, 60]), widened(s)
    parents, held = int32([-1] * 200), int32([0] * 3)

    def run():
        return s.cache.attend(q, table, lengths, offsets, tree=DraftTree(parents, offsets, held, nodes=100))

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    rng = random.Random(3)
    for new in ([30, 100, 60], [1, 1, 1], [0, 90, 0], [60, 0, 65], [0, 0, 0]):
        offsets.copy_(starts(new))
        held.copy_(int32([h - n for h, n in zip([90, 300, 65], new)]))
        trees = [random_tree(n, rng, "near") for n in new]
        flat = [p for t in trees for p in t]
        parents.copy_(int32(flat + [0] * (200 - len(flat))))
        q.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert not out[sum(new):].any()
        assert torch.equal(out, run())


def test_strided_queries_and_outputs_of_two_streams():
    """Queries that are part of a wider projection, and two calls at once on streams of their own."""
    s = Trees([700, 900], [9, 14], 2, 128, torch.bfloat16, 64, seed=11)
    s.dev_table = widened(s)
    wide = torch.randn(23, 3, 12, 128, generator=s.g).bfloat16().to(DEV)
    q = wide[:, 1, 2:10]
    want = s.cache.attend(q.contiguous(), s.dev_table, s.lengths(), s.offsets, tree=s.tree)
    assert torch.equal(s.cache.attend(q, s.dev_table, s.lengths(), s.offsets, tree=s.tree), want)
    lengths, got = s.lengths(), []
    torch.cuda.synchronize()
    for _ in range(2):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got += [s.cache.attend(q, s.dev_table, lengths, s.offsets, tree=s.tree) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def uneven(seqs, long=(0, 0.4, 1)):
    """Lengths of sequences of which few are long, and their nodes: mostly few, none for some."""
    rng = random.Random(seqs)
    before, counts = [rng.randint(0, 40) for _ in range(seqs)], [rng.randint(0, 3) for _ in range(seqs)]
    for i, part in enumerate(long):
        b = round(part * (seqs - 1))
        before[b], counts[b] = 2000 - 300 * i, (40, 5, 1)[i]
    return before, counts


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("seqs", [63, 64, 65, 130, 1030])
def test_few_long_ones_among_many(seqs, dtype):
    """As many sequences as a workgroup looks at, one more, and more than are listed at once; the long ones are cut."""
    print(f"many sequences {seqs} {dtype}", flush=True)
    s = Trees(*uneven(seqs), 2, 64, TYPES[dtype], 32, seed=seqs)
    s.check(8)
    s.check(8, window=64)
    s.check(34)
    s.dev_table = widened(s)
    s.check(2)


@pytest.mark.parametrize("before,after", [(0, 1), (70, 45)])
@pytest.mark.parametrize("seqs", [64, 65, 200])
def test_rows_that_none_of_many_sequences_has(seqs, before, after):
    was, counts = uneven(seqs)
    s = Trees(was, counts, 2, 64, torch.bfloat16, 32, seed=seqs)
    tokens = before + sum(counts) + after
    flat = [0] * before + [p for t in s.parents for p in t] + [0] * after
    offsets = starts(counts) + before
    q = torch.randn(tokens, 8, 64, generator=s.g).bfloat16()
    own = torch.zeros(tokens, dtype=torch.bool)
    own[before:before + sum(counts)] = True
    poison((q.shape, q.dtype), (q.shape[:2], torch.float32))
    got, lse = s.cache.attend(q.to(DEV), s.dev_table, s.lengths(), offsets, return_lse=True,
                              tree=DraftTree(int32(flat), offsets, int32(was), nodes=40))
    got, lse = got.cpu(), lse.cpu()
    assert not got[~own].any() and bool((lse[~own] == -math.inf).all())
    want, want_lse = s.reference(q[own], 64 ** -0.5)
    check(got[own], want, float(held_values(s.v).abs().max()), torch.bfloat16)
    assert float((lse[own].double() - want_lse).abs().max()) < 1e-3


@pytest.mark.parametrize("seqs", [64, 65])
def test_many_sequences_in_a_graph(seqs):
    """Lengths, trees and the sequences that are there change between replays; what is left of a replay is not used by the next."""
    was, counts = uneven(seqs)
    s = Trees(was, counts, 2, 64, torch.float32, 32, seed=seqs)
    tokens = sum(counts)
    q = torch.randn(tokens, 4, 64, generator=s.g).to(DEV)
    lengths, offsets, held, parents = s.lengths(), s.offsets.clone(), int32(was), int32([p for t in s.parents for p in t])

    def run():
        return s.cache.attend(q, s.dev_table, lengths, offsets, tree=DraftTree(parents, offsets, held, nodes=40))

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    rng = random.Random(7)
    for keep in (1., 0.5, 0.02, 0., 1.):
        new = [n if rng.random() < keep else 0 for n in counts]
        now = [h if n else 0 for h, n in zip(was, new)]
        trees = [random_tree(n, rng, "near") for n in new]
        flat = [p for t in trees for p in t]
        parents.copy_(int32(flat + [0] * (tokens - len(flat))))
        offsets.copy_(starts(new))
        held.copy_(int32(now))
        lengths.copy_(int32([h + n for h, n in zip(now, new)]))
        q.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert not out[sum(new):].any()
        assert torch.equal(out, run())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,hkv,group,page", [(128, 2, 4, 64), (64, 1, 8, 32), (80, 3, 4, 96), (256, 1, 4, 32), (33, 2, 5, 32)])
def test_many_columns_of_much_work(dtype, dim, hkv, group, page):
    """From 384 columns a sequence and 16384 blocks of all tiles on: prompt_kernel's, with trees; and windows, rows that no sequence
    has, a sequence without a node."""
    print(f"many columns {dtype} dim {dim} heads {hkv} x {group} page {page}", flush=True)
    for before, counts, shape in (([90, 40], [150, 117], "random"), ([300, 10, 1], [230, 65, 200], "near"),
                                  ([1, 40, 33, 0], [512, 200, 0, 200], "chain")):
        s = Trees(before, counts, hkv, dim, TYPES[dtype], page, seed=dim + len(counts), shape=shape)
        s.dev_table = widened(s, 2208)
        s.check(hkv * group)
        s.check(hkv * group, window=max(64, s.tree.nodes))
