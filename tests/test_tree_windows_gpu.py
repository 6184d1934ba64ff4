"""GPU tests of attention with trees and a window, in every kernel that such a call takes: a window bounds the work that the choice of
a kernel goes by, so these are long enough for each, and every test says which one it means.

Tolerance: test_kv_cache_gpu's."""

import math
import random

import pytest
import torch

from test_drafts_gpu import Trees, lines
from test_kv_cache_gpu import DEV, TYPES, check, held_values
from tree_paths import plan

pytestmark = pytest.mark.gpu


def reference(s, q, window):
    """(out, lse) in 64 bits, a sequence at a time, all keys that none of its nodes' windows leaves out."""
    group, scale, r = q.size(1) // s.hkv, s.dim ** -0.5, 0
    kv, vv = held_values(s.k), held_values(s.v)
    out, lse = torch.zeros(q.shape, dtype=torch.float64), torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    for b, (h, n) in enumerate(zip(s.before, s.counts)):
        if not n:
            continue
        ways = lines(s.parents[b])
        seen = torch.zeros(n, h + n, dtype=torch.bool)
        for i, way in enumerate(ways):
            seen[i, max(0, h + len(way) - window):h] = True
            seen[i, [h + j for j in way]] = True
        at = s.starts[b] + torch.arange(h + n)
        for head in range(q.size(1)):
            z = (q[r:r + n, head].double() @ kv[at, head // group].t() * scale).masked_fill(~seen, -math.inf)
            lse[r:r + n, head] = z.logsumexp(-1)
            out[r:r + n, head] = z.softmax(-1) @ vv[at, head // group]
        r += n
    return out, lse


def attend(s, heads, window, kernel, most=None):
    """A windowed call, of a kernel by its plan, against the definition."""
    tokens, seqs = sum(s.counts), len(s.counts)
    room = s.dev_table.size(1) * s.page
    assert plan(tokens, seqs, s.hkv, heads // s.hkv, s.dim, room, window, s.tree.nodes)[0] == kernel
    q = torch.randn(tokens, heads, s.dim, generator=s.g).to(s.dtype)
    out, lse = s.cache.attend(q.to(DEV), s.dev_table, s.lengths(), s.offsets, window=window, return_lse=True, tree=s.tree)
    want, want_lse = reference(s, q, window)
    check(out, want, float(held_values(s.v).abs().max()) if most is None else most, s.dtype)
    assert bool(((lse.cpu().double() - want_lse).abs() <= 3e-5 * (1 + want_lse.abs())).all())


# kernel, tokens held before, nodes, kv heads, query heads of each, page, window
CALLS = [("attend", [3000, 200, 1250], [1, 2, 1], 2, 4, 64, 1200),
         ("shared 16", [3000, 700, 1403], [2, 2, 1], 8, 8, 32, 1400),
         ("shared 16", [5001], [4], 16, 4, 96, 2500),
         ("shared 32", [3000, 700, 1403, 9], [7, 30, 12, 1], 4, 4, 64, 1400),
         ("shared 32", [2600, 40], [90, 70], 2, 4, 32, 2000),
         ("prompt", [6000, 2000], [60, 45], 8, 8, 64, 5300),
         ("prompt", [7000], [200], 4, 4, 32, 6000)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,shape", [(64, "near"), (64, "random"), (64, "chain"), (33, "near"), (128, "near")])
@pytest.mark.parametrize("kernel,before,counts,hkv,group,page,window", CALLS)
def test_windows(kernel, before, counts, hkv, group, page, window, dim, dtype, shape):
    print(f"window {kernel} {before} dim {dim} {dtype} {shape}", flush=True)
    s = Trees(before, counts, hkv, dim, TYPES[dtype], page, seed=dim + len(counts), shape=shape)
    attend(s, hkv * group, window, kernel)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("group,kernel", [(4, "shared 16"), (8, "shared 32")])
@pytest.mark.parametrize("seqs", [64, 65, 130])
def test_few_long_ones_among_many(seqs, group, kernel, dtype):
    """Lengths of which few reach past the window and are cut into chunks, with up to 64 sequences and with a list."""
    print(f"window, many sequences {seqs} {kernel} {dtype}", flush=True)
    rng = random.Random(seqs)
    before, counts = [rng.randint(0, 40) for _ in range(seqs)], [rng.randint(0, 3) for _ in range(seqs)]
    for i, b in enumerate((0, seqs // 2, seqs - 1)):
        before[b], counts[b] = 3000 - 300 * i, (20 if group == 8 else 4, 5, 1)[i]
    if group == 8:  # more than two nodes a sequence, for the kernel of 32 columns
        counts[1] += 2 * seqs + 1 - sum(counts)
    s = Trees(before, counts, 8, 64, TYPES[dtype], 32, seed=seqs, shape="near")
    attend(s, 8 * group, 1800, kernel)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("new,kernel", [(1, "shared 16"), (6, "shared 16"), (30, "shared 32"), (200, "prompt")])
def test_large_values_that_no_node_sees(new, kernel, dtype):
    """Values 2^30 (fp16: 2^20) times the others' just before every window, beside those of its first block: as if they were not there."""
    up = 2. ** 20 if dtype == "f16" else 2. ** 30
    held, window = 5600 if new == 200 else 4600, 5300 if new == 200 else 4100
    g = torch.Generator().manual_seed(new)
    k, v = torch.randn(held + new, 8, 64, generator=g), torch.randn(held + new, 8, 64, generator=g) * (2. ** -8 if dtype == "f16" else 1.)
    most = float(v.abs().max()) * 1.1  # what is held of a value may be a step off
    v[held + 1 - window - 25:held + 1 - window] *= up
    s = Trees([held], [new], 8, 64, TYPES[dtype], 32, seed=new, shape="chain", k=k, v=v)
    attend(s, 16, window, kernel, most)
