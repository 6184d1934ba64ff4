"""GPU tests of attention over the 4-bit cache where values' scales are subnormal numbers (spreads below some 1.8e-37), in every
kernel: such values are held as exactly as others, and must neither be lost nor make a sum infinite.

Tolerance: test_kv_cache_gpu's of the largest value, and what subnormal numbers add to it: half a step of the result's own
(2^-150 fp32, 2^-134 bf16), and of the sums, of up to 400 terms that are each rounded by 2^-150 and divided by weights whose
sum is at least 1: 400 2^-150 < 2^-141."""

import pytest
import torch

from test_drafts_gpu import DraftTree, int32
from test_kv_cache_gpu import DEV, OF_VALUES, OWN, Sequences, held_values, starts
from tree_paths import plan

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
HELD, DIM = 400, 64


def near(got, want, biggest, dtype):
    allowed = want.abs() * OWN[dtype] * 1.01 + OF_VALUES[dtype] * biggest + 2. ** -141
    allowed += 2. ** (-134 if dtype is torch.bfloat16 else -150)
    off = (got.cpu().double() - want).abs()
    assert bool((off <= allowed).all()), f"off by {float((off / allowed).max()):.3g} of what is allowed"


# kernel, new tokens, query heads (on two of keys), room of the table in tokens, and whether they are a tree
CALLS = [("attend", 1, 2, 416, False), ("prompt", 110, 8, 416, False), ("attend", 6, 8, 416, True), ("shared 16", 2, 8, 35200, True),
         ("shared 32", 6, 8, 35200, True), ("shared 32", 60, 8, 35200, True), ("prompt", 110, 8, 65600, True)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("where", ["all", "first", "first block of two", "last", "every second", "one"])
@pytest.mark.parametrize("kernel,new,heads,room,tree", CALLS)
def test_subnormal_scales(kernel, new, heads, room, tree, where, dtype):
    dt = TYPES[dtype]
    print(f"subnormal {kernel} {new} x {heads} {where} {dtype}", flush=True)
    assert plan(new, 1, 2, heads // 2, DIM, room, nodes=new if tree else 0)[0] == kernel
    g = torch.Generator().manual_seed(new + heads)
    v = torch.randn(HELD, 2, DIM, generator=g)
    at = torch.arange(HELD)
    small = {"all": at >= 0, "first": at < 100, "first block of two": at // 32 % 2 == 0, "last": at >= 290, "every second": at % 2 == 0,
             "one": at == HELD - new - 1}[where]
    v[small] *= 1e-38
    s = Sequences([HELD], 2, DIM, dt, 32, v=v, seed=new)
    scales = (s.v.float().amax(-1) - s.v.float().amin(-1)) / 15
    assert bool((scales[small] < torch.finfo(torch.float32).tiny).all()) and bool((scales[small] > 0).all())
    q = torch.randn(new, heads, DIM, generator=g).to(dt)
    want, _ = s.reference(q, [new], DIM ** -0.5, None)
    table = torch.cat([s.table, torch.full((1, room // 32 - s.table.size(1)), -7, dtype=torch.int32)], 1).to(DEV)
    chain = DraftTree(int32([i - 1 for i in range(new)]), starts([new]), int32([HELD - new]), nodes=new) if tree else None
    got = s.cache.attend(q.to(DEV), table, s.lengths(), starts([new]), tree=chain)
    near(got, want, float(held_values(s.v).abs().max()), dt)
