"""GPU tests that sums of attention with trees are held in 32 bits for every type, as causal attention's are.

Nodes that begin a sequence and come from none see themselves alone: the logarithm of the softmax's denominator is then one
score, and the output the value that is held.  A query's few large elements must not cost what the others add.

Tolerance, of A1 = scale s sum |q (c - 8)| and A2 = scale |z + 8 s| sum |q|, in 2^-24: products of queries and codes are exact; their sum,
in four matrix instructions at most, each rounded once and once more inside (8), then the scale, its products with s and z + 8 s
and that one's sum (4), two fused sums (2), the constants of base 2 and back (3): 17 A1; a query's own sum is rounded 34 times
more: 51 A2.  The output is rounded once from sums of three roundings, with a weight of 1."""

import pytest
import torch

from test_drafts_gpu import DraftTree, int32
from test_kv_cache_gpu import DEV, OWN, TYPES, Sequences, held_values, starts
from tree_paths import plan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", ["alike", "one large", "some large", "all positive, one large", "every size"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kernel,new,room", [("attend", [3, 2], 64), ("shared 16", [2] * 60, 35200), ("shared 16", [2] * 90, 35200),
                                             ("shared 32", [60, 40], 64), ("prompt", [110, 130], 65600)])
def test_scores_are_held_in_32_bits(kernel, new, room, dim, dtype, what):
    dt, seqs, hkv, group, tokens = TYPES[dtype], len(new), 2, 8 if kernel == "shared 16" else 4, sum(new)
    assert plan(tokens, seqs, hkv, group, dim, room, nodes=max(new))[0] == kernel
    s = Sequences(new, hkv, dim, dt, 32, seed=tokens)
    q = torch.randn(tokens, hkv * group, dim, generator=s.g)
    if what == "one large":
        q[..., 0] *= 200
    elif what == "some large":
        q[..., :4] *= 30
    elif what == "all positive, one large":
        q = q.abs()
        q[..., 0] = 300
    elif what == "every size":
        q = q.sign() * 2. ** (torch.rand(q.shape, generator=s.g) * 12 - 6)
    q = q.bfloat16().to(dt)  # no type rounds them to its operands
    table = torch.full((seqs, room // 32), -7, dtype=torch.int32)
    table[:, :s.table.size(1)] = s.table
    tree = DraftTree(int32([-1] * tokens), starts(new), int32([0] * seqs), nodes=max(new))
    out, lse = s.cache.attend(q.to(DEV), table.to(DEV), s.lengths(), starts(new), tree=tree, return_lse=True)
    kk, vv = (held_values(t).repeat_interleave(group, 1) for t in (s.k, s.v))
    x = s.k.float()
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step, low = ((high - low) / torch.tensor(15.)).bfloat16().double(), low.bfloat16().double()
    codes = ((held_values(s.k) - low) / step).round() - 8
    a1 = ((step * codes.abs()).repeat_interleave(group, 1) * q.double().abs()).sum(-1) * dim ** -0.5
    a2 = (low + 8 * step).abs().repeat_interleave(group, 1)[..., 0] * q.double().abs().sum(-1) * dim ** -0.5
    off = (lse.cpu().double() - (q.double() * kk).sum(-1) * dim ** -0.5).abs()
    print(f"{kernel} {dtype} dim {dim} {what}: {float((off / (a1 + a2)).max() * 2 ** 24):.1f} x 2^-24 of a score's terms", flush=True)
    assert bool((off <= 2. ** -24 * (17 * a1 + 51 * a2)).all())
    held = vv.abs().amax(-1, keepdim=True)
    assert bool(((out.cpu().double() - vv).abs() <= OWN[dt] * 1.01 * vv.abs() + 4 * 2. ** -24 * held).all())
