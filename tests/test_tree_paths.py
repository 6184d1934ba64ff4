"""That tree_paths.plan says what the library does: the sizes of its partial results are the library's workspaces."""

import random

import _hip
from tree_paths import plan


def test_the_plan_is_the_library_s():
    lib, rng, seen = _hip.lib(), random.Random(1), set()
    for _ in range(20000):
        seqs = rng.choice([0, 1, rng.randint(1, 80), round(10 ** rng.uniform(0, 3.5))])
        tokens = round(seqs * 10 ** rng.uniform(-0.3, 2.7))
        heads, group, dim = rng.randint(1, 16), rng.choice([1, 2, 3, 4, 8, 16]), rng.randint(1, 256)
        most = 32 * round(10 ** rng.uniform(0, 4))
        nodes = rng.choice([0, rng.randint(1, 512)])
        window = rng.choice([0, rng.randint(max(nodes, 1), max(nodes, 1) + 5000)])
        kernel, floats = plan(tokens, seqs, heads, group, dim, most, window, nodes)
        if nodes:
            size = lib.gptq2d_kv_attend_tree_workspace(tokens, seqs, heads, group, dim, most, window, nodes)
        else:
            size = lib.gptq2d_kv_attend_workspace(tokens, seqs, heads, group, dim, most, window)
        assert size == 4 * floats, (tokens, seqs, heads, group, dim, most, window, nodes, kernel)
        seen.add((kernel, bool(nodes), bool(floats)))
    assert len(seen) == 12, seen
