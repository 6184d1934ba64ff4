"""What an attention block refuses, it refuses before its cache has the call's tokens; on the CPU, with the launches left out."""

from types import SimpleNamespace

import pytest
import torch

import _hip
from kv_cache import KVCache4
from packed_serving import PackedAttention


@pytest.fixture
def parts(monkeypatch):
    """Layers that give zeros, and a cache of heads of 8 that notes what would be appended."""
    monkeypatch.setattr(_hip, "require_device", lambda t: None)
    cache = KVCache4(4, 2, 8, page_size=32, device="cpu")
    done = []
    monkeypatch.setattr(cache, "append", lambda *a: done.append("append"))
    monkeypatch.setattr(cache, "_call", lambda *a: done.append(a[1]))

    class Layer:
        columns = None

        def __init__(self, rows):
            self.words = torch.zeros(rows, 1)

        def __call__(self, x, adapters=None, index=None):
            return torch.zeros(x.size(0), self.words.size(0))

    return (Layer(32), Layer(16), Layer(16), Layer(32)), cache, done


def tree(tokens=6, seqs=2, nodes=4):
    return SimpleNamespace(tokens=tokens, seqs=seqs, nodes=nodes, device=torch.device("cpu"), positions=torch.zeros(tokens, dtype=torch.int32),
                           ancestors=torch.zeros(tokens, 1, dtype=torch.int32))


@pytest.mark.parametrize("what", ["no offsets", "other tokens", "other sequences", "window", "none of these"])
def test_trees(parts, what):
    layers, cache, done = parts
    block = PackedAttention(*layers, cache, heads=4, window=3 if what == "window" else 40)
    x, table, held = torch.zeros(6, 32), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    offsets = None if what == "no offsets" else torch.tensor([0, 4, 6], dtype=torch.int32)
    if what == "no offsets":
        x = x[:2]
    call = lambda: block(x, table, held, offsets, tree=tree(tokens=7 if what == "other tokens" else len(x),
                                                            seqs=3 if what == "other sequences" else 2))
    if what == "none of these":
        call()
        assert done == ["append", "attend_tree"]
    else:
        with pytest.raises(ValueError):
            call()
        assert done == []


@pytest.mark.parametrize("window", [0, -1, 1 << 30])
def test_windows(parts, window):
    layers, cache, _ = parts
    with pytest.raises(ValueError):
        PackedAttention(*layers, cache, heads=4, window=window)
