"""Trees of drafted tokens on the GPU (csrc/drafts.hip; no reference counterpart: the reference quantizes weights only).

A step that checks drafted tokens gives the model a tree of them for each sequence: node 0 is the token that is certain (the
last one chosen, not in the cache yet), the others are guesses of what follows their parent.  All nodes are appended to the
cache, attended at once, each to what was held before and to the nodes that it comes from, and the model chooses a token
after each.  The nodes that were guessed right, from node 0 on, are accepted.

    tree = DraftTree(parents, rows.offsets, rows.held, nodes=8)
    q, k = rotary(q, k, positions=tree.positions)                     # a node's place is that of its depth
    cache.append(k, v, table, rows.held, rows.offsets)
    out = cache.attend(q, table, lengths, rows.offsets, tree=tree)    # every layer
    accepted = tree.accept(drafted, chosen)
    cache.keep(table, lengths, rows.offsets, accepted.path, accepted.counts)
    pool.resize(rows.held + accepted.counts)                          # accepted.next are the next trees' nodes 0

No call synchronises with the host, and all of them may be captured in a hipGraph.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

import _hip

NODES = 512  # the most that a tree may have


class Accepted(NamedTuple):
    """``path`` [B, nodes] (int32): the accepted nodes' numbers, each a child of the one before, -1 behind them; ``counts`` [B]
    (int32): how many there are; ``next`` [B] (the tokens' type): the token chosen after the last one, -1 without a node."""
    path: torch.Tensor
    counts: torch.Tensor
    next: torch.Tensor


class DraftTree:
    """Trees of the packed rows ``offsets[b]`` to ``offsets[b + 1] - 1`` (int32 [B + 1]) of each sequence, which follow
    ``held[b]`` tokens (int32 [B]).  ``parents`` [tokens] (int32): the number of the earlier node of its sequence that a node
    follows; anything else: none.  ``nodes``: the most that a sequence has, up to 512 (known on the host).

    ``ancestors`` [tokens, ceil(nodes / 32)] (int32): bit j % 32 of word j / 32 is set for the nodes j that a node comes from and
    for itself; ``positions`` [tokens] (int32): held[b] and the nodes before it on its way.  Rows that no sequence has see
    nothing, at position 0; so do nodes past ``nodes`` but for what is held before, at held[b]."""

    def __init__(self, parents: torch.Tensor, offsets: torch.Tensor, held: torch.Tensor, *, nodes: int):
        _hip.require_device(parents)
        self.device, seqs = parents.device, held.numel()
        if not 1 <= nodes <= NODES:
            raise ValueError(f"a tree has 1 to {NODES} nodes, not {nodes}")
        for name, t, shape in (("parents", parents, (parents.numel(),)), ("offsets", offsets, (seqs + 1,)), ("held", held, (seqs,))):
            if t.dtype is not torch.int32 or t.shape != shape or t.device != self.device or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 {list(shape)} on the parents' device")
        self.parents, self.offsets, self.nodes, self.seqs, self.tokens = parents, offsets, nodes, seqs, parents.numel()
        self.ancestors = torch.empty(self.tokens, -(-nodes // 32), dtype=torch.int32, device=self.device)
        self.positions = torch.empty(self.tokens, dtype=torch.int32, device=self.device)
        _hip.launch("draft_tree", self.device, parents.data_ptr(), offsets.data_ptr(), held.data_ptr(), seqs, self.tokens, nodes,
                    self.ancestors.data_ptr(), self.positions.data_ptr())

    def accept(self, drafted: torch.Tensor, chosen: torch.Tensor) -> Accepted:
        """From node 0 of each sequence, each time to the first child whose ``drafted`` token is the one ``chosen`` after its
        parent (both [tokens], int32 or int64)."""
        for name, t in (("drafted", drafted), ("chosen", chosen)):
            if t.dtype not in (torch.int32, torch.int64) or t.dtype is not drafted.dtype or t.shape != (self.tokens,) or \
                    t.device != self.device or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 or int64 [{self.tokens}] on the tree's device, both of one type")
        path = torch.empty(self.seqs, self.nodes, dtype=torch.int32, device=self.device)
        counts = torch.empty(self.seqs, dtype=torch.int32, device=self.device)
        after = torch.empty(self.seqs, dtype=drafted.dtype, device=self.device)
        _hip.launch("draft_accept", self.device, self.parents.data_ptr(), self.offsets.data_ptr(), self.seqs, self.tokens,
                    self.nodes, drafted.data_ptr(), chosen.data_ptr(), drafted.dtype is torch.int64, path.data_ptr(),
                    counts.data_ptr(), after.data_ptr())
        return Accepted(path, counts, after)
