"""Which kernel a call of attention over the 4-bit cache takes: csrc's make_plan and make_tree_plan said again, so that a test can
say which one it means.  test_tree_paths.py holds it to the library's."""


def cdiv(a, b):
    return -(-a // b)


def plan(tokens, seqs, heads, group, dim, most, window=0, nodes=0):
    """(kernel, floats of its partial results) of a call of `tokens` rows of `seqs` sequences, `heads` kv heads that `group` query heads
    share each, a table with room for `most` tokens; of trees of up to `nodes` nodes, or (0) causal."""
    seqs += not seqs
    columns = tokens * group
    prompt = columns >= 96 * seqs
    ct = 128 if prompt else 16
    nd, slots = cdiv(dim, 64), columns // ct + seqs
    reach = min(most, window + (cdiv(nodes, 32) * 32 or ct)) if window else most
    blocks = reach // 32 + 2
    if nodes:
        wide = max(cdiv(columns, 32), seqs)
        total = blocks * wide * heads
        if columns < (256 if nd <= 2 else 384) * seqs or total < 16384 if prompt else total >= (4096 if seqs > 64 else 1024):
            cols = 16 if columns <= 16 * seqs else 32
            tiles, chunks = columns // cols + seqs, 3 * 1024 // heads + 1
            listed = 4 * (1 + 2 * tiles + chunks) if seqs > 64 else 0
            parts = (4 * chunks + 2) // 3 if blocks > 5 else 0
            return f"shared {cols}", listed + parts * heads * cols * (64 * nd + 2)
    tiles = max(cdiv(columns, ct), seqs)
    want = cdiv(blocks * tiles * heads, 768)
    if prompt:
        chunk = blocks if slots * heads >= 256 else max(want, 16)
    else:
        chunk = max(want, 4 if reach > 256 and cdiv(blocks, 4) * tiles * heads < 256 else 8)
    chunks = max(cdiv(blocks, chunk), 1)
    return "prompt" if prompt else "attend", slots * heads * chunks * ct * (64 * nd + 2) if chunks > 1 else 0
