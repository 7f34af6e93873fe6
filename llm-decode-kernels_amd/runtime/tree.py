"""Drafted token trees of speculative decoding, as the tree kernels read them (no counterpart in the reference, which
decodes one token per step). Node 0 is the pending token, node i + 1 the i-th drafted token; a node's parent has a lower
number."""
import torch

MAX_NODES = 1024


def tree_layout(parents):
    """parents[i] in 0 .. i: the node that drafted token i (node i + 1) follows -> (parents int32 [M], depth int32 [M],
    mask int64 [M, ceil(M / 64)]) with node 0 prepended: parent -1, depth 0. Bit j % 64 of mask[i, j // 64] is set for the
    nodes j on the path from node 0 to i, i among them."""
    up = [-1] + [int(p) for p in parents]
    M = len(up)
    if M > MAX_NODES:
        raise ValueError(f"a tree has at most {MAX_NODES} nodes, got {M}")
    words = (M + 63) // 64
    depth, rows = [0] * M, [1] * M
    for i in range(1, M):
        p = up[i]
        if not 0 <= p < i:
            raise ValueError(f"the parent of node {i} must be one of the nodes 0 .. {i - 1}, got {p}")
        depth[i] = depth[p] + 1
        rows[i] = rows[p] | 1 << i
    mask = torch.frombuffer(bytearray(b"".join(r.to_bytes(8 * words, "little") for r in rows)), dtype=torch.int64)
    return torch.tensor(up, dtype=torch.int32), torch.tensor(depth, dtype=torch.int32), mask.view(M, words)
