"""Layout of drafted trees on the host: depths and mask words against a walk up the parents."""
import pytest
import torch

import tree_ref as T
from helpers import gen
from runtime.tree import MAX_NODES, tree_layout


@pytest.mark.parametrize("M,branch", ((1, 1), (2, 1), (5, 3), (63, 2), (64, 4), (65, 3), (250, 4), (1024, 5), (1024, 1)))
def test_tree_layout(M, branch):
    parents = T.random_parents(M, branch, gen(M + branch))
    up, depth, mask = tree_layout(parents[1:])
    assert up.dtype == depth.dtype == torch.int32 and mask.dtype == torch.int64
    assert up.tolist() == parents
    rows = T.mask_rows(parents)
    assert mask.shape == (M, (M + 63) // 64)
    bits = mask[:, :, None] >> torch.arange(64) & 1
    want = torch.zeros(M, mask.size(1) * 64, dtype=torch.int64)
    want[:, :M] = rows
    assert torch.equal(bits.reshape(M, -1), want)
    assert depth.tolist() == [int(r.sum()) - 1 for r in rows]


def test_tree_layout_refusals():
    for bad in ((1,), (0, 2), (-1,), (0, 0, 7)):
        with pytest.raises(ValueError, match="parent of node"):
            tree_layout(bad)
    with pytest.raises(ValueError, match="at most"):
        tree_layout([0] * MAX_NODES)
    assert tree_layout(())[0].tolist() == [-1]
