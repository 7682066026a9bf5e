"""Prefixes that see themselves in both directions, on the host: which requests
may share blocks, and chunks that end inside a prefix."""
from types import SimpleNamespace

import pytest
import torch

from auto_infer_amd import ops
from auto_infer_amd.attention.metadata import step_plan
from auto_infer_amd.block_allocator import KVCacheManager, prefix_seed


def test_blocks_below_a_prefix_are_shared_with_the_same_prefix_only():
    bs = 4
    m = KVCacheManager(40, bs)
    a = list(range(20))
    blocks = m.allocate(20)
    m.register_prefix(a, blocks, prefix_seed(a, 10))
    same = a[:10] + [77] * 10                 # the prefix, then something else
    other = a[:5] + [88] + a[6:]              # the first block, then another prefix
    assert m.match_prefix(same, prefix_seed(same, 10)) == blocks[:2]
    assert m.match_prefix(a, prefix_seed(a, 10)) == blocks
    assert m.match_prefix(other, prefix_seed(other, 10)) == []
    assert m.match_prefix(a, prefix_seed(a, 12)) == []       # the same tokens, a longer prefix
    assert m.match_prefix(a, prefix_seed(a, 0)) == m.match_prefix(a) == []
    plain = m.allocate(20)
    m.register_prefix(a, plain)               # and causal requests among themselves
    assert m.match_prefix(a) == m.match_prefix(a, prefix_seed(a, 1)) == plain
    assert m.match_prefix(a, prefix_seed(a, 10)) == blocks


def test_a_chunk_that_ends_inside_a_prefix_is_refused():
    ops.check_prefixes([10, 0, 5, -2], [10, 12, 13, 14], [10, 4, 100, 1])
    ops.check_prefixes([50], [0], [10])                      # no rows in this step
    with pytest.raises(ValueError, match="request 1.*first chunk"):
        ops.check_prefixes([0, 30], [4, 24], [4, 20])
    with pytest.raises(ValueError, match="one entry"):
        ops.check_prefixes([0], [4, 24], [4, 20])
    ctx = SimpleNamespace(block_table=torch.zeros(1, 4, dtype=torch.int32), cu_seqlens_q=[20], seqlens_kv=[20],
                          aia_prefix_lens=[30])
    with pytest.raises(ValueError, match="first chunk"):
        step_plan(ctx, 4, 2, 64, 16)
