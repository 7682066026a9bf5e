"""Steps of block-sparse attention whose lengths do not describe their tokens."""
from types import SimpleNamespace

import pytest
import torch

from auto_infer_amd import ops
from auto_infer_amd.attention.metadata import step_sparse_plan
from tests import test_gpu_block_sparse as sparse

pytestmark = pytest.mark.gpu
DEV = "cuda"
BS, SELECTED = 16, 3


def step(lens, seed=0):
    """The step on the GPU, its plan and bounds that hold what nobody computed."""
    s = sparse.make(lens, 4, 2, 64, BS, seed=seed, spread=False)
    g = sparse.on_gpu(s)
    return s, g, sparse.make_plan(g, SELECTED), sparse.empty_bounds(s["nb"], 2, 64)


def all_calls(g, plan, bounds, scale):
    ops.summarize_blocks(g["kc"], plan, bounds, scale)
    selected = ops.select_blocks(g["q"], plan, bounds, scale)
    return selected, ops.paged_attention_sparse(g["q"], g["kc"], g["vc"], plan, selected, 0.125)


def test_lengths_that_end_behind_the_step():
    """A plan made again, in place, for requests whose new tokens are more than the
    step's: nothing is left of the plan before, whose last blocks have grown since."""
    s, g, plan, (bounds, scale) = step([(2, 40), (2, 70), (2, 23), (2, 130)])
    all_calls(g, plan, bounds, scale)
    bounds.fill_(55)
    g["cu"].copy_(torch.tensor([0, 3, 6, 9, 12]))
    g["lk"].add_(1)
    plan.replan()
    selected, out = all_calls(g, plan, bounds, scale)
    assert bool((bounds == 55).all()) and bool((selected == -1).all()) and bool(out.isnan().all())
    with pytest.raises(ValueError, match="does not describe"):
        plan.status()
    # and the plan of lengths that do describe it works again
    g["cu"].copy_(torch.tensor([0, 2, 4, 6, 8]))
    g["lk"].sub_(1)
    plan.replan()
    plan.status()
    selected, out = all_calls(g, plan, bounds, scale)
    sparse.check_attention(s, selected.cpu(), out.cpu(), 0.125)


@pytest.mark.parametrize("cu", [[0, 3, 2, 6, 8], [1, 2, 4, 6, 8], [0, 2, 4, 6, 9], [-1, 2, 4, 6, 8], [0, 2, 4, 9, 8]])
@pytest.mark.parametrize("copies", [1, 20])
def test_wrong_lengths(cu, copies):
    """Attention in a few work-groups a row, and (many tokens behind a long context) in
    ranges of the context."""
    lens = [(2, 300), (2, 70), (2, 23), (2, 130)]
    if copies > 1:
        cu = [copies * c for c in cu]
        lens = [(2 * copies, 6000), (2 * copies, 70), (2 * copies, 60), (2 * copies, 130)]
    s = sparse.make(lens, 8, 8, 128, BS, spread=False)
    g = sparse.on_gpu({**s, "cu": torch.tensor(cu, dtype=torch.int32)})
    plan, (bounds, scale) = sparse.make_plan(g, SELECTED), sparse.empty_bounds(s["nb"], 8, 128)
    selected, out = all_calls(g, plan, bounds, scale)
    assert bool((bounds == 77).all()) and bool((selected == -1).all()) and bool(out.isnan().all())
    with pytest.raises(ValueError, match="does not describe"):
        plan.status()


def test_lengths_that_end_before_the_step_leave_zeros():
    s, g, _, (bounds, scale) = step([(2, 40), (3, 70)])
    g["q"] = torch.cat((g["q"], g["q"][:3])).contiguous()
    plan = ops.BlockSparsePlan(g["table"], g["cu"], g["lk"], 8, 4, 2, 64, BS, SELECTED)
    plan.status()
    selected, out = all_calls(g, plan, bounds, scale)
    assert bool((selected[5:] == -1).all()) and bool((out[5:] == 0).all())
    sparse.check_attention(s, selected[:5].cpu(), out[:5].cpu(), 0.125)


def test_context_lengths_are_checked_where_asked(monkeypatch):
    s, g, _, _ = step([(2, 40), (2, 70)])
    ctx = SimpleNamespace(block_table=g["table"], cu_seqlens_q=[2, 4], seqlens_kv=[40, 70], aia_seqlens_kv=g["lk"],
                          aia_cu_seqlens_q=torch.tensor([0, 2, 5], dtype=torch.int32, device=DEV))
    step_sparse_plan(SimpleNamespace(**vars(ctx)), 4, 2, 64, BS, SELECTED, 1, 1)
    monkeypatch.setenv("AIA_CHECK_PLAN", "1")
    with pytest.raises(ValueError, match="does not describe"):
        step_sparse_plan(SimpleNamespace(**vars(ctx)), 4, 2, 64, BS, SELECTED, 1, 1)
    ctx.aia_cu_seqlens_q = g["cu"]
    step_sparse_plan(ctx, 4, 2, 64, BS, SELECTED, 1, 1)
