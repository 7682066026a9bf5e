"""Shared-prefix and block-sparse attention repeat themselves bit for bit: planned again,
in another workspace, and whatever that held."""
import pytest
import torch

from auto_infer_amd import ops
from tests import test_gpu_block_sparse as sparse
from tests import test_gpu_shared_prefix as shared

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (14, 2, 64)])
def test_shared_prefixes(hq, hkv, d, fp8):
    s = shared.make([(2048, [(1, 40 + 31 * i) for i in range(30)]), (512, [(3, 70), (100, 130), (2, 900)])], hq, hkv, d, 16, fp8)
    want, plan = shared.run(s)
    for fill in (0, 127, 255):
        space = torch.full_like(plan.workspace, fill)
        for _ in range(3):
            assert torch.equal(shared.run(s, workspace=space)[0], want)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lens", [[(1, 9000), (2, 4000), (1, 30)], [(80, 5000)], [(600, 6000), (3, 50)]])
def test_block_sparse(lens, fp8):
    s = sparse.make(lens, 16, 8, 128, 16, fp8, seed=2)
    g = sparse.on_gpu(s)

    def run(**kw):
        plan = sparse.make_plan(g, 40, 1, 2, **kw)
        bounds, scale = sparse.empty_bounds(s["nb"], 8, 128)
        ops.summarize_blocks(g["kc"], plan, bounds, scale, key_scale=g["ks"])
        selected = ops.select_blocks(g["q"], plan, bounds, scale)
        out = ops.paged_attention_sparse(g["q"], g["kc"], g["vc"], plan, selected, 0.1, key_scale=g["ks"], value_scale=g["vs"])
        return plan, (bounds, scale.view(torch.uint8), selected, out)
    plan, want = run()
    for fill in (0, 127, 255):
        space = torch.full_like(plan.workspace, fill)
        for _ in range(3):
            assert all(map(torch.equal, run(workspace=space)[1], want))
