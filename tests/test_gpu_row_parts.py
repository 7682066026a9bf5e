"""Rows whose keys are cut into parts, with values of very different sizes in them."""
import pytest
import torch

from auto_infer_amd import ops
from tests import test_gpu_block_sparse as sparse
from tests import test_gpu_shared_prefix as shared

pytestmark = pytest.mark.gpu
DEV = "cuda"
# Powers of two that each request's blocks are scaled by, in equal runs of the context.
SIZES = {
    "tiny": [-120], "least": [-127], "tiny_first": [-120, 0], "tiny_last": [0, -122], "apart": [60, -80],
    "apart_last": [-80, 60], "huge": [100], "four": [100, -110, 10, -40], "zeros_and_tiny": [None, -118],
}


def resize(s, sizes):
    """V's blocks scaled, None: to zero (in order of the requests, so shared blocks go by
    the last one)."""
    x = s["vc"].float()
    power = torch.zeros(x.shape[0], dtype=torch.int64)
    zero = torch.zeros(x.shape[0], dtype=torch.bool)
    for r, (_, lk) in enumerate(s["lens"]):
        n = -(-lk // s["bs"])
        for i in range(n):
            e, blk = sizes[i * len(sizes) // n], int(s["table"][r, i])
            power[blk], zero[blk] = e or 0, e is None
    x = torch.ldexp(x, power[:, None, None, None]) * ~zero[:, None, None, None]
    s["vc"] = x.bfloat16()
    s["vx"] = s["vc"].double()
    return s


def check(s, out, scale):
    """Weights and the output are rounded to bf16 (2^-8 relative at most), a part's values
    to fp16: 2^-11 of its largest, which is at most sum p max |v| over the part's keys. The
    float32 sums and exponentials are allowed half of that again.  Values below float32's
    and bf16's normal range (2^-126) may be flushed, a key's and the output's."""
    gq, at = s["hq"] // s["hkv"], 0
    assert bool(torch.isfinite(out).all())
    for r, (lq, lk) in enumerate(s["lens"]):
        blocks = s["table"][r, :-(-lk // s["bs"])].long()
        k, v = (s[c + "x"][blocks].flatten(0, 1)[:lk] for c in "kv")
        hidden = torch.arange(lk)[None] > (lk - lq + torch.arange(lq))[:, None]
        for h in range(s["hkv"]):
            q = s["q"][at:at + lq, h * gq:(h + 1) * gq].double().transpose(0, 1)
            p = torch.softmax((q @ k[:, h].t() * scale).masked_fill(hidden, float("-inf")), -1)
            want, size = (p @ v[:, h]).transpose(0, 1), (p @ v[:, h].abs()).transpose(0, 1)
            most = (p @ v[:, h].abs().amax(-1, keepdim=True)).transpose(0, 1)
            bound = 1.5 * (2.0 ** -8 * (size + want.abs()) + 2.0 ** -11 * most) + 2.0 ** -125
            err = (out[at:at + lq, h * gq:(h + 1) * gq].double() - want).abs()
            assert bool((err <= bound).all()), (r, h, float((err / bound).max()))
        at += lq


@pytest.mark.parametrize("hq,hkv,d,rows", [(16, 8, 128, 9), (14, 2, 64, 3), (32, 1, 128, 40)])
@pytest.mark.parametrize("sizes", sorted(SIZES))
def test_shared_prefixes(sizes, hq, hkv, d, rows):
    s = shared.make([(2048, [(1, 1500 + 7 * i) for i in range(rows)])], hq, hkv, d, 16, seed=rows)
    resize(s, SIZES[sizes])
    out, _ = shared.run(s)
    check(s, out, d ** -0.5)


@pytest.mark.parametrize("hq,hkv,d,lens", [(16, 8, 128, [(1, 4000), (2, 2500)]), (14, 2, 64, [(1, 3000)]),
                                           (16, 8, 128, [(70, 2500)])])
@pytest.mark.parametrize("sizes", sorted(SIZES))
def test_selected_blocks(sizes, hq, hkv, d, lens):
    """All blocks selected: few tokens in parts of their selection, 70 in ranges."""
    s = resize(sparse.make(lens, hq, hkv, d, 16, seed=d, spread=False), SIZES[sizes])
    g = sparse.on_gpu(s)
    n = max(-(-lk // 16) for _, lk in lens)
    selected = torch.full((s["t"], hkv, n), -1, dtype=torch.int32)
    for t, _, pos in sparse.tokens_of(s):
        selected[t, :, :pos // 16 + 1] = torch.arange(pos // 16 + 1)
    out = ops.paged_attention_sparse(g["q"], g["kc"], g["vc"], sparse.make_plan(g, n), selected.to(DEV), d ** -0.5)
    check(s, out.cpu(), d ** -0.5)
