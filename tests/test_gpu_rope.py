"""Rotary positions from positions against a float64 restatement (bound derived
in oracle/long_context.py)."""
import pytest
import torch

from auto_infer_amd import ops
from oracle import long_context as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

SCALINGS = {"none": None, "linear": {"type": "linear", "factor": 3.5},
            "yarn": {"type": "yarn", "factor": 32.0, "original_max_position": 32768}}


def run(T, hq, hkv, d, rotary, interleaved, scaling, norm, positions=None, in_place=False, seed=0, pad=0):
    gen = torch.Generator().manual_seed(seed)
    width = (hq + 2 * hkv) * d
    qkv = (torch.randn(T, width + pad, generator=gen) * 3).bfloat16()[:, :width]
    if positions is None:
        positions = torch.randint(0, 1 << 20, (T,), generator=gen)
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=gen)).bfloat16() if norm else None for _ in range(2))
    rope = ops.RotaryEmbedding(d, rotary_dim=rotary, base=1e6, interleaved=interleaved, scaling=scaling,
                               device=DEV)
    buf = qkv.to(DEV) if not pad else torch.empty(T, width + pad, dtype=torch.bfloat16, device=DEV)[:, :width]
    buf.copy_(qkv)
    more = {}
    if not in_place:
        more["out"] = (torch.full((T, hq, d), 7.0, dtype=torch.bfloat16, device=DEV),
                       torch.full((T, hkv, d), 7.0, dtype=torch.bfloat16, device=DEV))
    q, k, v = ops.rope_qk(buf, hq, hkv, positions.to(DEV), rope, None if wq is None else wq.to(DEV),
                          None if wk is None else wk.to(DEV), 1e-6, **more)
    torch.cuda.synchronize()
    if not in_place:
        assert torch.equal(buf.cpu(), qkv)
    assert torch.equal(v.cpu(), qkv[:, (hq + hkv) * d:].reshape(T, hkv, d))
    for got, x, w in ((q, qkv[:, :hq * d].reshape(T, hq, d), wq),
                      (k, qkv[:, hq * d:(hq + hkv) * d].reshape(T, hkv, d), wk)):
        ref, bound = oracle.rope(x, positions, rope.inv_freq, rope.attention_factor, interleaved, w)
        far = (got.cpu().double() - ref).abs()
        assert bool((far <= bound).all()), (far / bound.clamp(min=1e-30)).max().item()
    if in_place:
        assert q.data_ptr() == buf.data_ptr()


@pytest.mark.parametrize("d,rotary", [(128, None), (128, 64), (128, 16), (128, 96), (64, None), (64, 48), (64, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_parts_of_the_head(d, rotary, interleaved, norm):
    run(5, 14, 2, d, rotary, interleaved, None, norm, seed=d)


@pytest.mark.parametrize("scaling", list(SCALINGS))
@pytest.mark.parametrize("T,hq,hkv", [(1, 16, 8), (33, 28, 4), (3, 64, 8), (2, 1, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_scalings_and_heads(scaling, T, hq, hkv, in_place):
    run(T, hq, hkv, 128, None, False, SCALINGS[scaling], in_place, in_place=in_place, seed=T, pad=8 * T)


def test_far_and_negative_positions():
    """Angles stay exact where a float32 product is off by whole turns."""
    pos = torch.tensor([0, 1, -1, 2 ** 24 + 1, -(2 ** 30) - 7, 2 ** 31 + 5])
    run(6, 2, 1, 128, None, False, None, False, positions=pos)
    run(6, 2, 1, 64, None, True, SCALINGS["yarn"], True, positions=pos)


def test_given_frequencies():
    freq = [0.0, 1.0, -0.5, 3.0, 6.5, 1e-9, 2e-3, 0.25]
    rope = ops.RotaryEmbedding(64, rotary_dim=16, inv_freq=freq, attention_factor=0.5, device=DEV)
    gen = torch.Generator().manual_seed(1)
    qkv = torch.randn(4, 4 * 64, generator=gen).bfloat16()
    pos = torch.tensor([0, 7, 100000, 31])
    q, k, _ = ops.rope_qk(qkv.to(DEV), 2, 1, pos.to(DEV), rope)
    ref, bound = oracle.rope(qkv[:, :128].reshape(4, 2, 64), pos, freq, 0.5)
    assert bool(((q.cpu().double() - ref).abs() <= bound).all())


def test_an_empty_step():
    rope = ops.RotaryEmbedding(128, device=DEV)
    qkv = torch.empty(0, 4 * 128, dtype=torch.bfloat16, device=DEV)
    q, k, v = ops.rope_qk(qkv, 2, 1, torch.empty(0, dtype=torch.int64, device=DEV), rope)
    assert q.shape == (0, 2, 128) and k.shape == v.shape == (0, 1, 128)
