"""What a model asks the GQA backend for beyond the reference, on the CPU: the
op pair is replaced by one that keeps what it is given."""
from types import SimpleNamespace

import pytest
import torch

from auto_infer_amd import ops
from auto_infer_amd.attention import registry
from auto_infer_amd.attention.gqa import GqaHipBackend
from auto_infer_amd.attention.layers import rms_norm, rotate_half

HQ, HKV, D, HIDDEN, T = 4, 2, 64, 32, 5


def model(norm=False, **options):
    gen = torch.Generator().manual_seed(0)
    p = "model.layers.0.self_attn."
    w = {p + "qkv_proj.weight": torch.randn((HQ + 2 * HKV) * D, HIDDEN, generator=gen),
         p + "o_proj.weight": torch.eye(HQ * D)}
    if norm:
        w[p + "q_norm.weight"], w[p + "k_norm.weight"] = torch.rand(D, generator=gen), torch.rand(D, generator=gen)
    return SimpleNamespace(
        ATTENTION_FAMILY="gqa_hip", cfg=SimpleNamespace(head_dim=D, num_layers=1, rms_eps=1e-6), n_q_local=HQ,
        n_kv_local=HKV, device=torch.device("cpu"), dtype=torch.float32, w=w,
        layer_prefix=lambda i: f"model.layers.{i}.", **options)


def run(m, ctx):
    """(q, k, v) that the op pair gets, and the packed projection."""
    backend, _ = registry.build_attention_backend(m, "paged", 2, 16)
    kept = {}
    backend._write_kv = lambda layer, k, v, c: kept.update(k=k, v=v)
    backend._attn = lambda layer, q, k, v, c: kept.update(q=q) or q
    x = torch.randn(T, HIDDEN, generator=torch.Generator().manual_seed(1))
    backend.attention(0, x, ctx)
    qkv = x @ m.w["model.layers.0.self_attn.qkv_proj.weight"].t()
    q, k, v = (t.reshape(T, -1, D) for t in qkv.split((HQ * D, HKV * D, HKV * D), -1))
    return kept, (q, k, v)


@pytest.mark.parametrize("norm", [False, True])
def test_a_model_without_rotary_positions(norm):
    m = model(norm, aia_rope=False, alibi_slopes=torch.ones(HQ))
    kept, (q, k, v) = run(m, SimpleNamespace(cos=None, sin=None))
    if norm:
        q = rms_norm(q, m.w["model.layers.0.self_attn.q_norm.weight"], 1e-6)
        k = rms_norm(k, m.w["model.layers.0.self_attn.k_norm.weight"], 1e-6)
    assert torch.equal(kept["q"], q) and torch.equal(kept["k"], k) and torch.equal(kept["v"], v)


def test_rotary_rows_are_used_where_no_rope_is_given():
    cos, sin = torch.rand(T, 1, D), torch.rand(T, 1, D)
    kept, (q, k, v) = run(model(), SimpleNamespace(cos=cos, sin=sin))
    assert torch.equal(kept["q"], q * cos + rotate_half(q) * sin)
    assert torch.equal(kept["k"], k * cos + rotate_half(k) * sin) and torch.equal(kept["v"], v)


def test_missing_rotary_rows_are_named():
    with pytest.raises(ValueError, match="rope=False"):
        run(model(), SimpleNamespace(cos=None, sin=None))
    with pytest.raises(ValueError, match="rope must be"):
        GqaHipBackend(HQ, HKV, D, 1.0, 1, torch.device("cpu"), torch.float32, rope=True)
    rope = ops.RotaryEmbedding(D, device="cpu")
    assert GqaHipBackend(HQ, HKV, D, 1.0, 1, torch.device("cpu"), torch.float32, rope=rope).rope is rope


@pytest.mark.parametrize("family", ["gqa_hip", "gqa_hip_nz"])
def test_a_query_scale_of_the_models_own(family):
    for options, scale in (({}, D ** -0.5), ({"attn_scale": 144 ** -0.5, "attn_softcap": 50.0}, 144 ** -0.5)):
        m = model(**options)
        m.ATTENTION_FAMILY = family
        backend, _ = registry.build_attention_backend(m, "paged", 2, 16)
        mtp, _ = registry.build_mtp_attention_backend(m, "paged", "mtp.", 2, 16)
        for b in (backend, mtp):
            assert b.scale == scale and b.scores["softcap"] == options.get("attn_softcap", 0.0)
