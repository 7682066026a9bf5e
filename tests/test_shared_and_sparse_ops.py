"""Appending with rotation, shared prefixes and block-sparse attention on the CPU: the
calls that are refused, before any device call, and what the backend allocates."""
import math
from types import SimpleNamespace

import pytest
import torch

from auto_infer_amd import _native, ops
from auto_infer_amd.attention import registry
from auto_infer_amd.attention.gqa import GqaHipBackend
from auto_infer_amd.graph import DecodeGraph

INVALID, UNSUPPORTED, CAPACITY = _native.AIA_ERR_INVALID, _native.AIA_ERR_UNSUPPORTED, _native.AIA_ERR_CAPACITY


def call(name, *args):
    lib = _native.load()
    assert len(args) == len(_native.SIGNATURES[name])
    return getattr(lib, name)(*(t(a) if a is not None else None for a, t in zip(args, _native.SIGNATURES[name])))


def refused(name, good, cases):
    for code, kw, text in cases:
        assert call(name, *{**good, **kw}.values()) == code and text in _native.last_error(), (kw, _native.last_error())


def test_append_arguments():
    good = dict(qkv=16, ts=4096, tokens=4, hq=16, hkv=8, dim=128, pos=16, turns=16, rot=128, factor=1.0, inter=0,
                wq=None, wk=None, eps=1e-6, q=1 << 20, qts=2048, kc=16, vc=16, ks=None, vs=None, slots=16, bs=16,
                num=160, flags=0, stream=None)
    refused("aia_rope_append", good, [
        (INVALID, dict(tokens=-1), "bad sizes"), (INVALID, dict(hq=0), "bad sizes"), (INVALID, dict(bs=0), "bad sizes"),
        (INVALID, dict(num=161), "bad sizes"), (INVALID, dict(num=16 << 27), "bad sizes"),
        (INVALID, dict(hkv=70000), "bad sizes"), (INVALID, dict(flags=2), "flags"),
        (INVALID, dict(wk=16), "norm weights go together"), (INVALID, dict(ks=16), "go together"),
        (INVALID, dict(pos=None), "null"), (INVALID, dict(vc=None), "null"), (INVALID, dict(slots=None), "null"),
        (INVALID, dict(qkv=8), "aligned"), (INVALID, dict(kc=8), "aligned"), (INVALID, dict(wq=8, wk=16), "aligned"),
        (INVALID, dict(ts=4000), "token strides"), (INVALID, dict(qts=2044), "token strides"),
        (INVALID, dict(q=32, qts=4096), "overlaps"), (INVALID, dict(q=16, qts=2048), "overlaps"),
        (UNSUPPORTED, dict(dim=96), "head_dim"), (UNSUPPORTED, dict(rot=120), "rotary_dim"),
        (UNSUPPORTED, dict(ks=16, vs=16, flags=1), "NZ"),
        (UNSUPPORTED, dict(ks=16, vs=16, bs=8200, num=82000), "block_size")])
    assert call("aia_rope_append", *{**good, "tokens": 0}.values()) == 0


STEP = dict(batch=2, tokens=4, hq=16, hkv=8, dim=128)
BAD_STEPS = [(INVALID, dict(batch=-1), "bad sizes"), (INVALID, dict(tokens=-1), "bad sizes"),
             (INVALID, dict(hq=12), "bad sizes"), (INVALID, dict(hkv=0), "bad sizes"), (INVALID, dict(bs=0), "bad sizes"),
             (INVALID, dict(width=0), "bad sizes"), (UNSUPPORTED, dict(dim=96), "head_dim"),
             (UNSUPPORTED, dict(batch=10000), "requests"), (UNSUPPORTED, dict(bs=1 << 20, width=1 << 12), "2^31")]


def test_shared_arguments():
    import ctypes
    out = ctypes.c_int64(0)
    lib = _native.load()
    assert lib.aia_shared_workspace_bytes(2, 4, 16, 8, 128, 16, 8, ctypes.byref(out)) == 0 and out.value > 0
    assert lib.aia_shared_workspace_bytes(2, 4, 16, 8, 128, 16, 8, None) == INVALID
    ws = dict(ws=256, wsb=out.value, stream=None)
    plan = dict(cu=16, lk=16, gid=None, bt=16, bts=8, width=8, bs=16, **STEP, **ws)
    refused("aia_shared_plan", plan, BAD_STEPS + [
        (INVALID, dict(cu=None), "null"), (INVALID, dict(bt=None), "null"), (INVALID, dict(bts=7), "overlap"),
        (INVALID, dict(ws=272), "256-byte"), (INVALID, dict(ws=None), "256-byte"), (CAPACITY, dict(wsb=out.value - 1), "needed")])
    attn = dict(q=16, qts=2048, qhs=128, kc=16, vc=16, ks=None, vs=None, nb=4, cu=16, bt=16, bts=8, width=8, bs=16,
                **STEP, scale=0.1, out=16, ots=2048, ohs=128, **ws)
    refused("aia_paged_attention_shared", attn, BAD_STEPS + [
        (INVALID, dict(scale=0.0), "scale"), (INVALID, dict(scale=math.nan), "scale"), (INVALID, dict(q=None), "null"),
        (INVALID, dict(nb=0), "no blocks"), (INVALID, dict(ks=16), "go together"), (INVALID, dict(q=8), "aligned"),
        (INVALID, dict(qts=2047), "strides"), (INVALID, dict(ots=2047), "strides"), (INVALID, dict(nb=1 << 28), "slots"),
        (CAPACITY, dict(wsb=16), "needed")])
    assert call("aia_paged_attention_shared", *{**attn, "tokens": 0}.values()) == 0


def test_sparse_arguments():
    import ctypes
    out = ctypes.c_int64(0)
    lib = _native.load()
    assert lib.aia_sparse_workspace_bytes(2, 4, 16, 8, 128, 16, 8, 4, ctypes.byref(out)) == 0 and out.value > 0
    assert lib.aia_sparse_workspace_bytes(2, 4, 16, 8, 128, 16, 8, 4, None) == INVALID
    ws = dict(ws=256, wsb=out.value, stream=None)
    bad = BAD_STEPS + [(UNSUPPORTED, dict(sel=0), "selected"), (UNSUPPORTED, dict(sel=1025), "selected"),
                       (UNSUPPORTED, dict(hq=8 * 300), "query heads"), (INVALID, dict(ws=8), "256-byte"),
                       (CAPACITY, dict(wsb=16), "needed")]
    refused("aia_sparse_plan", dict(cu=16, lk=16, bt=16, bts=8, width=8, bs=16, **STEP, sel=4, **ws),
            bad + [(INVALID, dict(lk=None), "null"), (INVALID, dict(bts=4), "overlap")])
    refused("aia_summarize_blocks", dict(kc=16, ks=None, nb=4, bounds=16, bscale=16, bs=16, width=8, **STEP, sel=4, **ws),
            bad + [(INVALID, dict(kc=None), "null"), (INVALID, dict(nb=0), "no blocks"), (INVALID, dict(bounds=8), "aligned")])
    select = dict(q=16, qts=2048, qhs=128, bounds=16, bscale=16, nb=4, bt=16, bts=8, width=8, bs=16, **STEP, sel=4,
                  sink=1, local=1, out=16, ots=32, ohs=4, **ws)
    refused("aia_select_blocks", select, bad + [
        (INVALID, dict(sink=4), "do not fit"), (INVALID, dict(local=0), "do not fit"), (INVALID, dict(sink=-1), "do not fit"),
        (INVALID, dict(q=None), "null"), (INVALID, dict(q=8), "aligned"), (INVALID, dict(qhs=4), "strides")])
    attn = dict(q=16, qts=2048, qhs=128, kc=16, vc=16, ks=None, vs=None, nb=4, bt=16, bts=8, width=8, bs=16, **STEP,
                scale=0.1, s=16, sts=32, shs=4, sel=4, out=16, ots=2048, ohs=128, **ws)
    refused("aia_paged_attention_sparse", attn, bad + [
        (INVALID, dict(scale=-1.0), "scale"), (INVALID, dict(s=None), "null"), (INVALID, dict(vs=16), "go together"),
        (INVALID, dict(out=4), "aligned"), (INVALID, dict(vc=8), "aligned")])
    for name, args in (("aia_select_blocks", select), ("aia_paged_attention_sparse", attn)):
        assert call(name, *{**args, "tokens": 0}.values()) == 0


def test_cpu_tensors_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    for plan in (ops.SharedPrefixPlan, lambda *a: ops.BlockSparsePlan(*a, 4)):
        with pytest.raises(ValueError, match="GPU"):
            plan(torch.zeros(1, 4, dtype=torch.int32), i, i[:1], 1, 4, 2, 64, 16)
    rope = ops.RotaryEmbedding(64, device="cpu")
    c = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        ops.rope_append(torch.zeros(1, 192, dtype=torch.bfloat16), 1, 1, torch.zeros(1, dtype=torch.int64), rope, c, c, i[:1])


def backend(**kw):
    return GqaHipBackend(16, 8, 128, 0.1, 3, torch.device("cpu"), torch.bfloat16, **kw)


def test_backend_caches_with_bounds():
    for kv, n in (("bf16", 4), ("fp8", 6)):
        for cache in backend(kv_dtype=kv, sparse_blocks=8).alloc_kv_caches(10, 32):
            assert len(cache) == n and cache[0].shape == cache[1].shape == (10, 32, 8, 128)
            assert cache[-2].shape == (10, 8, 2, 128) and cache[-2].dtype == torch.int8
            assert cache[-1].shape == (10, 8) and cache[-1].dtype == ops.FP8_KV_SCALE
        assert len(backend(kv_dtype=kv, share_prefixes=True).alloc_kv_caches(10, 32)) == 3


def test_backend_refusals():
    for err, kw in ((ValueError, dict(sparse_blocks=3, sparse_sink=2, sparse_local=2)),
                    (ValueError, dict(sparse_blocks=3, sparse_local=0)),
                    (ValueError, dict(sparse_blocks=8, share_prefixes=True)),
                    (NotImplementedError, dict(sparse_blocks=8, kv_layout="nz")),
                    (NotImplementedError, dict(share_prefixes=True, kv_layout="nz")),
                    (NotImplementedError, dict(share_prefixes=True, softcap=30.0)),
                    (NotImplementedError, dict(sparse_blocks=8, alibi_slopes=torch.ones(16)))):
        with pytest.raises(err):
            backend(**kw)


def test_registry_passes_the_options_on():
    model = SimpleNamespace(
        ATTENTION_FAMILY="gqa_hip", cfg=SimpleNamespace(head_dim=128, num_layers=1, rms_eps=1e-6), n_q_local=16,
        n_kv_local=8, device=torch.device("cpu"), dtype=torch.bfloat16, w={}, layer_prefix=str,
        attn_sparse_blocks=9, attn_sparse_sink=2, attn_sparse_local=3)
    b, caches = registry.build_attention_backend(model, "paged", 2, 16)
    assert b.sparse == (9, 2, 3) and not b.share_prefixes and len(caches[0]) == 4
    del model.attn_sparse_blocks
    model.attn_share_prefixes = True
    b, _ = registry.build_mtp_attention_backend(model, "paged", "p.", 2, 16)
    assert b.sparse is None and b.share_prefixes


def test_decode_graph_refuses_caches_with_bounds():
    for kv in ("bf16", "fp8"):
        with pytest.raises(NotImplementedError, match="bounds"):
            DecodeGraph(None, backend(kv_dtype=kv, sparse_blocks=8).alloc_kv_caches(2, 16), num_q_heads=16, num_kv_heads=8)
    with pytest.raises(NotImplementedError, match="shared"):
        DecodeGraph(None, backend(kv_dtype="fp8").alloc_kv_caches(2, 16), num_q_heads=16, num_kv_heads=8,
                    share_prefixes=True, softcap=3.0)
