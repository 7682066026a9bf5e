"""8-bit caches, modified scores and rotary positions on the CPU: the oracle's
own checks, the rotary frequencies, and what the entry points refuse before any
device call."""
import ctypes
import math

import pytest
import torch

from auto_infer_amd import _native, ops
from auto_infer_amd.attention.gqa import GqaHipBackend
from oracle import long_context as oracle
from oracle.paged_attn import paged_attention

VP = ctypes.c_void_p


def test_e4m3_rounding_is_torchs():
    gen = torch.Generator().manual_seed(0)
    for scale in (200.0, 1.0, 0.01, 0.001):
        x = (torch.randn(20000, generator=gen) * scale).clamp(-448, 448)
        assert torch.equal(oracle.e4m3(x), x.to(torch.float8_e4m3fn).double())
    ties = torch.tensor([17.0, 19.0, 0.0009765625, 0.0029296875, 232.0, 240.0, 464.0 / 2])
    assert torch.equal(oracle.e4m3(ties), ties.to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("amax,e", [(448.0, 0), (448.1, 1), (224.0, -1), (0.0, -100), (2.0 ** -200, -100),
                                    (1.75 * 2.0 ** 127, 119), (3.3e38, 120)])
def test_needed_exponent(amax, e):
    assert oracle.needed_exp(amax) == e


def test_scales_do_not_depend_on_how_a_block_was_filled():
    """Powers of two: rows appended one by one leave what one write of all of
    them stores, as long as nothing falls below e4m3's normal range."""
    gen = torch.Generator().manual_seed(1)
    rows = torch.randn(16, 2, 8, generator=gen).sign() * (1 + torch.rand(16, 2, 8, generator=gen)) \
        * torch.exp2(torch.randint(0, 5, (16, 1, 1), generator=gen).float())
    rows = rows.bfloat16()
    one = torch.zeros(1, 16, 2, 8, dtype=torch.float64), torch.full((1, 2), -127)
    all_ = torch.zeros(1, 16, 2, 8, dtype=torch.float64), torch.full((1, 2), -127)
    for t in range(16):
        oracle.write_kv_fp8(rows[t:t + 1], *one, [t])
    oracle.write_kv_fp8(rows, *all_, list(range(16)))
    assert torch.equal(one[1], all_[1]) and torch.equal(one[0], all_[0])


def test_scored_attention_without_changes_is_the_oracles():
    gen = torch.Generator().manual_seed(2)
    q = torch.randn(8, 4, 16, generator=gen)
    k, v = torch.randn(7, 4, 2, 16, generator=gen), torch.randn(7, 4, 2, 16, generator=gen)
    bt = torch.tensor([[3, 1, 0, 0, 0], [2, 0, 5, 4, 6]])
    a = paged_attention(q, k, v, bt, [3, 8], [7, 18], 0.25)
    b, _ = oracle.scored_attention(q, k, v, bt, [3, 8], [7, 18], 0.25)
    assert (a - b).abs().max() < 1e-5
    # a prefix of all keys: no mask; a huge cap: none; slopes of zero: none
    full, _ = oracle.scored_attention(q, k, v, bt, [3, 8], [7, 18], 0.25, 1e6, torch.zeros(4), [7, 18])
    for h in range(4):
        kk = k[bt[0]].reshape(-1, 2, 16)[:7, h // 2].double()
        p = torch.softmax(q[:3, h].double() @ kk.t() * 0.25, -1)
        assert (full[:3, h] - p @ v[bt[0]].reshape(-1, 2, 16)[:7, h // 2].double()).abs().max() < 1e-9


def test_rotary_frequencies():
    r = ops.RotaryEmbedding(128, base=10000.0, device="cpu")
    assert r.turns.dtype == torch.int64 and r.turns.shape == (64,)
    for i in (0, 1, 33, 63):
        f = 10000.0 ** (-i / 64)
        turn = (int(r.turns[i]) % (1 << 64)) / 2 ** 64
        assert abs(turn - f / (2 * math.pi)) < 2e-16 and r.inv_freq[i] == pytest.approx(f, rel=1e-15)
    lin = ops.RotaryEmbedding(64, rotary_dim=32, scaling={"type": "linear", "factor": 4.0}, device="cpu")
    assert len(lin.inv_freq) == 16 and lin.inv_freq[3] == pytest.approx(10000.0 ** (-3 / 16) / 4)
    assert lin.attention_factor == 1.0
    yarn = ops.RotaryEmbedding(128, base=1e6, device="cpu",
                               scaling={"type": "yarn", "factor": 8.0, "original_max_position": 4096})
    assert yarn.attention_factor == pytest.approx(0.1 * math.log(8.0) + 1)
    base = [1e6 ** (-i / 64) for i in range(64)]
    turns = [4096 * f / (2 * math.pi) for f in base]
    for f, g, t in zip(yarn.inv_freq, base, turns):
        assert g / 8 * (1 - 1e-12) <= f <= g * (1 + 1e-12)
        if t > 40:
            assert f == pytest.approx(g)
        if t < 0.8:
            assert f == pytest.approx(g / 8)
    given = ops.RotaryEmbedding(64, rotary_dim=16, inv_freq=[0.5] * 8, attention_factor=2.0, device="cpu")
    assert given.inv_freq == [0.5] * 8 and given.attention_factor == 2.0
    far = ops.RotaryEmbedding(64, rotary_dim=16, inv_freq=[-0.5, 100.0] + [0.0] * 6, device="cpu")
    assert int(far.turns[0]) < 0 and int(far.turns[2]) == 0


@pytest.mark.parametrize("err,kw", [
    (NotImplementedError, dict(head_dim=96)), (NotImplementedError, dict(head_dim=64, rotary_dim=24)),
    (NotImplementedError, dict(head_dim=64, rotary_dim=80)), (NotImplementedError, dict(head_dim=64, rotary_dim=0)),
    (ValueError, dict(head_dim=64, base=0.0)), (ValueError, dict(head_dim=64, scaling={"type": "other"})),
    (ValueError, dict(head_dim=64, scaling={"type": "linear", "factor": 0})),
    (ValueError, dict(head_dim=64, scaling={"type": "linear", "factor": 2.0, "more": 1})),
    (ValueError, dict(head_dim=64, scaling={"type": "yarn", "factor": 2.0})),
    (ValueError, dict(head_dim=64, inv_freq=[1.0] * 31)),
    (ValueError, dict(head_dim=64, inv_freq=[float("nan")] * 32)),
    (ValueError, dict(head_dim=64, inv_freq=[1.0] * 32, scaling={"type": "linear", "factor": 2.0}))])
def test_rotary_refusals(err, kw):
    with pytest.raises(err):
        ops.RotaryEmbedding(device="cpu", **kw)


def test_cpu_tensors_are_refused():
    t = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    c = torch.zeros(2, 16, 1, 64, dtype=torch.uint8).view(ops.FP8_KV)
    s = torch.zeros(2, 1, dtype=torch.uint8).view(ops.FP8_KV_SCALE)
    with pytest.raises(ValueError, match="GPU"):
        ops.write_kv_fp8(t, t, c, c, s, s, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        ops.rope_qk(torch.zeros(1, 192, dtype=torch.bfloat16), 1, 1, torch.zeros(1, dtype=torch.int64),
                    ops.RotaryEmbedding(64, device="cpu"))


def call(name, *args):
    lib = _native.load()
    conv = []
    for a, t in zip(args, _native.SIGNATURES[name]):
        conv.append(t(a) if a is not None else None)
    assert len(args) == len(_native.SIGNATURES[name])
    return getattr(lib, name)(*conv)


def test_write_arguments_are_checked_before_any_device_call():
    good = dict(key=16, kts=1024, value=16, vts=1024, kc=16, vc=16, ks=16, vs=16, slots=16, tokens=4, heads=8,
                dim=128, bs=16, num=160, stream=None)

    def rc(**kw):
        return call("aia_kv_write_fp8", *{**good, **kw}.values())
    for kw, text in ((dict(tokens=-1), "bad sizes"), (dict(heads=0), "bad sizes"), (dict(bs=0), "bad sizes"),
                     (dict(num=161), "bad sizes"), (dict(num=16 << 27), "bad sizes"), (dict(key=None), "null"),
                     (dict(ks=None), "null"), (dict(value=None), "all be set"), (dict(vs=None), "all be set"),
                     (dict(kts=1000), "smaller"), (dict(vts=8), "smaller"), (dict(kc=8), "aligned")):
        assert rc(**kw) == _native.AIA_ERR_INVALID and text in _native.last_error(), kw
    for kw, text in ((dict(dim=96), "head_dim"), (dict(bs=8200, num=82000), "block_size"),
                     (dict(heads=70000, kts=70000 * 128, vts=70000 * 128), "heads")):
        assert rc(**kw) == _native.AIA_ERR_UNSUPPORTED and text in _native.last_error(), kw
    assert rc(tokens=0) == 0


def test_rope_arguments_are_checked_before_any_device_call():
    good = dict(qkv=16, ts=4096, tokens=4, hq=16, hkv=8, dim=128, pos=16, turns=16, rot=128, factor=1.0, inter=0,
                wq=None, wk=None, eps=1e-6, q=16, qts=2048, k=16, kts=1024, stream=None)

    def rc(**kw):
        return call("aia_rope_qk", *{**good, **kw}.values())
    for kw, text in ((dict(tokens=-1), "bad sizes"), (dict(hq=0), "bad sizes"), (dict(wq=16), "go together"),
                     (dict(pos=None), "null"), (dict(qkv=8), "aligned"), (dict(ts=3000), "token strides"),
                     (dict(qts=2049), "token strides"), (dict(kts=512), "token strides")):
        assert rc(**kw) == _native.AIA_ERR_INVALID and text in _native.last_error(), kw
    for kw, text in ((dict(dim=96), "head_dim"), (dict(rot=120), "rotary_dim"), (dict(rot=144), "rotary_dim"),
                     (dict(rot=0), "rotary_dim")):
        assert rc(**kw) == _native.AIA_ERR_UNSUPPORTED and text in _native.last_error(), kw
    assert rc(tokens=0) == 0


def test_scored_attention_arguments_are_checked_before_any_device_call():
    good = dict(q=16, qts=2048, qhs=128, kc=16, vc=16, bt=16, bts=16, cu=16, kv=16, batch=1, tokens=1, hq=16, hkv=8,
                dim=128, bs=16, nb=4, scale=0.1, out=16, ots=2048, ohs=128, kn=None, vn=None, knts=0, vnts=0,
                ks=16, vs=16, prefix=None, slopes=None, cap=0.0, waves=0, flags=0, ws=256, wsb=1 << 20, stream=None)

    def rc(**kw):
        return call("aia_paged_attention_gqa_ex", *{**good, **kw}.values())
    for kw, text in ((dict(vs=None), "go together"), (dict(kn=16, vn=16, knts=1024, vnts=1024), "aia_kv_write_fp8"),
                     (dict(cap=-1.0), "softcap"), (dict(cap=math.inf), "softcap"), (dict(cap=math.nan), "softcap"),
                     (dict(scale=0.0), "scale"), (dict(flags=4), "flags"), (dict(ws=272), "256-byte")):
        assert rc(**kw) == _native.AIA_ERR_INVALID and text in _native.last_error(), kw
    assert rc(flags=1) == _native.AIA_ERR_UNSUPPORTED and "NZ" in _native.last_error()
    assert rc(dim=96) == _native.AIA_ERR_UNSUPPORTED and "head_dim" in _native.last_error()
    assert rc(wsb=16) == _native.AIA_ERR_CAPACITY and "aia_paged_attention_gqa_ex" in _native.last_error()
    assert rc(tokens=0) == 0
    plan = dict(cu=16, kv=16, prefix=16, bt=16, bts=16, bs=16, batch=1, tokens=1, hq=16, hkv=8, dim=128, waves=0,
                ws=256, wsb=16, stream=None)
    assert call("aia_attn_plan_prefix", *{**plan, "prefix": None}.values()) == _native.AIA_ERR_INVALID
    assert "prefix_lens" in _native.last_error()
    assert call("aia_attn_plan_prefix", *{**plan, "dim": 512, "hkv": 1}.values()) == _native.AIA_ERR_UNSUPPORTED
    assert call("aia_attn_plan_prefix", *plan.values()) == _native.AIA_ERR_CAPACITY
    assert "aia_attn_plan_prefix" in _native.last_error()


def test_backend_allocates_8_bit_caches():
    b = GqaHipBackend(16, 8, 128, 0.1, 3, torch.device("cpu"), torch.bfloat16, kv_dtype="fp8")
    caches = b.alloc_kv_caches(10, 32)
    assert len(caches) == 3
    for k, v, ks, vs in caches:
        assert k.shape == v.shape == (10, 32, 8, 128) and k.dtype == torch.float8_e4m3fn
        assert ks.shape == vs.shape == (10, 8) and ks.dtype == torch.float8_e8m0fnu
    with pytest.raises(ValueError, match="kv_dtype"):
        GqaHipBackend(16, 8, 128, 0.1, 3, torch.device("cpu"), torch.bfloat16, kv_dtype="int4")
    with pytest.raises(NotImplementedError, match="NZ"):
        GqaHipBackend(16, 8, 128, 0.1, 3, torch.device("cpu"), torch.bfloat16, kv_dtype="fp8", kv_layout="nz")
