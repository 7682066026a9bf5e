"""Requests and rows that see no key: their outputs are zeros and they read no
row or slot of anyone else, whatever lies there."""
import pytest
import torch

from auto_infer_amd import ops, workloads
from oracle import long_context as oracle
from oracle.paged_attn import kv_write, mla_absorbed_attention, nz_from_nd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAN = float("nan")

# (query lengths, KV lengths, requests without keys)
STEPS = {
    "last": ([1, 2, 3], [40, 5, 0]),
    "middle": ([1, 3, 1, 2], [33, 0, 70, 2]),
    "all": ([1, 1], [0, 0]),
    "prompt": ([150, 160, 1], [150, 0, 90]),
    "decode_last": ([1] * 6, [300, 16, 1, 17, 2, 0]),
}


def make(name, hq, hkv, d, bs, seed=0):
    lqs, lks = STEPS[name]
    step = workloads.make_gqa_step(lqs=lqs, lks=[max(q, k) for q, k in zip(lqs, lks)], num_q_heads=hq,
                                   num_kv_heads=hkv, head_dim=d, block_size=bs, seed=seed, extra_blocks=1)
    step.seqlens_kv = list(lks)
    with_keys = torch.cat([torch.full((q,), k > 0) for q, k in zip(lqs, lks)])
    return step, with_keys


@pytest.mark.parametrize("kv", ["nd", "nz"])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (28, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("name", list(STEPS))
def test_new_rows_behind_the_request_are_not_read(name, hq, hkv, d, cap, kv):
    """With the K/V write in the attention call: the rows behind a request
    without keys (another request's, or memory behind the tensor) hold NaN."""
    bs = 16
    step, with_keys = make(name, hq, hkv, d, bs)
    T = step.num_tokens
    conv = nz_from_nd if kv == "nz" else (lambda x: x)
    dk, dv = conv(step.k_cache).to(DEV), conv(step.v_cache).to(DEV)
    new = []
    for rows in (step.k_new, step.v_new):       # rows of a longer buffer of NaN
        buf = torch.full((T + 200, hkv, d), NAN, dtype=torch.bfloat16, device=DEV)
        buf[:T] = rows.to(DEV)
        new.append(buf[:T])
    kv_write(step.k_new[with_keys], step.v_new[with_keys], step.k_cache, step.v_cache,
             step.slot_mapping[with_keys])
    plan = ops.AttentionPlan.from_lists(step.block_table.to(DEV), step.cu_seqlens_q, step.seqlens_kv, hq, hkv, d, bs)
    out = ops.paged_attention_gqa(step.q.to(DEV), dk, dv, plan, step.scale, key_new=new[0], value_new=new[1],
                                  kv_layout=kv, softcap=cap).cpu().double()
    ref, bound = oracle.scored_attention(step.q, step.k_cache, step.v_cache, step.block_table, step.cu_seqlens_q,
                                         step.seqlens_kv, step.scale, cap)
    assert bool((out[~with_keys] == 0).all())
    assert bool(((out - ref).abs() <= bound).all())
    assert torch.equal(dk.cpu(), conv(step.k_cache)) and torch.equal(dv.cpu(), conv(step.v_cache))


def behind_nan(cache, table):
    """The cache behind a block 0 of NaN, which no request with keys has."""
    return torch.cat([torch.full_like(cache[:1], NAN), cache]), table + 1


@pytest.mark.parametrize("kv", ["nd", "nz", "fp8"])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (28, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("name", list(STEPS))
def test_slots_of_others_stay_out(name, hq, hkv, d, cap, kv):
    """Zeros, whatever the pool's first block holds."""
    bs = 16
    step, with_keys = make(name, hq, hkv, d, bs, seed=1)
    keys, table = behind_nan(step.k_cache, step.block_table)
    values, _ = behind_nan(step.v_cache, table)
    more = {}
    if kv == "fp8":
        dk, dv = keys.to(torch.float8_e4m3fn), values.to(torch.float8_e4m3fn)
        one = torch.full((keys.shape[0], hkv), 127, dtype=torch.uint8, device=DEV).view(ops.FP8_KV_SCALE)
        keys, values = dk.float(), dv.float()
        dk, dv, more = dk.to(DEV), dv.to(DEV), dict(key_scale=one, value_scale=one)
    elif kv == "nz":
        dk, dv, more = nz_from_nd(keys).to(DEV), nz_from_nd(values).to(DEV), dict(kv_layout="nz")
    else:
        dk, dv = keys.to(DEV), values.to(DEV)
    plan = ops.AttentionPlan.from_lists(table.to(DEV), step.cu_seqlens_q, step.seqlens_kv, hq, hkv, d, bs)
    out = ops.paged_attention_gqa(step.q.to(DEV), dk, dv, plan, step.scale, softcap=cap, **more).cpu().double()
    ref, bound = oracle.scored_attention(step.q, keys, values, table, step.cu_seqlens_q, step.seqlens_kv, step.scale,
                                         cap)
    assert bool((out[~with_keys] == 0).all())
    assert bool(((out - ref).abs() <= bound).all())


@pytest.mark.parametrize("kv", ["nd", "nz"])
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (28, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("lq,lk", [(4, 2), (9, 1), (200, 100), (140, 3)])
def test_rows_in_front_of_the_first_key(lq, lk, hq, hkv, d, kv):
    """More query rows than keys: rows that see none give zeros beside rows that
    see a NaN."""
    bs = 16
    step = workloads.make_gqa_step(lqs=[lk, 1], lks=[lk, 30], num_q_heads=hq, num_kv_heads=hkv, head_dim=d,
                                   block_size=bs, seed=2)
    step.v_cache[step.block_table[0, (lk - 1) // bs], (lk - 1) % bs] = NAN
    q = torch.randn(lq + 1, hq, d, generator=torch.Generator().manual_seed(3)).bfloat16()
    conv = nz_from_nd if kv == "nz" else (lambda x: x)
    plan = ops.AttentionPlan.from_lists(step.block_table.to(DEV), [lq, lq + 1], [lk, 30], hq, hkv, d, bs)
    out = ops.paged_attention_gqa(q.to(DEV), conv(step.k_cache).to(DEV), conv(step.v_cache).to(DEV), plan, step.scale,
                                  kv_layout=kv).cpu()
    assert bool((out[:lq - lk] == 0).all())
    assert bool(torch.isnan(out[lq - 1]).all()) and bool(torch.isfinite(out[lq]).all())


@pytest.mark.parametrize("heads", [16, 20])
@pytest.mark.parametrize("name", list(STEPS))
def test_latent_attention(name, heads):
    """Absorbed MLA: zeros, whatever the pool's first block holds."""
    lqs, lks = STEPS[name]
    step = workloads.make_mla_step(lqs=lqs, lks=[max(q, k) for q, k in zip(lqs, lks)], num_heads=heads,
                                   block_size=16, seed=4)
    with_keys = torch.cat([torch.full((q,), k > 0) for q, k in zip(lqs, lks)])
    cache, table = behind_nan(step.cache, step.block_table)
    plan = ops.AttentionPlan.from_lists(table.to(DEV), step.cu_seqlens_q, lks, heads, 1, 512, 16)
    out = ops.paged_attention_mla(step.q_latent.to(DEV), cache.to(DEV), plan, step.scale).float().cpu()
    ref = mla_absorbed_attention(step.q_latent, cache, table, step.cu_seqlens_q, lks, step.scale, 512)
    assert bool((out[~with_keys] == 0).all())
    assert (out - ref)[with_keys].abs().max().item() <= 2e-2 if with_keys.any() else True


@pytest.mark.parametrize("lq,lk", [(4, 2), (200, 100)])
def test_latent_rows_in_front_of_the_first_key(lq, lk):
    heads, bs = 16, 16
    step = workloads.make_mla_step(lqs=[lk, 1], lks=[lk, 30], num_heads=heads, block_size=bs, seed=5)
    step.cache[step.block_table[0, (lk - 1) // bs], (lk - 1) % bs] = NAN
    q = torch.randn(lq + 1, heads, 576, generator=torch.Generator().manual_seed(3)).bfloat16()
    plan = ops.AttentionPlan.from_lists(step.block_table.to(DEV), [lq, lq + 1], [lk, 30], heads, 1, 512, bs)
    out = ops.paged_attention_mla(q.to(DEV), step.cache.to(DEV), plan, step.scale).cpu()
    assert bool((out[:lq - lk] == 0).all())
    assert bool(torch.isnan(out[lq - 1]).all()) and bool(torch.isfinite(out[lq]).all())
