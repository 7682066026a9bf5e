"""Requests and rows that see no key: their outputs are zeros and they read no
row or slot of anyone else, whatever lies there."""
import pytest
import torch

from auto_infer_amd import ops, workloads
from oracle import long_context as oracle
from oracle.paged_attn import kv_write, nz_from_nd

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
