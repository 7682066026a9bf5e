"""Modified scores and 8-bit caches at the ends of their ranges: rows split over
ranges that hold an infinity, caps past float32's squares."""
import pytest
import torch

from auto_infer_amd import ops, workloads
from oracle import long_context as oracle
from oracle.paged_attn import nz_from_nd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = float("inf")

# (query lengths, KV lengths, query and KV heads, head_dim, key ranges): ranges
# of thousands of keys, ranges of a few, prompt items cut into chunks
CUT = {
    "decode": ([1, 1], [6000, 40], 8, 2, 128, 2),
    "decode_short_ranges": ([1], [6000], 16, 8, 128, 0),
    "verify": ([3], [5000], 14, 2, 64, 2),
    "prompt": ([140], [4000], 8, 1, 128, 0),
    "prompt_d64": ([300], [5000], 14, 2, 64, 0),
}


def cut_step(name, size):
    lqs, lks, hq, hkv, d, waves = CUT[name]
    step = workloads.make_gqa_step(lqs=lqs, lks=lks, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, block_size=16,
                                   seed=7)
    step.q = step.q / 8           # nearly equal weights: the unnormalised sums grow with the keys
    step.v_cache = (step.v_cache.abs() + 0.5) * size
    return step, hq, hkv, d, waves


@pytest.mark.parametrize("kv", ["nd", "nz"])
@pytest.mark.parametrize("mod", [dict(softcap=20.0), dict(slopes=True)])
@pytest.mark.parametrize("size", [40.0, 3000.0, 2.0 ** 30])
@pytest.mark.parametrize("name", list(CUT))
def test_a_split_row_with_an_infinity_keeps_its_other_values(name, size, mod, kv):
    """One dim of one early key is infinite; the other dims' sums over a range
    exceed the partials' type unless they are scaled."""
    step, hq, hkv, d, waves = cut_step(name, size)
    step.v_cache[step.block_table[0, 6], 4, 0, 9] = INF
    slopes = torch.full((hq,), 2.0 ** -14) if mod.get("slopes") else None
    cap = mod.get("softcap", 0.0)
    conv = nz_from_nd if kv == "nz" else (lambda x: x)
    plan = ops.AttentionPlan.from_lists(step.block_table.to(DEV), step.cu_seqlens_q, step.seqlens_kv, hq, hkv, d, 16,
                                        num_waves=waves)
    out = ops.paged_attention_gqa(step.q.to(DEV), conv(step.k_cache).to(DEV), conv(step.v_cache).to(DEV), plan,
                                  step.scale, kv_layout=kv, softcap=cap,
                                  alibi_slopes=None if slopes is None else slopes.to(DEV)).cpu().double()
    ref, bound = oracle.scored_attention(step.q, step.k_cache, step.v_cache, step.block_table, step.cu_seqlens_q,
                                         step.seqlens_kv, step.scale, cap, slopes)
    fine = torch.isfinite(ref)
    assert not bool(fine.all()) and torch.equal(out[~fine], ref[~fine])
    assert bool(((out - ref).abs() <= bound)[fine].all())


@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("name", list(CUT))
def test_a_split_row_with_an_8_bit_value_past_the_range(name, cap):
    """An 8-bit value that stands for 2^128 is infinite as it is read (float32
    ends below it); the row's other dims are what they are."""
    step, hq, hkv, d, waves = cut_step(name, 1.0)
    nb = step.k_cache.shape[0]
    dk, dv = step.k_cache.to(torch.float8_e4m3fn), (step.v_cache * 64).to(torch.float8_e4m3fn)
    ks = torch.full((nb, hkv), 127, dtype=torch.uint8).view(ops.FP8_KV_SCALE)
    vs = torch.full((nb, hkv), 127, dtype=torch.uint8)
    blk = int(step.block_table[0, 6])
    dv[blk, :, 0] = 0.0
    vs[blk, 0] = 127 + 120
    vs = vs.view(ops.FP8_KV_SCALE)
    values = oracle.dequantised(dv, vs)
    dv[blk, 4, 0, 9] = 256.0
    values[blk, 4, 0, 9] = INF
    plan = ops.AttentionPlan.from_lists(step.block_table.to(DEV), step.cu_seqlens_q, step.seqlens_kv, hq, hkv, d, 16,
                                        num_waves=waves)
    out = ops.paged_attention_gqa(step.q.to(DEV), dk.to(DEV), dv.to(DEV), plan, step.scale, key_scale=ks.to(DEV),
                                  value_scale=vs.to(DEV), softcap=cap).cpu().double()
    ref, bound = oracle.scored_attention(step.q, oracle.dequantised(dk, ks), values, step.block_table,
                                         step.cu_seqlens_q, step.seqlens_kv, step.scale, cap)
    fine = torch.isfinite(ref)
    assert not bool(fine.all()) and torch.equal(out[~fine], ref[~fine])
    assert bool(((out - ref).abs() <= bound)[fine].all())

@pytest.mark.parametrize("lqs,lks", [([1, 3], [90, 40]), ([150], [200])])
@pytest.mark.parametrize("size", [1e8, 1e9, 1e10])
@pytest.mark.parametrize("cap", [1e17, 1e18, 1e19, 1e20, 1e30])
def test_scores_whose_squares_overflow_under_huge_caps(cap, size, lqs, lks):
    """Scores are so large that a row is the value of its first key; none of them
    is far past the cap, and all are finite."""
    hq, hkv, d, bs = 4, 2, 128, 16
    step = workloads.make_gqa_step(lqs=lqs, lks=lks, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, block_size=bs,
                                   seed=9)
    q, k = (step.q.float() * size).bfloat16(), (step.k_cache.float() * size / 10).bfloat16()
    plan = ops.AttentionPlan.from_lists(step.block_table.to(DEV), step.cu_seqlens_q, step.seqlens_kv, hq, hkv, d, bs)
    out = ops.paged_attention_gqa(q.to(DEV), k.to(DEV), step.v_cache.to(DEV), plan, step.scale, softcap=cap).cpu()
    assert bool(torch.isfinite(out).all())
    start = checked = 0
    far = 0.0
    for b, end in enumerate(step.cu_seqlens_q):
        kk = k[step.block_table[b].long()].double().reshape(-1, hkv, d)[:lks[b]]
        for h in range(hq):
            far = max(far, (kk[:, h // 2] @ q[start:end, h].double().t()).abs().max().item() * step.scale)
        start = end
    start = 0
    # the cap's error: 2^-18 of a score where all stay below three quarters of the
    # cap, else 2^-21 of the cap; the products' error: 128 sums of 2^-24 each
    cap_error = 2.0 ** -18 * far if far < 0.7 * cap else 2.0 ** -21 * cap + 2.0 ** -18 * far
    for b, end in enumerate(step.cu_seqlens_q):
        j = torch.arange(lks[b])
        blk = step.block_table[b].long()[j // bs]
        kk, vv = k[blk, j % bs].double(), step.v_cache[blk, j % bs]
        for i in range(end - start):
            n = lks[b] - (end - start) + i + 1
            for h in range(hq):
                s = kk[:n, h // 2] @ q[start + i, h].double() * step.scale
                s = cap * torch.tanh(s / cap)
                top = s.topk(min(2, n)).values
                if n == 1 or top[0] - top[1] > 2 * cap_error + 2.0 ** -14 * far + 200:
                    assert torch.equal(out[start + i, h], vv[s.argmax(), h // 2])
                    checked += 1
        start = end
    assert checked >= (0 if far > 8 * cap else 4)


def test_caps_past_the_range_are_refused():
    step = workloads.make_gqa_step(lqs=[1], lks=[9], num_q_heads=2, num_kv_heads=1, head_dim=64, block_size=16, seed=1)
    plan = ops.AttentionPlan.from_lists(step.block_table.to(DEV), step.cu_seqlens_q, step.seqlens_kv, 2, 1, 64, 16)
    with pytest.raises(ValueError, match="softcap"):
        ops.paged_attention_gqa(step.q.to(DEV), step.k_cache.to(DEV), step.v_cache.to(DEV), plan, step.scale,
                                softcap=2e38)
