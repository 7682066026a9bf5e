"""Paged attention over 8-bit caches and with modified scores against a float64
restatement, within the bound that the kernels' roundings leave (derived in
oracle/long_context.py)."""
import pytest
import torch

from auto_infer_amd import ops, workloads
from oracle import long_context as oracle
from oracle.paged_attn import nz_from_nd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

MODS = {
    "plain": {},
    "cap": dict(cap=5.0),
    "bias": dict(bias=True),
    "prefix": dict(prefix=True),
    "all": dict(cap=30.0, bias=True, prefix=True),
}


def quantised(x, seed):
    """A bf16 cache as e4m3 values and scales with per-block sizes."""
    gen = torch.Generator().manual_seed(seed)
    x = x.double() * torch.exp2(torch.randint(-3, 4, (x.shape[0], 1, x.shape[2], 1), generator=gen).double())
    e = torch.tensor([[oracle.needed_exp(v) for v in row] for row in x.abs().amax(dim=(1, 3)).tolist()])
    q = oracle.e4m3(x * torch.exp2(-e.double())[:, None, :, None]).to(torch.float8_e4m3fn)
    return q, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def run(lqs, lks, hq, hkv, d, bs, kv="nd", cap=0.0, bias=False, prefix=False, seed=0, fused=False,
        shared=0):
    step = workloads.make_gqa_step(lqs=lqs, lks=lks, num_q_heads=hq, num_kv_heads=hkv, head_dim=d,
                                   block_size=bs, seed=seed, extra_blocks=2)
    gen = torch.Generator().manual_seed(seed + 1)
    slopes = torch.exp2(-8.0 * torch.rand(hq, generator=gen)) if bias else None
    pre = None
    if prefix:
        pre = torch.tensor([[0, lk // 2, lk, lk + 9, -3, max(0, lk - lq)][int(torch.randint(6, (1,), generator=gen))]
                            for lq, lk in zip(lqs, lks)], dtype=torch.int32)
    keys, values = step.k_cache, step.v_cache
    more = {}
    if kv == "fp8":
        (kq, ks), (vq, vs) = quantised(keys, seed + 2), quantised(values, seed + 3)
        keys, values = oracle.dequantised(kq, ks), oracle.dequantised(vq, vs)
        dk, dv = kq.to(DEV), vq.to(DEV)
        more = dict(key_scale=ks.to(DEV), value_scale=vs.to(DEV))
    elif kv == "nz":
        dk, dv = nz_from_nd(keys).to(DEV), nz_from_nd(values).to(DEV)
        more = dict(kv_layout="nz")
    else:
        dk, dv = keys.to(DEV), values.to(DEV)
    if fused:          # the new rows come with the call
        from oracle.paged_attn import kv_write
        kv_write(step.k_new, step.v_new, keys, values, step.slot_mapping)
        more.update(key_new=step.k_new.to(DEV), value_new=step.v_new.to(DEV))
    plan = ops.AttentionPlan.from_lists(step.block_table.to(DEV), step.cu_seqlens_q, step.seqlens_kv, hq,
                                        hkv, d, bs, prefix_lens=None if pre is None else pre.to(DEV))
    out = ops.paged_attention_gqa(step.q.to(DEV), dk, dv, plan, step.scale, softcap=cap,
                                  alibi_slopes=None if slopes is None else slopes.to(DEV), **more)
    plan.status()
    ref, bound = oracle.scored_attention(step.q, keys, values, step.block_table, step.cu_seqlens_q,
                                         step.seqlens_kv, step.scale, cap, slopes,
                                         None if pre is None else pre.tolist())
    far = (out.cpu().double() - ref).abs()
    assert bool((far <= bound).all()), ((far - bound).max().item(), (far / bound.clamp(min=1e-30)).max().item())
    print(f"largest share of the bound {(far / bound.clamp(min=1e-30)).max().item():.3f}", flush=True)
    if fused:
        want = (nz_from_nd(keys), nz_from_nd(values)) if kv == "nz" else (keys, values)
        assert torch.equal(dk.cpu(), want[0]) and torch.equal(dv.cpu(), want[1])


# (lqs, lks): decode rows of the lengths where tiles and blocks end; verify
# rows; prompts; prompts beside decode rows; requests without keys, rows
# before the first key, requests without rows
STEPS = {
    "decode": ([1] * 12, [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 700]),
    "one_long": ([1], [5000]),
    "verify": ([3, 1, 2, 4, 3], [3, 40, 257, 4, 1000]),
    "short_prompts": ([7, 5, 9], [7, 40, 100]),
    "prompts": ([130, 65, 200], [130, 300, 200]),
    "mixed": ([1, 150, 1, 2, 90], [400, 150, 33, 70, 517]),
    "empty": ([1, 2, 0, 5, 1], [0, 40, 12, 3, 1]),
}
HEADS = {"16_8_128": (16, 8, 128), "28_4_128": (28, 4, 128), "14_2_64": (14, 2, 64), "5_5_64": (5, 5, 64),
         "20_1_128": (20, 1, 128)}


@pytest.mark.parametrize("mod", list(MODS))
@pytest.mark.parametrize("name", list(STEPS))
@pytest.mark.parametrize("heads", list(HEADS))
def test_fp8_caches(mod, name, heads):
    hq, hkv, d = HEADS[heads]
    lqs, lks = STEPS[name]
    run(lqs, lks, hq, hkv, d, 16, "fp8", seed=len(name) + hq, **MODS[mod])


@pytest.mark.parametrize("kv", ["nd", "nz"])
@pytest.mark.parametrize("mod", [m for m in MODS if m != "plain"])
@pytest.mark.parametrize("name", list(STEPS))
@pytest.mark.parametrize("heads", ["28_4_128", "14_2_64"])
def test_scored_bf16_caches(kv, mod, name, heads):
    hq, hkv, d = HEADS[heads]
    lqs, lks = STEPS[name]
    run(lqs, lks, hq, hkv, d, 16, kv, seed=len(name) + hq, fused=name in ("mixed", "decode", "prompts"),
        **MODS[mod])


@pytest.mark.parametrize("kv", ["nd", "fp8"])
@pytest.mark.parametrize("bs", [1, 3, 40, 64, 128, 300])
@pytest.mark.parametrize("name", ["decode", "mixed", "verify"])
def test_block_sizes(kv, bs, name):
    lqs, lks = STEPS[name]
    run(lqs, lks, 16, 8, 128, bs, kv, seed=bs, **MODS["all"])
    run(lqs, lks, 28, 4, 128, bs, kv, seed=bs + 1, **MODS["cap"])


@pytest.mark.parametrize("kv", ["nd", "fp8"])
def test_long_requests_are_split(kv):
    run([1, 1, 3], [9000, 70, 4100], 16, 2, 128, 64, kv, seed=3, **MODS["all"])
    run([140, 260], [2600, 3000], 8, 1, 128, 64, kv, seed=4, **MODS["all"])
    run([300], [4000], 14, 2, 64, 16, kv, seed=5, **MODS["all"])


@pytest.mark.parametrize("kv", ["nd", "nz", "fp8"])
@pytest.mark.parametrize("heads", ["28_4_128", "14_2_64", "16_8_128"])
@pytest.mark.parametrize("mod", ["cap", "bias", "all"])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(kv, heads, mod):
    """Infinities and NaN in later tokens' keys and values, and in slots past a
    request's end: rows that do not see them are as if they were not there."""
    hq, hkv, d = HEADS[heads]
    lqs, lks = [4, 150, 1, 90, 3], [37, 150, 64, 517, 1500]
    bs = 16
    step = workloads.make_gqa_step(lqs=lqs, lks=lks, num_q_heads=hq, num_kv_heads=hkv, head_dim=d,
                                   block_size=bs, seed=3, extra_blocks=2)
    m = MODS[mod]
    gen = torch.Generator().manual_seed(4)
    slopes = torch.exp2(-8.0 * torch.rand(hq, generator=gen)) if m.get("bias") else None
    pre = torch.tensor([0, 20, 10, 0, 0], dtype=torch.int32) if m.get("prefix") else None
    keys, values = step.k_cache, step.v_cache
    more = {}
    if kv == "fp8":
        (kq, ks), (vq, vs) = quantised(keys, 5), quantised(values, 6)
        keys, values = kq.float(), vq.float()

    def put(cache, request, position, head, dim, x):
        cache[step.block_table[request, position // bs], position % bs, head, dim] = x
    inf = float("nan") if kv == "fp8" else float("inf")
    put(values, 0, 35, 0, 3, inf), put(values, 0, 36, hkv - 1, 5, float("nan"))
    put(keys, 0, 36, 0, 7, float("nan"))
    put(values, 1, 149, 0, 0, float("nan")), put(values, 1, 120, hkv - 1, d - 1, inf)
    put(values, 1, 70, 0, d // 2, -inf), put(keys, 1, 131, hkv - 1, 1, inf)
    put(values, 3, 500, 0, 9, inf), put(values, 3, 516, hkv - 1, 9, float("nan"))
    put(values, 4, 1498, 0, 9, inf)
    for r, lk in enumerate(lks):               # slots past the end
        for p in range(lk, -(-lk // bs) * bs):
            put(values, r, p, slice(None), slice(None), float("nan"))
            put(keys, r, p, slice(None), slice(None), float("nan"))
    if kv == "fp8":
        kq, vq = keys.to(torch.float8_e4m3fn), values.to(torch.float8_e4m3fn)
        keys, values = oracle.dequantised(kq, ks), oracle.dequantised(vq, vs)
        dk, dv = kq.to(DEV), vq.to(DEV)
        more = dict(key_scale=ks.to(DEV), value_scale=vs.to(DEV))
    elif kv == "nz":
        dk, dv, more = nz_from_nd(keys).to(DEV), nz_from_nd(values).to(DEV), dict(kv_layout="nz")
    else:
        dk, dv = keys.to(DEV), values.to(DEV)
    plan = ops.AttentionPlan.from_lists(step.block_table.to(DEV), step.cu_seqlens_q, step.seqlens_kv, hq,
                                        hkv, d, bs, prefix_lens=None if pre is None else pre.to(DEV))
    out = ops.paged_attention_gqa(step.q.to(DEV), dk, dv, plan, step.scale, softcap=m.get("cap", 0.0),
                                  alibi_slopes=None if slopes is None else slopes.to(DEV), **more)
    ref, bound = oracle.scored_attention(step.q, keys, values, step.block_table, step.cu_seqlens_q,
                                         step.seqlens_kv, step.scale, m.get("cap", 0.0), slopes,
                                         None if pre is None else pre.tolist())
    got = out.cpu().double()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fine)
    assert 0.3 < fine.double().mean() < 1
    assert bool(((got - ref).abs() <= bound)[fine].all())


def test_capped_scores_far_past_the_cap():
    """Scores of +-1000 at a cap of 2: weights within e^4 of each other."""
    hq, hkv, d, bs = 4, 2, 64, 16
    step = workloads.make_gqa_step(lqs=[1, 70], lks=[50, 70], num_q_heads=hq, num_kv_heads=hkv, head_dim=d,
                                   block_size=bs, seed=1)
    q = (step.q * 60).bfloat16()
    plan = ops.AttentionPlan.from_lists(step.block_table.to(DEV), step.cu_seqlens_q, step.seqlens_kv, hq,
                                        hkv, d, bs)
    out = ops.paged_attention_gqa(q.to(DEV), step.k_cache.to(DEV), step.v_cache.to(DEV), plan, 1.0, softcap=2.0)
    ref, _ = oracle.scored_attention(q, step.k_cache, step.v_cache, step.block_table, step.cu_seqlens_q,
                                     step.seqlens_kv, 1.0, 2.0)
    _, bound = oracle.scored_attention(step.q, step.k_cache, step.v_cache, step.block_table,
                                       step.cu_seqlens_q, step.seqlens_kv, 1.0, 2.0)
    # saturated scores: the products' errors vanish in the cap, so the bound's
    # relative part applies to the output alone
    far = (out.cpu().double() - ref).abs()
    vmax = step.v_cache.abs().max().item()
    assert far.max().item() <= (2.0 ** -8 + 2.0 ** -10 + 2.0 ** -8) * vmax * 1.5


@pytest.mark.parametrize("cap", [1e-20, 1e-4, 0.01, 1.0, 1e3, 1e6, 1e20])
@pytest.mark.parametrize("zero", [False, True])
def test_caps_of_any_size(cap, zero):
    """Tiny caps (all weights equal in the limit), huge ones (no cap), and
    queries of zeros, whose scores are zero at any cap."""
    hq, hkv, d, bs = 4, 2, 128, 16
    step = workloads.make_gqa_step(lqs=[1, 70], lks=[50, 90], num_q_heads=hq, num_kv_heads=hkv, head_dim=d,
                                   block_size=bs, seed=8)
    q = step.q * 0 if zero else step.q
    plan = ops.AttentionPlan.from_lists(step.block_table.to(DEV), step.cu_seqlens_q, step.seqlens_kv, hq,
                                        hkv, d, bs)
    for slopes in (None, torch.full((hq,), 0.25)):
        out = ops.paged_attention_gqa(q.to(DEV), step.k_cache.to(DEV), step.v_cache.to(DEV), plan, step.scale,
                                      softcap=cap, alibi_slopes=None if slopes is None else slopes.to(DEV))
        ref, bound = oracle.scored_attention(q, step.k_cache, step.v_cache, step.block_table, step.cu_seqlens_q,
                                             step.seqlens_kv, step.scale, cap, slopes)
        assert bool(((out.cpu().double() - ref).abs() <= bound).all())


def test_fp8_pool_past_32_bits():
    """Blocks whose bytes lie past 2^32 (and slots past 2^22)."""
    hq, hkv, d, bs = 16, 8, 128, 128
    nb = (1 << 32) // (bs * hkv * d) + 40
    step = workloads.make_gqa_step(lqs=[1, 60], lks=[700, 300], num_q_heads=hq, num_kv_heads=hkv, head_dim=d,
                                   block_size=bs, seed=6)
    (kq, ks), (vq, vs) = quantised(step.k_cache, 1), quantised(step.v_cache, 2)
    used = step.k_cache.shape[0]
    at = torch.tensor([nb - 1 - 3 * i for i in range(used)], device=DEV)
    kc, vc = (torch.empty(nb, bs, hkv, d, dtype=torch.uint8, device=DEV) for _ in range(2))
    kse, vse = (torch.zeros(nb, hkv, dtype=torch.uint8, device=DEV) for _ in range(2))
    for pool, part in ((kc, kq), (vc, vq), (kse, ks), (vse, vs)):
        pool[at] = part.view(torch.uint8).to(DEV)
    table = at.int()[step.block_table.long().to(DEV)]
    plan = ops.AttentionPlan.from_lists(table, step.cu_seqlens_q, step.seqlens_kv, hq, hkv, d, bs)
    out = ops.paged_attention_gqa(step.q.to(DEV), kc.view(ops.FP8_KV), vc.view(ops.FP8_KV), plan, step.scale,
                                  key_scale=kse.view(ops.FP8_KV_SCALE), value_scale=vse.view(ops.FP8_KV_SCALE))
    ref, bound = oracle.scored_attention(step.q, oracle.dequantised(kq, ks), oracle.dequantised(vq, vs),
                                         step.block_table, step.cu_seqlens_q, step.seqlens_kv, step.scale)
    assert bool(((out.cpu().double() - ref).abs() <= bound).all())
