"""Seeded random steps through 8-bit cache writes, scored and 8-bit attention and
rotary positions: head counts and groups of every kind, odd block sizes, ragged
lengths, requests without rows or keys, rows behind the last request."""
import numpy as np
import pytest
import torch

from auto_infer_amd import ops, workloads
from oracle import long_context as oracle
from oracle.paged_attn import kv_write, nz_from_nd

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def lengths(rng):
    """(query lengths, KV lengths): decode, verify, prompts, mixtures."""
    kind = rng.choice(["decode", "verify", "prompts", "mixed"])
    lqs, lks = [], []
    for _ in range(int(rng.integers(1, 10))):
        if kind == "decode":
            lq = 1
        elif kind == "verify":
            lq = int(rng.integers(0, 6))
        elif kind == "prompts":
            lq = int(rng.integers(1, 260))
        else:
            lq = int(rng.choice([0, 1, 1, 1, 2, 5, 33, 130, 200]))
        lk = max(0, lq + int(rng.choice([0, 0, 1, 17, 100, 600])) + int(rng.choice([0, 0, 0, -1, -3])))
        lqs.append(lq)
        lks.append(lk)
    if sum(lqs) == 0:
        lqs[0], lks[0] = 1, max(lks[0], 1)
    return lqs, lks


HEADS = [(16, 8), (8, 8), (28, 4), (32, 4), (14, 2), (7, 1), (16, 1), (20, 1), (26, 1), (48, 16), (9, 9), (12, 3),
         (10, 5), (64, 8)]


@pytest.mark.parametrize("seed", range(60))
def test_attention(seed):
    rng = np.random.default_rng(1000 + seed)
    hq, hkv = HEADS[int(rng.integers(len(HEADS)))]
    d, bs = int(rng.choice([64, 128])), int(rng.choice([1, 5, 16, 16, 24, 32, 64, 128, 192]))
    lqs, lks = lengths(rng)
    kv = str(rng.choice(["nd", "nz", "fp8", "fp8"]))
    cap = float(rng.choice([0.0, 0.0, 2.0, 30.0]))
    bias, prefix = bool(rng.random() < 0.4), bool(rng.random() < 0.4)
    pad = int(rng.choice([0, 0, 3]))               # rows behind the last request
    print(seed, hq, hkv, d, bs, lqs, lks, kv, cap, bias, prefix, pad, flush=True)
    # (the generator's slots of rows before the first key are not used)
    step = workloads.make_gqa_step(lqs=[min(a, b) for a, b in zip(lqs, lks)], lks=lks, num_q_heads=hq,
                                   num_kv_heads=hkv, head_dim=d, block_size=bs, seed=seed, extra_blocks=1)
    gen = torch.Generator().manual_seed(seed)
    T = sum(lqs)
    cu = np.cumsum(lqs).tolist()
    q = torch.randn(T + pad, hq, d, generator=gen).bfloat16()
    keys, values = step.k_cache, step.v_cache
    slopes = torch.exp2(-8.0 * torch.rand(hq, generator=gen)) if bias else None
    pre = torch.tensor([int(rng.integers(-2, lk + 5)) for lk in lks], dtype=torch.int32) if prefix else None
    more = {}
    if kv == "fp8":
        slots = torch.arange(keys.shape[0] * bs, dtype=torch.int32, device=DEV)
        shape = tuple(keys.shape)
        dk, dv = (torch.zeros(shape, dtype=torch.uint8, device=DEV).view(ops.FP8_KV) for _ in range(2))
        ks, vs = (torch.zeros(shape[0], hkv, dtype=torch.uint8, device=DEV).view(ops.FP8_KV_SCALE) for _ in range(2))
        ops.write_kv_fp8(keys.view(-1, hkv, d).to(DEV), values.view(-1, hkv, d).to(DEV), dk, dv, ks, vs, slots)
        keys, values = oracle.dequantised(dk.cpu(), ks.cpu()), oracle.dequantised(dv.cpu(), vs.cpu())
        more = dict(key_scale=ks, value_scale=vs)
    else:
        if not (cap or bias or prefix):
            cap = 9.0
        conv = nz_from_nd if kv == "nz" else (lambda x: x)
        dk, dv = conv(keys).to(DEV), conv(values).to(DEV)
        more = dict(kv_layout=kv)
        if rng.random() < 0.5 and T and not pad and lqs == [min(a, b) for a, b in zip(lqs, lks)]:
            kv_write(step.k_new, step.v_new, keys, values, step.slot_mapping)
            more.update(key_new=step.k_new.to(DEV), value_new=step.v_new.to(DEV))
    plan = ops.AttentionPlan(step.block_table.to(DEV), torch.tensor([0] + cu, dtype=torch.int32, device=DEV),
                             torch.tensor(lks, dtype=torch.int32, device=DEV), T + pad, hq, hkv, d, bs,
                             prefix_lens=None if pre is None else pre.to(DEV))
    out = torch.full((T + pad, hq, d), 123.0, dtype=torch.bfloat16, device=DEV)
    ops.paged_attention_gqa(q.to(DEV), dk, dv, plan, step.scale, out=out, softcap=cap,
                            alibi_slopes=None if slopes is None else slopes.to(DEV), **more)
    plan.status()
    ref, bound = oracle.scored_attention(q[:T], keys, values, step.block_table, cu, lks, step.scale, cap, slopes,
                                         None if pre is None else pre.tolist())
    got = out.cpu().double()
    assert bool(((got[:T] - ref).abs() <= bound).all())
    assert bool((got[T:] == 123.0).all())


@pytest.mark.parametrize("seed", range(40))
def test_writes(seed):
    rng = np.random.default_rng(2000 + seed)
    gen = torch.Generator().manual_seed(seed)
    h, d = int(rng.choice([1, 2, 3, 4, 5, 8, 9])), int(rng.choice([64, 128]))
    bs = int(rng.choice([1, 2, 7, 16, 16, 17, 31, 32, 33, 64, 128, 129, 512]))
    nb = int(rng.integers(2, 40))
    vals = [oracle.e4m3(torch.randn(nb, bs, h, d, generator=gen) * 60) for _ in range(2)]
    exps = [torch.randint(-9, 4, (nb, h), generator=gen) for _ in range(2)]
    caches = [x.to(torch.float8_e4m3fn).to(DEV) for x in vals]
    scales = [(e + 127).to(torch.uint8).to(DEV).view(torch.float8_e8m0fnu) for e in exps]
    for _ in range(3):
        slots = []
        for _ in range(int(rng.integers(1, 30))):
            kind = rng.integers(4)
            at = int(rng.integers(nb * bs))
            if kind == 0:
                slots += [at]
            elif kind == 1:
                slots += list(range(at, min(nb * bs, at + int(rng.integers(1, 3 * bs + 2)))))
            elif kind == 2:
                slots += [-1] * int(rng.integers(1, 4)) + [at]
            else:
                slots += [int(s) for s in rng.integers(nb * bs, size=int(rng.integers(1, 9)))]
        slots = slots[:1500]
        rows = [(torch.randn(len(slots), h, d, generator=gen) * float(rng.choice([0.1, 1, 30]))).bfloat16()
                for _ in range(2)]
        st = torch.tensor(slots, dtype=torch.int32, device=DEV)
        ops.write_kv_fp8(rows[0].to(DEV), rows[1].to(DEV), caches[0], caches[1], scales[0], scales[1], st)
        for x in range(2):
            oracle.write_kv_fp8(rows[x], vals[x], exps[x], slots)
            assert torch.equal(scales[x].view(torch.uint8).cpu().int() - 127, exps[x].int()), (seed, h, d, bs, nb)
            assert torch.equal(caches[x].cpu().double(), vals[x]), (seed, h, d, bs, nb)


def test_the_largest_block():
    gen = torch.Generator().manual_seed(1)
    h, d, bs, nb = 2, 64, 8192, 2
    vals, exps = torch.zeros(nb, bs, h, d, dtype=torch.float64), torch.full((nb, h), -127)
    cache = torch.zeros(nb, bs, h, d, dtype=torch.uint8, device=DEV).view(ops.FP8_KV)
    scale = torch.zeros(nb, h, dtype=torch.uint8, device=DEV).view(ops.FP8_KV_SCALE)
    for first, n in ((0, 300), (300, 900), (7000, 1300), (9492, 1)):
        slots = list(range(first, first + n))
        rows = (torch.randn(n, h, d, generator=gen) * (1 + first)).bfloat16()
        ops.write_kv_fp8(rows.to(DEV), None, cache, None, scale, None, torch.tensor(slots, dtype=torch.int32, device=DEV))
        oracle.write_kv_fp8(rows, vals, exps, slots)
        assert torch.equal(scale.view(torch.uint8).cpu().int() - 127, exps.int())
        assert torch.equal(cache.cpu().double(), vals)


def test_a_step_of_a_thousand_requests_with_prefixes():
    """More segments than the planner keeps in registers."""
    rng = np.random.default_rng(5)
    lqs = [int(rng.choice([1, 1, 2, 4])) for _ in range(1200)]
    lks = [lq + int(rng.integers(0, 40)) for lq in lqs]
    hq, hkv, d, bs = 4, 2, 64, 16
    step = workloads.make_gqa_step(lqs=lqs, lks=lks, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, block_size=bs,
                                   seed=5)
    pre = torch.tensor([int(rng.integers(0, lk + 2)) for lk in lks], dtype=torch.int32)
    plan = ops.AttentionPlan.from_lists(step.block_table.to(DEV), step.cu_seqlens_q, step.seqlens_kv, hq, hkv, d, bs,
                                        prefix_lens=pre.to(DEV))
    out = ops.paged_attention_gqa(step.q.to(DEV), step.k_cache.to(DEV), step.v_cache.to(DEV), plan, step.scale)
    plan.status()
    ref, bound = oracle.scored_attention(step.q, step.k_cache, step.v_cache, step.block_table, step.cu_seqlens_q,
                                         step.seqlens_kv, step.scale, prefix=pre.tolist())
    assert bool(((out.cpu().double() - ref).abs() <= bound).all())
