"""Shared prefixes, block-sparse attention and appending with rotation at the ends of
their ranges: empty steps, groups of 256 heads, selections without a choice, caches whose
offsets pass 32 bits, and steps drawn by chance."""
import random

import pytest
import torch

from auto_infer_amd import ops
from oracle import block_sparse as ref
from tests import test_gpu_block_sparse as sparse
from tests import test_gpu_shared_prefix as shared

pytestmark = pytest.mark.gpu
DEV = "cuda"


def e8m0(e):
    return (e + 127).to(torch.uint8).to(DEV).view(torch.float8_e8m0fnu)


@pytest.mark.parametrize("batch", [0, 3])
def test_steps_without_tokens(batch):
    table = torch.zeros(max(1, batch), 4, dtype=torch.int32, device=DEV)
    cu = torch.zeros(batch + 1, dtype=torch.int32, device=DEV)
    lk = torch.full((batch,), 20, dtype=torch.int32, device=DEV)
    kc = torch.zeros(6, 16, 2, 64, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=DEV)
    plan = ops.BlockSparsePlan(table, cu, lk, 0, 4, 2, 64, 16, 3)
    bounds, scale = sparse.empty_bounds(6, 2, 64)
    before = bounds.clone()
    ops.summarize_blocks(kc, plan, bounds, scale)
    assert torch.equal(bounds, before)
    sel = ops.select_blocks(q, plan, bounds, scale)
    assert sel.shape == (0, 2, 3)
    assert ops.paged_attention_sparse(q, kc, kc, plan, sel, 0.1).shape == (0, 4, 64)
    both = ops.SharedPrefixPlan(table, cu, lk, 0, 4, 2, 64, 16)
    both.status()
    assert ops.paged_attention_shared(q, kc, kc, both, 0.1).shape == (0, 4, 64)
    rope = ops.RotaryEmbedding(64, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    out = ops.rope_append(torch.zeros(0, 8 * 64, dtype=torch.bfloat16, device=DEV), 4, 2, none.long(), rope, kc, kc, none)
    assert out.shape == (0, 4, 64)


@pytest.mark.parametrize("lens", [[(1, 300), (2, 77)], [(9, 40), (14, 60)]])
@pytest.mark.parametrize("signs", [1, -1, 0])
@pytest.mark.parametrize("d", [64, 128])
def test_whole_numbers_of_256_heads(d, signs, lens):
    """Sums over the heads from 0 to 127 * 256, of one sign or both."""
    s = sparse.make(lens, 256, 1, d, 4, seed=3)
    gen = torch.Generator().manual_seed(4)
    if signs:
        s["q"] = torch.full_like(s["q"], 127.0 * signs)
    else:
        s["q"] = torch.randint(-127, 128, s["q"].shape, generator=gen).bfloat16()
    b, e = sparse.random_bounds(s, 5)
    b[::5] = 127
    g = sparse.on_gpu(s)
    out = ops.select_blocks(g["q"], sparse.make_plan(g, 5, 1, 1), b.to(DEV), e8m0(e)).cpu()
    for t, r, pos in sparse.tokens_of(s):
        rows = s["table"][r].long()
        want = ref.select(s["q"][t], b[rows, 0, 0], b[rows, 0, 1], e[rows, 0], pos // 4 + 1, 5, 1, 1)
        assert out[t, 0].tolist() == want + [-1] * (5 - len(want)), t


@pytest.mark.parametrize("most", [60, 250, 1400, 9000])
def test_selections_without_a_choice(most):
    """All that is taken is always taken; or all scores are equal."""
    s = sparse.make([(1, most), (2, most - 7)], 4, 2, 64, 1, seed=2)
    b, e = sparse.random_bounds(s, 7)
    g = sparse.on_gpu(s)
    out = ops.select_blocks(g["q"], sparse.make_plan(g, 11, 4, 7), b.to(DEV), e8m0(e)).cpu()
    for t, _, pos in sparse.tokens_of(s):
        n = pos + 1
        assert out[t].tolist() == [list(range(4)) + list(range(n - 7, n))] * 2
    same, e = b[:1].expand_as(b).contiguous(), torch.zeros_like(e)
    out = ops.select_blocks(g["q"], sparse.make_plan(g, 30, 2, 3), same.to(DEV), e8m0(e)).cpu()
    for t, _, pos in sparse.tokens_of(s):
        n = pos + 1
        assert out[t].tolist() == [list(range(27)) + list(range(n - 3, n))] * 2


def test_entries_behind_padding_and_out_of_order():
    s = sparse.make([(3, 900)], 4, 2, 64, 4, seed=8, spread=False)
    g = sparse.on_gpu(s)
    rng = random.Random(1)
    sel = torch.tensor([[[rng.randint(-3, 230) for _ in range(140)] for _ in range(2)] for _ in range(3)], dtype=torch.int32)
    sel[0, 0, :70], sel[0, 0, 70:] = -1, torch.arange(3, 73)
    sel[0, 1, :64], sel[0, 1, 64:] = torch.arange(64), torch.arange(10, 86)
    sel[1, 0] = -1
    sel[1, 0, ::3] = torch.arange(0, 141, 3)[:47]
    out = ops.paged_attention_sparse(g["q"], g["kc"], g["vc"], sparse.make_plan(g, 140), sel.to(DEV), 0.125)
    sparse.check_attention(s, sel, out.cpu(), 0.125)


def test_caches_of_more_than_four_gigabytes():
    """The step's blocks lie at both ends of caches whose byte offsets and numbers of
    values pass 32 bits."""
    bs, hq, hkv, d, nb = 128, 16, 8, 128, 17000            # 2.2e9 values
    assert nb * bs * hkv * d > 2 ** 31
    kc = torch.empty(nb, bs, hkv, d, dtype=torch.bfloat16, device=DEV)
    vc = torch.empty_like(kc)
    lens = [(1, 700), (1, 650), (1, 300)]
    head = [nb - 1, 0, nb - 2]
    rows = [head + [nb - 3, 1, nb - 4], head + [2, nb - 5, 3], [nb - 6, 4, nb - 7]]
    table = torch.zeros(3, 7, dtype=torch.int32)
    for i, r in enumerate(rows):
        table[i, :len(r)] = torch.tensor(r)
    gen = torch.Generator().manual_seed(9)
    small, at = {}, sorted({b for r in rows for b in r})
    idx = torch.tensor(at)
    for name, cache in (("kx", kc), ("vx", vc)):
        x = torch.randn(len(at), bs, hkv, d, generator=gen).bfloat16()
        cache[idx.to(DEV)] = x.to(DEV)
        small[name] = x
    # each request's new token through rope_append, at its slot
    rope = ops.RotaryEmbedding(d, device=DEV)
    qkv = torch.randn(3, (hq + 2 * hkv) * d, generator=gen).bfloat16().to(DEV)
    pos = torch.tensor([lk - 1 for _, lk in lens], device=DEV)
    blocks = torch.tensor([rows[i][(lk - 1) // bs] for i, (_, lk) in enumerate(lens)])
    slots = (blocks * bs + torch.tensor([(lk - 1) % bs for _, lk in lens])).int().to(DEV)
    rq, rk, rv = ops.rope_qk(qkv.clone(), hq, hkv, pos, rope)
    q = ops.rope_append(qkv, hq, hkv, pos, rope, kc, vc, slots)
    assert torch.equal(q, rq)
    off = (slots % bs).long()
    assert torch.equal(kc[blocks.to(DEV), off], rk) and torch.equal(vc[blocks.to(DEV), off], rv)
    cu = torch.arange(4, dtype=torch.int32)
    place = torch.zeros(nb, dtype=torch.int32)
    place[idx] = torch.arange(len(at), dtype=torch.int32)
    s = dict(lens=lens, hq=hq, hkv=hkv, d=d, bs=bs, t=3, table=place[table.long()], q=q.cpu(),
             kx=kc[idx.to(DEV)].cpu().double(), vx=vc[idx.to(DEV)].cpu().double())
    lk = torch.tensor([n for _, n in lens], dtype=torch.int32, device=DEV)
    plan = ops.SharedPrefixPlan(table.to(DEV), cu.to(DEV), lk, 3, hq, hkv, d, bs)
    shared.check(s, ops.paged_attention_shared(q, kc, vc, plan, d ** -0.5).cpu())
    plan = ops.BlockSparsePlan(table.to(DEV), cu.to(DEV), lk, 3, hq, hkv, d, bs, 3, 1, 1)
    bounds, scale = sparse.empty_bounds(nb, hkv, d)
    bounds.random_(-20, 100)
    ops.summarize_blocks(kc, plan, bounds, scale)
    for i, blk in enumerate(blocks.tolist()):
        n = (lens[i][1] - 1) % bs + 1
        for h in range(hkv):
            hi, nlo, e = ref.block_bounds(kc[blk, :n, h].cpu().double())
            assert torch.equal(bounds[blk, h].cpu().long(), torch.stack([hi, nlo]))
            assert int(scale.view(torch.uint8)[blk, h]) == e + 127
    sel = ops.select_blocks(q, plan, bounds, scale)
    sparse.check_attention(s, sel.cpu(), ops.paged_attention_sparse(q, kc, vc, plan, sel, d ** -0.5).cpu(), d ** -0.5)


@pytest.mark.parametrize("seed", range(24))
def test_drawn_steps(seed):
    rng = random.Random(seed)
    hq, hkv, d = rng.choice(sparse.SHAPES)
    bs, fp8 = rng.choice([1, 3, 16, 32, 48, 64, 128, 200]), rng.random() < 0.5
    groups = [(rng.choice([0, 100, 128, 300, 900]), [(lq, lq + rng.randint(0, 200)) for lq in
               (rng.choice([0, 1, 1, 1, 2, 4, 30, 140]) for _ in range(rng.randint(1, 9)))]) for _ in range(rng.randint(1, 4))]
    s = shared.make(groups, hq, hkv, d, bs, fp8, seed=seed)
    out, _ = shared.run(s, by_id=rng.random() < 0.5)
    shared.check(s, out)
    lens = [(lq, lq + rng.randint(0, 1500)) for lq in (rng.choice([0, 1, 1, 2, 5, 40, 100]) for _ in range(rng.randint(1, 6)))]
    s = sparse.make(lens, hq, hkv, d, bs, fp8, seed=seed, spread=False)
    if s["t"] == 0:
        return
    g = sparse.on_gpu(s)
    n = rng.randint(2, 30)
    plan = sparse.make_plan(g, n, rng.randint(0, 1), 1)
    b, e = sparse.random_bounds(s, seed)
    sel = ops.select_blocks(g["q"], plan, b.to(DEV), e8m0(e)).cpu()
    some = {t for t in range(s["t"]) if s["t"] < 12 or rng.random() < 12 / s["t"]}
    for t, r, pos in sparse.tokens_of(s):
        if t in some:
            rows, h = s["table"][r].long(), rng.randrange(hkv)
            want = ref.select(s["q"][t, h * (hq // hkv):(h + 1) * (hq // hkv)], b[rows, h, 0], b[rows, h, 1], e[rows, h],
                              max(0, pos // bs + 1), n, plan.sink, 1)
            assert sel[t, h].tolist() == want + [-1] * (n - len(want)), (t, h)
    out = ops.paged_attention_sparse(g["q"], g["kc"], g["vc"], plan, sel.to(DEV), d ** -0.5, key_scale=g["ks"],
                                     value_scale=g["vs"])
    sparse.check_attention(s, sel, out.cpu(), d ** -0.5, some)


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64)])
def test_prompts_with_query_values_that_are_not_finite(hq, hkv, d):
    """They count as zero, beside tokens of the same tile that have none."""
    s = sparse.make([(45, 200)], hq, hkv, d, 3, seed=12)
    s["q"][3, 1, 5], s["q"][3, 2, 9], s["q"][20, 0, 0] = float("nan"), float("-inf"), float("inf")
    s["q"][21] = float("nan")
    s["q"][33, :, :] *= 2.0 ** 100
    s["q"][34, :, :] *= 2.0 ** -120
    b, e = sparse.random_bounds(s, 3)
    g = sparse.on_gpu(s)
    out = ops.select_blocks(g["q"], sparse.make_plan(g, 7, 1, 2), b.to(DEV), e8m0(e)).cpu()
    for t, r, pos in sparse.tokens_of(s):
        rows = s["table"][r].long()
        for h in range(hkv):
            q = s["q"][t, h * (hq // hkv):(h + 1) * (hq // hkv)]
            assert out[t, h].tolist() == ref.select(q, b[rows, h, 0], b[rows, h, 1], e[rows, h], pos // 3 + 1, 7, 1, 2), t


@pytest.mark.parametrize("most", [250, 383, 500, 639, 760, 1023, 2000, 4000, 8000, 8300])
def test_selections_over_tables_of_many_widths(most):
    s = sparse.make([(1, most), (1, most // 2), (1, 70)], 4, 2, 64, 1, seed=most)
    b, e = sparse.random_bounds(s, most)
    g = sparse.on_gpu(s)
    out = ops.select_blocks(g["q"], sparse.make_plan(g, 64, 1, 2), b.to(DEV), e8m0(e)).cpu()
    for t, r, pos in sparse.tokens_of(s):
        rows = s["table"][r].long()
        for h in range(2):
            want = ref.select(s["q"][t, 2 * h:2 * h + 2], b[rows, h, 0], b[rows, h, 1], e[rows, h], pos + 1, 64, 1, 2)
            assert out[t, h].tolist() == want, (t, h)
