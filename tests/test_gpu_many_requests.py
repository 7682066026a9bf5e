"""Shared prefixes and block-sparse steps of many requests (the planners go over them in
several passes, with more LDS than is given without asking), and selections in several
launches."""
import random

import pytest
import torch

from auto_infer_amd import ops
from oracle import block_sparse as ref
from tests import test_gpu_block_sparse as sparse
from tests import test_gpu_shared_groups as groups
from tests import test_gpu_shared_prefix as shared

pytestmark = pytest.mark.gpu
DEV = "cuda"


def many(batch, seed, bs=16):
    """Decode and verify rows of five documents of 128 to 640 keys, and some of none."""
    rng = random.Random(seed)
    reqs, of = [], {}
    for b in range(batch):
        doc, lq = rng.choice([None, 0, 1, 2, 3, 4]), rng.choice([1, 1, 1, 2])
        reqs.append((lq, [] if doc is None else [(doc, 128 * (doc + 1))], lq + rng.randint(0, 60)))
        if doc is not None:
            of.setdefault(doc, []).append(b)
    s = groups.build(reqs, 4, 2, 64, bs, seed=seed)
    for c in "kv":
        s[c + "c"], s[c + "s"] = torch.randn(s["nb"], bs, 2, 64, generator=s["gen"]).bfloat16(), None
        s[c + "x"] = s[c + "c"].double()
    s["q"] = torch.randn(s["t"], 4, 64, generator=s["gen"]).bfloat16()
    return s, {tuple(m): 128 * (doc + 1) for doc, m in of.items()}


def check_some(s, out, some):
    """``shared.check`` of some requests."""
    for b in some:
        t0, t1 = int(s["cu"][b]), int(s["cu"][b + 1])
        one = dict(s, lens=[s["lens"][b]], table=s["table"][b:b + 1], q=s["q"][t0:t1])
        shared.check(one, out[t0:t1])


@pytest.mark.parametrize("batch", [512, 513, 1025, 1755, 1756, 4096])
def test_shared_prefixes(batch):
    s, want = many(batch, batch)
    plan = groups.plan_of(s)
    assert groups.found(s, plan) == want
    out = ops.paged_attention_shared(s["q"].to(DEV), s["kc"].to(DEV), s["vc"].to(DEV), plan, 0.125).cpu()
    assert bool(torch.isfinite(out).all())
    check_some(s, out, [0, batch - 1, *random.Random(1).sample(range(batch), 40)])


def test_more_requests_are_refused():
    with pytest.raises(NotImplementedError, match="4097 requests"):
        groups.plan_of(many(4097, 1)[0])


@pytest.mark.parametrize("batch", [600, 2048])
def test_a_shared_step_in_a_graph(batch):
    """Planned and attended on each replay, for lengths and tables that change."""
    a, b = many(batch, 3)[0], many(batch, 4)[0]
    t = max(a["t"], b["t"])
    a["q"], b["q"] = (torch.cat((s["q"], s["q"][:t - s["t"]])) for s in (a, b))
    for s in (a, b):                       # as many tokens: the last request has the rest
        extra = t - s["t"]
        s["cu"][-1] += extra
        s["lk"][-1] += extra
        lq, lk = s["lens"][-1]
        s["lens"][-1] = (lq + extra, lk + extra)
        s["t"] = t
    width = max(a["table"].shape[1], b["table"].shape[1]) + 64
    nb = max(a["nb"], b["nb"])
    names = ("table", "cu", "lk", "q", "kc", "vc")
    for s in (a, b):
        s["table"] = torch.nn.functional.pad(s["table"], (0, width - s["table"].shape[1]))
        for c in "kv":
            s[c + "c"] = torch.cat((s[c + "c"], torch.zeros(nb - s["nb"], *s[c + "c"].shape[1:], dtype=torch.bfloat16)))
            s[c + "x"] = s[c + "c"].double()
    buf = {n: a[n].to(DEV) for n in names}
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        plan = ops.SharedPrefixPlan(buf["table"], buf["cu"], buf["lk"], t, 4, 2, 64, 16)
        out = ops.paged_attention_shared(buf["q"], buf["kc"], buf["vc"], plan, 0.125)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            plan.replan()
            ops.paged_attention_shared(buf["q"], buf["kc"], buf["vc"], plan, 0.125, out=out)
        for s in (a, b, a, b):
            for n in names:
                buf[n].copy_(s[n])
            graph.replay()
            stream.synchronize()
            plan.status()
            check_some(s, out.cpu(), [0, batch - 1, *random.Random(2).sample(range(batch), 15)])


@pytest.mark.parametrize("batch", [1023, 1025, 2049, 8192])
def test_block_sparse_steps(batch):
    rng = random.Random(batch)
    lens = [(lq, lq + rng.randint(0, 150)) for lq in (rng.choice([0, 1, 1, 1, 2, 5]) for _ in range(batch))]
    s = sparse.make(lens, 4, 2, 64, 16, seed=batch, spread=False)
    g = sparse.on_gpu(s)
    plan, (bounds, scale) = sparse.make_plan(g, 4), sparse.empty_bounds(s["nb"], 2, 64)
    plan.status()
    ops.summarize_blocks(g["kc"], plan, bounds, scale)
    sel = ops.select_blocks(g["q"], plan, bounds, scale)
    touched = sorted({int(s["table"][r, i]) for r, (lq, lk) in enumerate(lens) if lq for i in range((lk - lq) // 16, (lk - 1) // 16 + 1)})
    written = (bounds != 77).any(-1).any(-1).any(-1).nonzero().flatten().tolist()
    assert written == touched
    last = [(r, lk) for r, (lq, lk) in enumerate(lens) if lq]
    for r, lk in [last[0], last[-1], *rng.sample(last, 30)]:
        blk = int(s["table"][r, (lk - 1) // 16])
        hi, nlo, e = ref.block_bounds(s["kx"][blk, :(lk - 1) % 16 + 1, 1])
        assert torch.equal(bounds[blk, 1].cpu().long(), torch.stack([hi, nlo]))
        assert int(scale.view(torch.uint8)[blk, 1]) == e + 127
    out = ops.paged_attention_sparse(g["q"], g["kc"], g["vc"], plan, sel, 0.125).cpu()
    some = {0, s["t"] - 1, *rng.sample(range(s["t"]), 40)}
    sel = sel.cpu()
    for t, _, pos in sparse.tokens_of(s):
        if t in some and pos // 16 < 4:
            n = pos // 16 + 1
            assert sel[t].tolist() == [list(range(n)) + [-1] * (4 - n)] * 2
    sparse.check_attention(s, sel, out, 0.125, some)


@pytest.mark.parametrize("rows", [False, True])
def test_selections_in_several_launches(rows):
    """1,100 tokens of one prompt, or of as many requests, over 8,192 columns and 8 heads:
    1,024 tokens' scores at once."""
    t, width, hkv, d, nb = 1100, 8192, 8, 64, 400
    assert 1024 * width * hkv == 2 ** 26
    rng, gen = random.Random(5), torch.Generator().manual_seed(5)
    table = torch.randint(0, nb, (t if rows else 1, width), generator=gen, dtype=torch.int32)
    lens = [(1, rng.randint(1, 40000)) for _ in range(t)] if rows else [(t, 30011)]
    cu = [0]
    for lq, _ in lens:
        cu.append(cu[-1] + lq)
    q = torch.randn(t, hkv, d, generator=gen).bfloat16()
    b = torch.randint(-30, 127, (nb, hkv, 2, d), generator=gen, dtype=torch.int8)
    e = torch.randint(-3, 3, (nb, hkv), generator=gen)
    plan = ops.BlockSparsePlan(table.to(DEV), torch.tensor(cu, dtype=torch.int32, device=DEV),
                               torch.tensor([lk for _, lk in lens], dtype=torch.int32, device=DEV), t, hkv, hkv, d, 16, 20, 2, 3)
    scale = (e + 127).to(torch.uint8).to(DEV).view(torch.float8_e8m0fnu)
    out = ops.select_blocks(q.to(DEV), plan, b.to(DEV), scale).cpu()
    at = {tok: (r, pos) for tok, r, pos in sparse.tokens_of(dict(lens=lens))}
    for tok in (0, 1, 511, 1022, 1023, 1024, 1025, 1098, 1099):
        r, pos = at[tok]
        ids, h = table[r].long(), rng.randrange(hkv)
        want = ref.select(q[tok, h:h + 1], b[ids, h, 0], b[ids, h, 1], e[ids, h], pos // 16 + 1, 20, 2, 3)
        assert out[tok, h].tolist() == want + [-1] * (20 - len(want)), (tok, h)
    # each token's own block is the last that is taken
    vis = torch.tensor([at[i][1] // 16 + 1 for i in range(t)])
    assert torch.equal(out.amax(-1), (vis - 1)[:, None].expand(t, hkv).int())
    assert torch.equal((out >= 0).sum(-1), vis.clamp(max=20)[:, None].expand(t, hkv))
