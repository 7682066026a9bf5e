"""Block-sparse attention on the GPU against restatements in 64 bits: bounds and
selections bit for bit, attention within the roundings' bound."""
import random

import pytest
import torch

from oracle import block_sparse as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(lens, hq, hkv, d, bs, fp8=False, seed=0, extra=2, spread=True):
    """A step's tensors: lens = [(new tokens, context), ...]."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-lk // bs) for _, lk in lens]
    nb = sum(need) + extra
    ids = torch.randperm(nb, generator=gen, dtype=torch.int32)
    table = torch.zeros(len(lens), max(1, *need) + 1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    kc = torch.randn(nb, bs, hkv, d, generator=gen)
    vc = torch.randn(nb, bs, hkv, d, generator=gen)
    if spread:
        kc += torch.randn(nb, 1, hkv, d, generator=gen)
        kc *= torch.exp2(torch.randint(-3, 3, (nb, 1, hkv, 1), generator=gen).float())
    t = sum(lq for lq, _ in lens)
    s = dict(lens=lens, hq=hq, hkv=hkv, d=d, bs=bs, nb=nb, t=t, table=table,
             q=torch.randn(t, hq, d, generator=gen).bfloat16(), ks=None, vs=None)
    cu = [0]
    for lq, _ in lens:
        cu.append(cu[-1] + lq)
    s["cu"] = torch.tensor(cu, dtype=torch.int32)
    s["lk"] = torch.tensor([lk for _, lk in lens], dtype=torch.int32)
    if fp8:
        for name, x in (("k", kc), ("v", vc)):
            e = torch.randint(-4, 3, (nb, hkv), generator=gen)
            s[name + "c"] = x.to(torch.float8_e4m3fn)
            s[name + "s"] = (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
            s[name + "x"] = s[name + "c"].double() * torch.exp2(e.double())[:, None, :, None]
    else:
        s["kc"], s["vc"] = kc.bfloat16(), vc.bfloat16()
        s["kx"], s["vx"] = s["kc"].double(), s["vc"].double()
    return s


def on_gpu(s):
    return {k: v.to(DEV) if isinstance(v, torch.Tensor) and k not in ("kx", "vx") else v for k, v in s.items()}


def make_plan(g, selected, sink=1, local=1, **kw):
    from auto_infer_amd import ops
    return ops.BlockSparsePlan(g["table"], g["cu"], g["lk"], g["t"], g["hq"], g["hkv"], g["d"], g["bs"],
                               num_selected=selected, sink=sink, local=local, **kw)


def empty_bounds(nb, hkv, d):
    return (torch.full((nb, hkv, 2, d), 77, dtype=torch.int8, device=DEV),
            torch.full((nb, hkv), 33, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu))


def tokens_of(s):
    """(token, request, position) of each query token."""
    t = 0
    for r, (lq, lk) in enumerate(s["lens"]):
        for i in range(lq):
            yield t, r, lk - lq + i
            t += 1


SHAPES = [(16, 8, 128), (28, 4, 128), (14, 2, 64), (8, 8, 64), (6, 2, 128), (64, 2, 64), (5, 1, 128), (32, 1, 128)]
STEPS = {
    "decode": [(1, 1), (1, 700), (1, 16), (1, 17), (1, 333)],
    "verify": [(3, 3), (3, 500), (2, 129), (4, 64)],
    "prompt": [(70, 70), (33, 600), (1, 5)],
    "empty_request": [(0, 40), (2, 90), (0, 0), (1, 260)],
}


@pytest.mark.parametrize("bs", [1, 7, 16, 64, 128])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (14, 2, 64), (5, 1, 128), (6, 6, 64)])
@pytest.mark.parametrize("step", sorted(STEPS))
def test_bounds(step, hq, hkv, d, fp8, bs):
    from auto_infer_amd import ops
    s = make(STEPS[step], hq, hkv, d, bs, fp8, seed=bs + d)
    g = on_gpu(s)
    bounds, scale = empty_bounds(s["nb"], hkv, d)
    plan = make_plan(g, 4)
    ops.summarize_blocks(g["kc"], plan, bounds, scale, key_scale=g["ks"])
    b, e = bounds.cpu(), scale.view(torch.uint8).cpu().int() - 127
    want, wante = torch.full_like(b, 77), torch.full_like(e, 33 - 127)
    for r, (lq, lk) in enumerate(s["lens"]):
        if lq == 0 or lk == 0:
            continue
        for i in range((lk - lq) // bs, (lk - 1) // bs + 1):
            blk = int(s["table"][r, i])
            for h in range(hkv):
                hi, nlo, x = ref.block_bounds(s["kx"][blk, :min(bs, lk - i * bs), h])
                want[blk, h, 0], want[blk, h, 1], wante[blk, h] = hi, nlo, x
    assert torch.equal(b, want) and torch.equal(e, wante)


def test_bounds_of_odd_values():
    """Zeros, subnormals, infinities and NaN; slots behind the request's end are not read."""
    from auto_infer_amd import ops
    bs, d = 16, 64
    s = make([(16, 16)] * 6 + [(3, 3)], 1, 1, d, bs, seed=3)
    k = s["kc"]
    blk = s["table"][:, 0].tolist()
    k[blk[0]] = 0
    k[blk[1]] *= 2.0 ** -130
    k[blk[2], 3, 0, 5] = float("inf")
    k[blk[2], 4, 0, 6] = -float("inf")
    k[blk[2], 5, 0, 7] = float("nan")
    k[blk[3]] = float("nan")
    k[blk[4], 0] = 3.3e38
    k[blk[5]] = 1.0
    k[blk[5], 1, 0, 0] = 127.5            # not held by 127 units of 1
    k[blk[6], 3:] = float("nan")
    s["kx"] = k.double()
    g = on_gpu(s)
    bounds, scale = empty_bounds(s["nb"], 1, d)
    ops.summarize_blocks(g["kc"], make_plan(g, 4), bounds, scale)
    for r, (_, lk) in enumerate(s["lens"]):
        hi, nlo, e = ref.block_bounds(s["kx"][blk[r], :lk, 0])
        assert torch.equal(bounds[blk[r], 0, 0].cpu().long(), hi), r
        assert torch.equal(bounds[blk[r], 0, 1].cpu().long(), nlo), r
        assert int(scale.view(torch.uint8)[blk[r], 0]) - 127 == e, r


def random_bounds(s, seed, ties=False):
    gen = torch.Generator().manual_seed(seed)
    b = torch.randint(-127, 128, (s["nb"], s["hkv"], 2, s["d"]), generator=gen)
    b[:, :, 1] = torch.maximum(b[:, :, 1], -b[:, :, 0])
    e = torch.randint(-3, 2, (s["nb"], s["hkv"]), generator=gen)
    if ties:                             # a few different blocks, repeated
        b, e = b[torch.arange(s["nb"]) % 3], e[torch.arange(s["nb"]) % 3]
    return b.to(torch.int8), e


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("step", sorted(STEPS))
def test_selection(step, hq, hkv, d, ties):
    from auto_infer_amd import ops
    bs = 7
    s = make(STEPS[step], hq, hkv, d, bs, seed=hq)
    b, e = random_bounds(s, 5, ties)
    g = on_gpu(s)
    for selected, sink, local in ((1, 0, 1), (5, 1, 2), (24, 2, 1)):
        out = ops.select_blocks(g["q"], make_plan(g, selected, sink, local), b.to(DEV),
                                (e + 127).to(torch.uint8).to(DEV).view(torch.float8_e8m0fnu)).cpu()
        for t, r, pos in tokens_of(s):
            vis = max(0, pos // bs + 1)
            rows = s["table"][r].long()
            for h in range(hkv):
                q = s["q"][t, h * (hq // hkv):(h + 1) * (hq // hkv)]
                want = ref.select(q, b[rows, h, 0], b[rows, h, 1], e[rows, h], vis, selected, sink, local)
                assert out[t, h].tolist() == want + [-1] * (selected - len(want)), (t, h)


@pytest.mark.parametrize("most", [200, 300, 600, 900, 1500, 4097, 9000])
def test_selection_of_long_contexts(most):
    """Many blocks per row (every kernel that selects), values of the query that are not
    finite, strided queries."""
    from auto_infer_amd import ops
    s = make([(1, most), (2, 3 * most // 4 + 1)], 4, 2, 128, 1, seed=9)
    s["q"][0, 0, 3], s["q"][0, 1, 4], s["q"][1] = float("inf"), float("nan"), 0.0
    b, e = random_bounds(s, 6)
    g = on_gpu(s)
    wide = torch.zeros(s["t"], 9, 128, dtype=torch.bfloat16, device=DEV)
    wide[:, 2:6] = g["q"]
    out = ops.select_blocks(wide[:, 2:6], make_plan(g, 150, 3, 5), b.to(DEV),
                            (e + 127).to(torch.uint8).to(DEV).view(torch.float8_e8m0fnu)).cpu()
    for t, r, pos in tokens_of(s):
        rows = s["table"][r].long()
        for h in range(2):
            want = ref.select(s["q"][t, 2 * h:2 * h + 2], b[rows, h, 0], b[rows, h, 1], e[rows, h], pos + 1, 150, 3, 5)
            assert out[t, h].tolist() == want


@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_selection_of_prompts(hq, hkv, d):
    """Many tokens per request: tiles of several tokens, and of several requests."""
    from auto_infer_amd import ops
    s = make([(61, 300), (0, 9), (37, 37), (1, 200), (50, 90)], hq, hkv, d, 3, seed=hq + 1)
    b, e = random_bounds(s, 8)
    g = on_gpu(s)
    out = ops.select_blocks(g["q"], make_plan(g, 9, 1, 2), b.to(DEV),
                            (e + 127).to(torch.uint8).to(DEV).view(torch.float8_e8m0fnu)).cpu()
    for t, r, pos in tokens_of(s):
        if t % 5 and t not in (60, 61, 97, 98, 99):
            continue
        rows = s["table"][r].long()
        for h in range(hkv):
            q = s["q"][t, h * (hq // hkv):(h + 1) * (hq // hkv)]
            want = ref.select(q, b[rows, h, 0], b[rows, h, 1], e[rows, h], pos // 3 + 1, 9, 1, 2)
            assert out[t, h].tolist() == want + [-1] * (9 - len(want)), (t, h)


def random_selection(s, selected, seed):
    rng = random.Random(seed)
    out = torch.full((s["t"], s["hkv"], selected), -1, dtype=torch.int32)
    for t, r, pos in tokens_of(s):
        vis = max(0, pos // s["bs"] + 1)
        for h in range(s["hkv"]):
            n = rng.randint(0, min(vis, selected))
            out[t, h, :n] = torch.tensor(sorted(rng.sample(range(vis), n)), dtype=torch.int32)
    return out


def check_attention(s, sel, out, scale, tokens=None):
    """Within the roundings: weights and the output are rounded to bf16 (2^-8 relative
    each), parts of a row to fp16 (2^-11 of the part's largest value, at most the
    largest |v|), so |error| <= 2^-8 sum p |v| + 2^-8 |out| + 2^-11 max |v|; the float32
    sums and exponentials are allowed as much again."""
    hq, hkv, bs = s["hq"], s["hkv"], s["bs"]
    for t, r, pos in tokens_of(s):
        if tokens is not None and t not in tokens:
            continue
        rows = s["table"][r].long()
        n = max(0, pos + 1)
        nblk = -(-n // bs)
        k, v = (s[c][rows[:nblk]].flatten(0, 1)[:n] for c in ("kx", "vx"))
        for h in range(hkv):
            seen = torch.zeros(n, dtype=torch.bool)
            top = -1
            for e in sel[t, h].tolist():
                if e > top and e >= 0 and e * bs < n:
                    seen[e * bs:(e + 1) * bs] = True
                top = max(top, e)
            for j in range(hq // hkv):
                head = h * (hq // hkv) + j
                want = ref.attention(s["q"][t, head], k[:, h], v[:, h], seen, scale)
                size = ref.attention(s["q"][t, head], k[:, h], v[:, h].abs(), seen, scale)
                most = float(v[seen, h].abs().max()) if bool(seen.any()) else 0.0
                bound = 2.0 ** -7 * (size + want.abs()) + 2.0 ** -10 * most + 1e-30
                assert bool(((out[t, head].double() - want).abs() <= bound).all()), (t, head)


@pytest.mark.parametrize("bs", [1, 16, 24, 128])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("step", sorted(STEPS))
def test_attention(step, hq, hkv, d, fp8, bs):
    from auto_infer_amd import ops
    s = make(STEPS[step], hq, hkv, d, bs, fp8, seed=hq + bs, spread=False)
    g = on_gpu(s)
    selected = {1: 90, 16: 20, 24: 9, 128: 3}[bs]
    sel = random_selection(s, selected, 7)
    out = ops.paged_attention_sparse(g["q"], g["kc"], g["vc"], make_plan(g, selected), sel.to(DEV), d ** -0.5,
                                     key_scale=g["ks"], value_scale=g["vs"])
    check_attention(s, sel, out.cpu(), d ** -0.5)


def test_entries_that_do_not_ascend_are_left_out():
    from auto_infer_amd import ops
    s = make([(1, 100), (1, 40)], 4, 2, 64, 16, seed=2, spread=False)
    g = on_gpu(s)
    sel = torch.tensor([[[0, 0, 2, 1, 6], [3, -1, 4, 4, 9]], [[2, 2, 1, 0, -1], [5, 1, 0, -1, 2]]], dtype=torch.int32)
    out = ops.paged_attention_sparse(g["q"], g["kc"], g["vc"], make_plan(g, 5), sel.to(DEV), 0.125)
    check_attention(s, sel, out.cpu(), 0.125)
    assert bool((out[1, 2:] == 0).all())          # its first entry is not visible and hides the others


@pytest.mark.parametrize("fp8", [False, True])
def test_values_that_are_not_finite_stay_where_they_are_seen(fp8):
    from auto_infer_amd import ops
    bs, d = 16, 128
    s = make([(1, 90), (1, 90)], 4, 2, d, bs, fp8, seed=4, spread=False)
    bad = float("nan")
    table = s["table"]
    for r in range(2):
        for c in ("kc", "vc"):
            x = s[c].view(torch.uint8) if fp8 else s[c]
            x[int(table[r, 5]), 10:] = 0x7f if fp8 else bad       # behind the requests' ends
            x[int(table[r, 3])] = 0x7f if fp8 else bad            # a block that is not selected
    x = s["vc"].view(torch.uint8) if fp8 else s["vc"]
    x[int(table[1, 5]), 9, 1, 7] = 0x7f if fp8 else float("inf")  # the second request's last key
    g = on_gpu(s)
    sel = torch.tensor([0, 1, 5], dtype=torch.int32, device=DEV).expand(2, 2, 3)
    out = ops.paged_attention_sparse(g["q"], g["kc"], g["vc"], make_plan(g, 3), sel, d ** -0.5,
                                     key_scale=g["ks"], value_scale=g["vs"]).cpu()
    odd = ~torch.isfinite(out)
    want = torch.zeros_like(odd)
    want[1, 2:, 7] = True
    assert torch.equal(odd, want)
    if not fp8:
        assert bool((out[1, 2:, 7] == float("inf")).all())


def test_split_rows_equal_long_lists():
    """Few rows with long lists are cut over several work-groups."""
    from auto_infer_amd import ops
    s = make([(1, 9000)], 8, 1, 128, 32, seed=5, spread=False)
    g = on_gpu(s)
    sel = random_selection(s, 250, 8)
    sel[0, 0] = torch.arange(250, dtype=torch.int32) + 31
    out = ops.paged_attention_sparse(g["q"], g["kc"], g["vc"], make_plan(g, 250), sel.to(DEV), 128 ** -0.5)
    check_attention(s, sel, out.cpu(), 128 ** -0.5)


@pytest.mark.parametrize("hq,hkv,d,bs,fp8", [(4, 2, 128, 16, False), (7, 1, 128, 64, True), (40, 2, 64, 32, False),
                                             (6, 3, 64, 128, True), (2, 2, 128, 24, False)])
def test_long_chunks_take_the_context_in_ranges(hq, hkv, d, bs, fp8):
    from auto_infer_amd import ops
    s = make([(90, 13000), (3, 9001), (40, 40)], hq, hkv, d, bs, fp8, seed=11, spread=False)
    g = on_gpu(s)
    selected = 1500 // bs
    sel = random_selection(s, selected, 9)
    sel[5] = -1                                       # a token without a block
    sel[6, :, 1:] = -1                                # and with one
    out = ops.paged_attention_sparse(g["q"], g["kc"], g["vc"], make_plan(g, selected), sel.to(DEV), d ** -0.5,
                                     key_scale=g["ks"], value_scale=g["vs"]).cpu()
    assert bool((out[5] == 0).all())
    check_attention(s, sel, out, d ** -0.5, tokens=set(range(0, 95, 7)) | {5, 6, 89, 90, 92, 93, 132})


def test_chunks_of_several_launches():
    from auto_infer_amd import ops
    s = make([(1700, 7000)], 16, 16, 64, 16, seed=12, spread=False)
    g = on_gpu(s)
    gen = torch.Generator().manual_seed(1)
    sel = torch.rand(1700, 16, 270, generator=gen).topk(20, dim=-1).indices.sort(-1).values.int()
    out = ops.paged_attention_sparse(g["q"], g["kc"], g["vc"], make_plan(g, 20), sel.to(DEV), 0.125).cpu()
    check_attention(s, sel, out, 0.125, tokens={0, 1, 511, 512, 900, 1023, 1024, 1400, 1699})


def test_tokens_that_no_request_covers():
    from auto_infer_amd import ops
    s = make([(2, 50)], 4, 2, 64, 16, seed=6, spread=False)
    g = on_gpu(s)
    g["t"] = 5
    g["q"] = torch.randn(5, 4, 64, device=DEV).bfloat16()
    b, e = random_bounds(s, 6)
    plan = make_plan(g, 2)
    sel = ops.select_blocks(g["q"], plan, b.to(DEV), (e + 127).to(torch.uint8).to(DEV).view(torch.float8_e8m0fnu))
    assert bool((sel[2:] == -1).all()) and bool((sel[:2] >= 0).all())
    out = ops.paged_attention_sparse(g["q"], g["kc"], g["vc"], plan, sel, 0.125)
    assert bool((out[2:] == 0).all()) and bool((out[:2] != 0).any())
