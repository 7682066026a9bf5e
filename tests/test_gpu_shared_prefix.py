"""Attention with shared prefixes on the GPU against plain attention in 64 bits."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(groups, hq, hkv, d, bs, fp8=False, seed=0, shuffle=True):
    """groups: [(shared keys, [(new tokens, own keys with them), ...]), ...].  Requests
    come in random order; a group's rows begin with the same blocks."""
    gen = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    reqs = [(g, lq, n) for g, (_, members) in enumerate(groups) for lq, n in members]
    if shuffle:
        rng.shuffle(reqs)
    need = sum(s // bs for s, _ in groups) + sum(-(-(n + groups[g][0] % bs) // bs) + 1 for g, _, n in reqs) + 2
    ids = torch.randperm(need, generator=gen).tolist()
    heads = [[ids.pop() for _ in range(s // bs)] for s, _ in groups]
    lens, rows = [], []
    for g, lq, n in reqs:
        lk = groups[g][0] // bs * bs + n
        lens.append((lq, lk))
        rows.append(heads[g] + [ids.pop() for _ in range(-(-lk // bs) - len(heads[g]))])
    width = max(1, max(len(r) for r in rows) + 1)
    table = torch.zeros(len(rows), width, dtype=torch.int32)
    for i, r in enumerate(rows):
        table[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
    t = sum(lq for lq, _ in lens)
    cu = [0]
    for lq, _ in lens:
        cu.append(cu[-1] + lq)
    s = dict(lens=lens, hq=hq, hkv=hkv, d=d, bs=bs, t=t, table=table, ks=None, vs=None,
             groups=torch.tensor([g for g, _, _ in reqs], dtype=torch.int32),
             cu=torch.tensor(cu, dtype=torch.int32), lk=torch.tensor([lk for _, lk in lens], dtype=torch.int32),
             q=torch.randn(t, hq, d, generator=gen).bfloat16())
    for c in "kv":
        x = torch.randn(need, bs, hkv, d, generator=gen)
        if fp8:
            e = torch.randint(-2, 2, (need, hkv), generator=gen)
            s[c + "c"], s[c + "s"] = x.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
            s[c + "x"] = s[c + "c"].double() * torch.exp2(e.double())[:, None, :, None]
        else:
            s[c + "c"] = x.bfloat16()
            s[c + "x"] = s[c + "c"].double()
    return s


def run(s, scale=None, by_id=True, out=None, **kw):
    from auto_infer_amd import ops
    g = {k: v.to(DEV) if isinstance(v, torch.Tensor) and k not in ("kx", "vx") else v for k, v in s.items()}
    plan = ops.SharedPrefixPlan(g["table"], g["cu"], g["lk"], g["t"], g["hq"], g["hkv"], g["d"], g["bs"],
                                group_ids=g["groups"] if by_id else None, **kw)
    plan.status()
    out = ops.paged_attention_shared(g["q"], g["kc"], g["vc"], plan, scale or g["d"] ** -0.5, out=out,
                                     key_scale=g["ks"], value_scale=g["vs"])
    return out.cpu(), plan


def check(s, out, scale=None):
    """Weights are rounded to bf16 (2^-8 relative at most), the parts of a row to fp16
    (2^-11 of the largest value of the part's row, here at most 6) and the output to
    bf16: |error| <= 2^-8 (sum p |v| + |out|) + 2^-11 * 6, and half of that again for
    the float32 sums and exponentials."""
    scale = scale or s["d"] ** -0.5
    gq, at = s["hq"] // s["hkv"], 0
    for r, (lq, lk) in enumerate(s["lens"]):
        blocks = s["table"][r, :-(-lk // s["bs"])].long()
        k, v = (s[c + "x"][blocks].flatten(0, 1)[:lk] for c in "kv")
        hidden = torch.arange(lk)[None] > (lk - lq + torch.arange(lq))[:, None]
        for h in range(s["hkv"]):
            q = s["q"][at:at + lq, h * gq:(h + 1) * gq].double().transpose(0, 1)
            x = (q @ k[:, h].t() * scale).masked_fill(hidden, float("-inf"))
            p = torch.softmax(x, -1).nan_to_num(0.0)
            want, size = (p @ v[:, h]).transpose(0, 1), (p @ v[:, h].abs()).transpose(0, 1)
            bound = 1.5 * (2.0 ** -8 * (size + want.abs()) + 6 * 2.0 ** -11)
            err = (out[at:at + lq, h * gq:(h + 1) * gq].double() - want).abs()
            assert bool((err <= bound).all()), (r, lq, lk, h, float(err.max()))
        at += lq


SHAPES = [(16, 8, 128), (28, 4, 128), (14, 2, 64), (64, 8, 128), (5, 1, 128), (6, 3, 64), (10, 5, 64), (32, 1, 128)]
STEPS = {
    "one_group": [(512, [(1, n) for n in (1, 30, 17, 200, 64, 1, 5)])],
    "groups": [(0, [(1, 40), (1, 300)]), (256, [(1, 3), (1, 90), (2, 70)]), (130, [(3, 3), (1, 1)]),
               (700, [(1, 9)]), (200, [(4, 20), (2, 2), (1, 128)])],
    "verify": [(384, [(3, 3 + 7 * i) for i in range(11)])],
    "prompts": [(320, [(1, 5), (40, 60), (150, 150), (1, 64), (17, 33)])],
    "many": [(192, [(1, 1 + 3 * i) for i in range(70)])],
    "none": [(0, [(1, 1)]), (0, [(2, 100)]), (0, [(0, 60)]), (128, [(0, 10), (1, 10)])],
}


@pytest.mark.parametrize("bs", [1, 16, 24, 64, 128])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("step", sorted(STEPS))
def test_attention(step, hq, hkv, d, fp8, bs):
    s = make(STEPS[step], hq, hkv, d, bs, fp8, seed=bs + hq)
    out, _ = run(s)
    check(s, out)


@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 128), (32, 1, 128), (14, 2, 64), (28, 4, 64)])
def test_long_prefix_in_many_cuts(hq, hkv, d):
    """Rows of many parts, few rows (joined by four waves each) and many."""
    groups = [(6000, [(1, 100 + i) for i in range(40)]), (3000, [(2, 50 + i) for i in range(9)])]
    for g in (groups, groups[1:]):
        s = make(g, hq, hkv, d, 16, seed=1)
        out, _ = run(s)
        check(s, out)


def test_groups_by_first_block_or_wrong_groups_give_the_same():
    """What is shared follows from the block tables, whatever the groups say."""
    s = make(STEPS["groups"], 8, 2, 64, 16, seed=2)
    want, _ = run(s)
    check(s, want)
    out, _ = run(s, by_id=False)
    check(s, out)
    for ids in (torch.zeros_like(s["groups"]), torch.full_like(s["groups"], -1), torch.arange(len(s["groups"])).int() // 2):
        out, _ = run({**s, "groups": ids})
        check(s, out)


def test_keys_of_new_tokens_are_not_shared():
    """Rows that agree up to and into the new tokens' blocks: copies of one request."""
    s = make([(320, [(3, 70)])], 8, 2, 128, 16, seed=3)
    for k in ("table", "lk"):
        s[k] = torch.cat((s[k], s[k]))
    s["lens"] = s["lens"] * 2
    s["groups"] = torch.zeros(2, dtype=torch.int32)
    s["cu"] = torch.tensor([0, 3, 6], dtype=torch.int32)
    s["t"], s["q"] = 6, torch.randn(6, 8, 128).bfloat16()
    out, _ = run(s)
    check(s, out)


def test_rows_that_do_not_see_a_value_keep_clear_of_it():
    """NaN behind the requests' ends, and in the last new key: only its row sees it."""
    for fp8 in (False, True):
        s = make([(256, [(3, 40), (3, 40), (1, 9), (30, 50)])], 8, 2, 128, 16, fp8, seed=4, shuffle=False)
        v = s["vc"].view(torch.uint8) if fp8 else s["vc"]
        bad = 0x7f if fp8 else float("nan")
        last = []
        at = 0
        for r, (lq, lk) in enumerate(s["lens"]):
            v[int(s["table"][r, (lk - 1) // 16]), (lk - 1) % 16:] = bad
            at += lq
            last.append(at - 1)
        out, _ = run(s)
        nan = ~torch.isfinite(out).flatten(1).all(1)
        assert nan.nonzero().flatten().tolist() == last
        clean = torch.ones(s["t"], dtype=torch.bool)
        clean[last] = False
        assert bool(torch.isfinite(out[clean]).all())


def test_lengths_that_do_not_describe_the_step_give_nan():
    from auto_infer_amd import ops
    s = make([(256, [(1, 40), (1, 20)])], 8, 2, 64, 16, seed=5)
    g = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    for cu in ([0, 1, 3], [0, 2, 1], [1, 1, 2]):
        plan = ops.SharedPrefixPlan(g["table"], torch.tensor(cu, dtype=torch.int32, device=DEV), g["lk"], 2, 8, 2, 64, 16)
        out = ops.paged_attention_shared(g["q"], g["kc"], g["vc"], plan, 0.125)
        assert bool(out.isnan().all())
        with pytest.raises(ValueError, match="does not describe"):
            plan.status()


def test_strided_query_and_output():
    s = make(STEPS["groups"], 8, 2, 128, 16, seed=6)
    s["q"] = torch.randn(s["t"], 12, 128).bfloat16()[:, 2:10]
    out = torch.full((s["t"], 9, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    got, _ = run({**s, "q": s["q"]}, out=out[:, 1:])
    check(s, got)
    assert bool((out[:, 0] == 7).all())
