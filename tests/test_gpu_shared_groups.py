"""What the shared-prefix planner finds: which requests form a group, how many keys it
reads once for them, and which rows go with it.  (The results of the attention do not
depend on it, so they cannot show it.)"""
import random

import pytest
import torch

from tests import test_gpu_shared_prefix as shared

pytestmark = pytest.mark.gpu
DEV = "cuda"
MIN, TILE, UNIT = 128, 64, 128


def build(reqs, hq, hkv, d, bs, ids=None, seed=0, pad=1):
    """reqs: [(new tokens, [(name, keys), ...], own keys with the new ones), ...].  Keys of
    one name and place stand in the same blocks (so a name's keys are whole blocks)."""
    rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
    named, lens, rows, total = {}, [], [], 0
    for lq, parts, own in reqs:
        row, path = [], ()
        for name, n in parts:
            assert n % bs == 0
            path = (*path, name)
            kept = named.setdefault(path, [])
            while len(kept) < n // bs:
                kept.append(total)
                total += 1
            row += kept[:n // bs]
        lk = len(row) * bs + own
        own = -(-lk // bs) - len(row)
        rows.append(row + list(range(total, total + own)))
        total += own
        lens.append((lq, lk))
    ids_of = list(range(total))
    rng.shuffle(ids_of)
    table = torch.zeros(len(rows), max(map(len, rows)) + pad, dtype=torch.int32)
    for i, r in enumerate(rows):
        table[i, :len(r)] = torch.tensor([ids_of[b] for b in r], dtype=torch.int32)
    t, cu = sum(lq for lq, _ in lens), [0]
    for lq, _ in lens:
        cu.append(cu[-1] + lq)
    return dict(lens=lens, hq=hq, hkv=hkv, d=d, bs=bs, t=t, table=table, nb=total, ids=ids,
                cu=torch.tensor(cu, dtype=torch.int32), lk=torch.tensor([lk for _, lk in lens], dtype=torch.int32), gen=gen)


def plan_of(s):
    from auto_infer_amd import ops
    ids = None if s["ids"] is None else torch.tensor(s["ids"], dtype=torch.int32, device=DEV)
    plan = ops.SharedPrefixPlan(s["table"].to(DEV), s["cu"].to(DEV), s["lk"].to(DEV), s["t"], s["hq"], s["hkv"], s["d"],
                                s["bs"], group_ids=ids)
    plan.status()
    return plan


def found(s, plan):
    """{(members of a group): shared keys}, and the tokens in the order of its rows, as the
    plan's workspace has them: header, then per request its group's first one, the keys in
    common, its place; per token {request, index, first request, place}; the order; per
    group and request {first part, rows, first key, end key, first token, cuts, ..}."""
    B, T, ws = len(s["lens"]), s["t"], plan.workspace.cpu()
    at, out = 256, {}
    for name, n in (("lead", B), ("common", B), ("place", B), ("tokreq", 4 * T), ("order", T), ("ent", 16 * B)):
        out[name] = ws[at:at + 4 * n].view(torch.int32)
        at += (4 * n + 255) // 256 * 256
    lead, ent = out["lead"].tolist(), out["ent"].view(2 * B, 8)
    groups, orders = {}, {}
    for g in sorted(set(lead) - {-1}):
        _, rows, k0, k1, base = ent[g, :5].tolist()
        members = tuple(b for b in range(B) if lead[b] == g)
        assert members[0] == g and k0 == 0
        if rows == 0:
            continue
        tokens = [t for b in members for t in range(int(s["cu"][b]), int(s["cu"][b + 1]))]
        assert rows == len(tokens) * (s["hq"] // s["hkv"])
        orders[members] = out["order"][base:base + len(tokens)].tolist()
        assert orders[members] == tokens
        groups[members] = k1
    for b, (lq, lk) in enumerate(s["lens"]):       # each request's own keys follow
        keys = next((k for m, k in groups.items() if b in m), 0)
        _, rows, k0, k1, base = ent[B + b, :5].tolist()
        assert (rows, k1, base) == (lq * (s["hq"] // s["hkv"]), lk, int(s["cu"][b])) and k0 == min(keys, lk)
    return groups


def expected(s):
    """The rule, restated: a request's level is that of the most keys times requests that
    agree with it so far; requests of one level and block share what all of them have."""
    B, bs, group = len(s["lens"]), s["bs"], s["hq"] // s["hkv"]
    ids = s["ids"] or s["table"][:, 0].tolist()
    cached = [lk - lq if 0 < lq * group < UNIT and lk > lq and (s["ids"] is None or s["ids"][b] >= 0) else 0
              for b, (lq, lk) in enumerate(s["lens"])]

    def block(b, level):
        return int(s["table"][b, ((MIN << level) - 1) // bs])
    level = []
    for b in range(B):
        agree = []
        for o in range(B):
            far = 0
            if o != b and ids[o] == ids[b]:
                while (MIN << far) <= min(cached[b], cached[o]) and block(b, far) == block(o, far):
                    far += 1
            agree.append(far)
        saved = [(MIN << i) * sum(f > i for f in agree) for i in range(max(agree, default=0))]
        level.append(max(i for i, x in enumerate(saved) if x == max(saved)) if saved else -1)
    groups = {}
    for b in range(B):
        if level[b] >= 0:
            groups.setdefault((ids[b], level[b], block(b, level[b])), []).append(b)
    out = {}
    for members in groups.values():
        common = []
        for b in members:
            n = -(-cached[b] // bs)
            same = (s["table"][b, :n] == s["table"][members[0], :n]).tolist() + [False]
            common.append(min(cached[b], same.index(False) * bs))
        keys = min(common) // TILE * TILE
        if len(members) > 1 and keys >= MIN:
            out[tuple(members)] = keys
    return out


def check(s, want=None):
    got = found(s, plan_of(s))
    assert got == expected(s)
    if want is not None:
        assert got == want
    return got


DOC = [("doc", 4096)]
HEADS = dict(hq=16, hkv=8, d=64)


@pytest.mark.parametrize("bs", [16, 64, 128])
def test_all_requests_of_a_document(bs):
    check(build([(1, DOC, 1 + 37 * i) for i in range(9)], bs=bs, **HEADS), {tuple(range(9)): 4096})


@pytest.mark.parametrize("bs", [16, 64, 128])
@pytest.mark.parametrize("at", [0, 7, 15])
@pytest.mark.parametrize("odd", [(1, [("doc", 128)], 3000), (1, [("doc", 128)], 1), (1, [("doc", 512)], 40), (1, [], 60)])
def test_a_request_with_little_in_common_leaves_the_others_their_prefix(odd, at, bs):
    """In front of them, among them and behind them."""
    reqs = [(1, DOC, 1 + 5 * i) for i in range(15)]
    reqs.insert(at, odd)
    s = build(reqs, bs=bs, **HEADS)
    check(s, {tuple(b for b in range(16) if b != at): 4096})
    check({**s, "ids": [3] * 16}, {tuple(b for b in range(16) if b != at): 4096})


@pytest.mark.parametrize("bs", [16, 64, 128])
def test_a_request_in_the_first_block_only(bs):
    reqs = [(1, DOC, 9)] * 15 + [(1, [("doc", bs)], 5000)]
    check(build(reqs, bs=bs, **HEADS), {tuple(range(15)): 4096})


def test_families_behind_one_beginning():
    """They share by family where that saves more, else the beginning."""
    def step(system, first, second):
        return build([(1, [("system", system), (f"doc{i % 2}", (first, second)[i % 2])], 3 + i) for i in range(12)], bs=16, **HEADS)
    odd, even = tuple(range(1, 12, 2)), tuple(range(0, 12, 2))
    check(step(1024, 8192, 6144), {even: 9216, odd: 7168})
    check(step(4096, 512, 256), {tuple(range(12)): 4096})


@pytest.mark.parametrize("keys,want", [(0, 0), (64, 0), (112, 0), (127, 0), (128, 128), (144, 128), (191, 128), (192, 192)])
def test_from_128_keys_on_in_whole_tiles(keys, want):
    """127 keys: blocks of one key."""
    bs = 16 if keys % 16 == 0 else 1
    s = build([(2, [("p", keys)], 30), (1, [("p", keys)], 50), (1, [("p", keys)], 1)], bs=bs, **HEADS)
    check(s, {(0, 1, 2): want} if want else {})


def test_requests_of_a_whole_unit_do_not_share():
    reqs = [(1, DOC, 4), (63, DOC, 70), (64, DOC, 70), (3, DOC, 3), (200, DOC, 300)]
    check(build(reqs, bs=64, **HEADS), {(0, 1, 3): 4096})
    check(build(reqs, 28, 4, 128, 64), {(0, 3): 4096})


def test_group_ids():
    """They split what the tables would join; negative ones stand alone."""
    s = build([(1, DOC, 4 + i) for i in range(8)], bs=64, **HEADS)
    check({**s, "ids": [-1] * 8}, {})
    check({**s, "ids": list(range(8))}, {})
    check({**s, "ids": [0, 1, 0, 1, -1, 0, -7, 2]}, {(0, 2, 5): 4096, (1, 3): 4096})
    two = build([(1, [(f"doc{i % 2}", 1024)], 4 + i) for i in range(8)], bs=64, **HEADS)
    check({**two, "ids": [0] * 8}, {(0, 2, 4, 6): 1024, (1, 3, 5, 7): 1024})
    check(two, {(0, 2, 4, 6): 1024, (1, 3, 5, 7): 1024})


def test_new_tokens_are_not_shared():
    """Copies of one request: its last keys are new."""
    s = build([(3, DOC, 3), (3, DOC, 70)], bs=64, **HEADS)
    s["table"][0] = s["table"][1]
    check(s, {(0, 1): 4096})
    s["lk"][0], s["lens"][0] = 4096, (3, 4096)
    check(s, {(0, 1): 4032})


@pytest.mark.parametrize("name", sorted(shared.STEPS))
@pytest.mark.parametrize("hq,hkv,d,bs", [(16, 8, 128, 16), (28, 4, 128, 64), (14, 2, 64, 128)])
def test_steps_of_the_attention_tests(hq, hkv, d, bs, name):
    s = shared.make(shared.STEPS[name], hq, hkv, d, bs, seed=bs)
    s["ids"] = None
    check(s)
    check({**s, "ids": s["groups"].tolist()})


@pytest.mark.parametrize("seed", range(12))
def test_drawn_trees(seed):
    """Requests at random places of a tree of prefixes, and their attention."""
    rng = random.Random(seed)
    bs = rng.choice([1, 16, 64, 128])
    reqs = []
    for _ in range(rng.randint(2, 30)):
        parts = [(rng.randint(0, 2), bs * rng.choice([0, 1, 128 // bs, 300 // bs + 1, 1000 // bs + 1])) for _ in range(rng.randint(0, 3))]
        lq = rng.choice([1, 1, 1, 2, 5, 70])
        reqs.append((lq, [(n, k) for n, k in parts if k], lq + rng.randint(0, 400)))
    s = build(reqs, *rng.choice([(16, 8, 64), (28, 4, 128), (10, 2, 128)]), bs, seed=seed)
    if seed % 3 == 0:
        s["ids"] = [rng.randint(-1, 2) for _ in reqs]
    check(s)
    for c in "kv":
        x = torch.randn(s["nb"], bs, s["hkv"], s["d"], generator=s["gen"])
        s[c + "c"], s[c + "s"] = x.bfloat16(), None
        s[c + "x"] = s[c + "c"].double()
    s["q"] = torch.randn(s["t"], s["hq"], s["d"], generator=s["gen"]).bfloat16()
    s["groups"] = torch.tensor(s["ids"] or [0], dtype=torch.int32)
    out, _ = shared.run(s, by_id=s["ids"] is not None)
    shared.check(s, out)
