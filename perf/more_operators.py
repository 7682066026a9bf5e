"""Operators of serving long and shared contexts: appending to a paged cache with
the position rotation on the way, attention for a batch that shares a prefix, and
sparse attention over blocks that a cheap score selects.

Every case is one call of one operator on one layer's tensors of one step:

* ``append``: the Q and K heads of a packed qkv projection are normed (where the
  model does) and turned by their positions; K and V go to their slots of the paged
  caches, bf16 or 8-bit (e4m3 with a power of two for each block and head);
* ``shared``: paged attention of requests whose block tables begin with the same
  blocks, group by group;
* ``summary``: the 8-bit bounds of the keys of every cache block that the step
  wrote to;
* ``select``: the blocks that each query token and KV head will read, by an upper
  bound of their scores from those bounds;
* ``sparse``: paged attention over the selected blocks alone.

Head shapes are those the package is configured for elsewhere: 16/8/128, 28/4/128,
32/8/128, 64/8/128 and 14/2/64.  Lengths follow from the case alone
(``shape_seed``), values from ``prepare``'s seed.  The plain form computes in
float32 (angles and the bounds' products, which are whole numbers, in float64) and
rounds once at the end.
"""
import math
import random

import torch

own = False

DEV = "cuda"
E4M3_MAX = 448.0
MIN_EXP = -100           # smallest exponent of a block's scale
EPS = 1e-6
ROPE_BASE = 1e6

DEFAULTS = dict(op="append", hq=16, hkv=8, d=128, bs=128, rows=0, width=1, lo=1, hi=1, prompts=0,
                plo=0, phi=0, cached_hi=0, kv="bf16", groups=0, shared_lo=0, shared_hi=0, select=0,
                sink=1, local=2, rotary=0, interleaved=False, scaling="none", norm=False,
                shape_seed=1)


def _case(**kw):
    bad = set(kw) - set(DEFAULTS) - {"name"}
    assert not bad, bad
    return {**DEFAULTS, **kw}


def listed():
    return [
        # New tokens of a small decode batch: the smallest call, latency alone.
        _case(name="append_decode_b16", op="append", bs=16, rows=16, lo=100, hi=30000, norm=True,
              scaling="yarn", shape_seed=31),
        # A large model's decode batch into 8-bit caches.
        _case(name="append_decode_b128_8bit", op="append", hq=64, bs=32, rows=128, lo=100, hi=60000,
              kv="fp8", shape_seed=32),
        # Prompt chunks that begin and end inside blocks, half of each head turned.
        _case(name="append_prompts_8k", op="append", hq=28, hkv=4, prompts=5, plo=1000, phi=2300,
              cached_hi=900, rotary=64, interleaved=True, shape_seed=33),
        # A small batch behind one instruction.
        _case(name="shared_decode_b16", op="shared", bs=16, rows=16, lo=30, hi=900, groups=1,
              shared_lo=4096, shared_hi=4096, shape_seed=34),
        # Many users of a large model who ask about one long document.
        _case(name="shared_decode_b128", op="shared", hq=64, rows=128, lo=100, hi=2048, groups=1,
              shared_lo=32768, shared_hi=32768, shape_seed=35),
        # Speculative verify of samples from several prompts, 8-bit caches, head_dim 64,
        # odd lengths; a few requests share nothing.
        _case(name="shared_verify_d64_8bit", op="shared", hq=14, hkv=2, d=64, bs=16, rows=40, width=3,
              lo=3, hi=1500, groups=5, shared_lo=700, shared_hi=9000, kv="fp8", shape_seed=36),
        # Bounds after a decode step: every request's last block.
        _case(name="summary_decode_b64", op="summary", hq=32, bs=64, rows=64, lo=2000, hi=60000,
              shape_seed=37),
        # Bounds after a prompt step, small blocks.
        _case(name="summary_prompts_16k", op="summary", bs=16, prompts=8, plo=1500, phi=2500,
              cached_hi=300, shape_seed=38),
        # Decode over very long contexts: latency and the bounds' bytes.
        _case(name="select_decode_b8", op="select", hq=32, bs=32, rows=8, lo=60000, hi=131072,
              select=64, shape_seed=39),
        # One chunk of a long document, every token with blocks of its own.
        _case(name="select_chunk_at_32k", op="select", hq=28, hkv=4, bs=64, prompts=1, plo=512,
              phi=512, cached_hi=32300, select=32, shape_seed=40),
        # Attention of the two steps above.
        _case(name="sparse_decode_b8", op="sparse", hq=32, bs=32, rows=8, lo=60000, hi=131072,
              select=64, shape_seed=39),
        _case(name="sparse_chunk_at_32k", op="sparse", hq=28, hkv=4, bs=64, prompts=1, plo=512,
              phi=512, cached_hi=32300, select=32, shape_seed=40),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "shared", "shared", "summary", "select", "sparse"])
    hq, hkv, d = rng.choice([(16, 8, 128), (28, 4, 128), (32, 8, 128), (64, 8, 128), (14, 2, 64)])
    bs = rng.choice([16, 16, 32, 64, 128])
    kw = dict(op=op, hq=hq, hkv=hkv, d=d, bs=bs, kv=rng.choice(["bf16", "bf16", "fp8"]),
              shape_seed=rng.randrange(1 << 20))
    if op in ("append", "summary"):
        total = _log_int(rng, 1, 12000)
        if rng.random() < 0.5:
            lo = _log_int(rng, 1, 20000)
            kw.update(rows=min(total, 256), lo=lo, hi=3 * lo)
        else:
            phi = max(1, total // rng.choice([1, 3, 8]))
            kw.update(rows=rng.choice([0, 0, _log_int(rng, 1, 64)]), lo=1, hi=3000,
                      prompts=max(1, total // phi), plo=max(1, phi // 3), phi=phi,
                      cached_hi=rng.choice([0, 900]))
        if op == "append":
            kw.update(rotary=rng.choice([0, 0, d // 2, d // 4]), interleaved=rng.random() < 0.5,
                      scaling=rng.choice(["none", "linear", "yarn"]), norm=rng.random() < 0.5)
    elif op == "shared":
        rows, shi = _log_int(rng, 2, 128), _log_int(rng, 64, 32768)
        groups = rng.choice([1, 1, 2, max(1, rows // 7)])
        shi = min(shi, 100000 // groups)
        lo = min(_log_int(rng, 1, 1000), 60000 // rows)
        width = rng.choice([1, 1, 1, 2, 4])
        shi = min(shi, int(1.3e11 / (rows * width * hq * d * 4)))
        kw.update(rows=rows, width=width, lo=lo, hi=_log_int(rng, lo, 2 * lo + 1), groups=groups,
                  shared_hi=shi, shared_lo=max(1, shi // rng.choice([1, 1, 3])))
    else:
        kw.update(select=rng.choice([4, 16, 32, 64, 64, 100]), sink=rng.choice([0, 1, 1]),
                  local=rng.choice([1, 2, 2]))
        # a selection has something to choose from; attention takes short contexts too
        least = (kw["select"] + 3) * bs if op == "select" else 1
        if rng.random() < 0.6:
            lo = _log_int(rng, least, max(least, 60000))
            hi = min(131072, _log_int(rng, lo, 4 * lo + 1))
            kw.update(width=rng.choice([1, 1, 1, 2, 3]), lo=lo, hi=hi)
            kw["rows"] = max(1, min(_log_int(rng, 1, 64), int(1e9 / (hi * hkv * d))))
        else:
            phi = _log_int(rng, 2, 512)
            kw.update(prompts=rng.choice([1, 1, 2]), plo=max(1, phi // 2), phi=phi // 2 + 1,
                      cached_hi=_log_int(rng, max(16, least), 32000))
            if op == "select":
                kw["prompts"] = 1          # (several have cached parts from none to all)
    return _case(**kw)


# ------------------------------------------------------------------ lengths

def _shared(case):
    """(group of each request, shared keys of each group): requests of a group begin
    with the same whole blocks; group 0 shares nothing where there are several."""
    rng = random.Random(case["shape_seed"] + 3)
    n, bs = case["groups"], case["bs"]
    lens = [max(bs, rng.randint(case["shared_lo"], case["shared_hi"]) // bs * bs) for _ in range(n)]
    if n > 1:
        lens[0] = 0
    return [rng.randrange(n) for _ in range(case["rows"])], lens


def _lengths(case):
    """(new tokens, context length with them) of each request."""
    rng = random.Random(case["shape_seed"])
    out = []
    for _ in range(case["rows"]):
        out.append((case["width"], max(case["width"], rng.randint(case["lo"], case["hi"]))))
    for _ in range(case["prompts"]):
        lq = rng.randint(case["plo"], case["phi"])
        cached = case["cached_hi"] if case["prompts"] == 1 else rng.randint(0, case["cached_hi"])
        out.append((lq, lq + cached))
    if case["groups"]:       # the tails' lengths come on top of what is shared
        group, lens = _shared(case)
        out = [(lq, lk + lens[g]) for (lq, lk), g in zip(out, group)]
    return out


def _touched(case):
    """(request, logical block, keys that it holds) of each block the step wrote to."""
    bs, out = case["bs"], []
    for r, (lq, lk) in enumerate(_lengths(case)):
        out += [(r, i, min(bs, lk - i * bs)) for i in range((lk - lq) // bs, (lk - 1) // bs + 1)]
    return out


def _kept(case, nblk):
    """Blocks that a token with ``nblk`` visible ones selects."""
    return min(nblk, case["select"])


def work(case):
    hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["bs"]
    lens = _lengths(case)
    t = sum(lq for lq, _ in lens)
    cell = 1 if case["kv"] == "fp8" else 2
    if case["op"] == "append":
        rot = case["rotary"] or d
        scales = 2 * 2 * len(_touched(case)) * hkv if cell == 1 else 0
        return {"bytes": t * (2 * (2 * hq + 2 * hkv) * d + 2 * hkv * d * cell + 12) + scales,
                "flops": 3 * t * (hq + hkv) * rot}
    if case["op"] == "summary":
        keys = sum(n for _, _, n in _touched(case))
        return {"bytes": keys * hkv * d * cell + len(_touched(case)) * hkv * (2 * d + 1),
                "flops": 2 * keys * hkv * d}
    if case["op"] == "select":
        blocks = sum(-(-lk // bs) for _, lk in lens)
        pairs = sum((lk - lq + i) // bs + 1 for lq, lk in lens for i in range(lq))
        return {"bytes": 2 * t * hq * d + blocks * (hkv * (2 * d + 1) + 4) + 4 * t * hkv * case["select"],
                "flops": 2 * pairs * hq * 2 * d}
    io = 2 * 2 * t * hq * d
    if case["op"] == "sparse":
        seen, read = 0, 0
        for lq, lk in lens:
            most = 0
            for i in range(lq):
                p = lk - lq + i
                n = (_kept(case, p // bs + 1) - 1) * bs + p % bs + 1
                seen, most = seen + n, max(most, n)
            # a token's heads choose for themselves, and so does every token: at
            # least one token's keys are read, at most all
            read += min(lk, most)
        return {"bytes": io + 2 * read * hkv * d * cell + 4 * t * hkv * case["select"],
                "flops": 4 * hq * d * seen}
    group, shared = _shared(case)
    tails = sum(lk - shared[g] for (_, lk), g in zip(lens, group))
    keys = tails + sum(shared[g] for g in set(group))
    seen = sum(lq * (lk - lq) + lq * (lq + 1) // 2 for lq, lk in lens)
    return {"bytes": io + 2 * keys * hkv * d * cell, "flops": 4 * hq * d * seen}


# ------------------------------------------------------------------ inputs

def _rand(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _cache_values(gen, nb, case):
    """bf16 cache contents: a few channels of a head are much larger than the rest,
    as keys have them, and blocks differ in size and direction."""
    x = _rand(gen, nb, case["bs"], case["hkv"], case["d"])
    ch = torch.rand(case["hkv"], case["d"], generator=gen, device=DEV)
    x += _rand(gen, nb, 1, case["hkv"], case["d"])
    x *= torch.where(ch > 0.97, 5.0, 0.7)
    x *= torch.exp2(torch.randint(-2, 2, (nb, 1, case["hkv"], 1), generator=gen, device=DEV).float())
    return x.bfloat16()


def _needed_exp(amax, most):
    """Smallest e >= MIN_EXP with amax <= most * 2^e."""
    m, e = torch.frexp(amax.double() / most)       # amax / most = m 2^e, m in [0.5, 1)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.where(amax > 0, e, MIN_EXP).clamp(min=MIN_EXP).int()


def _quantised(x):
    """A bf16 cache (NB, bs, H, D) as e4m3 values and e8m0 scales (NB, H)."""
    x = x.float()
    e = _needed_exp(x.abs().amax(dim=(1, 3)), E4M3_MAX)
    q = torch.ldexp(x, -e[:, None, :, None]).to(torch.float8_e4m3fn)
    return q, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _tables(case, lens, seed):
    """Block tables, ids dealt in random order, and the number of blocks.  An append
    or a summary has only the blocks that its new rows touch."""
    bs = case["bs"]
    few = case["op"] in ("append", "summary")
    need = [-(-lk // bs) for _, lk in lens]
    group, shared = _shared(case) if case["groups"] else ([0] * len(lens), [0])
    first = [(lk - lq) // bs if few else shared[g] // bs for (lq, lk), g in zip(lens, group)]
    owned = [max(0, n - f) for n, f in zip(need, first)]
    nb = sum(owned) + sum(shared) // bs + 3
    ids = torch.randperm(nb, generator=torch.Generator().manual_seed(seed), dtype=torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32)
    at, heads = 0, []
    for n in shared:
        heads.append(ids[at:at + n // bs])
        at += n // bs
    for i, (f, n) in enumerate(zip(first, owned)):
        if not few:
            table[i, :f] = heads[group[i]]
        table[i, f:f + n] = ids[at:at + n]
        at += n
    return table, nb


def _selection(case, lens, gen):
    """Selected blocks (T, Hkv, select) of a step: the first ones, the last ones and
    others by chance, ascending, -1 behind them."""
    t, k = sum(lq for lq, _ in lens), case["select"]
    vis = torch.tensor([(lk - lq + i) // case["bs"] + 1 for lq, lk in lens for i in range(lq)], device=DEV)
    n = max(int(vis.max()), k)
    i = torch.arange(n, device=DEV)
    key = torch.rand(t, case["hkv"], n, generator=gen, device=DEV)
    v = vis[:, None, None]
    key += 2.0 * ((i < case["sink"]) | (i >= v - case["local"]))
    key.masked_fill_(i >= v, -1.0)
    top, at = key.topk(k, dim=-1)
    at = torch.where(top < 0, n, at).sort(dim=-1).values
    return torch.where(at == n, -1, at).int()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op, hq, hkv, d, bs = case["op"], case["hq"], case["hkv"], case["d"], case["bs"]
    lens = _lengths(case)
    t = sum(lq for lq, _ in lens)
    table, nb = _tables(case, lens, seed)
    s = {"case": case, "t": t, "table": table.to(DEV)}
    cu = [0]
    for lq, _ in lens:
        cu.append(cu[-1] + lq)
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
    s["lk"] = torch.tensor([lk for _, lk in lens], dtype=torch.int32, device=DEV)
    s["max_q"], s["max_k"] = max(lq for lq, _ in lens), max(lk for _, lk in lens)
    s["ks"] = s["vs"] = None
    caches = {"summary": "k", "select": ""}.get(op, "kv")
    for name in caches:
        x = _cache_values(gen, nb, case)
        s[name + "c"], s[name + "s"] = _quantised(x) if case["kv"] == "fp8" else (x, None)
    if op == "append":
        s["qkv"] = _rand(gen, t, (hq + 2 * hkv) * d).mul_(2).bfloat16()
        pos, slots = [], []
        for r, (lq, lk) in enumerate(lens):
            row = table[r].tolist()
            pos += range(lk - lq, lk)
            slots += [row[p // bs] * bs + p % bs for p in range(lk - lq, lk)]
        s["positions"] = torch.tensor(pos, device=DEV)
        s["slots"] = torch.tensor(slots, dtype=torch.int32, device=DEV)
        s["wq"] = s["wk"] = None
        if case["norm"]:
            s["wq"] = (1 + 0.2 * _rand(gen, d)).bfloat16()
            s["wk"] = (1 + 0.2 * _rand(gen, d)).bfloat16()
        s["q_out"] = torch.empty(t, hq, d, dtype=torch.bfloat16, device=DEV)
        if own:
            from auto_infer_amd import ops
            s["rope"] = ops.RotaryEmbedding(d, rotary_dim=case["rotary"] or d, base=ROPE_BASE,
                                            interleaved=case["interleaved"], scaling=_scaling(case),
                                            device=DEV)
        else:
            freq, factor = _frequencies(case)
            s["freq"], s["factor"] = freq.to(DEV), factor
        return s
    if op in ("shared", "select", "sparse"):
        s["q"] = _rand(gen, t, hq, d).bfloat16()
    if op == "shared":
        group, shared = _shared(case)
        s["group"] = torch.tensor(group, dtype=torch.int32, device=DEV)
        if not own:
            # rows of each group, one after another, -1 behind them
            of = [[] for _ in shared]
            for r, g in enumerate(group):
                of[g] += range(cu[r], cu[r + 1])
            most = max(len(x) for x in of)
            s["members"] = torch.tensor([x + [-1] * (most - len(x)) for x in of], device=DEV)
            place = [0] * t
            for g, x in enumerate(of):
                for i, tok in enumerate(x):
                    place[tok] = g * most + i
            s["place"] = torch.tensor(place, device=DEV)
            s["shared"] = torch.tensor(shared, device=DEV)
            lead = [group.index(g) if g in group else 0 for g in range(len(shared))]
            s["lead"] = torch.tensor(lead, device=DEV)
            s["max_shared"] = max(shared)
            s["max_tail"] = max(lk - shared[g] for (_, lk), g in zip(lens, group))
    if op in ("summary", "select"):
        s["bounds"] = torch.zeros(nb, hkv, 2, d, dtype=torch.int8, device=DEV)
        s["bs"] = torch.full((nb, hkv), 127, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
    if op == "summary":
        touched = _touched(case)
        s["blk"] = torch.tensor([int(table[r, i]) for r, i, _ in touched], device=DEV)
        s["held"] = torch.tensor([n for _, _, n in touched], device=DEV)
    if op == "select":
        x = torch.maximum(_rand(gen, nb, hkv, 2, d), _rand(gen, nb, hkv, 2, d)) + 0.3
        x[:, :, 1] = torch.maximum(x[:, :, 1], -x[:, :, 0])       # a least value up to the largest
        x *= torch.exp2(torch.randint(-1, 2, (nb, hkv, 1, 1), generator=gen, device=DEV).float())
        e = _needed_exp(x.abs().amax(dim=(2, 3)), 127)
        s["bounds"] = torch.ldexp(x, -e[:, :, None, None]).ceil_().to(torch.int8)
        s["bs"] = (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    if op == "sparse":
        s["selected"] = _selection(case, lens, gen)
    if own:
        from auto_infer_amd import ops
        # the step's plan, which a program makes once for all its layers
        args = (s["table"], s["cu"], s["lk"], t, hq, hkv, d, bs)
        if op == "shared":
            s["plan"] = ops.SharedPrefixPlan(*args, group_ids=s["group"])
        else:
            s["plan"] = ops.BlockSparsePlan(*args, num_selected=max(1, case["select"]),
                                            sink=min(case["sink"], max(0, case["select"] - case["local"])),
                                            local=case["local"] if case["select"] else 1)
    return s


# ------------------------------------------------------------------ append

def _scaling(case):
    if case["scaling"] == "linear":
        return {"type": "linear", "factor": 4.0}
    if case["scaling"] == "yarn":
        return {"type": "yarn", "factor": 32.0, "original_max_position": 32768}
    return None


def _frequencies(case):
    """Angle per position of each rotated pair (float64) and the factor on cos and
    sin.  The frequency-dependent scaling leaves pairs that turn more than 32 times
    within the original context, divides those that turn less than once by the factor
    and ramps in between."""
    dim = case["rotary"] or case["d"]
    freq = ROPE_BASE ** -(torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    sc = _scaling(case)
    if sc is None:
        return freq, 1.0
    if sc["type"] == "linear":
        return freq / sc["factor"], 1.0
    n = sc["original_max_position"]

    def pair(turns):     # the (fractional) pair that turns so often within n positions
        return dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(ROPE_BASE))
    lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), dim - 1)
    ramp = ((torch.arange(dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    return (freq / sc["factor"] * ramp + freq * (1 - ramp),
            0.1 * math.log(sc["factor"]) + 1.0)


def _rotated(x, w, cos, sin, interleaved):
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.to(x.dtype)
    half = cos.shape[-1]
    rot, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
    else:
        a, b = rot[..., :half], rot[..., half:]
    c, d = a * cos - b * sin, b * cos + a * sin
    rot = torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)
    return torch.cat((rot, rest), -1)


def _write_8bit(x, cache, scale, slots):
    """The plain form of one 8-bit cache's write, in place: over the whole pool, blocks
    without a new row keep what they hold."""
    nb, bs, h, d = cache.shape
    blk = (slots // bs).long()
    new = x.float()
    amax = torch.zeros(nb, h, device=DEV).index_reduce_(0, blk, new.abs().amax(-1), "amax")
    is_new = torch.zeros(nb * bs, dtype=torch.bool, device=DEV)
    is_new[slots.long()] = True
    is_new = is_new.view(nb, bs)
    old = scale.view(torch.uint8).int() - 127
    need = _needed_exp(amax, E4M3_MAX)
    # a block whose first slot is written starts anew
    e = torch.where(is_new[:, :1], need, torch.maximum(old, need))
    e = torch.where(is_new.any(1, keepdim=True), e, old)
    keep = torch.where(is_new[:, :1], torch.zeros_like(e), old - e)
    held = torch.ldexp(cache.float(), keep[:, None, :, None])
    held.view(nb * bs, h, d)[slots.long()] = torch.ldexp(new, -e[blk][:, :, None])
    cache.copy_(held.to(torch.float8_e4m3fn))
    scale.view(torch.uint8).copy_((e + 127).to(torch.uint8))


def _run_append(s):
    case = s["case"]
    hq, hkv, d, t = case["hq"], case["hkv"], case["d"], s["t"]
    if own:
        from auto_infer_amd import ops
        q = ops.rope_append(s["qkv"], hq, hkv, s["positions"], s["rope"], s["kc"], s["vc"], s["slots"],
                            s["wq"], s["wk"], EPS, q_out=s["q_out"], key_scale=s["ks"],
                            value_scale=s["vs"])
    else:
        angle = s["positions"].double()[:, None] * s["freq"]
        cos = (angle.cos() * s["factor"]).float()[:, None]
        sin = (angle.sin() * s["factor"]).float()[:, None]
        x = s["qkv"].float()
        q = _rotated(x[:, :hq * d].view(t, hq, d), s["wq"], cos, sin, case["interleaved"]).bfloat16()
        k = _rotated(x[:, hq * d:(hq + hkv) * d].view(t, hkv, d), s["wk"], cos, sin,
                     case["interleaved"]).bfloat16()
        v = s["qkv"][:, (hq + hkv) * d:].view(t, hkv, d)
        if case["kv"] == "fp8":
            _write_8bit(k, s["kc"], s["ks"], s["slots"])
            _write_8bit(v, s["vc"], s["vs"], s["slots"])
        else:
            s["kc"].view(-1, hkv, d)[s["slots"].long()] = k
            s["vc"].view(-1, hkv, d)[s["slots"].long()] = v
    out = {"q": q, "key_cache": s["kc"], "value_cache": s["vc"]}
    if case["kv"] == "fp8":
        out.update(key_scale=s["ks"], value_scale=s["vs"])
    return out


# ------------------------------------------------------------------ attention

def _values(cache, scale, blocks):
    """Cache blocks as float32 (..., bs, H, D)."""
    x = cache[blocks].float()
    if scale is not None:
        e = scale.view(torch.uint8)[blocks].int() - 127
        x = torch.ldexp(x, e[..., None, :, None])
    return x


def _part(x, v):
    """(largest score, sum of exponentials, weighted values) of masked scores x."""
    top = x.amax(-1, keepdim=True).clamp_(min=-3e38)
    x = x.sub_(top).exp_()
    return top, x.sum(-1, keepdim=True), torch.matmul(x, v)


def _run_shared(s):
    case = s["case"]
    hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["bs"]
    if own:
        from auto_infer_amd import ops
        return ops.paged_attention_shared(s["q"], s["kc"], s["vc"], s["plan"], d ** -0.5,
                                          key_scale=s["ks"], value_scale=s["vs"])
    g, t, nt = hq // hkv, s["t"], s["max_tail"]
    cu, lk = s["cu"].long(), s["lk"].long()
    lq = cu[1:] - cu[:-1]
    req = torch.repeat_interleave(torch.arange(lq.shape[0], device=DEV), lq, output_size=t)
    at = torch.arange(t, device=DEV) - cu[req]
    # what is shared, once for all rows of a group: (G, Hkv, rows * g, keys)
    sh, ng = s["shared"], s["shared"].shape[0]
    width = max(1, s["max_shared"] // bs)
    table = s["table"][s["lead"]][:, :width].long()
    k, v = (_values(s[c + "c"], s[c + "s"], table).flatten(1, 2).transpose(1, 2) for c in "kv")
    q = s["q"][s["members"].clamp(min=0)].float().view(ng, -1, hkv, g, d).permute(0, 2, 1, 3, 4).flatten(2, 3)
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(d ** -0.5)
    hidden = torch.arange(x.shape[-1], device=DEV) >= sh[:, None]
    top, total, o = (y.view(ng, hkv, -1, g, y.shape[-1]).transpose(1, 2).flatten(0, 1)[s["place"]]
                     for y in _part(x.masked_fill_(hidden[:, None, None], float("-inf")), v))
    # what each request has on its own
    first = sh[s["group"].long()]
    nblk = -(-nt // bs)
    cols = (first // bs)[:, None] + torch.arange(nblk, device=DEV)
    table = s["table"].gather(1, cols.clamp(max=s["table"].shape[1] - 1)).long()
    k, v = (_values(s[c + "c"], s[c + "s"], table).flatten(1, 2).transpose(1, 2) for c in "kv")
    i = torch.arange(s["max_q"], device=DEV)
    rows = torch.minimum(cu[:-1, None] + i, cu[1:, None] - 1)
    q = s["q"][rows].float().view(-1, s["max_q"], hkv, g, d).permute(0, 2, 1, 3, 4).flatten(2, 3)
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(d ** -0.5)
    hidden = torch.arange(x.shape[-1], device=DEV) > (lk - lq - first)[:, None, None] + i[:, None]
    hidden = hidden[:, :, None].expand(-1, -1, g, -1).flatten(1, 2)
    part = (y.view(-1, hkv, s["max_q"], g, y.shape[-1])[req, :, at]
            for y in _part(x.masked_fill_(hidden[:, None], float("-inf")), v))
    # joined
    top2, total2, o2 = part
    most = torch.maximum(top, top2)
    a, b = (top - most).exp(), (top2 - most).exp()
    total = a * total + b * total2
    o = (a * o + b * o2) / torch.where(total > 0, total, 1.0)
    return o.view(t, hq, d).bfloat16()


def _run_sparse(s):
    case = s["case"]
    hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["bs"]
    if own:
        from auto_infer_amd import ops
        return ops.paged_attention_sparse(s["q"], s["kc"], s["vc"], s["plan"], s["selected"], d ** -0.5,
                                          key_scale=s["ks"], value_scale=s["vs"])
    g, t = hq // hkv, s["t"]
    cu, lk = s["cu"].long(), s["lk"].long()
    lq = cu[1:] - cu[:-1]
    req = torch.repeat_interleave(torch.arange(lq.shape[0], device=DEV), lq, output_size=t)
    pos = (lk - lq)[req] + torch.arange(t, device=DEV) - cu[req]
    sel = s["selected"].long()                                           # (T, Hkv, K)
    blocks = s["table"].long()[req[:, None, None], sel.clamp(min=0)]
    head = torch.arange(hkv, device=DEV)[None, :, None]

    def rows(cache, scale):                                              # (T, Hkv, K bs, D)
        x = cache.transpose(1, 2)[blocks, head].float()
        if scale is not None:
            x = torch.ldexp(x, (scale.view(torch.uint8)[blocks, head].int() - 127)[..., None, None])
        return x.flatten(2, 3)
    k, v = rows(s["kc"], s["ks"]), rows(s["vc"], s["vs"])
    x = torch.matmul(s["q"].float().view(t, hkv, g, d), k.transpose(-1, -2)).mul_(d ** -0.5)
    key = sel[..., None] * bs + torch.arange(bs, device=DEV)
    hidden = ((sel < 0)[..., None] | (key > pos[:, None, None, None])).flatten(2, 3)
    _, total, o = _part(x.masked_fill_(hidden[:, :, None], float("-inf")), v)
    return (o / torch.where(total > 0, total, 1.0)).view(t, hq, d).bfloat16()


# ------------------------------------------------------------------ selection

def _run_summary(s):
    case = s["case"]
    if own:
        from auto_infer_amd import ops
        ops.summarize_blocks(s["kc"], s["plan"], s["bounds"], s["bs"], key_scale=s["ks"])
    else:
        x = _values(s["kc"], s["ks"], s["blk"])                          # (n, bs, H, D)
        behind = torch.arange(case["bs"], device=DEV)[:, None, None] >= s["held"][:, None, None, None]
        top = x.masked_fill(behind, float("-inf")).amax(1)
        low = x.neg_().masked_fill_(behind, float("-inf")).amax(1)
        both = torch.stack((top, low), 2)                                # (n, H, 2, D)
        e = _needed_exp(both.amax((2, 3)), 127)
        s["bounds"][s["blk"]] = torch.ldexp(both, -e[:, :, None, None]).ceil_().to(torch.int8)
        s["bs"].view(torch.uint8)[s["blk"]] = (e + 127).to(torch.uint8)
    return {"bounds": s["bounds"], "scale": s["bs"].view(torch.uint8)}


def _run_select(s):
    case = s["case"]
    if own:
        from auto_infer_amd import ops
        return ops.select_blocks(s["q"], s["plan"], s["bounds"], s["bs"])
    hq, hkv, d, bs, n = case["hq"], case["hkv"], case["d"], case["bs"], case["select"]
    g, t = hq // hkv, s["t"]
    cu, lk = s["cu"].long(), s["lk"].long()
    lq = cu[1:] - cu[:-1]
    req = torch.repeat_interleave(torch.arange(lq.shape[0], device=DEV), lq, output_size=t)
    at = torch.arange(t, device=DEV) - cu[req]
    vis = ((lk - lq)[req] + at) // bs + 1
    i = torch.arange(s["max_q"], device=DEV)
    rows = torch.minimum(cu[:-1, None] + i, cu[1:, None] - 1)
    q = s["q"].float().view(t, hkv, g * d)
    e = _needed_exp(q.abs().amax(-1), 127)
    q = torch.ldexp(q, -e[:, :, None]).round_().view(t, hkv, g, d)
    q = torch.stack((q.clamp(min=0).sum(2), (-q).clamp_(min=0).sum(2)), 2)[rows]   # (B, nq, Hkv, 2, D)
    table = s["table"].long()
    x = s["bounds"][table].permute(0, 2, 3, 4, 1).flatten(2, 3).double()           # (B, Hkv, 2 D, N)
    x = torch.matmul(q.flatten(3, 4).transpose(1, 2).double(), x)                  # (B, Hkv, nq, N)
    e = s["bs"].view(torch.uint8)[table].int().transpose(1, 2) - 127
    x = torch.ldexp(x.float(), e[:, :, None]).transpose(1, 2)[req, at]             # (T, Hkv, N)
    j = torch.arange(x.shape[-1], device=DEV)
    v = vis[:, None, None]
    always = (j < case["sink"]) | (j >= v - case["local"])
    x = torch.where(always, float("inf"), x).masked_fill_(j >= v, float("-inf"))
    order = x.sort(dim=-1, descending=True, stable=True).indices[..., :n]
    if order.shape[-1] < n:
        order = torch.nn.functional.pad(order, (0, n - order.shape[-1]), value=x.shape[-1])
    order = torch.where(order >= v, x.shape[-1], order).sort(dim=-1).values
    return torch.where(order == x.shape[-1], -1, order).int()


def run(state):
    return {"append": _run_append, "shared": _run_shared, "summary": _run_summary,
            "select": _run_select, "sparse": _run_sparse}[state["case"]["op"]](state)


# ------------------------------------------------------------------ 64 bits

def _exact_write(x, cache, scale, slots):
    """A cache's values and scales after the write, the new rows' before their last
    rounding."""
    nb, bs, h, d = cache.shape
    val, exp = cache.double(), scale.view(torch.uint8).long() - 127
    place = torch.full((nb * bs,), -1, dtype=torch.long, device=DEV)
    place[slots.long()] = torch.arange(slots.shape[0], device=DEV)
    place = place.view(nb, bs)
    for i in torch.unique(slots // bs).tolist():
        here = place[i] >= 0
        rows = x[place[i][here]]                                # (n, H, D)
        top = rows.bfloat16().double().abs().amax(dim=(0, 2))
        need = torch.ceil(torch.log2(top / 448.0) - 1e-12).long()
        need = torch.where(top <= 448.0 * 2.0 ** MIN_EXP, MIN_EXP, need)
        new = need if bool(here[0]) else torch.maximum(exp[i], need)
        if not bool(here[0]):
            val[i] *= torch.exp2((exp[i] - new).double())[None, :, None]
        val[i][here] = rows * torch.exp2(-new.double())[None, :, None]
        exp[i] = new
    return val, torch.exp2(exp.double())


def _exact_append(case, s):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    freq, factor = _frequencies(case)
    pos = s["positions"].double().cpu()
    z = torch.polar(torch.full((len(pos), len(freq)), float(factor), dtype=torch.float64),
                    pos[:, None] * freq)[:, None].to(DEV)
    half, turned = len(freq), []
    for x, w in ((s["qkv"][:, :hq * d], s["wq"]), (s["qkv"][:, hq * d:(hq + hkv) * d], s["wk"])):
        x = x.double().view(len(pos), -1, d).clone()
        if w is not None:
            x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
        if case["interleaved"]:
            first, second = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
        else:
            first, second = slice(0, half), slice(half, 2 * half)
        r = torch.complex(x[..., first], x[..., second]) * z
        x[..., first], x[..., second] = r.real, r.imag
        turned.append(x)
    q, k = turned
    v = s["qkv"][:, (hq + hkv) * d:].double().view(len(pos), hkv, d)
    if case["kv"] == "fp8":
        kc, ks = _exact_write(k, s["kc"], s["ks"], s["slots"])
        vc, vs = _exact_write(v, s["vc"], s["vs"], s["slots"])
        return {"q": q, "key_cache": kc, "value_cache": vc, "key_scale": ks, "value_scale": vs}
    kc, vc = s["kc"].double(), s["vc"].double()
    kc.view(-1, hkv, d)[s["slots"].long()] = k
    vc.view(-1, hkv, d)[s["slots"].long()] = v
    return {"q": q, "key_cache": kc, "value_cache": vc}


def _context(s, r, lk):
    """A request's keys and values in 64 bits, (lk, Hkv, D) each."""
    bs = s["case"]["bs"]
    blocks = s["table"][r, :-(-lk // bs)].long()
    out = []
    for c in "kv":
        x = s[c + "c"][blocks].double()
        if s[c + "s"] is not None:
            x = x * 2.0 ** (s[c + "s"].view(torch.uint8)[blocks].double() - 127)[:, None, :, None]
        out.append(x.flatten(0, 1)[:lk])
    return out


def _exact_attention(case, s):
    hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["bs"]
    out = torch.zeros(s["t"], hq, d, dtype=torch.float64, device=DEV)
    g, at = hq // hkv, 0
    for r, (lq, lk) in enumerate(_lengths(case)):
        k, v = _context(s, r, lk)
        pos = torch.arange(lk - lq, lk, device=DEV)[:, None]
        key = torch.arange(lk, device=DEV)[None]
        for h in range(hkv):
            hidden = key > pos
            if case["op"] == "sparse":
                sel = s["selected"][at:at + lq, h].long()
                mine = torch.zeros(lq, -(-lk // bs) + 1, dtype=torch.bool, device=DEV)
                mine.scatter_(1, torch.where(sel < 0, mine.shape[1] - 1, sel), True)
                hidden = hidden | ~mine[:, :-1].repeat_interleave(bs, 1)[:, :lk]
            q = s["q"][at:at + lq, h * g:(h + 1) * g].double().transpose(0, 1)     # (g, lq, d)
            x = torch.matmul(q, k[:, h].t().contiguous()) / math.sqrt(d)
            p = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1)
            out[at:at + lq, h * g:(h + 1) * g] = torch.matmul(p, v[:, h]).transpose(0, 1)
        at += lq
    return out


def _exact_summary(case, s):
    bounds, scale = s["bounds"].long(), s["bs"].view(torch.uint8).long()
    for r, i, n in _touched(case):
        b = int(s["table"][r, i])
        x = s["kc"][b, :n].double()
        if s["ks"] is not None:
            x = x * 2.0 ** (s["ks"].view(torch.uint8)[b].double() - 127)[None, :, None]
        most = x.abs().amax((0, 2))
        e = torch.full_like(most, MIN_EXP)
        while bool((most > 127 * 2.0 ** e).any()):
            e = e + (most > 127 * 2.0 ** e)
        step = (2.0 ** e)[:, None]
        bounds[b] = torch.stack((torch.ceil(x.amax(0) / step), -torch.floor(x.amin(0) / step)), 1).long()
        scale[b] = (e + 127).long()
    return {"bounds": bounds, "scale": scale}


def _exact_select(case, s):
    hq, hkv, bs, n = case["hq"], case["hkv"], case["bs"], case["select"]
    g, at = hq // hkv, 0
    out = torch.full((s["t"], hkv, n), -1, dtype=torch.int32, device=DEV)
    for r, (lq, lk) in enumerate(_lengths(case)):
        blocks = s["table"][r, :-(-lk // bs)].long()
        size = 2.0 ** (s["bs"].view(torch.uint8)[blocks].double() - 127)           # (N, Hkv)
        vis = torch.arange(lk - lq, lk, device=DEV)[:, None] // bs + 1
        j = torch.arange(len(blocks), device=DEV)[None]
        always = (j < case["sink"]) | (j >= vis - case["local"])
        for h in range(hkv):
            top, low = (s["bounds"][blocks, h, x].double() for x in (0, 1))        # (N, D)
            q = s["q"][at:at + lq, h * g:(h + 1) * g].double()                     # (lq, g, d)
            unit = 2.0 ** _needed_exp(q.abs().amax((1, 2)), 127).double()
            q = torch.round(q / unit[:, None, None])
            total = torch.zeros(lq, len(blocks), dtype=torch.float64, device=DEV)
            for x in q.unbind(1):
                for c in range(0, lq, 64):
                    y = x[c:c + 64, None]
                    total[c:c + 64] += torch.maximum(y * top, -y * low).sum(-1)
            score = (total.float().double() * size[None, :, h]).masked_fill(always, math.inf)
            score = score.masked_fill(j >= vis, -math.inf)
            order = torch.argsort(score, dim=-1, descending=True, stable=True)[:, :n]
            order = torch.where(order >= vis, 1 << 30, order).sort(dim=-1).values
            out[at:at + lq, h, :order.shape[1]] = torch.where(order == 1 << 30, -1, order).int()
        at += lq
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "summary":
        return _exact_summary(case, s)
    return _exact_select(case, s) if case["op"] == "select" else _exact_attention(case, s)
