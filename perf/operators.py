"""Operators of long-context serving: an 8-bit KV cache, the attention that
reads it, attention with modified scores, and rotary positions.

Every case is one call of one operator on one layer's tensors of one step:

* ``write``: new K/V rows into paged caches of e4m3 values with one
  power-of-two scale (e8m0) per cache block and head;
* ``attn``: paged attention over such caches (``kv="fp8"``), or with scores
  that are capped by a tanh, get a linear distance bias or see a prefix in
  both directions, over bf16 or 8-bit caches;
* ``rope``: (optional) per-head norms and rotary positions of a packed qkv
  projection, from positions rather than tables.

Head shapes are those the package is configured for elsewhere: 16/8/128,
28/4/128, 32/8/128, 64/8/128 and 14/2/64.  Lengths follow from the case alone
(``shape_seed``), values from ``prepare``'s seed.  The plain form computes in
float32 (angles in float64) and rounds once at the end.
"""
import math
import random

import torch

own = False

DEV = "cuda"
E4M3_MAX = 448.0
MIN_EXP = -100           # smallest exponent of a block scale
EPS = 1e-6

DEFAULTS = dict(op="attn", hq=16, hkv=8, d=128, bs=128, rows=0, width=1, lo=128, hi=2048,
                prompts=0, plo=0, phi=0, cached_hi=0, kv="bf16", cap=0.0, alibi=False,
                prefix=False, tokens=0, rotary=0, interleaved=False, scaling="none", norm=False,
                pos_hi=0, shape_seed=1)


def _case(**kw):
    bad = set(kw) - set(DEFAULTS) - {"name"}
    assert not bad, bad
    return {**DEFAULTS, **kw}


def listed():
    return [
        # New rows of a small decode batch, each somewhere inside its
        # request's last block: the smallest call, latency alone.
        _case(name="write_decode_b16", op="write", bs=16, rows=16, shape_seed=11),
        # A whole scheduler budget of prompt tokens: bandwidth.
        _case(name="write_prefill_16k", op="write", prompts=8, plo=2048, phi=2048, shape_seed=12),
        # Ragged prompt chunks that start and end inside blocks beside decode
        # rows, head_dim 64, small blocks.
        _case(name="write_ragged_d64", op="write", hq=14, hkv=2, d=64, bs=16, rows=33, prompts=7,
              plo=37, phi=1900, cached_hi=700, shape_seed=13),
        # Decode over 8-bit caches at a small batch.
        _case(name="fp8_decode_b16", rows=16, lo=128, hi=2048, kv="fp8", shape_seed=14),
        # A large model's decode batch: the bandwidth-bound extreme.
        _case(name="fp8_decode_b128", hq=64, rows=128, lo=1024, hi=8192, kv="fp8", bs=16,
              shape_seed=15),
        # One chunk of a long document: 512 tokens behind 32K cached ones.
        _case(name="fp8_chunk_at_32k", hq=28, hkv=4, prompts=1, plo=512, phi=512, cached_hi=32256,
              kv="fp8", shape_seed=16),
        # Speculative verify of two drafts per request, head_dim 64, odd
        # lengths, blocks of 16.
        _case(name="fp8_verify_d64", hq=14, hkv=2, d=64, bs=16, rows=24, width=3, lo=300, hi=5000,
              kv="fp8", shape_seed=17),
        # Decode of a model that caps its attention scores.
        _case(name="cap_decode_b64", hq=32, rows=64, lo=512, hi=4096, bs=32, cap=50.0,
              shape_seed=18),
        # New prompts of a model without rotary positions: a distance bias.
        _case(name="alibi_prompts", prompts=5, plo=37, phi=1500, bs=16, alibi=True, shape_seed=19),
        # Prompts whose first part (an image, an instruction) sees itself in
        # both directions, scores capped.
        _case(name="prefix_prompts_cap", hq=28, hkv=4, prompts=3, plo=600, phi=2000, prefix=True,
              cap=30.0, shape_seed=20),
        # Rotary positions of a decode step far into a context stretched by
        # frequency-dependent scaling.
        _case(name="rope_decode_b16", op="rope", tokens=16, scaling="yarn", norm=True,
              pos_hi=1 << 20, shape_seed=21),
        # The same for a prompt step, half of each head rotated, interleaved.
        _case(name="rope_prefill_8k", op="rope", hq=28, hkv=4, tokens=8192, rotary=64,
              interleaved=True, pos_hi=8192, shape_seed=22),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "attn", "attn", "attn", "attn", "rope"])
    hq, hkv, d = rng.choice([(16, 8, 128), (28, 4, 128), (32, 8, 128), (64, 8, 128), (14, 2, 64)])
    kw = dict(op=op, hq=hq, hkv=hkv, d=d, bs=rng.choice([16, 16, 32, 64, 128, 128]),
              shape_seed=rng.randrange(1 << 20))
    if op == "write":
        total = _log_int(rng, 1, 16384)
        if rng.random() < 0.5:
            kw["rows"] = min(total, 256)
        else:
            phi = max(1, total // rng.choice([1, 3, 8]))
            kw.update(rows=rng.choice([0, 0, _log_int(rng, 1, 64)]), prompts=max(1, total // phi),
                      plo=max(1, phi // 3), phi=phi, cached_hi=rng.choice([0, 900]))
    elif op == "attn":
        kw["kv"] = rng.choice(["fp8", "fp8", "bf16"])
        kw["cap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
        kw["alibi"] = rng.random() < 0.3
        kw["prefix"] = rng.random() < 0.3
        if kw["kv"] == "bf16" and not (kw["alibi"] or kw["prefix"]):
            kw["cap"] = kw["cap"] or 50.0
        if rng.random() < 0.55:
            lo = _log_int(rng, 1, 4096)
            hi = min(16384, _log_int(rng, lo, 16 * lo + 1))
            kw.update(width=rng.choice([1, 1, 1, 2, 3, 4]), lo=lo, hi=hi)
            kw["rows"] = max(1, min(_log_int(rng, 1, 128), int(5e8 / (hi * hkv * d))))
        else:
            phi = _log_int(rng, 9, 3000)
            n = max(1, min(_log_int(rng, 1, 8), 6000 // phi))
            room = max(0, int(4e8 / (n * hq * phi)) - phi)   # padded scores of the plain form
            kw.update(prompts=n, plo=max(1, phi // rng.choice([1, 2, 8])), phi=phi,
                      cached_hi=min(room, rng.choice([0, 0, 700, _log_int(rng, 512, 12000)])))
    else:
        kw.update(tokens=_log_int(rng, 1, 8192), rotary=rng.choice([0, 0, d // 2, d // 4]),
                  interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "yarn"]),
                  norm=rng.random() < 0.5, pos_hi=_log_int(rng, 2048, 1 << 20))
    return _case(**kw)


# ------------------------------------------------------------------ lengths

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
    return out


def _prefix_lengths(case):
    """Prefix of each request: none, part of the prompt or all of it."""
    rng = random.Random(case["shape_seed"] + 7)
    return [rng.choice([0, lk // 3, lk // 2, lk, rng.randint(0, lk)]) for _, lk in _lengths(case)]


def _visible(case):
    """Keys seen by all query tokens of the step, summed."""
    pre = _prefix_lengths(case) if case["prefix"] else [0] * len(_lengths(case))
    total = 0
    for (lq, lk), p in zip(_lengths(case), pre):
        first = lk - lq + 1                       # keys the first token sees
        p = min(p, lk)
        causal = lq * (first + lk) // 2
        short = max(0, min(lq, p - first))        # tokens that see the prefix instead
        total += causal + short * p - short * (2 * first + short - 1) // 2
    return total


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "rope":
        t, rot = case["tokens"], case["rotary"] or d
        return {"bytes": t * (2 * 2 * (hq + hkv) * d + 8), "flops": 3 * t * (hq + hkv) * rot}
    lens = _lengths(case)
    tokens = sum(lq for lq, _ in lens)
    if case["op"] == "write":
        blocks = sum((lk - 1) // case["bs"] - (lk - lq) // case["bs"] + 1 for lq, lk in lens)
        return {"bytes": tokens * (2 * hkv * d * 3 + 4) + 2 * blocks * hkv,
                "flops": 2 * tokens * hkv * d}
    keys = sum(lk for _, lk in lens)
    cell = 1 if case["kv"] == "fp8" else 2
    blocks = sum(-(-lk // case["bs"]) for _, lk in lens)
    scales = 2 * blocks * hkv if case["kv"] == "fp8" else 0
    return {"bytes": 2 * keys * hkv * d * cell + scales + 4 * blocks + 2 * 2 * tokens * hq * d,
            "flops": 4 * d * hq * _visible(case)}


# ------------------------------------------------------------------ inputs

def _rand(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _cache_values(gen, nb, case):
    """bf16 cache contents: a few channels of a head are much larger than the
    rest, as keys have them, and blocks differ in size."""
    x = _rand(gen, nb, case["bs"], case["hkv"], case["d"])
    ch = torch.rand(case["hkv"], case["d"], generator=gen, device=DEV)
    x *= torch.where(ch > 0.97, 6.0, 0.8)
    x *= torch.exp2(torch.randint(-2, 3, (nb, 1, case["hkv"], 1), generator=gen, device=DEV).float())
    return x.bfloat16()


def _needed_exp(amax):
    """Smallest e >= MIN_EXP with amax <= 448 * 2^e."""
    m, e = torch.frexp(amax / E4M3_MAX)            # amax / 448 = m 2^e, m in [0.5, 1)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.where(amax > 0, e, MIN_EXP).clamp(min=MIN_EXP).int()


def _quantised(x):
    """A bf16 cache (NB, bs, H, D) as e4m3 values and e8m0 scales (NB, H)."""
    x = x.float()
    e = _needed_exp(x.abs().amax(dim=(1, 3)))
    q = torch.ldexp(x, -e[:, None, :, None]).to(torch.float8_e4m3fn)
    return q, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["bs"]
    s = {"case": case}
    if case["op"] == "rope":
        t = case["tokens"]
        s["qkv"] = _rand(gen, t, (hq + 2 * hkv) * d).mul_(2).bfloat16()
        s["positions"] = torch.randint(0, case["pos_hi"], (t,), generator=gen, device=DEV)
        if case["norm"]:
            s["wq"] = (1 + 0.2 * _rand(gen, d)).bfloat16()
            s["wk"] = (1 + 0.2 * _rand(gen, d)).bfloat16()
        s["q_out"] = torch.empty(t, hq, d, dtype=torch.bfloat16, device=DEV)
        s["k_out"] = torch.empty(t, hkv, d, dtype=torch.bfloat16, device=DEV)
        if own:
            from auto_infer_amd import ops
            s["rope"] = ops.RotaryEmbedding(d, rotary_dim=case["rotary"] or d, base=ROPE_BASE,
                                            interleaved=case["interleaved"],
                                            scaling=_scaling(case), device=DEV)
        else:
            freq, factor = _frequencies(case)
            s["freq"], s["factor"] = freq.to(DEV), factor
        return s
    lens = _lengths(case)
    # blocks are dealt in random order, a few of the pool stay unused
    need = [-(-lk // bs) for _, lk in lens]
    if case["op"] == "write":      # only the blocks that the new rows touch
        need = [n - (lk - lq) // bs for n, (lq, lk) in zip(need, lens)]
    nb = sum(need) + 3
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.zeros(len(lens), max(need), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(perm[at:at + n], dtype=torch.int32)
        at += n
    if case["op"] == "write":
        k, v = (_cache_values(gen, nb, case) for _ in range(2))
        s["kc"], s["ks"] = _quantised(k)
        s["vc"], s["vs"] = _quantised(v)
        t = sum(lq for lq, _ in lens)
        # the new rows' own spread: larger than the cached ones' now and then
        grow = torch.exp2(torch.randint(-2, 4, (t, 1, 1), generator=gen, device=DEV).float())
        s["k"] = (_rand(gen, t, hkv, d) * grow).bfloat16()
        s["v"] = (_rand(gen, t, hkv, d) * grow).bfloat16()
        slots = []
        for i, (lq, lk) in enumerate(lens):
            off = (lk - lq) % bs
            row = table[i].tolist()
            slots += [row[p // bs] * bs + p % bs for p in range(off, off + lq)]
        s["slots"] = torch.tensor(slots, dtype=torch.int32, device=DEV)
        return s
    k, v = (_cache_values(gen, nb, case) for _ in range(2))
    if case["kv"] == "fp8":
        s["kc"], s["ks"] = _quantised(k)
        s["vc"], s["vs"] = _quantised(v)
    else:
        s["kc"], s["vc"], s["ks"], s["vs"] = k, v, None, None
    t = sum(lq for lq, _ in lens)
    s["q"] = _rand(gen, t, hq, d).bfloat16()
    cu = [0]
    for lq, _ in lens:
        cu.append(cu[-1] + lq)
    s["table"] = table.to(DEV)
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
    s["lk"] = torch.tensor([lk for _, lk in lens], dtype=torch.int32, device=DEV)
    s["max_q"], s["max_k"], s["t"] = max(lq for lq, _ in lens), max(lk for _, lk in lens), t
    s["slopes"] = s["prefix"] = None
    if case["alibi"]:
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, hq + 1, device=DEV) / hq)
    if case["prefix"]:
        s["prefix"] = torch.tensor(_prefix_lengths(case), dtype=torch.int32, device=DEV)
    if own:
        from auto_infer_amd import ops
        # the step's plan, which a program makes once for all its layers
        more = {"prefix_lens": s["prefix"]} if case["prefix"] else {}
        s["plan"] = ops.AttentionPlan(s["table"], s["cu"], s["lk"], t, hq, hkv, d, bs, **more)
    return s


# ------------------------------------------------------------------ write

def _write_one(x, cache, scale, slots):
    """The plain form of one cache's write, in place: over the whole pool,
    blocks without a new row keep what they hold."""
    nb, bs, h, d = cache.shape
    blk = (slots // bs).long()
    new = x.float()
    amax = torch.zeros(nb, h, device=DEV).index_reduce_(0, blk, new.abs().amax(-1), "amax")
    is_new = torch.zeros(nb * bs, dtype=torch.bool, device=DEV)
    is_new[slots.long()] = True
    is_new = is_new.view(nb, bs)
    old = scale.view(torch.uint8).int() - 127
    need = _needed_exp(amax)
    # a block whose first slot is written starts anew
    e = torch.where(is_new[:, :1], need, torch.maximum(old, need))
    e = torch.where(is_new.any(1, keepdim=True), e, old)
    # rows that stay in a block that does not start anew keep their values
    keep = torch.where(is_new[:, :1], torch.zeros_like(e), old - e)
    held = torch.ldexp(cache.float(), keep[:, None, :, None])
    held.view(nb * bs, h, d)[slots.long()] = torch.ldexp(new, -e[blk][:, :, None])
    cache.copy_(held.to(torch.float8_e4m3fn))
    scale.view(torch.uint8).copy_((e + 127).to(torch.uint8))


def _run_write(s):
    if own:
        from auto_infer_amd import ops
        ops.write_kv_fp8(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["slots"])
    else:
        _write_one(s["k"], s["kc"], s["ks"], s["slots"])
        _write_one(s["v"], s["vc"], s["vs"], s["slots"])
    # the exponents as whole numbers
    return {"key_cache": s["kc"], "key_exp": s["ks"].view(torch.uint8),
            "value_cache": s["vc"], "value_exp": s["vs"].view(torch.uint8)}


# ------------------------------------------------------------------ attention

def _gathered(cache, scale, table, n):
    """The first n cached rows of every request, (B, H, n, D) in float32."""
    x = cache[table.long()].float()                     # (B, W, bs, H, D)
    if scale is not None:
        e = scale.view(torch.uint8)[table.long()].int() - 127
        x = torch.ldexp(x, e[:, :, None, :, None])
    b, w, bs, h, d = x.shape
    return x.view(b, w * bs, h, d)[:, :n].transpose(1, 2)


def _run_attn(s):
    case = s["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if own:
        from auto_infer_amd import ops
        more = {}
        if case["kv"] == "fp8":
            more.update(key_scale=s["ks"], value_scale=s["vs"])
        return ops.paged_attention_gqa(s["q"], s["kc"], s["vc"], s["plan"], d ** -0.5,
                                       softcap=case["cap"], alibi_slopes=s["slopes"], **more)
    g = hq // hkv
    nq, nk = s["max_q"], s["max_k"]
    k = _gathered(s["kc"], s["ks"], s["table"], nk)
    v = _gathered(s["vc"], s["vs"], s["table"], nk)
    cu, lk = s["cu"].long(), s["lk"].long()
    lq = cu[1:] - cu[:-1]
    i = torch.arange(nq, device=DEV)
    rows = torch.minimum(cu[:-1, None] + i, cu[1:, None] - 1)              # (B, nq)
    q = s["q"][rows].float().view(-1, nq, hkv, g, d).permute(0, 2, 3, 1, 4)
    x = torch.matmul(q.reshape(-1, hkv, g * nq, d), k.transpose(-1, -2)).mul_(d ** -0.5)
    x = x.view(-1, hq, nq, nk)
    if case["cap"]:
        x = x.div_(case["cap"]).tanh_().mul_(case["cap"])
    pos = (lk - lq)[:, None] + i                                          # (B, nq)
    j = torch.arange(nk, device=DEV)
    if case["alibi"]:
        far = (pos[:, :, None] - j).abs().float()
        x = x.sub_(s["slopes"][:, None, None] * far[:, None])
    sees = j <= pos[:, :, None]
    if case["prefix"]:
        sees = sees | (j < s["prefix"][:, None, None])
    sees = sees & (j < lk[:, None, None])
    x = x.masked_fill_(~sees[:, None], float("-inf"))
    x = x.sub_(x.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(-1, hkv, g * nq, nk), v).view(-1, hq, nq, d)
    o = o / torch.where(total > 0, total, 1.0)
    req = torch.repeat_interleave(torch.arange(lq.shape[0], device=DEV), lq, output_size=s["t"])
    at = torch.arange(s["t"], device=DEV) - cu[req]
    return o.transpose(1, 2)[req, at].bfloat16()


# ------------------------------------------------------------------ rotary

ROPE_BASE = 1e6


def _scaling(case):
    if case["scaling"] == "linear":
        return {"type": "linear", "factor": 4.0}
    if case["scaling"] == "yarn":
        return {"type": "yarn", "factor": 32.0, "original_max_position": 32768}
    return None


def _frequencies(case):
    """Angle per position of each rotated pair (float64) and the factor on
    cos and sin.  The frequency-dependent scaling leaves pairs that turn more
    than 32 times within the original context, divides those that turn less
    than once by the factor and ramps in between."""
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


def _rotated(x, w, cos, sin, interleaved, eps=EPS):
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.to(x.dtype)
    half = cos.shape[-1]
    rot, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
    else:
        a, b = rot[..., :half], rot[..., half:]
    c, d = a * cos - b * sin, b * cos + a * sin
    rot = torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)
    return torch.cat((rot, rest), -1)


def _run_rope(s):
    case = s["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if own:
        from auto_infer_amd import ops
        q, k, _ = ops.rope_qk(s["qkv"], hq, hkv, s["positions"], s["rope"], s.get("wq"),
                              s.get("wk"), EPS, out=(s["q_out"], s["k_out"]))
        return q, k
    t = case["tokens"]
    angle = s["positions"].double()[:, None] * s["freq"]
    cos = (angle.cos() * s["factor"]).float()[:, None]
    sin = (angle.sin() * s["factor"]).float()[:, None]
    qkv = s["qkv"].float()
    q = qkv[:, :hq * d].view(t, hq, d)
    k = qkv[:, hq * d:(hq + hkv) * d].view(t, hkv, d)
    return tuple(_rotated(x, s.get(w), cos, sin, case["interleaved"]).bfloat16()
                 for x, w in ((q, "wq"), (k, "wk")))


def run(state):
    return {"write": _run_write, "attn": _run_attn, "rope": _run_rope}[state["case"]["op"]](state)


# ------------------------------------------------------------------ 64 bits

def _round_e4m3(x):
    """float64 to the nearest e4m3 value, ties to even (|x| <= 448)."""
    exp = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
    step = torch.exp2(exp - 3)
    return torch.round(x / step) * step


def _exact_write(x, cache, scale, slots):
    nb, bs, h, d = cache.shape
    val, exp = cache.double(), scale.view(torch.uint8).long() - 127
    out_val, out_exp = val.clone(), exp.clone()
    place = torch.full((nb * bs,), -1, dtype=torch.long, device=DEV)
    place[slots.long()] = torch.arange(slots.shape[0], device=DEV)
    place = place.view(nb, bs)
    for i in torch.unique(slots // bs).tolist():
        here = place[i] >= 0
        rows = x[place[i][here]].double()                       # (n, H, D)
        top = rows.abs().amax(dim=(0, 2))
        need = torch.ceil(torch.log2(top / 448.0) - 1e-12).long()
        need = torch.where(top <= 448.0 * 2.0 ** MIN_EXP, MIN_EXP, need)
        new = need if bool(here[0]) else torch.maximum(exp[i], need)
        if not bool(here[0]):
            out_val[i] = _round_e4m3(val[i] * torch.exp2((exp[i] - new).double())[None, :, None])
        out_val[i][here] = _round_e4m3(rows * torch.exp2(-new.double())[None, :, None])
        out_exp[i] = new
    return out_val, (out_exp + 127).to(torch.uint8)


def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["bs"]
    if case["op"] == "write":
        kv, ke = _exact_write(s["k"], s["kc"], s["ks"], s["slots"])
        vv, ve = _exact_write(s["v"], s["vc"], s["vs"], s["slots"])
        return {"key_cache": kv, "key_exp": ke, "value_cache": vv, "value_exp": ve}
    if case["op"] == "rope":
        freq, factor = _frequencies(case)
        pos = s["positions"].double().cpu()
        z = torch.polar(torch.full((len(pos), len(freq)), float(factor), dtype=torch.float64),
                        pos[:, None] * freq)[:, None].to(DEV)
        half, out = len(freq), []
        for x, w in ((s["qkv"][:, :hq * d], s.get("wq")),
                     (s["qkv"][:, hq * d:(hq + hkv) * d], s.get("wk"))):
            x = x.double().view(len(pos), -1, d).clone()
            if w is not None:
                x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
            if case["interleaved"]:
                first, second = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
            else:
                first, second = slice(0, half), slice(half, 2 * half)
            r = torch.complex(x[..., first], x[..., second]) * z
            x[..., first], x[..., second] = r.real, r.imag
            out.append(x)
        return tuple(out)
    out = torch.zeros(s["t"], hq, d, dtype=torch.float64, device=DEV)
    g, at = hq // hkv, 0
    pre = _prefix_lengths(case) if case["prefix"] else None
    for r, (lq, lk) in enumerate(_lengths(case)):
        blocks = s["table"][r, :-(-lk // bs)].long()
        k, v = s["kc"][blocks].double(), s["vc"][blocks].double()
        if case["kv"] == "fp8":
            k = k * 2.0 ** (s["ks"].view(torch.uint8)[blocks].double() - 127)[:, None, :, None]
            v = v * 2.0 ** (s["vs"].view(torch.uint8)[blocks].double() - 127)[:, None, :, None]
        k, v = k.flatten(0, 1)[:lk], v.flatten(0, 1)[:lk]
        pos = torch.arange(lk - lq, lk, device=DEV)[:, None]
        key = torch.arange(lk, device=DEV)[None]
        hidden = key > pos
        if pre is not None:
            hidden = hidden & (key >= pre[r])
        for h in range(hkv):
            q = s["q"][at:at + lq, h * g:(h + 1) * g].double().transpose(0, 1)     # (g, lq, d)
            x = torch.matmul(q, k[:, h].t().contiguous()) / math.sqrt(d)
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["alibi"]:
                x = x - s["slopes"][h * g:(h + 1) * g].double()[:, None, None] * (pos - key).abs()
            p = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1)
            out[at:at + lq, h * g:(h + 1) * g] = torch.matmul(p, v[:, h]).transpose(0, 1)
        at += lq
    return out
