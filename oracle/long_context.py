"""Plain float64 restatements of the operators around 8-bit caches, modified
scores and rotary positions, from their formulas.

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).  None of them has a
counterpart in the reference; they are written for checking, one value after
the other, not for speed.
"""
import math

import torch

E4M3_MAX = 448.0
MIN_EXP = -100


def e4m3(x):
    """float64 values to the nearest e4m3 value (ties to even; |x| <= 448; not
    finite: NaN): steps of 2^(e - 3) in [2^e, 2^(e + 1)), 2^-9 below 2^-6."""
    x = x.double()
    exp = torch.frexp(x)[1].clamp(min=-5) - 1
    step = torch.ldexp(torch.ones_like(x), exp - 3)
    out = torch.round(x / step) * step
    return torch.where(torch.isfinite(x), out, float("nan"))


def needed_exp(amax):
    """Least integer e >= MIN_EXP with amax <= 448 * 2^e."""
    e = MIN_EXP
    while amax > E4M3_MAX * 2.0 ** e:
        e += 1
    return e


def write_kv_fp8(rows, values, exps, slots):
    """In place over one cache: ``values`` (NB, bs, H, D) float64 e4m3 values,
    ``exps`` (NB, H) integers (a cached value stands for value * 2^exp), rows
    (T, H, D), slots a list."""
    nb, bs, heads, _ = values.shape
    blocks = {}
    for t, s in enumerate(slots):
        if 0 <= s < nb * bs:
            blocks.setdefault(s // bs, {})[s % bs] = t        # the last token stays
    for blk, placed in blocks.items():
        for h in range(heads):
            new = torch.stack([rows[t, h].double() for t in placed.values()])
            fin = new[torch.isfinite(new)].abs()
            need = needed_exp(fin.max().item() if fin.numel() else 0.0)
            old = int(exps[blk, h])
            e = need if 0 in placed else max(old, need)
            if 0 not in placed and e != old:
                for off in range(bs):
                    if off not in placed:
                        values[blk, off, h] = e4m3(values[blk, off, h] * 2.0 ** (old - e))
            for off, t in placed.items():
                values[blk, off, h] = e4m3(rows[t, h].double() * 2.0 ** -e)
            exps[blk, h] = e


def dequantised(cache, scale):
    """float64 values an 8-bit cache and its e8m0 scales stand for."""
    return cache.double() * torch.exp2(scale.view(torch.uint8).double() - 127)[:, None, :, None]


def scored_attention(query, keys, values, block_table, cu_seqlens_q, seqlens_kv, scale, softcap=0.0,
                     slopes=None, prefix=None):
    """Paged attention with modified scores in float64: query (T, Hq, D),
    keys / values (NB, bs, Hkv, D), the rest as ``paged_attn.paged_attention``.
    Returns (out, bound), both (T, Hq, D): ``bound`` is how far a kernel may be
    that takes scores and sums in float32, rounds the softmax weights to bf16
    and split rows' partials to fp16 (relative to the row's largest), and the
    output to bf16:
      (2^-8 + 2 eps) A + 2^-10 max_d A + 2^-8 |out|,
    A = sum_j p_j |v_j|, and eps = the error of a score: D 2^-24 sum_d |q_d k_d|
    scale for the products, 2^-21 of the cap or 2^-18 of the largest score for the
    tanh (the lesser), 2^-22 of the largest score for scaling, bias and exponent."""
    T, hq, d = query.shape
    bs, hkv = keys.shape[1], keys.shape[2]
    g = hq // hkv
    out = torch.zeros(T, hq, d, dtype=torch.float64)
    bound = torch.zeros_like(out)
    start = 0
    for b, end in enumerate(cu_seqlens_q):
        lq, lk = end - start, int(seqlens_kv[b])
        if lq and lk:
            j = torch.arange(lk)
            blk = block_table[b].long()[j // bs]
            k = keys[blk, j % bs].double()
            v = values[blk, j % bs].double()
            pos = torch.arange(lk - lq, lk)[:, None]
            seen = j[None] <= pos
            if prefix is not None:
                seen = seen | (j[None] < int(prefix[b]))
            for h in range(hq):
                q = query[start:end, h].double()
                kh, vh = k[:, h // g], v[:, h // g]
                s = q @ kh.t() * scale
                mag = q.abs() @ kh.abs().t() * scale
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                if slopes is not None:
                    s = s - float(slopes[h]) * (pos - j[None]).abs()
                s = s.masked_fill(~seen, -math.inf)
                top = s.amax(-1, keepdim=True)
                p = torch.where(seen, torch.exp(s - top.clamp(min=-1e300)), 0.0)
                total = p.sum(-1, keepdim=True)
                p = p / torch.where(total > 0, total, 1.0)
                # 0 * inf and 0 * NaN of keys that a row does not see are no part of its sum
                bad = ~torch.isfinite(vh)
                o = p @ torch.where(bad, 0.0, vh)
                if bad.any():
                    for i in range(lq):
                        o[i] = (p[i][seen[i], None] * vh[seen[i]]).sum(0)
                a = p @ torch.where(bad, 0.0, vh).abs()
                largest = torch.where(seen, s.abs(), 0.0).amax(-1, keepdim=True)
                eps = (d * 2.0 ** -24 * torch.where(seen, mag, 0.0).amax(-1, keepdim=True)
                       + torch.clamp(2.0 ** -18 * largest, max=2.0 ** -21 * softcap) + 2.0 ** -22 * largest)
                out[start:end, h] = o
                bound[start:end, h] = ((2.0 ** -8 + 2 * eps) * a + 2.0 ** -10 * a.amax(-1, keepdim=True)
                                       + 2.0 ** -8 * o.abs())
        start = end
    return out, bound


def rope(x, positions, inv_freq, factor=1.0, interleaved=False, weight=None, eps=1e-6):
    """Rotary positions of (T, H, D) rows, after an RMSNorm where ``weight`` is
    given.  Returns (out, bound): ``bound`` allows 2^-18 of a pair's length for
    the sine and cosine, 2^-20 for the float32 steps of norm and rotation, and
    the rounding to bf16."""
    x = x.double().clone()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    n = len(inv_freq)
    out, length = x.clone(), torch.zeros_like(x)
    for t, p in enumerate(positions.tolist()):
        for i, f in enumerate(inv_freq):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
            c, s = math.cos(p * f) * factor, math.sin(p * f) * factor
            out[t, :, a] = x[t, :, a] * c - x[t, :, b] * s
            out[t, :, b] = x[t, :, b] * c + x[t, :, a] * s
            length[t, :, a] = length[t, :, b] = (x[t, :, a].abs() + x[t, :, b].abs()) * abs(factor)
    length[..., 2 * n:] = x[..., 2 * n:].abs()
    return out, (2.0 ** -18 + 2.0 ** -20) * length + 2.0 ** -8 * out.abs() * (1 + 2.0 ** -8)
