"""Plain restatements, in 64 bits, of block-sparse attention: bounds of a block's
keys, the selection by them and attention over the selected blocks."""
import math

import torch

MIN_EXP = -100


def bound_exp(amax):
    """The least e >= -100 with amax <= 127 * 2^e."""
    e = MIN_EXP
    while amax > 127 * 2.0 ** e:
        e += 1
    return e


def block_bounds(keys):
    """(hi, nlo, e) of one block and head: keys (n, D) float64."""
    ok = torch.isfinite(keys)
    e = bound_exp(float(keys[ok].abs().max()) if bool(ok.any()) else 0.0)
    step = 2.0 ** e
    top = torch.where(ok, keys, -math.inf).amax(0)
    low = torch.where(ok, keys, math.inf).amin(0)
    hi, nlo = torch.ceil(top / step), torch.ceil(-low / step)
    bad = ~ok.all(0)
    return torch.where(bad, 127.0, hi).long(), torch.where(bad, 127.0, nlo).long(), e


def select(q, hi, nlo, exps, visible, count, sink, local):
    """Blocks of one token and KV head: q (g, D), hi / nlo (N, D) whole numbers, exps
    (N,)."""
    if visible <= count:
        return list(range(visible))
    q = q.double()
    ok = torch.isfinite(q)
    unit = 2.0 ** bound_exp(float(q[ok].abs().max()) if bool(ok.any()) else 0.0)
    whole = torch.where(ok, torch.round(torch.where(ok, q, 0.0) / unit), 0.0)
    score = []
    for i in range(visible):
        total = float((whole.clamp(min=0) @ hi[i].double() + (-whole).clamp(min=0) @ nlo[i].double()).sum())
        score.append(float(torch.tensor(total, dtype=torch.float64).float()) * 2.0 ** int(exps[i]))
    always = [i for i in range(visible) if i < sink or i >= visible - local]
    rest = sorted((i for i in range(visible) if i not in set(always)), key=lambda i: (-score[i], i))
    return sorted(always + rest[:count - len(always)])


def attention(q, k, v, seen, scale):
    """One query head: q (D,), k / v (n, D), seen (n,) truth values; float64."""
    if not bool(seen.any()):
        return torch.zeros(v.shape[1], dtype=torch.float64)
    x = (k[seen].double() @ q.double()) * scale
    return torch.softmax(x, 0) @ v[seen].double()
