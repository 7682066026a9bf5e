"""``ops.rope_append`` against ``rope_qk`` followed by a cache write, bit for bit (both
halves have tests of their own against restatements in 64 bits), and once against the
formulas."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def caches(kind, nb, bs, hkv, d, gen):
    if kind == "fp8":
        from auto_infer_amd import ops
        x = [torch.randint(0, 120, (nb, bs, hkv, d), generator=gen, dtype=torch.uint8).to(DEV).view(ops.FP8_KV)
             for _ in range(2)]
        s = [torch.randint(115, 130, (nb, hkv), generator=gen, dtype=torch.uint8).to(DEV).view(ops.FP8_KV_SCALE)
             for _ in range(2)]
        return x, s
    return [torch.randn(nb, bs, hkv, d, generator=gen).bfloat16().to(DEV) for _ in range(2)], [None, None]


def raw(t):
    return t.contiguous().view(torch.uint8) if t.element_size() == 1 else t.view(torch.int16)


def both(T, hq, hkv, d, bs, kind, rotary, inter, norm, slots, nb, seed, pad=0, out=False):
    """(q, caches, scales) of the one call and of the two."""
    from auto_infer_amd import ops
    gen = torch.Generator().manual_seed(seed)
    rope = ops.RotaryEmbedding(d, rotary_dim=rotary, base=1e4, interleaved=inter, device=DEV,
                               scaling={"type": "yarn", "factor": 8.0, "original_max_position": 4096})
    width = (hq + 2 * hkv) * d
    wide = torch.randn(T, width + pad, generator=gen).bfloat16().to(DEV)
    pos = torch.randint(-5, 1 << 40, (T,), generator=gen).to(DEV)
    w = [(1 + 0.3 * torch.randn(d, generator=gen)).bfloat16().to(DEV) if norm else None for _ in range(2)]
    slots = torch.tensor(slots, dtype=torch.int32, device=DEV)
    kv, sc = caches("fp8" if kind == "fp8" else "bf16", nb, bs, hkv, d, gen)
    results = []
    for one in (True, False):
        qkv = wide.clone()[:, :width]
        kc, vc = (x.clone() for x in kv)
        ks, vs = (x.clone() if x is not None else None for x in sc)
        if one:
            qo = torch.empty(T, hq, d, dtype=torch.bfloat16, device=DEV) if out else None
            q = ops.rope_append(qkv, hq, hkv, pos, rope, kc, vc, slots, *w, 1e-6, q_out=qo, key_scale=ks,
                                value_scale=vs, kv_layout="nz" if kind == "nz" else "nd")
            assert torch.equal(raw(qkv[:, hq * d:]), raw(wide[:, hq * d:width]))
            if out:
                assert torch.equal(raw(qkv), raw(wide[:, :width]))
        else:
            q, k, v = ops.rope_qk(qkv, hq, hkv, pos, rope, *w, 1e-6)
            if kind == "fp8":
                ops.write_kv_fp8(k, v, kc, vc, ks, vs, slots)
            elif kind == "nz":
                ops.write_kv_nz(k, v, kc, vc, slots)
            else:
                ops.write_kv(k, v, kc, vc, slots)
        results.append([q.contiguous(), kc, vc] + ([ks, vs] if kind == "fp8" else []))
    return results


def runs(T, bs, nb, seed, skip=False):
    """Slots of T tokens in runs that begin anywhere in a block; some outside."""
    rng = random.Random(seed)
    free = list(range(nb))
    rng.shuffle(free)
    out = []
    while len(out) < T:
        blk, off = free.pop(), rng.choice([0, 0, rng.randrange(bs)])
        n = min(T - len(out), rng.randint(1, bs - off))
        out += range(blk * bs + off, blk * bs + off + n)
    if skip:
        for i in rng.sample(range(T), max(1, T // 5)):
            out[i] = rng.choice([-1, nb * bs, nb * bs + 7])
    return out


@pytest.mark.parametrize("kind", ["bf16", "nz", "fp8"])
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (28, 4, 128), (14, 2, 64), (1, 1, 64), (64, 8, 128), (5, 5, 128)])
@pytest.mark.parametrize("T,bs", [(1, 16), (3, 1), (77, 16), (130, 32), (300, 128), (60, 24)])
def test_equals_rotation_then_write(T, bs, hq, hkv, d, kind):
    for i, (rotary, inter, norm) in enumerate([(d, False, True), (d // 2, True, False), (16, False, False),
                                               (48, False, True), (48, True, True)]):
        nb = T + 3
        got, want = both(T, hq, hkv, d, bs, kind, rotary, inter, norm, runs(T, bs, nb, i, skip=i > 2), nb, i,
                         pad=8 * (i % 2), out=i % 2 == 0)
        for a, b in zip(got, want):
            assert torch.equal(raw(a), raw(b)), (rotary, inter, norm)


@pytest.mark.parametrize("bs", [16, 128])
def test_slots_in_any_order_and_twice_8bit(bs):
    rng = random.Random(bs)
    slots = [rng.randrange(6 * bs) for _ in range(3 * bs)]
    got, want = both(3 * bs, 4, 2, 128, bs, "fp8", 96, False, True, slots, 6, 1)
    for a, b in zip(got, want):
        assert torch.equal(raw(a), raw(b))


def test_against_the_formulas():
    """float64: |q error| <= 2^-8 |q| (one rounding; the float32 steps in front, of a few
    2^-24 of a head's largest value, get 2^-20 of it)."""
    from auto_infer_amd import ops
    gen = torch.Generator().manual_seed(3)
    T, hq, hkv, d, bs = 33, 6, 3, 128, 16
    rope = ops.RotaryEmbedding(d, base=1e6, device=DEV)
    qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=gen).bfloat16()
    w = (1 + 0.3 * torch.randn(d, generator=gen)).bfloat16()
    pos = torch.randint(0, 1 << 20, (T,), generator=gen)
    kc, vc = (torch.zeros(5, bs, hkv, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    slots = torch.randperm(5 * bs, generator=gen)[:T].int()
    q = ops.rope_append(qkv.to(DEV), hq, hkv, pos.to(DEV), rope, kc, vc, slots.to(DEV), w.to(DEV), w.to(DEV))
    x = qkv.double()[:, :(hq + hkv) * d].view(T, hq + hkv, d)
    x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    a = pos.double()[:, None, None] * torch.tensor(rope.inv_freq, dtype=torch.float64)
    lo, hi = x[..., :d // 2], x[..., d // 2:]
    x = torch.cat((lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()), -1)
    got = torch.cat((q.cpu(), kc.cpu().view(-1, hkv, d)[slots.long()]), 1).double()
    assert bool(((got - x).abs() <= 2.0 ** -8 * x.abs() + 2.0 ** -20 * x.abs().amax(-1, keepdim=True)).all())
    assert torch.equal(vc.cpu().view(-1, hkv, d)[slots.long()], qkv[:, (hq + hkv) * d:].view(T, hkv, d))


def test_no_tokens():
    from auto_infer_amd import ops
    rope = ops.RotaryEmbedding(64, device=DEV)
    kc, vc = (torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = ops.rope_append(torch.empty(0, 8 * 64, dtype=torch.bfloat16, device=DEV), 4, 2,
                        torch.empty(0, dtype=torch.int64, device=DEV), rope, kc, vc,
                        torch.empty(0, dtype=torch.int32, device=DEV))
    assert q.shape == (0, 4, 64)
