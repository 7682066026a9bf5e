"""Outputs of rotary positions that share memory with the packed projection, or
with each other."""
import itertools

import pytest
import torch

from auto_infer_amd import _native, ops
from oracle import long_context as oracle

HQ, HKV, D = 4, 2, 64
WIDTH, NQ, NK = (HQ + 2 * HKV) * D, HQ * D, HKV * D
BASE = 1 << 20        # an address that nothing is read from: the calls are refused


def refused(tokens, ts, q, qts, k, kts):
    """q, k: elements from the projection's start."""
    args = (BASE, ts, tokens, HQ, HKV, D, 16, 16, D, 1.0, 0, None, None, 1e-6, BASE + 2 * q, qts, BASE + 2 * k, kts,
            None)
    lib = _native.load()
    conv = [t(a) if a is not None else None for a, t in zip(args, _native.SIGNATURES["aia_rope_qk"])]
    rc = lib.aia_rope_qk(*conv)
    return rc == _native.AIA_ERR_INVALID and "overlap" in _native.last_error()


@pytest.mark.parametrize("tokens,ts,q,qts,k,kts", [
    (5, WIDTH, 8, WIDTH, 1 << 16, NK),                  # shifted by a few elements
    (5, WIDTH, 0, NQ, 1 << 16, NK),                     # the same start, another stride
    (5, WIDTH, WIDTH, WIDTH, 1 << 16, NK),              # a row further on
    (5, WIDTH, 1 << 16, NQ, 0, WIDTH),                  # K onto the Q columns
    (5, WIDTH, 1 << 16, NQ, NQ + NK, WIDTH),            # K onto the V columns
    (5, 2 * WIDTH, WIDTH - 8, 2 * WIDTH, 1 << 16, NK),  # the row's end
    (5, 2 * WIDTH, 2 * WIDTH - 8, 2 * WIDTH, 1 << 16, NK),   # the next row's start
    (5, WIDTH, 1 << 16, NQ, (1 << 16) + 3 * NQ, NK),    # each other
    (5, WIDTH, 1 << 16, NQ + NK, (1 << 16) + NQ - 8, NQ + NK),
    (5, WIDTH, 4 * WIDTH + WIDTH - 8, NQ, 1 << 16, NK), # the last row's end
    (1, WIDTH, 8, WIDTH, 1 << 16, NK),
    (1, WIDTH, 0, NQ, NQ + 8, NK),
    (1, WIDTH, NQ, NQ, 1 << 16, NK),
    (2, WIDTH, -8, NQ, 1 << 16, NK),
])
def test_refused_overlaps(tokens, ts, q, qts, k, kts):
    assert refused(tokens, ts, q, qts, k, kts)


def share(a, alen, astride, b, blen, bstride, n):
    mine = {a + t * astride + i for t in range(n) for i in range(alen)}
    return any(b + t * bstride + i in mine for t in range(n) for i in range(blen))


def test_the_rule_is_exact_for_rows_of_one_stride():
    """The entry point's rule, restated on small numbers, against the sets of
    elements."""
    def rule(a, alen, b, blen, s, n):
        if a >= b + (n - 1) * s + blen or b >= a + (n - 1) * s + alen:
            return False
        if n == 1:
            return True
        d = (b - a) % s
        return d < alen or d + blen > s
    for s, alen, blen, n in itertools.product((3, 5, 6), (1, 2, 3), (1, 3), (1, 2, 3)):
        for b in range(-20, 21):
            assert rule(0, alen, b, blen, s, n) == share(0, alen, s, b, blen, s, n), (s, alen, blen, n, b)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 6])
def test_outputs_beside_the_projection(T):
    """Views of one wider tensor, the projection's own columns, and neighbours are
    taken; overlapping ones and overlapping projection rows are refused."""
    dev = "cuda:0"
    gen = torch.Generator().manual_seed(T)
    x = torch.randn(T, WIDTH, generator=gen).bfloat16()
    pos = torch.randint(0, 1000, (T,), generator=gen)
    rope = ops.RotaryEmbedding(D, device=dev)

    def check(q, k):
        for got, cols in ((q, x[:, :NQ]), (k, x[:, NQ:NQ + NK])):
            ref, bound = oracle.rope(cols.reshape(T, -1, D), pos, rope.inv_freq)
            assert bool(((got.cpu().double() - ref).abs() <= bound).all())
    wide = torch.zeros(T, 2 * WIDTH, dtype=torch.bfloat16, device=dev)
    qkv = wide[:, :WIDTH]
    qo, ko = wide[:, WIDTH:WIDTH + NQ].view(T, HQ, D), wide[:, WIDTH + NQ:WIDTH + NQ + NK].view(T, HKV, D)
    qkv.copy_(x)
    check(*ops.rope_qk(qkv, HQ, HKV, pos.to(dev), rope, out=(qo, ko))[:2])
    assert torch.equal(qkv.cpu(), x)
    own = qkv[:, :NQ].view(T, HQ, D), qkv[:, NQ:NQ + NK].view(T, HKV, D)
    check(*ops.rope_qk(qkv, HQ, HKV, pos.to(dev), rope, out=own)[:2])
    qkv.copy_(x)
    check(*ops.rope_qk(qkv, HQ, HKV, pos.to(dev), rope, out=(own[0], ko))[:2])
    qkv.copy_(x)
    for out in ((qkv[:, NK:NK + NQ].view(T, HQ, D), ko), (qo, qkv[:, NQ + NK:].view(T, HKV, D)),
                (qo, qo[:, :HKV]), (wide.view(-1)[8:8 + T * NQ].view(T, HQ, D), ko)):
        with pytest.raises(ValueError, match="overlap"):
            ops.rope_qk(qkv, HQ, HKV, pos.to(dev), rope, out=out)
    if T > 1:
        with pytest.raises(ValueError, match="qkv rows overlap"):
            ops.rope_qk(wide.as_strided((T, WIDTH), (WIDTH - 8, 1)), HQ, HKV, pos.to(dev), rope, out=(qo, ko))
    assert torch.equal(qkv.cpu(), x)
