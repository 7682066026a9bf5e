"""8-bit KV cache writes against a float64 restatement: every stored value and
every scale has to be equal (an e4m3 rounding and a power of two leave no
room)."""
import pytest
import torch

from auto_infer_amd import ops
from oracle import long_context as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def fresh(nb, bs, h, d, gen=None, exp_lo=-9, exp_hi=4):
    """A pool with random contents: (values, exps) for the oracle and the
    device tensors."""
    if gen is None:
        vals, exps = torch.zeros(nb, bs, h, d, dtype=torch.float64), torch.full((nb, h), -127)
    else:
        vals = oracle.e4m3(torch.randn(nb, bs, h, d, generator=gen) * 60)
        exps = torch.randint(exp_lo, exp_hi, (nb, h), generator=gen)
    cache = vals.to(torch.float8_e4m3fn).to(DEV)
    scale = (exps + 127).to(torch.uint8).to(DEV).view(torch.float8_e8m0fnu)
    return vals, exps, cache, scale


def check(cache, scale, vals, exps):
    got_e = scale.view(torch.uint8).cpu().int() - 127
    assert torch.equal(got_e, exps.int()), (got_e - exps.int()).abs().max()
    got = cache.cpu().double()
    nan = torch.isnan(vals)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], vals[~nan])


def write_both(k, v, slots, kv, vv):
    st = torch.tensor(slots, dtype=torch.int32, device=DEV)
    ops.write_kv_fp8(k.to(DEV), v.to(DEV), kv[2], vv[2], kv[3], vv[3], st)
    for rows, c in ((k, kv), (v, vv)):
        oracle.write_kv_fp8(rows, c[0], c[1], slots)
    for c in (kv, vv):
        check(c[2], c[3], c[0], c[1])


@pytest.mark.parametrize("d,h", [(128, 8), (128, 1), (64, 2), (64, 5)])
@pytest.mark.parametrize("bs", [1, 3, 16, 128, 300])
def test_prompts_and_decode_rows(d, h, bs):
    """Prompts that start and end inside blocks, then one row after the other
    behind them, growing the scales of their blocks."""
    gen = torch.Generator().manual_seed(d + bs)
    nb = 40 if bs < 16 else 12
    kv, vv = fresh(nb, bs, h, d, gen), fresh(nb, bs, h, d, gen)
    perm = torch.randperm(nb, generator=gen).tolist()
    n = min(2 * bs + max(1, bs // 2), 330)
    first = bs // 3
    at = [perm[p // bs] * bs + p % bs for p in range(first, first + n)]
    k = (torch.randn(n, h, d, generator=gen) * 3).bfloat16()
    v = torch.randn(n, h, d, generator=gen).bfloat16()
    write_both(k, v, at, kv, vv)
    for step in range(4):
        p = first + n + step
        if p // bs >= nb:
            break
        row = (torch.randn(1, h, d, generator=gen) * 4.0 ** step).bfloat16()
        write_both(row, -row, [perm[p // bs] * bs + p % bs], kv, vv)


@pytest.mark.parametrize("order", ["mixed", "reversed", "duplicates", "skipped"])
def test_slots_in_any_order(order):
    gen = torch.Generator().manual_seed(5)
    h, d, bs, nb = 3, 128, 16, 9
    kv, vv = fresh(nb, bs, h, d, gen), fresh(nb, bs, h, d, gen)
    slots = torch.randperm(nb * bs, generator=gen)[:70].tolist()
    if order == "reversed":
        slots = list(range(100, 20, -1))
    elif order == "duplicates":
        slots = slots[:20] + [slots[3], slots[3], slots[7]] + slots[:5] + [slots[19]] * 4
    elif order == "skipped":
        slots = [-1, slots[0], nb * bs, slots[1], -(2 ** 31), 2 ** 31 - 1] + slots[2:30] + [-7]
    k = (torch.randn(len(slots), h, d, generator=gen) * 9).bfloat16()
    v = torch.randn(len(slots), h, d, generator=gen).bfloat16()
    write_both(k, v, slots, kv, vv)


@pytest.mark.parametrize("bs", [16, 128, 1000])
def test_slots_in_any_order_of_a_long_step(bs):
    """Blocks whose tokens are spread over a step of several windows, runs that
    cross windows, and both in one call."""
    gen = torch.Generator().manual_seed(bs)
    h, d, nb = 2, 64, -(-4000 // bs)
    for kind in ("shuffled", "straight", "pieces"):
        kv, vv = fresh(nb, bs, h, d, gen), fresh(nb, bs, h, d, gen)
        slots = list(range(5, 5 + 900))
        if kind == "shuffled":
            slots = torch.randperm(nb * bs, generator=gen)[:700].tolist()
        elif kind == "pieces":
            slots = slots[300:] + [-1] * 7 + slots[:290] + [slots[40], slots[850]] + list(range(2000, 3100))
        k = (torch.randn(len(slots), h, d, generator=gen) * 9).bfloat16()
        v = torch.randn(len(slots), h, d, generator=gen).bfloat16()
        write_both(k, v, slots, kv, vv)


@pytest.mark.parametrize("bs,d", [(128, 128), (40, 64), (17, 128), (16, 128), (32, 64)])
def test_many_short_runs(bs, d):
    """A long step of decode rows and verify runs in blocks of their own, some
    blocks twice, at offsets where a block starts anew or goes on."""
    gen = torch.Generator().manual_seed(bs)
    h, nb = 5, 700
    kv, vv = fresh(nb, bs, h, d, gen), fresh(nb, bs, h, d, gen)
    slots = []
    for b in torch.randperm(nb, generator=gen).tolist():
        n, off = 1 + b % 3, int(torch.randint(0, bs - 3, (1,), generator=gen)) if b % 5 else 0
        slots += [b * bs + off + i for i in range(n)]
        if b % 40 == 7:                  # another run of the same block
            slots += [b * bs + bs - 1]
        if b % 40 == 9 and len(slots) > 9:   # of an earlier one
            slots += [slots[-9]]
    k = (torch.randn(len(slots), h, d, generator=gen) * 6).bfloat16()
    v = torch.randn(len(slots), h, d, generator=gen).bfloat16()
    write_both(k, v, slots, kv, vv)


def test_values_at_the_borders():
    """Largest values at and next to 448 * 2^e, ties of the rounding, zeros,
    subnormal and huge rows, and values that are not finite."""
    h, d, bs = 1, 64, 16
    rows = []
    for top in (448.0, 450.0, 446.0, 224.0, 7.0, 7.03125, 2.0 ** -120, 0.0, 3e38, 1.17e-38):
        r = torch.linspace(-1, 1, d, dtype=torch.float64) * top
        r[5] = top
        rows.append(r)
    rows.append(torch.arange(d) * 0.0625 + 17)          # halfway values at scale 1 and up
    rows.append(torch.where(torch.arange(d) % 3 == 0, float("inf"), torch.arange(d).double()))
    rows.append(torch.where(torch.arange(d) % 3 == 1, float("nan"), -torch.arange(d).double()))
    rows.append(torch.full((d,), float("-inf"), dtype=torch.float64))
    rows = torch.stack([r.double() for r in rows]).bfloat16()[:, None]
    for together in (False, True):
        kv, vv = fresh(16, bs, h, d), fresh(16, bs, h, d)
        slots = list(range(len(rows))) if together else [i * bs for i in range(len(rows))]
        write_both(rows, rows, slots, kv, vv)


def test_rows_in_strided_and_unaligned_buffers_and_a_single_cache():
    gen = torch.Generator().manual_seed(8)
    h, d, bs, nb, T = 4, 128, 16, 6, 21
    for off, width in ((0, 3 * h * d), (1, 2 * h * d + 1)):
        kv, vv = fresh(nb, bs, h, d, gen), fresh(nb, bs, h, d, gen)
        buf = torch.randn(T, width, generator=gen).bfloat16()
        k = buf[:, off:off + h * d].view(T, h, d) if off == 0 else None
        gbuf = buf.to(DEV)
        gk = gbuf.as_strided((T, h, d), (width, d, 1), off)
        gv = gbuf.as_strided((T, h, d), (width, d, 1), off + h * d)
        k = buf.as_strided((T, h, d), (width, d, 1), off)
        v = buf.as_strided((T, h, d), (width, d, 1), off + h * d)
        slots = [7 + i for i in range(T)]
        st = torch.tensor(slots, dtype=torch.int32, device=DEV)
        ops.write_kv_fp8(gk, gv, kv[2], vv[2], kv[3], vv[3], st)
        for rows, c in ((k, kv), (v, vv)):
            oracle.write_kv_fp8(rows, c[0], c[1], slots)
            check(c[2], c[3], c[0], c[1])
    kv = fresh(nb, bs, h, d, gen)
    ops.write_kv_fp8(gk, None, kv[2], None, kv[3], None, st)
    oracle.write_kv_fp8(k, kv[0], kv[1], slots)
    check(kv[2], kv[3], kv[0], kv[1])
    empty = torch.empty(0, h, d, dtype=torch.bfloat16, device=DEV)
    ops.write_kv_fp8(empty, empty, kv[2], kv[2], kv[3], kv[3], st[:0])


def test_a_long_step_and_far_blocks():
    """A step of several thousand tokens, and blocks whose bytes lie past
    2^32."""
    gen = torch.Generator().manual_seed(9)
    h, d, bs = 8, 128, 128
    nb = (1 << 32) // (bs * h * d) + 40
    cache = torch.empty(nb, bs, h, d, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    scale = torch.zeros(nb, h, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
    blocks = [nb - 1 - 2 * i for i in range(17)] + [3]
    slots = [b * bs + o for b in blocks for o in range(bs)][:2200]
    k = torch.randn(len(slots), h, d, generator=gen).bfloat16()
    ops.write_kv_fp8(k.to(DEV), None, cache, None, scale, None,
                     torch.tensor(slots, dtype=torch.int32, device=DEV))
    vals, exps = torch.zeros(len(blocks), bs, h, d, dtype=torch.float64), torch.full((len(blocks), h), -127)
    place = {b: i for i, b in enumerate(blocks)}
    oracle.write_kv_fp8(k, vals, exps, [place[s // bs] * bs + s % bs for s in slots])
    idx = torch.tensor(blocks, device=DEV)
    got = cache.view(torch.uint8)[idx].view(torch.float8_e4m3fn)
    used = 2200 - 17 * bs
    got[17, used:] = 0
    check(got, scale.view(torch.uint8)[idx].view(torch.float8_e8m0fnu), vals, exps)


def test_replays_from_a_graph_and_another_stream():
    gen = torch.Generator().manual_seed(10)
    h, d, bs, nb, T = 2, 64, 16, 8, 5
    kv, vv = fresh(nb, bs, h, d, gen), fresh(nb, bs, h, d, gen)
    k = torch.zeros(T, h, d, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    slots = torch.full((T,), -1, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.write_kv_fp8(k, v, kv[2], vv[2], kv[3], vv[3], slots)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            ops.write_kv_fp8(k, v, kv[2], vv[2], kv[3], vv[3], slots)
    for step in range(4):
        hk = (torch.randn(T, h, d, generator=gen) * 3.0 ** step).bfloat16()
        hv = torch.randn(T, h, d, generator=gen).bfloat16()
        at = torch.randperm(nb * bs, generator=gen)[:T]
        k.copy_(hk), v.copy_(hv), slots.copy_(at.int())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for rows, c in ((hk, kv), (hv, vv)):
            oracle.write_kv_fp8(rows, c[0], c[1], at.tolist())
            check(c[2], c[3], c[0], c[1])
