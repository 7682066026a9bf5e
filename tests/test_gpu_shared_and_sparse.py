"""Appending with rotation, shared prefixes and block-sparse attention as a server uses
them: through the GQA backend over prompt chunks and decode steps, from HIP graphs, on
streams of their own, and the calls that are refused."""
import numpy as np
import pytest
import torch

from auto_infer_amd import ops, packing
from auto_infer_amd.attention import registry
from auto_infer_amd.attention.gqa import GqaHipBackend
from auto_infer_amd.execution import BatchPlan, RequestView, ScheduledRequest
from auto_infer_amd.graph import DecodeGraph
from oracle import block_sparse as ref
from oracle import long_context as oracle
from oracle import pack
from tests.test_gpu_backend_options import make_context, make_model
from tests.test_gpu_block_sparse import empty_bounds, make, make_plan, on_gpu

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def rows_of(cache, scale=None):
    x = cache.cpu().double()
    if scale is not None:
        x = x * torch.exp2(scale.view(torch.uint8).cpu().double() - 127)[:, None, :, None]
    return x


def check(out, q, caches, ctx, d, fp8):
    """Against plain attention over the caches as they are; the parts of a row are
    rounded to fp16 (2^-11 of values of at most 8) on top of what the bound has."""
    keys, values = (rows_of(caches[i], caches[2 + i] if fp8 else None) for i in range(2))
    want, bound = oracle.scored_attention(q.cpu(), keys, values, ctx.block_table.cpu(), ctx.cu_seqlens_q,
                                          ctx.seqlens_kv, d ** -0.5)
    far = (out.cpu().double() - want).abs()
    assert bool((far <= bound + 8 * 2.0 ** -11).all()), (far - bound).max().item()


STEPS = [[(0, 300), (1, 9)], [(0, 1), (1, 250), (2, 40)], [(0, 1), (1, 1), (2, 3), (3, 20)], [(0, 1), (1, 1), (2, 1), (3, 1)]]


@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("rope", [True, False])
def test_backend_that_shares_prefixes(hq, hkv, d, kv_dtype, rope):
    """Requests 1 to 3 begin with request 0's blocks (as prefix caching hands them out)."""
    bs, nb = 16, 120
    emb = ops.RotaryEmbedding(d, base=1e5, device=DEV) if rope else False
    model = make_model(hq, hkv, d, 2, True, seed=d, kv_dtype=kv_dtype, aia_rope=emb, attn_share_prefixes=True)
    backend, caches = registry.build_attention_backend(model, "paged", nb, bs)
    gen = torch.Generator().manual_seed(2)
    perm = torch.randperm(nb, generator=gen).tolist()
    first = perm[:18]                                     # 288 keys
    tables = [first + perm[18 + 20 * i:38 + 20 * i] for i in range(4)]
    done = [0, 288, 288, 288]
    for step in STEPS:
        ctx, _ = make_context(backend, caches, [(tables[i], done[i], n) for i, n in step], bs)
        T = sum(n for _, n in step)
        for layer in range(2):
            x = torch.randn(T, hq * d, generator=gen).bfloat16().to(DEV)
            out = backend.attention(layer, x, ctx).view(T, hq, d)
            p = f"model.layers.{layer}.self_attn."
            qkv = x @ model.w[p + "qkv_proj.weight"].t()
            norms = (model.w[p + "q_norm.weight"], model.w[p + "k_norm.weight"])
            if rope:
                q, k, v = ops.rope_qk(qkv, hq, hkv, ctx.positions, emb, *norms, 1e-6)
                blocks, off = ctx.slot_mapping.long() // bs, ctx.slot_mapping.long() % bs
                if kv_dtype == "bf16":
                    assert torch.equal(caches[layer][0][blocks, off], k) and torch.equal(caches[layer][1][blocks, off], v)
            else:
                from auto_infer_amd.attention.layers import rms_norm
                q = rms_norm(qkv[:, :hq * d].reshape(T, hq, d), norms[0], 1e-6)
            check(out, q, caches[layer], ctx, d, kv_dtype == "fp8")
        for i, n in step:
            done[i] += n


@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 4, 128), (14, 2, 64)])
def test_backend_with_sparse_blocks(hq, hkv, d, kv_dtype):
    """Every step: the caches' bounds are those of what the blocks hold, the selection is
    the bounds', and the output is attention over it; enough blocks give plain attention."""
    bs, nb, picked = 16, 100, 5
    emb = ops.RotaryEmbedding(d, device=DEV)
    options = dict(kv_dtype=kv_dtype, aia_rope=emb, attn_sparse_local=1)
    model = make_model(hq, hkv, d, 1, True, seed=d, attn_sparse_blocks=picked, **options)
    backend, caches = registry.build_attention_backend(model, "paged", nb, bs)
    whole = make_model(hq, hkv, d, 1, True, seed=d, attn_sparse_blocks=40, **options)
    all_of, more = registry.build_attention_backend(whole, "paged", nb, bs)
    gen = torch.Generator().manual_seed(3)
    perm = torch.randperm(nb, generator=gen).tolist()
    tables, done = [perm[25 * i:25 * i + 25] for i in range(4)], [0] * 4
    fp8 = kv_dtype == "fp8"
    p = "model.layers.0.self_attn."
    for step in STEPS:
        rows = [(tables[i], done[i], n) for i, n in step]
        T = sum(n for _, n in step)
        x = torch.randn(T, hq * d, generator=gen).bfloat16().to(DEV)
        ctx, _ = make_context(all_of, more, rows, bs)
        dense = all_of.attention(0, x, ctx).view(T, hq, d)
        q = ops.rope_qk(x @ model.w[p + "qkv_proj.weight"].t(), hq, hkv, ctx.positions, emb,
                        model.w[p + "q_norm.weight"], model.w[p + "k_norm.weight"], 1e-6)[0]
        check(dense, q, more[0], ctx, d, fp8)
        ctx, _ = make_context(backend, caches, rows, bs)
        out = backend.attention(0, x, ctx).view(T, hq, d).cpu().double()
        cache = caches[0]
        keys, values = (rows_of(cache[i], cache[2 + i] if fp8 else None) for i in range(2))
        bounds, exps = cache[-2].cpu(), cache[-1].view(torch.uint8).cpu().int() - 127
        qc, t = q.cpu(), 0
        for (table, before, n) in rows:
            lk = before + n
            blocks = torch.tensor(table[:-(-lk // bs)])
            for j, blk in enumerate(blocks.tolist()):
                for h in range(hkv):
                    hi, nlo, e = ref.block_bounds(keys[blk, :min(bs, lk - j * bs), h])
                    assert torch.equal(bounds[blk, h, 0].long(), hi) and torch.equal(bounds[blk, h, 1].long(), nlo)
                    assert int(exps[blk, h]) == e
            k, v = (c[blocks].flatten(0, 1)[:lk] for c in (keys, values))
            for i in range(n):
                if i % 17 and n - i > 2:
                    t += 1
                    continue
                pos = before + i
                for h in range(hkv):
                    group = range(h * (hq // hkv), (h + 1) * (hq // hkv))
                    sel = ref.select(qc[t, group.start:group.stop], bounds[blocks, h, 0], bounds[blocks, h, 1],
                                     exps[blocks, h], pos // bs + 1, picked, 1, 1)
                    seen = torch.zeros(lk, dtype=torch.bool)
                    for b in sel:
                        seen[b * bs:(b + 1) * bs] = True
                    seen[pos + 1:] = False
                    for head in group:
                        want = ref.attention(qc[t, head], k[:, h], v[:, h], seen, d ** -0.5)
                        size = ref.attention(qc[t, head], k[:, h], v[:, h].abs(), seen, d ** -0.5)
                        bound = 2.0 ** -7 * (size + want.abs()) + 8 * 2.0 ** -11
                        assert bool(((out[t, head] - want).abs() <= bound).all()), (t, head)
                t += 1
        for i, n in step:
            done[i] += n


@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
def test_decode_graph_with_shared_prefixes(kv_dtype):
    """A captured gear (planner, writes, attention) replayed over growing requests with
    eager work between the replays; scratch rows of the gear included."""
    rng = np.random.default_rng(1)
    gear, maxb, bs, nb, hq, hkv, d, L = 8, 40, 16, 200, 16, 8, 128, 2
    stager = packing.DecodeInputStager(
        tid=torch.zeros(gear, dtype=torch.long, device=DEV),
        positions=torch.zeros(gear, dtype=torch.long, device=DEV),
        slots=torch.zeros(gear, dtype=torch.int32, device=DEV),
        block_table=torch.zeros(gear, maxb, dtype=torch.int32, device=DEV), block_size=bs, scratch0=nb - gear)
    g = torch.Generator(device=DEV).manual_seed(3)
    backend = GqaHipBackend(hq, hkv, d, d ** -0.5, L, DEV, torch.bfloat16, kv_dtype=kv_dtype)
    fp8 = kv_dtype == "fp8"
    caches = [tuple(c) if not fp8 else c for c in backend.alloc_kv_caches(nb, bs)]
    slots = torch.arange(nb * bs, dtype=torch.int32, device=DEV)
    for c in caches:
        rows = [torch.randn(nb * bs, hkv, d, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
        (ops.write_kv_fp8 if fp8 else ops.write_kv)(*rows, *c, slots)
    dg = DecodeGraph(stager, caches, num_q_heads=hq, num_kv_heads=hkv, share_prefixes=True)
    free = list(range(nb - gear))
    rng.shuffle(free)
    first = [free.pop() for _ in range(20)]
    reqs = {f"r{i}": dict(pos=lk - 1, blocks=[*(first if lk > 320 else ()), *(free.pop() for _ in range(lk // bs + 2))])
            for i, lk in enumerate([330, 500, 17, 345, 321])}
    for step in range(5):
        views = {rid: RequestView(rid, tuple(range(r["pos"] + 1)), r["pos"], 1, 1, ()) for rid, r in reqs.items()}
        plan = BatchPlan.make([ScheduledRequest(rid, 1, False, tuple(r["blocks"][:maxb])) for rid, r in reqs.items()],
                              views, {rid: r["blocks"][:maxb] for rid, r in reqs.items()})
        for buf in (dg.q, dg.k_new, dg.v_new):
            buf.copy_(torch.randn(buf.shape, generator=g, device=DEV, dtype=torch.bfloat16))
        torch.cuda.synchronize()
        dg.stage(plan)
        if dg.graph is None:
            dg.capture()
        else:
            dg.replay()
        torch.cuda.synchronize()
        exp = pack.decode_stage(plan, gear=gear, max_blocks=maxb, block_size=bs, scratch0=nb - gear)
        for layer in range(L):
            keys, values = (rows_of(caches[layer][i], caches[layer][2 + i] if fp8 else None) for i in range(2))
            if not fp8:
                at = torch.tensor(exp["slots"].tolist())
                assert torch.equal(keys.view(-1, hkv, d)[at], dg.k_new[layer].cpu().double())
            want, bound = oracle.scored_attention(dg.q[layer].cpu(), keys, values, torch.as_tensor(exp["block_table"]),
                                                  list(range(1, gear + 1)), list(exp["kv_lengths"]), d ** -0.5)
            far = (dg.out[layer].cpu().double() - want).abs()
            assert bool((far <= bound + 8 * 2.0 ** -11).all())
        for r in reqs.values():
            r["pos"] += 1


def test_a_whole_sparse_layer_in_one_graph():
    """Plan, append, bounds, selection and attention captured together and replayed over
    steps whose metadata changes in place, against the same calls made eagerly."""
    bs, hq, hkv, d, B, nb, W = 16, 16, 4, 128, 6, 200, 30
    gen = torch.Generator().manual_seed(5)
    rope = ops.RotaryEmbedding(d, device=DEV)
    table = torch.randperm(nb, generator=gen)[:B * W].view(B, W).int().to(DEV)
    cu = torch.arange(B + 1, dtype=torch.int32, device=DEV)
    lk = torch.tensor([1, 17, 100, 333, 16, 470], dtype=torch.int32, device=DEV)
    pos, slots = torch.zeros(B, dtype=torch.int64, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)
    qkv = torch.zeros(B, (hq + 2 * hkv) * d, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(B, hq, d, dtype=torch.bfloat16, device=DEV)
    caches = [torch.randn(nb, bs, hkv, d, generator=gen).bfloat16().to(DEV) for _ in range(2)]
    bounds = empty_bounds(nb, hkv, d)
    sel = torch.zeros(B, hkv, 6, dtype=torch.int32, device=DEV)
    out = torch.zeros(B, hq, d, dtype=torch.bfloat16, device=DEV)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        plan = ops.BlockSparsePlan(table, cu, lk, B, hq, hkv, d, bs, 6, 1, 2)

    def layer(plan, caches, bounds, sel, out):
        plan.replan()
        ops.rope_append(qkv, hq, hkv, pos, rope, *caches, slots, q_out=q)
        ops.summarize_blocks(caches[0], plan, *bounds)
        ops.select_blocks(q, plan, *bounds, out=sel)
        return ops.paged_attention_sparse(q, *caches, plan, sel, d ** -0.5, out=out)

    def advance(by):
        lk.add_(by)
        pos.copy_(lk.long() - 1)
        slots.copy_(table.gather(1, (pos // bs)[:, None])[:, 0] * bs + (pos % bs).int())
        qkv.copy_(torch.randn(qkv.shape, generator=gen).bfloat16())
    other = [c.clone() for c in caches], [b.clone() for b in bounds], sel.clone(), out.clone()
    advance(0)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        layer(plan, caches, bounds, sel, out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layer(plan, caches, bounds, sel, out)
    torch.cuda.synchronize()
    eager = ops.BlockSparsePlan(table, cu, lk, B, hq, hkv, d, bs, 6, 1, 2)
    for _ in range(4):
        layer(eager, *other)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(sel, other[2]) and torch.equal(out, other[3])
        assert torch.equal(bounds[0], other[1][0]) and torch.equal(caches[0], other[0][0])
        advance(1)
        torch.cuda.synchronize()


def test_two_plans_on_two_streams():
    """Two steps in flight with plans of their own give what each gives alone."""
    cases = [make([(1, 900)] * 20, 16, 8, 128, 16, seed=1, spread=False), make([(60, 700), (2, 90)], 8, 2, 64, 16, seed=2, spread=False)]
    tensors = [on_gpu(s) for s in cases]

    def run(i, stream):
        g = tensors[i]
        with torch.cuda.stream(stream):
            bounds = empty_bounds(g["nb"], g["hkv"], g["d"])
            plan = make_plan(g, 7, 1, 1)
            shared = ops.SharedPrefixPlan(g["table"], g["cu"], g["lk"], g["t"], g["hq"], g["hkv"], g["d"], g["bs"])
            ops.summarize_blocks(g["kc"], plan, *bounds)
            for r in range(g["table"].shape[0]):         # (blocks before the step's)
                bounds[0].index_fill_(0, g["table"][r, :g["lens"][r][1] // 32].long(), 3 + r)
                bounds[1].view(torch.uint8).index_fill_(0, g["table"][r, :g["lens"][r][1] // 32].long(), 127)
            bounds[0].clamp_(max=77)
            sel = ops.select_blocks(g["q"], plan, *bounds)
            return (sel, ops.paged_attention_sparse(g["q"], g["kc"], g["vc"], plan, sel, 0.1),
                    ops.paged_attention_shared(g["q"], g["kc"], g["vc"], shared, 0.1))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    alone = []
    for i in range(2):
        alone.append(run(i, streams[i]))
        torch.cuda.synchronize()
    for _ in range(3):
        got = [run(i, streams[i]) for i in (0, 1)]
        torch.cuda.synchronize()
        for a, b in zip(got, alone):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_plan_used_on_another_stream():
    s = make([(1, 900)] * 20, 16, 8, 128, 16, seed=1, spread=False)
    g = on_gpu(s)
    plan = ops.SharedPrefixPlan(g["table"], g["cu"], g["lk"], 20, 16, 8, 128, 16)
    want = ops.paged_attention_shared(g["q"], g["kc"], g["vc"], plan, 0.1)
    torch.cuda.synchronize()
    plan.replan()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.paged_attention_shared(g["q"], g["kc"], g["vc"], plan, 0.1)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_refusals():
    s = make([(1, 90), (2, 40)], 4, 2, 64, 16, seed=6)
    g = on_gpu(s)
    plan = make_plan(g, 3)
    shared = ops.SharedPrefixPlan(g["table"], g["cu"], g["lk"], 3, 4, 2, 64, 16)
    bounds = empty_bounds(g["nb"], 2, 64)
    sel = torch.zeros(3, 2, 3, dtype=torch.int32, device=DEV)
    q, kc, vc = g["q"], g["kc"], g["vc"]
    sc = torch.zeros(g["nb"], 2, dtype=torch.uint8, device=DEV).view(ops.FP8_KV_SCALE)
    for f in (lambda: make_plan(g, 3, 2, 2), lambda: make_plan(g, 3, 0, 0),
              lambda: ops.SharedPrefixPlan(g["table"], g["cu"][:-1], g["lk"], 3, 4, 2, 64, 16),
              lambda: ops.SharedPrefixPlan(g["table"].t(), g["cu"], g["lk"], 3, 4, 2, 64, 16),
              lambda: ops.SharedPrefixPlan(g["table"], g["cu"], g["lk"], 3, 4, 2, 64, 16, group_ids=g["lk"][:1]),
              lambda: ops.SharedPrefixPlan(g["table"], g["cu"], g["lk"], 3, 4, 2, 64, 16,
                                           workspace=torch.empty(64, dtype=torch.uint8, device=DEV)),
              lambda: ops.paged_attention_shared(q[:2], kc, vc, shared, 0.1),
              lambda: ops.paged_attention_shared(q, kc[:, :8], vc[:, :8], shared, 0.1),
              lambda: ops.paged_attention_shared(q, kc, vc[:2], shared, 0.1),
              lambda: ops.paged_attention_shared(q, kc, vc, shared, 0.0),
              lambda: ops.paged_attention_shared(q, kc, vc, shared, 0.1, key_scale=sc),
              lambda: ops.paged_attention_shared(q.float(), kc, vc, shared, 0.1),
              lambda: ops.paged_attention_sparse(q, kc, vc, plan, sel[:, :, :2], 0.1),
              lambda: ops.paged_attention_sparse(q, kc, vc, plan, sel.long(), 0.1),
              lambda: ops.paged_attention_sparse(q, kc, vc, plan, sel, 0.1, out=torch.empty(3, 4, 64, device=DEV)),
              lambda: ops.summarize_blocks(kc, plan, bounds[0][:2], bounds[1][:2]),
              lambda: ops.summarize_blocks(kc, plan, bounds[0], bounds[1], key_scale=sc),
              lambda: ops.select_blocks(q, plan, bounds[0][:, :1], bounds[1]),
              lambda: ops.select_blocks(q, plan, *bounds, out=sel[:, :, :2])):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(NotImplementedError):
        ops.SharedPrefixPlan(g["table"], g["cu"], g["lk"], 3, 4, 2, 96, 16)
    rope = ops.RotaryEmbedding(64, device=DEV)
    qkv = torch.zeros(3, 8 * 64, dtype=torch.bfloat16, device=DEV)
    pos, slots = torch.zeros(3, dtype=torch.int64, device=DEV), torch.arange(3, dtype=torch.int32, device=DEV)
    for f in (lambda: ops.rope_append(qkv, 4, 2, pos, rope, kc[:, :, :1], vc, slots),
              lambda: ops.rope_append(qkv, 4, 2, pos, rope, kc, vc, slots[:2]),
              lambda: ops.rope_append(qkv, 4, 2, pos[:2], rope, kc, vc, slots),
              lambda: ops.rope_append(qkv, 4, 2, pos, rope, kc, vc, slots, key_scale=sc),
              lambda: ops.rope_append(qkv, 4, 2, pos, rope, kc, vc, slots, kv_layout="nhd"),
              lambda: ops.rope_append(qkv, 4, 2, pos, rope, kc, vc, slots, q_out=qkv.view(3, 8, 64)[:, 1:5])):
        with pytest.raises(ValueError):
            f()


def test_backends_refuse_prefixes_seen_in_both_directions():
    model = make_model(8, 4, 128, 1, aia_rope=False)
    for options in (dict(attn_share_prefixes=True), dict(attn_sparse_blocks=4)):
        for k in ("attn_share_prefixes", "attn_sparse_blocks"):
            setattr(model, k, options.get(k, 0))
        backend, caches = registry.build_attention_backend(model, "paged", 4, 16)
        ctx, _ = make_context(backend, caches, [([0, 1], 0, 20)], 16)
        ctx.aia_prefix_lens = [5]
        with pytest.raises(NotImplementedError, match="both directions"):
            backend.attention(0, torch.zeros(20, 8 * 128, dtype=torch.bfloat16, device=DEV), ctx)
