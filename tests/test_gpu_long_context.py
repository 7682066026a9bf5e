"""8-bit caches, modified scores and rotary positions together, as a server uses
them: through the GQA backend over prompt chunks and decode steps, from a HIP
graph, on streams of their own, and the calls that are refused."""
import numpy as np
import pytest
import torch

from auto_infer_amd import ops, packing, workloads
from auto_infer_amd.attention import registry
from auto_infer_amd.attention.base import ForwardContext
from auto_infer_amd.attention.gqa import GqaHipBackend
from auto_infer_amd.execution import BatchPlan, RequestView, ScheduledRequest
from auto_infer_amd.graph import DecodeGraph
from oracle import long_context as oracle
from oracle import pack
from oracle.paged_attn import kv_write

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


class Request:
    def __init__(self, blocks, prefix):
        self.blocks, self.prefix, self.done = blocks, prefix, 0


def context(backend, caches, rows, bs):
    """rows: (request, new tokens)."""
    slots, pos, cu, kv, acc = [], [], [], [], 0
    bt = torch.zeros(len(rows), max(len(r.blocks) for r, _ in rows), dtype=torch.int32)
    for i, (r, n) in enumerate(rows):
        bt[i, :len(r.blocks)] = torch.tensor(r.blocks)
        for p in range(r.done, r.done + n):
            slots.append(r.blocks[p // bs] * bs + p % bs)
            pos.append(p)
        acc += n
        cu.append(acc)
        kv.append(r.done + n)
    ctx = ForwardContext(
        token_ids=torch.zeros(acc, dtype=torch.long, device=DEV),
        positions=torch.tensor(pos, device=DEV),
        slot_mapping=torch.tensor(slots, dtype=torch.int32, device=DEV), block_table=bt.to(DEV),
        cu_seqlens_q=cu, seqlens_kv=kv, attn_mask=None, attn_backend=backend, kv_caches=caches,
        is_decode=all(n == 1 for _, n in rows))
    ctx.aia_slots_from_block_table = True
    ctx.aia_prefix_lens = torch.tensor([r.prefix for r, _ in rows], dtype=torch.int32, device=DEV)
    return ctx, slots


@pytest.mark.parametrize("kv_dtype", ["fp8", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 4, 128), (14, 2, 64)])
def test_backend_over_chunks_and_decode_steps(kv_dtype, hq, hkv, d):
    """A backend with all of it: every step's caches equal the oracle's writes of
    the same K/V rows, and its output (an identity o_proj) is within the bound."""
    gen = torch.Generator().manual_seed(d)
    bs, nb, layers = 16, 80, 2
    hidden = hq * d
    w = {}
    for i in range(layers):
        p = f"model.layers.{i}.self_attn."
        w[p + "qkv_proj.weight"] = (torch.randn((hq + 2 * hkv) * d, hidden, generator=gen) / hidden ** 0.5)
        w[p + "q_norm.weight"] = 1 + 0.2 * torch.randn(d, generator=gen)
        w[p + "k_norm.weight"] = 1 + 0.2 * torch.randn(d, generator=gen)
        w[p + "o_proj.weight"] = torch.eye(hidden)
    w = {k: t.bfloat16().to(DEV) for k, t in w.items()}
    slopes = torch.exp2(-8.0 * torch.rand(hq, generator=gen))

    class Model:
        ATTENTION_FAMILY, KV_CACHE_DTYPE = "gqa_hip", kv_dtype
        attn_softcap = 20.0
        alibi_slopes = slopes.to(DEV)
        aia_rope = ops.RotaryEmbedding(d, rotary_dim=d // 2, interleaved=True, device=DEV,
                                       scaling={"type": "linear", "factor": 2.0})
        n_q_local, n_kv_local, device, dtype = hq, hkv, DEV, torch.bfloat16
        layer_prefix = staticmethod(lambda i: f"model.layers.{i}.")

        class cfg:
            head_dim, num_layers, rms_eps = d, layers, 1e-6
    Model.w = w
    backend, caches = registry.build_attention_backend(Model, "paged", nb, bs)
    assert isinstance(backend, GqaHipBackend) and len(caches) == layers
    perm = torch.randperm(nb, generator=gen).tolist()
    reqs = [Request(perm[20 * i:20 * i + 20], pre) for i, pre in enumerate((0, 37, 5))]
    ref = []
    for _ in range(layers):
        if kv_dtype == "fp8":
            ref.append([[torch.zeros(nb, bs, hkv, d, dtype=torch.float64), torch.full((nb, hkv), -127)]
                        for _ in range(2)])
        else:
            ref.append([torch.zeros(nb, bs, hkv, d, dtype=torch.bfloat16) for _ in range(2)])
    steps = [[(0, 50), (1, 150)], [(0, 1), (1, 70), (2, 9)], [(0, 1), (1, 1), (2, 1)], [(0, 2), (1, 1), (2, 130)],
             [(0, 1), (1, 1), (2, 1)]]
    for step in steps:
        rows = [(reqs[i], n) for i, n in step]
        ctx, slots = context(backend, caches, rows, bs)
        T = len(slots)
        for layer in range(layers):
            x = torch.randn(T, hidden, generator=gen).bfloat16().to(DEV)
            out = backend.attention(layer, x, ctx)
            p = f"model.layers.{layer}.self_attn."
            qkv = x @ w[p + "qkv_proj.weight"].t()
            q, k, v = (t.cpu() for t in ops.rope_qk(qkv, hq, hkv, ctx.positions, Model.aia_rope,
                                                    w[p + "q_norm.weight"], w[p + "k_norm.weight"], 1e-6))
            if kv_dtype == "fp8":
                for rows_, (vals, exps), cache, scale in ((k, ref[layer][0], *caches[layer][::2]),
                                                          (v, ref[layer][1], *caches[layer][1::2])):
                    oracle.write_kv_fp8(rows_, vals, exps, slots)
                    assert torch.equal(cache.cpu().double(), vals)
                    assert torch.equal(scale.view(torch.uint8).cpu().int() - 127, exps.int())
                keys, values = (c[0] * torch.exp2(c[1].double())[:, None, :, None] for c in ref[layer])
            else:
                kv_write(k, v, ref[layer][0], ref[layer][1], torch.tensor(slots))
                assert torch.equal(caches[layer][0].cpu(), ref[layer][0])
                assert torch.equal(caches[layer][1].cpu(), ref[layer][1])
                keys, values = ref[layer]
            want, bound = oracle.scored_attention(q, keys, values, ctx.block_table.cpu(), ctx.cu_seqlens_q,
                                                  ctx.seqlens_kv, d ** -0.5, 20.0, slopes,
                                                  ctx.aia_prefix_lens.tolist())
            far = (out.view(T, hq, d).cpu().double() - want).abs()
            assert bool((far <= bound).all()), (far / bound.clamp(min=1e-30)).max().item()
        for i, n in step:
            reqs[i].done += n


def test_decode_graph_over_8_bit_caches():
    """A captured gear (planner, writes, attention) replayed over steps with
    eager work between them; scratch rows of the gear included."""
    rng = np.random.default_rng(1)
    gear, maxb, bs, nb, hq, hkv, d, L = 8, 16, 16, 200, 16, 8, 128, 2
    stager = packing.DecodeInputStager(
        tid=torch.zeros(gear, dtype=torch.long, device=DEV),
        positions=torch.zeros(gear, dtype=torch.long, device=DEV),
        slots=torch.zeros(gear, dtype=torch.int32, device=DEV),
        block_table=torch.zeros(gear, maxb, dtype=torch.int32, device=DEV), block_size=bs, scratch0=nb - gear)
    g = torch.Generator(device=DEV).manual_seed(3)
    backend = GqaHipBackend(hq, hkv, d, d ** -0.5, L, DEV, torch.bfloat16, kv_dtype="fp8")
    caches = backend.alloc_kv_caches(nb, bs)
    for k, v, ks, vs in caches:           # earlier contents
        rows = [torch.randn(nb * bs, hkv, d, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
        ops.write_kv_fp8(*rows, k, v, ks, vs, torch.arange(nb * bs, dtype=torch.int32, device=DEV))
    ref = [[(c.cpu().double(), s.view(torch.uint8).cpu().int() - 127) for c, s in ((k, ks), (v, vs))]
           for k, v, ks, vs in caches]
    slopes = torch.exp2(-torch.arange(1, hq + 1).float() / 2)
    dg = DecodeGraph(stager, caches, num_q_heads=hq, num_kv_heads=hkv, softcap=30.0,
                     alibi_slopes=slopes.to(DEV))
    free = list(range(nb - gear))
    rng.shuffle(free)
    reqs = {}
    for i, lk in enumerate([5, 40, 17, 100, 63]):
        reqs[f"r{i}"] = dict(pos=lk - 1, blocks=[free.pop() for _ in range((lk + 5 + bs - 1) // bs)])
    for step in range(5):
        views = {rid: RequestView(rid, tuple(range(r["pos"] + 1)), r["pos"], 1, 1, ())
                 for rid, r in reqs.items()}
        plan = BatchPlan.make([ScheduledRequest(rid, 1, False, tuple(r["blocks"])) for rid, r in reqs.items()],
                              views, {rid: r["blocks"] for rid, r in reqs.items()})
        dg.q.copy_(torch.randn(dg.q.shape, generator=g, device=DEV, dtype=torch.bfloat16))
        for buf in (dg.k_new, dg.v_new):  # growing rows: scales grow now and then
            buf.copy_(torch.randn(buf.shape, generator=g, device=DEV, dtype=torch.bfloat16) * 2.0 ** step)
        torch.cuda.synchronize()
        dg.stage(plan)
        if dg.graph is None:
            dg.capture()
        else:
            dg.replay()
        torch.cuda.synchronize()
        exp = pack.decode_stage(plan, gear=gear, max_blocks=maxb, block_size=bs, scratch0=nb - gear)
        for layer in range(L):
            for rows, (vals, exps) in zip((dg.k_new[layer].cpu(), dg.v_new[layer].cpu()), ref[layer]):
                oracle.write_kv_fp8(rows, vals, exps, exp["slots"].tolist())
            for (vals, exps), c, s in zip(ref[layer], caches[layer][:2], caches[layer][2:]):
                assert torch.equal(c.cpu().double(), vals)
                assert torch.equal(s.view(torch.uint8).cpu().int() - 127, exps.int())
            keys, values = (v * torch.exp2(e.double())[:, None, :, None] for v, e in ref[layer])
            want, bound = oracle.scored_attention(dg.q[layer].cpu(), keys, values,
                                                  torch.as_tensor(exp["block_table"]),
                                                  list(range(1, gear + 1)), list(exp["kv_lengths"]), d ** -0.5,
                                                  30.0, slopes)
            assert bool(((dg.out[layer].cpu().double() - want).abs() <= bound).all())
        for r in reqs.values():
            r["pos"] += 1


def step_inputs(seed, lqs, lks, hq, hkv, d, bs):
    step = workloads.make_gqa_step(lqs=lqs, lks=lks, num_q_heads=hq, num_kv_heads=hkv, head_dim=d,
                                   block_size=bs, seed=seed)
    nb = step.k_cache.shape[0]
    backend = GqaHipBackend(hq, hkv, d, d ** -0.5, 1, DEV, torch.bfloat16, kv_dtype="fp8")
    cache = backend.alloc_kv_caches(nb, bs)[0]
    ops.write_kv_fp8(step.k_cache.view(-1, hkv, d).to(DEV), step.v_cache.view(-1, hkv, d).to(DEV), *cache,
                     torch.arange(nb * bs, dtype=torch.int32, device=DEV))
    return step, cache


def test_two_steps_in_flight_on_two_streams():
    """Two steps' plans, writes and attention interleaved on two streams give
    what each gives alone."""
    steps = [step_inputs(1, [1] * 9, [300 + 50 * i for i in range(9)], 16, 8, 128, 16),
             step_inputs(2, [130, 70, 1], [600, 70, 900], 28, 4, 128, 64)]
    heads = [(16, 8), (28, 4)]
    pre = torch.tensor([10, 0, 40], dtype=torch.int32, device=DEV)

    def run(i, stream):
        step, cache = steps[i]
        with torch.cuda.stream(stream):
            plan = ops.AttentionPlan.from_lists(step.block_table.to(DEV), step.cu_seqlens_q, step.seqlens_kv,
                                                *heads[i], 128, cache[0].shape[1],
                                                prefix_lens=pre if i else None)
            ops.write_kv_fp8(step.k_new.to(DEV), step.v_new.to(DEV), *cache, step.slot_mapping.to(DEV))
            return ops.paged_attention_gqa(step.q.to(DEV), cache[0], cache[1], plan, step.scale,
                                           key_scale=cache[2], value_scale=cache[3], softcap=25.0 * i)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    alone = []
    for i in range(2):
        alone.append(run(i, streams[i]))
        torch.cuda.synchronize()
    for _ in range(6):
        outs = [run(0, streams[0]), run(1, streams[1]), run(0, streams[0]), run(1, streams[1])]
        torch.cuda.synchronize()
        for i, o in enumerate(outs):
            assert torch.equal(o, alone[i % 2])


def test_an_empty_step_and_strided_outputs():
    step, cache = step_inputs(3, [2, 140], [50, 140], 14, 2, 64, 16)
    plan = ops.AttentionPlan.from_lists(step.block_table.to(DEV), step.cu_seqlens_q, step.seqlens_kv, 14, 2, 64, 16)
    q = step.q.to(DEV)
    kw = dict(key_scale=cache[2], value_scale=cache[3], softcap=9.0)
    want = ops.paged_attention_gqa(q, cache[0], cache[1], plan, step.scale, **kw)
    wide = torch.full((142, 16, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    got = ops.paged_attention_gqa(q, cache[0], cache[1], plan, step.scale, out=wide[:, 1:15, 64:], **kw)
    assert torch.equal(got, want)
    rest = wide.clone()
    rest[:, 1:15, 64:] = 3.0
    assert bool((rest == 3.0).all())
    sq = torch.empty(142, 20, 64, dtype=torch.bfloat16, device=DEV)[:, 3:17]
    sq.copy_(q)
    assert torch.equal(ops.paged_attention_gqa(sq, cache[0], cache[1], plan, step.scale, **kw), want)
    none = ops.AttentionPlan(torch.zeros(1, 1, dtype=torch.int32, device=DEV),
                             torch.zeros(1, dtype=torch.int32, device=DEV),
                             torch.zeros(0, dtype=torch.int32, device=DEV), 0, 14, 2, 64, 16)
    assert ops.paged_attention_gqa(q[:0], cache[0], cache[1], none, step.scale, **kw).shape == (0, 14, 64)


def test_query_lengths_that_do_not_fit_fill_the_output_with_nan():
    step, cache = step_inputs(4, [1, 1], [50, 20], 16, 8, 128, 16)
    cu = torch.tensor([0, 700, 1400], dtype=torch.int32, device=DEV)
    kv = torch.tensor([700, 700], dtype=torch.int32, device=DEV)
    for pre in (None, torch.zeros(2, dtype=torch.int32, device=DEV)):
        plan = ops.AttentionPlan(step.block_table.to(DEV), cu, kv, 2, 16, 8, 128, 16, prefix_lens=pre)
        out = ops.paged_attention_gqa(step.q.to(DEV), cache[0], cache[1], plan, step.scale,
                                      key_scale=cache[2], value_scale=cache[3], softcap=5.0)
        assert bool(torch.isnan(out.float()).all())
        with pytest.raises(ValueError, match="planner overflow"):
            plan.status()


def test_refused_calls():
    step, cache = step_inputs(5, [1, 3], [50, 20], 16, 8, 128, 16)
    kc, vc, ks, vs = cache
    plan = ops.AttentionPlan.from_lists(step.block_table.to(DEV), step.cu_seqlens_q, step.seqlens_kv, 16, 8, 128, 16)
    q, kn, vn = step.q.to(DEV), step.k_new.to(DEV), step.v_new.to(DEV)
    slots = step.slot_mapping.to(DEV)
    kb, vb = step.k_cache.to(DEV), step.v_cache.to(DEV)

    def attn(err, match, *a, **k):
        with pytest.raises(err, match=match):
            ops.paged_attention_gqa(*a, **k)
    f8 = dict(key_scale=ks, value_scale=vs)
    attn(ValueError, "value_scale", q, kc, vc, plan, 1.0, key_scale=ks)
    attn(ValueError, "key_cache must be", q, kc, vc, plan, 1.0)
    attn(ValueError, "key_cache must be", q, kb, vb, plan, 1.0, **f8)
    attn(ValueError, "write_kv_fp8", q, kc, vc, plan, 1.0, key_new=kn, value_new=vn, **f8)
    attn(NotImplementedError, "NZ", q, kc, vc, plan, 1.0, kv_layout="nz", **f8)
    attn(ValueError, "key_scale must be a contiguous", q, kc, vc, plan, 1.0, key_scale=ks[:-1], value_scale=vs)
    attn(ValueError, "key_scale must be torch", q, kc, vc, plan, 1.0, key_scale=ks.view(torch.uint8), value_scale=vs)
    attn(ValueError, "softcap", q, kb, vb, plan, 1.0, softcap=-1.0)
    attn(ValueError, "softcap", q, kb, vb, plan, 1.0, softcap=float("nan"))
    attn(ValueError, "softcap", q, kb, vb, plan, 1.0, softcap=float("inf"))
    attn(ValueError, "softcap", q, kb, vb, plan, 1.0, softcap=1e-31)
    attn(ValueError, "another shape", q[..., :64].contiguous(), kb[..., :64].contiguous(), vb[..., :64].contiguous(),
         plan, 1.0, softcap=1.0)
    attn(ValueError, "alibi_slopes must hold 16", q, kb, vb, plan, 1.0,
         alibi_slopes=torch.ones(8, device=DEV))
    attn(ValueError, "alibi_slopes must be", q, kb, vb, plan, 1.0,
         alibi_slopes=torch.ones(16, device=DEV, dtype=torch.bfloat16))
    attn(ValueError, "alibi_slopes must be on the GPU", q, kb, vb, plan, 1.0, alibi_slopes=torch.ones(16))
    attn(ValueError, "scale", q, kb, vb, plan, 0.0, softcap=1.0)
    with pytest.raises(ValueError, match="prefix_lens"):
        ops.AttentionPlan.from_lists(step.block_table.to(DEV), step.cu_seqlens_q, step.seqlens_kv, 16, 8, 128, 16,
                                     prefix_lens=torch.zeros(3, dtype=torch.int32, device=DEV))
    with pytest.raises(NotImplementedError, match="head_dim"):
        ops.AttentionPlan.from_lists(step.block_table.to(DEV), step.cu_seqlens_q, step.seqlens_kv, 16, 1, 512, 16,
                                     prefix_lens=torch.zeros(2, dtype=torch.int32, device=DEV))

    def write(match, *a):
        with pytest.raises(ValueError, match=match):
            ops.write_kv_fp8(*a)
    write("key_cache must be", kn, vn, kb, vb, ks, vs, slots)
    write("key_scale must be", kn, vn, kc, vc, ks.view(torch.uint8), vs, slots)
    write("do not match", kn[:, :4], vn, kc, vc, ks, vs, slots)
    write("slot_mapping", kn, vn, kc, vc, ks, vs, slots[:-1])
    write("slot_mapping must be", kn, vn, kc, vc, ks, vs, slots.long())
    write("value must match", kn, vn[:-1], kc, vc, ks, vs, slots)
    write("without value", kn, None, kc, vc, ks, None, slots)
    write("value_cache must match", kn, vn, kc, vc[:-1], ks, vs[:-1], slots)
    write("rows .heads, dim. must be contiguous", kn.transpose(0, 1).contiguous().transpose(0, 1), vn, kc, vc, ks, vs,
          slots)
    one = torch.zeros(1, 16, 128, dtype=torch.bfloat16, device=DEV)[:, ::2]      # a single token's rows too
    write("rows .heads, dim. must be contiguous", one, None, kc, None, ks, None, slots[:1])
    write("must be on the GPU", kn.cpu(), vn, kc, vc, ks, vs, slots)
    with pytest.raises(NotImplementedError, match="head_dim"):
        ops.write_kv_fp8(kn[..., :32].contiguous(), None, kc[..., :32].contiguous(), None, ks, None, slots)

    rope = ops.RotaryEmbedding(128, device=DEV)
    qkv = torch.zeros(4, 32 * 128, dtype=torch.bfloat16, device=DEV)
    pos = torch.zeros(4, dtype=torch.int64, device=DEV)
    for match, args, kw in (("width", (qkv, 16, 9, pos, rope), {}),
                            ("positions must be", (qkv, 16, 8, pos.int(), rope), {}),
                            ("positions must hold", (qkv, 16, 8, pos[:3], rope), {}),
                            ("RotaryEmbedding", (qkv, 16, 8, pos, None), {}),
                            ("go together", (qkv, 16, 8, pos, rope, torch.ones(128, device=DEV).bfloat16()), {}),
                            ("k_out must have shape", (qkv, 16, 8, pos, rope),
                             dict(out=(torch.empty(4, 16, 128, device=DEV).bfloat16(),
                                       torch.empty(4, 4, 128, device=DEV).bfloat16()))),
                            ("16-byte aligned", (torch.zeros(4, 32 * 128 + 1, device=DEV).bfloat16()[:, 1:], 16, 8,
                                                 pos, rope), {})):
        with pytest.raises(ValueError, match=match):
            ops.rope_qk(*args, **kw)


def test_a_whole_layer_in_a_graph():
    """Rotary positions, 8-bit write, planner with prefixes and capped attention
    captured in one graph; every replay, with new inputs, lengths and prefixes
    and eager work between, equals the eager calls."""
    hq, hkv, d, bs, nb, T = 28, 4, 128, 16, 90, 150
    gen = torch.Generator(device=DEV).manual_seed(2)
    rope = ops.RotaryEmbedding(d, base=1e6, device=DEV)
    qkv = torch.empty(T, (hq + 2 * hkv) * d, dtype=torch.bfloat16, device=DEV)
    pos = torch.zeros(T, dtype=torch.int64, device=DEV)
    slots = torch.full((T,), -1, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 1, 141, T], dtype=torch.int32, device=DEV)
    kv = torch.tensor([1, 140, 9], dtype=torch.int32, device=DEV)
    pre = torch.zeros(3, dtype=torch.int32, device=DEV)
    table = torch.randperm(nb, generator=torch.Generator().manual_seed(3)).int().view(3, 30).to(DEV)
    backend = GqaHipBackend(hq, hkv, d, d ** -0.5, 1, DEV, torch.bfloat16, kv_dtype="fp8")
    cache, twin = backend.alloc_kv_caches(nb, bs)[0], backend.alloc_kv_caches(nb, bs)[0]
    plan = ops.AttentionPlan(table, cu, kv, T, hq, hkv, d, bs, prefix_lens=pre)
    outs = [torch.empty(T, hq, d, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    rotated = (torch.empty(T, hq, d, dtype=torch.bfloat16, device=DEV),
               torch.empty(T, hkv, d, dtype=torch.bfloat16, device=DEV))

    def layer(c, out):
        q, k, v = ops.rope_qk(qkv, hq, hkv, pos, rope, out=rotated)
        ops.write_kv_fp8(k, v, *c, slots)
        plan.replan()
        ops.paged_attention_gqa(q, c[0], c[1], plan, d ** -0.5, out=out, key_scale=c[2], value_scale=c[3],
                                softcap=15.0)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        qkv.zero_()
        layer(twin, outs[1])
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            layer(cache, outs[0])
    torch.cuda.synchronize()
    rng = np.random.default_rng(4)
    for c in twin:
        c.view(torch.uint8).zero_()
    for step in range(5):
        lens = [int(rng.integers(1, 300)), 140 + int(rng.integers(0, 300)), 9 + int(rng.integers(0, 300))]
        p, s = [], []
        for r, (n, lk) in enumerate(zip((1, 140, 9), lens)):
            p += list(range(lk - n, lk))
            s += [int(table[r, x // bs]) * bs + x % bs for x in range(lk - n, lk)]
        qkv.copy_(torch.randn(qkv.shape, generator=gen, device=DEV) * 2.0 ** step)
        pos.copy_(torch.tensor(p)), slots.copy_(torch.tensor(s, dtype=torch.int32))
        kv.copy_(torch.tensor(lens, dtype=torch.int32))
        pre.copy_(torch.tensor([int(rng.integers(0, lk + 1)) for lk in lens], dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            layer(twin, outs[1])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        for a, b in zip(cache, twin):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
