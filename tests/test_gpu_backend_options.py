"""The GQA backend as models without rotary positions and requests with
prefixes use it, layer after layer."""
import pytest
import torch

from auto_infer_amd.attention import registry
from auto_infer_amd.attention.base import ForwardContext
from auto_infer_amd.attention.layers import rms_norm
from auto_infer_amd.block_allocator import KVCacheManager, prefix_seed
from oracle import long_context as oracle
from oracle.paged_attn import kv_write

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def make_model(hq, hkv, d, layers, norm=False, seed=0, kv_dtype="bf16", **options):
    gen = torch.Generator().manual_seed(seed)
    hidden, w = hq * d, {}
    for i in range(layers):
        p = f"model.layers.{i}.self_attn."
        w[p + "qkv_proj.weight"] = torch.randn((hq + 2 * hkv) * d, hidden, generator=gen) / hidden ** 0.5
        w[p + "o_proj.weight"] = torch.eye(hidden)
        if norm:
            w[p + "q_norm.weight"] = 1 + 0.2 * torch.randn(d, generator=gen)
            w[p + "k_norm.weight"] = 1 + 0.2 * torch.randn(d, generator=gen)

    class Model:
        ATTENTION_FAMILY, KV_CACHE_DTYPE = "gqa_hip", kv_dtype
        n_q_local, n_kv_local, device, dtype = hq, hkv, DEV, torch.bfloat16
        layer_prefix = staticmethod(lambda i: f"model.layers.{i}.")

        class cfg:
            head_dim, num_layers, rms_eps = d, layers, 1e-6
    Model.w = {k: t.bfloat16().to(DEV) for k, t in w.items()}
    for name, x in options.items():
        setattr(Model, name, x)
    return Model


def make_context(backend, caches, rows, bs):
    """rows: (blocks, computed tokens, new tokens); no cos / sin."""
    slots, pos, cu, kv, acc = [], [], [], [], 0
    bt = torch.zeros(len(rows), max(len(b) for b, _, _ in rows), dtype=torch.int32)
    for i, (blocks, done, n) in enumerate(rows):
        bt[i, :len(blocks)] = torch.tensor(blocks)
        slots += [blocks[p // bs] * bs + p % bs for p in range(done, done + n)]
        pos += list(range(done, done + n))
        acc += n
        cu.append(acc)
        kv.append(done + n)
    ctx = ForwardContext(
        token_ids=torch.zeros(acc, dtype=torch.long, device=DEV), positions=torch.tensor(pos, device=DEV),
        slot_mapping=torch.tensor(slots, dtype=torch.int32, device=DEV), block_table=bt.to(DEV), cu_seqlens_q=cu,
        seqlens_kv=kv, attn_mask=None, attn_backend=backend, kv_caches=caches,
        is_decode=all(n == 1 for _, _, n in rows))
    ctx.aia_slots_from_block_table = True
    return ctx, slots


@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("hq,hkv,d", [(8, 4, 128), (14, 2, 64)])
def test_a_model_that_tells_positions_by_the_bias_alone(hq, hkv, d, norm, kv_dtype):
    slopes = torch.exp2(-8.0 * torch.arange(1, hq + 1) / hq)
    model = make_model(hq, hkv, d, 1, norm, seed=d, kv_dtype=kv_dtype, aia_rope=False, alibi_slopes=slopes.to(DEV))
    bs, nb = 16, 40
    backend, caches = registry.build_attention_backend(model, "paged", nb, bs)
    gen = torch.Generator().manual_seed(1)
    perm = torch.randperm(nb, generator=gen).tolist()
    tables, done = [perm[:14], perm[14:28]], [0, 0]
    keys, values = (torch.zeros(nb, bs, hkv, d, dtype=torch.bfloat16) for _ in range(2))
    fp8 = [[torch.zeros(nb, bs, hkv, d, dtype=torch.float64), torch.full((nb, hkv), -127)] for _ in range(2)]
    p = "model.layers.0.self_attn."
    for new in ((20, 150), (1, 1), (70, 1), (1, 1)):
        ctx, slots = make_context(backend, caches, list(zip(tables, done, new)), bs)
        assert ctx.cos is None and ctx.sin is None
        x = torch.randn(sum(new), hq * d, generator=gen).bfloat16().to(DEV)
        out = backend.attention(0, x, ctx).view(-1, hq, d).cpu().double()
        qkv = x @ model.w[p + "qkv_proj.weight"].t()
        q, k, v = (t.reshape(sum(new), -1, d) for t in qkv.split((hq * d, hkv * d, hkv * d), -1))
        if norm:
            q, k = (rms_norm(t, model.w[p + n], 1e-6) for t, n in ((q, "q_norm.weight"), (k, "k_norm.weight")))
        if kv_dtype == "fp8":
            for rows, (vals, exps) in zip((k.cpu(), v.cpu()), fp8):
                oracle.write_kv_fp8(rows, vals, exps, slots)
            keys, values = (c * torch.exp2(e.double())[:, None, :, None] for c, e in fp8)
        else:
            kv_write(k.cpu(), v.cpu(), keys, values, torch.tensor(slots))
            assert torch.equal(caches[0][0].cpu(), keys) and torch.equal(caches[0][1].cpu(), values)
        ref, bound = oracle.scored_attention(q.cpu(), keys, values, ctx.block_table.cpu(), ctx.cu_seqlens_q,
                                             ctx.seqlens_kv, d ** -0.5, 0.0, slopes)
        assert bool(((out - ref).abs() <= bound).all())
        done = [a + b for a, b in zip(done, new)]


def forward(backend, caches, layers, emb, tokens, done, n, blocks, prefix, bs):
    """Rows [done, done + n) of one request through all layers (with residuals);
    returns each layer's (q, attention output) and the context."""
    ctx, _ = make_context(backend, caches, [(blocks, done, n)], bs)
    ctx.aia_prefix_lens = [prefix]
    x = emb[torch.tensor(tokens[done:done + n])].to(DEV)
    rows = []
    for layer in range(layers):
        attn, backend_attn = [], backend._attn

        def spy(i, q, k, v, c):
            attn.append(backend_attn(i, q, k, v, c))
            rows.append((q.clone(), attn[-1].clone()))
            return attn[-1]
        backend._attn = spy
        x = x + backend.attention(layer, x, ctx)
        backend._attn = backend_attn
    return rows, ctx


@pytest.mark.parametrize("hq,hkv,d", [(8, 4, 128), (14, 2, 64)])
def test_requests_with_a_prefix_share_blocks_through_two_layers(hq, hkv, d):
    """From the second layer on a block below the prefix depends on all of it:
    requests of the same prefix find the same keys and values, others must not
    share, and a chunk that ends inside the prefix is refused."""
    bs, nb, layers, prefix, total = 16, 40, 2, 40, 70
    model = make_model(hq, hkv, d, layers, seed=3, aia_rope=False, alibi_slopes=torch.full((hq,), 0.01, device=DEV))
    backend, caches = registry.build_attention_backend(model, "paged", nb, bs)
    gen = torch.Generator().manual_seed(5)
    emb = torch.randn(100, hq * d, generator=gen).bfloat16()
    a = torch.randint(100, (total,), generator=gen).tolist()
    other = a[:20] + [(t + 1) % 100 for t in a[20:prefix]] + a[prefix:]     # the same first block
    same = a[:prefix] + [(t + 1) % 100 for t in a[prefix:]]                 # the same prefix
    manager = KVCacheManager(nb, bs)
    tables = []
    for tokens in (a, other, same):
        hits = manager.match_prefix(tokens, prefix_seed(tokens, prefix))
        assert hits == (tables[0][:2] if tokens is same else [])
        manager.free(hits)
        tables.append(manager.allocate(total))
        forward(backend, caches, layers, emb, tokens, 0, total, tables[-1], prefix, bs)
        manager.register_prefix(tokens, tables[-1], prefix_seed(tokens, prefix))
    first = [caches[1][:, t[0]].float() for t in tables]
    assert (first[0] - first[1]).abs().max().item() > 0.05       # the second layer's first block
    for layer in range(layers):
        assert torch.equal(caches[layer][:, tables[0][:2]], caches[layer][:, tables[2][:2]])
    # the rest of a prompt behind two shared blocks, in one chunk that ends the prefix
    hits = manager.match_prefix(same, prefix_seed(same, prefix))
    table = hits + manager.allocate(total - len(hits) * bs)
    before = [caches[layer][:, hits].clone() for layer in range(layers)]
    rows, ctx = forward(backend, caches, layers, emb, same, len(hits) * bs, total - len(hits) * bs, table, prefix, bs)
    slopes = torch.full((hq,), 0.01)
    for layer, (q, out) in enumerate(rows):
        assert torch.equal(caches[layer][:, hits], before[layer])
        ref, bound = oracle.scored_attention(q.cpu(), caches[layer][0].cpu(), caches[layer][1].cpu(),
                                             ctx.block_table.cpu(), ctx.cu_seqlens_q, ctx.seqlens_kv, d ** -0.5, 0.0,
                                             slopes, [prefix])
        assert bool(((out.cpu().double() - ref).abs() <= bound).all())
    with pytest.raises(ValueError, match="first chunk"):
        forward(backend, caches, layers, emb, a, 0, prefix - 1, table, prefix, bs)


def test_checked_plans_read_device_prefixes_back(monkeypatch):
    model = make_model(4, 2, 64, 1, aia_rope=False)
    backend, caches = registry.build_attention_backend(model, "paged", 4, 16)
    x = torch.zeros(20, 256, dtype=torch.bfloat16, device=DEV)
    monkeypatch.setenv("AIA_CHECK_PLAN", "1")
    for prefix, fits in ((20, True), (21, False)):
        ctx, _ = make_context(backend, caches, [([0, 1], 0, 20)], 16)
        ctx.aia_prefix_lens = torch.tensor([prefix], dtype=torch.int32, device=DEV)
        if fits:
            backend.attention(0, x, ctx)
        else:
            with pytest.raises(ValueError, match="first chunk"):
                backend.attention(0, x, ctx)
