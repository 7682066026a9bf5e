"""GQA paged attention backend on the gfx950 kernels.

``GqaHipBackend`` is a drop-in for the reference's ``GqaFIABackend``
(auto_infer/layers/attention/gqa.py:52-94): same constructor arguments,
same KV-cache layout ``(2, num_blocks, block_size, n_kv, head_dim)`` per
layer (gqa.py:69-74), same sub-block math around the op pair (packed qkv
projection, optional Qwen3 QK-RMSNorm, NeoX RoPE, o_proj; gqa.py:27-49) and
the same op-pair seam ``_write_kv`` / ``_attn``.  Only the op pair differs:
the KV slot write and the split-K paged attention run as HIP kernels.
The backend is graph-capturable (no host sync, no allocation in ``_attn``
once the step's plan exists), so it serves both the "paged" and "graph"
modes.  With ``kv_layout="nz"`` it also takes the caches of the reference's
graph-mode backend (``GraphGqaBackend``, gqa.py:134-226): per layer a (k, v)
pair of (num_blocks, block_size, n_kv, head_dim) tensors whose memory is the
16-wide fractal NZ layout (viewed (num_blocks, n_kv * head_dim / 16,
block_size, 16) by npu_scatter_pa_kv_cache and FIA-v2, gqa.py:202-226).

Beyond the reference: ``kv_dtype="fp8"`` keeps the caches as e4m3 values with a
power-of-two scale per block and head, ``softcap`` / ``alibi_slopes`` modify the
scores, ``rope`` (an ``ops.RotaryEmbedding``) turns Q and K from
``ctx.positions`` instead of ``ctx.cos`` / ``ctx.sin`` (``rope=False``: a model
without rotary positions, Q and K stay as they are), and a context with
``aia_prefix_lens`` (one per request; a host list or device int32) lets all rows of a request
see its first keys.  ``share_prefixes=True`` reads the cache blocks that requests have in
common once for all of them (``ops.paged_attention_shared``; ``ctx.aia_group_ids`` names
the groups, else the first blocks do).  ``sparse_blocks=n`` lets every query token and KV
head attend n cache blocks that an upper bound of their scores selects
(``ops.select_blocks``), always the first ``sparse_sink`` and the last ``sparse_local``;
the layers' caches then carry the blocks' bounds.  With a ``rope``, one launch turns Q
and K and writes the caches (``ops.rope_append``) where the op pair is this class's own;
a replaced ``_write_kv`` or ``_attn`` is given K and V.
"""
import torch

from auto_infer_amd import ops
from auto_infer_amd.attention.base import AttentionBackend
from auto_infer_amd.attention.layers import lin, rms_norm, rotate_half
from auto_infer_amd.attention.metadata import step_plan, step_shared_plan, step_sparse_plan


class GqaHipBackend(AttentionBackend):

    def __init__(self, n_q_heads: int, n_kv_heads: int, head_dim: int, scale: float,
                 num_layers: int, device, dtype, w: dict = None, layer_prefix=None,
                 rms_eps=None, fuse_kv_write: bool = True, fuse_pre_attention: bool = True,
                 kv_layout: str = "nd", kv_dtype: str = "bf16", softcap: float = 0.0,
                 alibi_slopes=None, rope=None, share_prefixes: bool = False,
                 sparse_blocks: int = 0, sparse_sink: int = 1, sparse_local: int = 2):
        self.n_q_heads = n_q_heads
        self.n_kv_heads = n_kv_heads
        self.head_dim = head_dim
        self.scale = scale
        self.num_layers = num_layers
        self.device = device
        self.dtype = dtype
        self.w = w
        self.layer_prefix = layer_prefix or (lambda i: f"model.layers.{i}.")
        self.rms_eps = rms_eps
        # With fuse_kv_write, _write_kv defers the slot write to the attention
        # kernel of the following _attn (same cache contents, one launch less);
        # attention() always calls the two in that order.  The kernel writes
        # each new row at the slot its request's block table gives its
        # position, so the write is deferred only for contexts that declare
        # their slot_mapping equal to those slots
        # (ctx.aia_slots_from_block_table, set by this package's packers);
        # any other slot_mapping is written as given, by its own launch.
        self.fuse_kv_write = fuse_kv_write
        # With fuse_pre_attention, the split / QK-RMSNorm / RoPE steps run as
        # one in-place kernel over the qkv projection (bf16 rounding where the
        # torch ops round); q, k, v are then strided views of it.
        self.fuse_pre_attention = fuse_pre_attention
        if kv_layout not in ops.KV_LAYOUTS:
            raise ValueError(f"kv_layout must be one of {sorted(ops.KV_LAYOUTS)}")
        self.kv_layout = kv_layout
        if kv_dtype not in ("bf16", "fp8"):
            raise ValueError(f"kv_dtype must be bf16 or fp8, got {kv_dtype!r}")
        self.fp8 = kv_dtype == "fp8"
        if self.fp8 and kv_layout != "nd":
            raise NotImplementedError("8-bit caches have no NZ layout")
        self.scores = dict(softcap=softcap, alibi_slopes=alibi_slopes)
        if rope is not None and rope is not False and not isinstance(rope, ops.RotaryEmbedding):
            raise ValueError("rope must be an ops.RotaryEmbedding, False (no rotary positions) or None "
                             "(ctx.cos / ctx.sin)")
        self.rope = rope
        self.share_prefixes, self.sparse = bool(share_prefixes), None
        if sparse_blocks:
            if not (sparse_sink >= 0 and sparse_local >= 1 and sparse_sink + sparse_local <= sparse_blocks):
                raise ValueError(f"sparse_sink {sparse_sink} and sparse_local {sparse_local} do not fit "
                                 f"{sparse_blocks} blocks (sparse_local at least 1)")
            self.sparse = (int(sparse_blocks), int(sparse_sink), int(sparse_local))
        if self.share_prefixes or self.sparse:
            if self.share_prefixes and self.sparse:
                raise ValueError("share_prefixes and sparse_blocks exclude each other")
            if kv_layout != "nd":
                raise NotImplementedError("shared prefixes and sparse blocks have no NZ layout")
            if softcap != 0 or alibi_slopes is not None:
                raise NotImplementedError("shared prefixes and sparse blocks take no modified scores")
            self.fuse_kv_write = False      # the cache is written before it is read
        self._pending = None

    def alloc_kv_caches(self, num_blocks: int, block_size: int) -> list:
        if not self.sparse:
            return self._alloc(num_blocks, block_size)
        # per layer (k, v, ...) and the blocks' bounds and their scales
        shape = (num_blocks, self.n_kv_heads)
        return [(*cache, torch.zeros(*shape, 2, self.head_dim, device=self.device, dtype=torch.int8),
                 torch.zeros(shape, device=self.device, dtype=torch.uint8).view(ops.FP8_KV_SCALE))
                for cache in self._alloc(num_blocks, block_size)]

    def _alloc(self, num_blocks, block_size):
        if self.fp8:      # per layer (k, v, k scales, v scales)
            shape = (num_blocks, block_size, self.n_kv_heads, self.head_dim)

            def zeros(shape, dtype):      # byte 0: value 0, the smallest scale
                return torch.zeros(shape, device=self.device, dtype=torch.uint8).view(dtype)
            return [(zeros(shape, ops.FP8_KV), zeros(shape, ops.FP8_KV),
                     zeros((num_blocks, self.n_kv_heads), ops.FP8_KV_SCALE),
                     zeros((num_blocks, self.n_kv_heads), ops.FP8_KV_SCALE))
                    for _ in range(self.num_layers)]
        if self.kv_layout == "nz":      # GraphGqaBackend.alloc_kv_caches (gqa.py:195-204)
            shape = (num_blocks, block_size, self.n_kv_heads, self.head_dim)
            return [(torch.zeros(shape, device=self.device, dtype=self.dtype),
                     torch.zeros(shape, device=self.device, dtype=self.dtype))
                    for _ in range(self.num_layers)]
        shape = (2, num_blocks, block_size, self.n_kv_heads, self.head_dim)
        return [torch.zeros(shape, device=self.device, dtype=self.dtype)
                for _ in range(self.num_layers)]

    def _write(self, k, v, cache, slot_mapping):
        if self.fp8:
            ops.write_kv_fp8(k, v, *cache[:4], slot_mapping)
        elif self.kv_layout == "nz":
            ops.write_kv_nz(k, v, cache[0], cache[1], slot_mapping)
        else:
            ops.write_kv(k, v, cache[0], cache[1], slot_mapping)

    def attention(self, layer_idx: int, x: torch.Tensor, ctx) -> torch.Tensor:
        T = x.shape[0]
        n_q, n_kv, hd = self.n_q_heads, self.n_kv_heads, self.head_dim
        w = self.w
        p = self.layer_prefix(layer_idx) + "self_attn."
        qkv = lin(x, w[p + "qkv_proj.weight"], w.get(p + "qkv_proj.bias"))
        qn = w.get(p + "q_norm.weight")
        if self.rope is None and (ctx.cos is None or ctx.sin is None):
            raise ValueError("the context has no cos / sin: give the backend a rope, or rope=False "
                             "for a model without rotary positions")
        if self.rope is not None and self.rope is not False:
            if self.fuse_pre_attention and self._own_pair() and not self._deferred(T, ctx):
                cache = ctx.kv_caches[layer_idx]
                scales = dict(key_scale=cache[2], value_scale=cache[3]) if self.fp8 else {}
                q = ops.rope_append(qkv, n_q, n_kv, ctx.positions, self.rope, cache[0], cache[1],
                                    ctx.slot_mapping, qn,
                                    w.get(p + "k_norm.weight") if qn is not None else None,
                                    self.rms_eps if self.rms_eps is not None else 1e-6,
                                    kv_layout=self.kv_layout, **scales)
                o = self._attn(layer_idx, q, None, None, ctx).reshape(T, n_q * hd)
                return lin(o, w[p + "o_proj.weight"])
            q, k, v = ops.rope_qk(qkv, n_q, n_kv, ctx.positions, self.rope, qn,
                                  w.get(p + "k_norm.weight") if qn is not None else None,
                                  self.rms_eps if self.rms_eps is not None else 1e-6)
        elif self.rope is None and self._fusable(qkv, ctx):
            q, k, v = ops.qk_norm_rope(qkv, n_q, n_kv, ctx.cos, ctx.sin, qn,
                                       w.get(p + "k_norm.weight") if qn is not None else None,
                                       self.rms_eps if self.rms_eps is not None else 1e-6,
                                       head_dim=hd)
        else:
            q, k, v = qkv.split((n_q * hd, n_kv * hd, n_kv * hd), dim=-1)
            q = q.view(T, n_q, hd)
            k = k.view(T, n_kv, hd)
            v = v.view(T, n_kv, hd)
            if qn is not None:
                q = rms_norm(q, qn, self.rms_eps)
                k = rms_norm(k, w[p + "k_norm.weight"], self.rms_eps)
            if self.rope is None:
                q = q * ctx.cos + rotate_half(q) * ctx.sin
                k = k * ctx.cos + rotate_half(k) * ctx.sin
        self._write_kv(layer_idx, k, v, ctx)
        o = self._attn(layer_idx, q, k, v, ctx).reshape(T, n_q * hd)
        return lin(o, w[p + "o_proj.weight"])

    def _fusable(self, qkv, ctx):
        T = qkv.shape[0]
        def aligned(t):          # 16-byte accesses: 8-element strides, 16-byte base
            return t.stride(0) % 8 == 0 and t.data_ptr() % 16 == 0
        hd = self.head_dim
        return (self.fuse_pre_attention and hd in (128, 64) and qkv.dtype == torch.bfloat16
                and qkv.is_cuda and qkv.stride(-1) == 1 and aligned(qkv)
                and all(t.dtype == torch.bfloat16 and t.numel() == T * hd and t.stride(-1) == 1
                        and aligned(t) for t in (ctx.cos, ctx.sin)))

    def _own_pair(self):
        """Whether the op pair is this class's: one that replaces either gets K and V."""
        return (getattr(self._write_kv, "__func__", None) is GqaHipBackend._write_kv
                and getattr(self._attn, "__func__", None) is GqaHipBackend._attn)

    def _deferred(self, T, ctx):
        """Whether the attention kernel writes the new rows."""
        return (self.fuse_kv_write and not self.fp8 and getattr(ctx, "aia_slots_from_block_table", False)
                and T == ctx.slot_mapping.shape[0])

    def _write_kv(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor, ctx) -> None:
        cache = ctx.kv_caches[layer_idx]
        if self._deferred(k.shape[0], ctx):
            self._pending = (layer_idx, id(ctx), k, v)
            return
        self._write(k, v, cache, ctx.slot_mapping)

    def _attn(self, layer_idx: int, q, k, v, ctx) -> torch.Tensor:
        cache = ctx.kv_caches[layer_idx]
        if self.share_prefixes or self.sparse:
            return self._attn_blocks(q, cache, ctx)
        plan = step_plan(ctx, self.n_q_heads, self.n_kv_heads, self.head_dim, cache[0].shape[1])
        pending, self._pending = self._pending, None
        if pending is not None and pending[:2] == (layer_idx, id(ctx)):
            return ops.paged_attention_gqa(q, cache[0], cache[1], plan, self.scale,
                                           key_new=pending[2], value_new=pending[3],
                                           kv_layout=self.kv_layout, **self.scores)
        if pending is not None:      # a deferred write for another call: do it now
            lay, _, pk, pv = pending
            self._write(pk, pv, ctx.kv_caches[lay], ctx.slot_mapping)
        if self.fp8:
            return ops.paged_attention_gqa(q, cache[0], cache[1], plan, self.scale,
                                           key_scale=cache[2], value_scale=cache[3], **self.scores)
        return ops.paged_attention_gqa(q, cache[0], cache[1], plan, self.scale,
                                       kv_layout=self.kv_layout, **self.scores)

    def _attn_blocks(self, q, cache, ctx):
        """Attention over shared prefixes or selected blocks of written caches."""
        sizes = (self.n_q_heads, self.n_kv_heads, self.head_dim, cache[0].shape[1])
        scales = dict(key_scale=cache[2], value_scale=cache[3]) if self.fp8 else {}
        if self.share_prefixes:
            return ops.paged_attention_shared(q, cache[0], cache[1], step_shared_plan(ctx, *sizes),
                                              self.scale, **scales)
        plan = step_sparse_plan(ctx, *sizes, *self.sparse)
        bounds, bounds_scale = cache[-2:]
        ops.summarize_blocks(cache[0], plan, bounds, bounds_scale, key_scale=scales.get("key_scale"))
        selected = ops.select_blocks(q, plan, bounds, bounds_scale)
        return ops.paged_attention_sparse(q, cache[0], cache[1], plan, selected, self.scale, **scales)
