"""Torch-facing wrappers of the gfx950 kernels.

PyTorch owns every buffer (caches, metadata, workspace); these functions
check shapes/dtypes/devices on the host, then hand raw pointers and the
current HIP stream to the C ABI.  Nothing here computes on the CPU.
"""
import ctypes
import math

import torch

from auto_infer_amd import _native

_BF16 = torch.bfloat16
FP8_KV, FP8_KV_SCALE = torch.float8_e4m3fn, torch.float8_e8m0fnu   # 8-bit KV caches


# Pointers and streams go to the C-ABI as plain ints: every pointer
# parameter is declared c_void_p, which converts them (and None -> NULL).
# The checks raise behind their conditions (a message formatted on every call
# cost 0.1 - 0.4 us), and the stream's handle comes without a Stream object
# (0.1 us against 1.8; the public call where that one is absent).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device):
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _call_on(dev, name, *args):
    """An entry point's launch with GPU ``dev`` (an index) current: its stream
    handle may be the default stream's, which is that of the current device."""
    if _current_device() == dev:
        _native.call(name, *args)
    else:
        with torch.cuda.device(dev):
            _native.call(name, *args)


def _stream_of(dev):
    return (torch.cuda.current_stream(dev).cuda_stream if _raw_stream is None
            else _raw_stream(dev))


def _check_on(t, name, dtype, dev):
    """``t`` is a ``dtype`` tensor on GPU ``dev`` (an index: -1, a CPU tensor's,
    fails the first check of a call)."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.get_device() != dev or dev < 0:
        _check_device_tensor(t, name, dtype)
        raise ValueError(f"{name} must be on cuda:{dev}")


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _require(cond, msg):
    if not cond:
        raise ValueError(msg)


def _check_device_tensor(t, name, dtype=None):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU (no CPU fallback)")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")


def _row_stride(t, name):
    """Token stride of a (T, heads, dim) tensor whose (heads, dim) part is
    one contiguous row."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be (tokens, heads, dim)")
    s0, s1, s2 = t.stride()
    if s2 != 1 or s1 != t.shape[2]:
        raise ValueError(f"{name} rows (heads, dim) must be contiguous")
    return s0


def _token_stride(t, name):
    """``_row_stride``, but the row's length for a single token, whose stride
    means nothing."""
    ts = _row_stride(t, name)
    return ts if t.shape[0] > 1 else t.shape[1] * t.shape[2]


# ---------------------------------------------------------------- KV write

def qk_norm_rope(qkv, num_q_heads, num_kv_heads, cos, sin, q_norm_weight=None,
                 k_norm_weight=None, eps=1e-6, head_dim=128):
    """Fused pre-attention over a packed qkv projection, in place: optional
    per-head RMSNorm of the Q and K heads (Qwen3 QK-Norm) and NeoX RoPE with
    ``cos``/``sin`` of shape (T, 1, D) or (T, D), D = ``head_dim`` (128 or
    64).  Returns the (q, k, v) views of ``qkv`` -- (T, Hq, D), (T, Hkv, D),
    (T, Hkv, D) -- ready for ``paged_attention_gqa(q, ..., key_new=k,
    value_new=v)``.

    Replaces the split / rms_norm / rotary steps of the reference's
    ``_GqaProjRopeMixin.attention`` (auto_infer/layers/attention/gqa.py:
    27-49) with one kernel that rounds to bf16 where those ops round."""
    _check_device_tensor(qkv, "qkv", _BF16)
    _require(qkv.dim() == 2 and qkv.stride(1) == 1, "qkv must be (T, width) with unit inner stride")
    T, width = qkv.shape
    D = int(head_dim)
    if D not in (128, 64):
        raise NotImplementedError(f"qk_norm_rope: head_dim {D} (128 or 64)")
    if width != (num_q_heads + 2 * num_kv_heads) * D:
        raise ValueError(f"qkv width {width} != (Hq + 2 Hkv) x {D}")
    cs = []
    for t, name in ((cos, "cos"), (sin, "sin")):
        _check_device_tensor(t, name, _BF16)
        if not (t.shape[0] == T and t.shape[-1] == D and t.numel() == T * D and t.stride(-1) == 1):
            raise ValueError(f"{name} must hold one {D}-wide row per token")
        cs.append(t.stride(0))
    for t, name in ((q_norm_weight, "q_norm_weight"), (k_norm_weight, "k_norm_weight")):
        if t is not None:
            _check_device_tensor(t, name, _BF16)
            if t.numel() != D or not t.is_contiguous():
                raise ValueError(f"{name} must be {D} contiguous values")
    _native.call("aia_qk_norm_rope", _ptr(qkv), qkv.stride(0), T, num_q_heads, num_kv_heads, D,
                 _ptr(cos), cs[0], _ptr(sin), cs[1], _ptr(q_norm_weight), _ptr(k_norm_weight),
                 float(eps), _stream(qkv.device))
    q, k, v = qkv.split((num_q_heads * D, num_kv_heads * D, num_kv_heads * D), dim=-1)
    return q.view(T, num_q_heads, D), k.view(T, num_kv_heads, D), v.view(T, num_kv_heads, D)


class RotaryEmbedding:
    """Frequencies of rotary positions, for ``rope_qk``.

    ``rotary_dim`` (default ``head_dim``): the leading dims of each head that
    turn, a multiple of 16; ``interleaved``: pairs of neighbouring dims instead
    of dims half of the rotated part apart.  Pair i turns by
    ``base ** (-2 i / rotary_dim)`` per position, changed by ``scaling``:

    * ``{"type": "linear", "factor": f}``: all frequencies divided by f;
    * ``{"type": "yarn", "factor": f, "original_max_position": n}`` (optional
      ``beta_fast`` 32, ``beta_slow`` 1, ``attention_factor`` 0.1 ln f + 1 for f
      > 1): pairs that turn more than ``beta_fast`` times within n positions
      stay, those that turn less than ``beta_slow`` times are divided by f, a
      linear ramp over the pairs in between; cos and sin are multiplied by
      ``attention_factor``;

    or given as ``inv_freq`` (rotary_dim / 2 radians per position), with
    ``attention_factor`` for the factor on cos and sin.  The frequencies are
    kept on the device as 64-bit fractions of a turn (``turns``), so angles stay
    exact at far positions.
    """

    def __init__(self, head_dim, rotary_dim=None, base=10000.0, interleaved=False, scaling=None,
                 inv_freq=None, attention_factor=None, device="cuda"):
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        self.interleaved = bool(interleaved)
        n = self.rotary_dim // 2
        if self.head_dim not in (128, 64):
            raise NotImplementedError(f"RotaryEmbedding: head_dim {head_dim} (128 or 64)")
        if not 0 < self.rotary_dim <= self.head_dim or self.rotary_dim % 16:
            raise NotImplementedError(f"RotaryEmbedding: rotary_dim {rotary_dim} (a multiple of 16 "
                                      f"up to head_dim {head_dim})")
        factor = 1.0
        if inv_freq is not None:
            _require(scaling is None, "inv_freq and scaling exclude each other")
            freq = [float(f) for f in inv_freq]
            _require(len(freq) == n and all(math.isfinite(f) for f in freq),
                     f"inv_freq must hold {n} finite values")
        else:
            _require(base > 0, "base must be positive")
            freq = [float(base) ** (-2.0 * i / self.rotary_dim) for i in range(n)]
            if scaling is not None:
                freq, factor = self._scaled(freq, float(base), dict(scaling))
        if attention_factor is not None:
            factor = float(attention_factor)
        _require(math.isfinite(factor), "attention_factor must be finite")
        self.inv_freq, self.attention_factor = freq, factor
        # radians -> 2^-64 turns, modulo one turn, as a signed 64-bit word
        words = [int(math.ldexp(f / (2 * math.pi), 64)) % (1 << 64) for f in freq]
        self.turns = torch.tensor([w - (1 << 64) if w >> 63 else w for w in words],
                                  dtype=torch.int64).to(device)

    def _scaled(self, freq, base, sc):
        kind, f = sc.pop("type", None), float(sc.pop("factor", 0.0))
        _require(kind in ("linear", "yarn"), f"rotary scaling type {kind!r} (linear or yarn)")
        _require(f > 0 and math.isfinite(f), f"{kind} scaling needs a positive factor")
        if kind == "linear":
            _require(not sc, f"unknown entries of linear scaling: {sorted(sc)}")
            return [x / f for x in freq], 1.0
        n = sc.pop("original_max_position", 0)
        fast, slow = float(sc.pop("beta_fast", 32.0)), float(sc.pop("beta_slow", 1.0))
        att = sc.pop("attention_factor", None)
        _require(not sc, f"unknown entries of yarn scaling: {sorted(sc)}")
        _require(n > 0, "yarn scaling needs original_max_position")
        _require(fast >= slow > 0 and base > 1, "yarn scaling needs beta_fast >= beta_slow > 0 and "
                 "base > 1")
        d = self.rotary_dim

        def pair(turns):        # the pair that turns so often within n positions
            return d * math.log(n / (2 * math.pi * turns)) / (2 * math.log(base))
        lo = max(math.floor(pair(fast)), 0)
        hi = min(math.ceil(pair(slow)), d - 1)
        out = []
        for i, x in enumerate(freq):
            r = min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
            out.append(x * (1 - r) + x / f * r)
        if att is None:
            att = 0.1 * math.log(f) + 1.0 if f > 1 else 1.0
        return out, float(att)


def _rope_inputs(qkv, num_q_heads, num_kv_heads, positions, rope, q_norm_weight, k_norm_weight):
    """The checks of a packed qkv projection whose heads turn by positions; returns
    (device index, tokens, head_dim, width of Q, width of K, token stride)."""
    _require(isinstance(rope, RotaryEmbedding), "rope must be a RotaryEmbedding")
    _check_device_tensor(qkv, "qkv", _BF16)
    dev, D = qkv.get_device(), rope.head_dim
    if qkv.dim() != 2 or qkv.stride(1) != 1:
        raise ValueError("qkv must be (T, width) with unit inner stride")
    T, width = qkv.shape
    nq, nk = num_q_heads * D, num_kv_heads * D
    if num_q_heads <= 0 or num_kv_heads <= 0 or width != nq + 2 * nk:
        raise ValueError(f"qkv width {width} != (Hq + 2 Hkv) x {D}")
    _check_on(positions, "positions", torch.int64, dev)
    if positions.shape != (T,) or not positions.is_contiguous():
        raise ValueError("positions must hold one contiguous entry per token")
    if rope.turns.get_device() != dev:
        raise ValueError(f"rope must be on cuda:{dev}")
    if q_norm_weight is not None or k_norm_weight is not None:
        _require(q_norm_weight is not None and k_norm_weight is not None,
                 "q and k norm weights go together")
        for t, name in ((q_norm_weight, "q_norm_weight"), (k_norm_weight, "k_norm_weight")):
            _check_on(t, name, _BF16, dev)
            if t.numel() != D or not t.is_contiguous():
                raise ValueError(f"{name} must be {D} contiguous values")
    ts = qkv.stride(0) if T > 1 else width
    if ts < width:
        raise ValueError("qkv rows overlap")
    return dev, T, D, nq, nk, ts


def rope_qk(qkv, num_q_heads, num_kv_heads, positions, rope, q_norm_weight=None,
            k_norm_weight=None, eps=1e-6, out=None):
    """Rotary positions of the Q and K heads of a packed qkv projection (T, (Hq
    + 2 Hkv) D), with an optional per-head RMSNorm in front, one launch.

    ``positions`` (T,) int64, any values; ``rope`` a ``RotaryEmbedding`` of the
    same head_dim.  In place by default; ``out`` = (q_out, k_out), tensors (T,
    Hq, D) and (T, Hkv, D) that do not overlap ``qkv`` or each other (refused), leaves
    ``qkv`` as it is.
    Returns the rotated (q, k) and the V view, (T, heads, D) each.  Unlike
    ``qk_norm_rope`` (cos/sin rows, bf16 roundings of the separate ops) it
    computes the angles itself and rounds once."""
    dev, T, D, nq, nk, ts = _rope_inputs(qkv, num_q_heads, num_kv_heads, positions, rope,
                                         q_norm_weight, k_norm_weight)
    # (T, heads, D) views of the packed rows
    v = qkv.as_strided((T, num_kv_heads, D), (ts, D, 1), qkv.storage_offset() + nq + nk)
    if out is None:
        at = qkv.data_ptr()
        q = qkv.as_strided((T, num_q_heads, D), (ts, D, 1))
        k = qkv.as_strided((T, num_kv_heads, D), (ts, D, 1), qkv.storage_offset() + nq)
        q_at, q_ts, k_at, k_ts = at, ts, at + 2 * nq, ts
    else:
        q, k = out
        for t, name, heads in ((q, "q_out", num_q_heads), (k, "k_out", num_kv_heads)):
            _check_on(t, name, _BF16, dev)
            if t.shape != (T, heads, D):
                raise ValueError(f"{name} must have shape {(T, heads, D)}, got {tuple(t.shape)}")
        q_at, k_at = q.data_ptr(), k.data_ptr()
        q_ts, k_ts = _token_stride(q, "q_out"), _token_stride(k, "k_out")
    _call_on(dev, "aia_rope_qk", qkv.data_ptr(), ts, T, num_q_heads, num_kv_heads, D,
             positions.data_ptr(), rope.turns.data_ptr(), rope.rotary_dim, rope.attention_factor,
             rope.interleaved, _ptr(q_norm_weight), _ptr(k_norm_weight), eps, q_at, q_ts, k_at,
             k_ts, _stream_of(dev))
    return q, k, v


def rope_append(qkv, num_q_heads, num_kv_heads, positions, rope, key_cache, value_cache,
                slot_mapping, q_norm_weight=None, k_norm_weight=None, eps=1e-6, q_out=None,
                key_scale=None, value_scale=None, kv_layout="nd"):
    """``rope_qk`` and the cache write in one launch: the Q and K heads of a packed
    qkv projection (T, (Hq + 2 Hkv) D) are normed (with weights) and turned by their
    positions, K and V go to ``slot_mapping`` of the caches, turned Q is returned.

    ``positions`` / ``rope`` / norm weights as ``rope_qk`` takes them, with the same
    bits; caches (NB, bs, Hkv, D) bf16 (``kv_layout`` as in ``paged_attention_gqa``)
    or ``torch.float8_e4m3fn`` with ``key_scale`` / ``value_scale`` (as
    ``write_kv_fp8`` writes them).  Q is turned in place, or into ``q_out`` (T, Hq,
    D), which does not overlap ``qkv`` (refused); the K and V parts of ``qkv`` stay as
    they are.  ``slot_mapping`` (T,) int32: slots outside the cache are skipped; the
    slots of a call differ from each other (8-bit caches keep the last token of a
    slot, bf16 ones any)."""
    dev, T, D, nq, nk, ts = _rope_inputs(qkv, num_q_heads, num_kv_heads, positions, rope,
                                         q_norm_weight, k_norm_weight)
    if kv_layout not in KV_LAYOUTS:
        raise ValueError(f"kv_layout must be one of {sorted(KV_LAYOUTS)}")
    ks_at = vs_at = None
    if key_scale is not None or value_scale is not None:
        shape = _check_fp8_cache(key_cache, key_scale, "key_cache", "key_scale", dev)
        if _check_fp8_cache(value_cache, value_scale, "value_cache", "value_scale", dev) != shape:
            raise ValueError("value_cache must match key_cache")
        ks_at, vs_at = key_scale.data_ptr(), value_scale.data_ptr()
    else:
        _check_on(key_cache, "key_cache", _BF16, dev)
        _check_on(value_cache, "value_cache", _BF16, dev)
        shape = key_cache.shape
        if len(shape) != 4 or not (key_cache.is_contiguous() and value_cache.is_contiguous()):
            raise ValueError("caches must be contiguous (num_blocks, block_size, Hkv, D)")
        if value_cache.shape != shape:
            raise ValueError("value_cache must match key_cache")
    nb, bs, hkv, d = shape
    if hkv != num_kv_heads or d != D:
        raise ValueError(f"caches of {hkv} heads of {d}, not {num_kv_heads} of {D}")
    _check_on(slot_mapping, "slot_mapping", torch.int32, dev)
    if slot_mapping.shape != (T,) or not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be a contiguous 1-D tensor with one slot per token")
    if q_out is None:
        q = qkv.as_strided((T, num_q_heads, D), (ts, D, 1))
        q_ts = ts
    else:
        q = q_out
        _check_on(q, "q_out", _BF16, dev)
        if q.shape != (T, num_q_heads, D):
            raise ValueError(f"q_out must have shape {(T, num_q_heads, D)}, got {tuple(q.shape)}")
        q_ts = _token_stride(q, "q_out")
    _call_on(dev, "aia_rope_append", qkv.data_ptr(), ts, T, num_q_heads, num_kv_heads, D,
             positions.data_ptr(), rope.turns.data_ptr(), rope.rotary_dim, rope.attention_factor,
             rope.interleaved, _ptr(q_norm_weight), _ptr(k_norm_weight), eps, q.data_ptr(), q_ts,
             key_cache.data_ptr(), value_cache.data_ptr(), ks_at, vs_at, slot_mapping.data_ptr(), bs,
             nb * bs, KV_LAYOUTS[kv_layout], _stream_of(dev))
    return q


def _rope_rows(t, name, T, width):
    _check_device_tensor(t, name, _BF16)
    if not (t.shape[0] == T and t.shape[-1] == width and t.numel() == T * width and
            t.stride(-1) == 1):
        raise ValueError(f"{name} must hold one {width}-wide row per token")
    return t.stride(0)


def mla_kv_latent(ckv_full, norm_weight, eps, cos, sin, out=None):
    """Absorbed-MLA latent KV rows, one launch: ``[rms_norm(ckv), rope(
    interleave(k_pe))]`` of the kv_a_proj_with_mqa output ``ckv_full`` (T,
    576) with ``cos``/``sin`` (T, 1, 64).  Returns ``out`` (T, 1, 576), the
    reference's ``k_latent`` (auto_infer/layers/attention/mla.py:97-111)."""
    _check_device_tensor(ckv_full, "ckv_full", _BF16)
    _require(ckv_full.dim() == 2 and ckv_full.shape[1] == MLA_LATENT + MLA_ROPE and
             ckv_full.stride(1) == 1, "ckv_full must be (T, 576) with unit inner stride")
    T = ckv_full.shape[0]
    cts, sts = _rope_rows(cos, "cos", T, MLA_ROPE), _rope_rows(sin, "sin", T, MLA_ROPE)
    _check_device_tensor(norm_weight, "norm_weight", _BF16)
    _require(norm_weight.numel() == MLA_LATENT and norm_weight.is_contiguous(),
             "norm_weight must be 512 contiguous values")
    if out is None:
        out = torch.empty(T, 1, MLA_LATENT + MLA_ROPE, dtype=_BF16, device=ckv_full.device)
    _check_out(out, "out", (T, 1, MLA_LATENT + MLA_ROPE), ckv_full.device)
    _require(out.is_contiguous(), "out must be a contiguous (T, 1, 576) tensor")
    _native.call("aia_mla_kv_latent", _ptr(ckv_full), ckv_full.stride(0), T, _ptr(norm_weight),
                 float(eps), _ptr(cos), cts, _ptr(sin), sts, _ptr(out), MLA_LATENT + MLA_ROPE,
                 _stream(ckv_full.device))
    return out


def mla_q_latent(q, w_uk_t, cos, sin, out=None):
    """Absorbed-MLA latent query, one launch: ``[q_nope . W_UK, rope(
    interleave(q_pe))]`` for ``q`` (T, H, 192) = [nope 128, pe 64], with
    ``w_uk_t`` = W_UK transposed, (H, 512, 128) contiguous, and ``cos``/``sin``
    (T, 1, 64).  Returns ``out`` (T, H, 576), the reference's ``q_latent``
    (auto_infer/layers/attention/mla.py:93-107)."""
    _check_device_tensor(q, "q", _BF16)
    _require(q.dim() == 3 and q.shape[2] == 128 + MLA_ROPE and q.stride(2) == 1,
             "q must be (T, H, 192) with unit inner stride")
    T, H, _ = q.shape
    _check_device_tensor(w_uk_t, "w_uk_t", _BF16)
    _require(tuple(w_uk_t.shape) == (H, MLA_LATENT, 128) and w_uk_t.is_contiguous(),
             "w_uk_t must be a contiguous (H, 512, 128) tensor")
    cts, sts = _rope_rows(cos, "cos", T, MLA_ROPE), _rope_rows(sin, "sin", T, MLA_ROPE)
    if out is None:
        out = torch.empty(T, H, MLA_LATENT + MLA_ROPE, dtype=_BF16, device=q.device)
    _check_out(out, "out", (T, H, MLA_LATENT + MLA_ROPE), q.device)
    _native.call("aia_mla_q_latent", _ptr(q), q.stride(0), q.stride(1), T, H, _ptr(w_uk_t),
                 _ptr(cos), cts, _ptr(sin), sts, _ptr(out), out.stride(0), out.stride(1),
                 _stream(q.device))
    return out


# Query rows (tokens x heads) up to which mla_v_up beats the library GEMM, for
# programs that route by it: every count it takes, since long steps have a
# kernel of their own (16 heads: 192 tokens 6.2 -> 4.9 us, 2450 tokens 55 ->
# 12.9 against the library's 23.5).
MLA_V_UP_MAX_ROWS = 2 ** 31 - 1


def mla_v_up(o_latent, w_uv, out=None):
    """Absorbed-MLA value up-projection, one launch: ``einsum("tnl,nvl->tnv",
    o_latent[..., :512], W_UV)`` (auto_infer/layers/attention/mla.py:120-121)
    for ``o_latent`` (T, H, >= 512) and ``w_uv`` (H, 128, 512) contiguous.
    Returns ``out`` (T, H, 128); its (T, H * 128) view feeds o_proj."""
    _check_device_tensor(o_latent, "o_latent", _BF16)
    _require(o_latent.dim() == 3 and o_latent.shape[2] >= MLA_LATENT and o_latent.stride(2) == 1,
             "o_latent must be (T, H, >= 512) with unit inner stride")
    T, H, _ = o_latent.shape
    _check_device_tensor(w_uv, "w_uv", _BF16)
    _require(tuple(w_uv.shape) == (H, 128, MLA_LATENT) and w_uv.is_contiguous(),
             "w_uv must be a contiguous (H, 128, 512) tensor")
    if out is None:
        out = torch.empty(T, H, 128, dtype=_BF16, device=o_latent.device)
    _check_out(out, "out", (T, H, 128), o_latent.device)
    _native.call("aia_mla_v_up", _ptr(o_latent), o_latent.stride(0), o_latent.stride(1), T, H,
                 _ptr(w_uv), _ptr(out), out.stride(0), out.stride(1), _stream(o_latent.device))
    return out


def mtp_compact(preds, drafts, active_mask, hidden, positions, slots, scratch_positions,
                scratch_slots, *, accepted=None, out_hidden=None, out_tokens=None,
                out_positions=None, out_slots=None):
    """Accepted draft counts and the compaction of confirmed target rows for
    the MTP drafter, in one launch (reference: GraphMtpRunner._target_body,
    auto_infer/worker/graph_mtp_runner.py:224-248).  Shapes: preds (g, w)
    int64, drafts (g, w - 1) int64, active_mask (g,), hidden (g * w, H) bf16,
    positions / scratch_positions (g * w,) int64, slots / scratch_slots
    (g * w,) int32.  Outputs (allocated unless given, so a graph can pass
    fixed buffers): accepted (g,) int64, hidden (g * w, H), tokens and
    positions (g * w,) int64, slots (g * w,) int32.  Returns them as a tuple
    (accepted, hidden, tokens, positions, slots)."""
    _check_device_tensor(preds, "preds", torch.int64)
    _require(preds.dim() == 2 and preds.is_contiguous(), "preds must be a contiguous (g, w) tensor")
    g, w = preds.shape
    _require(1 <= g <= 64 and w >= 2, "gear must be in [1, 64] and query width >= 2")
    _check_device_tensor(drafts, "drafts", torch.int64)
    _require(tuple(drafts.shape) == (g, w - 1) and drafts.is_contiguous(),
             "drafts must be a contiguous (g, w - 1) tensor")
    _check_device_tensor(active_mask, "active_mask")
    active = active_mask.to(torch.int32).contiguous()
    _require(active.numel() == g, "active_mask must have g entries")
    _check_device_tensor(hidden, "hidden", _BF16)
    _require(hidden.dim() == 2 and hidden.shape[0] == g * w and hidden.stride(1) == 1,
             "hidden must be (g * w, H) with unit inner stride")
    H = hidden.shape[1]
    for t, name, dt in ((positions, "positions", torch.int64), (slots, "slots", torch.int32),
                        (scratch_positions, "scratch_positions", torch.int64),
                        (scratch_slots, "scratch_slots", torch.int32)):
        _check_device_tensor(t, name, dt)
        _require(t.numel() == g * w and t.is_contiguous(), f"{name} must hold g * w entries")
    dev = preds.device
    accepted = accepted if accepted is not None else torch.empty(g, dtype=torch.int64, device=dev)
    out_hidden = out_hidden if out_hidden is not None else torch.empty(g * w, H, dtype=_BF16, device=dev)
    out_tokens = out_tokens if out_tokens is not None else torch.empty(g * w, dtype=torch.int64, device=dev)
    out_positions = (out_positions if out_positions is not None
                     else torch.empty(g * w, dtype=torch.int64, device=dev))
    out_slots = out_slots if out_slots is not None else torch.empty(g * w, dtype=torch.int32, device=dev)
    _require(out_hidden.shape == (g * w, H) and out_hidden.stride(1) == 1 and out_hidden.dtype == _BF16,
             "out_hidden must be (g * w, H) bf16 with unit inner stride")
    _native.call("aia_mtp_compact", _ptr(preds), _ptr(drafts), _ptr(active), _ptr(hidden),
                 hidden.stride(0), _ptr(positions), _ptr(slots), _ptr(scratch_positions),
                 _ptr(scratch_slots), g, w, H, _ptr(accepted), _ptr(out_hidden),
                 out_hidden.stride(0), _ptr(out_tokens), _ptr(out_positions), _ptr(out_slots),
                 _stream(dev))
    return accepted, out_hidden, out_tokens, out_positions, out_slots


def write_kv(key, value, key_cache, value_cache, slot_mapping):
    """Scatter this step's K/V into the paged cache by slot index.

    Same call shape and semantics as the reference's ``write_kv``
    (auto_infer/layers/attention/base.py:41-45):
    ``key_cache.view(-1, Hkv, D)[slot_mapping[t]] = key[t]`` and the same for
    ``value``.  ``value``/``value_cache`` may be None to write a single
    cache (absorbed MLA).  Slots outside the cache are skipped.
    """
    _check_device_tensor(key, "key", _BF16)
    _check_device_tensor(key_cache, "key_cache", _BF16)
    _check_device_tensor(slot_mapping, "slot_mapping", torch.int32)
    _require(key_cache.is_contiguous(), "key_cache must be contiguous")
    _require(slot_mapping.dim() == 1 and slot_mapping.is_contiguous(),
             "slot_mapping must be a contiguous 1-D tensor")
    T = key.shape[0]
    _require(slot_mapping.shape[0] == T, "slot_mapping length must equal the token count")
    krow = key.shape[1] * key.shape[2]
    _require(key_cache.numel() % krow == 0 and key_cache.shape[-1] * key_cache.shape[-2] == krow,
             "key rows do not match the key cache's (heads, dim)")
    num_slots = key_cache.numel() // krow
    kts = _row_stride(key, "key")
    if value is not None:
        _check_device_tensor(value, "value", _BF16)
        _check_device_tensor(value_cache, "value_cache", _BF16)
        _require(value_cache.is_contiguous(), "value_cache must be contiguous")
        _require(value.shape[0] == T, "value must have as many tokens as key")
        vrow = value.shape[1] * value.shape[2]
        _require(value_cache.numel() // vrow == num_slots and
                 value_cache.shape[-1] * value_cache.shape[-2] == vrow,
                 "value rows do not match the value cache")
        vts = _row_stride(value, "value")
    else:
        _require(value_cache is None, "value_cache given without value")
        vrow, vts = 0, 0
    _native.call("aia_kv_write", _ptr(key), kts, _ptr(value), vts, _ptr(key_cache),
                 _ptr(value_cache), _ptr(slot_mapping), T, krow, vrow, num_slots,
                 _stream(key.device))


def write_kv_nz(key, value, key_cache, value_cache, slot_mapping):
    """The KV slot write into caches in the NZ layout of the reference's
    graph-mode backend (``npu_scatter_pa_kv_cache``, auto_infer/layers/
    attention/gqa.py:202-211): the caches are (NB, bs, Hkv, D) tensors whose
    memory is viewed (NB, Hkv*D/16, bs, 16).  ``value``/``value_cache`` may
    be None.  Slots outside the cache are skipped."""
    _check_device_tensor(key, "key", _BF16)
    _check_device_tensor(key_cache, "key_cache", _BF16)
    _check_device_tensor(slot_mapping, "slot_mapping", torch.int32)
    _require(key_cache.dim() == 4 and key_cache.is_contiguous(),
             "key_cache must be a contiguous (num_blocks, block_size, Hkv, D) tensor")
    _require(slot_mapping.dim() == 1 and slot_mapping.is_contiguous() and
             slot_mapping.shape[0] == key.shape[0], "slot_mapping must hold one slot per token")
    nb, bs, hkv, d = key_cache.shape
    row = hkv * d
    _require(key.dim() == 3 and key.shape[1] * key.shape[2] == row, "key rows do not match the cache")
    kts = _row_stride(key, "key")
    vts = 0
    if value is not None:
        _check_device_tensor(value, "value", _BF16)
        _check_device_tensor(value_cache, "value_cache", _BF16)
        _require(tuple(value_cache.shape) == tuple(key_cache.shape) and value_cache.is_contiguous(),
                 "value_cache must match key_cache")
        _require(tuple(value.shape) == tuple(key.shape), "value must match key")
        vts = _row_stride(value, "value")
    else:
        _require(value_cache is None, "value_cache given without value")
    _native.call("aia_kv_write_nz", _ptr(key), kts, _ptr(value), vts, _ptr(key_cache),
                 _ptr(value_cache), _ptr(slot_mapping), key.shape[0], row, bs, nb * bs,
                 _stream(key.device))


def _check_fp8_cache(cache, scale, cache_name, scale_name, dev):
    """An 8-bit cache (NB, bs, Hkv, D) and its scales (NB, Hkv); returns the
    cache's shape."""
    _check_on(cache, cache_name, FP8_KV, dev)
    _check_on(scale, scale_name, FP8_KV_SCALE, dev)
    shape = cache.shape
    if len(shape) != 4 or not cache.is_contiguous():
        raise ValueError(f"{cache_name} must be a contiguous (num_blocks, block_size, Hkv, D) tensor")
    if scale.shape != (shape[0], shape[2]) or not scale.is_contiguous():
        raise ValueError(f"{scale_name} must be a contiguous (num_blocks, Hkv) tensor")
    return shape


def write_kv_fp8(key, value, key_cache, value_cache, key_scale, value_scale, slot_mapping):
    """Scatter this step's bf16 K/V rows into 8-bit paged caches by slot index.

    ``key`` / ``value`` (T, Hkv, D), D 128 or 64; caches (NB, bs, Hkv, D)
    ``torch.float8_e4m3fn``; scales (NB, Hkv) ``torch.float8_e8m0fnu``, one power of two
    per block and head: a cached value stands for value * scale.  A block whose
    first slot is written starts anew (its other slots' contents are lost
    until they are written, which a paged cache does in order); in any other
    block the scale grows where the new rows need it and the block's other
    rows are rescaled; it stays grown when those rows are overwritten (rejected
    drafts), which costs the block's small values precision until it starts anew.
    Values that are not finite become NaN, magnitudes from 1.9375 * 2^127 on are
    read as infinities.  ``value``, its
    cache and its scale may be None.  Slots outside the cache are skipped; of
    tokens with the same slot the last one stays."""
    _check_device_tensor(key, "key", _BF16)
    dev = key.get_device()
    shape = _check_fp8_cache(key_cache, key_scale, "key_cache", "key_scale", dev)
    nb, bs, hkv, d = shape
    rows = key.shape
    if len(rows) != 3 or rows[1:] != shape[2:]:
        raise ValueError("key rows do not match the key cache's (heads, dim)")
    T = rows[0]
    _check_on(slot_mapping, "slot_mapping", torch.int32, dev)
    if slot_mapping.shape != (T,) or not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be a contiguous 1-D tensor with one slot per token")
    kts = _token_stride(key, "key")
    if value is not None:
        _check_on(value, "value", _BF16, dev)
        if _check_fp8_cache(value_cache, value_scale, "value_cache", "value_scale", dev) != shape:
            raise ValueError("value_cache must match key_cache")
        if value.shape != rows:
            raise ValueError("value must match key")
        vts = _token_stride(value, "value")
        v_at, vc_at, vs_at = value.data_ptr(), value_cache.data_ptr(), value_scale.data_ptr()
    else:
        _require(value_cache is None and value_scale is None,
                 "value_cache or value_scale given without value")
        vts, v_at, vc_at, vs_at = 0, None, None, None
    _call_on(dev, "aia_kv_write_fp8", key.data_ptr(), kts, v_at, vts, key_cache.data_ptr(), vc_at,
             key_scale.data_ptr(), vs_at, slot_mapping.data_ptr(), T, hkv, d, bs, nb * bs,
             _stream_of(dev))


KV_LAYOUTS = {"nd": 0, "nz": 1}   # nz: AIA_ATTN_KV_NZ


# ---------------------------------------------------------------- attention

def workspace_bytes(batch, num_tokens, num_q_heads, num_kv_heads, head_dim_v, num_waves=0):
    out = ctypes.c_int64(0)
    _native.call("aia_attn_workspace_bytes", batch, num_tokens, num_q_heads, num_kv_heads,
                 head_dim_v, num_waves, ctypes.byref(out))
    return out.value


_LAYOUT_KEYS = ("hdr", "seg", "wave", "part_ml", "part_o", "req", "mrg", "pf", "pfm", "pfw",
                "pf_ml", "pf_o", "total", "seg_cap", "mrg_cap", "pf_cap", "pf_unit_cap",
                "pf_mrg_cap", "waves", "pf_rows", "pf_keys")


def workspace_layout(batch, num_tokens, num_q_heads, num_kv_heads, head_dim_v, num_waves=0):
    """Byte offsets of a plan's parts in its workspace and the plan's
    capacities (``aia_attn_workspace_layout``), as a dict: for tools and
    tests that read a plan back."""
    vals = (ctypes.c_int64 * len(_LAYOUT_KEYS))()
    _native.call("aia_attn_workspace_layout", batch, num_tokens, num_q_heads, num_kv_heads,
                 head_dim_v, num_waves, vals, len(_LAYOUT_KEYS))
    return dict(zip(_LAYOUT_KEYS, vals))


class AttentionPlan:
    """Device metadata + split-K work plan of one step.

    Built once per step (all layers share it): ``cu_seqlens_q`` is the
    reference's cumulative query-length list with a leading 0 (B + 1
    entries), ``seqlens_kv`` the per-request KV lengths
    (forward_context.py:14-15), both int32 on the device.  The planner runs
    on the GPU, so device-produced metadata (the packing kernel) needs no
    host round trip.

    ``prefix_lens`` (B,) int32 on the device: the first keys of each request
    that all its rows see, in both directions (0 = none; more than the request
    has = all its keys).  GQA only.
    """

    def __init__(self, block_table, cu_seqlens_q, seqlens_kv, num_tokens, num_q_heads,
                 num_kv_heads, head_dim_v, block_size, num_waves=0, workspace=None, owned=None,
                 prefix_lens=None):
        _check_device_tensor(block_table, "block_table", torch.int32)
        _check_device_tensor(cu_seqlens_q, "cu_seqlens_q", torch.int32)
        _check_device_tensor(seqlens_kv, "seqlens_kv", torch.int32)
        _require(block_table.dim() == 2 and block_table.stride(1) == 1,
                 "block_table must be (batch, max_blocks) with unit column stride")
        batch = seqlens_kv.shape[0]
        _require(cu_seqlens_q.shape[0] == batch + 1, "cu_seqlens_q must have batch + 1 entries")
        _require(block_table.shape[0] >= batch, "block_table has fewer rows than requests")
        _require(cu_seqlens_q.is_contiguous() and seqlens_kv.is_contiguous(),
                 "metadata tensors must be contiguous")
        if prefix_lens is not None:
            _check_device_tensor(prefix_lens, "prefix_lens", torch.int32)
            _require(prefix_lens.shape == (batch,) and prefix_lens.is_contiguous() and
                     prefix_lens.device == block_table.device,
                     "prefix_lens must hold one contiguous entry per request")
        self.prefix_lens = prefix_lens
        self.block_table = block_table
        self.cu_seqlens_q = cu_seqlens_q
        self.seqlens_kv = seqlens_kv
        self.batch = batch
        self.num_tokens = int(num_tokens)
        self.num_q_heads = num_q_heads
        self.num_kv_heads = num_kv_heads
        self.head_dim_v = head_dim_v
        self.num_waves = num_waves
        self.block_size = int(block_size)
        nbytes = workspace_bytes(batch, self.num_tokens, num_q_heads, num_kv_heads, head_dim_v,
                                 num_waves)
        if workspace is None:
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=block_table.device)
        _check_device_tensor(workspace, "workspace", torch.uint8)
        _require(workspace.numel() >= nbytes, "attention workspace too small")
        self.workspace = workspace
        # streams the plan's own device tensors are known to be used on: the
        # caching allocator may hand their memory to the allocating stream's
        # next allocation once they are dropped, so every other stream that
        # reads or writes them is recorded (Tensor.record_stream)
        self._streams = {torch.cuda.current_stream(block_table.device)}
        self._owned = [workspace] if owned is None else [workspace, *owned]
        self.replan()

    def replan(self):
        """Re-run the device planner on the (possibly updated in place)
        metadata tensors; graph-capturable.  The plan is then valid on the
        current stream (attention calls on another stream wait for it)."""
        device = self.block_table.device
        self.stream = torch.cuda.current_stream(device)
        self._on = (device, self.stream.cuda_stream)
        self._use_on(self.stream)
        args = (_ptr(self.block_table), self.block_table.stride(0), self.block_size,
                self.batch, self.num_tokens, self.num_q_heads, self.num_kv_heads,
                self.head_dim_v, self.num_waves, _ptr(self.workspace),
                self.workspace.numel(), self._on[1])
        if self.prefix_lens is None:
            _call_on(device.index, "aia_attn_plan", _ptr(self.cu_seqlens_q), _ptr(self.seqlens_kv), *args)
        else:
            _call_on(device.index, "aia_attn_plan_prefix", _ptr(self.cu_seqlens_q), _ptr(self.seqlens_kv),
                         _ptr(self.prefix_lens), *args)

    def _use_on(self, stream):
        if stream not in self._streams:
            self._streams.add(stream)
            for t in self._owned:
                t.record_stream(stream)

    def status(self):
        """Synchronising check of the last plan: raises ValueError if the
        planner found more work than the workspace was sized for (query
        lengths that do not add up to ``num_tokens``); the kernels then ran
        an empty plan and the attention calls filled their outputs with
        NaN."""
        code = int(self.workspace[32:36].view(torch.int32).item())
        if code != 0:
            raise ValueError(f"attention planner overflow (status {code}): cu_seqlens_q does "
                             f"not describe {self.num_tokens} query tokens")

    @classmethod
    def from_lists(cls, block_table, cu_seqlens_q, seqlens_kv, num_q_heads, num_kv_heads,
                   head_dim_v, block_size, **kw):
        """From the reference's host lists (cumulative ends without the
        leading 0, per-request KV lengths)."""
        dev = block_table.device
        check_lists(cu_seqlens_q, seqlens_kv, block_table.shape[1] * block_size)
        cu = torch.tensor([0, *cu_seqlens_q], dtype=torch.int32).to(dev, non_blocking=True)
        kv = torch.tensor(list(seqlens_kv), dtype=torch.int32).to(dev, non_blocking=True)
        total = cu_seqlens_q[-1] if len(cu_seqlens_q) else 0
        return cls(block_table, cu, kv, total, num_q_heads, num_kv_heads, head_dim_v, block_size,
                   owned=[cu, kv], **kw)


def check_lists(cu_seqlens_q, seqlens_kv, max_context):
    """Host check of the reference's metadata lists (cumulative query ends,
    per-request KV lengths; forward_context.py:14-15): same length,
    non-decreasing ends, every KV length within the block table (the
    kernels read block ids up to it)."""
    _require(len(cu_seqlens_q) == len(seqlens_kv),
             "cu_seqlens_q and seqlens_kv must have one entry per request")
    prev = 0
    for end, lk in zip(cu_seqlens_q, seqlens_kv):
        _require(end >= prev, "cu_seqlens_q must be non-decreasing")
        _require(0 <= lk <= max_context,
                 f"KV length {lk} does not fit the block table ({max_context} slots)")
        prev = end


def check_prefixes(prefix_lens, cu_seqlens_q, seqlens_kv):
    """Host check of prefixes that all rows of a request see, against the step's
    lists: a prefix lies within what the request has after this step.  Its rows
    see all of it, so a chunk that ends inside it would leave them (and, layers
    on, their keys and values) without what follows."""
    _require(len(prefix_lens) == len(seqlens_kv), "prefix_lens must have one entry per request")
    prev = 0
    for i, (n, end, lk) in enumerate(zip(prefix_lens, cu_seqlens_q, seqlens_kv)):
        _require(end == prev or n <= lk,
                 f"request {i}: its prefix of {n} tokens ends behind the step's {lk}; a prefix must "
                 f"lie in the request's first chunk")
        prev = end


def _ready(plan, device):
    """Order the attention launch after the planner: on another stream, make
    the current stream wait for the plan's stream (not allowed while
    capturing a graph, where the plan must be made on the capturing stream)
    and record the plan's buffers as in use there.  Returns the current
    stream's handle."""
    raw = _stream(device)
    if plan._on == (device, raw):
        return raw
    cur = torch.cuda.current_stream(device)
    if cur != plan.stream:
        if torch.cuda.is_current_stream_capturing():
            raise ValueError("attention plan was made on another stream than the one being "
                             "captured; call plan.replan() on the capturing stream")
        cur.wait_stream(plan.stream)
        plan._use_on(cur)
    return raw


def _check_out(out, name, shape, device):
    """A caller-supplied output: bf16 on the same GPU, of ``shape``, unit
    inner stride, rows (heads, dim) not overlapping."""
    _check_device_tensor(out, name, _BF16)
    if out.device != device:
        raise ValueError(f"{name} must be on {device}")
    if out.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(out.shape)}")
    st = out.stride()
    if st[-1] != 1:
        raise ValueError(f"{name} must have unit inner stride")
    if len(st) == 3 and not (st[1] >= shape[2] and st[0] >= shape[1] * st[1]):
        raise ValueError(f"{name} rows must not overlap")


def paged_attention_gqa(query, key_cache, value_cache, plan, scale, out=None, flags=0,
                        key_new=None, value_new=None, kv_layout="nd", key_scale=None,
                        value_scale=None, softcap=0.0, alibi_slopes=None):
    """Paged GQA attention (reference base.py:48-61 FIA semantics).

    query (T, Hq, D) bf16 with D = 128 or 64; key/value caches (NB, bs, Hkv,
    D) bf16 contiguous; ``plan`` an ``AttentionPlan`` of this step (head_dim_v
    D).  Returns (T, Hq, D) bf16.  With ``key_new`` / ``value_new`` (this
    step's new rows, (T, Hkv, D)) the kernel also writes them into the caches
    at the slots the block table assigns (the fused form of ``write_kv``).
    ``kv_layout="nz"``: the caches hold the NZ layout of the reference's
    graph mode (see ``write_kv_nz``); results are the same as for the same
    values in the standard layout.

    8-bit caches: ``torch.float8_e4m3fn`` tensors with their ``key_scale`` /
    ``value_scale`` (see ``write_kv_fp8``, which also writes new rows: ``key_new``
    and the NZ layout are for bf16 caches).
    Modified scores, with query position i and key position j: ``softcap`` > 0
    (below 1e38) makes them ``softcap * tanh(scale * q.k / softcap)``; ``alibi_slopes`` (Hq,)
    float32 subtracts ``slope * |i - j|``; a plan with ``prefix_lens`` lets all
    rows of a request see its first keys.  Rows that see no key give zeros.
    """
    if kv_layout not in KV_LAYOUTS:
        raise ValueError(f"kv_layout must be one of {sorted(KV_LAYOUTS)}")
    flags |= KV_LAYOUTS[kv_layout]
    if (key_scale is not None or value_scale is not None or softcap != 0 or
            alibi_slopes is not None or plan.prefix_lens is not None):
        return _paged_attention_gqa_ex(query, key_cache, value_cache, plan, scale, out, flags,
                                       key_new, value_new, key_scale, value_scale, softcap,
                                       alibi_slopes)
    _check_device_tensor(query, "query", _BF16)
    _check_device_tensor(key_cache, "key_cache", _BF16)
    _check_device_tensor(value_cache, "value_cache", _BF16)
    _require(query.dim() == 3 and query.stride(2) == 1, "query must be (T, Hq, D), D contiguous")
    shape = query.shape
    T, hq, d = shape
    _require(key_cache.dim() == 4 and key_cache.is_contiguous() and value_cache.is_contiguous(),
             "caches must be contiguous (num_blocks, block_size, Hkv, D)")
    cshape = key_cache.shape
    nb, bs, hkv, dk = cshape
    _require(value_cache.shape == cshape, "value cache shape differs from key cache")
    _require(dk == d, "query head_dim differs from the cache's")
    _require(hq == plan.num_q_heads and hkv == plan.num_kv_heads and T == plan.num_tokens
             and bs == plan.block_size, "plan was made for another shape")
    device = query.device
    if out is None:
        out = torch.empty(shape, dtype=_BF16, device=device)
    else:
        _check_out(out, "out", shape, device)
    kn_ts = vn_ts = 0
    if key_new is not None or value_new is not None:
        _check_device_tensor(key_new, "key_new", _BF16)
        _check_device_tensor(value_new, "value_new", _BF16)
        rows = (T, hkv, d)
        _require(key_new.shape == rows and value_new.shape == rows,
                 "new K/V rows must be (tokens, Hkv, D)")
        kn_ts, vn_ts = _row_stride(key_new, "key_new"), _row_stride(value_new, "value_new")
    stream = _ready(plan, device)
    q_ts, q_hs, _ = query.stride()
    o_ts, o_hs, _ = out.stride()
    table, ws = plan.block_table, plan.workspace
    _native.call("aia_paged_attention_gqa", query.data_ptr(), q_ts, q_hs,
                 key_cache.data_ptr(), value_cache.data_ptr(), table.data_ptr(),
                 table.stride(0), plan.cu_seqlens_q.data_ptr(), plan.seqlens_kv.data_ptr(),
                 plan.batch, T, hq, hkv, d, bs, nb, float(scale), out.data_ptr(), o_ts,
                 o_hs, _ptr(key_new), _ptr(value_new), kn_ts, vn_ts, plan.num_waves,
                 flags, ws.data_ptr(), ws.numel(), stream)
    return out


def _paged_attention_gqa_ex(query, key_cache, value_cache, plan, scale, out, flags, key_new,
                            value_new, key_scale, value_scale, softcap, alibi_slopes):
    """``paged_attention_gqa`` over 8-bit caches or with modified scores."""
    _check_device_tensor(query, "query", _BF16)
    dev, shape = query.get_device(), query.shape
    if len(shape) != 3 or query.stride(2) != 1:
        raise ValueError("query must be (T, Hq, D), D contiguous")
    T, hq, d = shape
    ks_at = vs_at = kn_at = vn_at = None
    kn_ts = vn_ts = 0
    if key_scale is not None or value_scale is not None:
        cshape = _check_fp8_cache(key_cache, key_scale, "key_cache", "key_scale", dev)
        if _check_fp8_cache(value_cache, value_scale, "value_cache", "value_scale", dev) != cshape:
            raise ValueError("value cache shape differs from key cache")
        _require(key_new is None and value_new is None,
                 "8-bit caches are written by write_kv_fp8, not by key_new / value_new")
        ks_at, vs_at = key_scale.data_ptr(), value_scale.data_ptr()
    else:
        _check_on(key_cache, "key_cache", _BF16, dev)
        _check_on(value_cache, "value_cache", _BF16, dev)
        cshape = key_cache.shape
        if len(cshape) != 4 or not (key_cache.is_contiguous() and value_cache.is_contiguous()):
            raise ValueError("caches must be contiguous (num_blocks, block_size, Hkv, D)")
        if value_cache.shape != cshape:
            raise ValueError("value cache shape differs from key cache")
    nb, bs, hkv, dk = cshape
    if dk != d:
        raise ValueError("query head_dim differs from the cache's")
    if not (hq == plan.num_q_heads and hkv == plan.num_kv_heads and T == plan.num_tokens
            and bs == plan.block_size and d == plan.head_dim_v):
        raise ValueError("plan was made for another shape")
    if key_new is not None or value_new is not None:
        _check_on(key_new, "key_new", _BF16, dev)
        _check_on(value_new, "value_new", _BF16, dev)
        if key_new.shape != (T, hkv, d) or value_new.shape != (T, hkv, d):
            raise ValueError("new K/V rows must be (tokens, Hkv, D)")
        kn_ts, vn_ts = _row_stride(key_new, "key_new"), _row_stride(value_new, "value_new")
        kn_at, vn_at = key_new.data_ptr(), value_new.data_ptr()
    if alibi_slopes is not None:
        _check_on(alibi_slopes, "alibi_slopes", torch.float32, dev)
        if alibi_slopes.shape != (hq,) or not alibi_slopes.is_contiguous():
            raise ValueError(f"alibi_slopes must hold {hq} contiguous values")
    table, ws = plan.block_table, plan.workspace
    if table.get_device() != dev:
        raise ValueError("plan was made on another GPU")
    device = query.device
    if out is None:
        out = torch.empty(shape, dtype=_BF16, device=device)
    else:
        _check_out(out, "out", shape, device)
    stream = _ready(plan, device)
    q_ts, q_hs, _ = query.stride()
    o_ts, o_hs, _ = out.stride()
    _call_on(dev, "aia_paged_attention_gqa_ex", query.data_ptr(), q_ts, q_hs,
             key_cache.data_ptr(), value_cache.data_ptr(), table.data_ptr(), table.stride(0),
             plan.cu_seqlens_q.data_ptr(), plan.seqlens_kv.data_ptr(), plan.batch, T, hq, hkv, d,
             bs, nb, scale, out.data_ptr(), o_ts, o_hs, kn_at, vn_at, kn_ts, vn_ts, ks_at, vs_at,
             _ptr(plan.prefix_lens), _ptr(alibi_slopes), softcap, plan.num_waves, flags,
             ws.data_ptr(), ws.numel(), stream)
    return out


class _StepPlan:
    """What the plans of the operators below share: a step's metadata on one GPU,
    a workspace that its calls use, and the streams that they run on."""

    def _take(self, block_table, cu_seqlens_q, seqlens_kv, num_tokens, num_q_heads, num_kv_heads,
              head_dim, block_size):
        _check_device_tensor(block_table, "block_table", torch.int32)
        dev = block_table.get_device()
        _check_on(cu_seqlens_q, "cu_seqlens_q", torch.int32, dev)
        _check_on(seqlens_kv, "seqlens_kv", torch.int32, dev)
        _require(block_table.dim() == 2 and block_table.shape[1] > 0 and block_table.stride(1) == 1,
                 "block_table must be (batch, max_blocks) with unit column stride")
        _require(seqlens_kv.dim() == 1 and cu_seqlens_q.shape == (seqlens_kv.shape[0] + 1,),
                 "cu_seqlens_q must have batch + 1 entries")
        self.batch = seqlens_kv.shape[0]
        _require(block_table.shape[0] >= self.batch, "block_table has fewer rows than requests")
        _require(cu_seqlens_q.is_contiguous() and seqlens_kv.is_contiguous(),
                 "metadata tensors must be contiguous")
        self.block_table, self.cu_seqlens_q, self.seqlens_kv = block_table, cu_seqlens_q, seqlens_kv
        self.num_tokens, self.block_size = int(num_tokens), int(block_size)
        self.num_q_heads, self.num_kv_heads = int(num_q_heads), int(num_kv_heads)
        self.head_dim, self.device = int(head_dim), block_table.device
        # (a single row's stride means nothing)
        self._table_stride = block_table.stride(0) if block_table.shape[0] > 1 else block_table.shape[1]

    def _make(self, nbytes, workspace, owned):
        if workspace is None:
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        _check_on(workspace, "workspace", torch.uint8, self.device.index)
        _require(workspace.is_contiguous() and workspace.numel() >= nbytes, "workspace too small")
        self.workspace = workspace
        self._owned = [workspace, *(owned or ())]      # as AttentionPlan keeps them
        self._streams = {torch.cuda.current_stream(self.device)}
        self.replan()

    def replan(self):
        """Plan again from the (possibly updated in place) metadata tensors;
        graph-capturable.  The plan is then valid on the current stream."""
        self.stream = torch.cuda.current_stream(self.device)
        self._on = (self.device, self.stream.cuda_stream)
        self._use_on(self.stream)
        self._plan(self._on[1])

    def _use_on(self, stream):
        if stream not in self._streams:
            self._streams.add(stream)
            for t in self._owned:
                t.record_stream(stream)


def _attention_inputs(what, query, key_cache, value_cache, plan, key_scale, value_scale, out):
    """The checks of an attention call over a ``_StepPlan``; returns (device index,
    number of blocks, out)."""
    _check_device_tensor(query, "query", _BF16)
    dev, shape = query.get_device(), query.shape
    if shape != (plan.num_tokens, plan.num_q_heads, plan.head_dim) or query.stride(2) != 1:
        raise ValueError(f"{what}: query must be (T, Hq, D) of the plan's sizes, D contiguous")
    if plan.device.index != dev:
        raise ValueError("plan was made on another GPU")
    if key_scale is not None or value_scale is not None:
        cshape = _check_fp8_cache(key_cache, key_scale, "key_cache", "key_scale", dev)
        if _check_fp8_cache(value_cache, value_scale, "value_cache", "value_scale", dev) != cshape:
            raise ValueError("value cache shape differs from key cache")
    else:
        _check_on(key_cache, "key_cache", _BF16, dev)
        _check_on(value_cache, "value_cache", _BF16, dev)
        cshape = key_cache.shape
        if len(cshape) != 4 or not (key_cache.is_contiguous() and value_cache.is_contiguous()):
            raise ValueError("caches must be contiguous (num_blocks, block_size, Hkv, D)")
        if value_cache.shape != cshape:
            raise ValueError("value cache shape differs from key cache")
    if cshape[1:] != (plan.block_size, plan.num_kv_heads, plan.head_dim):
        raise ValueError("plan was made for another cache shape")
    if out is None:
        out = torch.empty(shape, dtype=_BF16, device=query.device)
    else:
        _check_out(out, "out", shape, query.device)
    return dev, cshape[0], out


class SharedPrefixPlan(_StepPlan):
    """A step of attention whose requests share prefixes, made once for all its
    layers, for ``paged_attention_shared``.

    Metadata as ``AttentionPlan`` takes it.  ``group_ids`` (B,) int32 on the device
    names requests that may share (negative: alone); without it, those with the same
    first block may.  What they share is found on the GPU: each goes with the ones that
    agree with it in most keys times requests, from 128 keys on and in powers of two, and
    such a group shares the leading keys, in front of the new tokens, for which all its
    block table rows agree.  A wrong group costs speed, never the result.  The plan holds scratch
    space, so its calls run on one stream at a time.
    """

    def __init__(self, block_table, cu_seqlens_q, seqlens_kv, num_tokens, num_q_heads, num_kv_heads,
                 head_dim, block_size, group_ids=None, workspace=None, owned=None):
        self._take(block_table, cu_seqlens_q, seqlens_kv, num_tokens, num_q_heads, num_kv_heads,
                   head_dim, block_size)
        if group_ids is not None:
            _check_on(group_ids, "group_ids", torch.int32, self.device.index)
            _require(group_ids.shape == (self.batch,) and group_ids.is_contiguous(),
                     "group_ids must hold one contiguous entry per request")
        self.group_ids = group_ids
        self._sizes = (self._table_stride, block_table.shape[1], self.block_size, self.batch,
                       self.num_tokens, self.num_q_heads, self.num_kv_heads, self.head_dim)
        nbytes = ctypes.c_int64(0)
        _native.call("aia_shared_workspace_bytes", self.batch, self.num_tokens, self.num_q_heads,
                     self.num_kv_heads, self.head_dim, self.block_size, block_table.shape[1],
                     ctypes.byref(nbytes))
        self._make(nbytes.value, workspace, owned)

    def _plan(self, stream):
        _call_on(self.device.index, "aia_shared_plan", self.cu_seqlens_q.data_ptr(),
                 self.seqlens_kv.data_ptr(), _ptr(self.group_ids), self.block_table.data_ptr(),
                 *self._sizes, self.workspace.data_ptr(), self.workspace.numel(), stream)

    def status(self):
        """Synchronising check of the last plan, as ``AttentionPlan.status``."""
        code = int(self.workspace[4:8].view(torch.int32).item())
        if code != 0:
            raise ValueError(f"shared-prefix planner (status {code}): cu_seqlens_q does not describe "
                             f"{self.num_tokens} query tokens")


def paged_attention_shared(query, key_cache, value_cache, plan, scale, out=None, key_scale=None,
                           value_scale=None):
    """Paged GQA attention of a step whose requests share prefixes: the results of
    ``paged_attention_gqa`` (but for roundings), with shared keys read once for all
    the requests of a group.

    query (T, Hq, D) bf16, D 128 or 64; caches (NB, bs, Hkv, D) bf16 or 8-bit with
    their scales (new rows written before, see ``rope_append``); ``plan`` a
    ``SharedPrefixPlan``.  Returns (T, Hq, D) bf16."""
    dev, nb, out = _attention_inputs("paged_attention_shared", query, key_cache, value_cache, plan,
                                     key_scale, value_scale, out)
    stream = _ready(plan, query.device)
    q_ts, q_hs, _ = query.stride()
    o_ts, o_hs, _ = out.stride()
    _call_on(dev, "aia_paged_attention_shared", query.data_ptr(), q_ts, q_hs, key_cache.data_ptr(),
             value_cache.data_ptr(), _ptr(key_scale), _ptr(value_scale), nb,
             plan.cu_seqlens_q.data_ptr(), plan.block_table.data_ptr(), *plan._sizes, scale,
             out.data_ptr(), o_ts, o_hs, plan.workspace.data_ptr(), plan.workspace.numel(), stream)
    return out


class BlockSparsePlan(_StepPlan):
    """A step of block-sparse attention, made once for all its layers.

    Metadata as ``AttentionPlan`` takes it.  Every query token and KV head attends
    at most ``num_selected`` (up to 1024) cache blocks: always the first ``sink``
    and the last ``local`` (at least 1) that it sees, and those of the highest
    score.  ``summarize_blocks``, ``select_blocks`` and ``paged_attention_sparse``
    take the plan; it holds their scratch space, so the plan's calls run on one
    stream at a time.
    """

    def __init__(self, block_table, cu_seqlens_q, seqlens_kv, num_tokens, num_q_heads, num_kv_heads,
                 head_dim, block_size, num_selected, sink=1, local=1, workspace=None, owned=None):
        self._take(block_table, cu_seqlens_q, seqlens_kv, num_tokens, num_q_heads, num_kv_heads,
                   head_dim, block_size)
        self.num_selected, self.sink, self.local = int(num_selected), int(sink), int(local)
        _require(self.sink >= 0 and self.local >= 1 and self.sink + self.local <= self.num_selected,
                 f"sink {sink} and local {local} do not fit {num_selected} selected blocks (local at "
                 f"least 1)")
        self._sizes = (block_table.shape[1], self.block_size, self.batch, self.num_tokens,
                       self.num_q_heads, self.num_kv_heads, self.head_dim)
        nbytes = ctypes.c_int64(0)
        _native.call("aia_sparse_workspace_bytes", self.batch, self.num_tokens, self.num_q_heads,
                     self.num_kv_heads, self.head_dim, self.block_size, block_table.shape[1],
                     self.num_selected, ctypes.byref(nbytes))
        self._make(nbytes.value, workspace, owned)

    def _plan(self, stream):
        width, bs, batch, *rest = self._sizes
        _call_on(self.device.index, "aia_sparse_plan", self.cu_seqlens_q.data_ptr(),
                 self.seqlens_kv.data_ptr(), self.block_table.data_ptr(), self._table_stride, width, bs,
                 batch, *rest, self.num_selected, self.workspace.data_ptr(), self.workspace.numel(),
                 stream)

    def status(self):
        """Synchronising check of the last plan: raises ValueError if cu_seqlens_q does not
        begin at 0, decreases or ends behind ``num_tokens``; ``summarize_blocks`` then
        wrote no bounds, nothing was selected and attention outputs are NaN."""
        code = int(self.workspace[8:12].view(torch.int32).item())
        if code != 0:
            raise ValueError(f"block-sparse planner (status {code}): cu_seqlens_q does not describe "
                             f"{self.num_tokens} query tokens")


def _check_bounds(bounds, bounds_scale, plan, dev):
    _check_on(bounds, "bounds", torch.int8, dev)
    _check_on(bounds_scale, "bounds_scale", FP8_KV_SCALE, dev)
    shape = bounds.shape
    if shape[1:] != (plan.num_kv_heads, 2, plan.head_dim) or not bounds.is_contiguous():
        raise ValueError("bounds must be a contiguous (num_blocks, Hkv, 2, D) tensor")
    if bounds_scale.shape != shape[:2] or not bounds_scale.is_contiguous():
        raise ValueError("bounds_scale must be a contiguous (num_blocks, Hkv) tensor")


def summarize_blocks(key_cache, plan, bounds, bounds_scale, key_scale=None):
    """8-bit bounds of the keys in every cache block that the step's new tokens lie
    in, for ``select_blocks``; call it after the step's keys are written.

    ``key_cache`` (NB, bs, Hkv, D) bf16, or ``torch.float8_e4m3fn`` with its
    ``key_scale``; ``plan`` a ``BlockSparsePlan``.  ``bounds`` (NB, Hkv, 2, D) int8
    receives the largest and the negated smallest key value per dim, as whole
    numbers times the power of two ``bounds_scale`` (NB, Hkv)
    ``torch.float8_e8m0fnu``, rounded up.  A block's bounds follow from what it holds
    of its request now, so rejected drafts leave no trace."""
    dev = plan.device.index
    if key_scale is not None:
        shape = _check_fp8_cache(key_cache, key_scale, "key_cache", "key_scale", dev)
    else:
        _check_on(key_cache, "key_cache", _BF16, dev)
        shape = key_cache.shape
        if len(shape) != 4 or not key_cache.is_contiguous():
            raise ValueError("key_cache must be a contiguous (num_blocks, block_size, Hkv, D) tensor")
    if shape[1:] != (plan.block_size, plan.num_kv_heads, plan.head_dim):
        raise ValueError("plan was made for another cache shape")
    _check_bounds(bounds, bounds_scale, plan, dev)
    if bounds.shape[0] != shape[0]:
        raise ValueError("bounds must have an entry per cache block")
    stream = _ready(plan, plan.device)
    width, bs, *rest = plan._sizes
    _call_on(dev, "aia_summarize_blocks", key_cache.data_ptr(), _ptr(key_scale), shape[0],
             bounds.data_ptr(), bounds_scale.data_ptr(), bs, width, *rest, plan.num_selected,
             plan.workspace.data_ptr(), plan.workspace.numel(), stream)


def select_blocks(query, plan, bounds, bounds_scale, out=None):
    """The cache blocks that each query token and KV head attends: (T, Hkv,
    num_selected) int32 block numbers within the request, ascending, -1 behind them.

    ``query`` (T, Hq, D) bf16 (rotated, as attention takes it); ``plan`` a
    ``BlockSparsePlan``; ``bounds`` / ``bounds_scale`` of ``summarize_blocks``.  A
    block's score bounds the sum of the group's products with its keys from above, up to
    the query's rounding, in whole numbers (8-bit query values and bounds), so the selection
    does not depend on any order of summation; of equal scores the lowest block wins.  The
    query's values are rounded to whole numbers of up to 127 of one power of two for all of
    the group's heads: a value below half of it, 1/127 to 1/254 of the group's largest,
    counts as zero, and so does all of a head whose values are."""
    _check_device_tensor(query, "query", _BF16)
    dev = query.get_device()
    if query.shape != (plan.num_tokens, plan.num_q_heads, plan.head_dim) or query.stride(2) != 1:
        raise ValueError("query must be (T, Hq, D) of the plan's sizes, D contiguous")
    if plan.device.index != dev:
        raise ValueError("plan was made on another GPU")
    _check_bounds(bounds, bounds_scale, plan, dev)
    shape = (plan.num_tokens, plan.num_kv_heads, plan.num_selected)
    if out is None:
        out = torch.empty(shape, dtype=torch.int32, device=query.device)
    else:
        _check_on(out, "out", torch.int32, dev)
        if out.shape != shape or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {shape} tensor")
    stream = _ready(plan, query.device)
    q_ts, q_hs, _ = query.stride()
    width, bs, *rest = plan._sizes
    _call_on(dev, "aia_select_blocks", query.data_ptr(), q_ts, q_hs, bounds.data_ptr(),
             bounds_scale.data_ptr(), bounds.shape[0], plan.block_table.data_ptr(), plan._table_stride,
             width, bs, *rest, plan.num_selected, plan.sink, plan.local, out.data_ptr(),
             shape[1] * shape[2], shape[2], plan.workspace.data_ptr(), plan.workspace.numel(), stream)
    return out


def paged_attention_sparse(query, key_cache, value_cache, plan, selected, scale, out=None,
                           key_scale=None, value_scale=None):
    """Paged attention over selected blocks alone: query head h of token t attends
    the keys of blocks ``selected[t, h // (Hq // Hkv)]`` up to its own position.

    query (T, Hq, D) bf16, D 128 or 64; caches (NB, bs, Hkv, D) bf16 or 8-bit with
    their scales; ``plan`` a ``BlockSparsePlan``; ``selected`` (T, Hkv,
    num_selected) int32 as ``select_blocks`` returns it: ascending block numbers
    within the request (an entry that is negative, past the token's own block or not
    above all before it is left out).  Returns (T, Hq, D) bf16; rows without a key
    give zeros."""
    dev, nb, out = _attention_inputs("paged_attention_sparse", query, key_cache, value_cache, plan,
                                     key_scale, value_scale, out)
    _check_on(selected, "selected", torch.int32, dev)
    if (selected.shape != (plan.num_tokens, plan.num_kv_heads, plan.num_selected)
            or selected.stride(2) != 1):
        raise ValueError("selected must be (T, Hkv, num_selected) with unit inner stride")
    stream = _ready(plan, query.device)
    q_ts, q_hs, _ = query.stride()
    o_ts, o_hs, _ = out.stride()
    s_ts, s_hs, _ = selected.stride()
    width, bs, *rest = plan._sizes
    _call_on(dev, "aia_paged_attention_sparse", query.data_ptr(), q_ts, q_hs, key_cache.data_ptr(),
             value_cache.data_ptr(), _ptr(key_scale), _ptr(value_scale), nb,
             plan.block_table.data_ptr(), plan._table_stride, width, bs, *rest, scale,
             selected.data_ptr(), s_ts, s_hs, plan.num_selected, out.data_ptr(), o_ts, o_hs,
             plan.workspace.data_ptr(), plan.workspace.numel(), stream)
    return out


MLA_LATENT, MLA_ROPE = 512, 64


def paged_attention_mla(q_latent, latent_cache, plan, scale, out=None, flags=0):
    """Absorbed-MLA latent attention (reference mla.py:76-122 semantics).

    q_latent (T, H, 576) bf16 = [W_UK-absorbed nope (512), rope (64)];
    latent_cache (NB, bs, 1, 576) bf16 contiguous; ``plan`` an
    ``AttentionPlan`` made with (num_q_heads=H, num_kv_heads=1,
    head_dim_v=512).  Returns the latent output (T, H, 512) bf16, i.e. the
    first kv_lora_rank values of attention with V = K.
    """
    _check_device_tensor(q_latent, "q_latent", _BF16)
    _check_device_tensor(latent_cache, "latent_cache", _BF16)
    _require(q_latent.dim() == 3 and q_latent.stride(2) == 1,
             "q_latent must be (T, H, 576), last dim contiguous")
    T, h, dk = q_latent.shape
    _require(dk == MLA_LATENT + MLA_ROPE, "q_latent last dim must be 576")
    _require(latent_cache.dim() == 4 and latent_cache.is_contiguous() and
             latent_cache.shape[2] == 1 and latent_cache.shape[3] == dk,
             "latent_cache must be contiguous (num_blocks, block_size, 1, 576)")
    nb, bs = latent_cache.shape[0], latent_cache.shape[1]
    _require(h == plan.num_q_heads and plan.num_kv_heads == 1 and plan.head_dim_v == MLA_LATENT
             and T == plan.num_tokens and bs == plan.block_size,
             "plan was not made for this MLA shape")
    _require(plan.prefix_lens is None, "MLA attention takes no prefix_lens")
    if out is None:
        out = torch.empty(T, h, MLA_LATENT, dtype=_BF16, device=q_latent.device)
    else:
        _check_out(out, "out", (T, h, MLA_LATENT), q_latent.device)
    stream = _ready(plan, q_latent.device)
    _native.call("aia_paged_attention_mla", _ptr(q_latent), q_latent.stride(0),
                 q_latent.stride(1), _ptr(latent_cache), _ptr(plan.block_table),
                 plan.block_table.stride(0), _ptr(plan.cu_seqlens_q), _ptr(plan.seqlens_kv),
                 plan.batch, T, h, MLA_LATENT, MLA_ROPE, bs, nb, float(scale), _ptr(out),
                 out.stride(0), out.stride(1), plan.num_waves, flags, _ptr(plan.workspace),
                 plan.workspace.numel(), stream)
    return out
