"""Per-step device metadata shared by every layer of a step.

The reference hands the attention op host lists (``ctx.cu_seqlens_q``
cumulative ends, ``ctx.seqlens_kv`` per request; forward_context.py:14-15)
and a device block table.  Our kernels read device int32 copies and a
split-K plan; both depend only on the step, so they are built once per
``ForwardContext`` (on first use, or by the GPU packer which attaches them
as ``ctx.aia_cu_seqlens_q`` / ``ctx.aia_seqlens_kv``) and cached on it.
Every context's plan owns its workspace, so steps in flight on different
streams do not share scratch memory.

A context may carry ``aia_prefix_lens``, one per request: the first keys of each
request that all its rows see.  From the second layer on, keys and values of the
prefix depend on all of it, so a prefix has to be computed within one step
(cached blocks of the same prefix in front), and its blocks are shared only
between requests of the same prefix (``block_allocator.prefix_seed``).  A host list
is checked for the first and uploaded; a device int32 tensor is taken as it is
(checked with ``AIA_CHECK_PLAN=1``).

Device metadata attached by a packer is not checked on the host.  Query
lengths that do not add up to the step's token count make the planner plan
nothing (status -1); the attention call then fills its output with NaN.
With ``AIA_CHECK_PLAN=1`` in the environment, the step plans also read the
status back after planning (one device synchronisation per step) and raise
the ValueError of the reference's stager contract
(prefill_input_stager.py:77-81).

``step_shared_plan`` and ``step_sparse_plan`` make the plans of attention with shared
prefixes (groups of requests from ``ctx.aia_group_ids``, device int32 with one entry per
request, else by their first blocks) and of block-sparse attention the same way.
"""
import os

import torch

from auto_infer_amd import ops


def _checking():
    return (os.environ.get("AIA_CHECK_PLAN", "0") == "1"
            and not torch.cuda.is_current_stream_capturing())


def _metadata(ctx, block_size):
    """(block table, cu_seqlens_q, seqlens_kv, query tokens, tensors made here, whether a
    packer attached the lengths) of a context, on the device."""
    bt = ctx.block_table
    cu = getattr(ctx, "aia_cu_seqlens_q", None)
    kv = getattr(ctx, "aia_seqlens_kv", None)
    if cu is None or kv is None:
        dev = bt.device
        ops.check_lists(ctx.cu_seqlens_q, ctx.seqlens_kv, bt.shape[1] * block_size)
        cu = torch.tensor([0, *ctx.cu_seqlens_q], dtype=torch.int32).to(dev)
        kv = torch.tensor(list(ctx.seqlens_kv), dtype=torch.int32).to(dev)
        ctx.aia_cu_seqlens_q, ctx.aia_seqlens_kv = cu, kv
        owned, packed = [cu, kv], False
    else:
        owned, packed = [], True
    T = int(ctx.cu_seqlens_q[-1]) if len(ctx.cu_seqlens_q) else 0
    if bt.dtype != torch.int32:
        bt = bt.to(torch.int32)
        owned.append(bt)
    return bt, cu, kv, T, owned, packed


def _plan_of(ctx, key, make):
    plans = getattr(ctx, "_aia_plans", None)
    if plans is None:
        plans = {}
        ctx._aia_plans = plans
    plan = plans.get(key)
    if plan is None:
        plan = plans[key] = make()
    return plan


def step_plan(ctx, num_q_heads, num_kv_heads, head_dim_v, block_size):
    def make():
        bt, cu, kv, T, owned, packed = _metadata(ctx, block_size)
        pre = getattr(ctx, "aia_prefix_lens", None)
        if pre is not None and not isinstance(pre, torch.Tensor):
            ops.check_prefixes(pre, ctx.cu_seqlens_q, ctx.seqlens_kv)
            pre = ctx.aia_prefix_lens = torch.tensor(list(pre), dtype=torch.int32).to(bt.device)
            owned.append(pre)
        elif pre is not None and _checking():
            ops.check_prefixes(pre.tolist(), ctx.cu_seqlens_q, ctx.seqlens_kv)
        # each context (one step in flight) gets its own workspace from the
        # caching allocator: two steps on two streams never share one, and the
        # plan records every stream it is used on, so the memory is not handed
        # out again while a step on another stream still reads it
        plan = ops.AttentionPlan(bt, cu, kv, T, num_q_heads, num_kv_heads, head_dim_v, block_size,
                                 owned=owned, prefix_lens=pre)
        if packed and _checking():
            plan.status()
        return plan
    return _plan_of(ctx, (num_q_heads, num_kv_heads, head_dim_v, block_size), make)


def _no_prefixes(ctx, what):
    if getattr(ctx, "aia_prefix_lens", None) is not None:
        raise NotImplementedError(f"{what} takes no prefixes that see themselves in both directions")


def step_shared_plan(ctx, num_q_heads, num_kv_heads, head_dim, block_size):
    def make():
        _no_prefixes(ctx, "attention with shared prefixes")
        bt, cu, kv, T, owned, packed = _metadata(ctx, block_size)
        plan = ops.SharedPrefixPlan(bt, cu, kv, T, num_q_heads, num_kv_heads, head_dim, block_size,
                                    group_ids=getattr(ctx, "aia_group_ids", None), owned=owned)
        if packed and _checking():
            plan.status()
        return plan
    return _plan_of(ctx, ("shared", num_q_heads, num_kv_heads, head_dim, block_size), make)


def step_sparse_plan(ctx, num_q_heads, num_kv_heads, head_dim, block_size, num_selected, sink, local):
    def make():
        _no_prefixes(ctx, "block-sparse attention")
        bt, cu, kv, T, owned, packed = _metadata(ctx, block_size)
        plan = ops.BlockSparsePlan(bt, cu, kv, T, num_q_heads, num_kv_heads, head_dim, block_size,
                                   num_selected, sink, local, owned=owned)
        if packed and _checking():
            plan.status()
        return plan
    return _plan_of(ctx, ("sparse", num_q_heads, num_kv_heads, head_dim, block_size, num_selected, sink,
                          local), make)
