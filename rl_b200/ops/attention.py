"""Attention ops: packed variable-length causal GQA attention (training and
prefill), paged-KV decode attention and KV-cache writes (rollout).

Reference counterparts: training attention is TE ``DotProductAttention`` over
packed THD sequences (native component N5, ``nemo_rl/models/megatron/data.py:1673``
builds the ``cu_seqlens``); rollout attention is vLLM / MCore paged attention
with ``block_size_tokens: 256`` (N15, ``examples/configs/grpo_math_1B.yaml:345``).

Layouts
-------
* packed: ``q [T, nq, hd]``, ``k, v [T, nkv, hd]`` (may be strided views of the
  QKV projection), ``cu_seqlens [B+1] int32``; output ``[T, nq, hd]`` and the
  per-row log-sum-exp ``lse [nq, T] fp32`` kept for the backward pass.
* paged cache: ``k_cache, v_cache [num_blocks, block_size, nkv, hd]``,
  ``block_tables [B, max_blocks] int32``, ``seq_lens [B] int32``;
  ``slot_mapping [T] int64`` = block * block_size + offset for writes.
* shared prefixes: rows ``[group_starts[g], group_starts[g+1])`` of a decode batch have the same
  keys in their first ``prefix_lens[g]`` positions (samples of one prompt);
  ``shared_prefix_decode_attention`` reads those once per group.
"""

from __future__ import annotations

import math
import os
from typing import NamedTuple, Optional

import torch

from rl_b200.ops._ext import add_launches, ext, use_native

__all__ = [
    "flash_attn_varlen",
    "flash_attn_varlen_ref",
    "PAGED_DECODE_GROUPS",
    "paged_decode_attention",
    "paged_decode_attention_ref",
    "SharedPrefixPlan",
    "shared_prefix_plan",
    "shared_prefix_decode_attention",
    "write_kv_cache",
    "write_kv_cache_ref",
]


def flash_attn_varlen_ref(q, k, v, cu_seqlens, scale: Optional[float] = None, causal: bool = True):
    """fp32 oracle: loop over packed sequences, explicit softmax."""
    T, nq, hd = q.shape
    nkv = k.shape[1]
    g = nq // nkv
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    out = torch.empty(T, nq, hd, dtype=torch.float32, device=q.device)
    lse = torch.empty(nq, T, dtype=torch.float32, device=q.device)
    cu = cu_seqlens.tolist()
    for b in range(len(cu) - 1):
        s, e = cu[b], cu[b + 1]
        if e <= s:
            continue
        qb = q[s:e].float().transpose(0, 1)                                  # [nq, L, hd]
        kb = k[s:e].float().transpose(0, 1).repeat_interleave(g, dim=0)      # [nq, L, hd]
        vb = v[s:e].float().transpose(0, 1).repeat_interleave(g, dim=0)
        sc = torch.matmul(qb, kb.transpose(-1, -2)) * scale
        if causal:
            L = e - s
            m = torch.ones(L, L, dtype=torch.bool, device=q.device).triu(1)
            sc = sc.masked_fill(m, float("-inf"))
        lse[:, s:e] = torch.logsumexp(sc, -1)
        out[s:e] = torch.matmul(torch.softmax(sc, -1), vb).transpose(0, 1)
    return out.to(q.dtype), lse


# RL_B200_ATTN_TC=0 keeps the forward on the mma.sync kernel (A/B timing)
_ATTN_TC = os.environ.get("RL_B200_ATTN_TC", "1") == "1"
# RL_B200_ATTN_TC_BWD=0 keeps the backward on the mma.sync kernel (A/B timing)
_TC_BWD = os.environ.get("RL_B200_ATTN_TC_BWD", "1") == "1"


def _tc_ok(*xs) -> bool:
    """The tcgen05 forward (``csrc/attention_sm100.cu``) takes head dim 128 bf16 views
    with contiguous heads and 16-byte aligned token rows (TMA tensor maps)."""
    return _ATTN_TC and all(x.dim() == 3 and x.shape[-1] == 128 and x.dtype == torch.bfloat16 and x.stride(2) == 1
                            and x.stride(1) == 128 and x.stride(0) % 8 == 0 and x.data_ptr() % 16 == 0 for x in xs)


def fa_forward(q, k, v, cu_seqlens, max_seqlen: int, scale: float, causal: bool):
    """Native varlen forward: (out, lse) from the tcgen05 kernel when it applies."""
    if os.environ.get("RLB_PROBE_ATTN_FP32") == "1":  # numerics probe only: fp32 attention
        o, lse = flash_attn_varlen_ref(q.float(), k.float(), v.float(), cu_seqlens, scale, causal)
        return o.to(q.dtype), lse
    if _tc_ok(q, k, v):
        return ext().flash_attn_fwd_tc(q, k, v, cu_seqlens, int(max_seqlen), float(scale), bool(causal))
    return ext().flash_attn_fwd(q, k, v, cu_seqlens, int(max_seqlen), float(scale), bool(causal))


def fa_seg_forward(q, k, v, seg, max_q: int, scale: float, cp_flags=None, cp_epoch: int = 0, cp_size: int = 0):
    """Native segment forward (context parallelism), tcgen05 when it applies."""
    if _tc_ok(q, k, v):
        return ext().flash_attn_seg_fwd_tc(q, k, v, seg, int(max_q), float(scale), cp_flags, int(cp_epoch),
                                           int(cp_size))
    return ext().flash_attn_seg_fwd(q, k, v, seg, int(max_q), float(scale), cp_flags, int(cp_epoch), int(cp_size))


def fa_backward(do, q, k, v, o, lse, cu_seqlens, max_seqlen: int, scale: float, causal: bool):
    """Native varlen backward: (dq, dk, dv), tcgen05 kernel when it applies."""
    do = do.contiguous()
    if _TC_BWD and _tc_ok(q, k, v, do) and o.is_contiguous():
        return ext().flash_attn_bwd_tc(do, q, k, v, o, lse, cu_seqlens, int(max_seqlen), float(scale), bool(causal))
    return ext().flash_attn_bwd(do, q, k, v, o, lse, cu_seqlens, int(max_seqlen), float(scale), bool(causal))


def fa_seg_backward(do, q, k, v, o, lse, seg, max_k: int, scale: float):
    """Native segment backward (context parallelism), tcgen05 when it applies."""
    do = do.contiguous()
    if _TC_BWD and _tc_ok(q, k, v, do) and o.is_contiguous():
        return ext().flash_attn_seg_bwd_tc(do, q, k, v, o, lse, seg, int(max_k), float(scale))
    return ext().flash_attn_seg_bwd(do, q, k, v, o, lse, seg, int(max_k), float(scale))


class _FlashAttnVarlen(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, max_seqlen, scale, causal):
        o, lse = fa_forward(q, k, v, cu_seqlens, int(max_seqlen), float(scale), bool(causal))
        ctx.save_for_backward(q, k, v, o, lse, cu_seqlens)
        ctx.meta = (int(max_seqlen), float(scale), bool(causal))
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, lse, cu = ctx.saved_tensors
        max_seqlen, scale, causal = ctx.meta
        dq, dk, dv = fa_backward(do, q, k, v, o, lse, cu, max_seqlen, scale, causal)
        return dq, dk, dv, None, None, None, None


def flash_attn_varlen(q, k, v, cu_seqlens, max_seqlen: int, scale: Optional[float] = None, causal: bool = True):
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[-1])
    if use_native(q):
        return _FlashAttnVarlen.apply(q, k, v, cu_seqlens, max_seqlen, scale, causal)
    return flash_attn_varlen_ref(q, k, v, cu_seqlens, scale, causal)[0]


class _FlashAttnSegments(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, seg, max_q, max_k, scale):
        o, lse = fa_seg_forward(q, k, v, seg, int(max_q), float(scale))
        ctx.save_for_backward(q, k, v, o, lse, seg)
        ctx.meta = (int(max_k), float(scale))
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, lse, seg = ctx.saved_tensors
        max_k, scale = ctx.meta
        dq, dk, dv = fa_seg_backward(do, q, k, v, o, lse, seg, max_k, scale)
        return dq, dk, dv, None, None, None, None


def flash_attn_segments(q, k, v, q_start, q_len, k_start, k_len, max_q: int, max_k: int, scale: float):
    """Segment ``s`` attends queries ``[q_start[s], +q_len[s])`` to keys
    ``[k_start[s], +k_len[s])``, causal with the last query aligned to the last
    key (context-parallel chunks against their sequence prefixes; segments may
    share keys).  Native kernels: the varlen flash-attention kernels of
    ``csrc/attention.cu`` with per-segment ranges."""
    seg = torch.stack([q_start, q_len, k_start, k_len], 1).to(torch.int32).contiguous()
    return _FlashAttnSegments.apply(q.contiguous(), k.contiguous(), v.contiguous(), seg, max_q, max_k, scale)


def flash_attn_varlen_fwd(q, k, v, cu_seqlens, max_seqlen: int, scale: Optional[float] = None,
                          causal: bool = True):
    """Forward only (prefill): returns (out, lse)."""
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[-1])
    if use_native(q):
        return fa_forward(q, k, v, cu_seqlens, int(max_seqlen), float(scale), bool(causal))
    return flash_attn_varlen_ref(q, k, v, cu_seqlens, scale, causal)


def write_kv_cache_ref(k, v, k_cache, v_cache, slot_mapping, k_scale: float = 1.0, v_scale: float = 1.0):
    nb, bs = k_cache.shape[:2]
    kc = k_cache.view(nb * bs, *k_cache.shape[2:])
    vc = v_cache.view(nb * bs, *v_cache.shape[2:])
    if kc.dtype == torch.float8_e4m3fn:
        k, v = (k.float() / k_scale).clamp(-448, 448), (v.float() / v_scale).clamp(-448, 448)
    kc[slot_mapping.long()] = k.to(kc.dtype)
    vc[slot_mapping.long()] = v.to(vc.dtype)


def write_kv_cache(k, v, k_cache, v_cache, slot_mapping, k_scale: float = 1.0, v_scale: float = 1.0):
    """Scatter ``k, v [T, nkv, hd]`` into the paged cache at ``slot_mapping``
    (an fp8 cache stores ``k / k_scale`` and ``v / v_scale``)."""
    if use_native(k):
        ext().write_kv_cache(k, v, k_cache, v_cache, slot_mapping, float(k_scale), float(v_scale))
    else:
        write_kv_cache_ref(k, v, k_cache, v_cache, slot_mapping, k_scale, v_scale)


def paged_decode_attention_ref(q, k_cache, v_cache, block_tables, seq_lens, scale: Optional[float] = None):
    B, nq, hd = q.shape
    nkv = k_cache.shape[2]
    bs = k_cache.shape[1]
    g = nq // nkv
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    out = torch.empty(B, nq, hd, dtype=torch.float32, device=q.device)
    for b in range(B):
        L = int(seq_lens[b])
        nblk = (L + bs - 1) // bs
        blocks = block_tables[b, :nblk].long()
        kb = k_cache[blocks].reshape(-1, nkv, hd)[:L].float()   # [L, nkv, hd]
        vb = v_cache[blocks].reshape(-1, nkv, hd)[:L].float()
        kb = kb.repeat_interleave(g, dim=1).transpose(0, 1)      # [nq, L, hd]
        vb = vb.repeat_interleave(g, dim=1).transpose(0, 1)
        sc = torch.einsum("hd,hld->hl", q[b].float(), kb) * scale
        out[b] = torch.einsum("hl,hld->hd", torch.softmax(sc, -1), vb)
    return out.to(q.dtype)


# query heads per KV head that the kernel of paged_decode_attention has (csrc/attention.cu)
PAGED_DECODE_GROUPS = (1, 2, 4, 8)


def paged_decode_attention(q, k_cache, v_cache, block_tables, seq_lens, scale: Optional[float] = None,
                           max_seq_len: int = 0, k_scale: float = 1.0, v_scale: float = 1.0):
    """One query token per sequence against its paged KV history (``seq_lens``
    includes the token just written).  fp8 caches are dequantised with the
    per-tensor ``k_scale`` / ``v_scale``."""
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[-1])
    if use_native(q):
        return ext().paged_decode_attn(q, k_cache, v_cache, block_tables, seq_lens, float(scale),
                                       int(max_seq_len), float(k_scale), float(v_scale))
    if k_cache.dtype != q.dtype:
        k_cache = k_cache.to(torch.float32) * k_scale
        v_cache = v_cache.to(torch.float32) * v_scale
    return paged_decode_attention_ref(q, k_cache, v_cache, block_tables, seq_lens, scale)


class SharedPrefixPlan(NamedTuple):
    """Work plan of :func:`shared_prefix_decode_attention` for one set of lengths."""

    buf: torch.Tensor
    rows: int
    groups: int
    heads: int
    kv_heads: int
    head_dim: int
    block_size: int
    max_blocks: int
    fp8: bool


def _check_groups(seq_lens, group_starts, prefix_lens):
    dev = seq_lens.device
    for t in (seq_lens, group_starts, prefix_lens):
        if t.dim() != 1 or t.dtype not in (torch.int32, torch.int64) or t.device != dev:
            raise ValueError("shared prefix: lengths and group starts must be integer vectors on one device, got "
                             f"{tuple(t.shape)} {t.dtype} on {t.device} (lengths on {dev})")
    if group_starts.shape[0] != prefix_lens.shape[0] + 1:
        raise ValueError(f"shared prefix: {prefix_lens.numel()} prefix lengths need {prefix_lens.numel() + 1} group "
                         f"starts, got {group_starts.numel()}")


def shared_prefix_plan(seq_lens, group_starts, prefix_lens, num_heads: int, num_kv_heads: int, head_dim: int,
                       block_size: int, max_blocks: int, fp8: bool = False) -> SharedPrefixPlan:
    """Plan the attention of one decode step: which CTA takes which keys of which rows.

    The plan depends on the lengths, the head, page and table sizes and the cache's type alone
    (lengths are read on the device, without a synchronisation), so one plan serves every layer of
    the step; lengths that change need a new one.  ``max_blocks`` is the width of the block tables,
    ``fp8`` says that the cache holds e4m3.  GPU only."""
    _check_groups(seq_lens, group_starts, prefix_lens)
    key = (int(num_heads), int(num_kv_heads), int(head_dim), int(block_size), int(max_blocks), bool(fp8))
    return SharedPrefixPlan(ext().shared_prefix_plan(group_starts, prefix_lens, seq_lens, *key), seq_lens.shape[0],
                            prefix_lens.shape[0], *key)


def shared_prefix_decode_attention(q, k_cache, v_cache, block_tables, seq_lens, group_starts, prefix_lens,
                                   scale: Optional[float] = None, k_scale: float = 1.0, v_scale: float = 1.0,
                                   plan: Optional[SharedPrefixPlan] = None):
    """:func:`paged_decode_attention` for rows that share prefixes, each read once for its group.

    ``q [B, nq, hd]`` (bf16 on a GPU), caches ``[blocks, block_size, nkv, hd]`` (bf16, or e4m3 with
    ``k_scale`` / ``v_scale``), ``block_tables [B, max_blocks]`` (complete for every row, its prefix
    included), ``seq_lens [B]``, ``group_starts [G+1]`` ascending, ``prefix_lens [G]``: the rows from
    ``group_starts[g]`` up to ``group_starts[g+1]`` hold equal keys and values in their first
    ``prefix_lens[g]`` positions, on the same pages or on copies.  Rows outside every group attend
    alone; a row of length 0 gives zeros and bounds no group.  A prefix longer than a row of its
    group is shared up to that row's length.

    On a GPU the softmax weights are rounded to bf16, or f16 with an e4m3 cache, for the product with V, and
    sums are taken in another order than row by row: results agree within those roundings, not bit for bit.

    ``plan`` (:func:`shared_prefix_plan` of the same lengths) saves planning once per layer; it is
    followed whatever the lengths are now.  Lengths and tables are device data: table entries
    outside the cache, lengths beyond the tables (or beyond what a plan numbers: at least 64 x 2^30 keys over
    KV heads x (2 rows + groups)) and group starts that descend are not followed but reported by
    :func:`rl_b200.ops._ext.check_device_errors`.
    """
    _check_groups(seq_lens, group_starts, prefix_lens)
    B = q.shape[0] if q.dim() == 3 else -1
    if B < 0 or k_cache.dim() != 4 or v_cache.shape != k_cache.shape or q.shape[2] != k_cache.shape[3] \
            or k_cache.shape[2] == 0 or q.shape[1] % k_cache.shape[2]:
        raise ValueError(f"shared prefix attention: q {tuple(q.shape)} with caches {tuple(k_cache.shape)}, "
                         f"{tuple(v_cache.shape)}")
    if block_tables.dim() != 2 or block_tables.shape[0] != B or seq_lens.shape[0] != B:
        raise ValueError(f"shared prefix attention: {B} queries, block tables {tuple(block_tables.shape)}, "
                         f"{seq_lens.shape[0]} lengths")
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[-1])
    if not use_native(q):
        if k_cache.dtype == torch.float8_e4m3fn:
            k_cache, v_cache = k_cache.float() * k_scale, v_cache.float() * v_scale
        out = torch.zeros_like(q, memory_format=torch.contiguous_format)
        live = seq_lens > 0
        if bool(live.any()):  # every row's table is complete: the grouping changes what is read, not the result
            out[live] = paged_decode_attention_ref(q[live], k_cache, v_cache, block_tables[live], seq_lens[live], scale)
        return out
    if plan is not None and plan[1:] != (B, prefix_lens.shape[0], q.shape[1], k_cache.shape[2], q.shape[2],
                                         k_cache.shape[1], block_tables.shape[1],
                                         k_cache.dtype == torch.float8_e4m3fn):
        raise ValueError(f"shared prefix attention: plan {plan[1:]} used for {B} rows, {prefix_lens.shape[0]} groups, "
                         f"q {tuple(q.shape)}, caches {tuple(k_cache.shape)}, tables {tuple(block_tables.shape)}")
    if plan is None:
        add_launches(1)  # the native call plans first
    return ext().shared_prefix_attn(q, k_cache, v_cache, block_tables, seq_lens, group_starts, prefix_lens,
                                    None if plan is None else plan.buf, scale, k_scale, v_scale)
