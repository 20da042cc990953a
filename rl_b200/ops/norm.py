"""RMSNorm and fused residual-add + RMSNorm with autograd.

Replaces the Transformer-Engine norm kernels the reference trains with (native
component N7 of the survey; called through MCore layers built in
``nemo_rl/models/megatron/setup.py:2520``).  On CUDA tensors the forward and
backward run in ``csrc/norm.cu``; the backward produces ``dx`` and a per-block
fp32 partial of ``dw`` that is reduced in the same launch sequence.

``rms_norm_fp8`` / ``add_rms_norm_fp8`` are the rollout's norms in front of an fp8
projection: the normalised rows leave as e4m3 values with one scale per 128 of
them, in one kernel and one pass over the residual stream.
"""

from __future__ import annotations

import torch

from rl_b200.ops._ext import ext, use_native

__all__ = ["rms_norm", "add_rms_norm", "rms_norm_ref", "add_rms_norm_ref", "rms_norm_fp8", "add_rms_norm_fp8"]


def rms_norm_ref(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.float()
    return y.to(x.dtype)


def add_rms_norm_ref(x: torch.Tensor, delta: torch.Tensor, w: torch.Tensor, eps: float):
    s = (x.float() + delta.float()).to(x.dtype)
    return rms_norm_ref(s, w, eps), s


def _weight_grad(w: torch.Tensor, dw_fp32: torch.Tensor):
    """Accumulate the fp32 weight gradient straight into ``w.main_grad`` when the
    optimizer attached one (no bf16 ``.grad`` round trip); else return it."""
    main = getattr(w, "main_grad", None)
    if main is not None:
        main.add_(dw_fp32.view_as(main))
        return None
    return dw_fp32.to(w.dtype)


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, eps):
        shape = x.shape
        x2 = x.reshape(-1, shape[-1]).contiguous()
        y, rstd = ext().rmsnorm_fwd(x2, w, eps)
        ctx.save_for_backward(x2, w, rstd)
        ctx.shape = shape
        return y.view(shape)

    @staticmethod
    def backward(ctx, dy):
        x2, w, rstd = ctx.saved_tensors
        dx, dw = ext().rmsnorm_bwd(dy.reshape(x2.shape).contiguous(), x2, w, rstd)
        return dx.view(ctx.shape), _weight_grad(w, dw), None


class _AddRMSNorm(torch.autograd.Function):
    """(y, s) = (rmsnorm(x + delta), x + delta): the residual add of one sub-layer
    fused with the normalisation that opens the next."""

    @staticmethod
    def forward(ctx, x, delta, w, eps):
        shape = x.shape
        x2 = x.reshape(-1, shape[-1]).contiguous()
        d2 = delta.reshape(-1, shape[-1]).contiguous()
        y, s, rstd = ext().add_rmsnorm_fwd(x2, d2, w, eps)
        ctx.save_for_backward(s, w, rstd)
        ctx.shape = shape
        return y.view(shape), s.view(shape)

    @staticmethod
    def backward(ctx, dy, ds):
        s, w, rstd = ctx.saved_tensors
        dy2 = dy.reshape(s.shape).contiguous()
        ds2 = None if ds is None else ds.reshape(s.shape).contiguous()
        dx, dw = ext().rmsnorm_bwd_add(dy2, s, w, rstd, ds2)
        dx = dx.view(ctx.shape)
        return dx, dx, _weight_grad(w, dw), None


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    if use_native(x):
        return _RMSNorm.apply(x, w, eps)
    return rms_norm_ref(x, w, eps)


def add_rms_norm(x: torch.Tensor, delta: torch.Tensor, w: torch.Tensor, eps: float = 1e-5):
    """Return ``(rmsnorm(x + delta) * w, x + delta)``."""
    if use_native(x):
        return _AddRMSNorm.apply(x, delta, w, eps)
    return add_rms_norm_ref(x, delta, w, eps)


def _check_norm_fp8(x: torch.Tensor, delta, w: torch.Tensor) -> None:
    H = x.shape[-1] if x.dim() else 0
    if H == 0 or H % 128:
        raise ValueError(f"rms_norm_fp8: the hidden size must be a multiple of 128, got shape {tuple(x.shape)}")
    if x.is_cuda and x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"rms_norm_fp8: bf16, fp16 or fp32 rows expected on a GPU, got {x.dtype}")
    if w.dim() != 1 or w.shape[0] != H or w.dtype != x.dtype or w.device != x.device:
        raise ValueError(f"rms_norm_fp8: weight {tuple(w.shape)} {w.dtype} on {w.device} for input "
                         f"{tuple(x.shape)} {x.dtype} on {x.device}")
    if delta is not None and (delta.shape != x.shape or delta.dtype != x.dtype or delta.device != x.device):
        raise ValueError(f"rms_norm_fp8: delta {tuple(delta.shape)} {delta.dtype} on {delta.device} for input "
                         f"{tuple(x.shape)} {x.dtype} on {x.device}")
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or (delta is not None and delta.requires_grad)):
        raise RuntimeError("rms_norm_fp8 has no gradient: call it under torch.no_grad() (rollout only)")


def _norm_fp8_ref(x: torch.Tensor, delta, w: torch.Tensor, eps: float, mx: bool):
    from rl_b200.ops.fp8_gemm import quant_act_mx
    from rl_b200.ops.quant import quant_fp8_group_ref

    y, s = (rms_norm_ref(x, w, eps), None) if delta is None else add_rms_norm_ref(x, delta, w, eps)
    y2 = y.reshape(-1, x.shape[-1])
    q, sc = quant_act_mx(y2) if mx else quant_fp8_group_ref(y2, 128, False)
    return q.view(x.shape), sc, s


def rms_norm_fp8(x: torch.Tensor, w: torch.Tensor, eps: float = 1e-5, mx: bool = True):
    """``rmsnorm(x) * w`` (rounded to ``x.dtype``) as e4m3 values with one scale per 128:
    ``(q like x, scales)``.

    ``mx``: power-of-two scales in the MN-major layout of :func:`rl_b200.ops.fp8_gemm.gemm_mxf8`
    (``[H/128, rows rounded up to 128]``, padding 1); otherwise fp32 scales ``[rows, H/128]`` for
    :func:`rl_b200.ops.fp8_gemm.gemm_fp8`.  The hidden size is a multiple of 128 (at most 16384 on a
    GPU).  For inference: an input that needs a gradient is refused.
    """
    _check_norm_fp8(x, None, w)
    return tuple(ext().rmsnorm_fp8(x, None, w, eps, mx, mx)) if x.is_cuda else _norm_fp8_ref(x, None, w, eps, mx)[:2]


def add_rms_norm_fp8(x: torch.Tensor, delta: torch.Tensor, w: torch.Tensor, eps: float = 1e-5, mx: bool = True):
    """``(q, scales, x + delta)``: :func:`rms_norm_fp8` of the residual sum, which is returned too."""
    _check_norm_fp8(x, delta, w)
    return tuple(ext().rmsnorm_fp8(x, delta, w, eps, mx, mx)) if x.is_cuda else _norm_fp8_ref(x, delta, w, eps, mx)
