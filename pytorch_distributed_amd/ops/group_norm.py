"""Group norm (+ residual, + activation) over channels-last activations.

GPU path = the kernels of ``csrc/kernels/group_norm.hip``; CPU path = stock PyTorch math.  Statistics belong to a
sample and a group of channels, so nothing crosses ranks or depends on the batch: where the batch of one rank is small,
this is the normalisation that needs neither running statistics nor SyncBatchNorm's all-reduces.
"""
from __future__ import annotations

from typing import Optional, Union

import torch
import torch.nn.functional as F

from . import _lib

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _act_code(act) -> tuple:
    """(kernel code, cap) of the activation argument: ``False`` / ``None``, ``True`` (ReLU), a positive number (ReLU clipped
    there) or ``"silu"``."""
    if act is False or act is None:
        return 0, 0.0
    if act is True:
        return 1, 0.0
    if isinstance(act, str):
        if act == "silu":
            return 3, 0.0
    elif isinstance(act, (int, float)) and 0.0 < float(act) < float("inf"):
        return 2, float(act)
    raise ValueError(f"group_norm_act: act must be False, True, a positive number or 'silu', not {act!r}")


def _check(x, num_groups, gamma, beta, residual, eps) -> int:
    if x.dim() < 2:
        raise ValueError("group_norm_act: x must be [N, ..., C]")
    if x.dtype not in _FLOATS:
        raise TypeError(f"group_norm_act: unsupported dtype {x.dtype}")
    C = x.shape[-1]
    groups = int(num_groups)
    if groups <= 0 or C == 0 or C % groups != 0:
        raise ValueError(f"group_norm_act: {C} channels do not divide into {num_groups} groups")
    if not float(eps) >= 0.0:
        raise ValueError("group_norm_act: eps must not be negative")
    if (gamma is None) != (beta is None):
        raise ValueError("group_norm_act: gamma and beta go together")
    for name, t in (("gamma", gamma), ("beta", beta)):
        if t is None:
            continue
        if t.shape != (C,) or t.dtype not in _FLOATS:
            raise ValueError(f"group_norm_act: {name} must be {C} floating-point numbers")
        if t.device != x.device:
            raise ValueError(f"group_norm_act: {name} is on {t.device}, x on {x.device}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError("group_norm_act: residual must have x's shape, dtype and device")
    return groups


def _plan(l, x, S: int, groups: int, backward: bool, *others) -> int:
    """0: a sample's groups stay in registers; otherwise the row chunks of the multi-pass kernels."""
    aligned = all(t is None or t.data_ptr() % 16 == 0 for t in (x,) + others)
    chunks = l.pda_group_norm_plan(_lib.dt(x), x.shape[0], S, x.shape[-1], groups, int(backward), int(aligned))
    if chunks < 0:
        _lib.check(chunks, "pda_group_norm_plan")
    return chunks


def _f32(p):
    return None if p is None else p.detach().float().contiguous()


class _GroupNormActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, residual, groups, act, cap, eps):
        l = _lib.lib()
        x = x.contiguous()
        residual = None if residual is None else residual.contiguous()
        N, C = x.shape[0], x.shape[-1]
        S = x.numel() // (N * C)
        out = torch.empty_like(x)
        ga, be = _f32(gamma), _f32(beta)
        with torch.cuda.device(x.device):
            chunks = _plan(l, x, S, groups, False, residual)
            part = torch.empty((N * chunks, C, 2), device=x.device, dtype=torch.float64) if chunks else None
            stats = torch.empty((N, groups, 2), device=x.device, dtype=torch.float64)
            _lib.check(l.pda_group_norm_fwd(_lib.dt(x), x.data_ptr(), _lib.ptr(residual), out.data_ptr(), _lib.ptr(ga),
                                            _lib.ptr(be), N, S, C, groups, eps, act, cap, chunks, _lib.ptr(part),
                                            stats.data_ptr(), _lib.stream()), "pda_group_norm_fwd")
        ctx.cfg = (groups, act, cap)
        # with no activation the residual passes its gradient on unread
        ctx.save_for_backward(x, gamma, beta, residual if act else None, stats)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        l = _lib.lib()
        x, gamma, beta, residual, stats = ctx.saved_tensors
        groups, act, cap = ctx.cfg
        dout = dout.contiguous()
        N, C = x.shape[0], x.shape[-1]
        S = x.numel() // (N * C)
        want_dx, want_g, want_b, want_res = ctx.needs_input_grad[:4]
        ga, be = _f32(gamma), _f32(beta)
        dres = dx = dgb = None
        if want_res:
            dres = dout if act == 0 else torch.empty_like(x)
        if want_dx or (want_res and act):
            dx = torch.empty_like(x)
        with torch.cuda.device(x.device):
            if want_g or want_b:
                dgb = torch.empty((2, C), device=x.device, dtype=torch.float32)
            if dx is not None or dgb is not None:
                chunks = _plan(l, x, S, groups, True, residual, dout)
                part = torch.empty((N * max(chunks, 1), C, 2), device=x.device, dtype=torch.float32)
                ab = torch.empty((N, groups, 2), device=x.device, dtype=torch.float32) if chunks else None
                _lib.check(l.pda_group_norm_bwd(_lib.dt(x), x.data_ptr(), _lib.ptr(residual), dout.data_ptr(), _lib.ptr(dx),
                                                _lib.ptr(dres) if act else 0, _lib.ptr(ga), _lib.ptr(be), stats.data_ptr(),
                                                N, S, C, groups, act, cap, chunks, part.data_ptr(), _lib.ptr(ab),
                                                0 if dgb is None else dgb[0].data_ptr(),
                                                0 if dgb is None else dgb[1].data_ptr(), _lib.stream()),
                           "pda_group_norm_bwd")
        dg = dgb[0].to(gamma.dtype) if want_g else None
        db = dgb[1].to(beta.dtype) if want_b else None
        return dx if want_dx else None, dg, db, dres, None, None, None, None


def group_norm_act_ref(x, groups, gamma, beta, residual, act, cap, eps):
    """Stock math, differentiable; statistics in fp64."""
    N, C = x.shape[0], x.shape[-1]
    v = x.reshape(N, x.numel() // (N * C), groups, C // groups).double()
    var, mean = torch.var_mean(v, dim=(1, 3), unbiased=False, keepdim=True)
    z = ((v - mean) * torch.rsqrt(var + eps)).reshape(x.shape)
    if gamma is not None:
        z = z * gamma.double() + beta.double()
    if residual is not None:
        z = z + residual.double()
    if act == 3:
        z = F.silu(z)
    elif act:
        z = torch.relu(z) if act == 1 else torch.clamp(z, 0.0, cap)
    return z.to(x.dtype)


def group_norm_act(x: torch.Tensor, num_groups: int, gamma: Optional[torch.Tensor] = None,
                   beta: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                   act: Union[bool, float, str] = False, eps: float = 1e-5) -> torch.Tensor:
    """``act(group_norm(x) * gamma + beta + residual)`` for ``x`` of shape ``[N, ..., C]`` (fp32, fp16 or bf16).

    The mean and the variance are those of one sample's ``C / num_groups`` adjacent channels at all its positions.
    ``act``: ``False`` (none), ``True`` (ReLU), a positive number (ReLU clipped there, 6 for ReLU6) or ``"silu"``.
    ``gamma`` and ``beta`` (``[C]``, both or neither) keep their own dtype.  Differentiable once, in ``x``, ``gamma``,
    ``beta`` and ``residual``; a sample whose values hold a NaN or an infinity gives NaN in that group."""
    groups = _check(x, num_groups, gamma, beta, residual, eps)
    code, cap = _act_code(act)
    if x.numel() == 0:
        # no positions: an empty result that still carries (zero) gradients
        out = x * 1.0 if residual is None else x + residual
        return out if gamma is None else out * gamma.to(x.dtype) + beta.to(x.dtype)
    if not x.is_cuda:
        return group_norm_act_ref(x, groups, gamma, beta, residual, code, cap, float(eps))
    return _GroupNormActFn.apply(x, gamma, beta, residual, groups, code, cap, float(eps))
