"""Group norm (+ residual, + activation) over channels-last activations.

GPU path = the kernels of ``csrc/kernels/group_norm.hip``; CPU path = stock PyTorch math.  Statistics belong to a
sample and a group of channels, so nothing crosses ranks or depends on the batch: where the batch of one rank is small,
this is the normalisation that needs neither running statistics nor SyncBatchNorm's all-reduces.
"""
from __future__ import annotations

import functools
import operator
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
    shape = x.shape
    if len(shape) < 2:
        raise ValueError("group_norm_act: x must be [N, ..., C]")
    if x.dtype not in _FLOATS:
        raise TypeError(f"group_norm_act: unsupported dtype {x.dtype}")
    C = shape[-1]
    groups = operator.index(num_groups)
    if groups <= 0 or C == 0 or C % groups != 0:
        raise ValueError(f"group_norm_act: {C} channels do not divide into {num_groups} groups")
    if not eps >= 0.0:
        raise ValueError("group_norm_act: eps must not be negative")
    if gamma is not None or beta is not None:
        if gamma is None or beta is None:
            raise ValueError("group_norm_act: gamma and beta go together")
        for name, t in (("gamma", gamma), ("beta", beta)):
            if t.shape != (C,) or t.dtype not in _FLOATS:
                raise ValueError(f"group_norm_act: {name} must be {C} floating-point numbers")
            if t.device != x.device:
                raise ValueError(f"group_norm_act: {name} is on {t.device}, x on {x.device}")
    if residual is not None and (residual.shape != shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError("group_norm_act: residual must have x's shape, dtype and device")
    return groups


def _f32(p):
    if p is None or (p.dtype is torch.float32 and p.is_contiguous()):
        return p
    return p.detach().float().contiguous()


@functools.lru_cache(maxsize=4096)
def _plan_of(code: int, N: int, S: int, C: int, groups: int, backward: int, aligned: bool) -> int:
    chunks = _lib.lib().pda_group_norm_plan(code, N, S, C, groups, backward, int(aligned))
    if chunks < 0:
        _lib.check(chunks, "pda_group_norm_plan")
    return chunks


def _plan(code: int, N: int, S: int, C: int, groups: int, backward: int, *tensors) -> int:
    """0: a sample's groups stay in registers; otherwise the row chunks of the multi-pass kernels."""
    aligned = True
    for t in tensors:
        if t is not None and t.data_ptr() % 16:
            aligned = False
    return _plan_of(code, N, S, C, groups, backward, aligned)


class _GroupNormActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, residual, groups, act, cap, eps):
        l = _lib.lib()
        x = x.contiguous()
        if residual is not None:
            residual = residual.contiguous()
        N, C = x.shape[0], x.shape[-1]
        S = x.numel() // (N * C)
        code = _lib.dt(x)
        out = torch.empty_like(x)
        ga, be = _f32(gamma), _f32(beta)
        with _lib.on_device_of(x):
            chunks = _plan(code, N, S, C, groups, 0, x, residual)
            part = torch.empty((N * chunks, C, 2), device=x.device, dtype=torch.float64) if chunks else None
            stats = torch.empty((N, groups, 2), device=x.device, dtype=torch.float64)
            _lib.check(l.pda_group_norm_fwd(code, x.data_ptr(), _lib.ptr(residual), out.data_ptr(), _lib.ptr(ga), _lib.ptr(be),
                                            N, S, C, groups, eps, act, cap, chunks, _lib.ptr(part), stats.data_ptr(),
                                            _lib.stream()), "pda_group_norm_fwd")
        ctx.cfg = (N, S, C, groups, act, cap)
        # with no activation the residual passes its gradient on unread
        ctx.save_for_backward(x, gamma, beta, residual if act else None, stats)
        return out

    @staticmethod
    def backward(ctx, dout):
        return _backward_once(ctx, dout) if torch.is_grad_enabled() else _backward(ctx, dout)


def _backward(ctx, dout):
    l = _lib.lib()
    x, gamma, beta, residual, stats = ctx.saved_tensors
    N, S, C, groups, act, cap = ctx.cfg
    dout = dout.contiguous()
    want_dx, want_g, want_b, want_res = ctx.needs_input_grad[:4]
    dres = dx = dg = db = None
    if want_res:
        dres = torch.empty_like(x) if act else dout
    if want_dx or (want_res and act):
        dx = torch.empty_like(x)
    params = want_g or want_b
    if dx is not None or params:
        code = _lib.dt(x)
        ga, be = _f32(gamma), _f32(beta)
        with _lib.on_device_of(x):
            chunks = _plan(code, N, S, C, groups, 1, x, residual, dout)
            # one buffer: the channels' sums, (chunked) the groups' two means, the parameters' gradients
            sums = N * (chunks or 1) * C * 2
            means = N * groups * 2 if chunks else 0
            work = torch.empty((sums + means,), device=x.device, dtype=torch.float32)
            if params:
                dg = torch.empty((C,), device=x.device, dtype=torch.float32)
                db = torch.empty((C,), device=x.device, dtype=torch.float32)
            at = work.data_ptr()
            _lib.check(l.pda_group_norm_bwd(code, x.data_ptr(), _lib.ptr(residual), dout.data_ptr(), _lib.ptr(dx),
                                            _lib.ptr(dres) if act else 0, _lib.ptr(ga), _lib.ptr(be), stats.data_ptr(), N, S, C,
                                            groups, act, cap, chunks, at, at + 4 * sums, _lib.ptr(dg), _lib.ptr(db),
                                            _lib.stream()), "pda_group_norm_bwd")
        if not want_g:
            dg = None
        elif gamma.dtype is not torch.float32:
            dg = dg.to(gamma.dtype)
        if not want_b:
            db = None
        elif beta.dtype is not torch.float32:
            db = db.to(beta.dtype)
    return dx if want_dx else None, dg, db, dres, None, None, None, None


# under create_graph: the gradients are marked as not differentiable again
_backward_once = torch.autograd.function.once_differentiable(_backward)


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
        z = torch.relu(z) if act == 1 else F.hardtanh(z, 0.0, cap)  # (clamp's gradient counts its borders as inside)
    return z.to(x.dtype)


def group_norm_act(x: torch.Tensor, num_groups: int, gamma: Optional[torch.Tensor] = None,
                   beta: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                   act: Union[bool, float, str] = False, eps: float = 1e-5) -> torch.Tensor:
    """``act(group_norm(x) * gamma + beta + residual)`` for ``x`` of shape ``[N, ..., C]`` (fp32, fp16 or bf16).

    The mean and the variance are those of one sample's ``C / num_groups`` adjacent channels at all its positions.
    ``act``: ``False`` (none), ``True`` (ReLU), a positive number (ReLU clipped there, 6 for ReLU6) or ``"silu"``.
    ``gamma`` and ``beta`` (``[C]``, both or neither) keep their own dtype.  Differentiable once, in ``x``, ``gamma``,
    ``beta`` and ``residual``; a sample whose values hold a NaN or an infinity gives NaN in that group.  Gradients are those of
    deviations (``sqrt(var + eps)``) between 1e-18 and 1e18, whose squares fp32 holds."""
    eps = float(eps)
    groups = _check(x, num_groups, gamma, beta, residual, eps)
    code, cap = _act_code(act)
    if x.numel() == 0:
        # no positions: an empty result that still carries (zero) gradients
        out = x * 1.0 if residual is None else x + residual
        return out if gamma is None else out * gamma.to(x.dtype) + beta.to(x.dtype)
    if not x.is_cuda:
        return group_norm_act_ref(x, groups, gamma, beta, residual, code, cap, eps)
    return _GroupNormActFn.apply(x, gamma, beta, residual, groups, code, cap, eps)
