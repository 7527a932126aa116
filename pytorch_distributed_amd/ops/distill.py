"""Distillation from a teacher's top logits.

``top_logits`` keeps of a teacher's row what a student is later trained on: its k largest logits, their classes and the
log-sum-exp of all others.  ``distill_loss`` is the Kullback-Leibler divergence of the student from that, forward and
backward; it stands beside ``cross_entropy``, whose loss on the labels is added by the caller where wanted.  GPU path =
the kernels of ``csrc/kernels/distill.hip``; CPU path = stock PyTorch math.
"""
from __future__ import annotations

import math
import operator
from typing import Optional, Tuple

import torch

from . import _lib

MAX_K = 1024
MAX_CLASSES = 1 << 20
MIN_TEMPERATURE, MAX_TEMPERATURE = 2.0 ** -20, 2.0 ** 20

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _temperature(t) -> float:
    t = float(t)
    if not (MIN_TEMPERATURE <= t <= MAX_TEMPERATURE):
        raise ValueError(f"temperature must lie between {MIN_TEMPERATURE} and {MAX_TEMPERATURE}, not {t}")
    return t


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``[rows, last]`` view (a copy only where the last dimension is strided or the leading ones do not collapse)."""
    r = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    return r if r.shape[1] <= 1 or r.stride(1) == 1 else r.contiguous()


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check_logits(name: str, logits: torch.Tensor) -> None:
    if logits.dim() < 1 or logits.dtype not in _FLOATS:
        raise TypeError(f"{name}: logits must be fp32, fp16 or bf16 rows of classes")
    V = logits.shape[-1]
    if V < 1 or V > MAX_CLASSES:
        raise ValueError(f"{name}: {V} classes; 1 to {MAX_CLASSES} are supported")


def top_logits_ref(logits, k, temperature):
    u = logits.double()
    # stable: equal values stay in the order of their classes; NaN first
    order = torch.sort(u, dim=-1, descending=True, stable=True).indices
    idx, left = order[..., :k].contiguous(), order[..., k:]
    if left.shape[-1] == 0:
        rest = torch.full(logits.shape[:-1], -math.inf, dtype=torch.float32, device=logits.device)
    else:
        rest = torch.logsumexp(u.gather(-1, left) / temperature, dim=-1).float()
    return logits.gather(-1, idx), idx, rest


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(values, indices, rest)`` of the ``k`` largest of every row of ``logits`` (``[..., classes]``).

    ``values`` ``[..., k]`` descend and keep the logits' dtype; of equal ones the lowest class comes first, and NaN counts
    as larger than every number.  ``indices`` are int64.  ``rest`` (fp32, ``[...]``) is
    ``log(sum(exp(z_j / temperature)))`` over the classes that were not taken, -inf where there are none (and an
    infinity where it leaves fp32: logits near fp32's ends with a temperature below one).  Not differentiable.
    ``1 <= k <= min(classes, 1024)``, ``2^-20 <= temperature <= 2^20``."""
    _check_logits("top_logits", logits)
    k, t = operator.index(k), _temperature(temperature)
    V = logits.shape[-1]
    if not 1 <= k <= min(V, MAX_K):
        raise ValueError(f"top_logits: k = {k} of {V} classes; 1 to {min(V, MAX_K)} are supported")
    if not logits.is_cuda or logits.numel() == 0:
        with torch.no_grad():
            return top_logits_ref(logits, k, t)
    l = _lib.lib()
    z = _rows(logits.detach() if logits.requires_grad else logits)
    lead = logits.shape[:-1]
    values = torch.empty(lead + (k,), device=z.device, dtype=z.dtype)
    indices = torch.empty(lead + (k,), device=z.device, dtype=torch.int64)
    rest = torch.empty(lead, device=z.device, dtype=torch.float32)
    with _lib.on_device_of(z):
        _lib.check(l.pda_top_logits(_lib.dt(z), z.data_ptr(), _row_stride(z), z.shape[0], V, k, t, values.data_ptr(),
                                    indices.data_ptr(), rest.data_ptr(), _lib.stream()), "pda_top_logits")
    return values, indices, rest


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, values, indices, rest, temperature, reduction):
        l = _lib.lib()
        z, v, i = _rows(logits), _rows(values), _rows(indices)
        if rest is not None:
            rest = rest.reshape(-1).float().contiguous()
        (rows, V), K = z.shape, v.shape[1]
        code, i64 = _lib.dt(z), int(i.dtype is torch.int64)
        with _lib.on_device_of(z):
            # what the rows leave for the backward pass: a shift and a factor each, then one number an entry
            left = torch.empty((rows, 2 + K), device=z.device, dtype=torch.float32)
            row_loss = torch.empty((rows,), device=z.device, dtype=torch.float32)
            loss = None if reduction == "none" else torch.empty((), device=z.device, dtype=torch.float32)
            at = left.data_ptr()
            _lib.check(l.pda_distill_fwd(code, z.data_ptr(), _row_stride(z), rows, V, v.data_ptr(), _lib.dt(v), _row_stride(v),
                                         i.data_ptr(), i64, _row_stride(i), _lib.ptr(rest), K, temperature,
                                         row_loss.data_ptr(), at, at + 8 * rows, _lib.ptr(loss),
                                         1.0 / rows if reduction == "mean" else 1.0, _lib.stream()), "pda_distill_fwd")
        ctx.save_for_backward(z, i, left)
        ctx.cfg = (logits.shape, temperature, reduction)
        if loss is not None:
            return loss
        return row_loss if logits.dim() == 2 else row_loss.view(logits.shape[:-1])

    @staticmethod
    def backward(ctx, g):
        return _backward_once(ctx, g) if torch.is_grad_enabled() else _backward(ctx, g)


def _backward(ctx, g):
    l = _lib.lib()
    z, i, left = ctx.saved_tensors
    shape, temperature, reduction = ctx.cfg
    rows, V = z.shape
    if g.dtype is not torch.float32 or not g.is_contiguous():
        g = g.float().contiguous()
    with _lib.on_device_of(z):
        dz = torch.empty((rows, V), device=z.device, dtype=z.dtype)
        at = left.data_ptr()
        _lib.check(l.pda_distill_bwd(_lib.dt(z), z.data_ptr(), _row_stride(z), rows, V, i.data_ptr(), int(i.dtype is torch.int64),
                                     _row_stride(i), i.shape[1], temperature, at, at + 8 * rows, g.data_ptr(),
                                     int(reduction == "none"), temperature / rows if reduction == "mean" else temperature,
                                     dz.data_ptr(), _lib.stream()), "pda_distill_bwd")
    return dz if len(shape) == 2 else dz.view(shape), None, None, None, None, None


# under create_graph: the gradient is marked as not differentiable again
_backward_once = torch.autograd.function.once_differentiable(_backward)


def distill_loss_ref(logits, values, indices, rest, temperature, reduction):
    """Stock math in fp64, differentiable in the logits."""
    V = logits.shape[-1]
    z, v, i = logits.reshape(-1, V).double(), values.reshape(-1, values.shape[-1]).double(), indices.reshape(-1, values.shape[-1])
    valid = (i >= 0) & (i < V)
    v = torch.where(valid, v / temperature, torch.full_like(v, -math.inf))
    # probabilities of entries of one class add up
    tm = v.amax(1, keepdim=True) if rest is None else torch.maximum(v.amax(1, keepdim=True), rest.reshape(-1, 1).double())
    some = valid.any(1) & ~(tm[:, 0] == -math.inf)
    keep = some[:, None]
    tau = torch.where(keep, v - torch.where(keep, tm, 0.0), -math.inf)
    left = torch.full_like(tm, -math.inf) if rest is None else torch.where(keep, rest.reshape(-1, 1).double() - tm, -math.inf)
    norm = torch.where(keep, tau.exp().sum(1, keepdim=True) + left.exp(), 1.0)
    slot = torch.where(valid, i, V).long()
    p = torch.zeros((z.shape[0], V + 1), dtype=torch.float64, device=z.device).scatter_add_(1, slot, tau.exp() / norm)[:, :V]
    taken = torch.zeros((z.shape[0], V + 1), dtype=torch.bool, device=z.device).scatter_(1, slot, True)[:, :V]
    # a row without entries is not read
    u = torch.where(keep, z, torch.zeros_like(z)) / temperature
    logq = torch.log_softmax(u, dim=1)
    on = p != 0
    terms = torch.where(on, p * (torch.where(on, p, 1.0).log() - torch.where(on, logq, 0.0)), 0.0)
    loss = terms.sum(1)
    if rest is not None:
        pr = (left.exp() / norm)[:, 0]
        has = (pr != 0) & some
        # nothing left outside the entries: log 0, whose gradient is that of the normaliser alone
        open_ = has & (~taken & (logq != -math.inf)).any(1)
        lt = torch.logsumexp(torch.where(open_[:, None], logq.masked_fill(taken, -math.inf), logq), dim=1)
        lt = torch.where(has & ~open_, -math.inf - torch.logsumexp(u, dim=1), lt)
        loss = loss + torch.where(has, pr * (torch.where(has, pr, 1.0).log() - torch.where(has, lt, 0.0)), 0.0)
    loss = torch.where(some, loss, 0.0) * temperature ** 2
    if reduction == "none":
        return loss.float().view(logits.shape[:-1])
    return (loss.mean() if reduction == "mean" else loss.sum()).float()


def distill_loss(logits: torch.Tensor, top_values: torch.Tensor, top_indices: torch.Tensor,
                 rest: Optional[torch.Tensor] = None, temperature: float = 1.0, reduction: str = "mean") -> torch.Tensor:
    """Distillation loss of ``logits`` (``[..., classes]``, fp32 / fp16 / bf16) against a teacher's top logits.

    ``top_values`` and ``top_indices`` (``[..., k]``, int64 or int32) are what :func:`top_logits` returned, or any entries of
    the same meaning; an index outside ``0 .. classes - 1`` marks an empty entry whose value is not looked at.  With
    ``T = temperature``, ``q = softmax(logits / T)`` and ``p`` the teacher's distribution, a row's loss is
    ``T^2 * sum(p * (log p - log q))``:

    * without ``rest`` the teacher is the softmax of its entries alone and every other class has probability zero;
    * with ``rest`` (``[...]``, at the same temperature) the classes that are not entries are one further class, whose
      probability is the teacher's ``exp(rest)`` and the student's sum over them.

    Entries of the same class add their probabilities.  A row without entries (or whose entries are all -inf, and ``rest`` with
    them) has loss and gradient zero, whatever its logits are.  ``reduction``: ``"mean"`` over all rows, ``"sum"`` or ``"none"``
    (``[...]``); the loss is fp32.  Differentiable once, in ``logits`` only.  ``k <= 1024``."""
    _check_logits("distill_loss", logits)
    t = _temperature(temperature)
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"distill_loss: unknown reduction {reduction!r}")
    lead = logits.shape[:-1]
    if top_values.dim() < 1 or top_values.shape != top_indices.shape or top_values.shape[:-1] != lead:
        raise ValueError(f"distill_loss: entries of shape {tuple(top_values.shape)} / {tuple(top_indices.shape)} do not go "
                         f"with logits of shape {tuple(logits.shape)}")
    if not 1 <= top_values.shape[-1] <= MAX_K:
        raise ValueError(f"distill_loss: {top_values.shape[-1]} entries a row; 1 to {MAX_K} are supported")
    if top_values.dtype not in _FLOATS:
        raise TypeError(f"distill_loss: unsupported dtype {top_values.dtype} of top_values")
    if top_indices.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"distill_loss: top_indices must be int64 or int32, not {top_indices.dtype}")
    if rest is not None and (rest.shape != lead or rest.dtype not in _FLOATS):
        raise ValueError(f"distill_loss: rest must be floating-point numbers of shape {tuple(lead)}")
    device = logits.device
    for name, x in (("top_values", top_values), ("top_indices", top_indices), ("rest", rest)):
        if x is not None and x.device != device:
            raise ValueError(f"distill_loss: {name} is on {x.device}, logits on {device}")
    if not logits.is_cuda or logits.numel() == 0:
        return distill_loss_ref(logits, top_values.detach(), top_indices, None if rest is None else rest.detach(), t, reduction)
    return _DistillFn.apply(logits, top_values, top_indices, rest, t, reduction)
