"""Group norm with an activation on the CPU: values, gradients and what it refuses."""
import pytest
import torch
import torch.nn.functional as F

from pytorch_distributed_amd import ops


@pytest.mark.parametrize("act", [False, True, 6.0, "silu"])
@pytest.mark.parametrize("residual", [False, True])
def test_group_norm_act_values(act, residual):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 5, 4, 12, generator=g) + 2.0
    res = torch.randn(3, 5, 4, 12, generator=g) if residual else None
    w, b = torch.randn(12, generator=g), torch.randn(12, generator=g)
    y = ops.group_norm_act(x, 3, w, b, res, act, 1e-3)
    z = F.group_norm(x.double().permute(0, 3, 1, 2), 3, w.double(), b.double(), 1e-3).permute(0, 2, 3, 1)
    z = z if res is None else z + res.double()
    ref = {False: lambda t: t, True: torch.relu, 6.0: lambda t: t.clamp(0, 6), "silu": F.silu}[act](z)
    # the result is rounded once from 64 bits
    assert y.dtype == torch.float32 and bool(((y.double() - ref).abs() <= 2.0 ** -23 * ref.abs() + 1e-12).all())


def test_group_norm_act_gradients_against_differences():
    """Central differences of step h: the error is that of the third derivative (h^2) and of the fp32 output (2^-24 / h)."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 3, 8, generator=g)
    w, b, res = torch.rand(8, generator=g) + 0.5, torch.randn(8, generator=g), torch.randn(2, 3, 8, generator=g)
    dy = torch.randn(2, 3, 8, generator=g).double()
    args = [t.clone().requires_grad_(True) for t in (x, w, b, res)]

    def f(x, w, b, r):
        return (ops.group_norm_act(x, 2, w, b, r, "silu", 1e-2).double() * dy).sum()

    grads = torch.autograd.grad(f(*args), args)
    h = 2.0 ** -7
    for k, t in enumerate((x, w, b, res)):
        for i in range(0, t.numel(), 5):
            lo, hi = [[v.clone() for v in (x, w, b, res)] for _ in range(2)]
            lo[k].view(-1)[i] -= h
            hi[k].view(-1)[i] += h
            num = (f(*hi) - f(*lo)) / (2 * h)
            # third derivatives of a normalised value reach a few tens here
            assert abs(float(num) - float(grads[k].reshape(-1)[i])) < 50 * h * h / 6 + 24 * 2.0 ** -24 * 4 / h


def test_group_norm_act_shapes():
    for shape in [(2, 8), (2, 3, 8), (1, 2, 3, 4, 8)]:
        assert ops.group_norm_act(torch.randn(shape), 4).shape == shape
    x = torch.randn(0, 4, 4, 8, requires_grad=True)
    w, b = torch.ones(8, requires_grad=True), torch.zeros(8, requires_grad=True)
    ops.group_norm_act(x, 4, w, b, None, True).sum().backward()
    assert x.grad.shape == x.shape and float(w.grad.abs().sum()) == 0.0 and float(b.grad.abs().sum()) == 0.0


def test_group_norm_act_refusals():
    x = torch.randn(2, 3, 8)
    w = torch.ones(8)
    bad = [dict(num_groups=3), dict(num_groups=0), dict(num_groups=4, eps=-1.0), dict(num_groups=4, eps=float("nan")),
           dict(num_groups=4, act="gelu"), dict(num_groups=4, act=-1.0), dict(num_groups=4, act=float("inf")),
           dict(num_groups=4, gamma=w), dict(num_groups=4, gamma=w, beta=torch.ones(4)),
           dict(num_groups=4, gamma=w.long(), beta=w.long()), dict(num_groups=4, residual=x[:1]),
           dict(num_groups=4, residual=x.half())]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.group_norm_act(x, **kw)
    with pytest.raises(TypeError):
        ops.group_norm_act(x.double(), 4)
    with pytest.raises(ValueError):
        ops.group_norm_act(torch.randn(8), 4)
