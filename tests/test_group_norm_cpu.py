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
    with pytest.raises(TypeError):
        ops.group_norm_act(x, 4.0)
    with pytest.raises(ValueError):
        ops.group_norm_act(torch.randn(8), 4)


def test_group_norm_module_and_refusals():
    from pytorch_distributed_amd import nn as pnn
    m = pnn.GroupNorm(4, 8)
    x = torch.randn(2, 3, 3, 8)
    assert torch.equal(m(x, x, True), ops.group_norm_act(x, 4, m.weight, m.bias, x, True))
    assert pnn.GroupNorm(2, 8, affine=False)(x).shape == x.shape
    for a in [(3, 8), (0, 8)]:
        with pytest.raises(ValueError):
            pnn.GroupNorm(*a)


@pytest.mark.parametrize("arch", ["resnet18", "resnext50_32x4d", "vgg11_bn", "densenet121", "mobilenet_v2", "shufflenet_v2_x0_5",
                                  "mnasnet0_5", "googlenet"])
def test_group_norm_in_place_of_batch_norm(arch):
    """Every family runs with group norm: one sample's logits do not depend on its batch, nor on training mode."""
    from pytorch_distributed_amd import nn as pnn, models
    torch.manual_seed(0)
    m = models.get_model(arch, num_classes=7)
    names = [n for n, _ in m.named_parameters()]
    pnn.GroupNorm.convert_group_norm(m, 32)
    assert [n for n, _ in m.named_parameters()] == names
    assert not any(isinstance(k, pnn.BatchNorm2d) for k in m.modules())
    for k in m.modules():
        if isinstance(k, pnn.Dropout):
            k.p = 0.0
    x = torch.randn(2, 3, 64, 64)
    m.train()
    out = m(x)
    # fp32 through some fifty layers, summed in another order for another batch size
    torch.testing.assert_close(m(x[:1]), out[:1], rtol=1e-3, atol=1e-3 * float(out.detach().abs().max()))
    out.square().mean().backward()
    grads = [p.grad for k in m.modules() if isinstance(k, pnn.GroupNorm) for p in (k.weight, k.bias)]
    assert all(g is not None and bool(torch.isfinite(g).all()) for g in grads)
    assert any(bool(g.any()) for g in grads)


def test_group_norm_resnet_layers_one_by_one():
    """The converted ResNet against the same parameters in torch.nn.functional, values and gradients."""
    from pytorch_distributed_amd import nn as pnn, models
    torch.manual_seed(1)
    m = pnn.GroupNorm.convert_group_norm(models.resnet18(num_classes=5), 16)
    m.set_input_normalization([0.4, 0.5, 0.6], [0.2, 0.3, 0.25], 0.5)
    x = torch.rand(2, 3, 40, 40)

    def gn(k, t):
        return F.group_norm(t, k.num_groups, k.weight, k.bias, k.eps)

    y = (x * 0.5 - torch.tensor([0.4, 0.5, 0.6]).view(1, 3, 1, 1)) / torch.tensor([0.2, 0.3, 0.25]).view(1, 3, 1, 1)
    y = F.max_pool2d(torch.relu(gn(m.bn1, F.conv2d(y, m.conv1.weight, None, 2, 3))), 3, 2, 1)
    for b in [b for l in (m.layer1, m.layer2, m.layer3, m.layer4) for b in l]:
        r = y if b.downsample is None else gn(b.downsample[1], F.conv2d(y, b.downsample[0].weight, None, b.stride))
        t = torch.relu(gn(b.bn1, F.conv2d(y, b.conv1.weight, None, b.stride, 1)))
        y = torch.relu(gn(b.bn2, F.conv2d(t, b.conv2.weight, None, 1, 1)) + r)
    want = m.fc(y.mean((2, 3)))
    gw = torch.autograd.grad(want.sum(), [m.conv1.weight, m.layer3[0].bn2.weight])
    got = m(x)
    gg = torch.autograd.grad(got.sum(), [m.conv1.weight, m.layer3[0].bn2.weight])
    torch.testing.assert_close(got, want, rtol=1e-3, atol=1e-4)
    for a, b in zip(gg, gw):
        torch.testing.assert_close(a, b, rtol=1e-2, atol=1e-3 * float(b.abs().max()))


@pytest.mark.parametrize("act,border", [(True, 0.0), (6.0, 0.0), (6.0, 6.0), (0.5, 0.5)])
def test_group_norm_act_no_gradient_on_a_border(act, border):
    """z exactly on a border (gamma 0, beta or the residual the border): no gradient comes through, as in relu and relu6."""
    g = torch.Generator().manual_seed(9)
    x, dy = torch.randn(2, 5, 8, generator=g), torch.randn(2, 5, 8, generator=g)
    for by_beta in (True, False):
        beta, res = (border, 0.0) if by_beta else (0.0, border)
        leaves = [t.requires_grad_(True) for t in (x.clone(), torch.zeros(8), torch.full((8,), beta), torch.full((2, 5, 8), res))]
        out = ops.group_norm_act(leaves[0], 2, leaves[1], leaves[2], leaves[3], act)
        assert torch.equal(out, torch.full_like(out, border))
        assert not any(bool(t.any()) for t in torch.autograd.grad(out, leaves, dy))


def test_convert_group_norm_of_a_module_with_two_names():
    """A BatchNorm that two parents (or one parent twice) hold becomes one GroupNorm everywhere."""
    from pytorch_distributed_amd import nn as pnn
    bn = pnn.BatchNorm2d(8)
    m = torch.nn.Module()
    m.first, m.again, m.inner = bn, bn, torch.nn.Sequential(bn, pnn.BatchNorm2d(8))
    pnn.GroupNorm.convert_group_norm(m, 4)
    assert not any(isinstance(k, pnn.BatchNorm2d) for k in (m.first, m.again, *m.inner))
    assert m.first is m.again is m.inner[0] and m.inner[1] is not m.first
    assert m.first.weight is bn.weight and m.first.num_groups == 4
