"""Group norm students of a teacher on the GPU: the converted models against the same parameters on the CPU, and a whole
step of both operators recorded and replayed."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

from pytorch_distributed_amd import engine, models, nn as pnn, ops, utils

DEV = "cuda"


@pytest.mark.parametrize("arch,groups", [("resnet18", 32), ("densenet121", 16), ("shufflenet_v2_x1_0", 8), ("mobilenet_v2", 8)])
def test_converted_model_matches_the_cpu(arch, groups):
    """fp32 on both sides: the bound is that of fp32 convolutions through the depth of the networks."""
    torch.manual_seed(0)
    cpu = pnn.GroupNorm.convert_group_norm(models.get_model(arch, num_classes=9), groups)
    for m in cpu.modules():
        if isinstance(m, pnn.Dropout):
            m.p = 0.0
    gpu = copy.deepcopy(cpu).to(DEV)
    x, t = torch.randn(4, 3, 64, 64), torch.randint(0, 9, (4,))
    out, ref = gpu(x.to(DEV)), cpu(x)
    torch.testing.assert_close(out.cpu(), ref, rtol=2e-3, atol=2e-3 * float(ref.detach().abs().max()))
    v, i, r = ops.top_logits(torch.randn(4, 9) * 2, 4, 2.0)
    (ops.cross_entropy(ref, t) + ops.distill_loss(ref, v, i, r, 2.0)).backward()
    (ops.cross_entropy(out, t.to(DEV)) + ops.distill_loss(out, v.to(DEV), i.to(DEV), r.to(DEV), 2.0)).backward()
    for (n, a), (_, b) in zip(gpu.named_parameters(), cpu.named_parameters()):
        err = float((a.grad.cpu() - b.grad).norm() / (b.grad.norm() + 1e-6))
        assert err < 2e-2, (n, err)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_student_and_teacher_step_recorded(dtype):
    torch.manual_seed(1)
    student = pnn.GroupNorm.convert_group_norm(models.resnet18(num_classes=40), 32).set_compute_dtype(dtype).to(DEV)
    teacher = engine.Teacher(models.resnet18(num_classes=40).set_compute_dtype(dtype).to(DEV), k=8, temperature=2.0, weight=0.5)
    x, t = torch.randn(8, 3, 64, 64, device=DEV), torch.randint(0, 40, (8,), device=DEV)
    params = list(student.parameters())

    def step():
        out = student(x)
        loss = teacher.loss(x, out, ops.cross_entropy(out, t))
        return (loss.detach(),) + torch.autograd.grad(loss, params)

    step()
    graphed = utils.GraphedStep(step, warmup=2)
    assert graphed.captured
    for k in range(3):
        x.copy_(torch.randn(8, 3, 64, 64, device=DEV))
        got = [g.clone() for g in graphed()]
        torch.cuda.synchronize()
        want = step()
        assert abs(float(got[0]) - float(want[0])) <= 1e-3 * (1 + abs(float(want[0])))
        for p, a, b in zip(params, got[1:], want[1:]):
            # weight gradients of the convolutions are summed in an order that varies
            assert float((a - b).norm()) <= 2e-2 * float(b.norm()) + 1e-5, p.shape


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("given", [torch.uint8, torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("norm", [False, True])
def test_group_norm_stem_input(dtype, given, norm, monkeypatch):
    """The stem's input in one pass, and with a gradient to the images by single steps (bf16 images likewise).  An element may differ by
    two roundings to fp32 and then by one step of the type, d; a sum of 147 of them is some 12 times its own spread, so the
    normalised output by 12 d and the sums' own 147 roundings."""
    torch.manual_seed(3)
    m = pnn.GroupNorm.convert_group_norm(models.resnet18(), 32).to(DEV).set_compute_dtype(dtype)
    if norm:
        m.set_input_normalization([0.4, 0.5, 0.6], [0.2, 0.3, 0.25], 1 / 255.0)
    x = torch.randint(0, 256, (3, 3, 40, 38), device=DEV).to(given)
    single = []
    monkeypatch.setattr(pnn, "to_nhwc", lambda t, f=pnn.to_nhwc: (single.append(t), f(t))[1])
    got = m._stem(x)
    assert bool(single) == (given is torch.bfloat16)
    xl = x.float().requires_grad_(True)
    want = m._stem(xl)
    assert torch.autograd.grad(want.float().square().sum(), xl)[0].abs().sum() > 0
    d = max(torch.finfo(dtype).eps, 2.0 ** -22)
    assert float((got - want).float().norm()) <= (12 * d + 147 * 2.0 ** -24) * float(want.float().norm())
