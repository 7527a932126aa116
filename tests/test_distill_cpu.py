"""A teacher's top logits and the distillation loss on them, on the CPU: values, gradients, refusals."""
import math

import pytest
import torch
import torch.nn.functional as F

from pytorch_distributed_amd import ops, nn as pnn, models


def test_top_logits_order():
    z = torch.tensor([[0.0, 3.0, -0.0, 3.0, float("-inf"), 1.0], [float("nan"), 5.0, float("inf"), 5.0, float("nan"), -1.0]])
    v, i, r = ops.top_logits(z, 4)
    assert i.tolist() == [[1, 3, 5, 0], [0, 4, 2, 1]]
    assert v[0].tolist() == [3.0, 3.0, 1.0, 0.0] and math.isnan(v[1, 0]) and v[1, 2:].tolist() == [float("inf"), 5.0]
    assert abs(float(r[0]) - 0.0) < 1e-6 and abs(float(r[1]) - math.log(math.exp(5) + math.exp(-1))) < 1e-5
    v, i, r = ops.top_logits(z[0], 6, 2.0)
    assert v.shape == (6,) and r.shape == () and float(r) == -math.inf


def test_top_logits_refusals():
    z = torch.randn(2, 5)
    for kw in (dict(k=0), dict(k=6), dict(k=2, temperature=0.0), dict(k=2, temperature=float("nan")),
               dict(k=2, temperature=float("inf")), dict(k=2, temperature=1e-9)):
        with pytest.raises(ValueError):
            ops.top_logits(z, **kw)
    with pytest.raises(TypeError):
        ops.top_logits(z, 2.5)
    with pytest.raises(TypeError):
        ops.top_logits(z.double(), 2)
    with pytest.raises(TypeError):
        ops.top_logits(z.long(), 2)
    with pytest.raises(ValueError):
        ops.top_logits(torch.empty(2, 0), 1)
    with pytest.raises(ValueError):
        ops.top_logits(torch.empty(1, (1 << 20) + 1), 1)
    with pytest.raises(ValueError):
        ops.top_logits(torch.empty(1, 4096), 1025)


@pytest.mark.parametrize("t", [1.0, 3.0])
def test_distill_loss_is_the_divergence_of_all_classes(t):
    """With every class an entry both forms are the divergence of the two softmaxes."""
    g = torch.Generator().manual_seed(1)
    z, teacher = torch.randn(6, 9, generator=g, requires_grad=True), torch.randn(6, 9, generator=g)
    v, i, r = ops.top_logits(teacher, 9, t)
    want = F.kl_div(F.log_softmax(z.double() / t, 1), F.softmax(teacher.double() / t, 1), reduction="none").sum(1) * t * t
    gw, = torch.autograd.grad(want.mean(), z)
    want = want.detach()
    for rest in (None, r):
        loss = ops.distill_loss(z, v, i, rest, t)
        assert abs(float(loss.detach()) - float(want.mean())) < 1e-6
        gz, = torch.autograd.grad(loss, z)
        assert float((gz - gw).abs().max()) < 1e-7


def _by_hand(z, v, i, rest, t):
    """One row, python numbers."""
    V = len(z)
    entries = [(a / t, c) for a, c in zip(v, i) if 0 <= c < V]
    if not entries or (all(a == -math.inf for a, _ in entries) and (rest is None or rest == -math.inf)):
        return 0.0
    total = sum(math.exp(a) for a, _ in entries) + (math.exp(rest) if rest is not None else 0.0)
    p = {}
    for a, c in entries:
        p[c] = p.get(c, 0.0) + math.exp(a) / total
    zs = sum(math.exp(a / t) for a in z)
    loss = sum(w * (math.log(w) - (z[c] / t - math.log(zs))) for c, w in p.items() if w > 0)
    if rest is not None and rest != -math.inf:
        pr = math.exp(rest) / total
        loss += pr * (math.log(pr) - math.log(sum(math.exp(z[c] / t) for c in range(V) if c not in p) / zs))
    return loss * t * t


@pytest.mark.parametrize("with_rest", [False, True])
def test_distill_loss_rows(with_rest):
    g = torch.Generator().manual_seed(2)
    inf = math.inf
    z = torch.randn(7, 6, generator=g)
    v = torch.randn(7, 3, generator=g)
    i = torch.tensor([[0, 1, 2], [-1, 4, 6], [3, 3, 5], [-1, -1, 9], [2, 0, 5], [1, 1, 1], [0, 2, 4]])
    v[1, 0], v[3] = float("nan"), float("nan")     # not looked at
    v[4] = torch.tensor([-inf, 1.0, 2.0])
    v[6] = -inf
    rest = torch.randn(7, generator=g) if with_rest else None
    if with_rest:
        rest[6] = -inf
    t = 2.0
    loss = ops.distill_loss(z, v, i, rest, t, "none")
    for k in range(7):
        want = _by_hand(z[k].tolist(), v[k].tolist(), i[k].tolist(), None if rest is None else float(rest[k]), t)
        assert abs(float(loss[k]) - want) < 1e-6 * (1 + abs(want)), k
    assert abs(float(ops.distill_loss(z, v, i, rest, t, "sum")) - float(loss.sum())) < 1e-5
    assert abs(float(ops.distill_loss(z, v, i.int(), rest, t)) - float(loss.mean())) < 1e-6
    # rows without entries: any logits, no gradient
    z[3], z[6] = float("nan"), inf
    zl = z.requires_grad_(True)
    loss = ops.distill_loss(zl, v, i, rest, t, "none")
    gz, = torch.autograd.grad(loss.sum(), zl)
    assert float(loss[3]) == 0 and float(loss[6]) == 0 and not bool(gz[3].any()) and not bool(gz[6].any())
    assert bool(torch.isfinite(gz).all())
    # differences, step h: h^2 times a third derivative below 1, and fp32's rounding of the loss
    h = 2.0 ** -6
    for k, c in [(0, 0), (0, 5), (1, 4), (2, 3), (4, 2), (5, 1), (5, 0)]:
        a, b = z.detach().clone(), z.detach().clone()
        a[k, c] += h
        b[k, c] -= h
        num = (ops.distill_loss(a, v, i, rest, t, "none")[k].double() - ops.distill_loss(b, v, i, rest, t, "none")[k].double()) / (2 * h)
        assert abs(float(num) - float(gz[k, c])) < h * h + 2.0 ** -24 * 8 / h


def closed_rows():
    """Rows whose student leaves nothing to the classes that are not entries while the teacher's rest has a share: the loss is inf, the
    gradient T (q - p) at the entries and zero elsewhere."""
    inf = math.inf
    z = torch.tensor([[1.0, 2.0, -inf, -inf], [0.5, -inf, 3.0, -inf], [0.3, -1.0, 2.0, 0.7], [0.1, 0.2, 0.3, 0.4]])
    v = torch.tensor([[0.2, 0.4, 0.0, 0.0], [1.0, 0.1, 0.3, 0.0], [0.1, 0.2, 0.3, 0.4], [0.1, 0.2, 0.3, 0.0]])
    i = torch.tensor([[0, 1, -1, -1], [0, 1, 2, -1], [0, 1, 2, 3], [0, 1, 2, -1]])
    rest = torch.tensor([0.5, -0.5, 0.25, 0.1])
    t = 2.0
    q = torch.softmax(z.double() / t, 1)
    tau = torch.where(i < 0, -inf, v.double() / t)
    p = torch.softmax(torch.cat([tau, rest.double()[:, None]], 1), 1)
    grad = torch.where(i < 0, 0.0, t * (q - p[:, :4]))   # entry k is class k in every row
    grad[3, 3] = t * (q[3, 3] - p[3, 4])                 # the last row is an open one
    return z, v, i, rest, t, grad


def test_distill_loss_nothing_left_outside_the_entries():
    z, v, i, rest, t, grad = closed_rows()
    z.requires_grad_(True)
    loss = ops.distill_loss(z, v, i, rest, t, "none")
    assert bool((loss[:3] == math.inf).all()) and bool(torch.isfinite(loss[3]))
    got, = torch.autograd.grad(loss, z, torch.ones(4))
    assert float((got.double() - grad).abs().max()) <= 2.0 ** -22


def test_distill_loss_refusals():
    z, v, i, r = torch.randn(4, 7), torch.randn(4, 2), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4)
    ops.distill_loss(z, v, i, r)
    bad = [(z, v[:3], i, r), (z, v, i[:, :1], r), (z, v, i, r[:3]), (z, v, i, r[:, None]), (z[None], v, i, r),
           (z, v[:, :0], i[:, :0], r), (z, v.expand(4, 2).repeat(1, 600), i.repeat(1, 600), r), (z, v, i, r.long())]
    for a in bad:
        with pytest.raises(ValueError):
            ops.distill_loss(*a)
    for a in [(z.double(), v, i, r), (z, v.double(), i, r), (z, v, i.short(), r), (z, v, i.float(), r)]:
        with pytest.raises(TypeError):
            ops.distill_loss(*a)
    for kw in (dict(temperature=0.0), dict(temperature=-1.0), dict(reduction="batchmean")):
        with pytest.raises(ValueError):
            ops.distill_loss(z, v, i, r, **kw)


def test_distill_loss_no_rows_and_leading_dimensions():
    z = torch.randn(2, 3, 9, requires_grad=True)
    v, i, r = ops.top_logits(z.detach() * 2, 4, 2.0)
    assert v.shape == (2, 3, 4) and r.shape == (2, 3)
    loss = ops.distill_loss(z, v, i, r, 2.0, "none")
    assert loss.shape == (2, 3)
    flat = ops.distill_loss(z.reshape(6, 9), v.reshape(6, 4), i.reshape(6, 4), r.reshape(6), 2.0, "none")
    assert torch.equal(loss.reshape(-1), flat)
    e = ops.distill_loss(torch.empty(0, 9), torch.empty(0, 4), torch.empty(0, 4, dtype=torch.int64), None, 1.0, "sum")
    assert float(e) == 0.0


def test_distillation_module_and_teacher():
    from pytorch_distributed_amd import engine
    torch.manual_seed(0)
    teacher_model, student = models.Net(), models.Net()
    teacher = engine.Teacher(teacher_model, k=4, temperature=2.0, weight=0.25)
    assert not teacher.model.training and not any(p.requires_grad for p in teacher.model.parameters())
    x = torch.randn(3, 1, 28, 28)
    student.eval()
    out = student(x)
    label = F.cross_entropy(out.float(), torch.tensor([1, 2, 3]))
    loss = teacher.loss(x, out, label)
    with torch.no_grad():
        v, i, r = ops.top_logits(teacher_model(x), 4, 2.0)
    want = 0.75 * label + 0.25 * pnn.DistillationLoss(2.0)(out, v, i, r)
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-6
    loss.backward()
    assert all(p.grad is None for p in teacher_model.parameters()) and any(bool(p.grad.any()) for p in student.parameters())
    with pytest.raises(ValueError):
        engine.Teacher(teacher_model, weight=1.5)


def test_group_norm_student_of_a_teacher_trains():
    """The operators together: a group norm student's gradients through the distillation loss, against differences."""
    torch.manual_seed(3)
    conv = pnn.Conv2d(3, 16, 3, 1, 1)
    gn = pnn.GroupNorm(4, 16)
    fc = pnn.Linear(16, 12)
    x, teacher_logits = torch.randn(2, 6, 6, 3), torch.randn(2, 12) * 3
    v, i, r = ops.top_logits(teacher_logits, 5, 2.0)

    def loss():
        return ops.distill_loss(fc(gn(conv(x), None, "silu").mean((1, 2))), v, i, r, 2.0)

    params = [gn.weight, gn.bias, fc.weight]
    grads = torch.autograd.grad(loss(), params)
    h = 2.0 ** -6
    for p, g in zip(params, grads):
        for k in (0, p.numel() - 1):
            with torch.no_grad():
                p.view(-1)[k] += h
                hi = float(loss())
                p.view(-1)[k] -= 2 * h
                lo = float(loss())
                p.view(-1)[k] += h
            # h^2 times a third derivative below 4, and the rounding of fp32 losses below 4
            assert abs((hi - lo) / (2 * h) - float(g.reshape(-1)[k])) < 4 * h * h + 2.0 ** -24 * 4 * 16 / h
