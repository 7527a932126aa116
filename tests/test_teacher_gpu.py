"""A student's recorded training steps under changing teachers."""
import copy
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu

from pytorch_distributed_amd import engine, models, nn as pnn, ops
from pytorch_distributed_amd.optim import FusedSGD

DEV = torch.device("cuda")


def test_recorded_steps_follow_the_teacher():
    """engine.train with --graph, one call after another on one optimizer: the gradients that the last step leaves are those of
    the call's own loss.  The learning rate is 0; weight gradients are summed in an order that varies (fp32, 1e-3)."""
    torch.manual_seed(0)
    student = models.resnet18(num_classes=10).to(DEV)
    twin = copy.deepcopy(student)
    opt = FusedSGD(student.parameters(), lr=0.0)
    x, t = torch.randn(8, 3, 64, 64), torch.randint(0, 10, (8,))
    args = SimpleNamespace(graph=True, steps_per_epoch=0, print_freq=100)
    a, b = (engine.Teacher(models.resnet18(num_classes=10).to(DEV), k=4, temperature=2.0, weight=w) for w in (0.5, 0.9))

    def want(teacher):
        out = twin(x.to(DEV))
        loss = ops.cross_entropy(out, t.to(DEV))
        if teacher is not None:
            loss = teacher.loss(x.to(DEV), out, loss)
        return [g.clone() for g in torch.autograd.grad(loss, list(twin.parameters()))]

    def check(teacher):
        expected = want(teacher)
        engine.train([(x, t)] * 6, student, pnn.CrossEntropyLoss(), opt, 0, DEV, args, teacher=teacher)
        torch.cuda.synchronize()
        graph = opt._pda_graph_state["graph"]
        assert graph is not None and graph.captured
        for p, g in zip(student.parameters(), expected):
            assert float((p.grad - g).norm()) <= 1e-3 * float(g.norm()) + 1e-6
        return graph

    first = check(None)
    assert check(None) is first     # the same loss: the same recording
    del first
    check(a)
    a.weight = 1.0
    check(a)
    check(b)
    check(None)
