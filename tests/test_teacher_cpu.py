"""What a teacher must leave alone in the training of its student."""
import pytest
import torch

from pytorch_distributed_amd import amp, engine, models, utils


def _args(*flags):
    return engine.build_parser().parse_args(["--num-classes", "10", "--teacher", "resnet18", *flags])


@pytest.fixture
def checkpoint(tmp_path):
    """A checkpoint as a run without dynamic loss scaling writes it."""
    torch.manual_seed(5)
    model = models.get_model("resnet18", num_classes=10)
    opt = torch.optim.SGD(model.parameters(), 0.1)
    state = utils.build_state(model, 0, "resnet18", 0.0, opt,
                              {"loss_scaler0": {"loss_scale": 1.0, "unskipped": 7, "skipped_steps": 3, "dynamic": False}})
    path = str(tmp_path / "teacher.pth.tar")
    torch.save(state, path)
    return path, model


def test_loading_a_teacher_leaves_the_loss_scaler(checkpoint):
    path, saved = checkpoint
    student = models.Net()
    opt = torch.optim.SGD(student.parameters(), 0.1)
    try:
        amp.initialize(student, opt, opt_level="O1", dtype=torch.float16, verbosity=0)
        before = amp.state_dict()
        assert before["loss_scaler0"]["dynamic"] and before["loss_scaler0"]["loss_scale"] > 1.0
        teacher = engine.make_teacher(_args("--teacher-checkpoint", path), "cpu")
        assert amp.state_dict() == before
        for a, b in zip(teacher.model.state_dict().values(), saved.state_dict().values()):
            assert torch.equal(a, b)
        # --resume still restores it
        utils.load_checkpoint(path, models.get_model("resnet18", num_classes=10))
        assert not amp.state_dict()["loss_scaler0"]["dynamic"]
    finally:
        amp.initialize(models.Net(), opt_level="O0", verbosity=0)


def test_recorded_steps_of_another_teacher_are_dropped():
    """What a recorded step holds of a teacher as constants is compared with the call's, by value where it may be changed in place."""
    class Opt:
        pass

    def recorded(teacher):
        opt._pda_graph_state = {"graph": Graph(), "eager": 3, "loss": engine._loss_constants(teacher), "metrics": None}
        opt.gone = False

    class Graph:
        def __del__(self):
            opt.gone = True

    def dropped(teacher):
        g = engine._graph_state(opt, teacher, "cpu")
        assert g is opt._pda_graph_state
        assert (g["graph"] is None) == opt.gone == (g["eager"] == 0)
        assert g["loss"] == engine._loss_constants(teacher)
        return opt.gone

    opt = Opt()
    assert engine._graph_state(opt, None, "cpu") is None
    a, b = engine.Teacher(models.Net()), engine.Teacher(models.Net())
    for was, now, drop in [(None, None, False), (a, a, False), (None, a, True), (a, None, True), (a, b, True)]:
        recorded(was)
        assert dropped(now) == drop
        assert not drop or engine._graph_state(opt, now, "cpu")["graph"] is None
    for name, value in [("weight", 0.25), ("k", 8), ("temperature", 1.0), ("model", models.Net())]:
        recorded(a)
        setattr(a, name, value)
        assert dropped(a)
        recorded(a)
        assert not dropped(a)


def test_a_teacher_without_a_checkpoint_is_the_same_everywhere():
    """Every rank builds its own: the weights must not hang on a rank's random state, and that state is left to the student."""
    made = []
    for seed, flags in [(1, ()), (2, ()), (3, ("--seed", "9"))]:
        torch.manual_seed(seed)
        state = torch.get_rng_state()
        made.append(engine.make_teacher(_args(*flags), "cpu").model.state_dict())
        assert torch.equal(torch.get_rng_state(), state)
    same = [all(torch.equal(made[0][k], m[k]) for k in made[0]) for m in made]
    assert same == [True, True, False]
