"""The example scripts with group norm and a teacher, on the CPU backends (tiny settings)."""
import os
import sys

import pytest

from test_examples_cpu import COMMON, EX, LAUNCH, free_port, run


def test_dataparallel_with_group_norm_and_teacher(tmp_path):
    out = run([sys.executable, os.path.join(EX, "1_dataparallel.py")] + COMMON +
              ["--group-norm", "16", "--teacher", "resnet18", "--distill-top", "4", "--distill-temperature", "2"], tmp_path)
    assert " * Acc@1" in out


def test_ddp_with_group_norm_and_teacher_of_a_checkpoint(tmp_path):
    run([sys.executable, os.path.join(EX, "1_dataparallel.py")] + COMMON, tmp_path)
    out = run(LAUNCH + ["--nproc_per_node=2", "--master_port", str(free_port()), os.path.join(EX, "2_distributed.py")] + COMMON +
              ["--group-norm", "8", "--teacher", "resnet18", "--teacher-checkpoint",
               str(tmp_path / "resnet18.checkpoint.pth.tar"), "--distill-weight", "1.0"], tmp_path)
    assert out.count(" * Acc@1") == 1


@pytest.mark.parametrize("flags", [["--distill-weight", "1.5", "--teacher", "resnet18"], ["--teacher", "no_such_arch"],
                                   ["--group-norm", "-4"]])
def test_refused_flags(tmp_path, flags):
    with pytest.raises(AssertionError):
        run([sys.executable, os.path.join(EX, "1_dataparallel.py")] + COMMON + flags, tmp_path)
