"""CPU-side checks of how the trainer's surface reaches the losses over a set of classes."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_photometric_path_needs_no_binding_of_the_class_losses():
    """vsl_vocab_binding.so is built for one torch and one Python; without it only its own losses are missing."""
    code = """
import sys, types
sys.modules["mde_amd.vsl_vocab_binding"] = None          # as if it were not there
import torch
import mde_amd.layers, mde_amd.ops, mde_amd.trainer_step
from mde_amd.trainer_loss import ViewSynthesisLoss
vs = ViewSynthesisLoss(types.SimpleNamespace(height=12, width=20))
maps = torch.zeros(1, 4, 12, 20)
for call in (lambda: vs.compute_bin_distillation(maps, maps, k=2),
             lambda: vs.compute_bin_cross_entropy(maps, torch.zeros(3, 4), torch.zeros(1, 12, 20, dtype=torch.int64))):
    try:
        call()
    except ImportError as e:
        assert "vsl_vocab_binding" in str(e)
    else:
        raise AssertionError("ran without its binding")
print("fine")
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip().endswith("fine"), done.stderr[-2000:]


@pytest.mark.parametrize("shape", [(1, 6, 3, 5), (1, 4, 3, 4), (2, 4, 3, 5), (4, 3, 5)])
def test_bins_of_student_and_teacher_have_to_be_the_same(shape):
    """A teacher of more bins would make its pixels NaN, one of fewer would be matched bin by bin with other depths."""
    import types

    import torch
    from mde_amd.trainer_loss import ViewSynthesisLoss
    vs = ViewSynthesisLoss(types.SimpleNamespace(height=3, width=5))
    with pytest.raises(ValueError, match="same bins"):
        vs.compute_bin_distillation(torch.zeros(1, 4, 3, 5), torch.zeros(shape), k=2)
    with pytest.raises(ValueError, match="GPU"):
        vs.compute_bin_distillation(torch.zeros(1, 4, 3, 5), torch.zeros(1, 4, 3, 5), k=2)
