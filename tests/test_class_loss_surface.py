"""CPU-side checks of how the trainer's surface reaches the losses over a set of classes."""
import os
import subprocess
import sys

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
