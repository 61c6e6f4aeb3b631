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


@pytest.mark.parametrize("rows,vocab,dim,kind", [(8192, 131072, 4096, 1), (8192, 131072, 4096, 0), (65536, 8192, 512, 1),
                                                 (16384, 50021, 768, 0), (32768, 32000, 1024, 2)])
def test_workspaces_stay_below_the_logits_of_large_problems(rows, vocab, dim, kind):
    """What the linear cross entropy is there to spare: rows * vocab float32."""
    import ctypes

    import mde_amd._abi as abi
    d = abi.LinearCeDesc(rows=rows, vocab=vocab, dim=dim, hidden_stride=dim, weight_stride=dim, ignore_index=-100, type=kind,
                         reduction=abi.REDUCE_MEAN, z_loss=0.0, hidden=1 << 20, weight=1 << 20, target=1 << 20)
    logits = rows * vocab * 4
    assert abi.lib.vsl_linear_ce_fwd_workspace_bytes(ctypes.byref(d)) < logits / 3
    assert abi.lib.vsl_linear_ce_bwd_workspace_bytes(ctypes.byref(d), 7) < logits * 0.7


def test_derivatives_of_few_classes_are_padded_to_a_tile():
    """92160 pixels, 128 depth bins, 256 features in bfloat16: hidden transposed (47 MB), the derivatives twice (24 MB each)."""
    import ctypes

    import mde_amd._abi as abi
    d = abi.LinearCeDesc(rows=92160, vocab=128, dim=256, hidden_stride=256, weight_stride=256, ignore_index=-100, type=1,
                         reduction=abi.REDUCE_MEAN, z_loss=0.0, hidden=1 << 20, weight=1 << 20, target=1 << 20, bias=1 << 20)
    need = 92160 * 256 * 2 + 2 * 92160 * 128 * 2
    assert need <= abi.lib.vsl_linear_ce_bwd_workspace_bytes(ctypes.byref(d), 7) < 1.25 * need
