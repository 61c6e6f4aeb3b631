"""Losses over a set of classes -- the tokens of a vocabulary, or the depth bins of a pixel -- on the HIP library:

    top_logits(logits, k, temperature)                       what a teacher hands on: its k largest logits of every row
    topk_distillation_loss(logits, values, indices, lse)     a student against them, with the gradient of its logits
    linear_cross_entropy(hidden, weight, target, bias)       cross entropy of a linear head in pieces of the vocabulary,
                                                             logits never kept, with the gradients of hidden, weight, bias

The last dimension is the classes (the features, for ``hidden`` and ``weight``); all others are rows, so a decoder's
[B, C, H, W] maps go in as ``maps.movedim(1, -1)``, which costs no copy in channels-last memory.  Tensors are float32,
bfloat16 or float16 (float64 is cast to float32 on load, as everywhere in this package); rows may be strided, everything
else is made contiguous.  Losses and statistics are float32, gradients have their tensor's type.

A logit of -infinity is a masked class.  A row in which nothing is left adds nothing and gets a zero gradient; NaN or
+infinity in a row, and a target or index outside the vocabulary, make that row's results NaN.  ``"mean"`` over no rows is
0.  Derivatives are first ones and backward ones; forward mode is refused.  Results are deterministic.  No host synchronisation: every call can be captured into a graph, its backward pass too
once no earlier result of the same leaves is alive (torch ends the process otherwise).

The functions are those of ``include/vsloss_vocab_torch.h``, where their arguments are checked, behind a small extension
module.  Calls of a few rows are bound by the host: an autograd node that runs without the interpreter takes a training
step of 200 rows x 1000 classes x 256 features from 128 to 77 us, a distillation step of 300 x 1000 from 102 to 59 us, the
top logits of 300 x 1000 from 16 to 8 us.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _abi

ctypes.CDLL(_abi.LIB_PATH, mode=ctypes.RTLD_GLOBAL)   # the binding finds the library's functions there
try:
    from . import vsl_vocab_binding as _binding
except ImportError as e:
    raise ImportError("vsl_vocab_binding.so is not built for this torch: run `python -c 'import __graft_entry__ as g; "
                      "g.build()'` -- there is no fallback implementation (%s)" % e) from e
_binding.errors_from(_abi.__name__)


class TopLogits(NamedTuple):
    values: torch.Tensor    # [..., k], the logits' type, larger first
    indices: torch.Tensor   # [..., k], int32
    lse: torch.Tensor       # [...], float32: log sum exp(logits / temperature) over the whole vocabulary


# ------------------------------------------------------------------ top logits
def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    """The ``k`` largest logits of every row, larger first, ties to the lower index, NaN above +infinity, and the log of
    the row's whole sum of exp(logits / temperature); 1 <= k <= min(classes, 256).  One pass over the logits; carries no
    gradient."""
    return TopLogits(*_binding.top_logits(logits, int(k), float(temperature)))


# ------------------------------------------------------------------ distillation
def topk_distillation_loss(logits: torch.Tensor, teacher_values: torch.Tensor, teacher_indices: torch.Tensor,
                           teacher_lse: Optional[torch.Tensor] = None, *, temperature: float = 1.0,
                           weights: Optional[torch.Tensor] = None, reduction: str = "mean") -> torch.Tensor:
    """temperature^2 * KL(teacher || student) from the teacher's top logits (``top_logits``), with the gradient of
    ``logits`` [..., classes].

    ``teacher_values`` / ``teacher_indices`` [..., k] (int32 or int64).  Without ``teacher_lse`` the teacher is the softmax
    of its k values / temperature.  With it ([...], the log of its whole sum at this temperature) the k classes keep their
    probabilities and what is left is one further class, against which the student puts the sum of its other
    probabilities; it is left out of a row where the student has no other class.  ``weights`` [...]: a row of weight 0 is
    not looked at; ``"mean"`` divides by their sum.  The teacher's tensors and the weights carry no gradient."""
    return _binding.topk_distillation_loss(logits, teacher_values, teacher_indices, teacher_lse, float(temperature), weights,
                                           reduction)


# ------------------------------------------------------------------ linear cross entropy
def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                         bias: Optional[torch.Tensor] = None, *, ignore_index: int = -100, z_loss: float = 0.0,
                         reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of ``hidden @ weight.T + bias`` against ``target``, plus ``z_loss`` times the square of every
    row's log sum, without keeping the logits: the forward pass reduces them tile by tile on the matrix cores, the
    backward pass makes them again in pieces of the vocabulary.

    ``hidden`` [..., dim], ``weight`` [classes, dim] and ``bias`` [classes] share one type; ``target`` [...] holds classes
    or ``ignore_index`` (such a row is left out of the mean and gets a zero gradient).  A class whose bias is -infinity is
    masked out.  Gradients reach ``hidden``, ``weight`` and ``bias``; in 16-bit types the derivative of a logit is rounded
    to that type before the two gradient products, which sum in float32."""
    return _binding.linear_cross_entropy(hidden, weight, target, bias, int(ignore_index), float(z_loss), reduction)
