"""The gated linear recurrence: SRU's state update (``c_t = f_t c_{t-1} + (1 - f_t) x_t``, sru/modules.py:283-318,
sru/csrc/sru_cuda_kernel.cu:60-78) with a forget gate ``f_t = sigmoid(g_t + bias)`` that does not look at the state
(``weight_c = 0``, the reference's ``v1`` gates).  A linear recurrence can be scanned in parallel along time, so that a
few long sequences use the whole GPU; the SRU scan of ``ops`` walks time step by step.

``gated_linear_recurrence(u, c0, bias, mask_pad, reverse)`` takes the projection's output with the gate index innermost,
as the SRU's U has it (k = 2: candidate, forget gate), and has its own backward pass
(``sru_b200_linear_recurrence_forward`` / ``_backward`` of the C ABI).  CUDA tensors only.
"""
from typing import Optional, Tuple

from torch import Tensor

from . import _lib


def gated_linear_recurrence(u: Tensor, c0: Optional[Tensor] = None, bias: Optional[Tensor] = None,
                            mask_pad: Optional[Tensor] = None, reverse: bool = False) -> Tuple[Tensor, Tensor]:
    """The recurrence over u (length, batch, 2 * hidden), or (batch, 2 * hidden) for a single step.

    u[..., 2j] is column j's candidate x and u[..., 2j + 1] its forget logit g (float32, float16 or bfloat16):

        f_t = sigmoid(g_t + bias),  c_t = f_t c_{t-1} + (1 - f_t) x_t,  h_t = c_t

    ``c0`` (batch, hidden) is the state before the first step (zeros when None), ``bias`` (hidden,) is added to the
    logits.  Where ``mask_pad`` (length, batch) is non-zero the position is padding: the state passes through, h and all
    gradients are 0 there, and what u holds there is not looked at.  ``reverse`` runs time from the last step to the
    first.  Returns ``h`` (length, batch, hidden) in u's type and the state after the last step (batch, hidden), always in
    float32: a sequence processed in chunks, the state handed on, loses nothing to the storage type.  Strided u with
    contiguous pairs (a batch-first tensor transposed, for instance) is read in place.  Differentiable once in u, c0 and
    bias, in reverse mode; a tensor that carries a forward-mode tangent is refused.
    """
    return _lib.call_native("gated_linear_recurrence", "linear_recurrence_fwd", "linear_recurrence_bwd", u, c0, bias, mask_pad, reverse)
