"""The orthogonalised update of a projection weight: Newton-Schulz steps on its gradient or momentum, as the Muon
optimiser takes them, on this package's tensor-core products (``sru_b200_orthogonalize`` of the C ABI).

The weights of an SRU stack are matrices (``weight``, ``weight_proj``; sru/modules.py:132-146), and layers of equal shape
can be stacked and updated in one call.  CUDA tensors only.
"""
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _lib


def orthogonalize(grad: Tensor, steps: int = 5, coefficients: Tuple[float, float, float] = (3.4445, -4.7750, 2.0315),
                  eps: float = 1e-7, out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """``grad`` (rows, cols) or (batch, rows, cols) -> a matrix (or matrices) of the same shape whose singular values are
    near 1 and whose singular vectors are grad's:

        X = grad / (|grad|_F + eps),  ``steps`` times  X <- a X + (b X X^T + c (X X^T)^2) X

    with X transposed where it is taller than wide.  float32, float16 or bfloat16 in; ``out_dtype`` (float16 or
    bfloat16, by default grad's type, bfloat16 for a float32 grad) out.  Repeated calls
    give identical bits.  Matrices whose rows or columns are contiguous are read in place.  No derivative flows
    through it, in either mode: the result is a constant to autograd.

    Accuracy (relative, Frobenius, default steps and coefficients).  The norm is summed in 64 bits and products in float32;
    the iterates have the bits that the result needs.  For a float16 result they are pairs of fp16 (22 bits): the result
    is the exact steps rounded once, 2.1e-4 off, 3e-4 at most (and 1e-8 more per column of the longer side,
    for the tensor cores' float32 sums), at 1.5 to 4 times the time of a bfloat16 one.  For a bfloat16
    result they have eleven bits (fp16, scaled clear of its subnormals), and what that costs depends on grad, because the steps
    multiply its smallest singular values, and the rounding of its largest elements with them, by up to a^steps (485): before the
    rounding to bfloat16 (1.7e-3) below 2e-3 for gradients that are mostly noise (with sixteen strong directions as well), 6e-3 for
    singular values that fall off as 1 / i, 3e-2 as 1 / i^2, 6e-2 for four strong directions over noise of a hundredth of their
    size (7e-4 as float16).  Storing such a grad as bfloat16 costs at least four times as much in the last three cases.
    """
    if len(coefficients) != 3:
        raise _lib.SruB200Error("coefficients must be (a, b, c), got %r" % (coefficients,))
    return _lib.call_native("orthogonalize", "orthogonalize", None, grad, steps, *coefficients, eps, out_dtype)
