"""The orthogonalised update of a projection weight: Newton-Schulz steps on its gradient or momentum, as the Muon
optimiser takes them, on this package's tensor-core products (``sru_b200_orthogonalize`` of the C ABI).

The weights of an SRU stack are matrices (``weight``, ``weight_proj``; sru/modules.py:132-146), and layers of equal shape
can be stacked and updated in one call.  CUDA tensors only.
"""
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _lib

_SIXTEEN = (torch.float16, torch.bfloat16)


def orthogonalize(grad: Tensor, steps: int = 5, coefficients: Tuple[float, float, float] = (3.4445, -4.7750, 2.0315),
                  eps: float = 1e-7, out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """``grad`` (rows, cols) or (batch, rows, cols) -> a matrix (or matrices) of the same shape whose singular values are
    near 1 and whose singular vectors are grad's:

        X = grad / (|grad|_F + eps),  ``steps`` times  X <- a X + (b X X^T + c (X X^T)^2) X

    with X transposed where it is taller than wide.  float32, float16 or bfloat16 in; ``out_dtype`` (float16 or
    bfloat16, by default grad's type, bfloat16 for a float32 grad) out.  The iterates are fp16 with float32 accumulation:
    the result is about 1e-3 (relative, Frobenius) off exact steps, before its rounding to ``out_dtype``.  Repeated calls
    give identical bits.  Matrices whose rows or columns are contiguous are read in place.  No gradient flows through it.
    """
    if len(coefficients) != 3:
        raise _lib.SruB200Error("coefficients must be (a, b, c), got %r" % (coefficients,))
    if _lib.timer is None and not _lib.nvtx_ranges:
        try:
            return _lib.native_op("orthogonalize")(grad, steps, *coefficients, eps, out_dtype)
        except RuntimeError as e:
            raise _lib.refused(e) from None
    if not grad.is_cuda:
        raise _lib.SruB200Error("sru_b200 has no CPU path: grad must be a CUDA tensor")
    if grad.dim() not in (2, 3):
        raise _lib.SruB200Error("grad must be (rows, cols) or (batch, rows, cols), got %s" % (tuple(grad.shape),))
    if grad.dtype not in (torch.float32,) + _SIXTEEN:
        raise _lib.SruB200Error("grad must be float32, float16 or bfloat16, got %s" % grad.dtype)
    if out_dtype is None:
        out_dtype = torch.bfloat16 if grad.dtype == torch.float32 else grad.dtype
    if out_dtype not in _SIXTEEN:
        raise _lib.SruB200Error("the result is float16 or bfloat16, got %s" % out_dtype)
    out = torch.empty(grad.shape, dtype=out_dtype, device=grad.device)
    if grad.numel() == 0:
        return out
    if grad.stride(-1) != 1 and grad.stride(-2) != 1:
        grad = grad.contiguous()
    grad = grad.detach()
    batch = grad.size(0) if grad.dim() == 3 else 1
    rows, cols = grad.shape[-2:]
    L = _lib.lib()
    a, b, c = (float(v) for v in coefficients)
    with torch.cuda.device(grad.device):
        nbytes = int(L.sru_b200_orthogonalize_workspace_bytes(batch, rows, cols))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=grad.device)
        _lib.call("orthogonalize", L.sru_b200_orthogonalize, _lib.ptr(out), _lib.ptr(grad), batch, rows, cols,
                  grad.stride(0) if grad.dim() == 3 else 0, grad.stride(-2), grad.stride(-1), int(steps), a, b, c,
                  float(eps), _lib.DTYPE_CODE[grad.dtype], _lib.DTYPE_CODE[out_dtype], _lib.ptr(ws), nbytes,
                  _lib.current_stream_ptr(grad.device))
    return out
