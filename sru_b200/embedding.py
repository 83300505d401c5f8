"""The token table in front of the first layer: scaled lookup and its gradient by sorted tokens.

The reference's language models take ``nn.Embedding`` for this (language_model/train_enwik8.py:56-62 reads its symbols
through one); ``embedding_lookup(tokens, weight, scale)`` multiplies by ``scale`` on the way and can write the
type the first projection consumes, so that neither is a pass of its own
(``sru_b200_embedding_forward`` / ``_backward`` of the C ABI).  CUDA tensors only.
"""
from typing import Optional

import torch
from torch import Tensor
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib

_SIXTEEN = (torch.float16, torch.bfloat16)


def _forward(tokens, weight, scale, out_dtype):
    n, (vocabulary, hidden) = tokens.numel(), weight.shape
    y = torch.empty(n, hidden, dtype=out_dtype, device=weight.device)
    if n:
        with torch.cuda.device(weight.device):
            _lib.call("embedding_fwd", _lib.lib().sru_b200_embedding_forward, _lib.ptr(y), _lib.ptr(tokens),
                      _lib.ptr(weight), n, vocabulary, hidden, weight.stride(0), scale, tokens.element_size(),
                      _lib.DTYPE_CODE[weight.dtype], _lib.DTYPE_CODE[out_dtype], _lib.current_stream_ptr(weight.device))
    return y


class _EmbeddingLookup(Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding_idx, out_dtype):
        ctx.save_for_backward(tokens)
        ctx.meta = (weight.shape, weight.dtype, scale, padding_idx)
        return _forward(tokens, weight.detach(), scale, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (tokens,) = ctx.saved_tensors
        (vocabulary, hidden), dtype, scale, padding_idx = ctx.meta
        dev, n = grad.device, tokens.numel()
        if not grad.is_contiguous():
            grad = grad.contiguous()
        out = torch.empty(vocabulary, hidden, dtype=dtype, device=dev)
        L = _lib.lib()
        nbytes = int(L.sru_b200_embedding_backward_workspace_bytes(n, vocabulary, hidden))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            _lib.call("embedding_bwd", L.sru_b200_embedding_backward, _lib.ptr(out), _lib.ptr(tokens), _lib.ptr(grad),
                      n, vocabulary, hidden, padding_idx, scale, tokens.element_size(), _lib.DTYPE_CODE[dtype],
                      _lib.DTYPE_CODE[grad.dtype], _lib.ptr(ws), nbytes, _lib.current_stream_ptr(dev))
        return None, out, None, None, None


def embedding_lookup(tokens: Tensor, weight: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None,
                     out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """``scale * weight[tokens]``: tokens of any shape (int32 or int64), weight (vocabulary, hidden) with contiguous rows.

    ``out_dtype`` None gives weight's type; a float32 weight may be read into float16 or bfloat16 (one rounding of the
    scaled value).  The gradient is dense, (vocabulary, hidden) in weight's type: each token's rows are summed in
    float32 in the order of their positions, without atomics, so that repeated calls give identical bits.  The row of
    ``padding_idx`` (negative values count from the end, as in ``nn.Embedding``) is read like any other and gets
    no gradient.  A token outside the table gives a row of zeros and no gradient, and raises the device error
    flag: ``_lib.check_device_error()`` then raises.
    """
    if _lib.timer is None and not _lib.nvtx_ranges:
        try:
            return _lib.native_op("embedding_lookup")(tokens, weight, scale, padding_idx, out_dtype)
        except RuntimeError as e:
            raise _lib.refused(e) from None
    if not weight.is_cuda or not tokens.is_cuda:
        raise _lib.SruB200Error("sru_b200 has no CPU path: tokens and weight must be CUDA tensors")
    if tokens.device != weight.device:
        raise _lib.SruB200Error("tokens are on %s, weight on %s" % (tokens.device, weight.device))
    if tokens.dtype not in (torch.int32, torch.int64):
        raise _lib.SruB200Error("tokens must be int32 or int64, got %s" % tokens.dtype)
    if weight.dim() != 2 or weight.size(0) < 1 or weight.size(1) < 1:
        raise _lib.SruB200Error("weight must be (vocabulary, hidden), got %s" % (tuple(weight.shape),))
    if weight.dtype not in (torch.float32,) + _SIXTEEN:
        raise _lib.SruB200Error("weight must be float32, float16 or bfloat16, got %s" % weight.dtype)
    out_dtype = out_dtype or weight.dtype
    if out_dtype != weight.dtype and not (weight.dtype == torch.float32 and out_dtype in _SIXTEEN):
        raise _lib.SruB200Error("a %s table cannot be read into %s" % (weight.dtype, out_dtype))
    vocabulary = weight.size(0)
    if padding_idx is None:
        padding_idx = -1
    else:
        if not -vocabulary <= padding_idx < vocabulary:
            raise _lib.SruB200Error("padding_idx %d is outside a table of %d rows" % (padding_idx, vocabulary))
        padding_idx %= vocabulary
    if weight.stride(1) != 1 or weight.stride(0) < weight.size(1):
        weight = weight.contiguous()
    flat = tokens.detach().reshape(-1)
    flat = flat if flat.is_contiguous() else flat.contiguous()
    if torch.is_grad_enabled() and weight.requires_grad:
        y = _EmbeddingLookup.apply(flat, weight, float(scale), padding_idx, out_dtype)
    else:
        y = _forward(flat, weight.detach(), float(scale), out_dtype)
    return y.view(*tokens.shape, weight.size(1))
