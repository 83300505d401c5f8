"""The token table in front of the first layer: scaled lookup and its gradient by sorted tokens.

The reference's language models take ``nn.Embedding`` for this (language_model/train_enwik8.py:56-62 reads its symbols
through one); ``embedding_lookup(tokens, weight, scale)`` multiplies by ``scale`` on the way and can write the
type the first projection consumes, so that neither is a pass of its own
(``sru_b200_embedding_forward`` / ``_backward`` of the C ABI).  CUDA tensors only.
"""
from typing import Optional

import torch
from torch import Tensor

from . import _lib


def embedding_lookup(tokens: Tensor, weight: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None,
                     out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """``scale * weight[tokens]``: tokens of any shape (int32 or int64), weight (vocabulary, hidden) with contiguous rows.

    ``out_dtype`` None gives weight's type; a float32 weight may be read into float16 or bfloat16 (one rounding of the
    scaled value).  The gradient is dense, (vocabulary, hidden) in weight's type: each token's rows are summed in
    float32 in the order of their positions, without atomics, so that repeated calls give identical bits.  The row of
    ``padding_idx`` (negative values count from the end, as in ``nn.Embedding``) is read like any other and gets
    no gradient.  A token outside the table gives a row of zeros and no gradient, and raises the device error
    flag: ``_lib.check_device_error()`` then raises.  Differentiable once, in reverse mode; a table that carries a
    forward-mode tangent is refused.
    """
    return _lib.call_native("embedding_lookup", "embedding_fwd", "embedding_bwd", tokens, weight, scale, padding_idx, out_dtype)
