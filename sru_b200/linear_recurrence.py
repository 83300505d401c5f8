"""The gated linear recurrence: SRU's state update (``c_t = f_t c_{t-1} + (1 - f_t) x_t``, sru/modules.py:283-318,
sru/csrc/sru_cuda_kernel.cu:60-78) with a forget gate ``f_t = sigmoid(g_t + bias)`` that does not look at the state
(``weight_c = 0``, the reference's ``v1`` gates).  A linear recurrence can be scanned in parallel along time, so that a
few long sequences use the whole GPU; the SRU scan of ``ops`` walks time step by step.

``gated_linear_recurrence(u, c0, bias, mask_pad, reverse)`` takes the projection's output with the gate index innermost,
as the SRU's U has it (k = 2: candidate, forget gate), and has its own backward pass
(``sru_b200_linear_recurrence_forward`` / ``_backward`` of the C ABI).  CUDA tensors only.
"""
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib

_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _rows(t: Tensor, unit: int) -> Tensor:
    """t (L, B, n) as the kernels read it: unit stride in the last dimension and every group of ``unit`` elements
    aligned to its size; other layouts are copied."""
    if t.stride(2) == 1 and t.data_ptr() % (unit * t.element_size()) == 0 and t.stride(0) % unit == 0 and t.stride(1) % unit == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _small(t: Optional[Tensor]) -> Optional[Tensor]:
    return None if t is None else t.detach().float().contiguous()


def _forward(u, c0, bias, mask, reverse, need_states):
    """u (L, B, 2d) -> h (L, B, d) in u's type, c_last (B, d) float32, states (or None)."""
    length, batch, d = u.size(0), u.size(1), u.size(2) // 2
    h = torch.empty(length, batch, d, dtype=u.dtype, device=u.device)
    c_last = torch.empty(batch, d, dtype=torch.float32, device=u.device)
    if length == 0 or batch == 0:
        return h, (c_last.copy_(c0) if c0 is not None else c_last.zero_()), None
    L = _lib.lib()
    states = None
    if need_states:
        nbytes = int(L.sru_b200_linear_recurrence_states_bytes(length, batch, d))
        states = torch.empty(nbytes // 4, dtype=torch.float32, device=u.device)
    with torch.cuda.device(u.device):
        _lib.call("linear_recurrence_fwd", L.sru_b200_linear_recurrence_forward,
                  _lib.ptr(h), _lib.ptr(c_last), _lib.ptr(states), _lib.ptr(u), _lib.ptr(bias), _lib.ptr(c0), _lib.ptr(mask),
                  length, batch, d, u.stride(0), u.stride(1), int(reverse), _lib.DTYPE_CODE[u.dtype],
                  _lib.current_stream_ptr(u.device))
    return h, c_last, states


class _GatedLinearRecurrence(Function):
    @staticmethod
    def forward(ctx, u, c0, bias, mask, reverse):
        ctx.set_materialize_grads(False)
        rows = _rows(u.detach(), 2)
        b = _small(bias)
        h, c_last, states = _forward(rows, _small(c0), b, mask, reverse, any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(rows, b, mask, states)
        ctx.reverse = reverse
        ctx.types = (None if c0 is None else c0.dtype, None if bias is None else bias.dtype)
        return h, c_last

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_h, grad_last):
        u, bias, mask, states = ctx.saved_tensors
        length, batch, d = u.size(0), u.size(1), u.size(2) // 2
        c0_dtype, bias_dtype = ctx.types
        dev = u.device
        need_bias = bias is not None and ctx.needs_input_grad[2]
        need_first = c0_dtype is not None and ctx.needs_input_grad[1]
        grad_u = torch.empty(length, batch, 2 * d, dtype=u.dtype, device=dev)
        grad_bias = torch.empty(d, dtype=torch.float32, device=dev) if need_bias else None
        grad_first = torch.empty(batch, d, dtype=torch.float32, device=dev) if need_first else None
        gl = None if grad_last is None else grad_last.float().contiguous()
        if length == 0 or batch == 0:
            if need_bias:
                grad_bias.zero_()
            if need_first:
                grad_first.zero_() if gl is None else grad_first.copy_(gl)
        else:
            gh = None if grad_h is None else _rows(grad_h.to(u.dtype), 1)
            L = _lib.lib()
            with torch.cuda.device(dev):
                nbytes = int(L.sru_b200_linear_recurrence_backward_workspace_bytes(length, batch, d, _lib.DTYPE_CODE[u.dtype])) if need_bias else 0
                ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
                _lib.call("linear_recurrence_bwd", L.sru_b200_linear_recurrence_backward,
                          _lib.ptr(grad_u), _lib.ptr(grad_bias), _lib.ptr(grad_first), _lib.ptr(u), _lib.ptr(bias),
                          _lib.ptr(states), _lib.ptr(mask), _lib.ptr(gh), _lib.ptr(gl), length, batch, d, u.stride(0),
                          u.stride(1), 0 if gh is None else gh.stride(0), 0 if gh is None else gh.stride(1),
                          int(ctx.reverse), _lib.DTYPE_CODE[u.dtype], _lib.ptr(ws), nbytes, _lib.current_stream_ptr(dev))
        return (grad_u if ctx.needs_input_grad[0] else None, grad_first.to(c0_dtype) if need_first else None,
                grad_bias.to(bias_dtype) if need_bias else None, None, None)


def _check(u: Tensor, t: Tensor, name: str, shape: tuple) -> None:
    if t.device != u.device:
        raise _lib.SruB200Error("%s is on %s, u on %s" % (name, t.device, u.device))
    if t.shape != shape:
        raise _lib.SruB200Error("%s must have shape %s, got %s" % (name, shape, tuple(t.shape)))
    if name != "mask_pad" and not t.is_floating_point():
        raise _lib.SruB200Error("%s must be a floating-point tensor, got %s" % (name, t.dtype))


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
    bias.
    """
    if _lib.timer is None and not _lib.nvtx_ranges:
        try:
            return _lib.native_op("gated_linear_recurrence")(u, c0, bias, mask_pad, reverse)
        except RuntimeError as e:
            raise _lib.refused(e) from None
    if not u.is_cuda:
        raise _lib.SruB200Error("sru_b200 has no CPU path: u must be a CUDA tensor")
    if u.dtype not in _TYPES:
        raise _lib.SruB200Error("gated_linear_recurrence takes float32, float16 or bfloat16, got %s" % u.dtype)
    if u.dim() not in (2, 3) or u.shape[-1] < 2 or u.shape[-1] % 2:
        raise _lib.SruB200Error("u must be (length, batch, 2 * hidden) or (batch, 2 * hidden), got %s" % (tuple(u.shape),))
    single = u.dim() == 2
    if single:
        u = u.unsqueeze(0)
        mask_pad = None if mask_pad is None else mask_pad.unsqueeze(0)
    length, batch, width = u.shape
    if c0 is not None:
        _check(u, c0, "c0", (batch, width // 2))
    if bias is not None:
        _check(u, bias, "bias", (width // 2,))
    if mask_pad is not None:
        _check(u, mask_pad, "mask_pad", (length, batch))
    mask = None if mask_pad is None else mask_pad.bool().contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (u, c0, bias)):
        h, c_last = _GatedLinearRecurrence.apply(u, c0, bias, mask, bool(reverse))
    else:
        h, c_last, _ = _forward(_rows(u.detach(), 2), _small(c0), _small(bias), mask, reverse, False)
    return (h.squeeze(0) if single else h), c_last
