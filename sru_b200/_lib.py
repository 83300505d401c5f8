"""ctypes access to libsru_b200.so (the C ABI of include/sru_b200.h).

There is no fallback: if the library is missing or fails to load, every operator raises.
"""
import ctypes
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libsru_b200.so")
TORCH_LIB_PATH = os.path.join(_HERE, "lib", "libsru_b200_torch.so")

SRU_F32, SRU_F16, SRU_BF16, SRU_F64 = 0, 1, 2, 3
DTYPE_CODE = {torch.float32: SRU_F32, torch.float16: SRU_F16, torch.bfloat16: SRU_BF16,
              torch.float64: SRU_F64}

_lib = None
_torch_ops_loaded = False

_vp = ctypes.c_void_p
_i64 = ctypes.c_int64
_int = ctypes.c_int


class SruB200Error(RuntimeError):
    pass


def lib():
    """The loaded C-ABI library.  Raises if it has not been built (python -m sru_b200.build)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise SruB200Error(
                "libsru_b200.so not found at %s: build it with `python -m sru_b200.build`; "
                "this package has no CPU or PyTorch fallback" % LIB_PATH)
        l = ctypes.CDLL(LIB_PATH)
        l.sru_b200_version.restype = _int
        l.sru_b200_last_error.restype = ctypes.c_char_p
        l.sru_b200_check_device_error.restype = _int
        l.sru_b200_check_device_error.argtypes = [_vp]
        l.sru_b200_set_option.restype = _int
        l.sru_b200_set_option.argtypes = [ctypes.c_char_p, _int]
        l.sru_b200_get_option.restype = _int
        l.sru_b200_get_option.argtypes = [ctypes.c_char_p]
        l.sru_b200_last_scan_kernel.restype = _int
        l.sru_b200_last_scan_kernel.argtypes = []
        l.sru_b200_launch_count.restype = _i64
        l.sru_b200_launch_count.argtypes = []
        l.sru_b200_scan_forward.restype = _int
        l.sru_b200_scan_forward.argtypes = [_vp] * 10 + [_i64, _i64, _i64, _int, _int, _int, _int, _int,
                                                         ctypes.c_double, _int, _int, _vp]
        l.sru_b200_scan_backward_workspace_bytes.restype = ctypes.c_size_t
        l.sru_b200_scan_backward_workspace_bytes.argtypes = [_i64, _i64, _i64, _int, _int, _int]
        l.sru_b200_scan_backward.restype = _int
        l.sru_b200_scan_backward.argtypes = [_vp] * 15 + [_i64, _i64, _i64, _int, _int, _int, _int, _int,
                                                          ctypes.c_double, _int, _int, _vp, ctypes.c_size_t, _vp]
        l.sru_b200_gemm.restype = _int
        l.sru_b200_gemm.argtypes = [_vp] * 4 + [_i64] * 6 + [_int] * 5 + [_vp]
        l.sru_b200_gate_bias_columns.restype = _int
        l.sru_b200_gate_bias_columns.argtypes = [_vp, _vp, _i64, _int, _vp]
        l.sru_b200_convert.restype = _int
        l.sru_b200_convert.argtypes = [_vp, _vp, _i64, _int, _int, _vp]
        l.sru_b200_gemm_workspace_bytes.restype = ctypes.c_size_t
        l.sru_b200_gemm_workspace_bytes.argtypes = [_i64, _i64, _i64, _int]
        l.sru_b200_gemm_ws.restype = _int
        l.sru_b200_gemm_ws.argtypes = [_vp] * 4 + [_i64] * 6 + [_int] * 5 + [_vp, ctypes.c_size_t, _vp]
        l.sru_b200_gemm_f32_workspace_bytes.restype = ctypes.c_size_t
        l.sru_b200_gemm_f32_workspace_bytes.argtypes = [_i64, _i64, _i64]
        l.sru_b200_gemm_f32.restype = _int
        l.sru_b200_gemm_f32.argtypes = [_vp] * 4 + [_i64] * 6 + [_int] * 3 + [_vp, ctypes.c_size_t, _vp]
        l.sru_b200_layer_norm_forward.restype = _int
        l.sru_b200_layer_norm_forward.argtypes = [_vp] * 6 + [_i64, _i64, ctypes.c_double, _int, _int, _vp]
        l.sru_b200_layer_norm_backward_workspace_bytes.restype = ctypes.c_size_t
        l.sru_b200_layer_norm_backward_workspace_bytes.argtypes = [_i64, _i64]
        l.sru_b200_layer_norm_backward.restype = _int
        l.sru_b200_layer_norm_backward.argtypes = [_vp] * 8 + [_i64, _i64, _int, _int, _vp, ctypes.c_size_t, _vp]
        l.sru_b200_linear_recurrence_states_bytes.restype = ctypes.c_size_t
        l.sru_b200_linear_recurrence_states_bytes.argtypes = [_i64] * 3
        l.sru_b200_linear_recurrence_forward.restype = _int
        l.sru_b200_linear_recurrence_forward.argtypes = [_vp] * 7 + [_i64] * 5 + [_int] * 2 + [_vp]
        l.sru_b200_linear_recurrence_backward_workspace_bytes.restype = ctypes.c_size_t
        l.sru_b200_linear_recurrence_backward_workspace_bytes.argtypes = [_i64] * 3 + [_int]
        l.sru_b200_linear_recurrence_backward.restype = _int
        l.sru_b200_linear_recurrence_backward.argtypes = [_vp] * 9 + [_i64] * 7 + [_int] * 2 + [_vp, ctypes.c_size_t, _vp]
        l.sru_b200_embedding_forward.restype = _int
        l.sru_b200_embedding_forward.argtypes = [_vp] * 3 + [_i64] * 4 + [ctypes.c_double] + [_int] * 3 + [_vp]
        l.sru_b200_embedding_backward_workspace_bytes.restype = ctypes.c_size_t
        l.sru_b200_embedding_backward_workspace_bytes.argtypes = [_i64] * 3
        l.sru_b200_embedding_backward.restype = _int
        l.sru_b200_embedding_backward.argtypes = [_vp] * 3 + [_i64] * 4 + [ctypes.c_double] + [_int] * 3 + [_vp, ctypes.c_size_t, _vp]
        l.sru_b200_orthogonalize_workspace_bytes.restype = ctypes.c_size_t
        l.sru_b200_orthogonalize_workspace_bytes.argtypes = [_i64] * 3
        l.sru_b200_orthogonalize_workspace_bytes_for.restype = ctypes.c_size_t
        l.sru_b200_orthogonalize_workspace_bytes_for.argtypes = [_i64] * 3 + [_int]
        l.sru_b200_orthogonalize.restype = _int
        l.sru_b200_orthogonalize.argtypes = ([_vp] * 2 + [_i64] * 6 + [_int] + [ctypes.c_double] * 4 + [_int] * 2
                                             + [_vp, ctypes.c_size_t, _vp])
        _lib = l
    return _lib


def load_torch_ops():
    """Registers torch.ops.sru_cuda.* (the reference's operator names) from the binding library."""
    global _torch_ops_loaded
    if not _torch_ops_loaded:
        if not os.path.exists(TORCH_LIB_PATH):
            raise SruB200Error("libsru_b200_torch.so not found at %s: run `python -m sru_b200.build`"
                               % TORCH_LIB_PATH)
        lib()
        torch.ops.load_library(TORCH_LIB_PATH)
        _torch_ops_loaded = True


def native_op(name):
    """``torch.ops.sru_b200.<name>``, whose refusals arrive as RuntimeError."""
    op = _native_ops.get(name)
    if op is None:
        load_torch_ops()
        op = _native_ops[name] = getattr(torch.ops.sru_b200, name).default
    return op


def call_native(op, name, backward_name, *args):
    """A native torch operator with autograd of its own.  With a timer or NVTX ranges installed its launches are bracketed
    like those of ``call``: the forward pass here, the backward pass by hooks on the operator's node of the graph."""
    fn = _native_ops.get(op) or native_op(op)
    try:
        if (timer is None and not nvtx_ranges) or not getattr(args[0], "is_cuda", False):
            return fn(*args)
        with torch.cuda.device(args[0].device):
            out = _watched(name, fn, *args)
    except RuntimeError as e:
        raise refused(e) from None
    if backward_name is not None:
        _watch_backward(backward_name, out)
    return out


def refused(error):
    """A refusal by a native operator as this package's error; anything else (out of memory, for instance) as it is."""
    return SruB200Error(str(error)) if type(error) is RuntimeError else error


_native_ops = {}

SCAN_KERNEL_NAMES = {0: "none", 1: "pipelined", 2: "generic", 3: "split"}


def set_option(name: str, value: int) -> None:
    """Sets a tuning option of the native library (see include/sru_b200.h); negative un-sets it."""
    check(lib().sru_b200_set_option(name.encode(), int(value)))


def get_option(name: str) -> int:
    return int(lib().sru_b200_get_option(name.encode()))


class options:
    """Context manager: ``with options(fwd_v=2, scan_stages=3): ...`` sets, then restores."""

    def __init__(self, **kw):
        self.kw = {k: v for k, v in kw.items() if v is not None}

    def __enter__(self):
        self.old = {k: get_option(k) for k in self.kw}
        for k, v in self.kw.items():
            set_option(k, v)
        return self

    def __exit__(self, *exc):
        for k, v in self.old.items():
            set_option(k, v)


def last_scan_kernel() -> str:
    """'pipelined', 'generic', 'split' or 'none': what this thread's last scan call launched."""
    return SCAN_KERNEL_NAMES.get(int(lib().sru_b200_last_scan_kernel()), "unknown")


def check(rc):
    if rc != 0:
        msg = lib().sru_b200_last_error().decode("utf-8", "replace")
        raise SruB200Error("sru_b200 call failed (%d): %s" % (rc, msg))


def ptr(t):
    return None if t is None else t.data_ptr()


def current_stream_ptr(device=None):
    return torch.cuda.current_stream(device).cuda_stream


def check_device_error(device=None):
    check(lib().sru_b200_check_device_error(current_stream_ptr(device)))


class KernelTimer:
    """Optional per-call timing with CUDA events on the launching stream (used by bench.py).

    Install with ``_lib.timer = KernelTimer()``; every C-ABI launch made through ``call`` is then
    bracketed by a pair of events recorded on the current stream.  ``summary()`` synchronises
    and returns ``{name: (calls, total_ms)}``.
    """

    def __init__(self):
        self.spans = {}

    def add(self, name, start, end):
        self.spans.setdefault(name, []).append((start, end))

    def summary(self):
        torch.cuda.synchronize()
        return {k: (len(v), sum(s.elapsed_time(e) for s, e in v)) for k, v in self.spans.items()}


timer = None          # a KernelTimer, or None
nvtx_ranges = os.environ.get("SRU_B200_NVTX", "0") not in ("", "0")   # see set_nvtx_ranges


def set_nvtx_ranges(enabled: bool) -> None:
    """Brackets every C-ABI launch with an NVTX range named after its kernel class ("scan_fwd", "gemm_wgrad", ...),
    so that a profiler can filter or group by it (for instance ``ncu --nvtx --nvtx-include "scan_bwd/"``).
    Off by default; also switched on by the environment variable SRU_B200_NVTX=1."""
    global nvtx_ranges
    nvtx_ranges = bool(enabled)


def __getattr__(name):
    """``launch_count``: kernels of this library launched so far, whoever called for them (bench.py reports the per-step
    figure); counted in the native library, where the launches are."""
    if name == "launch_count":
        return int(lib().sru_b200_launch_count())
    raise AttributeError("module %r has no attribute %r" % (__name__, name))


def call(name, fn, *args):
    """Invoke a C-ABI entry point, time it if a timer is installed."""
    return check(_watched(name, fn, *args))


def _watched(name, fn, *args):
    """fn(*args), in an NVTX range and between a pair of events where those are asked for."""
    ranged = nvtx_ranges
    if ranged:
        torch.cuda.nvtx.range_push(name)
    try:
        if timer is None:
            return fn(*args)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        out = fn(*args)
        end.record()
        timer.add(name, start, end)
        return out
    finally:
        if ranged:
            torch.cuda.nvtx.range_pop()


def _watch_backward(name, out):
    """The same around the backward pass of the operator that made ``out`` (a tensor or a tuple of them): its node is the
    first one of C++ behind the views."""
    node = (out if isinstance(out, torch.Tensor) else out[0]).grad_fn
    while node is not None and "CppNode" not in node.name():
        node = node.next_functions[0][0] if node.next_functions else None
    if node is None:
        return
    spans = []      # open ranges, innermost last: a node runs once per backward pass

    def before(grads):
        if nvtx_ranges:
            torch.cuda.nvtx.range_push(name)
        start = None
        if timer is not None:
            start = torch.cuda.Event(enable_timing=True)
            start.record()
        spans.append((start, nvtx_ranges))

    def after(grads_in, grads_out):
        start, ranged = spans.pop()
        if start is not None and timer is not None:
            end = torch.cuda.Event(enable_timing=True)
            end.record()
            timer.add(name, start, end)
        if ranged:
            torch.cuda.nvtx.range_pop()
    node.register_prehook(before)
    node.register_hook(after)
