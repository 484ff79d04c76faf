from __future__ import annotations

import torch

from . import _lib

_DT = {torch.float16: _lib.ESP_DTYPE_F16, torch.bfloat16: _lib.ESP_DTYPE_BF16, torch.float32: _lib.ESP_DTYPE_F32}


def dtype_tag(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}") from None


def dtype16_tag(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return _lib.ESP_DTYPE_BF16
    if t.dtype == torch.float16:
        return _lib.ESP_DTYPE_F16
    raise TypeError(f"expected float16 or bfloat16, not {t.dtype}")


def ptr(t):
    return 0 if t is None else t.data_ptr()


def stream_ptr() -> int:
    return torch.cuda.current_stream().cuda_stream


# torch's own accessors behind current_device() / current_stream(), without the Stream object that the latter builds (3 us per
# call, as much as the launch it is for)
_get_device = getattr(torch._C, "_cuda_getDevice", None)
_get_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def current_device() -> int:
    return _get_device() if _get_device is not None else torch.cuda.current_device()


def stream_of(device: int) -> int:
    """The current stream of a device, as the C ABI takes it."""
    return _get_stream(device) if _get_stream is not None else torch.cuda.current_stream(device).cuda_stream


def need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("the ESP attention ops run on CUDA tensors only (there is no CPU path)")


def need_here(first, *ts) -> int:
    """The device of the tensors (None is skipped, the first is a tensor), which must be the CURRENT CUDA device: the kernels are
    launched there, on its current stream."""
    d = first.get_device()
    if d < 0:
        raise RuntimeError("the ESP attention ops run on CUDA tensors only (there is no CPU path)")
    if d != current_device():
        raise RuntimeError(f"tensor on cuda:{d}, but the current CUDA device is cuda:{current_device()}: select the tensors' device first")
    for t in ts:
        if t is not None and t.get_device() != d:
            if t.get_device() < 0:
                raise RuntimeError("the ESP attention ops run on CUDA tensors only (there is no CPU path)")
            raise RuntimeError(f"tensor on cuda:{t.get_device()}, but the current CUDA device is cuda:{d}: all tensors of a call lie there")
    return d


_CODES = {torch.int8: _lib.ESP_CODE_INT8, torch.float8_e4m3fn: _lib.ESP_CODE_E4M3}


def code_tag(t: torch.Tensor) -> int:
    try:
        return _CODES[t.dtype]
    except KeyError:
        raise TypeError(f"8-bit rows are torch.int8 or torch.float8_e4m3fn, not {t.dtype}") from None


def need_i32(*ts):
    for t in ts:
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise TypeError("metadata vectors must be contiguous int32")


def idx64_flag(t: torch.Tensor) -> int:
    if t.dtype == torch.int64:
        return 1
    if t.dtype == torch.int32:
        return 0
    raise TypeError("index tensors must be int32 or int64")
