"""Argument checks and launches shared by the embedding and budget calls."""
from __future__ import annotations

import torch

from ._capi import INVALID_ARGUMENT, NOT_SUPPORTED, OUT_OF_RANGE, GsxError, check

FLOAT_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
INDEX_TYPES = {torch.int32: 12, torch.int64: 13}


def invalid(message: str):
    return GsxError(INVALID_ARGUMENT, message)


def type_code(t, types: dict, name: str) -> int:
    code = types.get(t.dtype)
    if code is None:
        raise GsxError(NOT_SUPPORTED, f"{name} must be one of {[str(k)[6:] for k in types]}, not {t.dtype}")
    return code


def on_device(device, *tensors):
    """Every tensor (None allowed) lives on the CUDA device `device`."""
    if device.type != "cuda":
        raise invalid("tensors must be on a CUDA device")
    for t in tensors:
        if t is not None and t.device != device:
            raise invalid(f"all tensors must be on {device}, one is on {t.device}")


def row_stride(t, dim: int, name: str) -> int:
    """Elements between the rows of t (.., dim), whose rows are contiguous and evenly spaced."""
    if t.is_contiguous():
        return dim
    if t.dim() == 2 and (t.stride(1) == 1 or dim == 1) and (t.stride(0) >= dim or t.shape[0] <= 1):
        return max(t.stride(0), dim)
    raise invalid(f"{name} must be contiguous, or 2-D with contiguous rows that do not overlap")


def group_stride(t, lead: int, name: str) -> int:
    """Elements between the groups that t's first `lead` dimensions number (row-major), evenly spaced."""
    step = None
    for d in range(lead - 1, -1, -1):
        if t.shape[d] == 1:
            continue
        if step is None:
            step, size = t.stride(d), t.shape[d]
        elif t.stride(d) != step * size:
            raise invalid(f"the leading dimensions of {name} must be evenly strided")
        else:
            size *= t.shape[d]
    return step or 0


def word(t, name: str):
    """Pointer of a one-element 32-bit flag tensor (None allowed)."""
    if t is None:
        return None
    if t.numel() != 1 or t.element_size() != 4:
        raise invalid(f"{name} must hold one 32-bit word")
    return t.data_ptr()


def below_2_31(*numbers):
    for v in numbers:
        if not 0 <= v < 2147483648:
            raise GsxError(OUT_OF_RANGE, f"counts and sizes must be in [0, 2^31), not {v}")


def empty(shape, dtype, device, stream):
    """A tensor whose memory belongs to `stream` (None: the device's current one)."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def launch(fn, device, stream, *args):
    """fn(*args, stream handle) with `device` current."""
    if stream is None:
        handle = torch._C._cuda_getCurrentRawStream(device.index)
    elif stream.device != device:
        raise invalid(f"stream must be on {device}, not {stream.device}")
    else:
        handle = stream.cuda_stream
    if torch._C._cuda_getDevice() == device.index:
        rc = fn(*args, handle)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, handle)
    if rc:
        check(rc)
