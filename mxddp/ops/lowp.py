"""What the operators for fp32, bf16 and fp16 tensors share: their types, rows and checks."""
from __future__ import annotations

import contextlib

import torch
import torch.autograd.forward_ad as forward_ad

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # csrc/lowp.h DType
MAX_ROWS = 2**23 - 1  # csrc/ops.h kMaxRows


def check_float(t: torch.Tensor, name: str, cpu_double: bool = False) -> None:
    if t.dtype not in DTYPES and not (cpu_double and t.dtype == torch.float64 and not t.is_cuda):
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")


def check_device(t: torch.Tensor | None, x: torch.Tensor, name: str) -> None:
    if t is not None and t.device != x.device:
        raise ValueError(f"{name} is on {t.device}, the input on {x.device}")


def has_derivative(*tensors: torch.Tensor | None) -> bool:
    """Whether autograd would carry a derivative through any of these: backward while it records, or a
    forward-mode tangent (which torch.no_grad does not turn off)."""
    backward, forward = torch.is_grad_enabled(), forward_ad._current_level >= 0
    if backward or forward:
        for t in tensors:
            if t is not None and (backward and t.requires_grad
                                  or forward and forward_ad.unpack_dual(t).tangent is not None):
                return True
    return False


def rows_of(t: torch.Tensor) -> torch.Tensor:
    """``t`` as [rows, last] with contiguous rows (any row stride), copied only where it must be."""
    n = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(t.numel() // n if n else 0, n)
    return t if t.stride(1) == 1 or n == 1 else t.contiguous()


def stream(t: torch.Tensor) -> int:
    """The current stream's handle, without the Stream object that ``ops.stream_of`` makes (1.8 us)."""
    return torch._C._cuda_getCurrentRawStream(t.device.index)


_HERE = contextlib.nullcontext()


def on_device(t: torch.Tensor):
    """Launches go to the current device: make it the tensor's."""
    if t.device.index == torch.cuda.current_device():
        return _HERE
    return torch.cuda.device(t.device)
