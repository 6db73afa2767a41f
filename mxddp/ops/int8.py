"""Linear layers in 8-bit integers (``csrc/int8_linear.hip``), beside ``ops.linear``.

A token (row of x) has one scale, its largest magnitude / 127, and so has each output channel of the
weight; the product runs on int8 matrix instructions with an exact int32 sum, and the epilogue
applies both scales, the bias and a ReLU.  Inference only: there is no gradient.
"""
from __future__ import annotations

import torch

from .. import native
from . import _native, _p
from .lowp import DTYPES, MAX_ROWS, check_device, check_float, has_derivative, on_device, rows_of, stream

MAX_K = 2**17 - 1  # products of 2^14 each whose sum stays below 2^31
MAX_LENGTH = 2**30   # csrc/ops.h kMaxLength: of a row that is quantised, and channels of a layer
_TINY = 2.0**-126
_MAX_LD = 2**22      # csrc/ops.h kInt8MaxLd


def quantize_rows(x: torch.Tensor):
    """``(q, scale)`` with x ~ q * scale[..., None]: int8 rows and one fp32 scale a row.

    ``scale = max|x| / 127`` (at least 2^-126) and ``q = x / scale`` rounded half to even, exactly.
    A row with an infinity or a NaN has a NaN scale and q = 0.  ``x``: [..., K], float32, bfloat16
    or float16, at most 8388607 rows, K at most 2^30.  Weights [out, in] give the per-channel scales that
    ``linear_int8`` takes.  The results carry no derivative, as those of ``detach``."""
    check_float(x, "quantize_rows: x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_LENGTH:
        raise ValueError(f"quantize_rows: x must be [..., K] with 1 <= K <= 2^30, got {tuple(x.shape)}")
    x = x.detach()
    if not _native(x):
        xd = x.double()
        top = xd.abs().amax(-1)
        ok = torch.isfinite(top)
        scale = torch.where(ok, (top / 127).float().clamp_min(_TINY), torch.full_like(top, float("nan")).float())
        q = torch.where(ok[..., None], (xd / scale.double()[..., None]).round(), torch.zeros_like(xd))
        return q.to(torch.int8), scale
    K = x.shape[-1]
    q = torch.empty(x.shape, device=x.device, dtype=torch.int8)
    scale = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
    x2 = rows_of(x)
    if x2.shape[0] > MAX_ROWS:
        raise ValueError(f"quantize_rows: {x2.shape[0]} rows, at most {MAX_ROWS}")
    with on_device(x2):
        native().quantize_rows(x2.data_ptr(), DTYPES[x2.dtype], x2.stride(0), q.data_ptr(), K, scale.data_ptr(),
                               x2.shape[0], K, stream(x2))
    return q, scale


def _row_stride(t):
    """Of a [rows, K] tensor; a single row has none that matters, whatever it was cut from: whole pieces."""
    return t.stride(0) if t.shape[0] > 1 else (t.shape[1] + 15) // 16 * 16


def _room(w, K):
    """Bytes that may be read of each of w's rows: whole 16-byte pieces where its memory goes on."""
    pieces = (K + 15) // 16 * 16
    if pieces == K:
        return K
    last = w.storage_offset() + (w.shape[0] - 1) * w.stride(0)
    return pieces if last + pieces <= w.untyped_storage().nbytes() else K


def linear_int8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None = None,
                relu: bool = False, x_scale: torch.Tensor | None = None, out_dtype: torch.dtype | None = None):
    """``relu?((q @ weight.T) * s[..., None] * weight_scale + bias)`` for (q, s) = quantize_rows(x).

    ``weight``: int8 [N, K], contiguous rows of any stride; ``weight_scale``: float32 [N];
    ``bias``: float32 [N].  ``x``: [..., K] in float32, bfloat16 or float16, or int8 with its
    ``x_scale`` [...] (``quantize_rows``: one quantised input for several layers).  The result has
    ``out_dtype`` (default: x's type, float32 for an int8 x).  K is at most 131071, and x has at most
    8388607 rows.  N is at most 2^30; on the GPU a layer of more than 134217712 channels (2^27 - 16) may
    be refused.  No gradient: an input that requires one is refused while autograd records, and one with
    a forward-mode tangent always.

    Rows of whole 16-byte pieces (K a multiple of 16, or a weight with padded rows as ``Int8Linear``
    keeps it) take the faster way into the large tiles."""
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_int8: x {tuple(x.shape)} does not fit weight {tuple(weight.shape)}")
    N, K = weight.shape
    if weight.dtype != torch.int8:
        raise TypeError(f"linear_int8: weight must be int8, got {weight.dtype}")
    if not 1 <= K <= MAX_K or not 1 <= N <= MAX_LENGTH:
        raise ValueError(f"linear_int8: weight {tuple(weight.shape)}: 1 <= K <= {MAX_K} and 1 <= N <= 2^30")
    given = x.dtype == torch.int8
    if given:
        if x_scale is None or x_scale.dtype != torch.float32 or x_scale.shape != x.shape[:-1]:
            raise ValueError("linear_int8: an int8 x needs its float32 x_scale, one a row")
    else:
        check_float(x, "linear_int8: x")
        if x_scale is not None:
            raise ValueError("linear_int8: x_scale goes with an int8 x")
    if has_derivative(x, weight_scale, bias, x_scale):
        raise RuntimeError("linear_int8 has no gradient: call it under torch.no_grad() or detach its inputs "
                           "(detach those with a forward-mode tangent)")
    out_dtype = out_dtype or (torch.float32 if given else x.dtype)
    if out_dtype not in DTYPES:
        raise TypeError(f"linear_int8: out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    for t, name in ((weight_scale, "weight_scale"), (bias, "bias")):
        if t is not None and (t.dtype != torch.float32 or t.shape != (N,)):
            raise ValueError(f"linear_int8: {name} must be float32 [{N}], got {t.dtype} {tuple(t.shape)}")
        check_device(t, x, name)
    check_device(weight, x, "weight")
    check_device(x_scale, x, "x_scale")
    if not _native(x):
        q, s = (x, x_scale) if given else quantize_rows(x)
        y = (q.double() @ weight.double().t()) * s.double()[..., None] * weight_scale.detach().double()
        if bias is not None:
            y = y + bias.detach().double()
        return (y.clamp_min(0) if relu else y).to(out_dtype)
    x2 = rows_of(x.detach())
    M = x2.shape[0]
    if M > MAX_ROWS:
        raise ValueError(f"linear_int8: {M} rows, at most {MAX_ROWS}")
    if (weight.stride(1) != 1 and K > 1) or _row_stride(weight) > _MAX_LD:
        weight = weight.contiguous()
    weight_scale = weight_scale.contiguous()
    bias = None if bias is None else bias.contiguous()
    y = torch.empty((*x.shape[:-1], N), device=x.device, dtype=out_dtype)
    C, xt, yt = native(), DTYPES.get(x2.dtype, -1), DTYPES[out_dtype]
    wargs = (weight.data_ptr(), _row_stride(weight), _room(weight, K), weight_scale.data_ptr(), _p(bias), y.data_ptr(), yt,
             M, N, K, bool(relu))
    with on_device(x2):
        if given:
            x2 = x2 if _row_stride(x2) <= _MAX_LD else x2.contiguous()
            C.linear_int8(x2.data_ptr(), _row_stride(x2), K, x_scale.contiguous().data_ptr(), *wargs, stream(x2))
        else:
            n = C.linear_int8_scratch(xt, yt, M, K)
            scratch = torch.empty((n,), device=x2.device, dtype=torch.int8) if n else None
            C.linear_int8_float(x2.data_ptr(), xt, x2.stride(0), *wargs, _p(scratch), stream(x2))
    return y
