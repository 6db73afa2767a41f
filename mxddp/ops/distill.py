"""Learning from a teacher's top logits (``csrc/distill.hip``), beside ``ops.cross_entropy``.

``top_logits`` keeps what a teacher's answer needs: its k largest logits, their classes, and the
logarithm of the whole sum of exponentials.  ``distill_loss`` is the student's loss against them,
with the labels' cross-entropy mixed in where it is asked for; its forward reads the logits once (twice
above a temperature of 8, where it adds up in 64 bits), its backward reads them once more and writes
their gradient.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .. import native
from . import _native, _p
from .lowp import DTYPES, MAX_ROWS, check_device, check_float, has_derivative, on_device, rows_of, stream

MAX_TOP = 256       # csrc/ops.h kTopMax
MAX_CLASSES = 2**30
_STATS = 12         # csrc/ops.h kDistillStats


class TopLogits(NamedTuple):
    values: torch.Tensor  # [..., k] in falling order, the logits' type
    index: torch.Tensor   # [..., k] int32 classes
    lse: torch.Tensor     # [...] float32: log sum exp(logits / temperature)


def _check_temperature(t) -> float:
    t = float(t)
    if not 1e-30 <= t <= 1e30:  # within them log2(e) / t is a normal fp32 number
        raise ValueError(f"temperature must be a positive number (1e-30 .. 1e30), got {t}")
    return t


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    """The k largest logits of each row, in falling order, equal ones by their class.

    ``logits``: [..., V] float32, bfloat16 or float16, at most 8388607 rows and 2^30 classes;
    1 <= k <= min(V, 256).  A NaN counts as the
    largest value.  ``lse`` is taken at ``temperature`` over all classes (infinite or NaN where the
    largest logit is).  The results carry no derivative, as those of ``detach``."""
    check_float(logits, "top_logits: logits")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_CLASSES:
        raise ValueError(f"top_logits: logits must be [..., V] with 1 <= V <= 2^30, got {tuple(logits.shape)}")
    V = logits.shape[-1]
    if not 1 <= k <= min(V, MAX_TOP):
        raise ValueError(f"top_logits: k must be within 1 .. {min(V, MAX_TOP)}, got {k}")
    temperature = _check_temperature(temperature)
    logits = logits.detach()
    if not _native(logits):
        values, index = torch.sort(logits, dim=-1, descending=True, stable=True)
        lse = torch.logsumexp(logits.double() / temperature, -1).float()
        return TopLogits(values[..., :k].contiguous(), index[..., :k].to(torch.int32), lse)
    z = rows_of(logits)
    rows = z.shape[0]
    if rows > MAX_ROWS:
        raise ValueError(f"top_logits: {rows} rows, at most {MAX_ROWS}")
    lead = logits.shape[:-1]
    values = torch.empty((*lead, k), device=z.device, dtype=z.dtype)
    index = torch.empty((*lead, k), device=z.device, dtype=torch.int32)
    lse = torch.empty(lead, device=z.device, dtype=torch.float32)
    with on_device(z):
        C = native()
        n = C.top_logits_scratch(rows, V, k)
        scratch = torch.empty((n,), device=z.device, dtype=torch.int64) if n else None
        C.top_logits(z.data_ptr(), DTYPES[z.dtype], z.stride(0), rows, V, k, temperature, values.data_ptr(),
                     index.data_ptr(), lse.data_ptr(), _p(scratch), stream(z))
    return TopLogits(values, index, lse)


def _args(z, tv, ti, target, tlse, stats, temperature, hard):
    return (z.data_ptr(), tv.data_ptr(), ti.data_ptr(), _p(target), _p(tlse), stats.data_ptr(), z.stride(0),
            z.shape[0], z.shape[1], tv.shape[1], DTYPES[z.dtype], DTYPES[tv.dtype], ti.dtype == torch.int64,
            target is not None and target.dtype == torch.int64, temperature, hard)


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, tv, ti, target, tlse, temperature, hard, reduction):
        C, (rows, V) = native(), z.shape
        # the rows' statistics and weight for the backward, then what is used up here: the rows'
        # losses (the result itself without a reduction) and the sums of a split row
        n = _STATS * rows + 1
        spare = (n + rows + 1) // 2 * 2  # 64-bit sums
        buf = torch.empty((spare + C.distill_scratch(rows, V),), device=z.device, dtype=torch.float32)
        loss = torch.empty(() if reduction != "none" else (rows,), device=z.device, dtype=torch.float32)
        per_row = reduction == "none"
        p = buf.data_ptr()
        with on_device(z):
            C.distill_fwd(*_args(z, tv, ti, target, tlse, buf, temperature, hard),
                          loss.data_ptr() if per_row else p + 4 * n, 0 if per_row else loss.data_ptr(),
                          reduction == "mean", p + 4 * spare, stream(z))
        ctx.save_for_backward(z, tv, ti, target, tlse, buf)
        ctx.args = (temperature, hard)
        ctx.per_row = per_row
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        z, tv, ti, target, tlse, buf = ctx.saved_tensors
        dz = torch.empty(z.shape, device=z.device, dtype=z.dtype)
        dloss = dloss.contiguous()
        with on_device(z):
            native().distill_bwd(*_args(z, tv, ti, target, tlse, buf, *ctx.args), dloss.data_ptr(), ctx.per_row,
                                 dz.data_ptr(), stream(z))
        return dz, None, None, None, None, None, None, None


def _gain(d):
    """x e^x - e^x + 1 = sum x^n (n - 1) / n!, for |x| <= 1/4 without the difference of near numbers."""
    near = d.abs() < 0.25
    x = torch.where(near, d, 0.0)
    series = torch.zeros_like(x)
    for n in range(14, 1, -1):
        series = series * x + (n - 1) / math.factorial(n)
    x = torch.where(near, 0.0, d)
    return torch.where(near, series * torch.where(near, d, 0.0) ** 2, x * x.exp() - torch.expm1(x))


def _distill_kd(z, tv, ti, tlse, temperature, used, counted):
    """Each row's KL(p || q), in 64 bits; of size 1 / T^2 and right to its last digits at any T: sums of
    exponentials are held by how far they are from the number of their terms, and what is added up has
    no negative part (``csrc/distill.hip``)."""
    V, k = z.shape[1], tv.shape[1]
    at = torch.where(used, ti, 0).long()
    slot = torch.where(used, at, V)
    place = torch.arange(k, device=z.device, dtype=torch.int32).expand(ti.shape)
    first = torch.full((z.shape[0], V + 1), k, dtype=torch.int32, device=z.device).scatter_reduce_(1, slot, place, "amin")
    named = first[:, :V] < k
    first = used & (first.gather(1, slot) == place)  # an entry that is its class's first
    # the student
    live = z.detach() != -math.inf
    top = z.detach().amax(1, keepdim=True)
    dz = z - torch.where(live.any(1, keepdim=True), top, 0.0)
    n, e = live.sum(1).double(), torch.where(live, torch.expm1(dz.detach() / temperature), 0.0).sum(1)
    whole, part = n.log(), torch.log1p(e / n)  # of log sum exp(dz / T); its derivative is logsumexp's
    total = torch.logsumexp(dz / temperature, 1)
    part = part + (total - total.detach())
    share = torch.softmax(dz / temperature, 1)
    # the teacher
    tv = tv.double()
    if tlse is not None:
        dt = torch.where(used, tv, 0.0)
        norm = torch.where(counted, tlse.double(), 0.0)
        log_ratio = whole + part - norm
    else:
        most = torch.where(used, tv, -math.inf).amax(1, keepdim=True)
        dt = torch.where(used, tv - most, 0.0)
        m = used.sum(1).double()
        p1 = torch.log1p(torch.where(used, torch.expm1(dt / temperature), 0.0).sum(1) / m)
        norm = m.log() + p1
        log_ratio = (whole - m.log()) + (part - p1)
    p = torch.where(used, (dt / temperature - norm[:, None]).exp(), 0.0)
    q = torch.where(used, share.gather(1, at), 0.0)
    d = (dt - dz.gather(1, at)) / temperature + log_ratio[:, None]  # log p - log q
    has_p = used & (p != 0)
    near = has_p & (d.detach().abs() < 0.25)
    far = torch.where(has_p & ~near, p * torch.where(has_p & ~near, d, 0.0), 0.0) - p + q
    kd = torch.where(near, q * _gain(torch.where(near, d, 0.0)), far).sum(1)
    less = torch.where(near, q * torch.expm1(torch.where(near, d, 0.0)), p - q).sum(1)  # sum p - sum q
    twice = torch.where(first, 0.0, q).sum(1)
    q_out = torch.where(live & ~named, share, 0.0).sum(1)
    rest = torch.zeros_like(kd)
    sum_p = torch.ones_like(kd)
    if tlse is not None:
        sum_p = p.sum(1)
        has = (live & ~named).any(1) & ~(sum_p >= 1)
        q_safe = torch.where(has & (q_out != 0), q_out, 1.0)
        over = -(less + twice) / q_safe  # rest / q_out - 1
        by_sum = (over.detach().abs() < 0.2) & (q_out.detach() != 0)
        rest = torch.where(has, 1 - sum_p, 0.0)
        r = torch.where(has, rest, 1.0)
        # log q_out, also where it is too small for a number: from the maximum outside
        out = torch.where(has[:, None], torch.where(live & ~named, dz, -math.inf), 0.0)
        most = out.detach().amax(1, keepdim=True)
        log_q = torch.logsumexp((out - most) / temperature, 1) + most[:, 0] / temperature - whole - part
        gain = torch.where(by_sum, q_out * _gain(torch.log1p(torch.where(by_sum, over, 0.0))),
                           r * (r.log() - log_q) - r + q_out)
        rest = torch.where(has, gain, (sum_p - 1) + q_out)
    else:
        rest = q_out
    return torch.where(used.any(1), kd + rest - twice, 0.0)


def _distill_rows(z, tv, ti, target, tlse, temperature, hard):
    """Each row's loss in plain torch (the CPU path), in 64 bits, and which rows count."""
    V = z.shape[1]
    used = (ti >= 0) & (ti < V) & (tv != -math.inf)
    counted = used.any(1) if target is None else (target >= 0) & (target < V)
    z = torch.where(counted[:, None], z.double(), 0.0)  # what a left-out row holds stays out
    used = used & counted[:, None]
    loss = torch.zeros_like(z[:, 0])
    if hard < 1:  # a weight of 0 takes the term out, whatever the teacher says
        loss = (1 - hard) * temperature * temperature * _distill_kd(z, tv, ti, tlse, temperature, used, counted)
    if hard > 0:
        y = torch.where(counted, target, 0).long()[:, None]
        top = z.detach().amax(1, keepdim=True)
        dz = z - torch.where(torch.isfinite(top), top, 0.0)  # a row of the type's lowest value keeps its log V
        loss = loss + hard * (torch.logsumexp(dz, 1) - dz.gather(1, y)[:, 0])
    return torch.where(counted, loss, 0.0), counted


def distill_loss(logits: torch.Tensor, top_values: torch.Tensor, top_index: torch.Tensor,
                 target: torch.Tensor | None = None, top_lse: torch.Tensor | None = None, temperature: float = 1.0,
                 hard_weight: float = 0.0, reduction: str = "mean"):
    """Distillation from a teacher's top logits; with p the teacher's and q = softmax(logits / T)

        loss = (1 - hard_weight) T^2 KL(p || q) + hard_weight cross_entropy(logits, target)

    (a term whose weight is 0 is left out, so with a weight of 1 the teacher's values are not looked at).

    ``logits``: [..., V], the student's, float32, bfloat16 or float16, at most 8388607 rows and 2^30
    classes.  ``top_values`` [..., k] (one
    of these types) and ``top_index`` [..., k] (int32 or int64): the teacher's logits for k <= 256
    named classes, as ``top_logits`` gives them.  An entry whose index lies outside [0, V) or whose
    value is -inf is unused; a class named twice has both entries' share.

    Without ``top_lse`` p is the softmax over the named classes.  With it ([...] float32, the
    teacher's log sum exp(t / T) at the same temperature) p is the teacher's true probability, and
    the rest of both distributions, outside the named classes, is compared as one more class (left
    out where the student gives nothing to the classes outside).

    ``target`` [...] (int32 or int64): the row's class; a row whose target lies outside [0, V) (such
    as -100) is left out: loss 0, gradient 0, not counted.  Without targets the rows with no used
    entry are left out.  ``reduction``: "mean" over the counted rows (0 if there are none), "sum", or
    "none" (each row's loss, [...]).  The loss is float32.  Only ``logits`` get a gradient, once
    differentiable; on the GPU a forward-mode tangent is refused.

    Both directions may be captured into a graph.  As for every operator, no loss of an earlier eager
    step may then still hold its autograd graph: torch would draw the stream on which that step met
    the parameters into the capture, which ends the process."""
    check_float(logits, "distill_loss: logits", cpu_double=True)
    check_float(top_values, "distill_loss: top_values", cpu_double=True)
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_CLASSES:
        raise ValueError(f"distill_loss: logits must be [..., V] with 1 <= V <= 2^30, got {tuple(logits.shape)}")
    lead, V = logits.shape[:-1], logits.shape[-1]
    if top_values.dim() < 1 or top_values.shape[:-1] != lead or top_index.shape != top_values.shape:
        raise ValueError(f"distill_loss: top_values {tuple(top_values.shape)} and top_index {tuple(top_index.shape)} "
                         f"must both be {tuple(lead)} + (k,)")
    k = top_values.shape[-1]
    if not 1 <= k <= MAX_TOP:
        raise ValueError(f"distill_loss: k must be within 1 .. {MAX_TOP}, got {k}")
    for t, name in ((top_index, "top_index"), (target, "target")):
        if t is not None and t.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"distill_loss: {name} must be int32 or int64, got {t.dtype}")
    if target is not None and target.shape != lead:
        raise ValueError(f"distill_loss: target must be {tuple(lead)}, got {tuple(target.shape)}")
    if top_lse is not None and (top_lse.dtype not in (torch.float32, torch.float64) or top_lse.shape != lead
                                or (logits.is_cuda and top_lse.dtype != torch.float32)):
        raise ValueError(f"distill_loss: top_lse must be float32 {tuple(lead)}, got {top_lse.dtype} "
                         f"{tuple(top_lse.shape)}")
    for t, name in ((top_values, "top_values"), (top_index, "top_index"), (target, "target"), (top_lse, "top_lse")):
        check_device(t, logits, name)
    if has_derivative(top_values, top_lse):
        raise ValueError("distill_loss: top_values and top_lse get no gradient; detach them")
    temperature, hard = _check_temperature(temperature), float(hard_weight)
    if not 0 <= hard <= 1:
        raise ValueError(f"distill_loss: hard_weight must be within 0 .. 1, got {hard_weight}")
    if hard > 0 and target is None:
        raise ValueError("distill_loss: hard_weight needs a target")
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"distill_loss: reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    z, tv, ti = rows_of(logits), top_values.reshape(-1, k), top_index.reshape(-1, k)
    target = None if target is None else target.reshape(-1)
    tlse = None if top_lse is None else top_lse.reshape(-1)
    if not _native(logits):
        loss, counted = _distill_rows(z, tv, ti, target, tlse, temperature, hard)
        loss = loss.reshape(lead) if reduction == "none" else loss.sum()
        loss = loss / counted.sum().clamp_min(1) if reduction == "mean" else loss
        return loss if logits.dtype == torch.float64 else loss.float()
    if z.shape[0] > MAX_ROWS:
        raise ValueError(f"distill_loss: {z.shape[0]} rows, at most {MAX_ROWS}")
    loss = _DistillLoss.apply(z, tv.contiguous(), ti.contiguous(), None if target is None else target.contiguous(),
                              None if tlse is None else tlse.contiguous(), temperature, hard, reduction)
    return loss.reshape(lead) if reduction == "none" else loss
