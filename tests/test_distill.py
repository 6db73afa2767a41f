"""A teacher's top logits and the distillation loss (ops.top_logits, ops.distill_loss) against their
definitions in 64 bits, on the CPU path and on the kernels.

Bounds, with E = 2^-24 (half a step of fp32).  A row's sum of exponentials s = sum exp((z - m) / T)
is of positive terms.  Each term's argument has three roundings (the difference, the factor, the
product), so it is off by at most 3 E d with d = (m - z) / T, and the exponential by one step more;
d exp(-d) summed over V classes is at most log(V) s.  Adding up: at most V / 64 terms in one thread's
chain and 64 steps of joining (each with an exponential that rescales).  So s is relatively off by at
most ES = (V / 64 + 64 + 3 log V + 4) E, and log s by that much absolutely.
"""
import math
from decimal import Decimal, localcontext

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from mxddp import ops
from mxddp.models.layers import Int8Linear, Linear

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]
E = 2.0**-24
INF = math.inf


def es(V):
    return (V / 64 + 64 + 3 * math.log(V + 1) + 4) * E


# ------------------------------------------------------------------------------------ top logits
def check_top(z, k, got, T=1.0):
    """z: [N, V] on the CPU."""
    zd = z.double()
    key = torch.where(torch.isnan(zd), torch.full_like(zd, INF), zd)
    # NaN first, then by value, then by class
    order = torch.stack([torch.tensor(sorted(range(z.shape[1]), key=lambda i: (not math.isnan(r[i]), -kr[i], i))[:k])
                         for r, kr in zip(zd.tolist(), key.tolist())]) if z.shape[0] else torch.zeros(0, k)
    order = order.long().reshape(z.shape[0], k)
    values, index, lse = (t.cpu() for t in got)
    assert index.dtype == torch.int32 and torch.equal(index.long(), order)
    want = z.gather(1, order)
    same = (values == want) | (torch.isnan(values) & torch.isnan(want))
    assert values.dtype == z.dtype and bool(same.all())
    wl = torch.logsumexp(zd / T, 1)
    m = (zd / T).amax(1).abs()
    fine = torch.isfinite(wl)
    assert torch.equal(torch.isnan(lse), torch.isnan(wl))
    assert torch.equal(lse[~fine & ~torch.isnan(wl)].double(), wl[~fine & ~torch.isnan(wl)])
    tol = es(z.shape[1]) + 4 * E * (m + wl.abs())
    assert bool(((lse.double() - wl).abs() <= tol)[fine].all())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,k", [(1, 1, 1), (3, 7, 7), (5, 10, 3), (2, 63, 63), (4, 65, 2), (3, 256, 256), (33, 1000, 10),
                                   (2, 1000, 200), (2, 8191, 64), (1, 8193, 64), (3, 16385, 256), (1, 50001, 100)])
def test_top_logits(dev, dtype, N, V, k):
    g = torch.Generator().manual_seed(V)
    z = (4 * torch.randn(N, V, generator=g)).to(dtype)
    T = [1.0, 2.0, 0.7][V % 3]
    check_top(z, k, ops.top_logits(z.to(dev), k, T), T)


def odd_rows(V, dtype):
    g = torch.Generator().manual_seed(V)
    low = torch.finfo(dtype).min
    r = torch.randn(V, generator=g).to(dtype)
    few = torch.randint(0, 3, (V,), generator=g).to(dtype)
    up = (torch.arange(V) % 2048).to(dtype).sort().values
    rows = [r, torch.zeros(V, dtype=dtype), few, up, up.flip(0), torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0).to(dtype)]
    for fill in (-INF, low):
        a = torch.full((V,), fill, dtype=dtype)
        rows.append(a.clone())
        a[[V - 1, V // 2, 3]] = torch.tensor([1.0, 2.0, 1.0]).to(dtype)
        rows.append(a)
    nan = r.clone()
    nan[[5, V - 2, V // 3]] = float("nan")
    one = r.clone()
    one[V - 1] = INF
    both = one.clone()
    both[2] = float("nan")
    peak = r.clone()
    peak[V // 2:V // 2 + 9] = 30
    late = torch.full((V,), -5.0, dtype=dtype)
    late[-70:] = torch.arange(70).to(dtype)
    return torch.stack(rows + [nan, one, both, peak, late, torch.full((V,), INF, dtype=dtype)])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,k", [(100, 8), (1500, 100), (9000, 64), (40000, 256)])
def test_top_logits_odd_rows(dev, dtype, V, k):
    """Ties, sorted rows either way, masks of -inf and of the lowest value, NaN, infinities, peaks."""
    z = odd_rows(V, dtype)
    check_top(z, k, ops.top_logits(z.to(dev), k))
    for i in range(z.shape[0]):  # one row at a time: long rows are then shared by several blocks
        check_top(z[i:i + 1], k, ops.top_logits(z[i:i + 1].to(dev), k))


@pytest.mark.parametrize("dev", DEVICES)
def test_top_logits_shapes(dev):
    g = torch.Generator().manual_seed(1)
    z = torch.randn(2, 3, 501, generator=g).to(torch.bfloat16)
    want = ops.top_logits(z.reshape(6, 501), 9)
    wide = torch.full((6, 600), 1e4, dtype=z.dtype, device=dev)
    wide[:, 33:534] = z.reshape(6, 501).to(dev)
    for v in (z.to(dev), wide[:, 33:534].reshape(2, 3, 501), z.to(dev).permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        got = ops.top_logits(v, 9)
        assert got.values.shape == (2, 3, 9) and got.lse.shape == (2, 3)
        check_top(z.reshape(6, 501), 9, [got.values.reshape(6, 9), got.index.reshape(6, 9), got.lse.reshape(6)])
    got = ops.top_logits(wide[:, 33:534], 9)
    assert torch.equal(got.index.cpu(), want.index)
    got = ops.top_logits(z[0, 0].to(dev), 9)
    assert got.lse.shape == () and torch.equal(got.index.cpu(), want.index[0])
    got = ops.top_logits(torch.empty(0, 5, device=dev), 2)
    assert got.values.shape == (0, 2) and got.lse.shape == (0,)
    one = z[:1, :1].expand(1, 4, 501)[0].to(dev)
    assert torch.equal(ops.top_logits(one.expand(4, 501), 9).index.cpu(), want.index[:1].expand(4, 9))


# --------------------------------------------------------------------------------- distill oracle
def times(share, bound):
    """share * bound, and 0 for a masked class: its exponential is 0 without error."""
    return torch.where(share == 0, 0.0, share * bound)


def oracle(z, tv, ti, target, tlse, T, h):
    """Rows' losses, rows counted, gradient of the sum of rows, and the bounds of both, in 64 bits
    from the formulas, entry by entry."""
    z, tv = z.detach().cpu().double(), tv.cpu().double()
    N, V = z.shape
    ti = ti.cpu().long()
    loss, counted = torch.zeros(N, dtype=torch.float64), torch.zeros(N, dtype=torch.bool)
    grad, tl, tg = torch.zeros(N, V, dtype=torch.float64), torch.zeros(N, dtype=torch.float64), torch.zeros(N, V, dtype=torch.float64)
    w = (1 - h) * T
    for r in range(N):
        used = (ti[r] >= 0) & (ti[r] < V) & (tv[r] != -INF)
        y = None if target is None else int(target[r])
        if (y is None and not used.any()) or (y is not None and not 0 <= y < V):
            continue
        counted[r] = True
        c, u = ti[r][used], tv[r][used] / T
        lz = torch.logsumexp(z[r] / T, 0)
        d = (z[r].amax() - z[r]) / T
        rel = es(V) + 4 * E * (d + 1)  # of one exponential over the sum
        q = (z[r] / T - lz).exp()
        p = u.new_zeros(0)
        if len(c):
            p = (u - (torch.logsumexp(u, 0) if tlse is None else tlse[r].cpu().double())).exp()
            lp = u - (torch.logsumexp(u, 0) if tlse is None else tlse[r].cpu().double())
            kd = torch.where(p > 0, p * (lp - (z[r][c] / T - lz)), 0.0).sum()
            # fp32 sum behind log z, and log p, log q in 64 bits
            err = p.sum() * es(V)
            mass = p.sum()
            eg = times(q, rel)
            big = torch.zeros(V, dtype=torch.float64).index_add(0, c, p)
        else:
            kd, err, mass, eg, big = 0.0, 0.0, 0.0, torch.zeros(V, dtype=torch.float64), 0.0
        far = 0.0
        if tlse is not None and len(c):
            out = torch.ones(V, dtype=torch.bool)
            out[c] = False
            rest = max(0.0, 1 - p.sum().item())
            if rest > 0 and out.any() and z[r][out].amax() > -INF:
                lo = torch.logsumexp(z[r][out] / T, 0)
                kd = kd + rest * (math.log(rest) - (lo - lz))
                # log q_rest = -log(1 + inside / outside): an error of the sum outside moves it by the
                # share inside only, so a small difference of p and q is not lost in their rest
                inside = q[~out].sum()
                err = err + rest * inside * (es(V) + 4 * E)
                qt = torch.where(out, (z[r] / T - lo).exp(), 0.0)
                do = (z[r][out].amax() - z[r]).clamp_min(0) / T
                mass, far = mass + rest, rest * qt
                # a class outside: one exponential times (q_rest - rest)
                diff = ((lo - lz).exp() * mass - rest).abs()
                eg = torch.where(out, times(diff * qt, es(V) + 4 * E * (do + 1)) + qt * inside * (es(V) + 4 * E), eg)
        g = w * (mass * q - far - big)
        own = torch.zeros(V, dtype=torch.float64).index_fill(0, c, 1.0) if tlse is not None else 1.0
        eg = w * (max(1.0, float(mass)) * eg + 4 * E * (mass * q * own + big))
        loss[r] = (1 - h) * T * T * kd
        tl[r] = (1 - h) * T * T * err
        if h > 0:
            l1 = torch.logsumexp(z[r], 0)
            loss[r] += h * (l1 - z[r][y])
            s1 = (z[r] - l1).exp()
            g = g + h * s1
            g[y] -= h
            eg = eg + h * times(s1, es(V) + 4 * E * (d * T + 1)) + 4 * E * h * s1
            eg[y] += 4 * E * h
            tl[r] += h * es(V)
        tl[r] += 2 * E * loss[r].abs()
        # the exponential of a far class is 0 below 2^-126; it is multiplied by at most w (1 / Z + rest /
        # Z_out) + h / Z_1 with all three sums >= 1 (each holds its own maximum), so by 2 w + h
        tg[r] = eg + 4 * E * g.abs() + 2.0**-126 * (2 * w + h)
        grad[r] = g
    return loss, counted, grad, tl, tg


def check_distill(dev, z, tv, ti, target=None, tlse=None, T=1.0, h=0.0, reduction="mean", leaf=None):
    """z: the logits on the CPU; leaf: the same values on `dev` in another layout."""
    zl = (z.to(dev) if leaf is None else leaf).detach().requires_grad_()
    mv = lambda t: None if t is None else t.to(dev)  # noqa: E731
    loss = ops.distill_loss(zl, mv(tv), mv(ti), target=mv(target), top_lse=mv(tlse), temperature=T, hard_weight=h,
                            reduction=reduction)
    rows, counted, grad, tl, tg = oracle(z, tv, ti, target, tlse, T, h)
    n = max(1, int(counted.sum()))
    if reduction == "none":
        share = torch.linspace(-1, 2, z.shape[0])
        want, tol = rows, tl
        g, = torch.autograd.grad(loss, zl, share.to(dev))
        share = share.double()
    else:
        f = 1 / n if reduction == "mean" else 1.0
        want, tol = rows.sum() * f, (tl.sum() + 3 * E * rows.abs().sum()) * f
        g, = torch.autograd.grad(loss * 1.0, zl)
        share = torch.full((z.shape[0],), f, dtype=torch.float64)
    assert loss.dtype == torch.float32 and loss.shape == want.shape
    far = (loss.detach().cpu().double() - want).abs()
    assert bool((far <= tol + 1e-37).all()), f"loss off by {(far / tol).max().item():.2f} of the bound"
    assert g.dtype == z.dtype and g.shape == z.shape
    wg = grad * share[:, None]
    fi = torch.finfo(z.dtype)
    tol = (tg + 3 * E * grad.abs()) * share[:, None].abs()
    # the result's type: half a step, and half a step of its subnormals
    tol = tol + fi.eps / 2 * (wg.abs() + tol) + fi.smallest_normal * fi.eps
    far = (g.cpu().double() - wg).abs()
    assert bool((far <= tol).all()), f"gradient off by {(far / tol).max().item():.2f} of the bound"
    return loss, g


def make(N, V, k, dtype, seed=0, T=1.0):
    g = torch.Generator().manual_seed(seed)
    teacher = (3 * torch.randn(N, V, generator=g)).to(dtype)
    z = (0.5 * teacher.float() + torch.randn(N, V, generator=g)).to(dtype)
    tv, ti, lse = ops.top_logits(teacher, k, T)
    y = torch.randint(V, (N,), generator=g)
    return z, tv, ti, y, lse


CASES = [(1, 1, 1), (2, 2, 1), (3, 7, 3), (5, 10, 10), (4, 65, 20), (9, 1000, 10), (3, 1000, 256), (2, 4099, 100),
         (2, 50001, 33), (1, 131075, 64)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("N,V,k", CASES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("T,h", [(1.0, 0.0), (2.0, 0.3), (1.0, 0.5), (0.7, 0.0), (4.0, 1.0)])
def test_distill_loss(dev, N, V, k, tail, T, h):
    dtype = TYPES[(V + N) % 3]
    z, tv, ti, y, lse = make(N, V, k, dtype, N + V, T)
    check_distill(dev, z, tv, ti, y if h > 0 else None, lse if tail else None, T, h)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_loss_types(dev, dtype, reduction, tail):
    """Every type, int64 indices and int32 targets, teacher values of another type, padded rows."""
    z, tv, ti, y, lse = make(12, 300, 17, torch.float32, 3, 2.0)
    z = z.to(dtype)
    y[[0, 5, 11]] = torch.tensor([-100, 300, -1])
    ti = ti.long()
    ti[4, :] = -1           # the teacher says nothing about this row
    ti[6, 5:] = 1 << 40     # a short list
    check_distill(dev, z, tv.to(torch.float16), ti, y.to(torch.int32), lse if tail else None, 2.0, 0.25, reduction)
    check_distill(dev, z, tv, ti, y, lse if tail else None, 2.0, 0.0, reduction)
    check_distill(dev, z, tv, ti, None, lse if tail else None, 2.0, 0.0, reduction)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("tail", [False, True])
def test_distill_loss_entries(dev, tail):
    """Classes named twice, the label among them and not, teacher values of -inf, all classes named."""
    V = 40
    z, tv, ti, y, lse = make(6, V, 8, torch.float32, 5)
    ti[0, 3] = ti[0, 1]
    ti[1, :] = ti[1, 0]
    tv[2, 4:] = -INF
    tv[3, :] = -INF
    y[0], y[1], y[2] = ti[0, 1], ti[1, 0], (ti[2, 0] + 1) % V
    for h in (0.0, 0.4):
        check_distill(dev, z, tv, ti, y if h else None, lse + 0.5 if tail else None, 1.0, h)
        check_distill(dev, z, tv, ti, y if h else None, lse + 0.5 if tail else None, 3.0, h)
    z, tv, ti, y, lse = make(5, V, V, torch.float32, 6)  # nothing outside: what 1 - sum p rounds to has no class
    check_distill(dev, z, tv, ti, y, lse if tail else None, 1.0, 0.1)
    check_distill(dev, z, tv, ti, None, lse + 0.1 if tail else None, 2.0, 0.0)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("fill", ["inf", "lowest"])
def test_distill_loss_masked_classes(dev, dtype, tail, fill):
    """Student logits masked with -inf or the type's lowest value: few classes left, all outside
    masked, all but the label masked."""
    V, k = 500, 6
    z, tv, ti, y, lse = make(4, V, k, dtype, 8)
    low = -INF if fill == "inf" else torch.finfo(dtype).min
    keep = torch.zeros(4, V, dtype=torch.bool)
    keep.scatter_(1, ti.long(), True)
    keep[1, 100:110] = True
    keep[3] = True
    y[0], y[1], y[2] = ti[0, 0], 105, ti[2, 1]
    z = torch.where(keep, z, low)
    for T, h in ((1.0, 0.0), (2.0, 0.3), (1.0, 0.5)):
        if tail and fill == "lowest" and dtype != torch.float16:
            # rest > 0 against classes at -1e38: the term is as large; keep rows that have others
            check_distill(dev, z[[1, 3]], tv[[1, 3]], ti[[1, 3]], y[[1, 3]] if h else None, lse[[1, 3]], T, h)
        else:
            check_distill(dev, z, tv, ti, y if h else None, lse if tail else None, T, h)


@pytest.mark.parametrize("dev", DEVICES)
def test_distill_loss_far_values(dev):
    """A student sure of one class, named or not: nothing overflows, the others' gradient stays."""
    V = 64
    z, tv, ti, y, lse = make(6, V, 5, torch.float32, 9)
    z[0, ti[0, 0].long()] = 200.0
    z[1, ti[1, 0].long()] = 1e4
    out = [int(i) for i in range(V) if i not in ti[2].tolist()][0]
    z[2, out] = 200.0
    z[3] += 1e4
    z[4] -= 3e4
    z[5] *= 50
    for T, h in ((1.0, 0.0), (1.0, 0.5), (2.0, 0.5)):
        check_distill(dev, z, tv, ti, y if h else None, lse, T, h)
        check_distill(dev, z, tv, ti, y if h else None, None, T, h)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("T", [1.0, 2.0])
def test_distill_loss_labels_alone(dev, dtype, tail, T):
    """hard_weight = 1 is the labels' cross-entropy: named classes that the student masks, teacher's
    values that are infinite or NaN and rows without any change nothing."""
    N, V, k = 6, 300, 5
    z, tv, ti, y, lse = make(N, V, k, dtype, 21, T)
    y = torch.where(y == ti[:, 0], (y + 1) % V, y)
    y[1] = ti[1, 1]
    z[0, ti[0, 0].long()] = -INF
    z[1, ti[1, 0].long()] = -INF
    tv[2, 1], tv[3, 0], ti[4] = INF, float("nan"), -1
    lse[5] = -1e30  # a normaliser that does not belong to the values: p overflows
    check_distill(dev, z[4:5], tv[4:5], ti[4:5], y[4:5], lse[4:5] if tail else None, T, 1.0)
    rows, counted, grad, tl, tg = oracle(z, tv, torch.full_like(ti, -1), y, None, T, 1.0)
    leaf = z.to(dev).requires_grad_()
    loss = ops.distill_loss(leaf, tv.to(dev), ti.to(dev), y.to(dev), lse.to(dev) if tail else None, T, 1.0, "none")
    g, = torch.autograd.grad(loss.sum(), leaf)
    assert bool(((loss.detach().cpu().double() - rows).abs() <= tl).all())
    fi = torch.finfo(dtype)
    tol = tg + fi.eps / 2 * (grad.abs() + tg) + fi.smallest_normal * fi.eps
    assert bool(((g.cpu().double() - grad).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [65537, 140001])
def test_distill_loss_whole_long_rows(cuda, dtype, V):
    """So many rows that each is one block's: longer ones than the classes whose marks are in LDS at a
    time.  The teacher's classes spread over the whole row; most rows are left out."""
    N, k = 520, 40
    g = torch.Generator().manual_seed(V)
    z = torch.zeros(N, V, dtype=dtype)
    rows = [0, 7, N - 1]
    z[rows] = (2 * torch.randn(3, V, generator=g)).to(dtype)
    tv = (torch.randn(N, k, generator=g) + 2).to(dtype)
    ti = torch.randint(V, (N, k), generator=g)
    ti[rows, 0] = V - 1
    lse = torch.full((N,), 8.0)
    y = torch.full((N,), -100)
    y[rows] = torch.tensor([3, 65536, V - 1])
    for T, h in ((1.0, 0.0), (2.0, 0.5)):
        check_distill("cuda", z, tv, ti, y, lse, T, h)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("V,k,T", [(300, 2, 4.0), (50000, 1, 4.0), (50000, 40, 8.0)])
def test_distill_loss_small_shares(dev, V, k, T):
    """Named classes that hold little, a student near its teacher: the loss is a small difference of
    the shares, and so is the gradient of every class outside."""
    g = torch.Generator().manual_seed(V)
    teacher = torch.randn(4, V, generator=g)
    z = teacher + 0.05 * torch.randn(4, V, generator=g)
    tv, ti, lse = ops.top_logits(teacher, k, T)
    check_distill(dev, z, tv, ti, None, lse, T)
    check_distill(dev, z, tv, ti, None, lse, T, 0.0, "none")


def oracle_decimal(z, tv, ti, target, tlse, T, h):
    """One row's loss and gradient from the formulas, in 160 digits, and the shares q and softmax(z)."""
    with localcontext() as c:
        c.prec = 160
        zero, one, T, w1 = Decimal(0), Decimal(1), Decimal(T), Decimal(1) - Decimal(h)
        z = [Decimal(v) if v != -INF else None for v in z]
        lse = lambda v: (lambda m: m + sum((x - m).exp() for x in v).ln())(max(v))  # noqa: E731
        zt = [None if v is None else v / T for v in z]
        total = lse([v for v in zt if v is not None])
        q = [zero if v is None else (v - total).exp() for v in zt]
        pairs = [(int(i), Decimal(v) / T) for i, v in zip(ti, tv) if 0 <= i < len(z) and v != -INF]
        norm = lse([u for _, u in pairs]) if tlse is None else Decimal(tlse)
        p = [(i, (u - norm).exp()) for i, u in pairs]
        mass = sum((x for _, x in p), zero)
        kd = sum((x * (u - norm - (zt[i] - total)) for (i, x), (_, u) in zip(p, pairs)), zero)
        out = [i for i in range(len(z)) if z[i] is not None and i not in {i for i, _ in p}]
        share, rest = mass, zero
        if tlse is not None and out and mass < 1:
            rest, share = one - mass, one
            outside = lse([zt[i] for i in out])
            kd += rest * (rest.ln() - (outside - total))
        grad = [share * x for x in q]
        for i in out:
            if rest > 0:
                grad[i] -= rest * (zt[i] - outside).exp()
        for i, x in p:
            grad[i] -= x
        loss, grad = w1 * T * T * kd, [w1 * T * g for g in grad]
        soft = [0.0] * len(z)
        if h > 0:
            l1 = lse([v for v in z if v is not None])
            loss += Decimal(h) * (l1 - z[target])
            for i, v in enumerate(z):
                if v is not None:
                    soft[i] = float((v - l1).exp())
                    grad[i] += Decimal(h) * (v - l1).exp()
            grad[target] -= Decimal(h)
        return float(loss), [float(g) for g in grad], [float(x) for x in q], soft


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("N,V,k,kind,T", [(3, 10, 10, "all", T) for T in (8.5, 20.0, 100.0, 1e4, 1e6, 1e12, 1e30)]
                         + [(3, 100, 40, "few", T) for T in (8.5, 20.0, 100.0, 1e4, 1e6, 1e12, 1e30)]
                         + [(2, 256, 256, "all", T) for T in (20.0, 1e6)] + [(3, 100, 40, "near", T) for T in (9.0, 1e4)]
                         + [(2, 200, 30, "masked", T) for T in (10.0, 1e3)] + [(2, 120, 24, "twice", T) for T in (20.0, 1e5)]
                         + [(1, 8200, 64, "few", T) for T in (12.0, 1e6)])
@pytest.mark.parametrize("tail,h", [(False, 0.0), (True, 0.0), (True, 0.3)])
def test_distill_loss_high_temperatures(dev, N, V, k, kind, T, tail, h):
    """T^2 KL keeps the size of the logits' differences at any T, and so does its gradient times 1 / T: with
    e the distance of two logarithms log p - log q (each right to a few steps U = 2^-53 of its parts, the
    sums of exponentials to (V / 64 + 64) U of how far their terms are from 1), KL is made of terms p e, each
    paired with its share so that none is negative, and the gradient of terms q (exp(e) - 1)."""
    dtype = TYPES[(N + V) % 3]
    g = torch.Generator().manual_seed(V + k)
    teacher = (3 * torch.randn(N, V, generator=g)).to(dtype)
    noise = 0.01 if kind == "near" else 1.0
    z = (teacher.float() * (1.0 if kind == "near" else 0.5) + noise * torch.randn(N, V, generator=g)).to(dtype)
    tv, ti = (t[:, :k].contiguous() for t in torch.sort(teacher, dim=1, descending=True))
    if kind == "masked":
        z[:, torch.randperm(V, generator=g)[:50]] = -INF
        z.scatter_(1, ti, tv - 1)
        ti[0, 3], tv[1, 5] = -1, -INF
    if kind == "twice":
        ti[:, 4], ti[:, 9], ti[:, 10] = ti[:, 1], ti[:, 2], ti[:, 2]
    lse = torch.logsumexp(teacher.double() / T, 1).float() if tail else None
    y = torch.arange(N) + 2 if h else None
    if h:
        z.scatter_(1, y[:, None], torch.where(z.gather(1, y[:, None]) == -INF, 0.0, z.gather(1, y[:, None])))
    leaf = z.to(dev, copy=True).requires_grad_()
    loss = ops.distill_loss(leaf, tv.to(dev), ti.to(dev), None if y is None else y.to(dev),
                            None if lse is None else lse.to(dev), T, h, "none")
    grad, = torch.autograd.grad(loss.sum(), leaf)
    fi = torch.finfo(dtype)
    for r in range(N):
        want, wg, q, soft = oracle_decimal(z[r].tolist(), tv[r].tolist(), ti[r].tolist(), None if y is None else int(y[r]),
                                           None if lse is None else lse[r].item(), T, h)
        zr = z[r][z[r] != -INF].double()
        gap = float(zr.max() - zr.min() + tv[r][tv[r] != -INF].double().max() - tv[r][tv[r] != -INF].double().min())
        high = gap if not tail else float(max(gap, tv[r][tv[r] != -INF].double().abs().max()))
        U = 2.0**-53 * 8 * (V / 64 + 64)
        ends = abs(lse[r].item()) + math.log(V) if tail else 0.0  # what does not shrink with 1 / T
        d = U * (high / T + ends)  # of one log p - log q
        largest = 2 * gap / T + (E * ends if tail else 0.0)  # how far apart p and q are
        tol = 2 * E * abs(want) + T * T * (d * largest + d * d) + h * es(V)
        got = loss[r].item()
        if abs(want) > 3.4e38:
            assert got == math.copysign(INF, want)
        else:
            assert abs(got - want) <= tol, (got, want, tol)
            if h == 0 and T <= (100 if tail else 1e6) and kind != "twice":  # the bound is far below the loss
                assert tol < 1e-3 * abs(want)
        wg, q, soft = (torch.tensor(v, dtype=torch.float64) for v in (wg, q, soft))
        far = (zr.max() - z[r].double()).clamp_max(1e300) / T
        hard = h * times(soft, es(V) + 4 * E * (far * T + 2)) + (4 * E * h if h else 0.0)
        tg = (16 + 8 * gap / T) * E * (wg.abs() + h * (soft + 1)) + T * q * d * 4 + hard
        if kind == "twice":  # two shares of one class side by side
            tg = tg + 16 * E * T * q
        tg = tg + fi.eps / 2 * 1.01 * (wg.abs() + tg) + fi.smallest_normal * fi.eps + 2.0**-126 * (2 * T + h)
        gr = grad[r].cpu().double()
        big = wg.abs() > fi.max
        assert bool(((gr - wg).abs() <= tg)[~big].all()), float(((gr - wg).abs() / tg)[~big].max())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("V,k,T", [(300, 2, 4.0), (50000, 1, 4.0), (50000, 40, 8.0), (4096, 20, 1.0), (50000, 40, 30.0)])
def test_distill_loss_small_losses(dev, V, k, T):
    """A student near its teacher and classes that hold little, against bounds far below the loss and the
    gradients.  An error of the sum S outside the named classes moves KD by (q_out - rest) d log S to first
    order and q_in q_out / 2 d log S^2 to second; log S is right to EO = (32 + 3 (V / 4096 + 1) + 3 log V + 8) E: a tile's 32
    terms added up in fp32, its rescaling at each of a thread's V / 4096 + 1 tiles, the exponents' three
    roundings and the exponential's; what is joined after that is in 64 bits."""
    g = torch.Generator().manual_seed(V + int(T))
    teacher = torch.randn(4, V, generator=g)
    z = teacher + 0.05 * torch.randn(4, V, generator=g)
    tv, ti, lse = ops.top_logits(teacher, k, T)
    leaf = z.to(dev, copy=True).requires_grad_()
    loss = ops.distill_loss(leaf, tv.to(dev), ti.to(dev), top_lse=lse.to(dev), temperature=T, reduction="none")
    grad, = torch.autograd.grad(loss.sum(), leaf)
    rows, _, wg, _, _ = oracle(z, tv, ti, None, lse, T, 0.0)
    eo = (32 + 3 * (V / 4096 + 1) + 3 * math.log(V + 1) + 8) * E
    q = torch.softmax(z.double() / T, 1)
    named = torch.zeros(4, V, dtype=torch.bool).scatter_(1, ti.long(), True)
    p = (tv.double() / T - lse.double()[:, None]).exp()
    rest, q_out = 1 - p.sum(1), torch.where(named, 0.0, q).sum(1)
    tol = T * T * (eo * (q_out - rest).abs() + eo * eo * (1 - q_out) + 2.0**-50 * math.log(V)) + 2 * E * rows
    assert bool((tol < 0.1 * rows).all()), (tol / rows).max()
    assert bool(((loss.detach().cpu().double() - rows).abs() <= tol).all())
    # a named class: q (exp(d) - 1) with d right to EO; one outside: q / q_out times (q_out - rest), right to
    # EO q_in q_out
    q_in = 1 - q_out
    tg = T * torch.where(named, q * eo, q / q_out[:, None] * (eo * q_in * q_out)[:, None]) + 16 * E * wg.abs()
    tg = tg + T * q * 2.0**-50 * math.log(V) + 2.0**-148 + 2.0**-126 * 2 * T
    assert bool((tg[named] < 0.05 * wg[named].abs().median()).all())
    assert bool((tg[~named] < 0.5 * wg[~named].abs()).all()), (tg / wg.abs())[~named].max()
    assert bool(((grad.cpu().double() - wg).abs() <= tg).all())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1.0, 4.0, 20.0])
def test_distill_loss_rows_of_one_value(dev, dtype, T):
    """Rows that hold one value everywhere, the type's lowest, its largest and others: the student knows
    nothing, the labels' loss is log V whatever the value, and so is KL to a teacher that is sure."""
    V = 24
    low, big = torch.finfo(dtype).min, torch.finfo(dtype).max
    z = torch.tensor([low, big, 0.0, -1e4, 3e4]).to(dtype)[:, None].expand(5, V)
    tv, ti = torch.tensor([[1e4, -3e4]]).to(dtype).expand(5, 2), torch.tensor([[3, 7]]).expand(5, 2)
    y = torch.full((5,), 7)
    leaf = z.to(dev, copy=True).requires_grad_()
    for h in (0.0, 0.5, 1.0):
        loss = ops.distill_loss(leaf, tv.to(dev), ti.to(dev), y.to(dev), None, T, h, "none")
        g, = torch.autograd.grad(loss.sum(), leaf)
        want = (h + (1 - h) * T * T) * math.log(V)
        assert bool(((loss.detach().cpu().double() - want).abs() <= (h + (1 - h) * T * T) * es(V) + 2 * E * want).all())
        wg = torch.full((V,), (h + (1 - h) * T) / V, dtype=torch.float64)
        wg[3] -= (1 - h) * T
        wg[7] -= h
        tol = es(V) * (h + (1 - h) * T) + torch.finfo(dtype).eps / 2 * 1.01 * wg.abs() + 2.0**-24
        assert bool(((g.cpu().double() - wg).abs() <= tol).all())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1.0, 8.0, 50.0, 1e6])
def test_distill_loss_little_left(dev, dtype, T):
    """Rows of which the student leaves little: only classes at the type's lowest value outside the named
    ones (they share the rest evenly), one class alone (its gradient is 0), a few, all of them named, and a
    teacher whose normaliser counts the masked classes too."""
    V, k = 30, 6
    g = torch.Generator().manual_seed(5)
    teacher = torch.randn(3, V, generator=g).to(dtype)
    z = (teacher.float() + torch.randn(3, V, generator=g)).to(dtype)
    tv, ti = (t[:, :k].contiguous() for t in torch.sort(teacher, dim=1, descending=True))
    lse = torch.logsumexp(teacher.double() / T, 1).float()
    out = torch.ones(3, V, dtype=torch.bool).scatter_(1, ti, False)
    z[0, out[0]] = torch.finfo(dtype).min
    z[1, torch.arange(V) != ti[1, 2]] = -INF
    z[2, out[2]] = -INF
    ti[1, [0, 1, 3, 4, 5]] = -1  # what the student masks is not named: its KL would be infinite
    leaf = z.to(dev, copy=True).requires_grad_()
    loss = ops.distill_loss(leaf, tv.to(dev), ti.to(dev), None, lse.to(dev), T, 0.0, "none")
    grad, = torch.autograd.grad(loss.sum(), leaf)
    fi = torch.finfo(dtype)
    for r in range(3):
        want, wg, q, _ = oracle_decimal(z[r].tolist(), tv[r].tolist(), ti[r].tolist(), None, lse[r].item(), T, 0.0)
        if r and abs(want) < 3.4e38:
            assert abs(loss[r].item() - want) <= T * T * es(V) + 2 * E * abs(want)
        wg, q = torch.tensor(wg, dtype=torch.float64), torch.tensor(q, dtype=torch.float64)
        # up to T = 8 the sums are fp32; above, a class's gradient is right to some steps of its own and
        # T q 2^-50 (sizes of lse and of d)
        tg = 32 * E * wg.abs() + T * q * (es(V) if T <= 8 else 2.0**-44)
        tg = tg + fi.eps / 2 * 1.01 * (wg.abs() + tg) + fi.smallest_normal * fi.eps + 2.0**-126 * 2 * T
        ok = (grad[r].cpu().double() - wg).abs() <= tg
        assert bool((ok | (wg.abs() > fi.max)).all()), (r, grad[r].tolist(), wg.tolist())


@pytest.mark.parametrize("dev", DEVICES)
def test_distill_loss_nothing(dev):
    """No rows; no row that counts; a left-out row whose logits and teacher hold NaN."""
    z, tv, ti, y, lse = make(4, 30, 3, torch.float32, 10)
    leaf = z[:0].to(dev).requires_grad_()
    for red, shape in (("mean", ()), ("sum", ()), ("none", (0,))):
        loss = ops.distill_loss(leaf, tv[:0].to(dev), ti[:0].to(dev), reduction=red)
        assert loss.shape == shape and (loss == 0).all()
        assert torch.autograd.grad(loss.sum(), leaf)[0].shape == (0, 30)
    for kw in ({"target": torch.full((4,), -100)}, {}):
        t = ti if kw else torch.full_like(ti, -1)
        leaf = z.to(dev).requires_grad_()
        loss = ops.distill_loss(leaf, tv.to(dev), t.to(dev), **{k: v.to(dev) for k, v in kw.items()})
        assert loss.item() == 0 and (torch.autograd.grad(loss, leaf)[0] == 0).all()
    y[1] = -100
    bad, btv, blse = z.clone(), tv.clone(), lse.clone()
    bad[1], btv[1], blse[1] = float("nan"), float("nan"), float("nan")
    for tl, bl in ((None, None), (lse, blse)):
        for h in (0.0, 0.5):
            leaf = bad.to(dev).requires_grad_()
            loss = ops.distill_loss(leaf, btv.to(dev), ti.to(dev), target=y.to(dev), hard_weight=h, temperature=2.0,
                                    top_lse=None if bl is None else bl.to(dev))
            g, = torch.autograd.grad(loss, leaf)
            clean, cg = check_distill(dev, z, tv, ti, y, tl, 2.0, h)
            if dev == "cuda":
                assert torch.equal(loss, clean) and torch.equal(g, cg)
            else:
                assert torch.allclose(loss, clean) and (g[1] == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_loss_layouts(dev, dtype):
    """Rows in a wider tensor at odd starts, more dimensions, classes not contiguous, shared rows."""
    N, V, k = 6, 333, 4
    z, tv, ti, y, lse = make(N, V, k, dtype, 11)
    for off, pad in ((0, 0), (1, 0), (3, 60), (8, 3)):
        wide = torch.full((N, off + V + pad), float("nan"), dtype=dtype, device=dev)
        wide[:, off:off + V] = z.to(dev)
        check_distill(dev, z, tv, ti, y, lse, 2.0, 0.5, leaf=wide[:, off:off + V])
    check_distill(dev, z, tv, ti, y, None, 1.0, 0.0, leaf=z.to(dev).t().contiguous().t())
    leaf = z.reshape(2, 3, V).to(dev).requires_grad_()
    args = [t.to(dev) for t in (tv.reshape(2, 3, k), ti.reshape(2, 3, k))]
    loss = ops.distill_loss(leaf, *args, target=y.reshape(2, 3).to(dev), hard_weight=0.5, reduction="none")
    assert loss.shape == (2, 3)
    g, = torch.autograd.grad(loss.sum(), leaf)
    want, _, grad, tl, tg = oracle(z, tv, ti, y, None, 1.0, 0.5)
    assert bool(((loss.detach().cpu().double().reshape(-1) - want).abs() <= tl).all())
    one = z[:1].to(dev).requires_grad_()  # one row of logits against all the teacher's rows
    loss = ops.distill_loss(one.expand(N, V), tv.to(dev), ti.to(dev), reduction="sum")
    g, = torch.autograd.grad(loss, one)
    _, _, grad, _, tg = oracle(z[:1].expand(N, V), tv, ti, None, None, 1.0, 0.0)
    eps = torch.finfo(dtype).eps / 2 * 8  # each row rounded, then up to N - 1 sums in the type
    bound = (tg + eps * grad.abs()).sum(0, keepdim=True) + eps * grad.abs().sum(0, keepdim=True) + 1e-6 * 8
    assert g.shape == (1, V) and bool(((g.cpu().double() - grad.sum(0, keepdim=True)).abs() <= bound).all())


def test_distill_gradient_by_differences():
    """The CPU path's gradient in 64 bits against differences, and the oracle's formulas against it."""
    for tail in (False, True):
        for T, h in ((1.0, 0.0), (2.0, 0.3)):
            z, tv, ti, y, lse = make(3, 12, 4, torch.float32, 12, T)
            z = z.double().requires_grad_()
            lse = lse if tail else None
            f = lambda v: ops.distill_loss(v, tv, ti, y, lse, T, h)  # noqa: E731
            assert torch.autograd.gradcheck(f, (z,), eps=1e-6, atol=1e-7)
            rows, _, grad, _, _ = oracle(z, tv, ti, y, lse, T, h)
            loss = f(z)
            assert abs(loss.item() - rows.mean().item()) < 1e-12
            assert torch.allclose(torch.autograd.grad(loss, z)[0], grad / 3, atol=1e-13)


@pytest.mark.gpu
def test_distill_gradient_by_differences_gpu(cuda):
    """The kernel's gradient along a direction against the oracle's loss on both sides of z."""
    z, tv, ti, y, lse = make(4, 700, 9, torch.float32, 13, 2.0)
    leaf = z.to(cuda).requires_grad_()
    ops.distill_loss(leaf, tv.to(cuda), ti.to(cuda), y.to(cuda), lse.to(cuda), 2.0, 0.3).backward()
    d = torch.randn(4, 700, generator=torch.Generator().manual_seed(1)).double()
    step = 1e-4
    hi, lo = (oracle(z.double() + s * step * d, tv, ti, y, lse, 2.0, 0.3)[0].mean() for s in (1, -1))
    slope = (leaf.grad.cpu().double() * d).sum()
    # the difference's own error: step^2 times a third derivative of order |d|^3 ~ 1e-7
    assert abs((hi - lo) / (2 * step) - slope) <= 1e-6 + 1e-5 * slope.abs()


def test_refusals():
    z, tv, ti, y, lse = make(4, 30, 3, torch.float32)
    d = ops.distill_loss
    for bad, err in [
        (lambda: ops.top_logits(z.double(), 2), TypeError),
        (lambda: ops.top_logits(z, 0), ValueError),
        (lambda: ops.top_logits(z, 31), ValueError),
        (lambda: ops.top_logits(torch.zeros(2, 400), 257), ValueError),
        (lambda: ops.top_logits(torch.tensor(1.0), 1), ValueError),
        (lambda: ops.top_logits(z, 2, temperature=0), ValueError),
        (lambda: ops.top_logits(z, 2, temperature=INF), ValueError),
        (lambda: d(z.to(torch.int32), tv, ti), TypeError),
        (lambda: d(z, tv.to(torch.int32), ti), TypeError),
        (lambda: d(z, tv, ti.float()), TypeError),
        (lambda: d(z, tv, ti.to(torch.int16)), TypeError),
        (lambda: d(z, tv, ti, target=y.float()), TypeError),
        (lambda: d(z, tv, ti, target=y[:3]), ValueError),
        (lambda: d(z, tv, ti, target=y[:, None]), ValueError),
        (lambda: d(z, tv[:, :2], ti), ValueError),
        (lambda: d(z, tv[:3], ti[:3]), ValueError),
        (lambda: d(z, tv[:, :0], ti[:, :0]), ValueError),
        (lambda: d(torch.zeros(2, 400), torch.zeros(2, 257), torch.zeros(2, 257, dtype=torch.int32)), ValueError),
        (lambda: d(z, tv, ti, top_lse=lse[:3]), ValueError),
        (lambda: d(z, tv, ti, top_lse=lse.half()), ValueError),
        (lambda: d(z, tv, ti, temperature=-1.0), ValueError),
        (lambda: d(z, tv, ti, temperature=float("nan")), ValueError),
        (lambda: d(z, tv, ti, target=y, hard_weight=1.5), ValueError),
        (lambda: d(z, tv, ti, target=y, hard_weight=float("nan")), ValueError),
        (lambda: d(z, tv, ti, hard_weight=0.5), ValueError),
        (lambda: d(z, tv, ti, reduction="max"), ValueError),
        (lambda: d(z, tv.clone().requires_grad_(), ti), ValueError),
        (lambda: d(z, tv, ti, top_lse=lse.clone().requires_grad_()), ValueError),
        (lambda: d(z, tv.to("meta"), ti), ValueError),
        (lambda: d(torch.empty(3, 0), tv[:3], ti[:3]), ValueError),
    ]:
        with pytest.raises(err):
            bad()


@pytest.mark.parametrize("dev", DEVICES)
def test_forward_mode_derivatives(dev):
    """The teacher's side with a tangent is refused, top_logits' results carry none; the student's gives
    the right one (CPU path) or is refused."""
    z, tv, ti, y, lse = (t.to(dev) for t in make(4, 30, 3, torch.float32))
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for bad in (lambda: ops.distill_loss(z, dual(tv), ti), lambda: ops.distill_loss(z, tv, ti, top_lse=dual(lse))):
            with pytest.raises(ValueError, match="detach"):
                bad()
            with torch.no_grad(), pytest.raises(ValueError, match="detach"):
                bad()
        got = ops.top_logits(dual(z), 3)
        assert all(forward_ad.unpack_dual(t).tangent is None for t in (got.values, got.lse))
        d = torch.randn(4, 30, generator=torch.Generator().manual_seed(1)).to(dev)
        if dev == "cuda":
            with pytest.raises((RuntimeError, NotImplementedError)):
                ops.distill_loss(forward_ad.make_dual(z, d), tv, ti)
        else:
            slope = forward_ad.unpack_dual(ops.distill_loss(forward_ad.make_dual(z.double(), d.double()), tv, ti)).tangent
            _, _, grad, _, _ = oracle(z, tv, ti, None, None, 1.0, 0.0)
            assert abs(slope - (grad * d).sum() / 4) < 1e-12


@pytest.mark.parametrize("t", [0.0, -1.0, 1e-40, 1e-31, 1e31, float("inf"), float("nan")])
def test_temperatures_refused(t):
    z = torch.zeros(2, 5)
    with pytest.raises(ValueError, match="temperature"):
        ops.top_logits(z, 2, t)
    with pytest.raises(ValueError, match="temperature"):
        ops.distill_loss(z, z[:, :2], torch.zeros(2, 2, dtype=torch.int32), temperature=t)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("t", [1e-30, 1e-3, 1e6, 1e30])
def test_temperatures_far(dev, t):
    """Temperatures up to both ends: with a small one a row's largest class has everything (its bf16
    values differ by more than 100 t), with a large one every unmasked class has the same share."""
    z = torch.randperm(200, generator=torch.Generator().manual_seed(1)).reshape(2, 100).float()
    z[:, 7] = -math.inf
    tv, ti, lse = ops.top_logits(z.to(dev), 10, t)
    want = torch.logsumexp(z.double() / t, 1)
    # half steps: the maximum times 1 / t, both rounded, and the result; a sum of 100 terms of at most 1 (its
    # exponents are 0, below -1000, or below 2^-12, so they hardly round)
    assert bool(((lse.cpu().double() - want).abs() <= 4 * E * want.abs() + 100 * E).all())
    zs = z.to(dev).requires_grad_()
    loss = ops.distill_loss(zs, tv, ti, temperature=t, reduction="none")  # the student is the teacher
    g, = torch.autograd.grad(loss.sum() / t, zs)
    q = torch.softmax(z.double() / t, 1)
    p = torch.zeros_like(q).scatter_(1, ti.cpu().long(), torch.softmax(tv.cpu().double() / t, 1))
    assert bool(((g.cpu().double() - (q - p)).abs() <= 200 * E * (q + p)).all())


@pytest.mark.gpu
def test_refusals_native(cuda):
    """The native entries refuse sizes that their kernels do not take; other devices are refused."""
    from mxddp import native

    C = native()
    with pytest.raises(RuntimeError):
        C.top_logits(0, 0, 8, 2, 8, 9, 1.0, 0, 0, 0, 0, 0)
    with pytest.raises(RuntimeError):
        C.top_logits(0, 0, 400, 2, 400, 257, 1.0, 0, 0, 0, 0, 0)
    with pytest.raises(RuntimeError):
        C.top_logits(0, 5, 8, 2, 8, 2, 1.0, 0, 0, 0, 0, 0)
    with pytest.raises(RuntimeError):
        C.distill_fwd(0, 0, 0, 0, 0, 0, 8, 2, 8, 300, 0, 0, False, False, 1.0, 0.0, 0, 0, True, 0, 0)
    with pytest.raises(RuntimeError):
        C.distill_bwd(0, 0, 0, 0, 0, 0, 8, 2, 8, 3, 0, 0, False, False, 1.0, 0.5, 0, False, 0, 0)
    z, tv, ti, y, lse = make(4, 30, 3, torch.float32)
    with pytest.raises(ValueError):
        ops.distill_loss(z.to(cuda), tv.to(cuda), ti)
    with pytest.raises(TypeError):
        ops.distill_loss(z.double().to(cuda), tv.to(cuda), ti.to(cuda))


@pytest.mark.gpu
@pytest.mark.parametrize("tail", [False, True])
def test_distill_autograd(cuda, tail):
    """Backward twice, a loss scaled in place, bitwise the same again, no second derivative, logits
    changed in between refused."""
    z, tv, ti, y, lse = make(40, 3000, 20, torch.bfloat16, 14)
    leaf = z.to(cuda).requires_grad_()
    args = (tv.to(cuda), ti.to(cuda), y.to(cuda), lse.to(cuda) if tail else None, 2.0, 0.5)
    loss = ops.distill_loss(leaf, *args)
    g1, = torch.autograd.grad(loss, leaf, retain_graph=True)
    g2, = torch.autograd.grad(loss, leaf, retain_graph=True)
    loss2 = ops.distill_loss(leaf, *args)
    g3, = torch.autograd.grad(loss2, leaf)
    assert torch.equal(g1, g2) and torch.equal(g1, g3) and torch.equal(loss, loss2)
    scaled = ops.distill_loss(leaf, *args)
    scaled *= 4
    g4, = torch.autograd.grad(scaled, leaf)
    assert torch.equal(g4.float(), 4 * g1.float())  # a power of two; no value is near the type's ends
    loss = ops.distill_loss(leaf, *args)
    g5, = torch.autograd.grad(loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g5.sum().backward()
    mid = leaf * 1
    loss = ops.distill_loss(mid, *args)
    mid.mul_(2)
    with pytest.raises(RuntimeError):
        loss.backward()


@pytest.mark.gpu
def test_distill_graph(cuda):
    """Teacher's top logits, loss and gradient captured into two graphs that replay in turn, with new
    logits each time and eager calls in between.  No eager autograd graph of a leaf lives while its
    backward is captured: torch would join the stream of that graph's leaf node into the capture."""
    N, V, k = 16, 20000, 12
    z, tv, ti, y, lse = make(N, V, k, torch.bfloat16, 15)
    teacher = torch.randn(N, V, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(cuda)
    y = y.to(cuda)

    def step(leaf, teacher):
        tv, ti, lse = ops.top_logits(teacher, k, 2.0)
        loss = ops.distill_loss(leaf, tv, ti, y, lse, 2.0, 0.5)
        return loss.detach(), torch.autograd.grad(loss, leaf)[0]

    graphs = []
    for i in range(2):
        leaf, tin = z.to(cuda).requires_grad_(), teacher.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(leaf, tin)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(leaf, tin)
        graphs.append((g, leaf, tin, out))
    for i in range(3):
        for j, (g, leaf, tin, out) in enumerate(graphs):
            with torch.no_grad():
                leaf.copy_(z.to(cuda) * (1 + i + 2 * j))
            tin.copy_(teacher * (1 + j) + i)
            g.replay()
        for j, (g, leaf, tin, out) in enumerate(graphs):
            loss, grad = step(leaf, tin)
            assert torch.equal(out[0], loss) and torch.equal(out[1], grad), (i, j)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V", [(520, 140001), (2, 140001)])
def test_distill_loss_long_rows_high_temperature(cuda, dtype, N, V):
    """Above T = 8: rows longer than the classes whose marks are in LDS at a time, in one block each and split
    over blocks; each of the named classes holds a percent of the row, so one that is taken for the wrong
    side shows.  Both passes repeat bit by bit."""
    k, T = 40, 20.0
    g = torch.Generator().manual_seed(V)
    rows = [0, N - 1]
    ti = torch.randint(V, (N, k), generator=g)
    ti[rows, 0], ti[rows, 1] = V - 1, 65536
    few = (2 * torch.randn(2, V, generator=g)).scatter_(1, ti[rows], 150.0).to(dtype)
    tv = (torch.randn(N, k, generator=g) + 148).to(dtype)
    lse = torch.full((N,), 12.0)
    y = torch.full((N,), -100)
    y[rows] = torch.tensor([3, V - 1])
    z = torch.zeros(N, V, dtype=dtype, device=cuda)
    z[rows] = few.to(cuda)
    z.requires_grad_()
    out = []
    for _ in range(2):
        loss = ops.distill_loss(z, tv.to(cuda), ti.to(cuda), y.to(cuda), lse.to(cuda), T, 0.5, "none")
        out.append((loss.detach(), torch.autograd.grad(loss.sum(), z)[0][rows].cpu().double()))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    want, _, grad, _, _ = oracle(few, tv[rows], ti[rows], y[rows], lse[rows], T, 0.5)
    assert (want > 1).all()
    # sums in 64 bits; the labels' in fp32: es(V) of its logarithm
    assert bool(((out[0][0][rows].cpu().double() - want).abs() <= 4 * E * want + es(V)).all())
    assert N == 2 or not out[0][0][1:-1].any()
    tol = 64 * E * (grad.abs() + T / V) + es(V) * torch.softmax(few.double(), 1)
    tol = tol + torch.finfo(dtype).eps / 2 * 1.01 * (grad.abs() + tol) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert bool(((out[0][1] - grad).abs() <= tol).all())


@pytest.mark.gpu
def test_distill_graph_high_temperature(cuda):
    """Loss and gradient above T = 8 captured, with rows that are split over blocks, and replayed with new
    logits and eager calls in between."""
    z, tv, ti, y, lse = make(3, 20000, 12, torch.float16, 18, 30.0)
    tv, ti, y, lse = tv.to(cuda), ti.to(cuda), y.to(cuda), lse.to(cuda)

    def step(leaf):
        loss = ops.distill_loss(leaf, tv, ti, y, lse, 30.0, 0.5)
        return loss.detach(), torch.autograd.grad(loss, leaf)[0]

    leaf = z.to(cuda).requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(leaf)
    for i in range(3):
        with torch.no_grad():
            leaf.copy_(z.to(cuda) * (1 + i))
        graph.replay()
        loss, grad = step(leaf)
        assert torch.equal(out[0], loss) and torch.equal(out[1], grad), i


@pytest.mark.gpu
def test_distill_other_stream(cuda):
    z, tv, ti, y, lse = make(8, 5000, 9, torch.float32, 16)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        check_distill("cuda", z, tv, ti, y, lse, 2.0, 0.5)
        check_top(z, 9, ops.top_logits(z.to(cuda), 9))
    st.synchronize()


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    """Rows that start behind 2^32 elements: the last ones have the right answers."""
    N, V, k = 33000, 131071, 5
    z = torch.zeros(N, V, dtype=torch.bfloat16, device=cuda)
    g = torch.Generator().manual_seed(17)
    last = (3 * torch.randn(6, V, generator=g)).to(torch.bfloat16)
    z[-6:] = last.to(cuda)
    tv, ti, lse = ops.top_logits(z, k)
    check_top(last, k, (tv[-6:], ti[-6:], lse[-6:]))
    y = torch.full((N,), -1, device=cuda)
    y[-6:] = 7
    z.requires_grad_()
    loss = ops.distill_loss(z, tv, ti, y, lse, 1.0, 0.5, "sum")
    dz, = torch.autograd.grad(loss, z)
    del z
    assert not dz[:1000].any() and not dz[16384 - 100:16384 + 100].any()
    rows, _, grad, tl, tg = oracle(last, tv[-6:], ti[-6:], torch.full((6,), 7), lse[-6:], 1.0, 0.5)
    assert abs(loss.item() - rows.sum().item()) <= (tl.sum() + 3 * E * rows.abs().sum()).item()
    tol = tg + 2.0**-8 * (grad.abs() + tg) + 1e-40
    assert bool(((dz[-6:].cpu().double() - grad).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,N,V", [(torch.bfloat16, 2048, 65536), (torch.float32, 700, 98304), (torch.float16, 1500, 98368)])
def test_distill_large_gradient(cuda, dtype, N, V):
    """A gradient of more than 256 MB: the same bits as those of its rows taken in smaller calls, and its
    last rows against the formula."""
    k, T, h = 40, 2.0, 0.3
    g = torch.Generator(device=cuda).manual_seed(23)
    z = (3 * torch.randn(N, V, generator=g, device=cuda)).to(dtype)
    tv, ti, lse = ops.top_logits(3 * torch.randn(N, V, generator=g, device=cuda), k, T)
    y = torch.randint(V, (N,), generator=g, device=cuda)

    def gradient(a, b):
        zs = z[a:b].detach().requires_grad_()
        loss = ops.distill_loss(zs, tv[a:b], ti[a:b], y[a:b], lse[a:b], T, h, "sum")
        return torch.autograd.grad(loss, zs)[0]

    whole = gradient(0, N)
    for a in list(range(0, N - 512, 512)) + [N - 512]:  # 512 rows: a block to a row, as in the whole
        assert torch.equal(whole[a:a + 512], gradient(a, a + 512))
    _, _, grad, _, tg = oracle(z[-3:].cpu(), tv[-3:].cpu(), ti[-3:].cpu(), y[-3:].cpu(), lse[-3:].cpu(), T, h)
    fi = torch.finfo(dtype)
    tol = tg + 3 * E * grad.abs()
    tol = tol + fi.eps / 2 * (grad.abs() + tol) + fi.smallest_normal * fi.eps
    assert bool(((whole[-3:].cpu().double() - grad).abs() <= tol).all())


@pytest.mark.parametrize("dev", DEVICES)
def test_teacher_to_student(dev):
    """The operators together: a teacher with int8 layers answers, its top logits are kept, a student
    learns from them; loss and the student's gradients against the same chain in 64 bits."""
    torch.manual_seed(3)
    D, H, V, N, k, T, h = 48, 96, 200, 24, 8, 2.0, 0.25
    l1, l2 = Linear(D, H, fuse_relu=True).to(dev), Linear(H, V).to(dev)
    with torch.no_grad():
        l2.weight.mul_(6)
    t1, t2 = Int8Linear.from_linear(l1), Int8Linear.from_linear(l2)
    student = Linear(D, V).to(dev)
    x, y = torch.randn(N, D).to(dev), torch.randint(V, (N,)).to(dev)
    with torch.no_grad():
        answer = t2(t1(x))
        top = ops.top_logits(answer, k, T)
    check_top(answer.cpu(), k, top, T)
    logits = student(x)
    loss = ops.distill_loss(logits, top.values, top.index, y, top.lse, T, h)
    loss.backward()
    rows, counted, grad, tl, tg = oracle(logits, top.values, top.index, y, top.lse, T, h)
    assert int(counted.sum()) == N
    assert abs(loss.item() - rows.mean().item()) <= (tl.mean() + 4 * E * rows.abs().mean()).item()
    dw = (grad.t() / N) @ x.cpu().double()
    # logits' gradient as bounded, then N products and sums in fp32
    tol = ((tg + (N + 3) * 2 * E * grad.abs()).t() / N) @ x.cpu().double().abs()
    assert bool(((student.weight.grad.cpu().double() - dw).abs() <= tol).all())
