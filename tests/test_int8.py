"""8-bit linear layers (ops.quantize_rows, ops.linear_int8, layers.Int8Linear) against the
definition in 64 bits.

The quantised values have one right answer each (the exact quotient, rounded half to even), so they
are compared bit for bit.  A product's sum is a whole number; what is left are the roundings of the
epilogue: the sum to fp32, two scales, the bias, and the result's type, each by half a step.
"""
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from mxddp import ops
from mxddp.models.layers import Int8Linear, Linear

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]
E = 2.0**-24


def oracle_quantize(x):
    """q and scale of [M, K] in 64 bits on the CPU; the quotient's rounding by comparison."""
    x = x.detach().cpu().double()
    top = x.abs().amax(1)
    scale = torch.maximum(top / 127, torch.tensor(2.0**-126, dtype=torch.float64)).float()
    d = x / scale.double()[:, None]
    low = d.floor()
    up = (d - low > 0.5) | ((d - low == 0.5) & (low.remainder(2) == 1))
    return (low + up).to(torch.int8), scale


def oracle_linear(q, s, w, ws, bias, relu):
    prod = (q.cpu().double() @ w.cpu().double().t()) * s.cpu().double()[:, None] * ws.cpu().double()
    y = prod if bias is None else prod + bias.cpu().double()
    return (y.clamp_min(0) if relu else y), prod


def check_linear(y, q, s, w, ws, bias, relu):
    want, prod = oracle_linear(q, s, w, ws, bias, relu)
    # sum to fp32 and two scales: 3 half steps of the product; bias: one of the result
    b = 0 if bias is None else bias.cpu().double().abs()
    tol = 3.01 * E * prod.abs() + 1.01 * E * (prod.abs() + b) + torch.finfo(y.dtype).eps / 2 * 1.001 * want.abs()
    tol = tol + torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps  # a subnormal's step
    far = (y.detach().cpu().double() - want).abs()
    assert y.shape == want.shape
    assert bool((far <= tol).all()), f"off by {(far / tol).max().item():.2f} of the bound"


def make(M, N, K, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, K, generator=g) * torch.exp(torch.randn(K, generator=g))).to(dtype)
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)
    ws = torch.rand(N, generator=g) * 0.01 + 1e-4
    return x, w, ws, torch.randn(N, generator=g)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (5, 64), (2, 1000), (7, 4097), (300, 129), (2, 40000), (1, 131071)])
def test_quantize_rows(dev, dtype, M, K):
    x = make(M, 1, K, dtype, M + K)[0]
    q, s = ops.quantize_rows(x.to(dev))
    wq, ws = oracle_quantize(x)
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and q.shape == x.shape and s.shape == (M,)
    assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu(), wq)


@pytest.mark.parametrize("dev", DEVICES)
def test_quantize_rows_halves(dev):
    """Quotients at and next to a half, either sign: scale 2^e exactly (127 2^e is the maximum)."""
    for e in (-126, -30, 0, 20):
        n = torch.arange(-127, 127, dtype=torch.float64)
        near = torch.stack([n + 0.5, (n + 0.5) * (1 + 2.0**-23), (n + 0.5) * (1 - 2.0**-23)]).reshape(-1)
        x = torch.cat([near, torch.tensor([127.0], dtype=torch.float64)]).clamp(-127, 127) * 2.0**e
        x = x.float()[None]
        q, s = ops.quantize_rows(x.to(dev))
        wq, ws = oracle_quantize(x)
        assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu(), wq), e


@pytest.mark.parametrize("dev", DEVICES)
def test_quantize_rows_halves_of_small_scales(dev):
    """The numbers next to a half at scales just above 2^-126 with an odd last place: half of such a
    scale is no number of fp32.  A number x and a scale s are multiples of 2^-149, so a quotient
    misses a half by nothing or by at least 2^-149 / (2 s) >= 2^-25."""
    g = torch.Generator().manual_seed(6)
    s = ((2**23 + torch.cat([torch.arange(1, 40, 2), torch.randint(2**22, (300,), generator=g) * 2 + 1])).double()
         * 2.0**-149)
    n = torch.arange(-126, 126, dtype=torch.float64) + 0.5
    step = torch.tensor([-1.0, 0.0, 1.0], dtype=torch.float64) * 2.0**-149
    x = ((n[None, :, None] * s[:, None, None]).float().double() + step).reshape(len(s), -1)
    x = torch.cat([x, 127 * s[:, None]], 1).float()
    wq, ws = oracle_quantize(x)
    assert int((ws == s.float()).sum()) > 300  # the rows' largest magnitudes give these scales
    q, sc = ops.quantize_rows(x.to(dev))
    assert torch.equal(sc.cpu(), ws) and torch.equal(q.cpu(), wq)
    # the product's own quantisation: y = q * scale * 2^126, rounded once, through a weight row of a single 1
    w = torch.zeros(1, x.shape[1], dtype=torch.int8)
    w[0, 7] = 1
    y = ops.linear_int8(x[:8].to(dev), w.to(dev), torch.full((1,), 2.0**126, device=dev))
    assert torch.equal(y.cpu()[:, 0], (wq[:8, 7].double() * ws[:8].double() * 2.0**126).float())


@pytest.mark.parametrize("dev", DEVICES)
def test_quantize_rows_values(dev):
    """Rows of zeros, subnormals, the largest numbers, and rows that are not finite."""
    big = torch.finfo(torch.float32).max
    x = torch.tensor([[0.0, -0.0, 0.0], [1e-44, -3e-45, 0.0], [big, -big, 1.0], [1.0, float("inf"), 2.0],
                      [float("nan"), 1.0, 0.0], [1.0, -float("inf"), float("nan")], [2.0, -1.0, 0.5]])
    q, s = ops.quantize_rows(x.to(dev))
    q, s = q.cpu(), s.cpu()
    fine = [0, 1, 2, 6]
    wq, ws = oracle_quantize(x[fine])
    assert torch.equal(q[fine], wq) and torch.equal(s[fine], ws)
    assert torch.isnan(s[[3, 4, 5]]).all() and (q[[3, 4, 5]] == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_quantize_rows_shapes(dev):
    x = torch.randn(2, 3, 50, generator=torch.Generator().manual_seed(0))
    want_q, want_s = oracle_quantize(x.reshape(6, 50))
    wide = torch.zeros(6, 77, device=dev)
    wide[:, 5:55] = x.reshape(6, 50).to(dev)
    for v in (x.to(dev), x.to(dev).transpose(0, 1).contiguous().transpose(0, 1),
              wide[:, 5:55].reshape(2, 3, 50), x.to(dev).permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        q, s = ops.quantize_rows(v)
        assert q.shape == (2, 3, 50) and s.shape == (2, 3)
        assert torch.equal(q.cpu().reshape(6, 50), want_q) and torch.equal(s.cpu().reshape(6), want_s)
    q, s = ops.quantize_rows(wide[:, 5:55])
    assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)
    q, s = ops.quantize_rows(x[0, 0].to(dev))
    assert torch.equal(q.cpu(), want_q[0]) and s.shape == () and s.item() == want_s[0].item()
    q, s = ops.quantize_rows(torch.empty(0, 9, device=dev))
    assert q.shape == (0, 9) and s.shape == (0,)


SIZES = [  # M, N, K: one token and few, rows of 16 bytes or not, tile edges, many tiles
    (1, 1, 1), (1, 10, 64), (1, 1000, 2048), (1, 4096, 512), (1, 513, 1001), (2, 100, 77), (3, 33, 4096),
    (8, 640, 256), (15, 257, 100), (16, 256, 1024), (17, 130, 1000), (31, 96, 784), (33, 1000, 1000), (63, 65, 127),
    (64, 64, 64), (65, 129, 66), (100, 300, 300), (128, 128, 128), (129, 257, 208), (250, 1000, 2048),
    (256, 256, 256), (257, 255, 1040), (300, 512, 48), (511, 513, 500), (1024, 1000, 16), (1500, 700, 136),
]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear_int8(dev, M, N, K):
    dtype = TYPES[(M + N) % 3]
    x, w, ws, b = make(M, N, K, dtype, M * 7 + N)
    q, s = oracle_quantize(x)
    args = (x.to(dev), w.to(dev), ws.to(dev))
    check_linear(ops.linear_int8(*args), q, s, w, ws, None, False)
    check_linear(ops.linear_int8(*args, b.to(dev), relu=True), q, s, w, ws, b, True)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(2309, 4100), (3999, 4050), (1000, 4000), (1100, 4100), (520, 3970), (20, 8200), (9, 8197)])
@pytest.mark.parametrize("K", [7, 16, 112, 128, 144, 250, 256, 384, 520, 640, 1008])
def test_linear_int8_tiles(cuda, M, N, K):
    """Every tile kernel (their choice goes by rounds over the machine), one stage of k to eight, k that
    ends in a stage, in a piece, and rows of no alignment; the oracle's product in 64 bits is exact."""
    g = torch.Generator(device=cuda).manual_seed(M + K)
    q = torch.randint(-127, 128, (M, K), generator=g, dtype=torch.int8, device=cuda)
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8, device=cuda)
    s, ws = torch.rand(M, generator=g, device=cuda), torch.rand(N, generator=g, device=cuda) * 1e-3
    b = torch.randn(N, generator=g, device=cuda)
    prod = (q.double() @ w.double().t().contiguous()) * s.double()[:, None] * ws.double()
    want = prod + b.double()
    y = ops.linear_int8(q, w, ws, b, x_scale=s)
    tol = 4.02 * E * prod.abs() + 1.01 * E * (b.double().abs() + want.abs())
    assert bool(((y.double() - want).abs() <= tol).all())
    # float tokens whose quantised values these are: rows of 127 at some place, a scale of 2^-7
    x = q.float()
    x[:, K // 2] = 127
    prod = (x.double() @ w.double().t().contiguous()) * 2.0**-7 * ws.double()
    y = ops.linear_int8((x * 2.0**-7).to(torch.bfloat16), w, ws, b, out_dtype=torch.float32)
    want = prod + b.double()
    tol = 4.02 * E * prod.abs() + 1.01 * E * (b.double().abs() + want.abs())
    assert bool(((y.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("M", range(1, 18))
@pytest.mark.parametrize("K", [9, 64, 961, 1000, 2040])
def test_linear_int8_few_tokens(dev, M, K):
    """Every number of tokens up to 17 of a float type, rows of different sizes of values, one of zeros and
    one that is not finite."""
    dtype = TYPES[M % 3]
    x, w, ws, b = make(M, 70, K, dtype, M * 31 + K)
    x = x * torch.logspace(-2, 2, M).to(dtype)[:, None]
    x[M // 2] = 0
    bad = M - 1 if M > 2 else -1
    q, s = oracle_quantize(x)
    if bad > 0:
        x[bad, K // 2] = math.inf
    y = ops.linear_int8(x.to(dev), w.to(dev), ws.to(dev), b.to(dev), out_dtype=torch.float32 if K == 64 else None)
    good = [m for m in range(M) if m != bad]
    check_linear(y[good], q[good], s[good], w, ws, b, False)
    assert bad < 0 or bool(torch.isnan(y[bad]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("M", [17, 24, 32])
@pytest.mark.parametrize("N,K", [(16384, 128), (16400, 520), (16385, 1001), (20001, 64), (16384, 16), (16399, 7), (32000, 1100)])
def test_linear_int8_wide(cuda, M, N, K):
    """Few tokens of very wide layers."""
    g = torch.Generator(device=cuda).manual_seed(M + N)
    q = torch.randint(-127, 128, (M, K), generator=g, dtype=torch.int8, device=cuda)
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8, device=cuda)
    s, ws = torch.rand(M, generator=g, device=cuda), torch.rand(N, generator=g, device=cuda) * 1e-3
    prod = (q.double() @ w.double().t().contiguous()) * s.double()[:, None] * ws.double()
    y = ops.linear_int8(q, w, ws, x_scale=s)
    assert bool(((y.double() - prod).abs() <= 4.02 * E * prod.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("off,ld,K", [(1, 1008, 1001), (3, 1002, 1000), (2, 130, 130), (5, 77, 70), (1, 16, 16),
                                      (4, 524, 516), (7, 4100, 4099), (15, 5001, 5000)])
@pytest.mark.parametrize("M,N", [(1, 300), (3, 8200), (12, 8200), (20, 333), (24, 8200), (100, 200), (700, 530)])
def test_linear_int8_views(cuda, off, ld, K, M, N):
    """Weights and int8 tokens that begin at any address, rows of any stride, storage that ends with the
    last row; tokens of a float type as well."""
    g = torch.Generator(device=cuda).manual_seed(off + M)

    def view(rows):
        flat = torch.randint(-127, 128, (off + (rows - 1) * ld + K,), generator=g, dtype=torch.int8, device=cuda)
        return flat.as_strided((rows, K), (ld, 1), off)

    w, q = view(N), view(M)
    s, ws = torch.rand(M, generator=g, device=cuda), torch.rand(N, generator=g, device=cuda) * 1e-3
    prod = (q.double() @ w.double().t().contiguous()) * s.double()[:, None] * ws.double()
    y = ops.linear_int8(q, w, ws, x_scale=s)
    assert bool(((y.double() - prod).abs() <= 4.02 * E * prod.abs()).all())
    x = q.float()
    x[:, K // 3] = -127
    prod = (x.double() @ w.double().t().contiguous()) * 2.0**-5 * ws.double()
    y = ops.linear_int8((x * 2.0**-5).to(torch.float16), w, ws, out_dtype=torch.float16).double()
    tol = 3.01 * E * prod.abs() + 2.0**-11 * 1.001 * prod.abs() + 2.0**-25
    assert bool(((y - prod).abs() <= tol).all())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("M,N,K", [(1, 300, 1024), (5, 77, 96), (5, 77, 99), (70, 200, 1000), (300, 300, 512)])
@pytest.mark.parametrize("out", TYPES)
def test_linear_int8_given(dev, M, N, K, out):
    """An int8 input with its scales, all 256 values on both sides (a weight may hold -128)."""
    g = torch.Generator().manual_seed(K)
    q = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8)
    s, ws = torch.rand(M, generator=g), torch.rand(N, generator=g) * 1e-3
    y = ops.linear_int8(q.to(dev), w.to(dev), ws.to(dev), x_scale=s.to(dev), out_dtype=out)
    assert y.dtype == out
    check_linear(y, q, s, w, ws, None, False)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("M", [1, 20, 200])
def test_linear_int8_largest_sums(dev, M):
    """Every product 2^14 over the longest rows: the sum is just below 2^31."""
    K, N = ops.int8.MAX_K, 20
    q = torch.full((M, K), -128, dtype=torch.int8, device=dev)
    w = torch.full((N, K), -128, dtype=torch.int8, device=dev)
    y = ops.linear_int8(q, w, torch.ones(N, device=dev), x_scale=torch.ones(M, device=dev))
    assert bool((y.double() == float(torch.tensor(K * 2**14, dtype=torch.float64).float())).all())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("M", [1, 6, 150])
def test_linear_int8_strides(dev, M):
    """Rows with other strides and starts: slices of wider tensors, a weight whose rows are padded."""
    N, K = 140, 112
    x, w, ws, b = make(M, N, K, torch.bfloat16)
    q, s = oracle_quantize(x)
    for off, pad in ((0, 16), (16, 48), (3, 5), (8, 8), (1, 15)):
        wide = torch.full((N, K + off + pad), 99, dtype=torch.int8, device=dev)
        wv = wide[:, off:off + K]
        wv.copy_(w)
        xw = torch.full((M, K + off + pad), float("nan"), dtype=x.dtype, device=dev)
        xv = xw[:, off:off + K]
        xv.copy_(x)
        check_linear(ops.linear_int8(xv, wv, ws.to(dev), b.to(dev)), q, s, w, ws, b, False)
        qw = torch.full((M, K + off + pad), 77, dtype=torch.int8, device=dev)
        qv = qw[:, off:off + K]
        qv.copy_(q)
        y = ops.linear_int8(qv, wv, ws.to(dev), b.to(dev), x_scale=s.to(dev))
        check_linear(y, q, s, w, ws, b, False)
    far = torch.zeros(N, 2**22 + 16, dtype=torch.int8, device=dev)[:, :K]  # rows further apart than a tile's offsets
    far.copy_(w)
    check_linear(ops.linear_int8(x.to(dev), far, ws.to(dev)), q, s, w, ws, None, False)
    # the weight's rows stored column by column; an input of more dimensions; every second scale
    wt = w.to(dev).t().contiguous().t()
    ws2 = torch.stack([ws, ws + 1], 1).to(dev)[:, 0]
    y = ops.linear_int8(x.to(dev)[None, :, None], wt, ws2, b.to(dev))
    assert y.shape == (1, M, 1, N)
    check_linear(y[0, :, 0], q, s, w, ws, b, False)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("M", [1, 40, 200])
def test_linear_int8_padded_tail(dev, M):
    """A weight whose padded rows end with the tensor's own memory, what lies there arbitrary."""
    N, K = 50, 1001
    x, w, ws, b = make(M, N, K, torch.float32)
    q, s = oracle_quantize(x)
    wide = torch.full((N, 1008), 127, dtype=torch.int8, device=dev)
    wide[:, :K] = w.to(dev)
    check_linear(ops.linear_int8(x.to(dev), wide[:, :K], ws.to(dev)), q, s, w, ws, None, False)
    flat = torch.full((N * 1008 - 7,), 127, dtype=torch.int8, device=dev)  # the last row ends at K
    view = flat.as_strided((N, K), (1008, 1))
    view.copy_(w)
    check_linear(ops.linear_int8(x.to(dev), view, ws.to(dev)), q, s, w, ws, None, False)


@pytest.mark.parametrize("dev", DEVICES)
def test_linear_int8_values(dev):
    """No tokens; a row that is not finite gives NaN there and nowhere else; a ReLU keeps NaN."""
    x, w, ws, b = make(40, 24, 64, torch.float32)
    y = ops.linear_int8(x[:0].to(dev), w.to(dev), ws.to(dev))
    assert y.shape == (0, 24)
    q, s = oracle_quantize(x)
    bad = x.clone()
    bad[3, 5] = float("inf")
    bad[17, 0] = float("nan")
    for relu in (False, True):
        y = ops.linear_int8(bad.to(dev), w.to(dev), ws.to(dev), b.to(dev), relu=relu).cpu()
        keep = [i for i in range(40) if i not in (3, 17)]
        assert torch.isnan(y[[3, 17]]).all()
        check_linear(y[keep], q[keep], s[keep], w, ws, b, relu)
    # scales whose product leaves fp32's range, with a sum of zero
    y = ops.linear_int8(torch.zeros(2, 64, dtype=torch.int8, device=dev), w.to(dev), torch.full((24,), 1e30, device=dev),
                        x_scale=torch.full((2,), 1e30, device=dev))
    assert (y == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("M", [1, 24, 70, 600])
def test_linear_int8_far_scales(dev, M):
    """Tokens of very large or very small values beside channel scales that bring the result back:
    no step of the epilogue leaves fp32's range where the result does not."""
    N, K = 130, 64
    x, w, _, b = make(M, N, K, torch.float32, M)
    x = x / x.abs().amax(1, keepdim=True)
    for top, scale, bias in ((1e37, 1e-8, 1e30), (3e38, 1e-30, 1.0), (1.0, 1e30, 1e30), (1e38, 1e-5, 1e38)):
        xt, ws, bt = x * top, (torch.rand(N, generator=torch.Generator().manual_seed(1)) + 0.5) * scale, b * bias
        q, s = oracle_quantize(xt)
        assert bool(torch.isfinite(oracle_linear(q, s, w, ws, bt, False)[0].float()).all())
        check_linear(ops.linear_int8(xt.to(dev), w.to(dev), ws.to(dev), bt.to(dev)), q, s, w, ws, bt, False)
        check_linear(ops.linear_int8(xt.to(dev), w.to(dev), ws.to(dev), relu=True), q, s, w, ws, None, True)
    # scales that are given: subnormal ones, the largest, zero and a negative one
    q = torch.randint(-127, 128, (M, K), generator=torch.Generator().manual_seed(2), dtype=torch.int8)
    for xs, scale in ((3e-42, 1e30), (3e38, 1e-10), (0.0, 1e30), (-3e37, 1e-10)):
        s = torch.full((M,), xs)
        s[::2] = 0.25  # tokens of ordinary scales beside them
        ws = torch.full((N,), scale)
        y = ops.linear_int8(q.to(dev), w.to(dev), ws.to(dev), b.to(dev), x_scale=s.to(dev))
        check_linear(y, q, s, w, ws, b, False)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("K", [1, 100, 4096])
def test_linear_int8_one_row_of_a_wide_tensor(dev, K):
    """A single row keeps the stride of the tensor it was cut from, however large: the last token of a
    sequence, a weight of one output channel, both."""
    T = (2**22 + K) // K + 1  # rows of T K > 2^22 elements
    g = torch.Generator().manual_seed(K)
    q = torch.randint(-127, 128, (1, T, K), generator=g, dtype=torch.int8)
    s = torch.rand(1, T, generator=g)
    w = torch.randint(-127, 128, (70, K), generator=g, dtype=torch.int8)
    ws = torch.rand(70, generator=g) * 1e-3
    qd, sd, wd, wsd = (t.to(dev) for t in (q, s, w, ws))
    y = ops.linear_int8(qd[:, -1], wd, wsd, x_scale=sd[:, -1])
    check_linear(y, q[:, -1], s[:, -1], w, ws, None, False)
    one = qd.reshape(1, T * K)[:, 3 * K:4 * K]  # the same for a weight
    y = ops.linear_int8(wd, one, wsd[:1], x_scale=wsd)
    check_linear(y, w, ws, one.cpu(), ws[:1], None, False)
    y = ops.linear_int8(qd[:, -2], one, wsd[:1], x_scale=sd[:, -2])
    check_linear(y, q[:, -2], s[:, -2], one.cpu(), ws[:1], None, False)
    x = qd.float()[:, -1]
    xq, xs = oracle_quantize(x)
    check_linear(ops.linear_int8(x, one, wsd[:1]), xq, xs, one.cpu(), ws[:1], None, False)
    gq, gs = ops.quantize_rows(x)
    assert torch.equal(gq.cpu(), xq) and torch.equal(gs.cpu(), xs)


def test_refusals():
    x, w, ws, b = make(4, 6, 8, torch.float32)
    for bad, err in [
        (lambda: ops.quantize_rows(x.double()), TypeError),
        (lambda: ops.quantize_rows(torch.tensor(1.0)), ValueError),
        (lambda: ops.quantize_rows(torch.empty(3, 0)), ValueError),
        (lambda: ops.linear_int8(x, w.float(), ws), TypeError),
        (lambda: ops.linear_int8(x.double(), w, ws), TypeError),
        (lambda: ops.linear_int8(x[:, :7], w, ws), ValueError),
        (lambda: ops.linear_int8(x, w[0], ws), ValueError),
        (lambda: ops.linear_int8(x, w, ws[:5]), ValueError),
        (lambda: ops.linear_int8(x, w, ws.double()), ValueError),
        (lambda: ops.linear_int8(x, w, ws, b.half()), ValueError),
        (lambda: ops.linear_int8(x, w, ws, b[:, None]), ValueError),
        (lambda: ops.linear_int8(x, w, ws, x_scale=torch.ones(4)), ValueError),
        (lambda: ops.linear_int8(x.to(torch.int8), w, ws), ValueError),
        (lambda: ops.linear_int8(x.to(torch.int8), w, ws, x_scale=torch.ones(3)), ValueError),
        (lambda: ops.linear_int8(x.to(torch.int8), w, ws, x_scale=torch.ones(4).double()), ValueError),
        (lambda: ops.linear_int8(x, w, ws, out_dtype=torch.int8), TypeError),
        (lambda: ops.linear_int8(x.clone().requires_grad_(), w, ws), RuntimeError),
        (lambda: ops.linear_int8(x, w, ws, b.clone().requires_grad_()), RuntimeError),
        (lambda: ops.linear_int8(x, w, ws.clone().requires_grad_()), RuntimeError),
        (lambda: ops.linear_int8(torch.zeros(1, 2**17), torch.zeros(2, 2**17, dtype=torch.int8), ws[:2]), ValueError),
        (lambda: ops.linear_int8(x, w, ws.to("meta")), ValueError),
    ]:
        with pytest.raises(err):
            bad()
    with torch.no_grad():
        ops.linear_int8(x.clone().requires_grad_(), w, ws)


def test_refusals_of_lengths():
    """Rows and layers whose ends the kernels' 32-bit places do not reach, on either device; the native
    entries refuse them before anything is launched."""
    from mxddp import native

    C = native()
    one = torch.zeros(1, 1, dtype=torch.bfloat16)
    for n in (2**30 + 1, 2**31 - 1, 2**31, 2**32 + 5):
        with pytest.raises(ValueError, match=r"2\^30"):
            ops.quantize_rows(one.expand(1, n))
        with pytest.raises(ValueError, match=r"2\^30"):
            ops.linear_int8(one, one.to(torch.int8).expand(n, 1), torch.ones(1).expand(n))
    for n in (2**30 + 1, 2**31 - 1):
        with pytest.raises(RuntimeError, match="bad sizes"):
            C.quantize_rows(0, 1, n, 0, n, 0, 1, n, 0)
        with pytest.raises(RuntimeError, match="bad sizes"):
            C.linear_int8(0, 16, 16, 0, 0, 16, 16, 0, 0, 0, 0, 1, n, 16, False, 0)
        with pytest.raises(RuntimeError, match="bad sizes"):
            C.linear_int8_float(0, 1, 16, 0, 16, 16, 0, 0, 0, 1, 1, n, 16, False, 0, 0)


@pytest.mark.gpu
def test_refusals_native(cuda):
    """The native entries refuse sizes that their kernels do not take."""
    from mxddp import native

    C = native()
    with pytest.raises(RuntimeError):
        C.linear_int8(0, 16, 16, 0, 0, 16, 16, 0, 0, 0, 0, 4, 4, 2**17, False, 0)
    with pytest.raises(RuntimeError):
        C.linear_int8(0, 16, 16, 0, 0, 16, 16, 0, 0, 0, 0, 4, 0, 16, False, 0)
    with pytest.raises(RuntimeError):
        C.quantize_rows(0, 0, 16, 0, 8, 0, 4, 16, 0)
    with pytest.raises(RuntimeError):
        C.quantize_rows(0, 3, 16, 0, 16, 0, 4, 16, 0)
    x = torch.randn(2, 8, device=cuda)
    with pytest.raises(ValueError):
        ops.linear_int8(x, torch.zeros(3, 8, dtype=torch.int8), torch.ones(3))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 24, 300])
def test_linear_int8_stream_and_graph(cuda, M):
    """On another stream, and captured: two graphs that replay in turn with new inputs."""
    N, K = 200, 520
    x, w, ws, b = make(M, N, K, torch.bfloat16)
    xg, wg, wsg, bg = (t.to(cuda) for t in (x, w, ws, b))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        y = ops.linear_int8(xg, wg, wsg, bg)
    st.synchronize()
    q, s = oracle_quantize(x)
    check_linear(y, q, s, w, ws, b, False)
    graphs = []
    for _ in range(2):
        xin = xg.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.linear_int8(xin, wg, wsg, bg)
        graphs.append((g, xin, out))
    for i in range(3):
        for j, (g, xin, out) in enumerate(graphs):
            xin.copy_(xg * (1 + i + 3 * j))
            g.replay()
        for j, (g, xin, out) in enumerate(graphs):
            assert torch.equal(out, ops.linear_int8(xin, wg, wsg, bg)), (i, j)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("bias,relu,K", [(True, True, 100), (False, False, 64), (True, False, 33)])
def test_int8_linear_layer(dev, bias, relu, K):
    """Int8Linear.from_linear: the layer's weight in int8, its outputs those of ops.linear_int8."""
    torch.manual_seed(0)
    lin = Linear(K, 30, bias=bias, fuse_relu=relu).to(dev)
    lay = Int8Linear.from_linear(lin)
    wq, ws = oracle_quantize(lin.weight)
    assert torch.equal(lay.weight[:, :K].cpu(), wq) and torch.equal(lay.weight_scale.cpu(), ws)
    x = torch.randn(5, 2, K)
    q, s = oracle_quantize(x.reshape(10, K))
    with torch.no_grad():
        y = lay(x.to(dev))
    b = lin.bias.detach().cpu() if bias else None
    check_linear(y.reshape(10, 30), q, s, wq, ws, b, relu)
    other = Int8Linear(K, 30, bias=bias, fuse_relu=relu).to(dev)
    other.load_state_dict(lay.state_dict())
    with torch.no_grad():
        assert torch.equal(other(x.to(dev)), y)
    assert sum(p.numel() for p in lay.parameters()) == 0


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("cast", ["half", "bfloat16", "double", "to", "type", "to_device"])
def test_int8_linear_layer_casts(dev, cast):
    """A whole model cast to another type, its 8-bit layers in it: they keep their bits and take inputs of
    the type; casting back and forth changes nothing; a move to a device goes through."""
    torch.manual_seed(1)
    lin = Linear(40, 30, fuse_relu=True)
    model = torch.nn.Sequential(Int8Linear.from_linear(lin), torch.nn.Identity(), Int8Linear.from_linear(Linear(30, 7)))
    want = {k: v.clone() for k, v in model.state_dict().items()}
    to = {"half": lambda m: m.half(), "bfloat16": lambda m: m.bfloat16(), "double": lambda m: m.double(),
          "to": lambda m: m.to(torch.float16), "type": lambda m: m.type(torch.bfloat16),
          "to_device": lambda m: m.to(dev, torch.bfloat16)}[cast]
    assert to(model) is model
    model.to(dev)
    for _ in range(2):
        got = model.state_dict()
        assert list(got) == list(want)
        for k, v in got.items():
            assert v.device.type == dev and v.dtype == want[k].dtype and torch.equal(v.cpu(), want[k]), k
        model.half().float()
    for dtype in TYPES:
        x = torch.randn(6, 40, generator=torch.Generator().manual_seed(2)).to(dtype)
        y = model[0](x.to(dev))
        assert y.dtype == dtype
        q, s = oracle_quantize(x)
        check_linear(y, q, s, want["0.weight"][:, :40], want["0.weight_scale"], want["0.bias"], True)
        assert model(x.to(dev)).dtype == dtype
    assert Int8Linear(5, 3, bias=False).half().bias is None
    empty = Int8Linear(5, 3).to("meta").half().to_empty(device=dev)
    assert empty.weight_scale.dtype == torch.float32 and empty.weight.device.type == dev


@pytest.mark.parametrize("dev", DEVICES)
def test_forward_mode_derivatives(dev):
    """linear_int8 refuses every input with a tangent (under no_grad too, which leaves forward mode on);
    quantize_rows' results carry none."""
    x, w, ws, b = (t.to(dev) for t in make(4, 6, 8, torch.float32))
    q, s = ops.quantize_rows(x)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for bad in (lambda: ops.linear_int8(dual(x), w, ws), lambda: ops.linear_int8(x, w, dual(ws)),
                    lambda: ops.linear_int8(x, w, ws, dual(b)), lambda: ops.linear_int8(q, w, ws, x_scale=dual(s))):
            with pytest.raises(RuntimeError, match="tangent"):
                bad()
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                bad()
        gq, gs = ops.quantize_rows(dual(x))
        assert forward_ad.unpack_dual(gs).tangent is None and torch.equal(gq, q) and torch.equal(gs, s)
        y = ops.linear_int8(x, w, ws, b)
    assert torch.equal(y, ops.linear_int8(x, w, ws, b))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda v: ops.linear_int8(v, w, ws), (x,), (x,))
