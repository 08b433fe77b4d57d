"""8-bit products where every bit is known, and fp32 results to fp32 accuracy.

Known operands.  Entries +-2^e with one e (-1, 0 or 1) for each row and block of 128: every block quantises exactly, products within a
block have one exponent, so the matrix unit's groups lose nothing, and sums are multiples of 1/4 below 4 K < 2^22: exact in fp32
in any order.  A term left out, taken twice or with a neighbour's scale shows in torch.equal.

fp32 results.  Their products are exact, the matrix unit adds eight neighbours with 25 bits below the largest, cutting each (an
error under 7 * 2^-25 of the largest), and groups and accumulator in fp32: K / 8 + 16 additions and a few for joined parts, bias
and alpha.  (1) Element by element those errors add up to less than 7 * 2^-25 * sum of the groups' largest + n 2^-24 sum |a||b|.
(2) Roundings are independent of each other and of the signs here, so over a whole result their squares add up: each is at most
2^-24 of a partial sum, partial sums grow like a random walk to w = sqrt(sum a^2 b^2), hence an error of sqrt(n) 2^-24 |w| at most,
a factor of two above what uniform roundings give; the squares of the groups' largest products add up to |w|^2 at most, and their
cuts so to 7 * 2^-25 |w|."""
import pytest
import torch

from tests.fp8_util import quantise
from tests.test_fp8_gpu import SHAPES, _matrix

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _ops():
    from celligner2_amd import ops
    return ops


def _signs(R, C, seed, rows=1):
    """+-2^e, one e for `rows` rows and 128 columns, fp32 on the device."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    e = torch.randint(-1, 2, (-(-R // rows), -(-C // 128)), generator=g, device=DEV).float()
    e = e.repeat_interleave(rows, 0)[:R].repeat_interleave(128, 1)[:, :C]
    return (torch.randint(0, 2, (R, C), generator=g, device=DEV).float() * 2 - 1) * torch.exp2(e)


def _exact(a, b):
    return torch.mm(a.double(), b.double().t().contiguous())


def _same(y, ref):
    want = ref.to(torch.float32).to(y.dtype)
    assert torch.equal(y, want), (y.dtype, (y != want).sum().item(), (y != want).nonzero()[0].tolist())


@pytest.mark.parametrize("M,N,K", SHAPES + [(64, 300, 70000), (128, 256, 19000), (100, 300, 12000), (300, 19001, 130)])
def test_every_term_counts_once(M, N, K):
    ops = _ops()
    x, w, w1 = _signs(M, K, M + K), _signs(N, K, N + K, 128), _signs(N, K, N + K + 1)
    bias = torch.randint(-9, 10, (N,), device=DEV).float()
    alpha = torch.tensor([0.5], device=DEV)
    ref, ref1 = _exact(x, w), _exact(x, w1)
    wq, w1q, xq, x5 = ops.quant_fp8(w, block_rows=128), ops.quant_fp8(w1), ops.quant_fp8(x), ops.quant_fp8(x, fmt="e5m2")
    for dt in DT.values():
        _same(ops.linear_fwd_fp8(x, wq, bias=bias, out_dtype=dt), ref + bias.double())
        _same(ops.linear_fwd_fp8(x.bfloat16(), w1q, out_dtype=dt), ref1)
        _same(ops.linear_fwd_fp8(xq, wq, out_dtype=dt), ref)
        _same(ops.linear_dgrad_fp8(x5, w1q, alpha=alpha, out_dtype=dt), ref1 * 0.5)


# How these are cut for 16-bit results: 256 x 256 tiles in four parts of the reduction; whole rounds of them for 16 384 columns and
# the rest in three parts; whole rounds and a rest that is not cut, ragged at every edge; 256 x 256 tiles alone.  `floats`: the
# workspace of that cut (fp32 results take fewer parts here), so that another cut shows.
@pytest.mark.parametrize("M,N,K,floats", [(1024, 4096, 8192, 4 * 1024 * 4096), (1024, 19000, 4096, 3 * 1024 * 2616),
                                          (777, 19001, 820, None), (4096, 4096, 300, 0)])
def test_large_cuts(M, N, K, floats):
    ops = _ops()
    if floats is not None:
        assert ops.linear_fp8_ws(M, N, K) == floats
    x, w = _signs(M, K, 1), _signs(N, K, 2)
    ref = _exact(x, w)
    bias = torch.randint(-9, 10, (N,), device=DEV).float()
    alpha = torch.tensor([0.25], device=DEV)
    wq = ops.quant_fp8(w)
    for dt in (torch.bfloat16, torch.float32, torch.float16):
        _same(ops.linear_fwd_fp8(ops.quant_fp8(x), wq, bias=bias, out_dtype=dt), ref + bias.double())
        for fmt in ("e4m3", "e5m2"):
            _same(ops.linear_dgrad_fp8(ops.quant_fp8(x, fmt=fmt), wq, alpha=alpha, out_dtype=dt), ref * 0.25)


def _fp32_result(y, a, b, extra=None):
    """y (fp32) against a b^T + extra in 64 bits; a, b fp64 on the CPU."""
    a, b, y = a.to(DEV), b.to(DEV), y.double()
    K = a.shape[1]
    n = K / 8 + 24
    ref = _exact(a, b) if extra is None else _exact(a, b) + extra.double()
    pad = torch.nn.functional.pad
    a8, b8 = pad(a.abs(), (0, -K % 8)).view(a.shape[0], -1, 8).amax(2), pad(b.abs(), (0, -K % 8)).view(b.shape[0], -1, 8).amax(2)
    err = (y - ref).abs()
    mag = _exact(a.abs(), b.abs()) + (0 if extra is None else extra.double().abs())
    lim = _exact(a8, b8) * 7 * 2.0 ** -25 + mag * n * 2.0 ** -24 + 1e-38
    assert (err <= lim).all(), (err / lim).max().item()
    walk = (_exact(a * a, b * b) + (0 if extra is None else extra.double() ** 2)).sqrt()
    assert err.norm() <= ((n ** 0.5) * 2.0 ** -24 + 7 * 2.0 ** -25) * walk.norm() + 1e-38, (err.norm() / walk.norm()).item()


@pytest.mark.parametrize("M,N,K", SHAPES + [(128, 256, 19000), (777, 820, 9001), (64, 300, 70000), (300, 515, 40000)])
def test_fp32_results_are_fp32(M, N, K):
    ops = _ops()
    x, xd = _matrix(M, K, "f32", M + N + K, 3)
    w, wd = _matrix(N, K, "f32", M * N + K)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(5)).to(DEV)
    wq = ops.quant_fp8(wd, block_rows=128)
    a, b = quantise(x)[0], quantise(w, 128)[0]
    y = ops.linear_fwd_fp8(xd, wq, out_dtype=torch.float32)
    _fp32_result(y, a, b)
    _fp32_result(ops.linear_fwd_fp8(xd, wq, bias=bias, out_dtype=torch.float32), a, b, bias)
    assert torch.equal(ops.linear_fwd_fp8(ops.quant_fp8(xd), wq, out_dtype=torch.float32), y)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("M,N,K", [(5, 130, 66), (130, 257, 129), (777, 82, 515), (1500, 300, 900)])
def test_fp32_gradients_are_fp32(M, N, K, fmt):
    """The weight gradient in its default type and the input gradient in fp32, against the formulas and as derivatives of <dy, y>:
    <gradient, step> is the difference of the 64-bit <dy, y> over that step (y is linear in x and in w)."""
    ops = _ops()
    x, xd = _matrix(M, K, "f32", 1, 1)
    w, wd = _matrix(N, K, "f32", 2, spread=0.5)
    dy, dyd = _matrix(M, N, "bf16", 3, 2)
    wq, wt = ops.quant_fp8(wd, block_rows=128, layout="both")
    xq, xt = ops.quant_fp8(xd, layout="both")
    dq, dt = ops.quant_fp8(dyd, layout="both", fmt=fmt)
    W, D, Dt, Xt = quantise(w, 128)[0], quantise(dy, 1, fmt)[0], quantise(dy.t(), 1, fmt)[0], quantise(x.t())[0]
    dx, dw = ops.linear_dgrad_fp8(dq, wt, out_dtype=torch.float32), ops.linear_wgrad_fp8(dt, xt)
    assert dw.dtype == torch.float32
    _fp32_result(dx, D, W.t().contiguous())
    _fp32_result(dw, Dt, Xt)
    g = torch.Generator().manual_seed(9)
    X = quantise(x)[0]
    for got, n, f, at in ((dx, N, lambda v: (D * (v @ W.t())).sum(), X), (dw, M, lambda v: (Dt.t() * (Xt.t() @ v.t())).sum(), W)):
        step = torch.randn(at.shape, generator=g, dtype=torch.float64)
        num = f(at + step) - f(at)
        mag = (D.abs() @ W.abs() if got is dx else Dt.abs() @ Xt.abs().t()) * step.abs()
        # (the kernel's bound as above, with a group's largest below its sum; 64-bit rounding of the two values of f)
        lim = mag.sum() * (7 * 2.0 ** -25 + (n / 8 + 24) * 2.0 ** -24) + (f(at).abs() + mag.sum()) * 1e-11
        assert ((got.cpu().double() * step).sum() - num).abs() <= lim


@pytest.mark.parametrize("M", [3, 40, 200])
def test_fp32_results_at_the_ends_of_the_range(M):
    """Blocks at fp32's largest and smallest numbers: an element that rounds up to 2^128 counts as that, elements below 2^-132 to
    within 2^-133; NaN and infinities reach their own row only."""
    ops = _ops()
    K, N = 300, 140
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g)
    x[0] *= 2.0 ** -118
    x[0, 5] = 3e-39
    x[1] = x[1].clamp(-1, 1) * torch.finfo(torch.float32).max
    x[1, 7] = torch.finfo(torch.float32).max
    w *= 2.0 ** -20
    w[0] *= 2.0 ** -100
    w[1, 0] = 2.0 ** 100
    wq = ops.quant_fp8(w.to(DEV))
    a, b = quantise(x)[0], quantise(w)[0]
    assert a[1, 7] == 2.0 ** 128
    ref, mag = a @ b.t(), a.abs() @ b.abs().t()
    ends = 2.0 ** -133 * (a.abs().sum(1)[:, None] + b.abs().sum(1)[None])
    y = ops.linear_fwd_fp8(x.to(DEV), wq, out_dtype=torch.float32).cpu().double()
    fits = mag * 1.01 < torch.finfo(torch.float32).max
    assert fits[0].all() and fits[2:].all() and fits[1].float().mean() > 0.9
    err = (y - ref).abs()
    assert (err[fits] <= (mag * (K / 8 + 31) * 2.0 ** -24 + ends + 1e-38)[fits]).all()
    x[0, 3], x[1, 4] = float("nan"), float("inf")
    y = ops.linear_fwd_fp8(x.to(DEV), wq, out_dtype=torch.float32).cpu()
    assert torch.isnan(y[:2]).all() and torch.isfinite(y[2:]).all()
    d = ops.linear_dgrad_fp8(ops.quant_fp8(x.to(DEV), fmt="e5m2"), wq, out_dtype=torch.float32).cpu()
    assert torch.isnan(d[0]).all() and not torch.isfinite(d[1]).any() and torch.isfinite(d[2:]).all()
