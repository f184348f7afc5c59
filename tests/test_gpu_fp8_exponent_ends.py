"""Products with an fp32 result whose blocks lie at the ends of the exponents.

A value q 2^e may be as small as 2^-142 (e5m2 2^-16 at e = -126) and as large as 2^128 (fp32's largest block, rounded up): bf16, which the fp32 results'
form multiplies in, holds neither.  The products themselves are what counts: against blocks from the definition in 64 bits every result with
sum |terms| under 2^127 is off by at most (K + 64) 2^-23 sum |terms| (one rounding per addition; the terms are exact), plus K terms that may be lost
under fp32's least normal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from test_gpu_fp8 import blocks64, fp8      # noqa: F401 (a fixture)


def check(got, va, vb, K):
    want, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    got, sure = got.cpu().double(), mag < 2.0 ** 127
    assert sure.any()
    tol = (K + 64) * 2.0 ** -23 * mag + K * 2.0 ** -126
    bad = ~((got - want).abs() <= tol) & sure
    assert not bad.any(), f'{int(bad.sum())} of {int(sure.sum())} outside, worst {float(((got - want).abs() / tol)[sure].nan_to_num(nan=math.inf).max()):.3g} of the bound'
    over = (mag >= 2.0 ** 129) & (want.abs() >= 2.0 ** 129)
    assert not torch.isfinite(got[over]).any()


def rows(R, K, seed, low, high):
    """Every row's blocks of sizes between 2^low and 2^high, a few of zeros."""
    g = torch.Generator().manual_seed(seed)
    nb = -(-K // 128)
    e = torch.randint(low, high + 1, (R, nb), generator=g).float().repeat_interleave(128, 1)[:, :K]
    x = (torch.rand(R, K, generator=g, dtype=torch.float64) * 2 - 1) * torch.exp2(e.double())
    x[torch.rand(R, nb, generator=g).lt(0.1).repeat_interleave(128, 1)[:, :K]] = 0
    return x.float()


@pytest.mark.parametrize('fa', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('fb', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('swap', [False, True])
@pytest.mark.parametrize('M,K,N', [(40, 256, 30), (300, 700, 260)])
def test_small_blocks(fp8, M, K, N, swap, fa, fb):          # noqa: F811
    """Blocks down to the last that do not vanish, beside ordinary ones, against large ones."""
    for low, high in ((-134, -118), (-128, -120), (-135, 0)):
        a, b = rows(M, K, 1, low, high), rows(N, K, 2, 50, 100)
        if swap:
            a, b = rows(M, K, 2, 50, 100), rows(N, K, 1, low, high)
        got = fp8.matmul(fp8.quantize(a.cuda(), fa), fp8.quantize(b.cuda(), fb), torch.float32)
        check(got, blocks64(a, fa)[0], blocks64(b, fb)[0], K)


@pytest.mark.parametrize('fa', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('fb', ['e4m3', 'e5m2'])
def test_large_blocks(fp8, fa, fb):                         # noqa: F811
    """Magnitudes that round up to 2^128, in either operand, beside ordinary and small rows and columns."""
    K = 300
    a, b = rows(70, K, 3, -100, -30), rows(66, K, 4, -60, 0)
    top = torch.finfo(torch.float32).max
    a[3, 5], a[3, 200], a[40, 130], b[7, 9], b[7, 290], b[50, 131] = top, -top, 1.99 * 2.0 ** 127, -top, top, 1.95 * 2.0 ** 127
    a[10:20] = rows(10, K, 5, -134, -120)
    b[20:25] = rows(5, K, 6, -134, -120)
    got = fp8.matmul(fp8.quantize(a.cuda(), fa), fp8.quantize(b.cuda(), fb), torch.float32)
    check(got, blocks64(a, fa)[0], blocks64(b, fb)[0], K)


@pytest.mark.parametrize('M,K,N', [(4200, 1024, 4100), (64, 4096, 64)])
def test_large_tiles_and_parts(fp8, M, K, N):               # noqa: F811
    """The 256 x 256 tiles, and a contraction in parts, with a few extreme rows and columns."""
    g = torch.Generator().manual_seed(0)
    a, b = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g)
    a[M // 2] *= 2.0 ** -128
    b[N // 3] *= 2.0 ** 100
    a[5, 7] = torch.finfo(torch.float32).max
    got = fp8.matmul(fp8.quantize(a.cuda()), fp8.quantize(b.cuda()), torch.float32).cpu()
    pick = [0, 4, 5, M // 2, M - 1]
    va, vb = blocks64(a[pick], 'e4m3')[0], blocks64(b, 'e4m3')[0]
    check(got[pick], va, vb, K)


def test_linear_and_gradients_of_small_fp32_values(fp8):    # noqa: F811
    x, w, gy = rows(50, 300, 1, -133, -120), rows(40, 300, 2, 60, 70), rows(50, 40, 3, 60, 70)
    got = fp8.linear(x.cuda(), fp8.quantize(w.cuda()))
    check(got, blocks64(x, 'e4m3')[0], blocks64(w, 'e4m3')[0], 300)
    dw = fp8.linear_backward(gy.cuda(), x.cuda(), None, need_dx=False)[1]
    check(dw, blocks64(gy.t().contiguous(), 'e4m3')[0], blocks64(x.t().contiguous(), 'e4m3')[0], 50)


@pytest.mark.parametrize('fmt', ['e4m3', 'e5m2'])
def test_weight_gradient_of_the_largest_bf16_values(fp8, fmt):      # noqa: F811
    """bf16 magnitudes that would round up to 2^128: the gradient's kernel holds them as the 8-bit value below (1.875 2^127 in e4m3, 1.75 2^127 in e5m2),
    still within half a step of theirs."""
    g = torch.Generator().manual_seed(0)
    gy, x = torch.randn(300, 40, generator=g).bfloat16(), (torch.randn(300, 70, generator=g) * 2.0 ** -60).bfloat16()
    top = torch.finfo(torch.bfloat16).max
    gy[3, 5], gy[299, 5], gy[200, 39], gy[130, 0] = top, -top, 1.9453125 * 2.0 ** 127, 1.9296875 * 2.0 ** 127

    def v(t, f):
        q = blocks64(t.t().contiguous(), f)[0]
        return torch.where(q.abs() == 2.0 ** 128, q.sign() * {'e4m3': 1.875, 'e5m2': 1.75}[f] * 2.0 ** 127, q)
    dw = fp8.linear_backward(gy.cuda(), x.cuda(), None, fmt, need_dx=False)[1]
    assert torch.isfinite(dw).all() and v(gy, fmt).abs().max() == {'e4m3': 1.875, 'e5m2': 1.75}[fmt] * 2.0 ** 127
    check(dw, v(gy, fmt), v(x, 'e4m3'), 300)
    dw = fp8.linear_backward(x.cuda(), gy.cuda(), None, fmt, need_dx=False)[1]
    assert torch.isfinite(dw).all()
    check(dw, v(x, fmt), v(gy, 'e4m3'), 300)


def test_nonfinite_and_extreme_rows_leave_the_others(fp8):  # noqa: F811
    """fp32 results: rows and columns that hold a NaN, an infinity or extreme values change no bit of the others, which do not meet them."""
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(200, 500, generator=g), torch.randn(150, 500, generator=g)
    clean = fp8.linear(x.cuda(), fp8.quantize(w.cuda())).cpu()
    x[3, 7], x[50, 499], x[130, 200], x[131] = math.inf, math.nan, torch.finfo(torch.float32).max, x[131] * 2.0 ** -130
    w[5, 0], w[149, 300], w[70] = -math.inf, math.nan, w[70] * 2.0 ** -128
    got = fp8.linear(x.cuda(), fp8.quantize(w.cuda())).cpu()
    rows, cols = torch.ones(200, dtype=torch.bool), torch.ones(150, dtype=torch.bool)
    rows[[3, 50, 130, 131]] = False
    cols[[5, 149, 70]] = False
    assert torch.equal(got[rows][:, cols], clean[rows][:, cols])
    assert torch.isnan(got[[3, 50]]).all() and torch.isnan(got[:, [5, 149]]).all()
    assert torch.isfinite(got[131][cols]).all() and torch.isfinite(got[rows][:, 70]).all() and (got[131][cols] != 0).any() and (got[rows][:, 70] != 0).any()
