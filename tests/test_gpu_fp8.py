"""8-bit block products (autolabel_amd.fp8, csrc/fp8.hip) against plain 64-bit implementations.

Quantised values and exponents are held bit-exact.

A product with an fp32 result: the terms qx qw 2^(ex + ew) are exact, and so are their products in fp32, so it is off by at most one rounding
per addition, (K + splits) 2^-23 sum |terms| (2^-23 and not 2^-24: the matrix instruction's own additions may truncate).

A product with a 16-bit result runs on the 8-bit matrix instruction, which cuts every term of a step off at 2^-13 of the step's largest (a
property of the hardware, measured on single steps).  A term's error is then below 2^-13 max |term|, of either sign with the term's, uniform:
variance 2^-26 max^2 / 3; over K terms sqrt(K / 3) 2^-13 max, and six of those hold for every one of some million results (1e-9 each outside).
The largest term is taken over the whole row and column.  On top half a step of the type, fp16 2^-11, bf16 2^-8 of the value, fp16 2^-25 near
zero.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EMAX = {'e4m3': 8, 'e5m2': 15}
DIGITS = {'e4m3': (3, -6), 'e5m2': (2, -14)}
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 0.0}


@pytest.fixture(scope='module')
def fp8():
    from autolabel_amd import fp8, hip
    hip.require_gpu()
    hip.lib()
    return fp8


def blocks64(x, fmt):
    """(values q 2^e [R, K], exponents e [R, blocks]) in 64 bits, from the definition; x on the CPU.  A block with a NaN or an infinity: NaN."""
    x = x.double()
    R, K = x.shape
    nb = -(-K // 128)
    pad = torch.zeros(R, nb * 128, dtype=torch.float64)
    pad[:, :K] = x
    b = pad.view(R, nb, 128)
    bad = ~torch.isfinite(b).all(-1)
    b = torch.where(bad[..., None], torch.ones_like(b), b)
    m, ex = torch.frexp(b.abs().amax(-1))          # max = m 2^ex, m in [1/2, 1)
    e = ex - 1 - EMAX[fmt] + (2 * m > 1.75).int()
    e = torch.where(m == 0, torch.zeros_like(e), e.clamp(min=-126))
    v = torch.ldexp(b, -e[..., None].double())
    digits, lowest = DIGITS[fmt]
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v)[1] - 1).clamp(min=lowest).double() - digits)
    q = torch.round(v / step) * step
    val = torch.ldexp(q, e[..., None].double())
    val = torch.where(bad[..., None], torch.full_like(val, math.nan), val)
    return val.reshape(R, -1)[:, :K], q.reshape(R, -1), e, bad


def hard(R, K, dtype, seed=0, nonfinite=False):
    """Rows of very different sizes, with zeros, powers of two, ties, the edges of the 8-bit ranges, and subnormals of the type."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K, generator=g) * torch.exp2(torch.randint(-12, 8, (R, 1), generator=g).float())
    x = torch.where(torch.rand(R, K, generator=g) < 0.2, torch.zeros(()), x)
    x = torch.where(torch.rand(R, K, generator=g) < 0.1, torch.exp2(torch.randint(-14, 10, (R, K), generator=g).float()), x)
    if R > 3:
        x[1] = 0
        x[2, :] = 448.0
        x[3, 0] = 449.0
    if R > 5:
        x[4] = x[4].sign() * torch.randint(1, 64, (K,), generator=g) / 16 + 0.0     # many ties
        x[5] *= {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -130, torch.float32: 2.0 ** -132}[dtype]
    if nonfinite and R > 8:
        x[6, K // 2] = math.inf
        x[7, 0] = math.nan
        x[8, K - 1] = -math.inf
    return x.to(dtype)


def check_blocks(got, x, fmt):
    val, q, e, bad = blocks64(x, fmt)
    K, nb = x.shape[1], e.shape[1]
    gq, gs = got.q.cpu().float().double(), got.scale.cpu()
    assert got.q.shape[1] == nb * 128 and gs.shape[1] == (nb + 3) // 4 * 4
    ok = ~bad[..., None].expand(-1, -1, 128).reshape(bad.shape[0], -1)
    assert torch.equal(gq[ok], q[ok])
    assert torch.isnan(gq[~ok]).all()
    assert torch.equal(gs[:, :nb][~bad].int() - 127, e[~bad])
    assert (gs[:, nb:] == 127).all()
    return val


@pytest.mark.parametrize('fmt', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('R,K', [(1, 1), (7, 77), (33, 128), (130, 129), (64, 512), (9, 1000)])
def test_quantize_is_bit_exact(fp8, R, K, dtype, fmt):
    x = hard(R, K, dtype, seed=R * K, nonfinite=True)
    check_blocks(fp8.quantize(x.cuda(), fmt), x, fmt)
    check_blocks(fp8.quantize(x.cuda(), fmt, transpose=True), x.t().contiguous(), fmt)


def test_quantize_every_fp16_value(fp8):
    """All 63488 finite fp16 values, one to a block beside a fixed partner: every rounding of the conversion."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = x[torch.isfinite(x)].view(-1, 1)
    x = torch.cat([x, torch.ones_like(x)], 1)
    for fmt in ('e4m3', 'e5m2'):
        check_blocks(fp8.quantize(x.cuda(), fmt), x, fmt)


def test_quantize_views(fp8):
    """Pitches, odd offsets, transposed and expanded views."""
    base = hard(70, 301, torch.float16, seed=3)
    d = base.cuda()
    for v in (lambda t: t[3:60, 5:140], lambda t: t[:, 1:2], lambda t: t.t()[:130], lambda t: t[10:11].expand(40, -1), lambda t: t[:, 7:8].expand(-1, 200),
              lambda t: t[::2, 1:300]):
        check_blocks(fp8.quantize(v(d)), v(base).contiguous(), 'e4m3')
        check_blocks(fp8.quantize(v(d), transpose=True), v(base).t().contiguous(), 'e4m3')


def product_bound(va, vb, K, dtype, relu=False):
    y = va @ vb.t()
    mag = va.abs() @ vb.abs().t()
    tol = (K + 64) * 2.0 ** -23 * mag + 1e-40
    if dtype != torch.float32:
        # the largest term of each (row, column): at most the product of the operands' largest, and exactly found where that is cheap
        M, N = va.shape[0], vb.shape[0]
        if M * N * K <= 1 << 26:
            most = torch.stack([(va[i].abs() * vb.abs()).amax(1) for i in range(M)])
        else:
            most = va.abs().amax(1)[:, None] * vb.abs().amax(1)[None]
        tol = tol + 6 * math.sqrt(K / 3) * 2.0 ** -13 * most + HALF_STEP[dtype] * y.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
    if relu:
        y = torch.where(y > 0, y, torch.zeros_like(y))
    return y, tol


def check(got, want, tol):
    got = got.cpu().double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f'{int(bad.sum())} of {bad.numel()} outside, worst {float(((got - want).abs() / tol).max()):.2f} of the bound'


@pytest.mark.parametrize('fa', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('fb', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
def test_matmul_formats_and_types(fp8, fa, fb, dtype):
    a, b = hard(75, 300, torch.float16, seed=1), torch.randn(66, 300, generator=torch.Generator().manual_seed(2)) * 0.05
    va, vb = blocks64(a, fa)[0], blocks64(b, fb)[0]
    want, tol = product_bound(va, vb, 300, dtype)
    if dtype == torch.float16:
        assert want.abs().max() < 65504
    check(fp8.matmul(fp8.quantize(a.cuda(), fa), fp8.quantize(b.cuda(), fb), dtype), want, tol)


SHAPES = [(1, 1, 1), (1, 512, 512), (2, 128, 3), (31, 129, 33), (64, 512, 512), (65, 528, 64), (128, 16, 16), (200, 640, 130), (257, 512, 300),
          (5, 4096, 40), (3, 1030, 1000), (300, 1536, 96), (1000, 77, 130), (129, 2048, 257), (70, 700, 200), (33, 893, 70), (130, 1000, 768),
          (65, 1024, 1024), (1, 300, 1500), (70, 384, 1500), (9, 250, 2000), (700, 256, 31)]


@pytest.mark.parametrize('relu', [False, True])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('M,K,N', SHAPES)
def test_linear(fp8, M, K, N, dtype, relu):
    g = torch.Generator().manual_seed(M + K + N)
    x = (torch.randn(M, K, generator=g) * torch.rand(M, 1, generator=g) * 3).to(dtype)
    w = torch.randn(N, K, generator=g) / math.sqrt(K)
    want, tol = product_bound(blocks64(x, 'e4m3')[0], blocks64(w, 'e4m3')[0], K, dtype, relu)
    got = fp8.linear(x.cuda(), fp8.quantize(w.cuda()), relu=relu)
    assert got.dtype == dtype
    check(got, want, tol)


def test_linear_many_rows(fp8):
    """More rows than one pass of any grid, an odd last tile."""
    g = torch.Generator().manual_seed(0)
    M, K, N = 70001, 136, 72
    x, w = torch.randn(M, K, generator=g).half(), torch.randn(N, K, generator=g)
    want, tol = product_bound(blocks64(x, 'e4m3')[0], blocks64(w, 'e4m3')[0], K, torch.float32)
    check(fp8.linear(x.cuda(), fp8.quantize(w.cuda()), out_dtype=torch.float32), want, tol)


def test_linear_shapes_views_and_empty(fp8):
    g = torch.Generator().manual_seed(0)
    w = torch.randn(20, 40, generator=g)
    wq = fp8.quantize(w.cuda())
    x = torch.randn(6, 5, 90, generator=g).half()
    xv = x[:, 1:4, 3:83:2]
    got = fp8.linear(xv.cuda(), wq)
    assert got.shape == (6, 3, 20)
    want, tol = product_bound(blocks64(xv.reshape(-1, 40), 'e4m3')[0], blocks64(w, 'e4m3')[0], 40, torch.float16)
    check(got.reshape(-1, 20), want, tol)
    xd = x.cuda()[:, 2, 11:51]                         # row pitch 450, odd offset
    want, tol = product_bound(blocks64(x[:, 2, 11:51], 'e4m3')[0], blocks64(w, 'e4m3')[0], 40, torch.float16)
    check(fp8.linear(xd, wq), want, tol)
    assert fp8.linear(torch.empty(0, 40, device='cuda', dtype=torch.bfloat16), wq).shape == (0, 20)
    assert fp8.linear(torch.empty(3, 0, 40, device='cuda'), wq).shape == (3, 0, 20)
    one = fp8.linear(x[0, 0, :40].cuda(), wq)          # a vector
    assert one.shape == (20,)


@pytest.mark.parametrize('fx', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('fw', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('K', [200, 600, 1200])
def test_linear_formats(fp8, fx, fw, K):
    g = torch.Generator().manual_seed(K)
    x, w = torch.randn(150, K, generator=g).bfloat16(), torch.randn(90, K, generator=g) / math.sqrt(K)
    want, tol = product_bound(blocks64(x, fx)[0], blocks64(w, fw)[0], K, torch.bfloat16)
    check(fp8.linear(x.cuda(), fp8.quantize(w.cuda(), fw), fmt=fx), want, tol)


def test_linear_out(fp8):
    x, wq = torch.randn(7, 30, 96, device='cuda').half(), fp8.quantize(torch.randn(40, 96, device='cuda'))
    want = fp8.linear(x, wq)
    out = torch.full((9, 30, 40), 7.0, device='cuda', dtype=torch.float16)
    got = fp8.linear(x, wq, out=out[1:8])
    assert got.data_ptr() == out[1:8].data_ptr() and torch.equal(out[1:8], want)
    assert (out[0] == 7).all() and (out[8] == 7).all()           # what lies beside is left as it was
    out32 = torch.empty(7, 30, 40, device='cuda')
    assert torch.equal(fp8.linear(x, wq, out=out32), fp8.linear(x, wq, out_dtype=torch.float32))
    for bad in (out[:6], out[1:8].transpose(0, 1), torch.empty(7, 30, 40)):
        with pytest.raises(ValueError, match='out must be'):
            fp8.linear(x, wq, out=bad)
    with pytest.raises(ValueError, match='out must be'):
        fp8.linear(x, wq, out=out32, out_dtype=torch.float16)
    sq = fp8.quantize(torch.randn(96, 96, device='cuda'))
    with pytest.raises(ValueError, match='overlap'):
        fp8.linear(x, sq, out=x)


@pytest.mark.parametrize('M,K,N', [(129, 1, 1), (256, 3, 5), (128, 7, 1), (135, 2, 9), (383, 8, 8), (4096, 40, 1), (8, 1, 1), (7, 1, 1), (1, 8, 8), (1, 3, 4),
                                   (66000, 300, 300), (65536, 264, 520), (640, 30, 400)])
def test_weight_gradient_edges(fp8, M, K, N):
    """Where a piece of eight columns would reach over the tensors' end: both stand alone at the end of their memory here (a pool's block is larger,
    but what lies behind is NaN, and must not be met)."""
    r = torch.Generator().manual_seed(M + K + N)
    x, gy = torch.randn(M, K, generator=r).half(), (torch.randn(M, N, generator=r) * 0.1).half()
    xd, gd = torch.full((M * K + 64,), math.nan, device='cuda').half(), torch.full((M * N + 64,), math.nan, device='cuda').half()
    xd[:M * K], gd[:M * N] = x.cuda().reshape(-1), gy.cuda().reshape(-1)
    dw = fp8.linear_backward(gd[:M * N].view(M, N), xd[:M * K].view(M, K), None, need_dx=False)[1]
    want, tol = product_bound(blocks64(gy.t().contiguous(), 'e4m3')[0], blocks64(x.t().contiguous(), 'e4m3')[0], M, torch.float32)
    check(dw, want, tol)


def test_weight_gradient_pitches_and_types(fp8):
    r = torch.Generator().manual_seed(0)
    base_x, base_g = torch.randn(500, 301, generator=r).half(), torch.randn(500, 205, generator=r).half()
    for xs, gs in ((slice(5, 140), slice(3, 80)), (slice(0, 301), slice(204, 205)), (slice(1, 257), slice(0, 128))):
        x, gy = base_x[:, xs], base_g[:, gs]
        want, tol = product_bound(blocks64(gy.t().contiguous(), 'e5m2')[0], blocks64(x.t().contiguous(), 'e4m3')[0], 500, torch.float32)
        check(fp8.linear_backward(base_g.cuda()[:, gs], base_x.cuda()[:, xs], None, 'e5m2', need_dx=False)[1], want, tol)
        # g and x of different types: 16-bit beside fp32
        check(fp8.linear_backward(base_g.cuda()[:, gs].float(), base_x.cuda()[:, xs], None, 'e5m2', need_dx=False)[1], want, tol)


def test_weight_gradient_nonfinite_columns_stay_in_their_columns(fp8):
    r = torch.Generator().manual_seed(0)
    x, gy = torch.randn(1000, 70, generator=r).half(), torch.randn(1000, 40, generator=r).half()
    x[300, 11], x[999, 69], gy[0, 3], gy[500, 39] = math.inf, math.nan, -math.inf, math.nan
    for fmt in ('e4m3', 'e5m2'):
        dw = fp8.linear_backward(gy.cuda(), x.cuda(), None, fmt, need_dx=False)[1].cpu()
        bad = torch.zeros(40, 70, dtype=torch.bool)
        bad[:, [11, 69]] = True
        bad[[3, 39]] = True
        assert torch.isnan(dw[bad]).all() and torch.isfinite(dw[~bad]).all()


def test_linear_nonfinite_rows_stay_in_their_rows(fp8):
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(100, 300, generator=g).half(), torch.randn(70, 300, generator=g)
    x[3, 7], x[50, 299], x[99, 128] = math.inf, math.nan, -math.inf
    for relu in (False, True):
        y = fp8.linear(x.cuda(), fp8.quantize(w.cuda()), relu=relu).cpu()
        bad = torch.zeros(100, dtype=torch.bool)
        bad[[3, 50, 99]] = True
        assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()


def test_linear_extreme_scales(fp8):
    """Blocks at the ends of the exponents: the scales' product is taken in full, results under fp32's range become subnormal or 0."""
    x = torch.full((4, 256), 1.0)
    x[0] *= 2.0 ** 100; x[1] *= 2.0 ** -100; x[2] *= 2.0 ** -140; x[3, :128] = 0
    w = torch.full((3, 256), 1.0)
    w[0] *= 2.0 ** -90; w[1] *= 2.0 ** 20
    want = blocks64(x, 'e4m3')[0] @ blocks64(w, 'e4m3')[0].t()
    got = fp8.linear(x.cuda(), fp8.quantize(w.cuda())).cpu()
    want = want.float()                                # 256 x 2^100 x 2^20 = 2^128 is infinite in fp32, 2^-182 is 0
    assert math.isinf(want[0, 1]) and want[1, 0] == 0
    normal = want.abs() >= 2.0 ** -126
    assert torch.equal(got[normal], want[normal]) and (got[~normal].abs() < 2.0 ** -126).all()


BACK = [(1, 1, 1), (3, 40, 17), (128, 128, 128), (1003, 77, 130), (4096, 512, 512), (20000, 96, 40), (257, 640, 65), (129, 16, 300)]


@pytest.mark.parametrize('gfmt', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('M,K,N', BACK)
def test_linear_backward(fp8, M, K, N, dtype, gfmt):
    r = torch.Generator().manual_seed(M + K + N)
    x = torch.randn(M, K, generator=r).clamp(min=0).to(dtype)
    gy = (torch.randn(M, N, generator=r) * 0.1 * torch.rand(M, 1, generator=r)).to(dtype)
    w = torch.randn(N, K, generator=r) / math.sqrt(K)
    dx, dw = fp8.linear_backward(gy.cuda(), x.cuda(), fp8.quantize(w.t().cuda()), grad_fmt=gfmt)
    want, tol = product_bound(blocks64(gy, gfmt)[0], blocks64(w.t().contiguous(), 'e4m3')[0], N, dtype)
    assert dx.dtype == dtype and dw.dtype == torch.float32
    check(dx, want, tol)
    want, tol = product_bound(blocks64(gy.t().contiguous(), gfmt)[0], blocks64(x.t().contiguous(), 'e4m3')[0], M, torch.float32)
    check(dw, want, tol)


def test_linear_backward_parts_views_and_empty(fp8):
    r = torch.Generator().manual_seed(0)
    w = torch.randn(24, 40, generator=r).cuda()
    x, gy = torch.randn(5, 60, 40, generator=r).half().cuda(), torch.randn(5, 60, 24, generator=r).half().cuda()
    wt = fp8.quantize(w.t())
    dx, dw = fp8.linear_backward(gy, x, wt)
    assert dx.shape == x.shape and dw.shape == w.shape
    assert torch.equal(fp8.linear_backward(gy, x, None, need_dx=False)[1], dw)
    only = fp8.linear_backward(gy, x, wt, need_dw=False)
    assert only[1] is None and torch.equal(only[0], dx)
    one = torch.ones((), device='cuda').half().expand(5, 60, 24)       # what sum().backward() hands over
    a, b = fp8.linear_backward(one, x, wt), fp8.linear_backward(one.contiguous(), x, wt)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    dx, dw = fp8.linear_backward(gy[:0], x[:0], wt)
    assert dx.shape == (0, 60, 40) and torch.equal(dw, torch.zeros_like(w))


def test_the_same_bits_every_time(fp8):
    r = torch.Generator().manual_seed(0)
    x, gy = torch.randn(30011, 200, generator=r).half().cuda(), torch.randn(30011, 90, generator=r).half().cuda()
    w = torch.randn(90, 200, generator=r).cuda()
    wq, wt = fp8.quantize(w), fp8.quantize(w.t())
    first = (fp8.linear(x, wq), *fp8.linear_backward(gy, x, wt))
    for _ in range(3):
        again = (fp8.linear(x, wq), *fp8.linear_backward(gy, x, wt))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_two_streams_at_once(fp8):
    r = torch.Generator().manual_seed(0)
    w = torch.randn(512, 512, generator=r).cuda()
    wq, wt = fp8.quantize(w), fp8.quantize(w.t())
    xs = [torch.randn(5000, 512, generator=r).half().cuda() for _ in range(2)]
    want = [(fp8.linear(x, wq), *fp8.linear_backward(x, x, wt)) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            for _ in range(5):
                got[i] = (fp8.linear(xs[i], wq), *fp8.linear_backward(xs[i], xs[i], wt))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_captured_and_replayed(fp8):
    r = torch.Generator().manual_seed(0)
    w = torch.randn(96, 300, generator=r).cuda()
    x, gy = torch.randn(3000, 300, generator=r).half().cuda(), torch.randn(3000, 96, generator=r).half().cuda()
    wq, wt = fp8.quantize(w), fp8.quantize(w.t())
    body = lambda: (fp8.linear(x, wq, relu=True), *fp8.linear_backward(gy, x, wt))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                  # two graphs of the same call, replayed in turn
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = body()
        graphs.append((gr, out))
    for i in range(4):
        x.copy_(torch.randn(3000, 300, generator=r))
        gy.copy_(torch.randn(3000, 96, generator=r) * 0.1)
        for gr, out in graphs:
            gr.replay()
            want = body()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_linear_module_gradients(fp8):
    """Linear against the formulas in 64 bits, and against a plain layer: its gradients are those of the plain layer up to 8-bit rounding."""
    torch.manual_seed(0)
    layer = fp8.Linear(100, 36, device='cuda')
    assert list(layer.state_dict()) == ['weight']
    x = torch.randn(7, 50, 100, device='cuda', requires_grad=True)
    gy = torch.randn(7, 50, 36, device='cuda')
    y = layer(x)
    y.backward(gy)
    w = layer.weight.detach().cpu()
    flat = lambda t: t.detach().cpu().reshape(-1, t.shape[-1])
    want, tol = product_bound(blocks64(flat(x), 'e4m3')[0], blocks64(w, 'e4m3')[0], 100, torch.float32)
    check(flat(y), want, tol)
    want, tol = product_bound(blocks64(flat(gy), 'e4m3')[0], blocks64(w.t().contiguous(), 'e4m3')[0], 36, torch.float32)
    check(flat(x.grad), want, tol)
    want, tol = product_bound(blocks64(flat(gy).t().contiguous(), 'e4m3')[0], blocks64(flat(x).t().contiguous(), 'e4m3')[0], 350, torch.float32)
    check(layer.weight.grad, want, tol)
    # each operand's value is off by at most half a step of e4m3, 2^-4 of itself (a block's small values: 2^-10 of its largest magnitude,
    # the half step under the smallest normal): every product of a sum by 2^-3 + 2^-8 plus those floors
    a, b = flat(gy).double(), w.double()
    plain, mag = a @ b, (a.abs() + 2.0 ** -10 * a.abs().amax(1, keepdim=True)) @ (b.abs() + 2.0 ** -10 * b.abs().amax(0, keepdim=True))
    assert ((flat(x.grad).double() - plain).abs() <= (2.0 ** -3 + 2.0 ** -8) * mag).all()


def test_linear_module_only_asked_gradients(fp8):
    layer = fp8.Linear(64, 32, grad_fmt='e5m2', device='cuda', dtype=torch.bfloat16)
    x = torch.randn(10, 64, device='cuda', dtype=torch.bfloat16)
    layer(x).sum().backward()
    assert layer.weight.grad.dtype == torch.bfloat16 and x.grad is None
    layer.weight.requires_grad_(False)
    x.requires_grad_(True)
    layer(x).sum().backward()
    assert x.grad.shape == x.shape


def test_gpu_refusals(fp8):
    x, w = torch.randn(4, 40, device='cuda'), fp8.quantize(torch.randn(8, 40, device='cuda'))
    with pytest.raises(ValueError, match='columns'):
        fp8.linear(x[:, :39], w)
    with pytest.raises(ValueError, match='columns'):
        fp8.matmul(fp8.quantize(x[:, :39]), w)
    with pytest.raises(ValueError, match='different devices|no CPU path'):
        fp8.linear(x.cpu(), w)
    with pytest.raises(ValueError, match='rows'):
        fp8.linear_backward(x[:3], x, w)
    with pytest.raises(ValueError, match='weight_t is'):
        fp8.linear_backward(x, x, w)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('M,K,N', [(3841, 200, 3777), (64, 1000, 4096), (1000, 700, 1300), (1920, 2048, 1024), (100, 4100, 120), (1100, 130, 2300)])
def test_matmul_tiles_and_parts(fp8, M, K, N, dtype):
    """Large and small tiles, one row tile and many, numbers of tiles that eight does not divide, contractions in one part and in several."""
    g = torch.Generator().manual_seed(M + K + N)
    a, b = torch.randn(M, K, generator=g) * torch.rand(M, 1, generator=g), torch.randn(N, K, generator=g) / math.sqrt(K)
    want, tol = product_bound(blocks64(a, 'e4m3')[0], blocks64(b, 'e4m3')[0], K, dtype)
    check(fp8.matmul(fp8.quantize(a.cuda()), fp8.quantize(b.cuda()), dtype), want, tol)


@pytest.mark.parametrize('M,K,N', [(1, 1000, 4000), (512, 900, 1100), (513, 900, 1100), (600, 1024, 1024), (64, 500, 4100), (2304, 100, 200), (900, 60, 520)])
def test_linear_parts(fp8, M, K, N):
    """Either side of where one launch does it, and row ranges and column parts that eight does not divide."""
    g = torch.Generator().manual_seed(M + K + N)
    x, w = (torch.randn(M, K, generator=g) * torch.rand(M, 1, generator=g)).half(), torch.randn(N, K, generator=g) / math.sqrt(K)
    want, tol = product_bound(blocks64(x, 'e4m3')[0], blocks64(w, 'e4m3')[0], K, torch.float16)
    check(fp8.linear(x.cuda(), fp8.quantize(w.cuda())), want, tol)


@pytest.mark.parametrize('M,K,N', [(1200, 1300, 1100), (300, 2100, 600), (128, 600, 4100)])
def test_weight_gradient_few_parts(fp8, M, K, N):
    g = torch.Generator().manual_seed(M + K + N)
    x, gy = torch.randn(M, K, generator=g).half(), (torch.randn(M, N, generator=g) * 0.1).half()
    want, tol = product_bound(blocks64(gy.t().contiguous(), 'e5m2')[0], blocks64(x.t().contiguous(), 'e4m3')[0], M, torch.float32)
    check(fp8.linear_backward(gy.cuda(), x.cuda(), None, 'e5m2', need_dx=False)[1], want, tol)


def test_linear_out_tells_autograd(fp8):
    """A tensor saved for a backward pass and then written into: the backward pass must refuse, as for torch's own operations."""
    w = fp8.quantize(torch.eye(64, device='cuda'))
    x, out = torch.ones(5, 64, device='cuda'), torch.ones(5, 64, device='cuda')
    leaf = torch.ones(5, 64, device='cuda', requires_grad=True)
    loss = (leaf * out).sum()
    fp8.linear(x, w, out=out)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()
    with torch.inference_mode():
        o = torch.empty(5, 64, device='cuda')
        assert torch.equal(fp8.linear(x, w, out=o), x)


@pytest.mark.parametrize('fmt', ['e4m3', 'e5m2'])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('M,K,N', [(1, 1025, 5), (1, 1086, 1059), (130, 1033, 384), (385, 1100, 384), (385, 1100, 385), (384, 1151, 400), (128, 2048, 128), (5, 4095, 129),
                                   (3000, 1153, 40)])
def test_linear_rows_cut_on_the_way_to_tiles(fp8, M, K, N, dtype, fmt):
    """More columns than registers hold, few rows or few columns of results: x a view between NaN columns, its last piece of any length."""
    g = torch.Generator().manual_seed(M + K + N)
    x = (torch.randn(M, K, generator=g) * torch.rand(M, 1, generator=g)).to(dtype)
    w = torch.randn(N, K, generator=g) / math.sqrt(K)
    wide = torch.full((M, K + 11), math.nan, dtype=dtype, device='cuda')
    wide[:, 3:3 + K] = x.cuda()
    want, tol = product_bound(blocks64(x, fmt)[0], blocks64(w, 'e4m3')[0], K, dtype)
    ws = fp8.quantize(w.cuda())
    got = fp8.linear(wide[:, 3:3 + K], ws, fmt=fmt)
    check(got, want, tol)
    assert torch.equal(got, fp8.linear(x.cuda(), ws, fmt=fmt))


def test_linear_cut_rows_nonfinite_and_broadcast(fp8):
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(200, 1300, generator=g).half(), torch.randn(300, 1300, generator=g) / 36
    sq = fp8.quantize(w.cuda())
    clean = fp8.linear(x.cuda(), sq)
    bad = x.clone()
    bad[7, 1299], bad[150, 0], bad[151, 700] = math.nan, math.inf, -math.inf
    got, rows = fp8.linear(bad.cuda(), sq), [7, 150, 151]
    keep = [i for i in range(200) if i not in rows]
    assert torch.isnan(got[rows]).all() and torch.equal(got[keep], clean[keep])
    one = x[:1].cuda().expand(200, 1300)
    assert torch.equal(fp8.linear(one, sq), fp8.linear(one.contiguous(), sq))
