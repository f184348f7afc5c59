"""Global gradient norm and clipping (autolabel_amd.clip, csrc/clip.hip) against plain 64-bit arithmetic.

The sum of squares is taken in fp64, so the norm is off by its one rounding to fp32 (2^-24) and n additions of 2^-53; the factor by one more
rounding, and a scaled gradient by one more of its type (fp32 2^-24, fp16 2^-11, bf16 2^-8; fp16 2^-25 and bf16 / fp32 2^-134 / 2^-150 near zero).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


@pytest.fixture(scope='module')
def clip():
    from autolabel_amd import clip, hip
    hip.require_gpu()
    hip.lib()
    return clip


def lists():
    g = torch.Generator().manual_seed(0)
    r = lambda n, dt, s=1.0: (torch.randn(n, generator=g) * s).to(dt)
    f16, bf16, f32 = torch.float16, torch.bfloat16, torch.float32
    return {
        'one value': [r(1, f32)],
        'one odd': [r(1001, bf16)],
        'mixed': [r(7, f16), r(0, f32), r(8192, f32), r(8193, bf16), r(1, f16), r(40000, f32, 1e-3), r(3, bf16)],
        'many': [r(1 + 37 * i % 501, (f32, f16, bf16)[i % 3]) for i in range(391)],
        'empty tail': [r(10, f32)] + [r(0, f32)] * 250 + [r(5, f16)],
        'zeros': [torch.zeros(300), torch.zeros(20, dtype=f16)],
        'huge': [r(5000, f32, 1e25)],
        'small': [r(5000, f32, 1e-30)],
        'large': [r(9000001, f32)],
    }


@pytest.mark.parametrize('name', list(lists()))
@pytest.mark.parametrize('how', ['in place', 'out', 'idle', 'idle out', 'norm'])
def test_against_64_bits(clip, name, how):
    host = lists()[name]
    norm = math.sqrt(sum(float((t.double() ** 2).sum()) for t in host))
    max_norm = (0.3 * norm if how in ('in place', 'out', 'norm') else 2 * norm + 1)
    dev = [t.cuda() for t in host]
    out = [torch.full_like(t, 7) for t in dev] if 'out' in how else None
    got = clip.grad_norm(dev) if how == 'norm' else clip.clip_grad_norm_(dev, max_norm, out=out)
    assert got.dtype == torch.float32 and got.shape == ()
    n = sum(t.numel() for t in host)
    assert abs(float(got) - norm) <= (2.0 ** -24 + n * 2.0 ** -53) * norm
    factor = 1.0 if how == 'norm' else min(1.0, max_norm / (norm + 1e-6))
    for h, d, o in zip(host, dev, out or dev):
        if out is not None or how == 'norm':
            assert torch.equal(d.cpu(), h)
        want = h.double() * factor
        tol = 0 if factor == 1.0 else (2 * 2.0 ** -24 + HALF_STEP[h.dtype]) * want.abs() * (1 + 2.0 ** -8) + TINY[h.dtype]
        assert ((o.cpu().double() - want).abs() <= tol).all()


def test_loss_scale(clip):
    host = lists()['mixed']
    norm = math.sqrt(sum(float((t.double() ** 2).sum()) for t in host))
    scale = torch.tensor([1024.0], device='cuda')
    dev = [t.cuda() for t in host]
    got = clip.clip_grad_norm_(dev, norm / 4096, loss_scale=scale)       # a quarter of norm / 1024
    assert abs(float(got) - norm / 1024) <= 2.0 ** -23 * norm / 1024
    factor = (norm / 4096) / (norm / 1024 + 1e-6)
    for h, d in zip(host, dev):
        want = h.double() * factor
        assert ((d.cpu().double() - want).abs() <= (2.0 ** -22 + HALF_STEP[h.dtype]) * want.abs() * 1.01 + TINY[h.dtype]).all()


@pytest.mark.parametrize('bad', [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
def test_a_norm_that_is_not_finite_scales_nothing(clip, bad, dtype):
    host = [torch.ones(300), torch.ones(20000, dtype=dtype), torch.ones(5)]
    host[1][12345] = bad
    dev, out, flag = [t.cuda() for t in host], None, torch.zeros(1, dtype=torch.int32, device='cuda')
    norm = clip.clip_grad_norm_(dev, 1.0, found_inf=flag)
    assert not math.isfinite(float(norm)) and int(flag) == 1
    assert all(torch.equal(d.cpu().nan_to_num(nan=-5), h.nan_to_num(nan=-5)) for d, h in zip(dev, host))
    out, flag = [torch.empty_like(t) for t in dev], torch.zeros(1, dtype=torch.int32, device='cuda')
    clip.clip_grad_norm_(dev, 1.0, out=out, found_inf=flag)
    assert int(flag) == 1
    assert all(torch.equal(d.cpu().nan_to_num(nan=-5), h.nan_to_num(nan=-5)) for d, h in zip(out, host))
    flag.zero_()
    clip.clip_grad_norm_([torch.ones(10, device='cuda')], 1.0, found_inf=flag)
    assert int(flag) == 0


def test_fp32_overflow_of_the_norm_itself(clip):
    t = torch.full((5000,), 3e38, device='cuda')       # every value finite, the norm 2.1e40
    flag = torch.zeros(1, dtype=torch.int32, device='cuda')
    assert math.isinf(float(clip.clip_grad_norm_([t], 1.0, found_inf=flag))) and int(flag) == 1
    assert (t == 3e38).all()


def test_views_and_layouts(clip):
    g = torch.Generator().manual_seed(0)
    base = torch.randn(4000, generator=g)
    d = base.cuda()
    a, b = d[1:1002], d[1003:3999].half()[5:]          # odd offsets: fp32 aligned to 4, fp16 to 2 bytes
    cl = torch.randn(3, 5, 4, 7, generator=g).cuda().to(memory_format=torch.channels_last)
    tr = torch.randn(30, 50, generator=g).cuda().t()
    host = [t.cpu().clone() for t in (a, b, cl, tr)]
    norm = math.sqrt(sum(float((t.double() ** 2).sum()) for t in host))
    clip.clip_grad_norm_([a, b, cl, tr], norm / 2)
    for h, t in zip(host, (a, b, cl, tr)):
        assert ((t.cpu().double() - h.double() / 2).abs() <= (2.0 ** -20 + HALF_STEP[h.dtype]) * h.double().abs() + TINY[h.dtype]).all()
    assert d[0] == base[0].cuda() and d[1002] == base[1002].cuda() and (d[3999:] == base[3999:].cuda()).all()


def test_max_norm_edges(clip):
    t = torch.randn(1000, device='cuda')
    same = t.clone()
    clip.clip_grad_norm_(t, math.inf)
    assert torch.equal(t, same)
    clip.clip_grad_norm_([t], 0.0)
    assert (t == 0).all()


def test_the_same_bits_every_time_and_in_a_graph(clip):
    g = torch.Generator().manual_seed(0)
    dev = [torch.randn(n, generator=g).cuda() for n in (1000003, 17, 5000)]
    out = [torch.empty_like(t) for t in dev]
    body = lambda: clip.clip_grad_norm_(dev, 1.0, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = body()
    for i in range(4):
        for t in dev:
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        first = (float(norm), [o.clone() for o in out])
        assert float(body()) == first[0]
        assert all(torch.equal(a, b) for a, b in zip(first[1], out)), i


def test_refusals(clip):
    t = torch.randn(100, device='cuda')
    with pytest.raises(RuntimeError, match='share memory'):
        clip.clip_grad_norm_([t, t], 1.0)
    with pytest.raises(RuntimeError, match='share memory'):
        clip.clip_grad_norm_([t[:60], t[50:]], 1.0)
    with pytest.raises(RuntimeError, match='share memory'):
        clip.clip_grad_norm_([t[:50], t[50:]], 1.0, out=[t[50:], t[:50]])
    assert float(clip.grad_norm([t, t])) > 0            # nothing is written: the same tensor may be counted twice
    with pytest.raises(ValueError, match='one run of memory'):
        clip.clip_grad_norm_([t[::2]], 1.0)
    with pytest.raises(ValueError, match='max_norm'):
        clip.clip_grad_norm_([t], -1.0)
    with pytest.raises(ValueError, match='outputs'):
        clip.clip_grad_norm_([t], 1.0, out=[t, t])
    with pytest.raises(ValueError, match='output 0'):
        clip.clip_grad_norm_([t], 1.0, out=[t.half()])
    with pytest.raises(ValueError, match='different devices'):
        clip.clip_grad_norm_([t, t.cpu()], 1.0)
