"""Clipping factors under fp32's normal range: very large gradients and small bounds.

The factor is held as f 2^-s with f normal, and a value is v f 2^-s with v f rounded once (no overflow: f < 1, no underflow: see below) and the
power of two exact, but where the result is subnormal.  So a result is off by the factor's rounding and the norm's (2^-24 each, the norm's fp64 sum
n 2^-53), the product's (2^-24) and its type's: fp32 2^-24 or half its least subnormal 2^-150 -- as for any other factor."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('how', ['in place', 'out'])
@pytest.mark.parametrize('size, max_norm', [(1e36, 1.0), (4e36, 1e-3), (4e36, 1e-6), (2.0 ** 115, 2.0 ** -30), (1e36, 1e-12), (3e36, 1e-20)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_small_factors(dtype, size, max_norm, how):
    from autolabel_amd import clip
    g = torch.Generator().manual_seed(0)
    host = [(torch.randn(5000, generator=g) * size).to(dtype), (torch.randn(33, generator=g) * size * 2.0 ** -40).to(dtype)]
    norm = math.sqrt(sum(float((t.double() ** 2).sum()) for t in host))
    assert norm < 3.4e38
    ratio = max_norm / (norm + 1e-6)
    dev = [t.cuda() for t in host]
    out = [torch.empty_like(t) for t in dev] if how == 'out' else None
    clip.clip_grad_norm_(dev, max_norm, out=out)
    half, tiny = (2.0 ** -24, 2.0 ** -150) if dtype == torch.float32 else (2.0 ** -8, 2.0 ** -134)
    for h, o in zip(host, out or dev):
        want = h.double() * ratio
        tol = (3 * 2.0 ** -24 + half) * want.abs() * (1 + 2.0 ** -8) + tiny * (1 + 2.0 ** -8)
        assert ((o.cpu().double() - want).abs() <= tol).all(), float(((o.cpu().double() - want).abs() / tol).max())
