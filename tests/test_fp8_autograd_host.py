"""fp8.linear on an x that requires a gradient: refused while gradients are tracked, its result would carry none."""
import pytest
import torch

from autolabel_amd import fp8


def blocks(rows, cols):
    nb = (cols + 127) // 128
    return fp8.Fp8Blocks(torch.zeros(rows, nb * 128).to(torch.float8_e4m3fn), torch.full((rows, (nb + 3) // 4 * 4), 127, dtype=torch.uint8), cols)


def test_linear_refuses_what_autograd_would_miss():
    w, x = blocks(4, 100), torch.zeros(3, 100, requires_grad=True)
    for bad in (x, x * 2, x.reshape(3, 1, 100)):
        with pytest.raises(ValueError, match='requires a gradient'):
            fp8.linear(bad, w)
        with pytest.raises(ValueError, match='requires a gradient'):
            fp8.linear(bad, w, out=torch.zeros(*bad.shape[:-1], 4))
        with torch.no_grad(), pytest.raises(ValueError, match='no CPU path'):       # (allowed: it gets as far as the device)
            fp8.linear(bad, w)
    with pytest.raises(ValueError, match='no CPU path'):
        fp8.linear(x.detach(), w)
    # the gradients' own products are not tracked a second time, whatever their operands ask for
    with pytest.raises(ValueError, match='no CPU path'):
        fp8.linear_backward(torch.zeros(3, 4, requires_grad=True), x, blocks(100, 4))
