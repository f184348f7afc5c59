"""Sizes that the C entry points' 32-bit arguments cannot hold are refused (they used to wrap: 2^32 + 128 columns were taken for 128)."""
import pytest
import torch

from autolabel_amd import fp8, hip


@pytest.mark.parametrize('cols', [fp8.MOST + 1, 1 << 31, (1 << 32) + 128, 1 << 40])
@pytest.mark.parametrize('transpose', [False, True])
def test_columns_over_32_bits(cols, transpose):
    with pytest.raises(ValueError, match='columns'):
        fp8.quantize(torch.empty(2, cols, dtype=torch.float16, device='meta'), transpose=transpose)
    with pytest.raises(ValueError, match='columns'):
        fp8.linear_backward(torch.empty(2, 8, device='meta'), torch.empty(2, cols, device='meta'), None, need_dx=False)
    with pytest.raises(ValueError, match='columns'):
        fp8.linear_backward(torch.empty(2, cols, device='meta'), torch.empty(2, 8, device='meta'), None, need_dx=False)


@pytest.mark.parametrize('rows', [fp8.MOST + 1, 1 << 31, (1 << 32) + 1])
def test_blocks_over_32_bits(rows):
    many = fp8.Fp8Blocks(torch.empty(rows, 128, dtype=torch.float8_e4m3fn, device='meta'), torch.empty(rows, 4, dtype=torch.uint8, device='meta'), 128)
    few = fp8.Fp8Blocks(torch.empty(4, 128, dtype=torch.float8_e4m3fn, device='meta'), torch.empty(4, 4, dtype=torch.uint8, device='meta'), 128)
    with pytest.raises(ValueError, match='rows'):
        fp8.matmul(few, many)
    with pytest.raises(ValueError, match='rows'):
        fp8.matmul(many, few)
    with pytest.raises(ValueError, match='rows'):
        fp8.linear(torch.empty(4, 128, device='meta'), many)


def test_the_longest_contraction():
    """Sizes are rounded up to whole tiles in 32 bits: the last 256 numbers under 2^31 would run over."""
    A = 1 << 20
    big = (1 << 31) - 255
    with pytest.raises(RuntimeError, match='sizes'):
        hip.call('aln_fp8_linear', A, 0, 0, 0, A, 1 << 31, A, 1 << 24, 0, 4, 8, big, A, 8, 0, 0, A, 1 << 40, None)
    with pytest.raises(RuntimeError, match='values'):
        hip.call('aln_fp8_quantize', A, 0, 0, 4, big, 0, A, 1 << 31, A, 1 << 24, None)
    with pytest.raises(RuntimeError, match='values'):
        hip.call('aln_fp8_quantize_t', A, 0, 0, 4, big, 0, A, 128, A, 4, None)
    with pytest.raises(RuntimeError, match='sizes'):
        hip.call('aln_fp8_nt', A, 1 << 31, A, 1 << 24, 0, A, 1 << 31, A, 1 << 24, 0, 4, 8, big, A, 8, 0, 0, A, 1 << 40, None)
