"""Which way fp8.linear takes beyond 1024 columns, seen from the workspace it asks for: the blocks of x for two launches, parts alone for one."""
import pytest

from autolabel_amd import hip


@pytest.mark.parametrize('m, k, n', [(129, 4096, 4096), (257, 4096, 4096), (384, 4096, 4096), (384, 2048, 4096)])
def test_more_than_one_row_tile_is_quantised_once(m, k, n):
    """(measured the other way round: rows cut again by every column tile take up to 45% longer)"""
    L = hip.lib()
    assert L.aln_fp8_linear_ws_bytes(m, n, k, 0, 0, 0) >= m * -(-k // 128) * 129 + L.aln_fp8_nt_ws_bytes(m, n, k)


@pytest.mark.parametrize('m, k, n', [(1, 4096, 4096), (64, 4096, 4096), (128, 4096, 4096), (200000, 1100, 300)])
def test_one_row_tile_or_few_columns_are_cut_on_the_way(m, k, n):
    assert hip.lib().aln_fp8_linear_ws_bytes(m, n, k, 0, 0, 0) % (4 * m * n) == 0
