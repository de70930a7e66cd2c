"""Pointers that are not aligned as their element type are refused by the
cache-bounding operators before anything is launched (no GPU needed)."""
import pytest

from tests.test_bounded_cache_cpu import INVALID, P, chunk, evict, rows, weights


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("arg", ["tables", "row_table", "ctx"])
def test_rows_refuse(arg, off):
    assert rows(**{arg: P + off}) == INVALID
    assert weights(**{arg: P + off}) == INVALID


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("arg", ["tables", "tiles"])
def test_tiles_refuse(arg, off):
    assert chunk(**{arg: P + off}) == INVALID


@pytest.mark.parametrize("off", [1, 2, 3])
def test_weight_sums_refuse(off):
    assert weights(w=P + off) == INVALID


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("arg", ["tables", "row_table", "ctx", "next", "known", "w", "w_out", "pos", "pos_out", "ws"])
def test_evict_refuses(arg, off):
    assert evict(**{arg: P + off}) == INVALID
