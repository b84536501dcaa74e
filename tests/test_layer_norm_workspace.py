"""Bytes of the layer norm's backward workspace (host code; no GPU needed)."""

import pytest

import molnex_amd.kernels  # noqa: F401
from molnex_amd import _lib

SIZE = _lib.load().mnx_layer_norm_bwd_workspace_bytes


@pytest.mark.parametrize("rows", [0, 1, 63, 512, 5000, 1_000_000])
@pytest.mark.parametrize("width", [1, 333, 8192])
def test_rows_in_registers(rows, width):
    """Two sums a column for each of up to 512 workgroups, and two numbers a row."""
    assert SIZE(rows, width) <= min(max(rows, 1), 512) * 2 * width * 4 + 8 * rows + 512
    assert SIZE(rows, width) >= min(max(rows, 1), 512) * 2 * width * 4


@pytest.mark.parametrize("rows", [0, 1, 63, 64, 512, 20_000, 1_000_000])
@pytest.mark.parametrize("width", [8193, 70_001, 1 << 20, 1 << 24])
def test_wide_rows(rows, width):
    """Two sums a column for each strip of 64 rows, 256 strips at most, and two numbers a row: 1/32 of a float32 input
    and a little more."""
    strips = min(max(rows // 64, 1), 256)
    assert strips * 2 * width * 4 + 8 * rows <= SIZE(rows, width) <= strips * 2 * width * 4 + 8 * rows + 512
