"""Sizes that the kernels of caches in 8 bits count in 31 bits, refused past them, without a GPU (placeholder pointers that are
never followed)."""

import pytest

from dropkv_b200 import _lib

P = 4096  # a placeholder device address


@pytest.mark.parametrize("block,D,aligned", [(1024, 1 << 21, False), (1024, 1 << 24, True), (1000, 2147484, False)])
def test_store_rows_fp8_refuses_pages_past_31_bits(block, D, aligned):
    """A row to a page whose elements (or vectors of eight) pass 2^31 - 2048, the count of what follows a scale that grows."""
    rows, page = (D, D, D) if aligned else (D + 1, D + 1, D + 1), (block * D, block * D, D)
    lib = _lib.load()
    rc = lib.dropkv_store_rows_fp8(P, *rows, P, *rows, P, P, *page, P, *page, P, 1, 1, P, 1, 1, 2, block, 2, 2, 1, 2, D, None)
    assert rc == _lib.ERR_UNSUPPORTED and "too large" in lib.dropkv_last_error().decode()
