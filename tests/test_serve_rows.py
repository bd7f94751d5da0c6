"""CPU: a batch of max_rows rows each whose row numbers would pass 31 bits is
refused, as the kernels count rows in 32-bit integers."""
import ctypes

import pytest

import quantr
from test_serve_args import P, TOO_LARGE, batch, pool, ref, tables


@pytest.mark.parametrize("B,rows", [(4, 1 << 29), (65535, 32769), (2, 2 ** 31 - 1)])
def test_too_many_rows(B, rows):
    L, b = quantr.lib(), batch(B=B, max_rows=rows)
    for f in ("quantr_kv8_append_dev", "quantr_kv8_read_dev"):
        assert getattr(L, f)(P, 128, P, 128, 0, ref(pool()), ref(tables()), ref(b), 0, None) == TOO_LARGE
    small = pool(n_kv_heads=1, n_layers=1)
    assert L.quantr_kv8_attend_dev(P, 64, P, 64, 1, 1, ref(small), ref(tables(max_pages=1)), ref(b), 0, ctypes.c_float(1.0), 0,
                                   64, None, P, 1 << 30, None) == TOO_LARGE
