"""Sizes and factors that the cache's entry points refuse because a kernel's
32-bit numbers would not hold what follows from them."""
import pytest

from test_kv4_abi import ALL, attention, cache, rows

INT_MAX = 2 ** 31 - 1


@pytest.mark.parametrize("f", ALL)
@pytest.mark.parametrize("size", [INT_MAX, INT_MAX - 30, 2 ** 31 - 4096])
def test_rows_and_batches_near_two_to_31(tb, f, size):
    S = tb.Status
    assert f(tb, cache(tb), rows(tb, n=size)) == S.SHAPE
    assert f(tb, cache(tb), rows(tb, batch=size)) == S.SHAPE
    assert "4097" in tb.lib().tb_last_error().decode()
