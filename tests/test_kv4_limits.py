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


def test_groups_of_heads_that_pass_two_to_31_elements(tb):
    S = tb.Status
    for dim, heads in ((64, 2 ** 25), (128, 2 ** 24), (128, 2 ** 29)):
        c, r = cache(tb, heads=1, dim=dim), rows(tb, n=1)
        assert attention(tb, c, r, heads=heads) == S.SHAPE
        assert "q_heads / kv_heads" in tb.lib().tb_last_error().decode()
        assert tb.kv4_attention_workspace(c, r, heads, 1, 1000) == 0


def test_factors_that_pass_fp32(tb):
    """Each scale is an FP32 number, their product is not."""
    S = tb.Status
    for ks, scale in ((2.0 ** 100, 2.0 ** 30), (2.0 ** 100, -2.0 ** 30), (2.0 ** 64, 2.0 ** 64), (2.0 ** 60, 2.0 ** 67 * 1.9)):
        assert attention(tb, cache(tb, ks=ks), rows(tb), scale=scale) == S.INVALID_ARGUMENT
        assert "softmax_scale * k_scale" in tb.lib().tb_last_error().decode()
