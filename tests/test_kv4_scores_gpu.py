"""Attention over the FP4 cache where the factor of the scores or the queries
lie at the ends of their ranges."""
import numpy as np
import pytest

from test_kv4_gpu import LONG, Batch, error_word  # noqa: F401 (error_word: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_len", [None, LONG])
@pytest.mark.parametrize("scale", [0.0, 2.0 ** -120, -2.0 ** -120])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_small_factors_of_large_queries(tb, cuda, n, scale, max_len):
    """BF16 queries near 2^118 under a factor of 0 (all tokens weigh alike) and
    of 2^-120 (ordinary scores)."""
    bt = Batch(tb, cuda, [n + 60, n + 300], [n, n], page=16, heads=1, dim=64, typ="bf16", seed=n)
    bt.fill_fast()
    q, _ = bt.queries(4)
    q *= 2.0 ** 118
    out, lse = bt.attend(q, 4, scale, max_len=max_len)
    bt.check(out, lse, q, 4, scale)


@pytest.mark.parametrize("max_len", [None, LONG])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_large_factor_of_zero_products(tb, cuda, n, max_len):
    """Keys of zero: all scores are zero whatever the queries and the factor."""
    bt = Batch(tb, cuda, [n + 60, n + 300], [n, n], page=16, heads=1, dim=64, typ="bf16", seed=n)
    bt.fill_fast()
    for page in range(bt.host.pages):
        bt.host.data[page, :bt.host.codes] = 0
    bt.upload()
    q, _ = bt.queries(4)
    q *= 2.0 ** 120
    out, lse = bt.attend(q, 4, 2.0 ** 40, max_len=max_len)
    bt.check(out, lse, q, 4, 2.0 ** 40)
