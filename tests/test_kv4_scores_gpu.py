"""Attention over the FP4 cache where the factor of the scores or the queries
lie at the ends of their ranges."""
import math

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


@pytest.mark.parametrize("max_len", [None, LONG])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_infinite_query_beside_large_ones(tb, cuda, n, max_len):
    """BF16 rows that hold -inf where all keys are positive, beside values far
    outside FP16: all their scores are -inf.  The other rows stay as they are."""
    bt = Batch(tb, cuda, [n + 60, n + 300], [n, n], page=16, heads=1, dim=64, typ="bf16", seed=n)
    bt.fill_fast()
    for page in range(bt.host.pages):
        at = bt.host.data[page, :bt.host.codes].reshape(16, 32)
        at[:, 0] = 0x20 | at[:, 0] & 7  # token's first value 1.0, the second not negative
    bt.upload()
    q, _ = bt.queries(2)
    clean, clean_lse = bt.attend(q, 2, 0.1, max_len=max_len)
    q[0, 0], q[0, 1:64] = -math.inf, 3e38
    q[-1, 64], q[-1, 65] = -math.inf, -1e10
    out, lse = bt.attend(q, 2, 0.1, max_len=max_len)
    for row, head in ((0, 0), (bt.total - 1, 1)):
        assert bool((out[row, 64 * head:64 * head + 64] == 0).all()) and lse[row, head].item() == -math.inf
        clean[row, 64 * head:64 * head + 64], clean_lse[row, head] = 0, -math.inf
    assert cuda.equal(out, clean) and cuda.equal(lse, clean_lse)


@pytest.mark.parametrize("max_len", [None, LONG])
@pytest.mark.parametrize("size", [-1.6e38, 1.6e38])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_scores_near_the_ends_of_fp32(tb, cuda, n, size, max_len):
    """All scores of a row are the same number, near an end of FP32's range: the
    output is the mean of the values seen, lse that number.  The products are
    sums of 64 equal terms and differ in no bit, so neither do the weights; the
    mean takes FP16's half step for each weight, FP32 sums and BF16's half step."""
    bt = Batch(tb, cuda, [n + 60, n + 700], [n, n], page=16, heads=1, dim=64, typ="bf16", k_scale=1.0, seed=n)
    bt.fill_fast()
    for page in range(bt.host.pages):
        bt.host.data[page, :bt.host.codes] = 0x22
        bt.host.data[page, bt.host.codes:bt.host.codes + bt.host.scales] = 0x38
    bt.upload()
    q, _ = bt.queries(2)
    q.fill_(math.copysign(2.0 ** 115, size))
    scale = abs(size) / 2.0 ** 121
    out, lse = bt.attend(q, 2, scale, max_len=max_len)
    o, ls = out.double().cpu().numpy().reshape(bt.total, 2, 64), lse.double().cpu().numpy()
    for b in range(2):
        v = bt.tokens(b, True)[:, 0]
        for i in range(n):
            seen = v[:bt.lens[b] - n + i + 1]
            want, mass = seen.mean(axis=0), abs(seen).mean(axis=0)
            tol = (2.0 ** -11 + 2.0 ** -20 + len(seen) * 2.0 ** -23) * mass + 2.0 ** -8 * abs(want)
            assert (abs(o[bt.cu[b] + i] - want) <= tol).all(), (b, i)
            assert (abs(ls[bt.cu[b] + i] - size) <= 2.0 ** -20 * abs(size)).all(), (b, i)
