"""Rows of the FP4 cache's attention whose weight lies on a first token of no
value, so that the output is the sum of the small weights behind it."""
import math

import numpy as np
import pytest

import kv4_oracle as K
from test_kv4_gpu import EPS, LONG, Batch, error_word  # noqa: F401 (error_word: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_len", [None, LONG])
@pytest.mark.parametrize("gap", [12.0, 18.3, 21.7, 24.4, 26.2])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1, 3, 6, 40, 300])
def test_small_weights_behind_a_first_token(tb, cuda, n, dim, gap, max_len):
    """All tokens but the first weigh 2^-gap of it; its value is zero, theirs
    positive.

    The bound: P is held in FP16 with the row's largest at 2^6 or above, so a
    weight of 2^-gap of the largest is at 2^(6 - gap) or above and off by at most
    half a step, 2^-11 of itself or 2^-25 (FP16's subnormal steps are 2^-24), which
    is 2^(gap - 31) of itself.  (From 33 packed rows on the largest may be at 2^5,
    but there the small weights are powers of two here, and exact.)  The other
    terms are those of kv4_oracle.tolerances."""
    bt = Batch(tb, cuda, [n + 99, n + 420], [n, n], page=16, heads=1, dim=dim, k_scale=1.0, v_scale=2.0 ** 16, seed=n + dim)
    for b, length in enumerate(bt.lens):
        for pos in range(length):
            page, place = bt.place(b, pos)
            for is_v in (False, True):
                cs, ss = bt.host.parts(page, 0, place, is_v)
                bt.host.data[page, ss] = 0x38  # 1.0
                if is_v:
                    bt.host.data[page, cs] = 0 if pos == 0 else (bt.rng.integers(1, 8, dim // 2) * 16 +
                                                                bt.rng.integers(1, 8, dim // 2))
                else:
                    bt.host.data[page, cs] = 0x22 if pos == 0 else 0x00  # ones, zeros
    bt.upload()
    q, _ = bt.queries(2)
    q.fill_(1.0)
    scale = float(np.float32(gap * math.log(2) / dim))
    out, lse = bt.attend(q, 2, scale, max_len=max_len)
    o = out.double().cpu().numpy().reshape(bt.total, 2, dim)
    ls, qq = lse.double().cpu().numpy(), q.double().cpu().numpy().reshape(bt.total, 2, dim)
    for b in range(2):
        r = slice(bt.cu[b], bt.cu[b] + n)
        want = K.attention(bt.tokens(b, False), bt.tokens(b, True), qq[r], bt.lens[b] - n, scale)
        _, t_lse = K.tolerances(*want, bt.lens[b], dim, EPS["f16"])
        absv, reach, top = want[2:]
        e = (dim + 8) * 2.0 ** -23 * reach + 2.0 ** -21 * top + 2.0 ** -21
        part = 2.0 ** -11 + 2.0 ** (gap - 31) + np.expm1(2 * e) + bt.lens[b] * 2.0 ** -23 + 2.0 ** -20
        t_out = part[..., None] * absv * 1.01 + EPS["f16"] * np.abs(want[0]) + 2.0 ** -25
        err = np.abs(o[r] - want[0])
        assert np.all(err <= t_out), f"off by {np.max(err / np.maximum(want[0], 2.0 ** -25)):.3g} of the output"
        assert np.all(np.abs(ls[r] - want[1]) <= t_lse)
