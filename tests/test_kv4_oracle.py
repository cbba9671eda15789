"""The numpy statement of the cache (kv4_oracle.py) against independent ones."""
import numpy as np
import pytest

import kv4_oracle as K
import oracle as O


@pytest.mark.parametrize("g", [1.0, 0.0137, 2.0 ** -9])
def test_quantize_is_the_nearest(g):
    """Scale and codes by brute force over all candidates; ties to the smaller."""
    g = float(np.float32(g))
    rng = np.random.default_rng(3)
    x = rng.normal(size=(40, 64)) * np.exp(3 * rng.normal(size=(40, 1))) * g * 40
    x = x.astype(np.float16).astype(np.float64)
    x[0], x[1, :16] = 0.0, 6 * g * 0.4375  # zero blocks; an exact scale
    codes, scales = K.quantize(x, g)
    steps = K.scale_steps()
    for r in range(40):
        for b in range(4):
            blk = x[r, 16 * b:16 * b + 16]
            s = steps[np.argmin(np.abs(np.abs(blk).max() / (6 * g) - steps))]
            assert steps[scales[r, b]] == s
            for i in range(16):
                c = codes[r, 8 * b + i // 2]
                c = c >> 4 if i % 2 == 0 else c & 15
                want = np.argmin(np.abs(abs(blk[i]) - K.MAGS * s * g)) if s else 0
                assert c & 7 == want and (c >> 3) == (s > 0 and np.signbit(blk[i]))


def test_quantize_agrees_with_the_two_level_quantizer():
    """With that quantizer's tensor scale, the codes and scales differ only
    where its FP32 arithmetic rounds a border."""
    x = O.normal(5, (64, 256), 1.0)
    q, s, g = O.quantize_nvfp4(x)
    codes, scales = K.quantize(x, g)
    assert np.mean(scales != s) < 1e-3 and np.mean(codes != q) < 1e-3


def test_special_values():
    x = np.zeros((4, 16))
    x[0, 3], x[1, 5], x[2] = np.nan, np.inf, -1e-30
    codes, scales = K.quantize(x, 1.0)
    assert scales[:, 0].tolist() == [0x7F, 0x7E, 0, 0]
    assert not codes[0].any() and codes[1].tolist() == [0, 0, 0x07, 0, 0, 0, 0, 0] and not codes[2:].any()


def test_tokens_round_trip():
    c = K.Cache(3, 16, 2, 64, 0.01, 0.02, page_stride=2 * 16 * 72 + 32)
    rng = np.random.default_rng(1)
    k, v = rng.normal(size=(2, 2, 64))
    c.write(2, 15, k, v)
    for is_v, x, g in ((False, k, c.k_scale), (True, v, c.v_scale)):
        back = c.token(2, 15, is_v).astype(np.float64) * g
        assert O.rel_frob(back, x) < 0.2
        # codes and scales lie where the header says
        base = (16 * 32 + 16 * 4) * is_v
        assert np.array_equal(c.data[2, base + 15 * 32:base + 16 * 32], K.quantize(x, g)[0][0])
        assert np.array_equal(c.data[2, base + 16 * 32 + 15 * 4:base + 16 * 36], K.quantize(x, g)[1][0])


def test_attention_of_one_token_is_its_value():
    rng = np.random.default_rng(2)
    k, v, q = rng.normal(size=(5, 1, 16)), rng.normal(size=(5, 1, 16)), rng.normal(size=(1, 3, 16))
    out, lse, *_ = K.attention(k, v, q, 4, 0.5, window=1)
    np.testing.assert_allclose(out[0], np.repeat(v[4], 3, axis=0))
    np.testing.assert_allclose(lse[0], 0.5 * q[0] @ k[4, 0])
    out, lse, *_ = K.attention(k, v, q, -1, 0.5)
    assert not out.any() and np.isneginf(lse).all()
