"""Rows of the FP4 key/value cache's calls that cu_rows places outside the
caller's arrays: the sequence's other rows keep their token numbers, and the
error word says so."""
import numpy as np
import pytest

import kv4_oracle as K
from test_kv4_gpu import EPS, LONG, Batch, error_word, to_bits  # noqa: F401 (error_word: a fixture)

pytestmark = pytest.mark.gpu


def cut_batch(tb, cuda, n, lost, front, **kw):
    """Three sequences; `lost` rows of the last lie behind the arrays, `front`
    rows of the first before them."""
    bt = Batch(tb, cuda, [n + 30, 7, n + 41], [n, 2, n], **kw)
    bt.cu = (bt.cu - front).astype(np.int32)
    bt.total = int(bt.cu[-1]) - lost
    bt.index()
    return bt


def rows_inside(bt):
    """(sequence, row of the arrays, token) of the rows that are there."""
    for b, n in enumerate(bt.n):
        for i in range(n):
            if 0 <= bt.cu[b] + i < bt.total:
                yield b, int(bt.cu[b]) + i, bt.lens[b] - n + i


@pytest.mark.parametrize("n,lost,front", [(5, 2, 0), (5, 0, 3), (40, 25, 4), (300, 299, 0)])
def test_append_with_rows_behind_the_arrays(tb, cuda, n, lost, front):
    bt = cut_batch(tb, cuda, n, lost, front, page=16, heads=2, dim=64, seed=n)
    val, words = to_bits(bt.rng.normal(size=(bt.total, 2, 2, 64)).astype(np.float32), "f16")
    dev = cuda.from_numpy(words.copy()).cuda()
    tb.kv4_append(bt.cache, bt.rows, tb.Format.F16, dev.data_ptr(), dev.data_ptr() + 256, k_stride=256, v_stride=256)
    assert tb.device_error() == 2
    for b, row, pos in rows_inside(bt):
        bt.host.write(*bt.place(b, pos), *val[row])
    np.testing.assert_array_equal(bt.dev.cpu().numpy().reshape(bt.host.data.shape), bt.host.data)


@pytest.mark.parametrize("n,lost,front", [(5, 2, 0), (5, 0, 3), (40, 25, 4), (300, 299, 0)])
def test_read_with_rows_behind_the_arrays(tb, cuda, n, lost, front):
    bt = cut_batch(tb, cuda, n, lost, front, page=16, heads=2, dim=64, seed=n)
    bt.fill_fast()
    k, v = (cuda.full((bt.total, 128), 7.0, dtype=cuda.float16, device="cuda") for _ in range(2))
    tb.kv4_read(bt.cache, bt.rows, tb.Format.F16, k, v)
    assert tb.device_error() == 2
    for is_v, got in ((False, k), (True, v)):
        want = np.full((bt.total, 128), 7.0, np.float16)
        g = np.float32(bt.host.v_scale if is_v else bt.host.k_scale)
        for b, row, pos in rows_inside(bt):
            want[row] = (bt.host.token(*bt.place(b, pos), is_v).astype(np.float32) * g).reshape(-1).astype(np.float16)
        np.testing.assert_array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("window", [0, 9])
@pytest.mark.parametrize("max_len", [None, LONG])
@pytest.mark.parametrize("n,lost,front", [(5, 2, 0), (5, 0, 3), (40, 25, 4), (300, 299, 0), (300, 20, 7)])
def test_attention_with_rows_behind_the_arrays(tb, cuda, n, lost, front, max_len, window):
    bt = cut_batch(tb, cuda, n, lost, front, page=16, heads=1, dim=64, seed=n)
    bt.fill_fast()
    q, _ = bt.queries(2)
    out, lse = bt.attend(q, 2, 0.1, window=window, max_rows=n, max_len=max_len)
    assert tb.device_error() == 2
    kv = [(bt.tokens(b, False), bt.tokens(b, True)) for b in range(3)]
    o, ls, qq = (x.double().cpu().numpy() for x in (out, lse, q))
    for b, row, pos in rows_inside(bt):
        want = K.attention(*kv[b], qq[row].reshape(1, 2, 64), pos, 0.1, window)
        t_out, t_lse = K.tolerances(*want, bt.lens[b], 64, EPS["f16"])
        assert np.all(np.abs(o[row].reshape(1, 2, 64) - want[0]) <= t_out), (b, row)
        assert np.all(np.abs(ls[row] - want[1]) <= t_lse), (b, row)


@pytest.mark.parametrize("cu", [[0, 3, 2, 6], [0, 2, 6, 7], [-1, 2, 4, 6]])
def test_each_fault_of_cu_rows_is_reported(tb, cuda, cu):
    """Decreasing, behind the arrays, before them: by each call, alone."""
    bt = Batch(tb, cuda, [40, 40, 40], [2, 2, 2], page=16, heads=1, dim=64, seed=9)
    bt.fill_fast()
    bt.cu = np.array(cu, np.int32)
    bt.index()
    q, _ = bt.queries(2)
    k, v = (cuda.zeros((6, 64), dtype=cuda.float16, device="cuda") for _ in range(2))
    tb.kv4_read(bt.cache, bt.rows, tb.Format.F16, k, v)
    assert tb.device_error() == 2
    tb.kv4_append(bt.cache, bt.rows, tb.Format.F16, k, v)
    assert tb.device_error() == 2
    for max_len in (None, LONG):
        bt.attend(q, 2, 0.1, max_rows=4, max_len=max_len)
        assert tb.device_error() == 2
