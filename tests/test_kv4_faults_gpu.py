"""What attention over the FP4 cache does with batches that their host-side
numbers or page tables describe wrongly."""
import numpy as np
import pytest

import kv4_oracle as K
from test_kv4_gpu import EPS, LONG, Batch, error_word  # noqa: F401 (error_word: a fixture)

pytestmark = pytest.mark.gpu


def check_row(bt, out, lse, q, q_heads, scale, b, i, keep=None):
    """Row i of sequence b against 64-bit sums over the tokens `keep` (all)."""
    d = bt.host.dim
    pos = bt.lens[b] - bt.n[b] + i
    keep = np.arange(bt.lens[b]) if keep is None else np.asarray(keep)
    k, v = bt.values[b][0][keep], bt.values[b][1][keep]
    m = int((keep <= pos).sum())
    row = int(bt.cu[b]) + i
    qq = q[row].double().cpu().numpy().reshape(1, q_heads, d)
    want = K.attention(k[:m], v[:m], qq, m - 1, scale)
    t_out, t_lse = K.tolerances(*want, bt.lens[b], d, EPS[bt.typ])
    got = out[row].double().cpu().numpy().reshape(1, q_heads, d)
    assert np.all(np.abs(got - want[0]) <= t_out), (b, i)
    ls = lse[row].double().cpu().numpy()[None]
    seen = np.isfinite(want[1])
    assert np.array_equal(np.isneginf(ls), ~seen) and np.all(np.abs(ls[seen] - want[1][seen]) <= t_lse[seen]), (b, i)


@pytest.mark.parametrize("max_len", [100, LONG])
@pytest.mark.parametrize("others", [0, 10])
def test_more_row_tiles_than_max_rows_has(tb, cuda, others, max_len):
    """A sequence of three tiles of 256 packed rows where max_rows gives room for
    one: the first tile's rows are right, the others' left as they were, and the
    error word says so.  With and without shares of a unit's tokens (max_len), in
    a batch of like sequences and one whose items are drawn (others)."""
    n, length = 300, 900
    bt = Batch(tb, cuda, [50] * (others // 2) + [length] + [50] * (others // 2),
               [1] * (others // 2) + [n] + [1] * (others // 2), page=16, heads=1, dim=64, seed=others)
    bt.fill_fast()
    bt.values = [(bt.tokens(b, False), bt.tokens(b, True)) for b in range(len(bt.n))]
    q, _ = bt.queries(2)
    out, lse = bt.attend(q, 2, 0.1, max_rows=40, max_len=max_len)
    assert tb.device_error() == 4
    for b in range(len(bt.n)):
        for i in range(bt.n[b]):
            if i < 128:
                check_row(bt, out, lse, q, 2, 0.1, b, i)
            else:
                row = int(bt.cu[b]) + i
                assert bool((out[row] == 7).all()) and bool((lse[row] == 7).all())


@pytest.mark.parametrize("max_len", [None, LONG])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_pages_outside_the_cache_count_in_neither_output(tb, cuda, max_len, n):
    """Tokens of pages that are not there are in neither the output nor its lse."""
    lens = [100, 1500]
    bt = Batch(tb, cuda, lens, [n, n], page=16, heads=1, dim=64, seed=36)
    bt.fill_fast()
    bt.values = [(bt.tokens(b, False), bt.tokens(b, True)) for b in range(2)]
    q, _ = bt.queries(2)
    bt.table[0, 2], bt.table[1, 5], bt.table[1, 60] = bt.host.pages, -1, 2 ** 31 - 1
    bt.index()
    out, lse = bt.attend(q, 2, 0.1, max_len=max_len)
    assert tb.device_error() == 2
    for b, hidden in ((0, [2]), (1, [5, 60])):
        keep = [p for p in range(lens[b]) if p // 16 not in hidden]
        for i in range(n):
            check_row(bt, out, lse, q, 2, 0.1, b, i, keep)


def test_no_rows_by_max_rows(tb, cuda):
    """max_rows 0: nothing is written and nothing reported."""
    bt = Batch(tb, cuda, [100, 60], [1, 3], page=16, heads=1, dim=64, seed=38)
    bt.fill_fast()
    q, _ = bt.queries(2)
    for max_len in (100, LONG):
        out, lse = bt.attend(q, 2, 0.1, max_rows=0, max_len=max_len)
        assert bool((out == 7).all()) and bool((lse == 7).all())
        assert tb.device_error() == 0


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("typ,q_heads", [("f16", 1), ("bf16", 3)])
def test_nan_values_in_whole_and_partly_seen_tiles(tb, cuda, typ, q_heads, page):
    """NaN blocks of V in tiles of 128 tokens that all rows see whole, in those
    that they see in part, and in one that has a page missing: each row has a NaN
    where it sees one, and only there."""
    n, lens = 300, [1500, 1000]
    bt = Batch(tb, cuda, lens, [n, n], page=page, heads=1, dim=64, typ=typ, seed=page)
    bt.fill_fast()
    missing = 512 // page  # of sequence 0
    bad = {0: [(200, 0), (700, 1), (1205, 2), (1350, 1), (1499, 3)], 1: [(0, 3), (701, 2), (999, 0)]}
    if page == 16:
        bad[0].append((530, 3))  # beside the missing page in its tile
    for b, blocks in bad.items():
        for pos, x in blocks:
            pg, place = bt.place(b, pos)
            ss = bt.host.parts(pg, 0, place, True)[1]
            bt.host.data[pg, ss.start + x] = 0x7F
    bt.upload()
    bt.table[0, missing] = -1
    bt.index()
    q, _ = bt.queries(q_heads)
    out, lse = bt.attend(q, q_heads, 0.1)
    assert tb.device_error() == 2
    assert bool(lse.isfinite().all())
    o = out.float().cpu().numpy().reshape(-1, q_heads, 4, 16)
    for b, blocks in bad.items():
        for i in range(n):
            pos = lens[b] - n + i
            want = np.zeros(4, bool)
            want[[x for p, x in blocks if p <= pos and not (b == 0 and p // page == missing)]] = True
            got = np.isnan(o[bt.cu[b] + i])
            assert np.array_equal(got, np.broadcast_to(want[None, :, None], got.shape)), (b, i)
