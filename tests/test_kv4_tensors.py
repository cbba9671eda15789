"""Which tensors the cache's Python structures take."""
import pytest

torch = pytest.importorskip("torch")


def test_index_arrays_are_dense_int32(tb):
    n = torch.tensor([3, 1, 4], dtype=torch.int32)
    cu = torch.zeros(4, dtype=torch.int32)
    cu[1:] = n.cumsum(0)
    lens, table = torch.full((3,), 20, dtype=torch.int32), torch.arange(6, dtype=torch.int32).view(3, 2)
    r = tb.KV4Rows(cu, lens, table, 3, 2, 8)
    assert (r.cu_rows, r.seq_lens, r.block_table) == (cu.data_ptr(), lens.data_ptr(), table.data_ptr())
    with pytest.raises(ValueError, match="cu_rows must be int32"):
        tb.KV4Rows(torch.cat([n[:1] * 0, n]).cumsum(0), lens, table, 3, 2, 8)  # int64
    with pytest.raises(ValueError, match="seq_lens must be int32"):
        tb.KV4Rows(cu, lens.float(), table, 3, 2, 8)
    with pytest.raises(ValueError, match="block_table must be int32"):
        tb.KV4Rows(cu, lens, table.long(), 3, 2, 8)
    wide = torch.arange(15, dtype=torch.int32).view(3, 5)
    with pytest.raises(ValueError, match="block_table must be contiguous"):
        tb.KV4Rows(cu, lens, wide[:, :2], 3, 2, 8)
    with pytest.raises(ValueError, match="seq_lens must be contiguous"):
        tb.KV4Rows(cu, torch.zeros(6, dtype=torch.int32)[::2], table, 3, 2, 8)
    for kw in (dict(cu=cu[:3]), dict(lens=lens[:2]), dict(table=table[:2])):
        a = dict(cu=cu, lens=lens, table=table) | kw
        with pytest.raises(ValueError, match="fewer than"):
            tb.KV4Rows(a["cu"], a["lens"], a["table"], 3, 2, 8)
    # an idle batch needs none of them
    tb.KV4Rows(None, None, None, 0, 0, 0)
    tb.KV4Rows(cu[:0], lens[:0], table[:0], 0, 2, 8)


def test_pages_lie_where_the_cache_looks(tb):
    size = tb.kv4_page_bytes(16, 2, 64)
    dense = torch.zeros(5, size, dtype=torch.uint8)
    assert tb.KV4Cache(dense, 5, 16, 2, 64).data == dense.data_ptr()
    tb.KV4Cache(dense.view(-1), 5, 16, 2, 64)
    tb.KV4Cache(dense.view(torch.int32), 5, 16, 2, 64)
    with pytest.raises(ValueError, match="fewer than 6 pages"):
        tb.KV4Cache(dense, 6, 16, 2, 64)
    # the pages of one layer among those of three
    layers = torch.zeros(5, 3, size, dtype=torch.uint8)
    c = tb.KV4Cache(layers[:, 1], 5, 16, 2, 64, page_stride=3 * size)
    assert c.data == layers.data_ptr() + size
    for bad in (dict(), dict(page_stride=2 * size)):
        with pytest.raises(ValueError, match="apart"):
            tb.KV4Cache(layers[:, 1], 5, 16, 2, 64, **bad)
    with pytest.raises(ValueError, match="apart"):
        tb.KV4Cache(layers[:, :, ::2], 5, 16, 2, 64)
    # dense, with room behind each page; the last one may end without it
    tb.KV4Cache(layers.view(-1)[:4 * 3 * size + size], 5, 16, 2, 64, page_stride=3 * size)
    with pytest.raises(ValueError, match="fewer than 5 pages"):
        tb.KV4Cache(layers.view(-1)[:4 * 3 * size], 5, 16, 2, 64, page_stride=3 * size)
    tb.KV4Cache(None, 0, 16, 2, 64)
