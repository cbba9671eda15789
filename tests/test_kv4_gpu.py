"""The block-scaled FP4 key/value cache on the GPU: rows written and read back
bit for bit against the oracle, attention against 64-bit sums over the oracle's
values, with tolerances from the kernels' arithmetic (kv4_oracle.tolerances)."""
import math

import numpy as np
import pytest

import kv4_oracle as K
import oracle as O
from gpu_util import to_dev

pytestmark = pytest.mark.gpu

LONG = 10 ** 6  # a max_len for which sequences are shared by runs of chunks
EPS = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step


@pytest.fixture(autouse=True)
def error_word(tb, cuda):
    """Each test starts with a clear error word and, unless it reads it itself,
    leaves it clear."""
    tb.device_error()
    yield
    assert tb.device_error() == 0


def dtype(torch, typ):
    return torch.float16 if typ == "f16" else torch.bfloat16


def fmt(tb, typ):
    return tb.Format.F16 if typ == "f16" else tb.Format.BF16


class Batch:
    """Sequences of a host cache: lengths, rows, page table, and the device copies."""

    def __init__(self, tb, torch, lens, n, *, page=16, heads=2, dim=64, k_scale=0.011, v_scale=0.007, stride=0, pad=0,
                 typ="f16", seed=0, spare=2, width=None):
        self.tb, self.torch, self.typ = tb, torch, typ
        self.lens, self.n, self.rng = list(lens), list(n), np.random.default_rng(seed)
        per = [-(-x // page) for x in lens]
        self.host = K.Cache(sum(per) + spare, page, heads, dim, k_scale, v_scale, stride, seed=seed + 1)
        order = self.rng.permutation(sum(per) + spare).astype(np.int32)
        self.table = np.full((len(lens), max(width or 0, max(per, default=0), 1)), -5, np.int32)
        at = 0
        for b, p in enumerate(per):
            self.table[b, :p] = order[at:at + p]
            at += p
        self.cu = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        self.total = int(self.cu[-1]) + pad
        self.dev = to_dev(torch, self.host.data)
        self.index()
        self.cache = tb.KV4Cache(self.dev, self.host.pages, page, heads, dim, k_scale, v_scale, stride)

    def index(self):
        t = self.torch
        self.d_cu, self.d_lens, self.d_table = (t.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()
                                                for x in (self.cu, self.lens, self.table))
        self.rows = self.tb.KV4Rows(self.d_cu, self.d_lens, self.d_table, len(self.lens), self.table.shape[1], self.total)

    def place(self, b, pos):
        return self.table[b, pos // self.host.page], pos % self.host.page

    def fill(self, spread=0.5):
        """Write every token of every sequence from normal values, on both sides."""
        h, d = self.host.heads, self.host.dim
        for b, n in enumerate(self.lens):
            for pos in range(n):
                x = self.rng.normal(size=(2, h, d)) * np.exp(spread * self.rng.normal(size=(2, h, 1)))
                self.host.write(*self.place(b, pos), x[0], x[1])
        self.upload()

    def fill_fast(self):
        """Codes of any kind and ordinary scale bytes everywhere a token lies."""
        self.host.data[:] = self.rng.integers(0, 256, self.host.data.shape, dtype=np.uint8)
        for page in range(self.host.pages):
            for h in range(self.host.heads):
                for v in (False, True):
                    b = h * self.host.head_bytes + (self.host.codes + self.host.scales if v else 0) + self.host.codes
                    self.host.data[page, b:b + self.host.scales] = self.rng.integers(0x28, 0x50, self.host.scales)
        self.upload()

    def upload(self):
        self.dev.copy_(self.torch.from_numpy(self.host.data.reshape(-1)))

    def tokens(self, b, is_v):
        """[len, heads, dim] float64 values of a sequence, tensor scale included."""
        g = self.host.v_scale if is_v else self.host.k_scale
        out = np.zeros((self.lens[b], self.host.heads, self.host.dim))
        for pos in range(self.lens[b]):
            out[pos] = self.host.token(*self.place(b, pos), is_v).astype(np.float64) * g
        return out

    def queries(self, q_heads, std=1.0, stride=0):
        t = self.torch
        w = q_heads * self.host.dim
        q = t.from_numpy(self.rng.normal(size=(self.total, w)) * std).to(dtype(t, self.typ)).cuda()
        if stride:
            wide = t.full((self.total, stride), float("nan"), dtype=q.dtype, device="cuda")
            wide[:, :w] = q
            return wide, q
        return q, q

    def attend(self, q, q_heads, scale, window=0, sinks=0, max_rows=None, max_len=None, lse=True, q_stride=0,
               out_stride=0, workspace=None, stream=None):
        t, tb = self.torch, self.tb
        max_rows = max(self.n, default=0) if max_rows is None else max_rows
        max_len = max(self.lens, default=0) if max_len is None else max_len
        out = t.full((self.total, out_stride or q_heads * self.host.dim), 7.0, dtype=dtype(t, self.typ), device="cuda")
        ls = t.full((self.total, q_heads), 7.0, dtype=t.float32, device="cuda") if lse else None
        need = tb.kv4_attention_workspace(self.cache, self.rows, q_heads, max_rows, max_len)
        ws = t.full((max(need, 16),), 0xFF, dtype=t.uint8, device="cuda") if workspace is None else workspace
        tb.kv4_attention(self.cache, self.rows, fmt(tb, self.typ), q, out, ls, q_heads, max_rows, max_len, scale,
                         window=window, sinks=sinks, q_stride=q_stride, out_stride=out_stride, workspace=ws,
                         workspace_bytes=need, stream=stream)
        t.cuda.synchronize()
        return out, ls

    def check(self, out, lse, q, q_heads, scale, window=0, sinks=0):
        """Rows of every sequence against the oracle; rows of nobody untouched."""
        d = self.host.dim
        o = out.double().cpu().numpy()[:, :q_heads * d].reshape(self.total, q_heads, d)
        ls = None if lse is None else lse.double().cpu().numpy()
        qq = q.double().cpu().numpy()[:, :q_heads * d].reshape(self.total, q_heads, d)
        for b, n in enumerate(self.n):
            r = slice(self.cu[b], self.cu[b] + n)
            want = K.attention(self.tokens(b, False), self.tokens(b, True), qq[r], self.lens[b] - n, scale, window, sinks)
            t_out, t_lse = K.tolerances(*want, self.lens[b], d, EPS[self.typ])
            err = np.abs(o[r] - want[0])
            assert np.all(np.isfinite(o[r])) and np.all(err <= t_out), \
                f"sequence {b}: out off by {np.max(err - t_out):.3g} more than allowed at {np.argwhere(err > t_out)[:3]}"
            if ls is None:
                continue
            seen = np.isfinite(want[1])
            assert np.array_equal(np.isneginf(ls[r]), ~seen)
            assert np.all(np.abs(ls[r][seen] - want[1][seen]) <= t_lse[seen])
        assert np.all(o[self.cu[-1]:] == 7.0)
        if ls is not None:
            assert np.all(ls[self.cu[-1]:] == 7.0)

    def run(self, q_heads, scale=None, std=1.0, **kw):
        """Both ways of sharing a sequence: short (clusters) and long (runs of
        chunks), chosen by max_len."""
        scale = self.host.dim ** -0.5 if scale is None else scale
        q, dense = self.queries(q_heads, std)
        for max_len in (kw.pop("max_len", None), LONG):
            out, lse = self.attend(q, q_heads, scale, max_len=max_len, **kw)
            self.check(out, lse, dense, q_heads, scale, kw.get("window", 0), kw.get("sinks", 0))


# ---- append ------------------------------------------------------------------------------

def to_bits(x, typ):
    """float32 array -> (values as the type holds them, torch-ready 16-bit words)."""
    if typ == "f16":
        h = x.astype(np.float16)
        return h.astype(np.float64), h.view(np.int16)
    b = x.astype(np.float32).view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    r = np.where(np.isnan(x), np.uint16(0x7FC0), r)
    return (r.astype(np.uint32) << 16).view(np.float32).astype(np.float64), r.view(np.int16)


def append_and_compare(bt, x, stride_extra=0):
    """x [total, 2, heads, dim] float32; the device cache afterwards equals the host's."""
    t, h, d = bt.torch, bt.host.heads, bt.host.dim
    val, words = to_bits(x, bt.typ)
    row = 2 * h * d + stride_extra
    buf = t.full((bt.total, row), -1, dtype=t.int16, device="cuda")
    buf[:, :2 * h * d] = t.from_numpy(words.reshape(bt.total, -1).copy()).cuda()
    base = buf.data_ptr()
    bt.tb.kv4_append(bt.cache, bt.rows, fmt(bt.tb, bt.typ), base, base + 2 * h * d, k_stride=row, v_stride=row)
    t.cuda.synchronize()
    for b, n in enumerate(bt.n):
        for i in range(n):
            pos = bt.lens[b] - n + i
            bt.host.write(*bt.place(b, pos), val[bt.cu[b] + i, 0], val[bt.cu[b] + i, 1])
    got = bt.dev.cpu().numpy().reshape(bt.host.data.shape)
    np.testing.assert_array_equal(got, bt.host.data)


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("lens,n,page,heads,dim,pad,stride", [
    ([1], [1], 16, 1, 16, 0, 0),
    ([5, 0, 17, 33], [5, 0, 1, 20], 16, 2, 64, 3, 0),
    ([40, 129, 64], [40, 1, 64], 64, 3, 128, 0, 0),
    ([70], [69], 32, 1, 80, 0, 32 * 90 + 160),
    ([9, 31], [9, 2], 128, 2, 256, 1, 0),
    ([300, 513, 1], [300, 400, 1], 32, 8, 128, 0, 0),  # the kernel with many rows a CTA
    ([1000], [999], 16, 5, 240, 0, 0),
])
def test_append_matches_oracle(tb, cuda, typ, lens, n, page, heads, dim, pad, stride):
    bt = Batch(tb, cuda, lens, n, page=page, heads=heads, dim=dim, typ=typ, stride=stride, pad=pad, seed=dim + len(lens))
    x = bt.rng.normal(size=(bt.total, 2, heads, dim)) * np.exp(1.5 * bt.rng.normal(size=(bt.total, 2, heads, 1)))
    x[:, :, :, : 16] *= 0.001  # a block of small values beside ordinary ones
    append_and_compare(bt, x.astype(np.float32), stride_extra=8)


def test_append_more_rows_than_one_cta_per_sm(tb, cuda):
    """Enough rows for the many-row kernel, whose last CTA is ragged."""
    bt = Batch(tb, cuda, [5000, 37], [4999, 37], page=64, heads=2, dim=32, typ="bf16", seed=3)
    append_and_compare(bt, bt.rng.normal(size=(bt.total, 2, 2, 32)).astype(np.float32))


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("g", [1.0, 0.125, 2.0 ** -9, 0.0137])
def test_append_at_the_borders(tb, cuda, typ, g):
    """Values on and next to the borders between codes and between scales, with
    scales for which the borders are numbers of the type; zeros of both signs,
    subnormals, infinities and NaN."""
    heads, dim = 4, 128
    bt = Batch(tb, cuda, [600], [600], page=16, heads=heads, dim=dim, typ=typ, k_scale=g, v_scale=g, seed=11)
    x = bt.rng.normal(size=(600, 2, heads, dim)).astype(np.float32)
    blk = x.reshape(-1, 16)
    steps = O.e4m3_scale_values()[:127].astype(np.float64)
    mids = (steps[1:] + steps[:-1]) / 2
    with np.errstate(over="ignore"):
        for i in range(blk.shape[0]):
            s = steps[1 + i % 126]
            what = i % 5
            if what == 0:    # the largest value on a scale's border or one step of the type beside it
                top = 6 * g * mids[(i // 5) % 126]
                blk[i] *= top / 8
                blk[i, i % 16] = top * (1 + [0, 2.0 ** -8, -2.0 ** -8, 2.0 ** -10, -2.0 ** -10][(i // 7) % 5])
            elif what == 1:  # a block of scale s whose values lie on the codes' borders
                blk[i] = g * s * np.concatenate([K.MIDS, -K.MIDS, [6, -6]])
            elif what == 2:  # beside them
                f = 1 + [2.0 ** -8, -2.0 ** -8, 2.0 ** -10, -2.0 ** -10][(i // 5) % 4]
                blk[i] = g * s * np.concatenate([K.MIDS * f, -K.MIDS * f, [6, 6]])
            elif what == 3:
                blk[i] *= 10.0 ** bt.rng.uniform(-8, 5)
            else:
                blk[i] = [[0.0] * 16, [-0.0] * 16, [1e-7] * 16, [np.inf] + [1.0] * 15, [np.nan] + [2.0] * 15,
                          [-np.inf] * 16, [np.nan] * 16, [3e38] * 16, [-1e-40] * 16][(i // 5) % 9]
        append_and_compare(bt, x)


def test_append_leaves_out_what_has_no_place(tb, cuda):
    """A page outside the cache, a slot outside the table, more rows than
    tokens, rows outside `rows`: nothing is written there, the rest is, and the
    error word says so."""
    bt = Batch(tb, cuda, [40, 20, 50, 30], [40, 20, 50, 30], page=16, heads=2, dim=64, seed=5)
    bt.table[0, 1] = bt.host.pages      # tokens 16..31 of sequence 0
    bt.table[1, 0] = -1                 # tokens 0..15 of sequence 1
    bt.lens[2] = 30                     # 50 rows for 30 tokens
    bt.total -= 5                       # the last five rows are outside
    bt.index()
    x = bt.rng.normal(size=(bt.total, 2, 2, 64)).astype(np.float32)
    val, words = to_bits(x, "f16")
    dev = cuda.from_numpy(words.copy()).cuda()
    tb.kv4_append(bt.cache, bt.rows, tb.Format.F16, dev.data_ptr(), dev.data_ptr() + 2 * 2 * 64, k_stride=256, v_stride=256)
    assert tb.device_error() == 2
    # cu's end passes `rows`: sequence 3 has 25 rows, its last 25 tokens
    for b, (n, ln) in enumerate([(40, 40), (20, 20), (50, 30), (25, 30)]):
        for i in range(n):
            pos = ln - n + i
            if pos < 0 or not 0 <= bt.table[b, pos // 16] < bt.host.pages:
                continue
            bt.host.write(*bt.place(b, pos), val[bt.cu[b] + i, 0], val[bt.cu[b] + i, 1])
    np.testing.assert_array_equal(bt.dev.cpu().numpy().reshape(bt.host.data.shape), bt.host.data)


# ---- read back ---------------------------------------------------------------------------

def expect_read(bt, b, i, is_v):
    """The row's values as the output type: FP32 product, rounded once."""
    g = np.float32(bt.host.v_scale if is_v else bt.host.k_scale)
    x = bt.host.token(*bt.place(b, bt.lens[b] - bt.n[b] + i), is_v) * g
    return bt.torch.from_numpy(x.astype(np.float32)).to(dtype(bt.torch, bt.typ)).float().numpy()


def read_and_compare(bt, stride_extra=0):
    t, h, d = bt.torch, bt.host.heads, bt.host.dim
    w = h * d + stride_extra
    out = [t.full((bt.total, w), 7.0, dtype=dtype(t, bt.typ), device="cuda") for _ in range(2)]
    bt.tb.kv4_read(bt.cache, bt.rows, fmt(bt.tb, bt.typ), out[0], out[1], k_stride=w, v_stride=w)
    t.cuda.synchronize()
    for is_v in (False, True):
        got = out[is_v].float().cpu().numpy()
        want = np.full_like(got, 7.0)
        for b, n in enumerate(bt.n):
            for i in range(n):
                want[bt.cu[b] + i, :h * d] = expect_read(bt, b, i, is_v).reshape(-1)
        np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("lens,n,page,heads,dim,pad,extra", [
    ([1], [1], 16, 1, 16, 0, 0),
    ([5, 0, 17, 33], [5, 0, 1, 20], 16, 2, 64, 3, 8),
    ([40, 129, 64], [40, 129, 64], 64, 3, 128, 0, 0),
    ([70], [69], 32, 1, 80, 0, 16),
    ([9, 31], [9, 2], 128, 2, 256, 1, 0),
    ([2500, 513], [2500, 511], 32, 8, 128, 2, 0),
])
def test_read_matches_oracle(tb, cuda, typ, lens, n, page, heads, dim, pad, extra):
    bt = Batch(tb, cuda, lens, n, page=page, heads=heads, dim=dim, typ=typ, pad=pad, seed=dim)  # any bytes at all
    read_and_compare(bt, extra)


def test_read_every_code_and_scale(tb, cuda):
    """One page of 1024 tokens: every code byte under every scale byte."""
    bt = Batch(tb, cuda, [1024], [1024], page=1024, heads=8, dim=128, k_scale=1.0, v_scale=3.7, spare=0)
    c = np.arange(256, dtype=np.uint8)
    for h in range(8):
        for is_v in (False, True):
            b = h * bt.host.head_bytes + (bt.host.codes + bt.host.scales if is_v else 0)
            n = 1024 * 8  # blocks of 16
            blk = np.arange(n) + h * n
            bt.host.data[0, b + bt.host.codes:b + bt.host.codes + n] = (blk // 32).astype(np.uint8)
            bt.host.data[0, b:b + n * 8] = c[(8 * blk[:, None] + np.arange(8)) % 256].reshape(-1)
    bt.upload()
    read_and_compare(bt)


def test_read_leaves_out_what_has_no_place(tb, cuda):
    bt = Batch(tb, cuda, [40, 20], [40, 20], page=16, heads=2, dim=64, seed=6)
    bt.table[0, 2] = 1 << 30
    bt.lens[1] = 12
    bt.index()
    k, v = (cuda.full((60, 128), 7.0, dtype=cuda.float16, device="cuda") for _ in range(2))
    tb.kv4_read(bt.cache, bt.rows, tb.Format.F16, k, v)
    assert tb.device_error() == 2
    assert bool((k[32:40] == 7).all()) and bool((v[40:48] == 7).all())
    assert not bool((k[:32] == 7).all(dim=1).any()) and not bool((v[48:] == 7).all(dim=1).any())


# ---- attention ---------------------------------------------------------------------------

@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("heads,q_heads", [(1, 1), (2, 8), (1, 7), (2, 32)])
def test_step_lengths(tb, cuda, typ, dim, page, heads, q_heads):
    """One row per sequence, lengths around the chunks, the warps and the pages."""
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 65, 255, 257, 300]
    bt = Batch(tb, cuda, lens, [1] * len(lens), page=page, heads=heads, dim=dim, typ=typ, seed=dim + page + q_heads, pad=2)
    bt.fill_fast()
    bt.run(q_heads)


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_step_split(tb, cuda, typ, dim, page):
    """Sequences long enough to be shared by several CTAs, beside short ones."""
    lens = [2600, 1, 40, 0, 1500, 1025]
    bt = Batch(tb, cuda, lens, [1, 1, 1, 0, 1, 1], page=page, heads=2, dim=dim, typ=typ, seed=page)
    bt.fill_fast()
    assert tb.kv4_attention_workspace(bt.cache, bt.rows, 8, 1, LONG) > 0
    bt.run(8)


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("n", [2, 3, 4, 5, 8, 9, 16, 17, 33])
def test_few_rows(tb, cuda, typ, n):
    """2 to 33 rows of 4 heads: one, two and four tiles of eight, and several of 32."""
    bt = Batch(tb, cuda, [n, n + 1, 100, 1300, 50], [n, n, n, n, 1], page=16, heads=2, dim=128, typ=typ, seed=n, pad=1)
    bt.fill_fast()
    bt.run(8)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (32, 4), (33, 31), (100, 33), (1000, 0), (1, 5000),
                                          (2 ** 31 - 1, 2 ** 31 - 1), (0, 9)])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_window_and_sinks(tb, cuda, dim, window, sinks, n):
    lens = [n, 64 + n, 301, 1200]
    bt = Batch(tb, cuda, lens, [n] * 4, page=32, heads=1, dim=dim, seed=window % 1000 + sinks % 1000 + n)
    bt.fill_fast()
    bt.run(4, window=window, sinks=sinks)


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("dim,page,heads,q_heads,window,sinks", [
    (64, 16, 2, 8, 0, 0), (128, 64, 1, 4, 0, 0), (128, 16, 2, 2, 0, 0), (64, 128, 1, 7, 50, 3), (128, 32, 1, 8, 130, 0)])
def test_prompts(tb, cuda, typ, dim, page, heads, q_heads, window, sinks):
    """Whole prompts, a chunk behind cached tokens, a single row, an idle sequence."""
    bt = Batch(tb, cuda, [130, 300, 257, 90, 20], [130, 100, 257, 1, 0], page=page, heads=heads, dim=dim, typ=typ, seed=dim,
               pad=5)
    bt.fill_fast()
    bt.run(q_heads, window=window, sinks=sinks)


@pytest.mark.parametrize("page,dim", [(64, 128), (256, 64), (1024, 128), (128, 128), (16, 64)])
def test_long_prompt(tb, cuda, page, dim):
    """Row tiles of 256 and tokens shared by several CTAs, pages below and above the tile."""
    bt = Batch(tb, cuda, [1500], [700], page=page, heads=1, dim=dim, typ="bf16", seed=2)
    bt.fill_fast()
    bt.run(2)


@pytest.mark.parametrize("batch", [40, 700, 2100])
def test_unlike_sequences(tb, cuda, batch):
    """Many single rows, some idle sequences, and prompts of one to several row
    tiles among them, the first and the last included."""
    n = [1 if b % 9 else 0 for b in range(batch)]
    lens = [5 + b % 40 for b in range(batch)]
    for b, rows, length in ((0, 40, 50), (7, 600, 600), (8, 130, 700), (batch // 2, 9, 300), (batch - 1, 300, 310)):
        n[b], lens[b] = rows, length
    bt = Batch(tb, cuda, lens, n, page=32, heads=1, dim=64, typ="bf16", seed=batch, pad=2)
    bt.fill_fast()
    bt.run(4)


@pytest.mark.parametrize("n", [1, 40])
def test_cache_of_many_gigabytes(tb, cuda, n):
    """Pages 700 MB apart, so that offsets pass 32 bits: written, read, attended."""
    apart = 700 * 2 ** 20
    bt = Batch(tb, cuda, [70 + n, 90], [n, n], page=16, heads=2, dim=64, seed=80 + n, spare=0)
    bt.fill()
    far = cuda.empty((bt.host.pages, apart), dtype=cuda.uint8, device="cuda")
    size = bt.host.stride
    small = cuda.from_numpy(bt.host.data[:, :size].copy()).cuda()
    assert far.numel() > 2 ** 32
    far[:, :size] = small
    far[:, size:size + 4096] = 0xA5
    bt.cache = tb.KV4Cache(far, bt.host.pages, 16, 2, 64, bt.host.k_scale, bt.host.v_scale, apart)
    bt.run(8)
    val, words = to_bits(bt.rng.normal(size=(bt.total, 2, 2, 64)).astype(np.float32), "f16")
    kv = cuda.from_numpy(words).cuda()
    tb.kv4_append(bt.cache, bt.rows, tb.Format.F16, kv.data_ptr(), kv.data_ptr() + 256, k_stride=256, v_stride=256)
    for b in range(2):
        for i in range(n):
            bt.host.write(*bt.place(b, bt.lens[b] - n + i), *val[bt.cu[b] + i])
    assert np.array_equal(far[:, :size].cpu().numpy(), bt.host.data)
    assert bool((far[:, size:size + 4096] == 0xA5).all())
    read_and_compare(bt)
    bt.run(8)


@pytest.mark.parametrize("n", [33, 127, 128, 129, 255, 256, 257, 300])
def test_row_tiles(tb, cuda, n):
    """One query head per KV head: rows around the tiles of 128 and 256."""
    bt = Batch(tb, cuda, [n, n + 77], [n, n], page=32, heads=1, dim=64, seed=n, pad=1)
    bt.fill_fast()
    bt.run(1)


@pytest.mark.parametrize("n", [1, 3, 40])
def test_peaked_and_flat_scores(tb, cuda, n):
    """Scores of hundreds, where all weight lies on one token, scores near zero,
    and a negative scale."""
    bt = Batch(tb, cuda, [700, 1400], [n, n], page=16, heads=1, dim=64, seed=21)
    bt.fill_fast()
    bt.run(4, std=20.0)
    bt.run(4, std=1e-4)
    bt.run(4, scale=-0.3)
    bt.run(4, scale=0.0)


def test_rising_scores(tb, cuda):
    """Keys that grow along the sequence, so that the running maximum moves often."""
    bt = Batch(tb, cuda, [1200, 500], [1, 40], page=16, heads=1, dim=64, k_scale=1.0, seed=22)
    bt.fill_fast()
    for b, n in enumerate(bt.lens):
        for pos in range(n):
            page, place = bt.place(b, pos)
            cs, ss = bt.host.parts(page, 0, place, False)
            bt.host.data[page, cs], bt.host.data[page, ss] = 0x22, 0x20 + pos // 40
    bt.upload()
    q, dense = bt.queries(4)
    q.abs_()
    for max_len in (None, LONG):
        out, lse = bt.attend(q, 4, 1.0, max_len=max_len)
        bt.check(out, lse, q, 4, 1.0)


@pytest.mark.parametrize("magnitude", [2.0 ** 100, 2.0 ** 15, 2.0 ** -60, 2.0 ** -120])
def test_bf16_queries_outside_fp16(tb, cuda, magnitude):
    """BF16 rows far outside FP16's range, each of its own magnitude."""
    for n in (1, 40):
        bt = Batch(tb, cuda, [200, 80], [n, n], page=16, heads=1, dim=128, typ="bf16", seed=23)
        bt.fill_fast()
        q, _ = bt.queries(4)
        q *= magnitude
        q[0, :128] = 0.0
        scale = 0.05 / magnitude
        out, lse = bt.attend(q, 4, scale)
        bt.check(out, lse, q, 4, float(np.float32(scale)))


@pytest.mark.parametrize("max_len", [None, LONG])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_what_lies_behind_a_sequence_is_not_seen(tb, cuda, max_len, n):
    """NaN scales behind the sequences' ends, in unused pages and in unused
    table entries change nothing."""
    lens = [n + 5, 100, 1203]
    bt = Batch(tb, cuda, lens, [n] * 3, page=64, heads=2, dim=128, seed=31)
    bt.fill_fast()
    q, _ = bt.queries(4)
    first = [x.clone() for x in bt.attend(q, 4, 0.1, max_len=max_len)]
    used = {(int(bt.table[b, p // 64]), p % 64) for b in range(3) for p in range(lens[b])}
    for page in range(bt.host.pages):
        for place in range(64):
            if (page, place) not in used:
                for h in range(2):
                    for v in (False, True):
                        cs, ss = bt.host.parts(page, h, place, v)
                        bt.host.data[page, ss] = 0x7F + 0x80 * (place & 1)
    bt.upload()
    again = bt.attend(q, 4, 0.1, max_len=max_len)
    assert cuda.equal(first[0], again[0]) and cuda.equal(first[1], again[1])
    bt.check(*again, q, 4, 0.1)


@pytest.mark.parametrize("max_len", [None, LONG])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("n,others", [(1, 0), (3, 0), (40, 0), (40, 6)])
def test_nan_tokens_reach_the_rows_that_see_them(tb, cuda, max_len, where, n, others):
    """A cached NaN block is seen or hidden like any other token."""
    window, sinks = 50, 2
    lens = [400, 1300]
    bt = Batch(tb, cuda, lens + [30] * others, [n, n] + [1] * others, page=16, heads=1, dim=128, seed=33)
    bt.fill_fast()
    bad = {0: [1, 200, 345, 360, 399], 1: [0, 100, 1251]}  # positions
    for b, ps in bad.items():
        for p in ps:
            page, place = bt.place(b, p)
            cs, ss = bt.host.parts(page, 0, place, where == "v")
            bt.host.data[page, ss.start + 2] = 0x7F  # values 32..47
    bt.upload()
    q, _ = bt.queries(2)
    out, lse = bt.attend(q, 2, 0.1, window=window, sinks=sinks, max_len=max_len)
    o = out.float().cpu().numpy().reshape(-1, 2, 128)
    for b in range(2):
        for i in range(n):
            pos = lens[b] - n + i
            seen = [p for p in bad[b] if K.sees(pos, p, window, sinks)]
            row = o[bt.cu[b] + i]
            nan = np.zeros(128, bool)
            if seen:
                nan[(slice(None) if where == "k" else slice(32, 48))] = True
            np.testing.assert_array_equal(np.isnan(row), np.broadcast_to(nan, row.shape), err_msg=f"{b} {i}")
            ls = lse[bt.cu[b] + i].cpu().numpy()
            assert np.all(np.isnan(ls)) if seen and where == "k" else np.all(np.isfinite(ls))
    # without them: the hidden ones change nothing in rows that see none
    ok = ~np.isnan(o).any(axis=(1, 2))
    for b, ps in bad.items():
        for p in ps:
            page, place = bt.place(b, p)
            cs, ss = bt.host.parts(page, 0, place, where == "v")
            bt.host.data[page, ss.start + 2] = 0x30
    bt.upload()
    clean = bt.attend(q, 2, 0.1, window=window, sinks=sinks, max_len=max_len)[0].float().cpu().numpy().reshape(-1, 2, 128)
    np.testing.assert_array_equal(o[ok], clean[ok])


@pytest.mark.parametrize("max_len", [None, LONG])
@pytest.mark.parametrize("n", [1, 40])
def test_nan_queries_stay_in_their_rows(tb, cuda, max_len, n):
    bt = Batch(tb, cuda, [80, 1400], [n, n], page=16, heads=1, dim=64, typ="bf16", seed=34)
    bt.fill_fast()
    q, _ = bt.queries(2)
    clean = bt.attend(q, 2, 0.1, max_len=max_len)[0].clone()
    q[n, 3] = float("nan")
    out, lse = bt.attend(q, 2, 0.1, max_len=max_len)
    assert bool(out[n, :64].isnan().all()) and bool(lse[n, 0].isnan())
    same = cuda.ones_like(out, dtype=cuda.bool)
    same[n, :64] = False
    assert cuda.equal(out[same], clean[same])


@pytest.mark.parametrize("max_len", [None, LONG])
@pytest.mark.parametrize("n", [2, 40])
def test_rows_that_see_nothing(tb, cuda, max_len, n):
    """More rows than tokens: the rows before the first token are zero, lse -inf.
    Sequences without tokens."""
    bt = Batch(tb, cuda, [5, 0, 3], [5, 0, 3], page=16, heads=1, dim=64, seed=35)
    bt.fill_fast()
    bt.n, bt.lens = [n, n, 0], [1, 0, 3]
    bt.cu = np.array([0, n, 2 * n, 2 * n], np.int32)
    bt.total = 2 * n + 1
    bt.index()
    q, _ = bt.queries(2)
    out, lse = bt.attend(q, 2, 0.1, max_len=max_len)
    bt.check(out, lse, q, 2, 0.1)
    assert bool((out[:n - 1] == 0).all()) and bool(cuda.isneginf(lse[:n - 1]).all())
    assert bool((out[n:2 * n] == 0).all()) and bool((out[2 * n:] == 7).all())


@pytest.mark.parametrize("max_len", [None, LONG])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_pages_outside_the_cache_are_not_seen(tb, cuda, max_len, n):
    lens = [100, 1500]
    bt = Batch(tb, cuda, lens, [n, n], page=16, heads=1, dim=64, seed=36)
    bt.fill_fast()
    q, _ = bt.queries(2)
    good = bt.table.copy()
    bt.table[0, 2], bt.table[1, 5], bt.table[1, 60] = bt.host.pages, -1, 2 ** 31 - 1
    bt.index()
    out, lse = bt.attend(q, 2, 0.1, max_len=max_len)
    assert tb.device_error() == 2
    for b, hidden in ((0, [2]), (1, [5, 60])):
        keep = [p for p in range(lens[b]) if p // 16 not in hidden]
        bt.table[:] = good
        k, v = bt.tokens(b, False)[keep], bt.tokens(b, True)[keep]
        for i in range(n):
            pos = lens[b] - n + i
            m = sum(1 for p in keep if p <= pos)
            qq = q[bt.cu[b] + i].double().cpu().numpy().reshape(1, 2, 64)
            want = K.attention(k[:m], v[:m], qq, m - 1, 0.1)
            t_out, t_lse = K.tolerances(*want, lens[b], 64, EPS["f16"])
            got = out[bt.cu[b] + i].double().cpu().numpy().reshape(1, 2, 64)
            assert np.all(np.abs(got - want[0]) <= t_out)


@pytest.mark.parametrize("max_len", [None, LONG])
@pytest.mark.parametrize("gone", ["none", "other"])
@pytest.mark.parametrize("n,page", [(1, 16), (1, 64), (3, 32), (40, 16), (40, 32), (300, 16)])
def test_pages_out_of_sight_may_be_gone(tb, cuda, max_len, gone, n, page):
    """Entries of pages behind the window: no page, or one of NaN blocks that
    another sequence holds.  The results stay and nothing is reported."""
    window, sinks = 70, 5
    lens = [1500, 777 + n]
    bt = Batch(tb, cuda, lens, [n, n], page=page, heads=2, dim=64, seed=37, spare=1)
    bt.fill_fast()
    free = next(p for p in range(bt.host.pages) if p not in bt.table)
    bt.host.data[free] = 0x7F
    bt.upload()
    q, _ = bt.queries(4)
    want = bt.attend(q, 4, 0.1, window=window, sinks=sinks, max_len=max_len)
    for b in range(2):
        oldest = lens[b] - n - window + 1
        for slot in range(-(-lens[b] // page)):
            if slot * page >= sinks and (slot + 1) * page <= oldest:
                bt.table[b, slot] = -1 if gone == "none" else free
    bt.index()
    got = bt.attend(q, 4, 0.1, window=window, sinks=sinks, max_len=max_len)
    assert cuda.equal(got[0], want[0]) and cuda.equal(got[1], want[1])


def test_lengths_outside_the_table(tb, cuda):
    """A length that passes the table or is negative: the error word, and rows
    of the other sequences as before."""
    bt = Batch(tb, cuda, [100, 64, 90], [1, 1, 1], page=16, heads=1, dim=64, seed=37)
    bt.fill_fast()
    q, _ = bt.queries(2)
    out0 = bt.attend(q, 2, 0.1)[0].clone()
    for bad in (10 ** 9, -4, 2 ** 31 - 1, -2 ** 31):
        for max_len in (100, LONG):
            bt.d_lens[1] = bad
            out, _ = bt.attend(q, 2, 0.1, max_len=max_len)
            assert tb.device_error() == 2
            same = (out[::2].float() - out0[::2].float()).abs().max().item()
            assert same <= 2 * 2.0 ** -10 * out0.abs().max().item()


def test_more_rows_than_max_rows_is_reported(tb, cuda):
    bt = Batch(tb, cuda, [2000, 90], [40, 40], page=16, heads=1, dim=64, seed=38)
    bt.fill_fast()
    q, _ = bt.queries(2)
    for max_len in (100, LONG):
        bt.attend(q, 2, 0.1, max_rows=1, max_len=max_len)
        assert tb.device_error() == 4


@pytest.mark.parametrize("max_rows,max_len", [(1, 64), (1, 10 ** 6), (9, 10 ** 6), (100, 10), (100, 10 ** 6)])
def test_bounds_may_be_loose(tb, cuda, max_rows, max_len):
    """max_len only steers the split, max_rows may be larger than any."""
    bt = Batch(tb, cuda, [1800, 70], [1, 1], page=16, heads=2, dim=64, seed=39)
    bt.fill_fast()
    bt.run(4, max_rows=max_rows, max_len=max_len)


@pytest.mark.parametrize("max_len", [None, LONG])
@pytest.mark.parametrize("n", [1, 6, 40])
def test_strides_and_no_lse(tb, cuda, max_len, n):
    bt = Batch(tb, cuda, [60, 1300], [n, n], page=32, heads=2, dim=64, stride=2 * 32 * 72 + 4096, seed=40, pad=1)
    bt.fill_fast()
    wide, q = bt.queries(4, stride=4 * 64 + 24)
    out, _ = bt.attend(wide, 4, 0.125, lse=False, q_stride=4 * 64 + 24, out_stride=4 * 64 + 40, max_len=max_len)
    bt.check(out, None, q, 4, 0.125)
    assert bool((out[:, 256:] == 7).all())


@pytest.mark.parametrize("max_len", [2100, LONG])
@pytest.mark.parametrize("n", [1, 6, 40])
def test_same_bits_again_and_in_a_graph(tb, cuda, n, max_len):
    """Two runs, a captured one and its replays give the same bits; a replay
    follows the lengths, rows and table that the device holds then."""
    bt = Batch(tb, cuda, [900, 2100, 30], [n, n, n], page=16, heads=2, dim=128, seed=41)
    bt.fill_fast()
    q, _ = bt.queries(8)
    out0, lse0 = (x.clone() for x in bt.attend(q, 8, 0.09, max_len=max_len))
    out1, lse1 = bt.attend(q, 8, 0.09, max_len=max_len)
    assert cuda.equal(out0, out1) and cuda.equal(lse0, lse1)
    need = tb.kv4_attention_workspace(bt.cache, bt.rows, 8, n, max_len)
    ws = cuda.empty(max(need, 16), dtype=cuda.uint8, device="cuda")
    out, lse = cuda.zeros_like(out0), cuda.zeros_like(lse0)
    s = cuda.cuda.Stream()
    graph = cuda.cuda.CUDAGraph()
    s.wait_stream(cuda.cuda.current_stream())
    with cuda.cuda.graph(graph, stream=s):
        tb.kv4_attention(bt.cache, bt.rows, tb.Format.F16, q, out, lse, 8, n, max_len, 0.09, workspace=ws,
                         workspace_bytes=need)
    graph.replay()
    cuda.cuda.synchronize()
    assert cuda.equal(out0, out) and cuda.equal(lse0, lse)
    bt.lens = [700, 2000, 29]
    bt.d_lens.copy_(cuda.tensor(bt.lens, dtype=cuda.int32))
    graph.replay()
    graph.replay()
    cuda.cuda.synchronize()
    bt.check(out, lse, q, 8, 0.09)
    # the eager call follows too
    out1, lse1 = bt.attend(q, 8, 0.09, max_len=max_len)
    assert cuda.equal(out, out1) and cuda.equal(lse, lse1)


@pytest.mark.parametrize("max_len", [None, LONG])
@pytest.mark.parametrize("n", [1, 6, 40, 300])
def test_out_over_the_queries(tb, cuda, max_len, n):
    """out may be q itself."""
    bt = Batch(tb, cuda, [n + 400, n + 20, 90], [n, n, 1], page=16, heads=2, dim=128, seed=95, pad=1)
    bt.fill_fast()
    q, _ = bt.queries(8)
    out, lse = bt.attend(q, 8, 0.09, max_len=max_len)
    need = tb.kv4_attention_workspace(bt.cache, bt.rows, 8, n, max_len or max(bt.lens))
    ws = cuda.full((max(need, 16),), 0xFF, dtype=cuda.uint8, device="cuda")
    both, lse2 = q.clone(), cuda.full_like(lse, 7.0)
    tb.kv4_attention(bt.cache, bt.rows, tb.Format.F16, both, both, lse2, 8, n, max_len or max(bt.lens), 0.09,
                     workspace=ws, workspace_bytes=need)
    assert cuda.equal(both[:-1], out[:-1]) and cuda.equal(lse, lse2) and cuda.equal(both[-1], q[-1])


def test_generation_in_one_graph(tb, cuda):
    """A step of a generation, captured once: a token written, then attended.
    Each replay reads the lengths, the pages and the new values from the device."""
    bt = Batch(tb, cuda, [31, 140], [1, 1], page=16, heads=2, dim=128, seed=90, spare=4)
    bt.fill()
    val, words = to_bits(bt.rng.normal(size=(3, 2, 2, 2, 128)).astype(np.float32), "f16")
    kv = cuda.from_numpy(words[0].copy()).cuda()
    q, _ = bt.queries(8)
    out = cuda.full((2, 1024), 7.0, dtype=cuda.float16, device="cuda")
    lse = cuda.full((2, 8), 7.0, dtype=cuda.float32, device="cuda")
    need = tb.kv4_attention_workspace(bt.cache, bt.rows, 8, 1, LONG)
    ws = cuda.full((need,), 0xFF, dtype=cuda.uint8, device="cuda")

    def step(stream):
        tb.kv4_append(bt.cache, bt.rows, tb.Format.F16, kv, kv.data_ptr() + 512, k_stride=512, v_stride=512, stream=stream)
        tb.kv4_attention(bt.cache, bt.rows, tb.Format.F16, q, out, lse, 8, 1, LONG, 0.09, workspace=ws,
                         workspace_bytes=need, stream=stream)

    side = cuda.cuda.Stream()
    graph = cuda.cuda.CUDAGraph()
    cuda.cuda.synchronize()
    with cuda.cuda.graph(graph, stream=side):
        step(side)
    free = [p for p in range(bt.host.pages) if p not in bt.table]
    for i in range(3):
        if i:
            bt.lens = [x + 1 for x in bt.lens]
            for b in range(2):
                if (bt.lens[b] - 1) % 16 == 0:
                    at = (bt.lens[b] - 1) // 16
                    if at == bt.table.shape[1]:
                        pytest.fail("the table is too narrow")
                    bt.table[b, at] = free.pop()
            bt.d_lens.copy_(cuda.tensor(bt.lens, dtype=cuda.int32))
            bt.d_table.copy_(cuda.from_numpy(bt.table))
            kv.copy_(cuda.from_numpy(words[i].copy()))
        for b in range(2):
            bt.host.write(*bt.place(b, bt.lens[b] - 1), *val[i, b])
        graph.replay()
        cuda.cuda.synchronize()
        bt.check(out, lse, q, 8, 0.09)


def test_streams_side_by_side(tb, cuda):
    """Calls on two streams at once, a workspace each."""
    bts = [Batch(tb, cuda, [3000, 50 + i], [1, 1], page=16, heads=2, dim=128, seed=50 + i) for i in range(2)]
    for bt in bts:
        bt.fill_fast()
    qs = [bt.queries(8)[0] for bt in bts]
    need = tb.kv4_attention_workspace(bts[0].cache, bts[0].rows, 8, 1, LONG)
    outs = [cuda.zeros((2, 1024), dtype=cuda.float16, device="cuda") for _ in bts]
    wss = [cuda.empty(need, dtype=cuda.uint8, device="cuda") for _ in bts]
    cuda.cuda.synchronize()
    streams = [cuda.cuda.Stream() for _ in bts]
    for _ in range(20):
        for bt, q, out, ws, st in zip(bts, qs, outs, wss, streams):
            tb.kv4_attention(bt.cache, bt.rows, tb.Format.F16, q, out, None, 8, 1, LONG, 0.09, workspace=ws,
                             workspace_bytes=need, stream=st)
    cuda.cuda.synchronize()
    for bt, q, out in zip(bts, qs, outs):
        bt.check(out, None, q, 8, 0.09)


def test_workspace_is_asked_for(tb, cuda):
    bt = Batch(tb, cuda, [3000], [1], page=16, heads=1, dim=64, seed=60)
    q, _ = bt.queries(2)
    need = tb.kv4_attention_workspace(bt.cache, bt.rows, 2, 1, LONG)
    assert need > 0
    out = cuda.zeros((1, 128), dtype=cuda.float16, device="cuda")
    ws = cuda.empty(need + 16, dtype=cuda.uint8, device="cuda")
    for w, nb, st in ((None, 0, "WORKSPACE"), (ws, need - 1, "WORKSPACE"), (ws.data_ptr() + 4, need, "ALIGNMENT")):
        with pytest.raises(tb.TBError) as e:
            tb.kv4_attention(bt.cache, bt.rows, tb.Format.F16, q, out, None, 2, 1, LONG, 0.1, workspace=w, workspace_bytes=nb)
        assert e.value.status == tb.Status[st]


def test_workspace_of_a_padded_batch(tb, cuda):
    """Rows of nobody, far more than the others, do not swell the workspace."""
    bt = Batch(tb, cuda, [1500], [20], page=16, heads=2, dim=64, seed=61, pad=9000)
    bt.fill_fast()
    assert tb.kv4_attention_workspace(bt.cache, bt.rows, 8, 20, LONG) < 64 * 2 ** 20
    bt.run(8)


@pytest.mark.parametrize("typ", ["f16", "bf16"])
def test_prompt_then_steps(tb, cuda, typ):
    """The operators together, as a generation runs them: a prompt's rows are
    written and attend, then rows one by one; then the cache is read back."""
    heads, qh, dim, page = 2, 8, 128, 16
    final = [45, 130]
    bt = Batch(tb, cuda, final, final, page=page, heads=heads, dim=dim, typ=typ, seed=70)
    lens = [40, 125]
    x = bt.rng.normal(size=(sum(final), 2, heads, dim)).astype(np.float32)
    val, words = to_bits(x, typ)
    start = np.concatenate([[0], np.cumsum(final)])
    for step in range(6):
        bt.n = list(lens) if step == 0 else [1, 1]
        bt.lens = [n + step for n in lens]
        bt.cu = np.concatenate([[0], np.cumsum(bt.n)]).astype(np.int32)
        bt.total = int(bt.cu[-1])
        bt.index()
        take = np.concatenate([np.arange(bt.lens[b] - bt.n[b], bt.lens[b]) + start[b] for b in range(2)])
        kv = cuda.from_numpy(words[take].copy()).cuda()
        base = kv.data_ptr()
        tb.kv4_append(bt.cache, bt.rows, fmt(tb, typ), base, base + 2 * heads * dim, k_stride=2 * heads * dim,
                      v_stride=2 * heads * dim)
        for b in range(2):
            for i in range(bt.n[b]):
                bt.host.write(*bt.place(b, bt.lens[b] - bt.n[b] + i), *val[take[bt.cu[b] + i]])
        bt.run(qh)
    bt.n = list(bt.lens)
    bt.cu = np.concatenate([[0], np.cumsum(bt.n)]).astype(np.int32)
    bt.total = int(bt.cu[-1])
    bt.index()
    read_and_compare(bt)
    # the values that came in are near the values held: 4 bits and a scale per 16
    k, v = (cuda.zeros((bt.total, heads * dim), dtype=dtype(cuda, typ), device="cuda") for _ in range(2))
    tb.kv4_read(bt.cache, bt.rows, fmt(tb, typ), k, v)
    take = np.concatenate([np.arange(bt.lens[b]) + start[b] for b in range(2)])
    want = val[take, 0].reshape(bt.total, -1)
    assert O.rel_frob(k.float().cpu().numpy(), want) < 0.15
    # a page's codes and scales are what tb_decode_nvfp4 reads
    page0 = int(bt.table[0, 0])
    part = bt.dev[page0 * bt.host.stride:][:bt.host.codes]
    sc = bt.dev[page0 * bt.host.stride + bt.host.codes:][:bt.host.scales]
    dec = cuda.empty(page * dim, dtype=cuda.float16, device="cuda")
    tb.decode_nvfp4(part, sc, dec, page * dim)
    want = np.stack([bt.host.token(page0, p, False)[0] for p in range(page)]).reshape(-1)
    np.testing.assert_array_equal(dec.float().cpu().numpy(), want)
