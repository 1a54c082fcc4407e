"""Rows into a paged cache and back (jl_kv_write_dev, jl_kv_read_dev) against the plain statement of them.

Bars: exact.  16-bit rows are the value rounded to nearest even; 8-bit rows the quantizer's arithmetic in f32 (the quotient by 127, its
reciprocal, halves away from zero), read back as one f32 product rounded to the type asked for.  Nothing else in the pools changes."""
import numpy as np
import pytest

from jitllm_amd import quant
from jitllm_amd.hipmem import DeviceArray, Graph, Stream
from test_gpu_norm_rows import at_offset, bf16_bits, dtype, stored, values

pytestmark = pytest.mark.gpu

KINDS = [quant.F16, quant.BF16, quant.I8]
PLAIN = [quant.F32, quant.F16, quant.BF16]


def as_f32(a, t):
    return values(a, t).astype(np.float32)


def quantized(x):
    """f32 rows -> (int8, f32 scales)."""
    x = x.astype(np.float32)
    amax = np.abs(x).max(-1, keepdims=True)
    step = (amax / np.float32(127)).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        inv = (np.float32(1) / step).astype(np.float32)
        inv = np.where(inv < np.inf, inv, np.float32(0))
        v = (x * inv).astype(np.float64)
    q = np.where(np.isfinite(v), np.sign(v) * np.floor(np.abs(v) + 0.5), 0)
    return q.astype(np.int8), step[..., 0]


class Cache:
    """A cache in device memory beside its statement in numpy: k, v as [n_page][n_kv][page][d] (bits), scales."""

    def __init__(self, t, n_kv, d, page, table, n_page, order="heads", seed=0, gap=0):
        self.t, self.n_kv, self.d, self.page, self.n_page = t, n_kv, d, page, n_page
        self.table = np.ascontiguousarray(table, np.uint32)
        rng = np.random.default_rng(seed)
        shape = (n_page, n_kv, page, d)
        if t == quant.I8:
            self.k, self.v = (rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2))
            self.ks, self.vs = ((0.005 + 0.02 * rng.random(shape[:3])).astype(np.float32) for _ in range(2))
        else:
            self.k, self.v = (stored(rng.standard_normal(shape).astype(np.float32), t) for _ in range(2))
            self.ks = self.vs = None
        self.order, self.row = order, d + gap      # "heads": [page][head][place], "places": [page][place][head]; gap between rows
        self.upload()

    def lay(self, a):
        a = np.concatenate([a, np.full((*a.shape[:3], self.row - self.d), 99, a.dtype)], -1)
        return np.ascontiguousarray(a if self.order == "heads" else a.transpose(0, 2, 1, 3))

    def unlay(self, a):
        return (a if self.order == "heads" else a.transpose(0, 2, 1, 3))[..., : self.d]

    def upload(self):
        self.kd, self.vd, self.td = DeviceArray(self.lay(self.k)), DeviceArray(self.lay(self.v)), DeviceArray(self.table)
        self.ksd, self.vsd = (DeviceArray(s) if s is not None else None for s in (self.ks, self.vs))

    def handle(self, dev, **kw):
        strides = {} if self.order == "heads" and self.row == self.d else \
            dict(row_stride=self.row, head_stride=self.page * self.row, page_stride=self.n_kv * self.page * self.row) if self.order == "heads" else \
            dict(row_stride=self.n_kv * self.row, head_stride=self.row, page_stride=self.n_kv * self.page * self.row)
        return dev.kv_cache(self.t, self.n_kv, self.d, self.page, self.n_page, self.kd.ptr, self.vd.ptr, self.td.ptr, self.table.shape[0],
                            self.table.shape[1], k_scale=self.ksd.ptr if self.ksd else None, v_scale=self.vsd.ptr if self.vsd else None,
                            **{**strides, **kw})

    def place(self, seq, pos):
        """(page, slot), or None."""
        if seq >= self.table.shape[0] or pos // self.page >= self.table.shape[1]:
            return None
        p = int(self.table[seq, pos // self.page])
        return (p, int(pos % self.page)) if p < self.n_page else None

    def write(self, k, v, seq, pos):
        for x, pool, scales in ((k, self.k, self.ks), (v, self.v, self.vs)):
            if x is None:
                continue
            if self.t == quant.I8:
                q, s = quantized(x)
            else:
                with np.errstate(over="ignore"):
                    q, s = stored(x, self.t), None
            for i in range(len(pos)):
                at = self.place(int(seq[i]), int(pos[i]))
                if at:
                    pool[at[0], :, at[1]] = q[i]
                    if s is not None:
                        scales[at[0], :, at[1]] = s[i]

    def read(self, which, seq, pos):
        """f32 rows [n][n_kv][d]."""
        pool, scales = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        out = np.zeros((len(pos), self.n_kv, self.d), np.float32)
        for i in range(len(pos)):
            at = self.place(int(seq[i]), int(pos[i]))
            if at:
                row = pool[at[0], :, at[1]]
                out[i] = row.astype(np.float32) * scales[at[0], :, at[1], None] if self.t == quant.I8 else as_f32(row, self.t)
        return out

    def check(self):
        for d, a, s, sd in ((self.kd, self.k, self.ks, self.ksd), (self.vd, self.v, self.vs, self.vsd)):
            got = d.get()
            assert np.array_equal(self.unlay(got).view(np.uint8), np.ascontiguousarray(a).view(np.uint8))
            if self.row > self.d:
                assert np.all(got[..., self.d:] == got.dtype.type(99))
            if s is not None:
                assert np.array_equal(sd.get().view(np.uint32), s.view(np.uint32))


def table_of(rng, lens, page, spare=1):
    need = [-(-n // page) for n in lens]
    n_page = sum(need) + spare
    order = rng.permutation(n_page).astype(np.uint32)
    table, at = np.full((len(lens), max(max(need), 1)), n_page, np.uint32), 0
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k]
        at += k
    return table, n_page


def same(got, want_f32, t):
    with np.errstate(over="ignore", invalid="ignore"):
        want = stored(want_f32, t)
    if t == quant.BF16:
        nan = np.isnan(want_f32)
        assert np.array_equal(got[~nan], want[~nan]) and np.all((got[nan] & 0x7fff) > 0x7f80)
    else:
        assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("x", PLAIN)
@pytest.mark.parametrize("ntok, n_kv, d, page, order, gap", [(1, 1, 16, 16, "heads", 0), (1, 8, 128, 16, "heads", 0), (37, 3, 64, 16, "places", 0), (50, 5, 80, 32, "heads", 16),
                                                             (20, 2, 256, 64, "places", 16), (9, 7, 192, 16, "heads", 0), (300, 4, 96, 128, "places", 0), (5, 1, 48, 1024, "heads", 0)])
def test_rows_written_and_read(dev, t, x, ntok, n_kv, d, page, order, gap):
    rng = np.random.default_rng(ntok * 1000 + d)
    lens = [max(1, ntok // 2 + 3), ntok + 20, 5]
    table, n_page = table_of(rng, lens, page)
    c = Cache(t, n_kv, d, page, table, n_page, order, gap=gap)
    places = [(s, p) for s, n in enumerate(lens) for p in range(n)]
    pick = rng.permutation(len(places))[:ntok]
    seq, pos = np.array([places[i] for i in pick], np.uint32).T
    k, v = (stored((rng.standard_normal((ntok, n_kv, d)) * rng.choice([0.01, 1, 30], (ntok, n_kv, 1))).astype(np.float32), x) for _ in range(2))
    kd, vd, sd, pd = (DeviceArray(np.ascontiguousarray(a)) for a in (k, v, seq, pos))
    h = c.handle(dev)
    assert dev.kv_write_dev(h, kd.ptr, vd.ptr, x, pd.ptr, ntok, seq=sd.ptr)
    c.write(as_f32(k, x), as_f32(v, x), seq, pos)
    dev.synchronize()
    c.check()
    for to in PLAIN:
        yk, yv = (DeviceArray(np.full((ntok + 1, n_kv, d), 77, dtype(to))) for _ in range(2))
        assert dev.kv_read_dev(h, yk.ptr, yv.ptr, to, pd.ptr, ntok, seq=sd.ptr)
        dev.synchronize()
        for got, which in ((yk.get(), "k"), (yv.get(), "v")):
            same(got[:ntok], c.read(which, seq, pos), to)
            assert np.all(got[ntok] == dtype(to)(77))


def test_tokens_without_a_place(dev):
    """No such sequence, positions behind the table, pages that are none: left alone, and read as zeros."""
    rng = np.random.default_rng(4)
    table = np.array([[2, 0xFFFFFFFF, 1], [4, 3, 77]], np.uint32)          # four pages: 4, 77 and 2^32 - 1 are none
    for t in KINDS:
        c = Cache(t, 2, 64, 16, table, 4)
        seq = np.array([0, 0, 0, 1, 1, 2, 0xFFFFFFFF, 1, 0, 1], np.uint32)
        pos = np.array([3, 20, 40, 5, 20, 0, 0, 47, 48, 0xFFFFFFFF], np.uint32)
        k, v = (rng.standard_normal((10, 2, 64)).astype(np.float32) for _ in range(2))
        kd, vd, sd, pd = (DeviceArray(a) for a in (k, v, seq, pos))
        h = c.handle(dev)
        assert dev.kv_write_dev(h, kd.ptr, vd.ptr, quant.F32, pd.ptr, 10, seq=sd.ptr)
        c.write(k, v, seq, pos)
        y = DeviceArray(np.full((10, 2, 64), 5, np.float32))
        assert dev.kv_read_dev(h, None, y.ptr, quant.F32, pd.ptr, 10, seq=sd.ptr)
        dev.synchronize()
        c.check()
        want = c.read("v", seq, pos)
        assert np.array_equal(y.get(), want) and np.all(want[[1, 3, 5, 6, 7, 8, 9]] == 0) and np.any(want[4] != 0)


def test_one_of_the_two_and_strides(dev):
    """Keys alone, values alone, rows inside a wider fused projection, off 16-byte boundaries; a sequence a token without seq."""
    rng = np.random.default_rng(5)
    for t in KINDS:
        c = Cache(t, 2, 32, 16, np.array([[0], [1], [2]]), 3)
        wide = rng.standard_normal((3, 201)).astype(np.float32)      # q | k | v, k from 65 on: rows at any 4-byte boundary
        buf, at = at_offset(wide, 1)
        pos = np.array([7, 0, 15], np.uint32)
        pd = DeviceArray(pos)
        h = c.handle(dev)
        k = wide[:, 65:129].reshape(3, 2, 32)
        assert dev.kv_write_dev(h, at + 65 * 4, None, quant.F32, pd.ptr, 3, k_stride=201)
        c.write(k, None, range(3), pos)
        dev.synchronize()
        c.check()
        assert dev.kv_write_dev(h, None, at + 129 * 4, quant.F32, pd.ptr, 3, v_stride=201)
        c.write(None, wide[:, 129:193].reshape(3, 2, 32), range(3), pos)
        dev.synchronize()
        c.check()
        out, to = at_offset(np.full((3, 90), 3, np.uint16), 3)
        assert dev.kv_read_dev(h, to + 2 * 11, None, quant.BF16, pd.ptr, 3, k_stride=90)
        dev.synchronize()
        got = out.get()[3:].reshape(3, 90)
        assert np.array_equal(got[:, 11:75].reshape(3, 2, 32), bf16_bits(c.read("k", range(3), pos)))
        assert np.all(got[:, :11] == 3) and np.all(got[:, 75:] == 3)


def test_values_at_the_ends_of_their_types(dev):
    """Halfway values, zeros, rows under 2^-121, the largest f32, infinities and NaN."""
    d = 32
    rows = np.zeros((8, 1, d), np.float32)
    rows[0, 0] = np.arange(d) - 15.5                               # amax 16.5: halves fall on both sides
    rows[1, 0, :4] = [127, 0.5, -0.5, 1.5]                         # step 1: exact halves, away from zero
    rows[3, 0] = 1e-37
    rows[4, 0, :2] = [3.4e38, -1e38]
    rows[5, 0, 3] = np.inf
    rows[6, 0, 3] = np.nan
    rows[7, 0, :3] = [65504, 65519.996, 65520]                     # the border of f16's infinity
    pos = np.arange(8, dtype=np.uint32)
    for t in KINDS:
        c = Cache(t, 1, d, 16, np.array([[0]]), 1)
        kd, pd, sd = DeviceArray(rows), DeviceArray(pos), DeviceArray(np.zeros(8, np.uint32))
        y = DeviceArray(np.zeros_like(rows))
        h = c.handle(dev)
        assert dev.kv_write_dev(h, kd.ptr, kd.ptr, quant.F32, pd.ptr, 8, seq=sd.ptr) and dev.kv_read_dev(h, y.ptr, None, quant.F32, pd.ptr, 8, seq=sd.ptr)
        dev.synchronize()
        got = y.get()
        if t == quant.I8:
            with np.errstate(invalid="ignore"):
                assert np.all(np.isnan(got[5])) and np.all(np.isnan(got[6])) and np.all(got[3] == 0) and np.all(got[2] == 0)
            assert list(got[1, 0, :4]) == [127, 1, -1, 2]
            q, s = quantized(rows)
            for i in (0, 1, 4, 7):
                assert np.array_equal(got[i], q[i].astype(np.float32) * s[i, 0])
        else:
            with np.errstate(over="ignore"):
                same(stored(got, quant.F32), as_f32(stored(rows, t), t) if t != quant.BF16 else np.where(np.isnan(rows), rows, as_f32(bf16_bits(rows), t)), quant.F32)


def test_pools_of_more_than_four_gib(dev):
    """Pages that lie past 32-bit offsets, of bytes and of elements."""
    rng = np.random.default_rng(6)
    n_kv, d, page = 2, 64, 16
    stride = (1 << 32) + 160                                          # elements: 8 GiB and a little between two pages
    big = DeviceArray(shape=((stride + n_kv * d * page) * 2,), dtype=np.uint8)
    table = DeviceArray(np.array([[1, 0]], np.uint32))
    h = dev.kv_cache(quant.F16, n_kv, d, page, 2, big.ptr, big.ptr, table.ptr, 1, 2, page_stride=stride)
    k = rng.standard_normal((20, n_kv, d)).astype(np.float32)
    kd, y, pd, sd = DeviceArray(k), DeviceArray(np.zeros_like(k)), DeviceArray(np.arange(20, dtype=np.uint32)), DeviceArray(np.zeros(20, np.uint32))
    assert dev.kv_write_dev(h, kd.ptr, None, quant.F32, pd.ptr, 20, seq=sd.ptr) and dev.kv_read_dev(h, y.ptr, None, quant.F32, pd.ptr, 20, seq=sd.ptr)
    dev.synchronize()
    assert np.array_equal(y.get(), k.astype(np.float16).astype(np.float32))
    big.free()


def test_captured_and_on_a_stream_of_the_callers(dev):
    """A graph of a write and a read, replayed over new rows and places, between eager calls."""
    rng = np.random.default_rng(8)
    st = Stream()
    table, n_page = table_of(rng, [64, 64, 64], 16)
    c = Cache(quant.I8, 3, 96, 16, table, n_page)
    h = c.handle(dev)
    kd, vd = (DeviceArray(np.zeros((3, 3, 96), np.float32)) for _ in range(2))
    y, pd = DeviceArray(np.zeros((3, 3, 96), np.float32)), DeviceArray(np.zeros(3, np.uint32))

    def calls(s):
        assert dev.kv_write_dev(h, kd.ptr, vd.ptr, quant.F32, pd.ptr, 3, stream=s) and dev.kv_read_dev(h, y.ptr, None, quant.F32, pd.ptr, 3, stream=s)

    try:
        with Graph.capture(st.handle) as g:
            calls(st.handle)
        for i in range(5):
            k, v, pos = rng.standard_normal((3, 3, 96)).astype(np.float32), rng.standard_normal((3, 3, 96)).astype(np.float32), rng.integers(0, 64, 3).astype(np.uint32)
            kd.put(k); vd.put(v); pd.put(pos)
            if i % 2:
                calls(st.handle)
            else:
                g.launch()
            st.synchronize()
            c.write(k, v, range(3), pos)
            c.check()
            assert np.array_equal(y.get(), c.read("k", range(3), pos))
    finally:
        st.destroy()
