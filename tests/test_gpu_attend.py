"""Attention of new tokens over a paged cache (jl_attend_dev) against the definition in 64 bits over the cache's own bits.

Bars, with u = 2^-24 (half a step of f32).  A score is scale * (q . k) in f32: d products and their sums round, q's pieces keep 22 bits at least
(f16 and int8 caches: two of eleven; 24 over bf16), the factors of scale, log2 e and an int8 row's scale round once each:
    E = scale * sum |q k| * (d u + 2^-22 + 8 u)                              (a cap adds cap * 2^-21: tanh by an exponential of 2^-23 and a quotient)
A weight e^(s - m) carries E twice (s and m), the subtraction's and the exponential's roundings, 4 u (1 + |s|), and its pieces: 2^-21 (f16), 2^-16 (two
of bf16) or 2^-23 (three).  Its smallest in f16 lie 2^-38 under the largest.  Sums of n weights in f32: a quarter of the positions a wavefront, in every piece
a product of its own, joined in at most 512 parts, so (3 n / 4 + 600) u.  With A = sum w |v| / sum w, numerator and denominator together:
    |out - want| <= A * (2 (2 E + 4 u (1 + |s|)) + pieces + 2 (3 n / 4 + 600) u) + n 2^-38 max |v| + half a step of out's type."""
import numpy as np
import pytest

from jitllm_amd import quant
from jitllm_amd.device import Device
from jitllm_amd.hipmem import DeviceArray, Graph, Stream, mem_info
from test_gpu_kv_cache import KINDS, PLAIN, Cache, table_of
from test_gpu_norm_rows import STEP, at_offset, dtype, stored, values

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(c, q, seq, length, scale, window=0, cap=0.0, sink=None):
    """out, its bar, lse, its bar: [ntok][n_head][d] and [ntok][n_head]; q as numbers."""
    ntok, n_head, d = q.shape
    group = n_head // c.n_kv
    out, bar = np.zeros((ntok, n_head, d)), np.zeros((ntok, n_head, d))
    lse, lbar = np.full((ntok, n_head), -np.inf), np.zeros((ntok, n_head))
    bf = c.t == quant.BF16
    scale = float(np.float32(scale))
    for t in range(ntok):
        s, n = int(seq[t]), int(length[t])
        if s >= c.table.shape[0]:
            n = 0
        n = min(n, c.table.shape[1] * c.page)
        lo = max(0, n - window) if window else 0
        pos = np.array([p for p in range(lo, n) if c.table[s, p // c.page] < c.n_page], np.int64)
        if pos.size:
            pages, slots = c.table[s, pos // c.page].astype(np.int64), pos % c.page
            num = lambda a: (a.astype(np.float64) if c.t == quant.I8 else values(a, c.t))
            k, v = num(c.k[pages, :, slots]), num(c.v[pages, :, slots])
            if c.t == quant.I8:
                k, v = k * c.ks[pages, :, slots][..., None].astype(np.float64), v * c.vs[pages, :, slots][..., None].astype(np.float64)
        for h in range(n_head):
            x, e = np.zeros(0), np.zeros(0)
            if pos.size:
                kh, vh, qh = k[:, h // group], v[:, h // group], q[t, h].astype(np.float64)
                x, e = scale * (kh @ qh), abs(scale) * (np.abs(kh) @ np.abs(qh)) * (d * U + 2.0 ** -22 + 8 * U)
                if cap:
                    x, e = cap * np.tanh(x / cap), e + cap * 2.0 ** -21
            full = x if sink is None else np.append(x, np.float64(sink[h]))
            if not full.size:
                continue
            m = full.max()
            w = np.exp(x - m)
            total = np.exp(full - m).sum()
            big, far = (e.max() if e.size else 0.0), max(np.abs(full).max(), 0.0)
            rel = 2 * big + 4 * U * (1 + far)
            sums = (0.75 * pos.size + 600) * U
            lse[t, h] = m + np.log(total)
            lbar[t, h] = rel + sums + 4 * U * abs(lse[t, h]) + 2.0 ** -22
            if pos.size:
                out[t, h] = w @ vh / total
                a = w @ np.abs(vh) / total
                bar[t, h] = a * (2 * rel + (2.0 ** -16 if bf else 2.0 ** -21) + 2 * sums) + pos.size * 2.0 ** -38 * np.abs(vh).max()
    return out, bar, lse, lbar


def run(dev, c, q, qt, ot, seq, length, scale, window=0, cap=0.0, sink=None, want_lse=True, stream=None, **kw):
    ntok, n_head, d = q.shape
    qd, ld = DeviceArray(stored(q.astype(np.float32), qt)), DeviceArray(np.ascontiguousarray(length, np.uint32))
    sd = None if seq is None else DeviceArray(np.ascontiguousarray(seq, np.uint32))
    out, lse = DeviceArray(np.full((ntok + 1, n_head, d), 77, dtype(ot))), DeviceArray(np.full((ntok + 1, n_head), 77, np.float32))
    snk = None if sink is None else DeviceArray(np.ascontiguousarray(sink, np.float32))
    assert dev.attend_dev(c.handle(dev), out.ptr, qd.ptr, n_head, ld.ptr, ntok, scale, seq=sd.ptr if sd else None, q_type=qt, out_type=ot, window=window,
                          softcap=cap, sink=snk.ptr if snk else None, lse=lse.ptr if want_lse else None, stream=stream, **kw)
    dev.synchronize()
    got, gl = out.get(), lse.get()
    assert np.all(got[ntok] == dtype(ot)(77)) and np.all(gl[ntok] == 77)
    return values(got[:ntok], ot), gl[:ntok].astype(np.float64)


def check(got, lse, ref, ot):
    out, bar, wl, lbar = ref
    small = 2.0 ** -25 if ot == quant.F16 else 2.0 ** -130
    with np.errstate(invalid="ignore"):
        off = np.abs(got - out) - (bar + (np.abs(out) + bar) * STEP[ot] + small)
    assert not np.any(np.isnan(got)) and np.all(off <= 0), (float(np.nanmax(off)), np.argwhere(~(off <= 0))[:5])
    if lse is not None:
        fine = np.isfinite(wl)
        assert np.array_equal(lse[~fine], wl[~fine])
        assert np.all(np.abs(lse[fine] - wl[fine]) <= lbar[fine])


def attend(dev, t, lens, seq, length, n_kv, group, d, qt=quant.F32, ot=quant.F32, page=16, order="heads", gap=0, seed=0, peak=1.0, **kw):
    rng = np.random.default_rng(seed + 17 * d + n_kv)
    table, n_page = table_of(rng, lens, page)
    c = Cache(t, n_kv, d, page, table, n_page, order, seed, gap)
    q = values(stored((peak * rng.standard_normal((len(length), n_kv * group, d))).astype(np.float32), qt), qt)
    sink = rng.standard_normal(n_kv * group).astype(np.float32) if kw.pop("sinks", False) else None
    scale = 1 / np.sqrt(d)
    got, lse = run(dev, c, q, qt, ot, seq, length, scale, sink=sink, **kw)
    check(got, lse, reference(c, q, range(len(length)) if seq is None else seq, length, scale, kw.get("window", 0), kw.get("cap", 0.0), sink), ot)


# every type of cache, query and result, a token a sequence
@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("qt", PLAIN)
@pytest.mark.parametrize("ot", PLAIN)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_types(dev, t, qt, ot, d):
    lens = [1, 37, 300]
    attend(dev, t, lens, None, lens, 2, 4, d, qt, ot, peak=2.0)


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("d", [16, 32, 48, 80, 96, 112, 160, 192, 240])
def test_row_widths(dev, t, d):
    lens = [1, 15, 16, 17, 129, 260]
    attend(dev, t, lens, None, lens, 3, 2, d)


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 15, 16, 17, 32, 33, 48])
def test_heads_that_share(dev, t, group):
    lens = [5, 200, 64]
    attend(dev, t, lens, None, lens, 2, group, 64 if group > 8 else 128, ot=quant.BF16 if group == 3 else quant.F32)


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("page, order, gap", [(16, "places", 0), (32, "heads", 16), (64, "places", 32), (256, "heads", 0), (4096, "heads", 0)])
def test_pages_and_strides(dev, t, page, order, gap):
    lens = [1, 31, 32, 33, 127, 128, 129, 1000]
    attend(dev, t, lens, None, lens, 2, 4, 96, page=page, order=order, gap=gap)


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("n", [2, 16, 128, 5000, 20011])
def test_lengths_of_one_sequence(dev, t, n):
    attend(dev, t, [n], None, [n], 2, 4, 64, peak=2.0)


@pytest.mark.parametrize("t", KINDS)
def test_many_sequences_and_workgroups(dev, t):
    """More units than workgroups, and cuts through most of them."""
    rng = np.random.default_rng(3)
    lens = [int(v) for v in rng.integers(1, 500, 300)] + [7001]
    attend(dev, t, lens, None, lens, 4, 2, 64, page=32)


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("window", [1, 16, 100, 128, 1000])
def test_windows_and_sinks(dev, t, window):
    lens = [1, 90, 128, 513, 2000]
    attend(dev, t, lens, None, lens, 2, 8, 64, window=window, sinks=True, ot=quant.BF16)


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("cap", [5.0, 50.0])
def test_caps(dev, t, cap):
    lens = [3, 400]
    attend(dev, t, lens, None, lens, 2, 2, 128, cap=cap, peak=8.0)


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("per, group, d", [(2, 4, 128), (5, 2, 256), (5, 2, 64), (7, 1, 96), (3, 16, 64), (20, 4, 64), (70, 1, 128), (33, 5, 128), (50, 4, 192)])
def test_several_tokens_of_a_sequence(dev, t, per, group, d):
    """Drafted tokens and prompts: token i of a sequence sees its own position and those before."""
    lens = [per, per + 1, per + 130, per + 500]
    seq = np.repeat(np.arange(4), per)
    length = np.concatenate([np.arange(n - per, n) + 1 for n in lens])
    attend(dev, t, lens, seq, length, 2, group, d, qt=quant.BF16 if d == 64 else quant.F32)
    attend(dev, t, lens, seq, length, 2, group, d, window=40, sinks=True)


@pytest.mark.parametrize("t", KINDS)
def test_tokens_in_any_order(dev, t):
    """Sequences mixed, lengths that differ within a sequence, the same token twice, and an encoder's states seen in full by all."""
    rng = np.random.default_rng(9)
    lens = [300, 40, 1]
    seq = rng.integers(0, 3, 61)
    length = np.array([rng.integers(0, lens[s] + 1) for s in seq])
    attend(dev, t, lens, seq, length, 2, 3, 64)
    attend(dev, t, lens, np.repeat([0, 1, 2], [20, 9, 4]), np.repeat(lens, [20, 9, 4]), 2, 3, 128)


@pytest.mark.parametrize("t", KINDS)
def test_rows_that_see_nothing(dev, t):
    """Length zero, no such sequence, all pages missing, a page missing in the middle, lengths behind the table."""
    rng = np.random.default_rng(10)
    table = np.array([[0, 9, 2, 3], [9, 9, 0xFFFFFFFF, 9], [4, 5, 6, 7], [1, 8, 9, 9]], np.uint32)     # nine pages: 9 is none
    c = Cache(t, 2, 64, 32, table, 9)
    seq, length = [0, 1, 2, 2, 3, 4, 0xFFFFFFFF, 0, 2], [100, 128, 0, 0xFFFFFFFF, 128, 5, 7, 33, 129]
    for sink in (None, rng.standard_normal(6).astype(np.float32)):
        q = rng.standard_normal((9, 6, 64)).astype(np.float32)
        got, lse = run(dev, c, q, quant.F32, quant.F32, seq, length, 0.2, sink=sink)
        check(got, lse, reference(c, q, seq, length, 0.2, sink=sink), quant.F32)
        for t0 in (1, 2, 5, 6):
            assert np.all(got[t0] == 0) and np.all(lse[t0] == (-np.inf if sink is None else sink))


@pytest.mark.parametrize("t", KINDS)
def test_what_is_hidden_may_be_anything(dev, t):
    """NaN and infinities in places that no token sees, and in places that only later tokens of a prompt see: those alone have NaN."""
    rng = np.random.default_rng(11)
    table, n_page = table_of(rng, [50, 90], 16)
    c = Cache(t, 2, 64, 16, table, n_page)
    seq, length = np.array([0] * 6 + [1] * 6), np.array([41, 42, 43, 44, 45, 46, 60, 61, 62, 63, 64, 65])
    q = rng.standard_normal((12, 4, 64)).astype(np.float32)
    ref = reference(c, q, seq, length, 0.125)

    def spoil(s, p, bad):
        pg, at = c.place(s, p)
        for pool, scales in ((c.k, c.ks), (c.v, c.vs)):
            if t == quant.I8:
                scales[pg, :, at] = bad
            else:
                pool[pg, :, at] = stored(np.full((2, 64), bad, np.float32), t)

    for p in range(46, 50):
        spoil(0, p, np.nan)
    for p in range(66, 90):
        spoil(1, p, [np.inf, np.nan, -np.inf][p % 3])
    c.upload()
    got, lse = run(dev, c, q, quant.F32, quant.F32, seq, length, 0.125)
    check(got, lse, ref, quant.F32)
    spoil(0, 43, np.nan)          # seen by tokens of length 44 and more
    spoil(1, 62, np.nan)
    c.upload()
    got, lse = run(dev, c, q, quant.F32, quant.F32, seq, length, 0.125)
    clean = (length <= 43) | ((seq == 1) & (length <= 62))
    check(got[clean], lse[clean], [a[clean] for a in ref], quant.F32)
    assert np.all(np.isnan(got[~clean]))


@pytest.mark.parametrize("t", [quant.F16, quant.BF16])
def test_large_and_small_values(dev, t):
    """Scores far apart, values at the ends of the type, queries from 1e-20 to 1e4."""
    rng = np.random.default_rng(12)
    table, n_page = table_of(rng, [700], 16)
    c = Cache(t, 1, 128, 16, table, n_page)
    c.v = stored(values(c.v, t).astype(np.float32) * rng.choice([1e-7, 1.0, 3e4 / 6], c.v.shape[:3] + (1,)).astype(np.float32), t)
    c.upload()
    for size in (1e-20, 1e-3, 30.0, 1e4):
        q = (size * rng.standard_normal((1, 4, 128))).astype(np.float32)
        got, lse = run(dev, c, q, quant.F32, quant.F32, None, [700], 0.0884)
        check(got, lse, reference(c, q, [0], [700], 0.0884), quant.F32)


def test_scales_of_an_int8_cache_far_apart(dev):
    rng = np.random.default_rng(13)
    table, n_page = table_of(rng, [900, 33], 16)
    c = Cache(quant.I8, 2, 64, 16, table, n_page)
    c.vs = (c.vs * 2.0 ** rng.integers(-40, 30, c.vs.shape)).astype(np.float32)
    c.vs[table[1, 0]] = 0
    c.upload()
    q = rng.standard_normal((2, 6, 64)).astype(np.float32)
    got, lse = run(dev, c, q, quant.F32, quant.F32, None, [900, 33], 0.125)
    check(got, lse, reference(c, q, [0, 1], [900, 33], 0.125), quant.F32)


def test_strides_of_q_and_out(dev):
    """A query inside a wider projection, a result into one, off 16-byte boundaries."""
    rng = np.random.default_rng(14)
    table, n_page = table_of(rng, [100, 50, 3], 16)
    for ot, off in ((quant.F32, 1), (quant.BF16, 3), (quant.F16, 0)):
        c = Cache(quant.F16, 2, 64, 16, table, n_page)
        wide = rng.standard_normal((3, 512)).astype(np.float32)
        qd, ld = DeviceArray(wide), DeviceArray(np.array([100, 50, 3], np.uint32))
        out, at = at_offset(np.full((3, 301), 7, dtype(ot)), off)
        assert dev.attend_dev(c.handle(dev), at, qd.ptr + 4 * 64, 4, ld.ptr, 3, 0.125, q_stride=512, out_type=ot, out_stride=301)
        dev.synchronize()
        got = out.get()[off:].reshape(3, 301)
        assert np.all(got[:, 256:] == dtype(ot)(7))
        check(values(got[:, :256], ot).reshape(3, 4, 64), None, reference(c, wide[:, 64:320].reshape(3, 4, 64), range(3), [100, 50, 3], 0.125), ot)


def test_pools_of_more_than_four_gib(dev):
    rng = np.random.default_rng(15)
    n_kv, d, page = 2, 64, 16
    stride = (1 << 32) + 160
    big = DeviceArray(shape=((stride + n_kv * d * page) * 2,), dtype=np.uint8)
    table = DeviceArray(np.array([[1, 0]], np.uint32))
    small = Cache(quant.F16, n_kv, d, page, np.array([[1, 0]]), 2)
    h = dev.kv_cache(quant.F16, n_kv, d, page, 2, big.ptr, big.ptr, table.ptr, 1, 2, page_stride=stride)
    small.v = small.k
    rows, pos, seq = values(small.k, quant.F16), np.arange(32, dtype=np.uint32), np.zeros(32, np.uint32)
    rows = np.ascontiguousarray(np.concatenate([rows[1], rows[0]], 1).transpose(1, 0, 2).astype(np.float32))
    rd, pd, sd = DeviceArray(rows), DeviceArray(pos), DeviceArray(seq)
    assert dev.kv_write_dev(h, rd.ptr, None, quant.F32, pd.ptr, 32, seq=sd.ptr)
    q = rng.standard_normal((1, 4, d)).astype(np.float32)
    qd, ld, out = DeviceArray(q), DeviceArray(np.array([32], np.uint32)), DeviceArray(np.zeros_like(q))
    assert dev.attend_dev(h, out.ptr, qd.ptr, 4, ld.ptr, 1, 0.125)
    dev.synchronize()
    check(out.get().astype(np.float64), None, reference(small, q, [0], [32], 0.125), quant.F32)
    big.free()


def test_captured_replayed_and_on_other_streams(dev):
    """A graph over growing lengths, replayed between eager calls of other shapes on the same workspace; the same bits as eager."""
    rng = np.random.default_rng(16)
    table, n_page = table_of(rng, [3000, 200], 32)
    c, st = Cache(quant.I8, 2, 128, 32, table, n_page), Stream()
    q = rng.standard_normal((2, 8, 128)).astype(np.float32)
    qd, ld, out = DeviceArray(q), DeviceArray(np.array([5, 5], np.uint32)), DeviceArray(np.zeros_like(q))
    h = c.handle(dev)
    other = Cache(quant.BF16, 3, 64, 16, np.array([[0, 1, 2]]), 3)
    dev.reserve_attend(256)
    call = lambda s: dev.attend_dev(h, out.ptr, qd.ptr, 8, ld.ptr, 2, 0.1, stream=s)
    try:
        with Graph.capture(st.handle) as g:
            assert call(st.handle)
        for i, length in enumerate(([1, 1], [3000, 200], [128, 129], [0, 7], [2047, 3], [2048, 100])):
            ld.put(np.array(length, np.uint32))
            q = rng.standard_normal((2, 8, 128)).astype(np.float32)
            qd.put(q)
            g.launch()
            st.synchronize()
            first = out.get()
            check(first.astype(np.float64), None, reference(c, q, [0, 1], length, 0.1), quant.F32)
            attend(dev, quant.BF16, [100 + i, 40], None, [100 + i, 40], 3, 2, 64)
            out.put(np.zeros_like(first))
            assert call(st.handle)
            st.synchronize()
            assert np.array_equal(out.get().view(np.uint32), first.view(np.uint32))
    finally:
        st.destroy()
    del other


def test_a_reserved_workspace_and_two_launches():
    with Device(device=0) as d:
        d.reserve_attend(256)
        table, n_page = table_of(np.random.default_rng(1), [4000] * 8, 64)
        for dim, t in ((64, quant.I8), (128, quant.F16), (256, quant.BF16)):
            c = Cache(t, 4, dim, 64, table, n_page)
            q, ld = DeviceArray(np.ones((8, 16, dim), np.float32)), DeviceArray(np.full(8, 4000, np.uint32))
            out = DeviceArray(np.zeros((8, 16, dim), np.float32))
            before, n = mem_info()[0], d.launch_count()
            assert d.attend_dev(c.handle(d), out.ptr, q.ptr, 16, ld.ptr, 8, 0.1)
            d.synchronize()
            assert mem_info()[0] == before and d.launch_count() - n <= 2


def test_a_token_alone_and_among_others(dev):
    """The same token in calls of its own and of many: the definition's value each time."""
    rng = np.random.default_rng(18)
    lens = [700, 20, 1300, 64]
    table, n_page = table_of(rng, lens, 16)
    c = Cache(quant.BF16, 2, 128, 16, table, n_page)
    q = rng.standard_normal((4, 8, 128)).astype(np.float32)
    ref = reference(c, q, range(4), lens, 0.09)
    got, lse = run(dev, c, q, quant.F32, quant.F32, None, lens, 0.09)
    check(got, lse, ref, quant.F32)
    for t in range(4):
        got, lse = run(dev, c, q[t:t + 1], quant.F32, quant.F32, [t], [lens[t]], 0.09)
        check(got, lse, [a[t:t + 1] for a in ref], quant.F32)


@pytest.fixture(params=[1, 2], ids=["units whole", "shares"])
def form(dev, request):
    """Which of the two ways more than sixteen columns a unit are divided among the workgroups."""
    dev.set_tuning(attend__whole=request.param)
    yield request.param
    dev.set_tuning(attend__whole=0)


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("per, group, d", [(16, 2, 64), (17, 1, 80), (33, 4, 128), (64, 1, 256), (130, 2, 48), (9, 8, 192)])
def test_prompts_in_both_divisions(dev, form, t, per, group, d):
    """Units that end inside a sequence, sequences that end inside a unit, the last unit short; with and without what came before the prompt."""
    lens = [per, per + 1, per + 200, per + 63, per + 64]
    seq = np.repeat(np.arange(5), per)
    length = np.concatenate([np.arange(n - per, n) + 1 for n in lens])
    attend(dev, t, lens, seq, length, 2, group, d, qt=quant.F16, ot=quant.BF16)
    attend(dev, t, lens, seq, length, 2, group, d, window=50, sinks=True, cap=20.0)
    n = 3 * per // 2
    attend(dev, t, lens, seq[:n], length[:n], 2, group, d)


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("ot", PLAIN)
def test_prompts_of_each_type_in_both_divisions(dev, form, t, ot):
    lens = [90, 70]
    seq, length = np.repeat([0, 1], [60, 70]), np.concatenate([np.arange(31, 91), np.arange(1, 71)])
    for qt in PLAIN:
        attend(dev, t, lens, seq, length, 3, 2, 128, qt, ot)


@pytest.mark.parametrize("t", KINDS)
def test_hidden_places_in_both_divisions(dev, form, t):
    """A prompt whose later positions hold NaN: only the tokens that see them have it.  Tokens that see nothing between those that do."""
    rng = np.random.default_rng(21)
    table, n_page = table_of(rng, [300, 80], 16)
    c = Cache(t, 2, 64, 16, table, n_page)
    seq, length = np.repeat([0, 1], [100, 40]), np.concatenate([np.arange(170, 270), np.arange(31, 71)])
    length[[3, 50, 120]] = 0
    seq[[7, 130]] = 9
    q = rng.standard_normal((140, 4, 64)).astype(np.float32)
    ref = reference(c, q, seq, length, 0.125)
    for s, p in [(0, 200), (0, 257), (0, 269), (0, 275), (1, 60), (1, 71), (1, 79)]:
        pg, at = c.place(s, p)
        for pool, scales in ((c.k, c.ks), (c.v, c.vs)):
            if t == quant.I8:
                scales[pg, :, at] = np.nan
            else:
                pool[pg, :, at] = stored(np.full((2, 64), np.nan, np.float32), t)
    c.upload()
    got, lse = run(dev, c, q, quant.F32, quant.F32, seq, length, 0.125)
    clean = (seq == 9) | ((seq == 0) & (length <= 200)) | ((seq == 1) & (length <= 60))
    check(got[clean], lse[clean], [a[clean] for a in ref], quant.F32)
    assert np.all(np.isnan(got[~clean])) and np.all(got[[3, 50, 120, 7, 130]] == 0)


def test_prompts_on_a_stream_of_the_callers(dev, form):
    """More than sixteen columns a unit captured and replayed over other lengths, between eager calls; the same bits as eager."""
    rng = np.random.default_rng(22)
    table, n_page = table_of(rng, [600, 300], 32)
    c, st = Cache(quant.BF16, 2, 128, 32, table, n_page), Stream()
    seq = np.repeat([0, 1], 45)
    q = stored(rng.standard_normal((90, 8, 128)).astype(np.float32), quant.BF16)
    qd, sd, ld, out = DeviceArray(q), DeviceArray(seq.astype(np.uint32)), DeviceArray(np.ones(90, np.uint32)), DeviceArray(np.zeros((90, 8, 128), np.uint16))
    h = c.handle(dev)
    dev.reserve_attend(128)
    call = lambda s: dev.attend_dev(h, out.ptr, qd.ptr, 8, ld.ptr, 90, 0.1, seq=sd.ptr, q_type=quant.BF16, out_type=quant.BF16, stream=s)
    try:
        with Graph.capture(st.handle) as g:
            assert call(st.handle)
        for n in (45, 300, 64, 128):
            length = np.concatenate([np.arange(2 * n - 45, 2 * n) + 1, np.arange(n - 45, n) + 1])
            ld.put(length.astype(np.uint32))
            g.launch()
            st.synchronize()
            first = out.get()
            check(values(first, quant.BF16), None, reference(c, values(q, quant.BF16), seq, length, 0.1), quant.BF16)
            attend(dev, quant.F16, [70], np.zeros(40, int), np.arange(31, 71), 2, 2, 64)
            out.put(np.zeros_like(first))
            assert call(st.handle)
            st.synchronize()
            assert np.array_equal(out.get(), first)
    finally:
        st.destroy()


@pytest.mark.parametrize("per", [1, 24])
def test_weights_of_an_int8_cache_are_split_as_they_are_rounded(dev, per):
    """Tens of thousands of weights that each count, over scales of every size: where a weight times its row's scale falls next to a half step of f16, its two pieces
    still add up to it."""
    rng = np.random.default_rng(40)
    lens = [12 + per] * (64 // per + 1)
    table, n_page = table_of(rng, lens, 16)
    c = Cache(quant.I8, 8, 64, 16, table, n_page)
    c.k[:] //= 16
    c.vs[:] = 0.01 + 0.03 * rng.random(c.vs.shape)
    c.upload()
    seq = np.repeat(np.arange(len(lens)), per)
    length = np.concatenate([np.arange(12, 12 + per) + 1 for _ in lens])
    q = rng.standard_normal((len(seq), 64, 64)).astype(np.float32)
    got, lse = run(dev, c, q, quant.F32, quant.F32, seq, length, 0.125)
    check(got, lse, reference(c, q, seq, length, 0.125), quant.F32)


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("way", [dict(attend__form=1), dict(attend__form=4, attend__whole=1), dict(attend__form=4, attend__whole=2), dict(attend__form=8, attend__whole=1),
                                 dict(attend__form=8, attend__whole=2)], ids=lambda w: " ".join(f"{k[8:]} {v}" for k, v in w.items()))
def test_every_way_of_putting_tokens_together(dev, t, way):
    """Few and many tokens in each of the forms, whichever would be taken for them."""
    dev.set_tuning(**way)
    try:
        for per, group, d in ((2, 1, 64), (5, 3, 128), (19, 4, 256), (70, 20, 96)):
            lens = [per, per + 150, per + 33]
            seq = np.repeat(np.arange(3), per)
            length = np.concatenate([np.arange(n - per, n) + 1 for n in lens])
            attend(dev, t, lens, seq, length, 2, group, d, qt=quant.BF16, ot=quant.F16)
            attend(dev, t, lens, seq, length, 2, group, d, window=70, sinks=True)
    finally:
        dev.set_tuning(attend__form=0, attend__whole=0)


@pytest.mark.parametrize("form", [1, 4, 8])
def test_thousands_of_tokens(dev, form):
    """More units than a workgroup has threads to count them, sequences in turn, and a few tokens that see nothing."""
    rng = np.random.default_rng(50)
    lens = [400, 37, 900]
    seq = np.repeat([0, 2, 1, 2, 0], [1300, 1500, 37, 1100, 1200])
    length = np.array([rng.integers(0, lens[s] + 1) for s in seq])
    dev.set_tuning(attend__form=form, attend__whole=2)
    try:
        attend(dev, quant.F16, lens, seq, length, 1, 1, 16, ot=quant.F16)
    finally:
        dev.set_tuning(attend__form=0, attend__whole=0)
    many = rng.integers(0, 38, 3000)
    attend(dev, quant.I8, [37], np.zeros(3000, int), many, 1, 1, 16)
    attend(dev, quant.BF16, lens * 700, None, np.array(lens * 700) // 20, 1, 2, 16, window=9)


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("whole", [1, 2])
@pytest.mark.parametrize("d, group", [(64, 8), (128, 4), (256, 2), (80, 20)])
def test_few_tokens_in_both_divisions(dev, t, whole, d, group):
    """A unit a workgroup, and shares that are joined, for single tokens and for a few of a sequence, whichever would be taken for them."""
    dev.set_tuning(attend__form=1, attend__whole=whole)
    try:
        for ot in PLAIN:
            lens = [1, 37, 0, 300, 1500]
            attend(dev, t, [max(n, 1) for n in lens], None, lens, 2, group, d, quant.BF16, ot, sinks=ot == quant.F16, window=200 if ot == quant.BF16 else 0)
        lens = [3, 200, 700]
        attend(dev, t, lens, np.repeat(np.arange(3), 3), np.concatenate([np.arange(n - 3, n) + 1 for n in lens]), 2, group, d)
    finally:
        dev.set_tuning(attend__form=0, attend__whole=0)
