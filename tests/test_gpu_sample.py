"""A token a row of logits (jl_sample_dev) against the definition, in 64 bits and with whole numbers for the ties.

Bars: the token is the definition's, always; prob is off by no more than its sums of weights kept to 2^-44 (n 2^-45 of them) and its rounding to f32."""
import numpy as np
import pytest

from jitllm_amd import quant
from jitllm_amd.device import Device
from jitllm_amd.hipmem import DeviceArray, Graph, Stream, mem_info
from test_gpu_kv_cache import PLAIN
from test_gpu_norm_rows import STEP, at_offset, stored, values

pytestmark = pytest.mark.gpu


def reference(x, u, temp=1.0, k=0, p=1.0, low=0.0):
    """(token, prob) of one row."""
    x = x.astype(np.float64)
    n = x.size
    live = np.flatnonzero(x > -np.inf)
    if not live.size:
        return n, 0.0
    if not temp > 0:
        return int(live[np.argmax(x[live])]), 1.0
    order = live[np.lexsort((live, -x[live]))]
    m = x[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x[order] == m, 1.0, np.exp((x[order] - m) / np.float64(np.float32(temp))))
    if k:
        order, w = order[:k], w[:k]
    if p < 1:
        c = np.cumsum(w)
        end = int(np.argmax(c >= np.float64(np.float32(p)) * c[-1])) + 1
        order, w = order[:end], w[:end]
    if low > 0:
        end = max(1, int((w >= np.float64(np.float32(low))).sum()))
        order, w = order[:end], w[:end]
    by = np.argsort(order)
    order, w = order[by], w[by]
    c = np.cumsum(w)
    over = np.flatnonzero(c > np.float64(u) * c[-1])
    at = over[0] if over.size else np.flatnonzero(w > 0)[-1]
    return int(order[at]), w[at] / c[-1]


def run(dev, x, t, u, stream=None, address=None, stride=0, prob=True, **settings):
    rows, n = x.shape
    keep = [DeviceArray(stored(x, t)), DeviceArray(np.ascontiguousarray(u, np.float32))]
    token, pr = DeviceArray(np.full(rows + 1, 12345, np.uint32)), DeviceArray(np.full(rows + 1, 7, np.float32))
    kw = {}
    for name, a in settings.items():
        if a is not None:
            keep.append(DeviceArray(np.broadcast_to(np.asarray(a, np.uint32 if name == "top_k" else np.float32), (rows,)).copy()))
            kw[name] = keep[-1].ptr
    assert dev.sample_dev(address or keep[0].ptr, rows, n, keep[1].ptr, token.ptr, type=t, stride=stride, prob=pr.ptr if prob else None, stream=stream, **kw)
    dev.synchronize()
    assert token.get()[rows] == 12345 and pr.get()[rows] == 7
    return token.get()[:rows], pr.get()[:rows]


def check(dev, x, t, u, temperature=None, top_k=None, top_p=None, min_p=None, **kw):
    x = values(stored(x, t), t).astype(np.float32)
    rows = x.shape[0]
    token, prob = run(dev, x, t, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, **kw)
    of = lambda a, off: np.broadcast_to(np.asarray(off if a is None else a), (rows,))
    for r in range(rows):
        want = reference(x[r], np.float32(u[r]), of(temperature, 1.0)[r], int(of(top_k, 0)[r]), float(np.float32(of(top_p, 1.0)[r])),
                         float(np.float32(of(min_p, 0.0)[r])))
        assert token[r] == want[0], (r, token[r], want)
        assert abs(prob[r] - want[1]) <= want[1] * (2.0 ** -24 + x.shape[1] * 2.0 ** -44) + 2.0 ** -43
    return token


def logits(rng, rows, n, spread=2.0):
    x = (spread * rng.standard_normal((rows, n))).astype(np.float32)
    for r in range(rows):
        x[r, rng.integers(0, n, 8)] += 8 * rng.random(8).astype(np.float32)
    return x


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=0.8, top_k=40, top_p=0.95),
            dict(temperature=1.3, top_k=300, top_p=0.99, min_p=0.001), dict(temperature=0.0), dict(top_p=0.0), dict(top_p=0.5, min_p=0.3)]


@pytest.mark.parametrize("n", [1, 2, 3, 64, 1000, 4095, 4096, 4097, 32000, 131072])
@pytest.mark.parametrize("settings", SETTINGS, ids=lambda s: ",".join(f"{k}={v}" for k, v in s.items()) or "plain")
def test_settings(dev, n, settings):
    rng = np.random.default_rng(n)
    rows = 6 if n < 5000 else 3
    check(dev, logits(rng, rows, n), quant.F32, rng.random(rows).astype(np.float32), **settings)


@pytest.mark.parametrize("t", PLAIN)
@pytest.mark.parametrize("rows, n", [(1, 200003), (5, 50257), (300, 1031), (64, 8192), (2, 524288)])
def test_every_row_its_own_settings(dev, t, rows, n):
    rng = np.random.default_rng(rows + n)
    check(dev, logits(rng, rows, n), t, rng.random(rows).astype(np.float32), temperature=rng.choice([0.0, 0.3, 1.0, 2.0], rows), top_k=rng.choice([0, 1, 7, 60, 5000, n + 3], rows),
          top_p=rng.choice([0.1, 0.8, 0.999, 1.0, 1.5], rows), min_p=rng.choice([0.0, 0.01, 0.5, 1.0, 2.0], rows))


@pytest.mark.parametrize("settings", [dict(), dict(top_k=3000), dict(top_p=0.4), dict(top_k=5000, top_p=0.7, min_p=0.1)], ids=str)
def test_rows_of_equals(dev, settings):
    """All values one, two values, a few: ties by the thousand, cut by index; and a flat row, whose nucleus is most of it."""
    rng = np.random.default_rng(3)
    n = 9001
    x = np.zeros((6, n), np.float32)
    x[0] = -3.25
    x[1] = rng.choice([1.0, 1.5], n)
    x[2] = rng.choice([-0.0, 0.0], n)
    x[3] = rng.integers(-3, 3, n)
    x[4] = 1e-3 * rng.standard_normal(n)
    x[5] = (1 + 1e-6 * rng.integers(0, 40, n)).astype(np.float32)
    for u in (0.0, 0.37, 0.5, 0.99999994):
        check(dev, x, quant.F32, np.full(6, u, np.float32), **settings)


def test_rows_with_infinities_and_nans(dev):
    rng = np.random.default_rng(4)
    x = logits(rng, 9, 3001)
    x[0, ::2] = -np.inf
    x[1] = -np.inf
    x[2] = np.nan
    x[3, 5] = np.nan
    x[4, [7, 100, 2000]] = np.inf
    x[5] = np.where(rng.random(3001) < 0.9, -np.inf, x[5])
    x[6] = -np.inf
    x[6, 77] = -1e30
    x[7] = 3e38
    x[7, 9] = -3e38
    x[8] = np.where(np.arange(3001) % 3 == 0, np.nan, -np.inf)
    for s in (dict(), dict(top_k=50), dict(top_p=0.8), dict(temperature=0.0), dict(top_k=2, top_p=0.5, min_p=0.2)):
        token = check(dev, x, quant.F32, rng.random(9).astype(np.float32), **s)
        assert token[1] == token[2] == token[8] == 3001 and token[6] == 77 and token[4] in (7, 100, 2000)


def test_numbers_at_the_ends(dev):
    """u at 0, just below 1, at and over 1, negative, NaN; temperatures from the smallest to infinity; settings that are no numbers."""
    rng = np.random.default_rng(5)
    x = logits(rng, 6, 777)
    check(dev, x, quant.F32, np.array([0.0, np.nextafter(np.float32(1), np.float32(0)), 1.0, 7.0, -1.0, np.nan], np.float32))
    check(dev, x, quant.F32, rng.random(6).astype(np.float32), temperature=np.array([1e-45, 1e-20, 1e10, np.inf, -1.0, np.nan], np.float32))
    a = run(dev, x, quant.F32, np.full(6, 0.5, np.float32), top_p=np.nan, min_p=np.nan)[0]
    assert np.array_equal(a, check(dev, x, quant.F32, np.full(6, 0.5, np.float32)))


def test_every_token_has_its_share(dev):
    """The token as u goes through a grid: the steps of the distribution's sums."""
    x = np.array([[0.0, 1.0, -1.0, 2.0, -np.inf, 1.0]], np.float32)
    w = np.exp(x[0] - 2)
    c = np.cumsum(w / w.sum())
    us = np.linspace(0, 1, 400, endpoint=False).astype(np.float32)
    token, prob = run(dev, np.repeat(x, 400, 0), quant.F32, us)
    assert np.array_equal(token, [int(np.argmax(c > float(v))) for v in us])
    assert np.allclose(prob, (w / w.sum())[token], rtol=1e-6)


@pytest.mark.parametrize("t, off", [(quant.F32, 1), (quant.F16, 1), (quant.BF16, 3), (quant.F32, 0)])
def test_strides_and_alignment(dev, t, off):
    rng = np.random.default_rng(6)
    x = values(stored(logits(rng, 4, 1234), t), t).astype(np.float32)
    wide = np.full((4, 1301), 50.0, np.float32)       # what lies behind a row would win
    wide[:, :1234] = x
    buf, at = at_offset(stored(wide, t), off)
    u = rng.random(4).astype(np.float32)
    token, _ = run(dev, x, t, u, address=at, stride=1301, top_k=30)
    assert list(token) == [reference(x[r], u[r], k=30)[0] for r in range(4)]
    token, prob = run(dev, x, t, u, address=at, stride=1301, prob=False)
    assert list(token) == [reference(x[r], u[r])[0] for r in range(4)] and np.all(prob == 7)


def test_the_same_in_every_call(dev):
    """A row's token does not depend on the rows beside it, nor on the stream; captured, and replayed over new numbers."""
    rng = np.random.default_rng(7)
    n, rows, st = 50000, 300, Stream()
    x, u = logits(rng, rows, n, 0.5), rng.random(rows).astype(np.float32)
    many = run(dev, x, quant.F32, u, top_p=0.9)
    for r in (0, 150, 299):
        one = run(dev, x[r:r + 1], quant.F32, u[r:r + 1], top_p=0.9)
        assert one[0][0] == many[0][r] and one[1][0] == many[1][r]
    xd, ud, p, token = DeviceArray(x[:4]), DeviceArray(u[:4]), DeviceArray(np.full(4, 0.9, np.float32)), DeviceArray(np.zeros(4, np.uint32))
    try:
        with Graph.capture(st.handle) as g:
            assert dev.sample_dev(xd.ptr, 4, n, ud.ptr, token.ptr, top_p=p.ptr, stream=st.handle)
        for i in range(5):
            u = rng.random(4).astype(np.float32)
            x[:4] = x[rng.permutation(4)]
            ud.put(u)
            xd.put(x[:4])
            g.launch()
            st.synchronize()
            assert list(token.get()) == [reference(x[r], u[r], p=float(np.float32(0.9)))[0] for r in range(4)]
            run(dev, x[:7], quant.F32, rng.random(7).astype(np.float32), top_k=9)
    finally:
        st.destroy()


@pytest.mark.parametrize("n", [200, 5000, 70001])
@pytest.mark.parametrize("k", [63, 64, 65, 128, 700, 1023, 1024, 1025, 4000])
def test_as_many_as_asked_for(dev, n, k):
    """The k largest, alone and with a share of their sum, around the sizes at which they are held in another way."""
    rng = np.random.default_rng(k)
    x = logits(rng, 3, n, 1.0)
    x[2] = np.round(x[2], 1)          # ties by the hundred
    u = rng.random(3).astype(np.float32)
    check(dev, x, quant.F32, u, top_k=k)
    check(dev, x, quant.F32, u, top_k=k, top_p=0.97, min_p=0.001)
    check(dev, x, quant.BF16, u, top_k=k, top_p=0.6, temperature=2.0)


def test_more_rows_than_a_pass_has(dev):
    rng = np.random.default_rng(31)
    x = logits(rng, 2100, 300)
    check(dev, x, quant.F16, rng.random(2100).astype(np.float32), top_k=rng.choice([0, 5, 90], 2100), top_p=rng.choice([0.5, 0.9, 1.0], 2100))


def test_a_reserved_workspace():
    with Device(device=0) as d:
        d.reserve_sample(5000)          # (a pass's rows, whatever is asked for)
        rng = np.random.default_rng(32)
        for rows, n in ((1, 100), (1500, 2000), (7, 131072)):
            xd, ud = DeviceArray(logits(rng, rows, n)), DeviceArray(rng.random(rows).astype(np.float32))
            p, token = DeviceArray(np.full(rows, 0.9, np.float32)), DeviceArray(np.zeros(rows, np.uint32))
            before = mem_info()[0]
            assert d.sample_dev(xd.ptr, rows, n, ud.ptr, token.ptr, top_p=p.ptr) and d.sample_dev(xd.ptr, rows, n, ud.ptr, token.ptr)
            d.synchronize()
            assert mem_info()[0] == before and np.all(token.get() < n)
