"""Rows normed between two projections (jl_norm_rows_dev) against the definition in 64 bits.

Bars.  h: the bits of f32(resid + f32(alpha * x)).  y: the f64 value narrowed once, so half a step of its type -- f32 2^-24,
f16 2^-11 (below 2^-14 an absolute 2^-25), bf16 2^-8 of the value, plus the narrowing to f32 on the way and the f64 sum's own
error, together under 2^-23.  q, as, sum16: the bits jl_quantize_act_dev makes of the f32 y."""
import numpy as np
import pytest

import oracle
from jitllm_amd import quant
from jitllm_amd.device import Device
from jitllm_amd.hipmem import DeviceArray, Graph, Stream

pytestmark = pytest.mark.gpu

POISON = np.float32(-7e30)
STEP = {quant.F32: 2.0 ** -24, quant.F16: 2.0 ** -11, quant.BF16: 2.0 ** -8}


def bf16_bits(a):
    b = np.ascontiguousarray(a, np.float32).view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def stored(a, t):
    """f32 values as an array of type t."""
    return a.astype(np.float32) if t == quant.F32 else a.astype(np.float16) if t == quant.F16 else bf16_bits(a)


def values(a, t):
    return a.astype(np.float64) if t != quant.BF16 else (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def dtype(t):
    return {quant.F32: np.float32, quant.F16: np.float16, quant.BF16: np.uint16}[t]


def poison(shape, t):
    return DeviceArray(stored(np.full(shape, -60000.0, np.float32), t))


def at_offset(a, elems):
    """a in device memory, `elems` elements behind a 16-byte boundary: (buffer, address)."""
    buf = DeviceArray(np.concatenate([np.zeros(elems, a.dtype), a.ravel()]))
    return buf, buf.ptr + elems * a.dtype.itemsize


def reference(x, resid, alpha, w, eps):
    h = x.astype(np.float32) if resid is None else (resid + np.float32(alpha) * x.astype(np.float32)).astype(np.float32)
    d = h.astype(np.float64)
    y = d * (1.0 if w is None else w.astype(np.float64)) / np.sqrt((d * d).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
    return h, y


def check_y(got, want, t):
    y32 = want.astype(np.float32).astype(np.float64)
    got = values(got, t)
    small = 2.0 ** -25 if t == quant.F16 else 2.0 ** -130
    assert np.all(np.abs(got - y32) <= np.abs(want) * (STEP[t] + 2.0 ** -23) + small)


@pytest.mark.parametrize("rows, n", [(1, 1), (1, 4096), (2, 4), (3, 61), (5, 64), (7, 96), (9, 128), (4, 132), (3, 255), (5, 256), (3, 512), (2, 777),
                                     (5, 1024), (3, 1025), (2, 1028), (3, 2880), (1, 5000), (2, 7168), (300, 4096), (700, 1536), (2, 16384),
                                     (1, 20001), (2, 32768), (1, 65536), (1, 65533), (4099, 64), (1000, 200)])
def test_f32_rows(dev, rows, n):
    rng = np.random.default_rng(rows * 100003 + n)
    x, resid = rng.standard_normal((rows, n), np.float32), 3 * rng.standard_normal((rows, n), np.float32)
    w = (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)
    h, y = reference(x, resid, 0.75, w, 1e-5)
    xd, rd, wd, hd, yd = DeviceArray(x), DeviceArray(resid), DeviceArray(w), poison((rows + 1, n), quant.F32), poison((rows + 1, n), quant.F32)
    assert dev.norm_rows_dev(xd.ptr, rows, n, wd.ptr, 1e-5, resid=rd.ptr, alpha=0.75, resid_out=hd.ptr, y=yd.ptr)
    dev.synchronize()
    assert np.array_equal(hd.get()[:rows].view(np.uint32), h.view(np.uint32))
    check_y(yd.get()[:rows], y, quant.F32)
    assert np.all(yd.get()[rows] == -60000.0) and np.all(hd.get()[rows] == -60000.0)


@pytest.mark.parametrize("xt", [quant.F32, quant.F16, quant.BF16])
@pytest.mark.parametrize("yt", [quant.F32, quant.F16, quant.BF16])
@pytest.mark.parametrize("n, off", [(128, 0), (2048, 0), (2048, 1), (333, 0), (1500, 2)])
def test_types_and_alignments(dev, xt, yt, n, off):
    rows = 6
    rng = np.random.default_rng(n + 7 * xt + yt + off)
    x = stored(rng.standard_normal((rows, n)), xt)
    w = (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)
    resid = rng.standard_normal((rows, n)).astype(np.float32)
    _, y = reference(values(x, xt), resid, 1.0, w, 1e-6)
    keep, xp = at_offset(x, off)
    rd, wd = DeviceArray(resid), DeviceArray(w)
    ybuf, yp = at_offset(stored(np.zeros((rows, n)), yt), off)
    assert dev.norm_rows_dev(xp, rows, n, wd.ptr, 1e-6, x_type=xt, resid=rd.ptr, y=yp, y_type=yt)
    dev.synchronize()
    check_y(ybuf.get()[off:].reshape(rows, n), y, yt)


@pytest.mark.parametrize("n, xs, rs, ys", [(128, 160, 132, 256), (130, 131, 130, 135), (2048, 2052, 2048, 4096), (2048, 2049, 2050, 2051)])
def test_strides_leave_what_lies_between(dev, n, xs, rs, ys):
    rows = 5
    rng = np.random.default_rng(n + xs)
    x, resid = rng.standard_normal((rows, xs)).astype(np.float32), rng.standard_normal((rows, rs)).astype(np.float32)
    h, y = reference(x[:, :n], resid[:, :n], 1.0, None, 1e-5)
    xd, rd, hd, yd = DeviceArray(x), DeviceArray(resid), poison((rows, rs), quant.F32), poison((rows, ys), quant.F32)
    assert dev.norm_rows_dev(xd.ptr, rows, n, None, 1e-5, x_stride=xs, resid=rd.ptr, resid_stride=rs, resid_out=hd.ptr, y=yd.ptr, y_stride=ys)
    dev.synchronize()
    assert np.array_equal(hd.get()[:, :n], h) and np.all(hd.get()[:, n:] == -60000.0)
    check_y(yd.get()[:, :n], y, quant.F32)
    assert np.all(yd.get()[:, n:] == -60000.0)


@pytest.mark.parametrize("window", [32, 64, 128, 256])
@pytest.mark.parametrize("rows, n", [(1, 32), (3, 64), (2, 96), (5, 128), (2, 160), (3, 256), (3, 288), (2, 1024), (2, 1056), (3, 2880), (2, 4096), (300, 4096), (1, 14336)])
def test_int8_form_is_the_quantizers(dev, window, rows, n):
    dev.SetActWindow(window)
    rng = np.random.default_rng(n + rows)
    x = (rng.standard_normal((rows, n)) * np.exp(rng.standard_normal((rows, 1)))).astype(np.float32)
    x[0, : min(32, n)] = 0.0                                   # a window of zeros
    w = (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)
    xd, wd, yd = DeviceArray(x), DeviceArray(w), poison((rows, n), quant.F32)
    q, s, h = DeviceArray(shape=(rows, n), dtype=np.int8, fill=99), poison((rows, n // 32), quant.F32), poison((rows, n // 16), quant.F32)
    assert dev.norm_rows_dev(xd.ptr, rows, n, wd.ptr, 1e-5, y=yd.ptr, q=q.ptr, a_s=s.ptr, sum16=h.ptr)
    dev.synchronize()
    q2, s2, h2 = DeviceArray(shape=(rows, n), dtype=np.int8, fill=0), poison((rows, n // 32), quant.F32), poison((rows, n // 16), quant.F32)
    assert dev.quantize_act_dev(yd.ptr, rows, n, q2.ptr, s2.ptr, h2.ptr)
    dev.synchronize()
    assert np.array_equal(q.get(), q2.get()) and np.array_equal(s.get(), s2.get()) and np.array_equal(h.get(), h2.get())
    for r in (0, rows - 1):
        want = oracle.quantize_act(yd.get()[r], window)
        assert np.array_equal(q.get()[r], want[0]) and np.array_equal(s.get()[r], want[1]) and np.array_equal(h.get()[r], want[2])
    # the int8 form alone, from misaligned rows
    keep, xp = at_offset(x, 1)
    assert dev.norm_rows_dev(xp, rows, n, wd.ptr, 1e-5, q=q2.ptr, a_s=s2.ptr, sum16=h2.ptr)
    dev.synchronize()
    assert np.array_equal(q.get(), q2.get()) and np.array_equal(s.get(), s2.get()) and np.array_equal(h.get(), h2.get())
    dev.SetActWindow(32)


@pytest.mark.parametrize("rows, n", [(300, 288), (300, 512), (300, 2048), (2, 7168), (300, 7168), (300, 14336), (3, 32768), (2, 32800), (300, 40000), (1, 65536)])
def test_int8_form_over_the_sizes_of_a_workgroup(dev, rows, n):
    test_int8_form_is_the_quantizers(dev, 256, rows, n)


def test_in_place(dev):
    """resid_out over resid and y over x: as with buffers of their own."""
    rows, n = 37, 2880
    rng = np.random.default_rng(5)
    x, resid, w = (rng.standard_normal(s).astype(np.float32) for s in ((rows, n), (rows, n), (n,)))
    xd, rd, wd, hd, yd = DeviceArray(x), DeviceArray(resid), DeviceArray(w), poison((rows, n), quant.F32), poison((rows, n), quant.F32)
    assert dev.norm_rows_dev(xd.ptr, rows, n, wd.ptr, 1e-5, resid=rd.ptr, resid_out=hd.ptr, y=yd.ptr)
    assert dev.norm_rows_dev(xd.ptr, rows, n, wd.ptr, 1e-5, resid=rd.ptr, resid_out=rd.ptr, y=xd.ptr)
    dev.synchronize()
    assert np.array_equal(rd.get(), hd.get()) and np.array_equal(xd.get(), yd.get())


@pytest.mark.parametrize("n", [100, 4096])
def test_no_number_stays_in_its_row(dev, n):
    """A NaN or an infinity spoils its own row; zeros give zeros, eps 0 among them no number; values whose squares pass f32 do not."""
    x = np.random.default_rng(n).standard_normal((6, n)).astype(np.float32)
    x[1, 3], x[2, 5], x[3], x[4] = np.nan, np.inf, 0.0, x[4] * np.float32(1e30)
    xd, yd = DeviceArray(x), poison((6, n), quant.F32)
    assert dev.norm_rows_dev(xd.ptr, 6, n, None, 1e-5, y=yd.ptr)
    dev.synchronize()
    y = yd.get()
    assert np.all(np.isnan(y[1])) and np.isnan(y[2, 5]) and np.all(y[2, 6:] == 0) and np.all(y[3] == 0)
    for r in (0, 4, 5):
        check_y(y[r:r + 1], reference(x[r:r + 1], None, 1.0, None, 1e-5)[1], quant.F32)
    assert dev.norm_rows_dev(xd.ptr, 6, n, None, 0.0, y=yd.ptr)
    dev.synchronize()
    assert np.all(np.isnan(yd.get()[3])) and np.all(np.isfinite(yd.get()[0]))


def test_offsets_past_32_bits(dev):
    """Rows a stride of 2^30 elements apart: the sixth starts past 2^32 elements, of two bytes each (10.7 GB)."""
    n, rows, xs = 256, 6, 1 << 30
    x = bf16_bits(np.random.default_rng(9).standard_normal((rows, n)))
    big = DeviceArray(shape=(5 * xs + n,), dtype=np.uint16)
    from jitllm_amd.hipmem import check, hip
    for r in range(rows):
        check(hip().hipMemcpy(big.ptr + r * xs * 2, np.ascontiguousarray(x[r]).ctypes.data, n * 2, 1), "hipMemcpy")
    yd = poison((rows, n), quant.F32)
    assert dev.norm_rows_dev(big.ptr, rows, n, None, 1e-5, x_type=quant.BF16, x_stride=xs, y=yd.ptr)
    dev.synchronize()
    check_y(yd.get(), reference(values(x, quant.BF16), None, 1.0, None, 1e-5)[1], quant.F32)
    big.free()


def test_captured_and_replayed_on_a_stream_of_the_callers(dev):
    rows, n = 64, 4096
    rng = np.random.default_rng(11)
    st = Stream()
    xd, rd, yd = DeviceArray(shape=(rows, n), dtype=np.float32, fill=0), DeviceArray(shape=(rows, n), dtype=np.float32, fill=0), poison((rows, n), quant.F32)
    with Graph.capture(st.handle) as g:
        assert dev.norm_rows_dev(xd.ptr, rows, n, None, 1e-5, resid=rd.ptr, resid_out=rd.ptr, y=yd.ptr, stream=st.handle)
    for _ in range(3):
        x, resid = rng.standard_normal((rows, n)).astype(np.float32), rng.standard_normal((rows, n)).astype(np.float32)
        xd.put(x)
        rd.put(resid)
        g.launch()
        st.synchronize()
        h, y = reference(x, resid, 1.0, None, 1e-5)
        assert np.array_equal(rd.get(), h)
        check_y(yd.get(), y, quant.F32)
    st.destroy()


def test_one_launch(dev):
    x, y = DeviceArray(shape=(40, 4096), dtype=np.float32, fill=1), poison((40, 4096), quant.F32)
    before = dev.launch_count()
    assert dev.norm_rows_dev(x.ptr, 40, 4096, None, 1e-5, y=y.ptr)
    assert dev.launch_count() == before + 1
    dev.synchronize()
