"""A block's step through the calls around its projections and the projections themselves, one after the other on a stream of the
caller's.  Every step against the plain statement of it over the values that the step before left: the norm and the adapters in 64 bits,
the projections and the mixture against the oracle (a projection by NMSE 1e-10, like for like; the mixture, whose down projection
quantizes what gate and up gave, by rel-L2 1e-3)."""
import numpy as np
import pytest

import oracle
from conftest import nmse, rel_l2
from jitllm_amd import quant, synth
from jitllm_amd.hipmem import DeviceArray, Stream
from test_gpu_moe import _oracle_block
from test_gpu_moe_select import reference as select_reference
from test_gpu_norm_rows import check_y, reference as norm_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 5, 40])
def test_every_step_of_a_block(dev, rows):
    dev.SetActWindow(256)
    st, t, window = Stream(), quant.Q4_K, 256
    rng = np.random.default_rng(rows)
    e, kv, ne, ku, f, rank, na = 512, 256, 16, 4, 256, 16, 3
    num = lambda *s: rng.standard_normal(s).astype(np.float32)
    w0 = [synth.quantized_weights(t, r, e, seed=r) for r in (e, kv)]
    bank0 = [np.concatenate([synth.quantized_weights(t, r, c, seed=100 * i + x) for x in range(ne)]) for i, (r, c) in enumerate(((f, e), (f, e), (e, f)))]
    wq, wk = (DeviceArray(v) for v in w0)
    banks = [DeviceArray(v) for v in bank0]
    x, resid, w, fan = num(rows, e), num(rows, e), 1 + num(e) / 10, np.float32(1 / np.sqrt(e))
    a, b = [(num(na, rank, e) * fan).astype(np.float16) for _ in range(2)], [num(na, n, rank).astype(np.float16) for n in (e, kv)]
    ids, router, bias = rng.integers(0, na + 1, rows).astype(np.uint32), num(ne, e) * fan, 0.1 * num(ne)
    bias[3] = -np.inf
    xd, rd, wd, yd = DeviceArray(x), DeviceArray(resid), DeviceArray(w), DeviceArray(np.zeros((rows, e), np.float32))
    q, k = (DeviceArray(np.zeros((rows, n), np.float32)) for n in (e, kv))
    ad, bd, idd = [DeviceArray(v) for v in a], [DeviceArray(v) for v in b], DeviceArray(ids)
    routerd, biasd, logits = DeviceArray(router), DeviceArray(bias), DeviceArray(np.zeros((rows, ne), np.float32))
    sel, wt = DeviceArray(np.zeros((rows, ku), np.uint32)), DeviceArray(np.zeros((rows, ku), np.float32))
    s = st.handle
    try:
        assert dev.norm_rows_dev(xd.ptr, rows, e, wd.ptr, 1e-5, resid=rd.ptr, resid_out=rd.ptr, y=yd.ptr, stream=s)
        assert dev.matmul_dev(q.ptr, t, wq.ptr, yd.ptr, e, e, rows, stream=s) and dev.matmul_dev(k.ptr, t, wk.ptr, yd.ptr, kv, e, rows, stream=s)
        st.synchronize()
        h, y = norm_reference(x, resid, 1.0, w, 1e-5)
        assert np.array_equal(rd.get(), h)
        check_y(yd.get(), y, quant.F32)
        y0, base = yd.get(), [q.get(), k.get()]
        for got, weights, n in zip(base, w0, (e, kv)):
            assert nmse(got, oracle.matmul_q8act_f64(t, weights, y0, n, e, rows, window).reshape(rows, n)) <= 1e-10
        assert dev.adapter_group_dev([q.ptr, k.ptr], [q.ptr, k.ptr], [e, kv], [v.ptr for v in ad], [v.ptr for v in bd], quant.F16, na, rank, yd.ptr, e, idd.ptr, rows,
                                     stream=s)
        assert dev.moe_logits_dev(logits.ptr, 0, routerd.ptr, yd.ptr, ne, e, rows, stream=s)
        assert dev.moe_select_dev(logits.ptr, rows, ne, ku, sel.ptr, ku, wt.ptr, score=1, bias=biasd.ptr, n_group=4, k_group=2, group_top=2, scale=2.0, stream=s)
        assert dev.moe_ffn_dev(rd.ptr, t, *[v.ptr for v in banks], yd.ptr, sel.ptr, ku, wt.ptr, rows, ku, ne, f, e, stream=s)
        st.synchronize()
        y64 = y0.astype(np.float64)
        for o, bs, ai, bi in ((q, base[0], a[0], b[0]), (k, base[1], a[1], b[1])):
            want, most = bs.astype(np.float64), np.zeros_like(bs, np.float64)
            for r in np.nonzero(ids < na)[0]:
                ar, br = ai[ids[r]].astype(np.float64), bi[ids[r]].astype(np.float64)
                want[r] += br @ (ar @ y64[r])
                most[r] = np.abs(br) @ (np.abs(ar) @ np.abs(y64[r]))
            assert np.all(np.abs(o.get() - want) <= 2.0 ** -24 * ((e + rank + 4) * most + np.abs(want)))
        l = logits.get()
        want = router.astype(np.float64) @ y64.T
        assert np.all(np.abs(l - want.T) <= 2.0 ** -24 * e * (np.abs(router.astype(np.float64)) @ np.abs(y64.T)).T)
        ws, ww = select_reference(l, ku, 1, bias, 4, 2, 2, True, 2.0)
        assert np.array_equal(sel.get(), ws) and np.all(np.abs(wt.get() - ww) <= np.abs(ww) * 20 * 2.0 ** -24)
        mix = _oracle_block(t, *bank0, y0, sel.get(), wt.get(), ne, f, e, window)
        assert rel_l2(rd.get().astype(np.float64) - h, mix) <= 1e-3
    finally:
        st.destroy()
        dev.SetActWindow(32)
