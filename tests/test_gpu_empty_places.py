"""A selection with empty places (jl_moe_select_dev) through the mixture's calls one after the other: grouping, matvecs, combine."""
import numpy as np
import pytest

from conftest import rel_l2
from jitllm_amd import quant, synth
from test_gpu_moe import _oracle_block

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows, left", [(5, 2), (70, 2), (70, 0), (33, 1), (200, 3)])
def test_empty_places_through_the_single_calls(dev, devbuf, rows, left):
    """`left` of six experts in service, four wanted: the places left over have no column, and the combine adds nothing for them.  Their
    pos was filled with no column before the grouping; y holds NaN wherever no column is."""
    n, k, f, e, t, window = 6, 4, 256, 256, quant.Q4_K, 256
    dev.SetActWindow(window)
    try:
        rng = np.random.default_rng(rows + left)
        bank0 = [np.concatenate([synth.quantized_weights(t, r, c, seed=10 * i + x) for x in range(n)]) for i, (r, c) in enumerate(((f, e), (f, e), (e, f)))]
        gate, up, down = (devbuf(b) for b in bank0)
        x, resid = rng.standard_normal((rows, e)).astype(np.float32), rng.standard_normal((rows, e)).astype(np.float32)
        bias = np.full(n, -np.inf, np.float32)
        bias[rng.permutation(n)[:left]] = 0.0
        logits, biasd, xd = devbuf(rng.standard_normal((rows, n)).astype(np.float32)), devbuf(bias), devbuf(x)
        sel, wt = devbuf(np.zeros((rows, k), np.uint32)), devbuf(np.zeros((rows, k), np.float32))
        assert dev.moe_select_dev(logits.ptr, rows, n, k, sel.ptr, k, wt.ptr, score=1, bias=biasd.ptr)
        start, perm, pos = devbuf(shape=(n + 1,), dtype=np.uint32, fill=0), devbuf(np.zeros(rows * k, np.uint32)), devbuf(np.full(rows * k, 0xFFFFFFFF, np.uint32))
        nan = np.float32(np.nan)
        g, u, y = (devbuf(shape=(rows * k, w), dtype=np.float32, fill=nan) for w in (f, f, e))
        out = devbuf(resid)
        assert dev.moe_group_dev(sel.ptr, k, rows, k, n, start.ptr, perm.ptr, pos.ptr)
        dev.synchronize()
        live = int(start.get()[n])
        assert live == rows * left and np.count_nonzero(pos.get() != 0xFFFFFFFF) == live
        assert dev.moe_matvec_dev(g.ptr, u.ptr, t, gate.ptr, up.ptr, xd.ptr, None, perm.ptr, start.ptr, n, rows * k, f, e)
        assert dev.moe_matvec_dev(y.ptr, None, t, down.ptr, None, g.ptr, u.ptr, None, start.ptr, n, rows * k, e, f)
        dev.synchronize()
        yh = y.get()
        yh[live:] = nan
        y.put(yh)
        assert dev.moe_combine_dev(out.ptr, y.ptr, wt.ptr, sel.ptr, k, pos.ptr, rows, k, e)
        dev.synchronize()
        got = out.get().astype(np.float64) - resid
        want = _oracle_block(t, *bank0, x, sel.get(), wt.get(), n, f, e, window)
        assert np.all(np.sort(sel.get(), 1)[:, left:] == n)
        if left:
            assert rel_l2(got, want) <= 1e-3
        else:
            assert np.all(got == 0)
    finally:
        dev.SetActWindow(32)
