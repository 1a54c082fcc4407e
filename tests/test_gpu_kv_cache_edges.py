"""Orders of a paged cache's pages by the strides that a call works out by itself (jl_kv_write_dev, jl_kv_read_dev, jl_attend_dev)."""
import numpy as np
import pytest

from jitllm_amd import quant
from jitllm_amd.hipmem import DeviceArray
from test_gpu_attend import check, reference, run
from test_gpu_kv_cache import KINDS, Cache, table_of

pytestmark = pytest.mark.gpu


class Shared(Cache):
    """Its handle names the rows' and the heads' strides alone, or a table row longer than its pages."""

    def handle(self, dev, **kw):
        strides = dict(row_stride=self.n_kv * self.row, head_stride=self.row) if self.order == "places" else dict(row_stride=self.row) if self.row > self.d else {}
        return dev.kv_cache(self.t, self.n_kv, self.d, self.page, self.n_page, self.kd.ptr, self.vd.ptr, self.td.ptr, *self.table.shape,
                            k_scale=self.ksd.ptr if self.ksd else None, v_scale=self.vsd.ptr if self.vsd else None, **strides, **kw)


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("order, gap", [("heads", 0), ("heads", 16), ("places", 0), ("places", 16)])
def test_page_strides_left_out(dev, t, order, gap):
    """Every row of three sequences written, read back and attended to."""
    rng = np.random.default_rng(3 + gap)
    lens, n_kv, d = [40, 17, 64], 3, 64
    table, n_page = table_of(rng, lens, 16)
    c = Shared(t, n_kv, d, 16, table, n_page, order, gap=gap)
    seq, pos = np.repeat(np.arange(3), lens).astype(np.uint32), np.concatenate([np.arange(n) for n in lens]).astype(np.uint32)
    n = len(seq)
    k, v = (rng.standard_normal((n, n_kv, d)).astype(np.float32) for _ in range(2))
    kd, vd, sd, pd, y = DeviceArray(k), DeviceArray(v), DeviceArray(seq), DeviceArray(pos), DeviceArray(np.zeros_like(k))
    h = c.handle(dev)
    assert dev.kv_write_dev(h, kd.ptr, vd.ptr, quant.F32, pd.ptr, n, seq=sd.ptr) and dev.kv_read_dev(h, None, y.ptr, quant.F32, pd.ptr, n, seq=sd.ptr)
    c.write(k, v, seq, pos)
    dev.synchronize()
    c.check()
    assert np.array_equal(y.get(), c.read("v", seq, pos))
    q = rng.standard_normal((3, 2 * n_kv, d)).astype(np.float32)
    got, lse = run(dev, c, q, quant.F32, quant.F32, None, lens, 0.125)
    check(got, lse, reference(c, q, range(3), lens, 0.125), quant.F32)
