"""Attention over a paged cache (jl_attend_dev) at the ends of what a cache and a call may hold, against the definition and the bars of test_gpu_attend."""
import numpy as np
import pytest

from jitllm_amd import quant
from jitllm_amd.device import Device
from jitllm_amd.hipmem import DeviceArray, mem_info
from test_gpu_attend import check, reference, run
from test_gpu_kv_cache import Cache, table_of

pytestmark = pytest.mark.gpu

WAYS = [dict(attend__form=f, attend__whole=w) for f in (1, 4, 8) for w in (1, 2)]


@pytest.fixture(params=WAYS, ids=lambda w: " ".join(f"{k[8:]} {v}" for k, v in w.items()))
def way(dev, request):
    """Each form, in units and in shares."""
    dev.set_tuning(**request.param)
    yield request.param
    dev.set_tuning(attend__form=0, attend__whole=0)


def causal(lens, per):
    """The last `per` tokens of each sequence: their sequences, and the positions that they see."""
    return np.repeat(np.arange(len(lens)), per), np.concatenate([np.arange(n - per, n) + 1 for n in lens])


@pytest.mark.parametrize("signs", ["negative", "mixed", "largest negative"])
@pytest.mark.parametrize("per, group, d", [(1, 4, 64), (3, 2, 128), (40, 2, 64), (24, 4, 256)])
def test_scales_of_either_sign(dev, way, signs, per, group, d):
    """A row of 8-bit values is its scale times them, whatever the scale's sign."""
    rng = np.random.default_rng(60 + per)
    lens = [per, per + 20, per + 300]
    table, n_page = table_of(rng, lens, 16)
    c = Cache(quant.I8, 2, d, 16, table, n_page)
    sign = lambda s: -np.ones(s.shape) if signs == "negative" else rng.choice([-1.0, 1.0], s.shape) if signs == "mixed" else np.where(s > 0.015, -40.0, 1.0)
    c.ks, c.vs = (c.ks * np.sign(sign(c.ks))).astype(np.float32), (c.vs * sign(c.vs)).astype(np.float32)
    c.upload()
    seq, length = causal(lens, per)
    q = rng.standard_normal((len(seq), 2 * group, d)).astype(np.float32)
    got, lse = run(dev, c, q, quant.F32, quant.F32, seq, length, 0.125)
    check(got, lse, reference(c, q, seq, length, 0.125), quant.F32)


@pytest.mark.parametrize("per, group, d", [(3, 2, 128), (16, 1, 64), (40, 2, 64), (24, 4, 256)])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 40, np.inf])
def test_a_scale_that_only_a_later_token_sees(dev, way, size, per, group, d):
    """The 8-bit row of a unit's last token may be larger than all others by any factor: the tokens before it, which do not see it, keep their bits."""
    rng = np.random.default_rng(70 + per)
    lens = [per, per + 20, per + 300]
    table, n_page = table_of(rng, lens, 16)
    c = Cache(quant.I8, 2, d, 16, table, n_page)
    c.vs = (c.vs * np.float32(2.0 ** -30)).astype(np.float32)
    for s, n in enumerate(lens):
        page, at = c.place(s, n - 1)
        c.vs[page, :, at] *= np.float32(size)
    c.upload()
    seq, length = causal(lens, per)
    q = rng.standard_normal((len(seq), 2 * group, d)).astype(np.float32)
    got, lse = run(dev, c, q, quant.F32, quant.F32, seq, length, 0.125)
    last = length == np.array(lens)[seq]
    with np.errstate(invalid="ignore"):
        ref = reference(c, q, seq, length, 0.125)
    check(got[~last], lse[~last], [a[~last] for a in ref], quant.F32)
    if np.isinf(size):
        assert np.all(np.isnan(got[last]) | np.isinf(got[last]))
    else:
        check(got[last], lse[last], [a[last] for a in ref], quant.F32)


def test_a_workspace_of_one_size_for_a_row_width():
    """The first call that divides positions among the workgroups sizes the workspace for every other over rows of that width."""
    with Device(device=0) as d:
        table, n_page = table_of(np.random.default_rng(1), [3000] * 4, 64)
        c = Cache(quant.F16, 4, 128, 64, table, n_page)
        q, out = DeviceArray(np.ones((2000, 16, 128), np.float32)), DeviceArray(np.zeros((2000, 16, 128), np.float32))
        seq, ld = DeviceArray(np.repeat(np.arange(4, dtype=np.uint32), 500)), DeviceArray(np.full(2000, 3000, np.uint32))
        h = c.handle(d)
        call = lambda ntok: d.attend_dev(h, out.ptr, q.ptr, 16, ld.ptr, ntok, 0.1, seq=seq.ptr)
        d.set_tuning(attend__form=1, attend__whole=2)
        assert call(1)
        d.synchronize()
        before = mem_info()[0]
        for form in (1, 4, 8):
            d.set_tuning(attend__form=form)
            for ntok in (4, 100, 2000):
                assert call(ntok)
        d.synchronize()
        assert mem_info()[0] == before
