"""Attention over a paged cache (jl_attend_dev) at the ends of what a cache and a call may hold, against the definition and the bars of test_gpu_attend."""
import numpy as np
import pytest

from jitllm_amd import quant
from jitllm_amd.device import Device
from jitllm_amd.hipmem import DeviceArray, mem_info
from test_gpu_attend import check, reference, run
from test_gpu_kv_cache import KINDS, Cache, table_of

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


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("scale, cap", [(-0.125, 0.0), (-0.125, 20.0), (0.0, 0.0), (-0.0, 5.0), (-1e-30, 0.0)])
def test_scales_of_the_scores(dev, way, t, scale, cap):
    """Below zero: the smallest product has the most weight.  Zero: every position the same."""
    rng = np.random.default_rng(80)
    for per, group, d in ((1, 4, 64), (3, 2, 128), (40, 2, 64)):
        lens = [per, per + 20, per + 300]
        table, n_page = table_of(rng, lens, 16)
        c = Cache(t, 2, d, 16, table, n_page)
        seq, length = causal(lens, per)
        q = rng.standard_normal((len(seq), 2 * group, d)).astype(np.float32)
        got, lse = run(dev, c, q, quant.F32, quant.F32, seq, length, scale, cap=cap)
        check(got, lse, reference(c, q, seq, length, scale, cap=cap), quant.F32)


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("pages", [3, 4000])
def test_tables_longer_than_their_sequences(dev, t, pages):
    """A table sized for far more positions than its sequences have, its rows apart: what lies behind a sequence's pages is no page, and what lies between the rows is not read."""
    rng = np.random.default_rng(81)
    for per, group, d in ((1, 4, 128), (3, 2, 64), (40, 2, 128), (300, 1, 64)):
        lens = [per, per + 20, per + 300]
        table, n_page = table_of(rng, lens, 16)
        c = Cache(t, 2, d, 16, np.concatenate([table, np.full((3, pages), n_page, np.uint32)], 1), n_page)
        wide = np.concatenate([c.table, np.zeros((3, 5), np.uint32)], 1)      # (page 0: read, it would be seen)
        c.td = DeviceArray(wide)
        make = c.handle
        c.handle = lambda dev: make(dev, table_stride=wide.shape[1])
        seq, length = causal(lens, per)
        q = rng.standard_normal((len(seq), 2 * group, d)).astype(np.float32)
        got, lse = run(dev, c, q, quant.F32, quant.F32, seq, length, 0.125)
        check(got, lse, reference(c, q, seq, length, 0.125), quant.F32)
        length[per - 1::per] = 0xFFFFFFFF          # behind the table: all that it holds
        got, lse = run(dev, c, q, quant.F32, quant.F32, seq, length, 0.125)
        check(got, lse, reference(c, q, seq, length, 0.125), quant.F32)


@pytest.mark.parametrize("t", KINDS)
def test_a_prompt_and_single_tokens_in_one_call(dev, way, t):
    """One sequence's prompt between the next tokens of twenty others."""
    rng = np.random.default_rng(82)
    lens = [int(v) for v in rng.integers(1, 400, 21)]
    lens[7] = 500
    seq = np.concatenate([np.arange(7), np.full(120, 7), np.arange(8, 21)])
    length = np.concatenate([lens[:7], np.arange(380, 500) + 1, lens[8:]])
    table, n_page = table_of(rng, lens, 32)
    c = Cache(t, 2, 64, 32, table, n_page)
    q = rng.standard_normal((len(seq), 8, 64)).astype(np.float32)
    got, lse = run(dev, c, q, quant.F32, quant.F32, seq, length, 0.125)
    check(got, lse, reference(c, q, seq, length, 0.125), quant.F32)
