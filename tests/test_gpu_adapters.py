"""Low-rank adapters beside shared projections (jl_adapter_group_dev) against a plain statement in 64 bits.

Bars.  Whole numbers small enough that every product and sum is exact in f32: the exact result, whatever the order.  Random
values: a sum of n f32 products in any order is off by at most n 2^-24 of the sum of their magnitudes (n = k for A x, rank for
B u, one each for the scale and the base), so with S = |scale| |B| (|A| |x|):  |out - exact| <= 2^-24 ((k + rank + 4) S + |out|)
and, since errors of random sign grow as the root of their number, the 2-norm over a result of at least a thousand values within
2^-24 (4 sqrt(k + rank) root-sum-square of the same products + |out|)."""
import numpy as np
import pytest

from jitllm_amd import quant, synth
from jitllm_amd.hipmem import DeviceArray, Graph, Stream, mem_info

pytestmark = pytest.mark.gpu

TYPES = {"f32": quant.F32, "f16": quant.F16, "bf16": quant.BF16}


def bf16_bits(a):
    b = np.ascontiguousarray(a, np.float32).view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def stored(a, t):
    return a.astype(np.float32) if t == "f32" else a.astype(np.float16) if t == "f16" else bf16_bits(a)


def values(a, t):
    return a.astype(np.float64) if t != "bf16" else (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Case:
    """Operands of a call, whole numbers or random, and what it has to give."""

    def __init__(self, seed, ntok, k, rows, rank, n_adapter, t="f16", xt="f32", ids=None, ranks=None, whole=False, base=True, scale=True):
        rng = np.random.default_rng(seed)
        num = (lambda *s: rng.integers(-2, 3, s).astype(np.float32)) if whole else (lambda *s: rng.standard_normal(s).astype(np.float32))
        self.ntok, self.k, self.rows, self.rank, self.n_adapter, self.t, self.xt = ntok, k, rows, rank, n_adapter, t, xt
        x = stored(num(ntok, k), xt)
        a, b = [stored(num(n_adapter, rank, k), t) for _ in rows], [stored(num(n_adapter, r, rank), t) for r in rows]
        self.base = [num(ntok, r) if base else None for r in rows]
        self.ids = (rng.integers(0, n_adapter + 1, ntok) if ids is None else np.asarray(ids)).astype(np.uint32)
        self.ranks = None if ranks is None else np.asarray(ranks, np.uint32)
        self.scale = None if not scale else rng.integers(1, 4, n_adapter).astype(np.float32) if whole else (0.5 + rng.random(n_adapter)).astype(np.float32)
        self.want, self.most, self.rss = [], [], []
        for i, r in enumerate(rows):
            w = np.zeros((ntok, r)) if self.base[i] is None else self.base[i].astype(np.float64)
            s, q = np.zeros((ntok, r)), np.zeros((ntok, r))
            for e in range(n_adapter):
                of, rk = np.nonzero(self.ids == e)[0], rank if ranks is None else min(int(ranks[e]), rank)
                if not len(of):
                    continue
                xe, ae, be = values(x[of], xt), values(a[i][e, :rk], t), values(b[i][e, :, :rk], t)
                g = 1.0 if self.scale is None else float(self.scale[e])
                w[of] += g * (xe @ ae.T) @ be.T
                s[of] = g * (np.abs(xe) @ np.abs(ae).T) @ np.abs(be).T
                q[of] = g * g * (xe ** 2 @ ae.T ** 2) @ be.T ** 2
            self.want.append(w), self.most.append(s), self.rss.append(q)
        self.d = dict(x=DeviceArray(x), ids=DeviceArray(self.ids), ranks=None if ranks is None else DeviceArray(self.ranks),
                      scale=None if self.scale is None else DeviceArray(self.scale), a=[DeviceArray(v) for v in a], b=[DeviceArray(v) for v in b],
                      base=[None if v is None else DeviceArray(v) for v in self.base],
                      out=[DeviceArray(np.full((ntok + 1, r), -7e30, np.float32)) for r in rows])

    def call(self, dev, in_place=False, stream=None):
        d = self.d
        p = lambda v: None if v is None else v.ptr
        if in_place:
            for o, v in zip(d["out"], self.base):
                o.put(np.concatenate([v, np.full((1, v.shape[1]), -7e30, np.float32)]))
        return dev.adapter_group_dev([o.ptr for o in d["out"]], [o.ptr for o in d["out"]] if in_place else [p(v) for v in d["base"]], self.rows,
                                     [v.ptr for v in d["a"]], [v.ptr for v in d["b"]], TYPES[self.t], self.n_adapter, self.rank, d["x"].ptr, self.k,
                                     d["ids"].ptr, self.ntok, scale=p(d["scale"]), ranks=p(d["ranks"]), x_type=TYPES[self.xt], stream=stream)

    def check(self, exact=False):
        for i, o in enumerate(self.d["out"]):
            got = o.get()
            assert np.all(got[-1] == np.float32(-7e30)), "wrote past the last token"
            got, w, u = got[:-1], self.want[i], 2.0 ** -24
            if exact:
                assert np.array_equal(got, w.astype(np.float32)) and np.all(np.abs(w) < 2 ** 24)
                continue
            assert np.all(np.abs(got - w) <= u * ((self.k + self.rank + 4) * self.most[i] + np.abs(w)) + 1e-30)
            if w.size >= 1000:
                assert np.linalg.norm(got - w) <= u * (4 * np.sqrt((self.k + self.rank) * self.rss[i].sum()) + np.linalg.norm(w))
            none = self.ids >= self.n_adapter
            if self.base[i] is not None:
                assert np.array_equal(got[none], self.base[i][none]), "a token without an adapter is its base"


# tokens from one on, ranks that fill no vector and no tile, ragged rows
SHAPES = [(1, 32, [1], 1, 1), (1, 4096, [4096], 16, 3), (2, 64, [17], 3, 2), (3, 96, [300], 5, 4), (5, 256, [129, 64, 1], 8, 3), (7, 2880, [720], 20, 2),
          (16, 512, [256, 256], 16, 5), (17, 1024, [1000], 31, 20), (33, 128, [65, 33], 64, 2), (64, 2048, [512, 128, 128], 16, 64), (65, 352, [77], 33, 3),
          (100, 160, [515], 128, 7), (128, 1024, [1028], 64, 1), (129, 96, [31, 1000, 5, 260], 12, 130), (257, 544, [640], 48, 4), (300, 64, [2000], 96, 2),
          (513, 256, [100], 257, 2), (40, 128, [96], 512, 3), (1000, 288, [144, 160], 24, 9)]


@pytest.fixture(params=["chosen", "one", "dots", "matrix", "matrix+sum"])
def form(dev, request):
    """Every form of the call beside the one it chooses ("adapter.form"; one that has no kernel for a rank is not taken)."""
    dev.set_tuning(adapter__form={"chosen": 0, "one": 1, "dots": 2, "matrix": 3, "matrix+sum": 4}[request.param])
    yield
    dev.set_tuning(adapter__form=0)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ntok, k, rows, rank, n_adapter", SHAPES)
def test_whole_numbers_are_exact(dev, form, ntok, k, rows, rank, n_adapter, t):
    c = Case(ntok + rank, ntok, k, rows, rank, n_adapter, t=t, whole=True)
    assert c.call(dev)
    dev.synchronize()
    c.check(exact=True)


@pytest.mark.parametrize("slices", [1, 3, 16])
@pytest.mark.parametrize("sets", [1, 2, 4])
def test_cuts_of_the_work(dev, form, slices, sets):
    dev.set_tuning(adapter__slices=slices, adapter__sets=sets)
    for ntok, k, rows, rank in ((5, 1120, [700], 40), (130, 2080, [513, 1030], 12)):
        c = Case(slices + sets, ntok, k, rows, rank, 3, whole=True, ranks=[rank, 3, 5])
        assert c.call(dev)
        dev.synchronize()
        c.check(exact=True)
    dev.set_tuning(adapter__slices=0, adapter__sets=0)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("xt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ntok, k, rows, rank, n_adapter", [(1, 4096, [2048], 16, 3), (9, 2880, [720, 100], 20, 2), (48, 1024, [1000], 64, 8), (200, 1536, [1031], 40, 3),
                                                            (700, 512, [512, 256], 64, 2)])
def test_types(dev, form, ntok, k, rows, rank, n_adapter, xt, t):
    c = Case(7 * ntok + k, ntok, k, rows, rank, n_adapter, t=t, xt=xt)
    assert c.call(dev)
    dev.synchronize()
    c.check()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ntok", [1, 12, 90, 400])
def test_ranks_of_their_own(dev, form, ntok, t):
    """Each adapter its rank, none among them, more than the bank's among them; what the banks hold past it is not used."""
    ranks = [0, 1, 5, 16, 23, 24, 1000, 7]
    c = Case(ntok, ntok, 320, [200, 72], 24, 8, t=t, ranks=ranks, whole=True)
    for bank, axis in ((c.d["a"], 1), (c.d["b"], 2)):
        for v in bank:
            h = v.get()
            for e, r in enumerate(ranks):
                if axis == 1:
                    h[e, r:] = stored(np.float32([np.nan]), t)[0]
                else:
                    h[e, :, r:] = stored(np.float32([np.nan]), t)[0]
            v.put(h)
    assert c.call(dev)
    dev.synchronize()
    c.check(exact=True)


@pytest.mark.parametrize("ntok", [3, 64, 500])
def test_no_number_stays_with_its_tokens(dev, form, ntok):
    """An adapter of NaN and infinity, and a token of NaN: no other token sees them."""
    c = Case(ntok, ntok, 256, [130], 16, 3, whole=True, ids=np.arange(ntok) % 4)
    for v in (c.d["a"][0], c.d["b"][0]):
        h = v.get()
        h[1] = np.nan
        h[1, 0] = np.inf
        v.put(h)
    x = c.d["x"].get()
    x[2] = np.inf
    c.d["x"].put(x)
    assert c.call(dev)
    dev.synchronize()
    got = c.d["out"][0].get()[:-1]
    fine = (c.ids != 1) & (np.arange(ntok) != 2)
    assert np.array_equal(got[fine], c.want[0][fine].astype(np.float32))
    assert np.all(np.isnan(got[c.ids == 1])) and not np.any(np.isfinite(got[2]))


@pytest.mark.parametrize("ntok", [1, 20, 300])
def test_in_place_without_base_and_without_scale(dev, form, ntok):
    c = Case(ntok, ntok, 512, [192, 48], 16, 4, whole=True)
    assert c.call(dev, in_place=True)
    dev.synchronize()
    c.check(exact=True)
    c = Case(ntok, ntok, 512, [192, 48], 16, 4, whole=True, base=False, scale=False)
    assert c.call(dev)
    dev.synchronize()
    c.check(exact=True)


@pytest.mark.parametrize("order", ["one", "none", "sorted", "runs", "each its own", "past the last", "blocks"])
@pytest.mark.parametrize("ntok", [6, 64, 380])
def test_orders_of_the_tokens(dev, form, ntok, order):
    na = ntok if order == "each its own" else 5
    rng = np.random.default_rng(ntok)
    ids = {"one": np.full(ntok, 3), "none": np.full(ntok, 0xFFFFFFFF), "sorted": np.sort(rng.integers(0, 6, ntok)),
           "runs": np.repeat([2, 5, 0, 4], -(-ntok // 4))[:ntok], "each its own": rng.permutation(ntok),
           "past the last": np.where(np.arange(ntok) % 3 == 0, 5, np.where(np.arange(ntok) % 3 == 1, 1 << 31, 4)),
           "blocks": np.arange(ntok) // 16 % 6}[order]
    c = Case(ntok + 1, ntok, 128, [100, 36], 16, na, whole=True, ids=ids)
    assert c.call(dev)
    dev.synchronize()
    c.check(exact=True)


def test_a_call_after_a_larger_one(dev, form):
    """The workspace holds what an earlier call left: nothing of it is read."""
    for ntok, rank, na in ((600, 96, 3), (20, 8, 2), (3, 64, 1), (250, 33, 4)):
        c = Case(ntok, ntok, 256, [90, 130], rank, na, whole=True, ranks=None if rank != 33 else [0, 33, 4, 9])
        assert c.call(dev)
        dev.synchronize()
        c.check(exact=True)


@pytest.mark.parametrize("ntok, rank", [(1, 16), (24, 16), (24, 64), (300, 64), (5000, 16)])
def test_captured_and_replayed(dev, form, ntok, rank):
    """Two graphs of one context, their calls replayed in turn between eager calls and after the workspace has grown."""
    st = Stream()
    dev.reserve_adapters(ntok, 2, rank)
    c, e = (Case(s, ntok, 512, [200, 60], rank, 4, whole=True) for s in (1, 2))
    graphs = []
    for v in (c, e):
        with Graph.capture(st.handle) as g:
            assert v.call(dev, stream=st.handle)
        graphs.append(g)
    big = Case(3, 4 * ntok, 128, [64] * 4, min(512, 4 * rank), 2, whole=True)
    for turn in range(3):
        for v, g in ((c, graphs[0]), (e, graphs[1])):
            for o in v.d["out"]:
                o.put(np.full(o.shape, -7e30, np.float32))
            v.d["x"].put(-v.d["x"].get())             # other inputs each time: the adapters' part changes sign
            for i, b in enumerate(v.base):
                v.want[i] = 2 * b - v.want[i]
            g.launch()
            st.synchronize()
            v.check(exact=True)
        assert big.call(dev)
        dev.synchronize()
        big.check(exact=True)
    st.destroy()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rank", [3, 8, 11, 16, 20, 24, 33, 61, 100])
def test_an_infinity_stays_in_its_column(dev, form, rank, t):
    """Wherever it stands in a row of B, also where rows are read in pieces that overlap; other columns and adapters are as without it."""
    c = Case(rank, 6, 64, [70], rank, 2, t=t, whole=True, ids=[0, 1, 0, 2, 1, 0], scale=False)
    h = c.d["b"][0].get()
    cols = [0, 31, 69]
    for i, col in enumerate(cols):
        h[1, col, [0, rank // 2, rank - 1][i]] = stored(np.float32([np.inf]), t)[0]
    c.d["b"][0].put(h)
    assert c.call(dev)
    dev.synchronize()
    got, hit = c.d["out"][0].get()[:-1], np.zeros((6, 70), bool)
    hit[np.ix_([1, 4], cols)] = True
    assert np.all(~np.isfinite(got[hit])) and np.array_equal(got[~hit], c.want[0].astype(np.float32)[~hit])


def test_reserved_calls_allocate_nothing(dev):
    dev.reserve_adapters(700, 3, 80)
    c = Case(5, 700, 128, [64, 64, 64], 80, 2, whole=True)
    before = mem_info()[0]
    assert c.call(dev)
    dev.synchronize()
    assert mem_info()[0] == before
    c.check(exact=True)


@pytest.mark.parametrize("which", [2, 3])
def test_a_reservation_covers_every_cut_of_the_work(dev, which):
    """3000 tokens of sixteen slices each would be more sums than are reserved for 3000 tokens."""
    from jitllm_amd.device import Device
    c = Case(6, 3000, 16384, [64], 64, 2, t="bf16", xt="bf16", whole=True)
    own = Device(0)
    try:
        own.set_tuning(adapter__form=which)
        own.reserve_adapters(3000, 1, 64)
        assert Case(7, 3, 64, [8], 4, 1).call(own)
        own.synchronize()
        before = mem_info()[0]
        assert c.call(own)
        own.synchronize()
        assert mem_info()[0] == before
        c.check(exact=True)
    finally:
        own.close()


@pytest.mark.parametrize("which", [0, 3])
@pytest.mark.parametrize("ntok, n_adapter, rank", [(5000, 8192, 3), (70000, 5, 4), (4097, 1, 40)])
def test_many_tokens_and_many_adapters(dev, which, ntok, n_adapter, rank):
    dev.set_tuning(adapter__form=which)
    c = Case(ntok, ntok, 32, [12], rank, n_adapter, whole=True)
    assert c.call(dev)
    dev.synchronize()
    dev.set_tuning(adapter__form=0)
    c.check(exact=True)


def test_same_bits_every_time(dev, form):
    for ntok in (5, 64, 400):
        c = Case(ntok, ntok, 1024, [300], 32, 3)
        assert c.call(dev)
        dev.synchronize()
        first = c.d["out"][0].get()
        assert c.call(dev)
        dev.synchronize()
        assert np.array_equal(first, c.d["out"][0].get())


def test_banks_past_32_bits(dev):
    """The last of 1100 adapters of 2^21 elements starts past 2^31 elements of its bank."""
    k, rows, rank, na, ntok = 4096, 4096, 512, 1100, 3
    from jitllm_amd.hipmem import check, hip
    c = Case(1, ntok, k, [rows], rank, 1, whole=True, ids=[0, 0, 1])
    a, b = (DeviceArray(shape=(na * rank * k,), dtype=np.float16) for _ in range(2))
    one = rank * k * 2
    check(hip().hipMemcpy(a.ptr + (na - 1) * one, c.d["a"][0].ptr, one, 3), "hipMemcpy")
    check(hip().hipMemcpy(b.ptr + (na - 1) * one, c.d["b"][0].ptr, one, 3), "hipMemcpy")
    ids, scale = DeviceArray(np.uint32([na - 1, na - 1, na])), DeviceArray(np.full(na, c.scale[0], np.float32))
    d = c.d
    assert dev.adapter_group_dev([d["out"][0].ptr], [d["base"][0].ptr], [rows], [a.ptr], [b.ptr], quant.F16, na, rank, d["x"].ptr, k, ids.ptr, ntok, scale=scale.ptr)
    dev.synchronize()
    c.check(exact=True)
    a.free(), b.free()


def test_a_block_step_around_its_projections(dev):
    """Norm, the projections with their adapters, the router and the mixture, one after the other on a stream of the caller's, as
    a program runs them: every step against the plain statement of it over the values the step before left."""
    from test_gpu_moe_select import reference as select_reference
    from test_gpu_norm_rows import check_y, reference as norm_reference
    dev.SetActWindow(256)
    st, t = Stream(), quant.Q4_K
    for rows in (1, 6, 90):
        rng = np.random.default_rng(rows)
        e, kv, ne, ku, f, rank, na = 512, 256, 16, 4, 256, 16, 3
        num = lambda *s: rng.standard_normal(s).astype(np.float32)
        wq, wk = (DeviceArray(synth.quantized_weights(t, r, e, seed=r)) for r in (e, kv))
        banks = [DeviceArray(synth.quantized_weights(t, ne * r, c, seed=5 + i)) for i, (r, c) in enumerate(((f, e), (f, e), (e, f)))]
        x, resid, w = num(rows, e), num(rows, e), 1 + num(e) / 10
        xd, rd, wd, yd = DeviceArray(x), DeviceArray(resid), DeviceArray(w), DeviceArray(np.zeros((rows, e), np.float32))
        q, k = (DeviceArray(np.zeros((rows, n), np.float32)) for n in (e, kv))
        fan = np.float32(1 / np.sqrt(e))
        a, b = [(num(na, rank, e) * fan).astype(np.float16) for _ in range(2)], [num(na, n, rank).astype(np.float16) for n in (e, kv)]
        ad, bd, ids = [DeviceArray(v) for v in a], [DeviceArray(v) for v in b], rng.integers(0, na + 1, rows).astype(np.uint32)
        idd, router, bias = DeviceArray(ids), num(ne, e) * fan, 0.1 * num(ne)
        routerd, biasd, logits = DeviceArray(router), DeviceArray(bias), DeviceArray(np.zeros((rows, ne), np.float32))
        sel, wt = DeviceArray(np.zeros((rows, ku), np.uint32)), DeviceArray(np.zeros((rows, ku), np.float32))
        s = st.handle
        # twice, so that the second run follows the first's leftovers
        for _ in range(2):
            rd.put(resid)
            assert dev.norm_rows_dev(xd.ptr, rows, e, wd.ptr, 1e-5, resid=rd.ptr, resid_out=rd.ptr, y=yd.ptr, stream=s)
            assert dev.matmul_dev(q.ptr, t, wq.ptr, yd.ptr, e, e, rows, stream=s) and dev.matmul_dev(k.ptr, t, wk.ptr, yd.ptr, kv, e, rows, stream=s)
            st.synchronize()
            base = [q.get(), k.get()]
            assert dev.adapter_group_dev([q.ptr, k.ptr], [q.ptr, k.ptr], [e, kv], [v.ptr for v in ad], [v.ptr for v in bd], quant.F16, na, rank, yd.ptr, e, idd.ptr,
                                         rows, stream=s)
            assert dev.moe_logits_dev(logits.ptr, 0, routerd.ptr, yd.ptr, ne, e, rows, stream=s)
            assert dev.moe_select_dev(logits.ptr, rows, ne, ku, sel.ptr, ku, wt.ptr, score=1, bias=biasd.ptr, n_group=4, k_group=2, group_top=2, scale=2.0, stream=s)
            st.synchronize()
            h, y = norm_reference(x, resid, 1.0, w, 1e-5)
            assert np.array_equal(rd.get(), h)
            check_y(yd.get(), y, quant.F32)
            y64 = yd.get().astype(np.float64)
            for o, bs, ai, bi in ((q, base[0], a[0], b[0]), (k, base[1], a[1], b[1])):
                want, most = bs.astype(np.float64), np.zeros_like(bs, np.float64)
                for r in range(rows):
                    if ids[r] < na:
                        want[r] += bi[ids[r]].astype(np.float64) @ (ai[ids[r]].astype(np.float64) @ y64[r])
                        most[r] = np.abs(bi[ids[r]].astype(np.float64)) @ (np.abs(ai[ids[r]].astype(np.float64)) @ np.abs(y64[r]))
                assert np.all(np.abs(o.get() - want) <= 2.0 ** -24 * ((e + rank + 4) * most + np.abs(want)))
            ws, ww = select_reference(logits.get(), ku, 1, bias, 4, 2, 2, True, 2.0)
            assert np.array_equal(sel.get(), ws) and np.all(np.abs(wt.get() - ww) <= np.abs(ww) * 20 * 2.0 ** -24)
            before = rd.get()
            assert dev.moe_ffn_dev(rd.ptr, t, *[v.ptr for v in banks], yd.ptr, sel.ptr, ku, wt.ptr, rows, ku, ne, f, e, stream=s)
            st.synchronize()
            assert np.all(np.isfinite(rd.get())) and np.any(rd.get() != before)
    st.destroy()
    dev.SetActWindow(32)
