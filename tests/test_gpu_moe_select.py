"""The router's general form (jl_moe_select_dev) against a plain statement of it: scores in f64 narrowed to f32, the order by
(f32 choice descending, index ascending), so the selection is equal; weights to 20 roundings of f32 (a score each, up to sixteen
additions, the quotient and the scale), 20 * 2^-24 of the value."""
import numpy as np
import pytest

from jitllm_amd import quant, synth
from jitllm_amd.hipmem import DeviceArray, Graph, Stream

pytestmark = pytest.mark.gpu

NONE = np.uint32(0xABCDABCD)


def reference(logits, k, score, bias, n_group, k_group, top, renorm, scale):
    rows, n = logits.shape
    l = logits.astype(np.float64)
    with np.errstate(all="ignore"):
        if score == 0:
            e = np.exp(l - np.max(l, axis=1, keepdims=True))
            s64 = e / e.sum(1, keepdims=True)
        else:
            s64 = 1.0 / (1.0 + np.exp(-l))
        s = s64.astype(np.float32)
        c = s if bias is None else s + bias
    sel, wt = np.full((rows, k), n, np.uint32), np.zeros((rows, k))
    for r in range(rows):
        can = (logits[r] != -np.inf) & (c[r] > -np.inf)       # (no number: not greater)
        if n_group > 1:
            size, worth = n // n_group, []
            for g in range(n_group):
                best = sorted((c[r, e] for e in range(g * size, (g + 1) * size) if can[e]), reverse=True)[:top]
                if best:
                    worth.append((-(best[0] + best[1] if len(best) > 1 else best[0]), g))
            kept = {g for _, g in sorted(worth)[:k_group]}
            can = can & np.isin(np.arange(n) // size, list(kept))
        order = sorted((-c[r, e], e) for e in np.nonzero(can)[0])[:k]
        total = sum(float(s[r, e]) for _, e in order)         # of the narrowed scores, as the weights are defined
        for i, (_, e) in enumerate(order):
            sel[r, i], wt[r, i] = e, float(s[r, e]) / ((total + 1e-20) if renorm else 1.0) * np.float64(np.float32(scale))
    return sel, wt


def run(dev, logits, k, score=0, bias=None, n_group=1, k_group=1, top=1, renorm=True, scale=1.0, stride=None, stream=None):
    rows, n = logits.shape
    stride = stride or k
    ld, bd = DeviceArray(logits), None if bias is None else DeviceArray(bias)
    sel, wt = DeviceArray(np.full((rows + 1, stride), NONE)), DeviceArray(np.full((rows + 1, k), -7.0, np.float32))
    before = dev.launch_count()
    assert dev.moe_select_dev(ld.ptr, rows, n, k, sel.ptr, stride, wt.ptr, score=score, bias=None if bd is None else bd.ptr, n_group=n_group,
                              k_group=k_group, group_top=top, renorm=renorm, scale=scale, stream=stream)
    assert dev.launch_count() == before + 1
    dev.synchronize()
    s, w = sel.get(), wt.get()
    assert np.all(s[rows] == NONE) and np.all(s[:, k:] == NONE) and np.all(w[rows] == -7.0), "wrote past its operands"
    return s[:rows, :k], w[:rows]


def check(dev, logits, k, **kw):
    got = run(dev, logits, k, **kw)
    kw.pop("stride", None)
    full = dict(score=0, bias=None, n_group=1, k_group=1, top=1, renorm=True, scale=1.0)
    full.update(kw)
    sel, wt = reference(logits, k, **full)
    assert np.array_equal(got[0], sel)
    assert np.all(np.abs(got[1] - wt) <= np.abs(wt) * 20 * 2.0 ** -24 + 1e-37)


SIZES = [1, 2, 3, 7, 16, 33, 64, 65, 100, 128, 129, 160, 255, 256, 257, 384, 512, 513, 777, 1000, 1024]


@pytest.fixture(params=["chosen", "packed", "whole"])
def form(dev, request):
    """The kernel's two ways to select, beside the one it chooses ("moe.select")."""
    dev.set_tuning(moe__select={"chosen": 0, "packed": 1, "whole": 2}[request.param])
    yield
    dev.set_tuning(moe__select=0)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("n", SIZES)
def test_sizes(dev, form, n, score):
    rng = np.random.default_rng(n)
    for k in sorted({1, min(2, n), min(8, n), min(13, n), min(16, n)}):
        logits = rng.standard_normal((9, n)).astype(np.float32)
        check(dev, logits, k, score=score, stride=k + 1)
        check(dev, logits, k, score=score, bias=(0.1 * rng.standard_normal(n)).astype(np.float32), renorm=False, scale=2.5)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("top", [1, 2])
@pytest.mark.parametrize("n, n_group, k_group, k", [(256, 8, 4, 8), (8, 8, 3, 3), (16, 8, 2, 4), (160, 8, 3, 6), (64, 64, 16, 16), (1024, 64, 5, 16), (384, 4, 1, 10),
                                                    (1000, 2, 1, 16), (63, 7, 7, 9), (66, 2, 1, 5), (1024, 2, 2, 8), (128, 16, 1, 8), (256, 4, 2, 8), (12, 3, 2, 8)])
def test_groups(dev, form, n, n_group, k_group, k, top, score):
    rng = np.random.default_rng(n + n_group + k)
    logits, bias = rng.standard_normal((17, n)).astype(np.float32), (0.2 * rng.standard_normal(n)).astype(np.float32)
    check(dev, logits, k, score=score, bias=bias, n_group=n_group, k_group=k_group, top=top, scale=1.5)
    check(dev, logits, k, score=score, n_group=n_group, k_group=k_group, top=top)
    bias[rng.permutation(n)[: n // 3]] = -np.inf
    check(dev, logits, k, score=score, bias=bias, n_group=n_group, k_group=k_group, top=top)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("n, groups", [(40, 1), (256, 8), (600, 1)])
def test_ties_go_to_the_lowest_index(dev, form, n, groups, score):
    rng = np.random.default_rng(n)
    logits = rng.integers(-1, 2, (33, n)).astype(np.float32)
    kw = dict(score=score, n_group=groups, k_group=max(1, groups // 2), top=2 if groups > 1 else 1)
    check(dev, logits, 8, **kw)
    check(dev, np.zeros((3, n), np.float32), 8, **kw)
    check(dev, np.full((2, n), 60.0, np.float32), 8, **kw)             # scores that narrow to one value
    logits = (30 + rng.standard_normal((9, n))).astype(np.float32)
    check(dev, logits, 8, **kw)
    bias = rng.choice(np.float32([-1.0, 0.0, -0.0]), n).astype(np.float32)
    check(dev, np.full((4, n), -120.0, np.float32), 8, bias=bias, **kw)  # choices of either zero


def test_masks(dev, form):
    """Experts out of service by logit or bias, fewer than are wanted, none at all; the type's lowest value is a number."""
    n, k = 70, 8
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((8, n)).astype(np.float32)
    logits[1, 5:] = -np.inf                  # five left
    logits[2] = -np.inf                      # none
    logits[3, 1:] = -np.inf                  # one
    logits[4] = np.finfo(np.float32).min
    logits[5, ::2] = np.finfo(np.float32).min
    logits[6, 7] = np.inf
    logits[7, 9] = np.nan
    for score in (0, 1):
        check(dev, logits, k, score=score)
        check(dev, logits, k, score=score, n_group=7, k_group=2, top=2)
    bias = np.full(n, -np.inf, np.float32)
    bias[[3, 40, 69]] = [0.1, np.nan, -5.0]
    for score in (0, 1):
        check(dev, logits, k, score=score, bias=bias)
        check(dev, logits, k, score=score, bias=bias, n_group=7, k_group=7, top=2)
    sel, wt = run(dev, logits, k, score=0)
    for r in (2, 6, 7):                      # nothing, +infinity under the softmax, a NaN under the softmax
        assert np.all(sel[r] == n) and np.all(wt[r] == 0)
    sel, wt = run(dev, logits, k, score=1)
    assert sel[6, 0] == 7 and wt[6, 0] > 0 and 9 not in sel[7] and np.all(wt[7] > 0)


@pytest.mark.parametrize("n", [200, 384, 1024])
def test_choices_that_share_their_high_bits(dev, form, n):
    """Choices a few steps of f32 apart, in any order: packed keys (22 bits) cannot tell them, whole ones do.  A handful of them
    among others, then more than the 64 that are put in order, the whole row."""
    rng = np.random.default_rng(n)
    for close in (2, 5, 30, 63, 64, 65, 100, n):
        logits = (rng.standard_normal((6, n)) - 3).astype(np.float32)
        for row in logits:
            at = rng.permutation(n)[: min(close, n)]
            row[at] = np.float32(1.0) + rng.integers(0, 40, len(at)).astype(np.float32) * np.float32(2.0 ** -23)
        check(dev, logits, 8, score=1)
        check(dev, logits, 16, score=0, bias=np.zeros(n, np.float32))


def test_softmax_without_bias_is_the_router(dev):
    """What jl_moe_route_dev selects and weighs, bit for bit in the selection."""
    for n, k in ((128, 8), (256, 4), (1000, 16)):
        logits = np.random.default_rng(n).standard_normal((200, n)).astype(np.float32)
        ld, sel, wt = DeviceArray(logits), DeviceArray(np.full((200, k), NONE)), DeviceArray(np.zeros((200, k), np.float32))
        assert dev.moe_route_dev(ld.ptr, 200, n, k, sel.ptr, k, wt.ptr)
        dev.synchronize()
        got = run(dev, logits, k)
        assert np.array_equal(got[0], sel.get()) and np.allclose(got[1], wt.get(), rtol=20 * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("rows", [1, 5, 64, 1000, 70001])
def test_many_rows(dev, rows):
    n, k = 96, 6
    logits = np.random.default_rng(rows).standard_normal((rows, n)).astype(np.float32)
    bias = (0.1 * np.random.default_rng(1).standard_normal(n)).astype(np.float32)
    sel, wt = run(dev, logits, k, score=1, bias=bias, n_group=4, k_group=2, top=2)
    at = np.unique(np.concatenate([np.arange(min(rows, 40)), np.arange(max(0, rows - 40), rows), np.random.default_rng(2).integers(0, rows, 100)]))
    want = reference(logits[at], k, 1, bias, 4, 2, 2, True, 1.0)
    assert np.array_equal(sel[at], want[0]) and np.all(np.abs(wt[at] - want[1]) <= want[1] * 20 * 2.0 ** -24)


def test_captured_and_replayed(dev):
    rows, n, k = 50, 256, 8
    rng = np.random.default_rng(21)
    st = Stream()
    bias = (0.1 * rng.standard_normal(n)).astype(np.float32)
    ld, bd, sel, wt = DeviceArray(np.zeros((rows, n), np.float32)), DeviceArray(bias), DeviceArray(np.full((rows, k), NONE)), DeviceArray(np.zeros((rows, k), np.float32))
    with Graph.capture(st.handle) as g:
        assert dev.moe_select_dev(ld.ptr, rows, n, k, sel.ptr, k, wt.ptr, score=1, bias=bd.ptr, n_group=8, k_group=4, group_top=2, stream=st.handle)
    for _ in range(3):
        logits = rng.standard_normal((rows, n)).astype(np.float32)
        ld.put(logits)
        g.launch()
        st.synchronize()
        want = reference(logits, k, 1, bias, 8, 4, 2, True, 1.0)
        assert np.array_equal(sel.get(), want[0]) and np.all(np.abs(wt.get() - want[1]) <= want[1] * 20 * 2.0 ** -24)
    st.destroy()


def test_an_empty_place_adds_nothing_to_the_mixture(dev):
    """A selection with empty places through the routed block: as the same block over the experts that were selected, to the 1e-3
    of a mixture block whose columns may run in another form (a 32-bit sum on a border of the int8 steps moves a value by one)."""
    dev.SetActWindow(256)
    rows, n, k, f, e, t = 5, 6, 4, 256, 256, quant.Q4_K
    rng = np.random.default_rng(8)
    banks = [DeviceArray(synth.quantized_weights(t, n * r, c, seed=s)) for s, (r, c) in enumerate(((f, e), (f, e), (e, f)))]
    x, resid = rng.standard_normal((rows, e)).astype(np.float32), rng.standard_normal((rows, e)).astype(np.float32)
    bias = np.full(n, -np.inf, np.float32)
    bias[[1, 4]] = 0.0                                     # two of six in service, four wanted
    ld, bd, xd = DeviceArray(rng.standard_normal((rows, n)).astype(np.float32)), DeviceArray(bias), DeviceArray(x)
    sel, wt = DeviceArray(np.zeros((rows, k), np.uint32)), DeviceArray(np.zeros((rows, k), np.float32))
    assert dev.moe_select_dev(ld.ptr, rows, n, k, sel.ptr, k, wt.ptr, bias=bd.ptr)
    got, want = DeviceArray(resid), DeviceArray(resid)
    dev.synchronize()
    assert np.all(np.sort(sel.get(), 1) == [1, 4, n, n])
    assert dev.moe_ffn_dev(got.ptr, t, *[b.ptr for b in banks], xd.ptr, sel.ptr, k, wt.ptr, rows, k, n, f, e)
    sel2, wt2 = DeviceArray(sel.get()[:, :2].copy()), DeviceArray(wt.get()[:, :2].copy())
    assert dev.moe_ffn_dev(want.ptr, t, *[b.ptr for b in banks], xd.ptr, sel2.ptr, 2, wt2.ptr, rows, 2, n, f, e)
    dev.synchronize()
    moved = np.linalg.norm(want.get() - resid)
    assert moved > 0 and np.linalg.norm(got.get() - want.get()) <= 1e-3 * moved
    dev.SetActWindow(32)
