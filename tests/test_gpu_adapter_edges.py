"""Adapters (jl_adapter_group_dev) where a caller's numbers are at an end of their range, against the plain statement in
test_gpu_adapters."""
import numpy as np
import pytest

from test_gpu_adapters import Case, form, stored, values  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sets", [-1, -(1 << 31), 3, 5, 1 << 24, (1 << 31) - 1])
def test_a_tuned_cut_outside_its_range(dev, sets):
    """"adapter.sets" and "adapter.slices" are brought into their range: a workgroup has a first column and columns."""
    dev.set_tuning(adapter__form=2, adapter__sets=sets, adapter__slices=sets)
    try:
        for form in (2, 3, 4):
            dev.set_tuning(adapter__form=form)
            c = Case(7, 9, 288, [1300, 70], 24, 3, whole=True)
            assert c.call(dev)
            dev.synchronize()
            c.check(exact=True)
    finally:
        dev.set_tuning(adapter__form=0, adapter__sets=0, adapter__slices=0)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("exponent", [-110, -100, -60, 20])
def test_small_values_are_exact_in_every_form(dev, form, exponent, t):  # noqa: F811
    """x of 24 bits from 2^-110 on: one product by a power of two and nothing to add, so no form rounds."""
    ntok, k, rows = 70, 64, 5
    rng = np.random.default_rng(exponent + 200)
    c = Case(1, ntok, k, [rows], 1, 1, t=t, ids=np.zeros(ntok), base=False, scale=False)
    x, a = np.zeros((ntok, k), np.float32), np.zeros((1, 1, k), np.float32)
    x[:, 37] = (1 + rng.integers(0, 1 << 23, ntok) / 2.0 ** 23) * 2.0 ** exponent
    a[0, 0, 37] = 2.0 ** 100
    c.d["x"].put(x), c.d["a"][0].put(stored(a, t)), c.d["b"][0].put(stored(np.ones((1, rows, 1), np.float32), t))
    assert c.call(dev)
    dev.synchronize()
    assert np.array_equal(c.d["out"][0].get()[:-1], np.repeat(x[:, 37:38] * np.float32(2.0 ** 100), rows, 1))


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_no_finite_number_in_every_form(dev, form, t):  # noqa: F811
    """An infinity in x, in A or in a column of B, and a sum past f32: no finite number where the formula has none, the formula's elsewhere."""
    ntok, k, rows, rank = 66, 96, 70, 9
    c = Case(2, ntok, k, [rows], rank, 3, t=t, whole=True, ids=np.arange(ntok) % 4)
    x, a, b = c.d["x"].get(), c.d["a"][0].get(), c.d["b"][0].get()
    x[4, 7], x[8] = np.inf, 3e38                                   # both of adapter 0
    a[0, :, 7], a[0, 0, :] = stored(np.float32([1]), t)[0], stored(np.float32([2]), t)[0]
    b[0, :, 0] = stored(np.float32([1]), t)[0]
    a[1, 4, 9] = stored(np.float32([np.inf]), t)[0]
    x[:, 9] = 1
    b[1, :, 4] = stored(np.float32([1]), t)[0]
    b[2, 33, 8] = stored(np.float32([np.inf]), t)[0]
    c.d["x"].put(x), c.d["a"][0].put(a), c.d["b"][0].put(b)
    assert c.call(dev)
    dev.synchronize()
    got, bad = c.d["out"][0].get()[:-1], np.zeros((ntok, rows), bool)
    bad[[4, 8]] = True
    bad[c.ids == 1] = True
    u2 = values(x, "f32")[c.ids == 2] @ values(a, t)[2].T              # (a zero that meets the infinity is no number either)
    bad[c.ids == 2, 33] = True
    assert np.all(~np.isfinite(got[bad])) and np.all(np.isfinite(got[~bad]))
    two = got[c.ids == 2]
    keep = np.arange(rows) != 33
    want = c.base[0][c.ids == 2] + c.scale[2] * (u2 @ np.where(np.isfinite(values(b, t)[2]), values(b, t)[2], 0).T)
    assert np.array_equal(two[:, keep], want[:, keep].astype(np.float32))
