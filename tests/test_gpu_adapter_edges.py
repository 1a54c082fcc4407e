"""Adapters (jl_adapter_group_dev) where a caller's numbers are at an end of their range, against the plain statement in
test_gpu_adapters."""
import pytest

from test_gpu_adapters import Case

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
