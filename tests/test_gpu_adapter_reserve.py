"""jl_reserve_adapters: a reserved call allocates nothing, in every form and cut, on a context of its own whose workspace is what was
reserved and no more; the same calls without a reservation show that the free memory would have told."""
import numpy as np
import pytest

from jitllm_amd.device import Device
from jitllm_amd.hipmem import mem_info
from test_gpu_adapters import Case

pytestmark = pytest.mark.gpu

# tokens, k, rows, rank, adapters: several projections, ranks that fill no tile, the most adapters, one token of the largest rank
CALLS = [(20000, 64, [8, 8, 8], 33, 5), (20000, 32, [4], 80, 1), (9000, 1024, [8, 12, 4, 8], 80, 3), (12000, 32, [8], 33, 8192), (40000, 64, [16, 16], 3, 64),
         (3000, 16384, [8, 8], 64, 7), (1500, 2048, [8] * 4, 512, 2)]


def own(tuned):
    d = Device(0)
    d.set_tuning(adapter__form=tuned)
    d.reserve_adapters(1, 1, 1)
    assert Case(7, 3, 64, [8], 4, 1).call(d)     # (whatever the first launch of a context brings)
    d.synchronize()
    return d


@pytest.mark.parametrize("tuned", [0, 2, 3, 4])
@pytest.mark.parametrize("ntok, k, rows, rank, n_adapter", CALLS)
def test_a_reserved_call_allocates_nothing(tuned, ntok, k, rows, rank, n_adapter):
    c = Case(ntok, ntok, k, rows, rank, n_adapter, whole=True)
    less = Case(1, max(1, ntok // 16), k, rows[:1], max(1, rank // 2), n_adapter, whole=True)     # within the same reservation: more slices a token
    d = own(tuned)
    try:
        d.reserve_adapters(ntok, len(rows), rank)
        before = mem_info()[0]
        for v in (c, less, c):
            assert v.call(d)
            d.synchronize()
            assert mem_info()[0] == before
        c.check(exact=True)
        less.check(exact=True)
    finally:
        d.close()


def test_without_a_reservation_it_does():
    ntok, k, rows, rank, n_adapter = CALLS[0]
    c = Case(ntok, ntok, k, rows, rank, n_adapter, whole=True)
    d = own(3)
    try:
        before = mem_info()[0]
        assert c.call(d)
        d.synchronize()
        assert mem_info()[0] < before
        c.check(exact=True)
    finally:
        d.close()
