"""Adapters of large banks (jl_adapter_group_dev): how a call is cut and which form it takes goes by how many adapters there are, its
result and its time by how many of them its tokens carry."""
import numpy as np
import pytest

from jitllm_amd import quant
from test_gpu_adapters import Case, form  # noqa: F401
from test_gpu_dispatch_times import us

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("met", [1, 3, 60])
@pytest.mark.parametrize("ntok, n_adapter, rank", [(60, 700, 12), (90, 8192, 4), (700, 300, 40), (2500, 1000, 9)])
def test_most_of_a_bank_lies_idle(dev, form, ntok, n_adapter, rank, met):  # noqa: F811
    ids = np.random.default_rng(met).permutation(n_adapter)[:met][np.arange(ntok) * met // ntok]
    c = Case(ntok + met, ntok, 64, [33, 20], rank, n_adapter, whole=True, ids=ids)
    assert c.call(dev)
    dev.synchronize()
    c.check(exact=True)


class Bank:
    """Operands whose values nobody reads: 16-bit adapters beside `rows`, `met` of n_adapter carried in runs."""

    def __init__(self, dev, devbuf, ntok, k, rows, rank, n_adapter, met):
        z = lambda *s: devbuf(shape=s, dtype=np.uint16, fill=0)
        self.keep = x, a, b = z(ntok, k), z(n_adapter, rank, k), z(n_adapter, rows, rank)
        self.out = devbuf(shape=(ntok, rows), dtype=np.float32, fill=0)
        self.ids = devbuf((np.arange(ntok) * met // ntok * (n_adapter // met)).astype(np.uint32))
        self.call = lambda: dev.adapter_group_dev([self.out.ptr], [self.out.ptr], [rows], [a.ptr], [b.ptr], quant.BF16, n_adapter, rank, x.ptr, k, self.ids.ptr, ntok,
                                                  x_type=quant.BF16)


def test_a_prompt_beside_a_large_bank_takes_the_matrix_cores(dev, devbuf):
    """2048 tokens of three adapters: four launches, of a bank of 512 as of one of three."""
    for n_adapter in (3, 512):
        c = Bank(dev, devbuf, 2048, 2048, 4096, 64, n_adapter, 3)
        assert c.call()
        before = dev.launch_count()
        assert c.call()
        assert dev.launch_count() == before + 4
        dev.synchronize()


@pytest.mark.parametrize("ntok", [1024, 2048])
def test_an_idle_bank_costs_little(dev, devbuf, ntok):
    """512 adapters of which three are met, rank 64: within 1.6 times the best form and cut there is.  (By the size of the bank
    alone, 2 and 3 times.)"""
    c = Bank(dev, devbuf, ntok, 4096, 4096, 64, 512, 3)
    t = us(dev, {"chosen": ({}, c.call), "dots": (dict(adapter__form=2), c.call), "matrix": (dict(adapter__form=3, adapter__slices=16), c.call),
                 "matrix+sum": (dict(adapter__form=4, adapter__slices=16), c.call)})
    assert t["chosen"] <= 1.6 * min(t.values()), t
