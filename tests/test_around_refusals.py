"""What the calls around the projections refuse (jl_norm_rows_dev, jl_moe_select_dev, jl_adapter_group_dev), without a GPU: a
context bound to no device.  Every check of arguments comes before the device, so a refused call says so here; one that passes
them fails with the device."""
import pytest

from jitllm_amd import quant
from jitllm_amd.device import Device, DeviceError

P = 4096     # an aligned address nobody reads


@pytest.fixture(scope="module")
def nodev():
    d = Device(device=-1)
    yield d
    d.close()


def _says(call, what):
    """None: the arguments pass and the device is missing; False: declined; else a text of the error."""
    if what is False:
        assert call() is False
        return
    with pytest.raises(DeviceError, match="hipSetDevice|SetDevice" if what is None else what):
        call()


NORM = dict(x=P, rows=3, n=64, w=P, eps=1e-5, y=P)


@pytest.mark.parametrize("change, what", [
    ({}, None),
    (dict(w=None), None),
    (dict(resid=P, resid_out=P), None),
    (dict(q=P, a_s=P, sum16=P), None),
    (dict(n=65536), None),
    (dict(n=63), None),
    (dict(x=P + 4), None),                        # an element at a time
    (dict(x=P + 2, x_type=quant.BF16), None),
    (dict(rows=0), "bad operand"),
    (dict(rows=-1), "bad operand"),
    (dict(n=0), "bad operand"),
    (dict(x=0), "bad operand"),
    (dict(y=None), "no output"),
    (dict(resid_out=P), "without resid"),
    (dict(q=P), "come together"),
    (dict(a_s=P, sum16=P), "come together"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(x_stride=63), "stride"),
    (dict(y_stride=32), "stride"),
    (dict(resid=P, resid_stride=1), "stride"),
    (dict(x_type=quant.Q8_0), False),
    (dict(y_type=2), False),
    (dict(n=65540), False),
    (dict(x=P + 1), False),
    (dict(x=P + 2), False),
    (dict(w=P + 2), False),
    (dict(y=P + 1, y_type=quant.F16), False),
    (dict(n=48, q=P, a_s=P, sum16=P), False),     # not whole blocks of 32
    (dict(q=P + 4, a_s=P, sum16=P), False),
    (dict(rows=(1 << 31) - 1, n=2048), False),    # more threads than a launch has
])
def test_norm_rows_refusals(nodev, change, what):
    _says(lambda: nodev.norm_rows_dev(**{**NORM, **change}), what)


SELECT = dict(logits=P, rows=3, n_expert=64, k_used=4, sel=P, sel_stride=4, wt=P)


@pytest.mark.parametrize("change, what", [
    ({}, None),
    (dict(bias=P, score=1, n_group=8, k_group=2, group_top=2), None),
    (dict(k_used=16, sel_stride=16, n_group=4, k_group=1, group_top=1), None),
    (dict(n_expert=1024), None),
    (dict(n_group=0), None),
    (dict(rows=0), "bad operand"),
    (dict(n_expert=0), "bad operand"),
    (dict(k_used=0), "bad operand"),
    (dict(sel_stride=3), "bad operand"),
    (dict(logits=0), "bad operand"),
    (dict(wt=0), "bad operand"),
    (dict(scale=float("inf")), "scale"),
    (dict(n_group=-1), "groups"),
    (dict(n_group=4, k_group=0), "groups"),
    (dict(n_group=4, k_group=5), "groups"),
    (dict(score=2), False),
    (dict(n_expert=1025), False),
    (dict(k_used=17, sel_stride=17), False),
    (dict(n_expert=3), False),                    # fewer experts than are used
    (dict(n_group=3, k_group=2), False),          # no divisor
    (dict(n_expert=130, n_group=65, k_group=65), False),
    (dict(n_group=4, k_group=2, group_top=3), False),
    (dict(n_group=32, k_group=1, group_top=1), False),   # a group of two, four wanted
    (dict(logits=P + 2), False),
    (dict(rows=(1 << 31) - 1), False),
])
def test_moe_select_refusals(nodev, change, what):
    _says(lambda: nodev.moe_select_dev(**{**SELECT, **change}), what)


ADAPT = dict(outs=[P], bases=[P], rows=[40], a=[P], b=[P], t=quant.F16, n_adapter=2, rank=8, x=P, k=64, ids=P, ntok=3)


@pytest.mark.parametrize("change, what", [
    ({}, None),
    (dict(bases=None), None),
    (dict(bases=[None], scale=P, ranks=P, x_type=quant.BF16, t=quant.F32), None),
    (dict(outs=[P] * 4, bases=[P] * 4, rows=[1, 2, 3, 4], a=[P] * 4, b=[P] * 4), None),
    (dict(outs=[], bases=[], rows=[], a=[], b=[]), "bad group"),
    (dict(rank=0), "bad group"),
    (dict(n_adapter=0), "bad group"),
    (dict(ntok=0), "bad group"),
    (dict(k=0), "bad group"),
    (dict(x=0), "bad group"),
    (dict(ids=0), "bad group"),
    (dict(outs=[0]), "null operand"),
    (dict(a=[0]), "null operand"),
    (dict(rows=[0]), "no rows"),
    (dict(t=quant.Q4_K), False),
    (dict(x_type=quant.MXFP4), False),
    (dict(k=48), False),
    (dict(rank=513), False),
    (dict(n_adapter=8193), False),
    (dict(a=[P + 8]), False),
    (dict(x=P + 4), False),
    (dict(outs=[P + 2]), False),
    (dict(ids=P + 1), False),
    (dict(ntok=(1 << 31) - 1), False),
])
def test_adapter_group_refusals(nodev, change, what):
    _says(lambda: nodev.adapter_group_dev(**{**ADAPT, **change}), what)


def test_five_projections_are_no_group(nodev):
    with pytest.raises(IndexError):
        nodev.adapter_group_dev(**{**ADAPT, "outs": [P] * 5})


def test_reserve_adapters_refusals(nodev):
    _says(lambda: nodev.reserve_adapters(1, 1, 1), None)
    _says(lambda: nodev.reserve_adapters(0, 1, 1), "reserve adapters")
    _says(lambda: nodev.reserve_adapters(1, 5, 1), "reserve adapters")
