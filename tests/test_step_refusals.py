"""What the calls of a decode step refuse (jl_kv_write_dev, jl_kv_read_dev, jl_attend_dev, jl_sample_dev), without a GPU: a context bound to no
device.  Every check of arguments comes before the device, so a refused call says so here; one that passes them fails with the device."""
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


CACHE = dict(t=quant.F16, n_kv=2, d=64, page_size=16, n_page=9, k=P, v=P, table=P, n_seq=3, table_pages=4)
CACHES = [
    ({}, None),
    (dict(t=quant.BF16), None),
    (dict(t=quant.I8, k_scale=P, v_scale=P), None),
    (dict(d=256, page_size=1 << 20), None),
    (dict(row_stride=128, head_stride=64, page_stride=4096), None),
    (dict(table_stride=7), None),
    (dict(n_kv=0), "cache"),
    (dict(d=0), "cache"),
    (dict(page_size=0), "cache"),
    (dict(n_page=0), "cache"),
    (dict(n_seq=0), "cache"),
    (dict(table_pages=-1), "cache"),
    (dict(k=0), "null cache"),
    (dict(v=0), "null cache"),
    (dict(table=0), "null cache"),
    (dict(t=quant.I8), "scales"),
    (dict(t=quant.I8, k_scale=P), "scales"),
    (dict(table_stride=3), "table_stride"),
    (dict(row_stride=48), "stride"),
    (dict(head_stride=32), "stride"),
    (dict(page_stride=16), "stride"),
    (dict(t=quant.F32), False),
    (dict(t=quant.Q8_0), False),
    (dict(d=72), False),
    (dict(d=272), False),
    (dict(page_size=8), False),
    (dict(page_size=48), False),
    (dict(page_size=1 << 30), False),              # four of them are 2^32 positions
    (dict(row_stride=72), False),
    (dict(page_stride=4100), False),
    (dict(k=P + 8), False),
    (dict(table=P + 2), False),
    (dict(t=quant.I8, k_scale=P + 4, v_scale=P), False),
]
ROWS = dict(k=P, v=P, type=quant.F32, pos=P, ntok=3)
ATTEND = dict(out=P, q=P, n_head=8, len=P, ntok=3, scale=0.125)


@pytest.mark.parametrize("change, what", CACHES)
def test_cache_refusals(nodev, change, what):
    c = nodev.kv_cache(**{**CACHE, **change})
    _says(lambda: nodev.kv_write_dev(c, **ROWS), what)
    _says(lambda: nodev.kv_read_dev(c, **ROWS), what)
    _says(lambda: nodev.attend_dev(c, **ATTEND), what)


@pytest.mark.parametrize("change, what", [
    ({}, None),
    (dict(k=None), None),
    (dict(v=None, seq=P, type=quant.BF16), None),
    (dict(k=P + 4, k_stride=129), None),
    (dict(k=None, v=None), "bad operand"),
    (dict(pos=0), "bad operand"),
    (dict(ntok=0), "bad operand"),
    (dict(ntok=-3), "bad operand"),
    (dict(k_stride=127), "stride"),
    (dict(v_stride=1), "stride"),
    (dict(type=quant.Q4_K), False),
    (dict(type=quant.I8), False),
    (dict(k=P + 2), False),
    (dict(v=P + 1, type=quant.F16), False),
    (dict(pos=P + 2), False),
    (dict(seq=P + 1), False),
    (dict(ntok=(1 << 31) - 1), False),             # more threads than a launch has
])
def test_row_refusals(nodev, change, what):
    c = nodev.kv_cache(**CACHE)
    _says(lambda: nodev.kv_write_dev(c, **{**ROWS, **change}), what)
    _says(lambda: nodev.kv_read_dev(c, **{**ROWS, **change}), what)


@pytest.mark.parametrize("change, what", [
    ({}, None),
    (dict(seq=P, window=5, softcap=30.0, sink=P, lse=P, q_type=quant.F16, out_type=quant.BF16), None),
    (dict(n_head=2), None),
    (dict(n_head=256), None),
    (dict(out=P + 4), None),
    (dict(out_stride=513), None),
    (dict(q=0), "bad operand"),
    (dict(out=0), "bad operand"),
    (dict(len=0), "bad operand"),
    (dict(ntok=0), "bad operand"),
    (dict(n_head=0), "bad operand"),
    (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"),
    (dict(softcap=-1.0), "softcap"),
    (dict(softcap=float("inf")), "softcap"),
    (dict(window=-1), "window"),
    (dict(q_stride=511), "stride"),
    (dict(out_stride=64), "stride"),
    (dict(n_head=9), False),
    (dict(q_type=quant.Q8_0), False),
    (dict(out_type=quant.I8), False),
    (dict(q=P + 4), False),
    (dict(q_stride=514), False),
    (dict(q_stride=516, q_type=quant.F16), False),
    (dict(out=P + 2), False),
    (dict(len=P + 2), False),
    (dict(lse=P + 1), False),
])
def test_attend_refusals(nodev, change, what):
    c = nodev.kv_cache(**CACHE)
    _says(lambda: nodev.attend_dev(c, **{**ATTEND, **change}), what)


def test_a_cache_is_a_cache(nodev):
    for other in (None, 7, b"x" * 200, nodev.packed_bank(P, P, P, 0, 1)):
        with pytest.raises(TypeError, match="kv_cache"):
            nodev.attend_dev(other, **ATTEND)
        with pytest.raises(TypeError, match="kv_cache"):
            nodev.kv_read_dev(other, **ROWS)


SAMPLE = dict(logits=P, rows=3, n=1000, u=P, token=P)


@pytest.mark.parametrize("change, what", [
    ({}, None),
    (dict(temperature=P, top_k=P, top_p=P, min_p=P, prob=P, type=quant.BF16, stride=1001), None),
    (dict(n=524288), None),
    (dict(logits=P + 4), None),
    (dict(logits=0), "bad operand"),
    (dict(u=0), "bad operand"),
    (dict(token=0), "bad operand"),
    (dict(rows=0), "bad operand"),
    (dict(n=0), "bad operand"),
    (dict(stride=999), "stride"),
    (dict(type=quant.Q6_K), False),
    (dict(n=524289), False),
    (dict(rows=(1 << 20) + 1), False),
    (dict(logits=P + 2), False),
    (dict(logits=P + 1, type=quant.F16), False),
    (dict(prob=P + 2), False),
    (dict(top_k=P + 1), False),
])
def test_sample_refusals(nodev, change, what):
    _says(lambda: nodev.sample_dev(**{**SAMPLE, **change}), what)


def test_reserve_refusals(nodev):
    _says(lambda: nodev.reserve_attend(128), None)
    _says(lambda: nodev.reserve_attend(0), "reserve attend")
    _says(lambda: nodev.reserve_sample(64), None)
    _says(lambda: nodev.reserve_sample(0), "reserve sample")
