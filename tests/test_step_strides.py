"""Orders of a cache's pages, heads and places by their strides, without a GPU: what shares no elements passes every check of arguments (and fails with the missing
device), what does is refused."""
import pytest

from jitllm_amd import quant
from test_step_refusals import ATTEND, CACHE, P, ROWS, _says, nodev  # noqa: F401

D, KV, S, N = 64, 4, 16, 9


@pytest.mark.parametrize("order", ["page head place", "page place head", "head page place", "head place page", "place page head", "place head page"])
@pytest.mark.parametrize("gap", [0, 16])
@pytest.mark.parametrize("t", [quant.F16, quant.I8])
def test_every_order(nodev, order, gap, t):  # noqa: F811
    """Back to back in any order, rows with a gap behind them or not; an element less in the outer or the middle stride and rows overlap."""
    stride, at = {}, D + gap
    for dim in reversed(order.split()):
        stride[dim] = at
        at *= dict(page=N, head=KV, place=S)[dim]
    make = lambda **s: nodev.kv_cache(**{**CACHE, "t": t, "n_kv": KV, "n_page": N, "d": D, "k_scale": P, "v_scale": P, "page_size": S, "page_stride": s["page"],
                                         "head_stride": s["head"], "row_stride": s["place"]})
    _every = lambda c, what: [_says(lambda: f(c, **kw), what) for f, kw in ((nodev.kv_write_dev, ROWS), (nodev.kv_read_dev, ROWS), (nodev.attend_dev, ATTEND))]
    _every(make(**stride), None)
    outer, middle, _ = order.split()
    for dim in (outer, middle):
        _every(make(**{**stride, dim: stride[dim] - gap - 16}), "overlap|shorter")


@pytest.mark.parametrize("strides, what", [
    (dict(row_stride=KV * D, head_stride=D), None),                        # the order of the header's example: pages behind one another
    (dict(row_stride=KV * D + 32, head_stride=D), None),
    (dict(row_stride=D, head_stride=D), "overlap"),
    (dict(row_stride=D, head_stride=D * S - 16), "overlap"),
    (dict(row_stride=KV * D - 16, head_stride=D), "overlap"),
    (dict(row_stride=KV * D, head_stride=D, page_stride=KV * D), "overlap"),
    (dict(page_stride=KV * S * D - 16), "overlap"),
    (dict(page_stride=(1 << 63) + 16), None),
    (dict(row_stride=3 * D, head_stride=2 * D), "overlap"),
    (dict(n_kv=1, head_stride=D), None),                                   # one head: its stride is met by nothing
    (dict(n_page=1, page_stride=D), None),
    (dict(n_kv=1, n_page=1, head_stride=D, page_stride=D, row_stride=D), None),
])
def test_strides(nodev, strides, what):  # noqa: F811
    c = nodev.kv_cache(**{**CACHE, "n_kv": KV, "n_page": N, "d": D, "page_size": S, **strides})
    _says(lambda: nodev.kv_write_dev(c, **ROWS), what)
    _says(lambda: nodev.attend_dev(c, **ATTEND), what)
