"""Tuning of the calls of a decode step, without a GPU: a value that names no form is refused where it is set, since a call could take none of them."""
import pytest

from jitllm_amd import quant
from jitllm_amd.device import DeviceError
from test_step_refusals import ATTEND, CACHE, P, _says, nodev  # noqa: F401


@pytest.mark.parametrize("form", [2, 3, 5, 16, -1, 1 << 30])
def test_forms_that_are_none(nodev, form):  # noqa: F811
    for before in (0, 1, 4, 8):
        nodev.set_tuning(attend__form=before)
        with pytest.raises(DeviceError, match="attend.form"):
            nodev.set_tuning(attend__form=form)
    nodev.set_tuning(attend__form=0)


@pytest.mark.parametrize("form", [0, 1, 4, 8])
@pytest.mark.parametrize("whole", [0, 1, 2, 3, -1])
@pytest.mark.parametrize("ntok", [1, 3, 16, 3000])
def test_every_form_serves_every_call(nodev, form, whole, ntok):  # noqa: F811
    """Up to the device, which is missing here: few and many tokens, heads that share a key head by the dozen or not at all."""
    nodev.set_tuning(attend__form=form, attend__whole=whole)
    try:
        for n_head in (2, 8, 34, 200):
            for t in (quant.F16, quant.I8):
                c = nodev.kv_cache(**{**CACHE, "t": t, "k_scale": P, "v_scale": P})
                _says(lambda: nodev.attend_dev(c, **{**ATTEND, "seq": P, "ntok": ntok, "n_head": n_head}), None)
    finally:
        nodev.set_tuning(attend__form=0, attend__whole=0)
