"""Sampling (jl_sample_dev) where a row's values and settings are both at an end of their range, against the definition."""
import numpy as np
import pytest

from jitllm_amd import quant
from test_gpu_sample import check, logits, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("settings", [dict(), dict(top_k=2), dict(top_k=40), dict(top_p=0.5), dict(min_p=0.3), dict(top_k=5, top_p=0.9, min_p=0.1)], ids=str)
@pytest.mark.parametrize("n", [70, 5001])
def test_infinities_at_an_infinite_temperature(dev, n, settings):
    """An infinity is larger than the rest at every temperature and shares with its equals: of three, by thirds (of two where the first two are asked for or reach the half)."""
    rng = np.random.default_rng(n)
    at = [5, 33, n - 2]
    u = np.array([0.0, 0.2, 0.4, 0.6, 0.9, 0.9999999], np.float32)
    x = logits(rng, len(u), n)
    x[:, at] = np.inf
    for temperature in (np.inf, 3e38, 1.0, 1e-45):
        token, prob = run(dev, x, quant.F32, u, temperature=np.float32(temperature), **settings)
        share = 2 if settings.get("top_k") == 2 or settings.get("top_p") == 0.5 else 3
        assert list(token) == [at[min(int(v * share), share - 1)] for v in u.astype(np.float64)], temperature
        assert np.array_equal(prob, np.full(len(u), np.float32(1.0 / share)))


@pytest.mark.parametrize("settings", [dict(), dict(top_k=7), dict(top_p=0.6), dict(top_p=0.9), dict(min_p=0.3), dict(top_k=30, top_p=0.8), dict(top_p=0.7, min_p=0.05)], ids=str)
@pytest.mark.parametrize("n", [70, 5001])
@pytest.mark.parametrize("temperature", [1e38, 3e38, np.inf])
def test_distances_beyond_the_type(dev, n, temperature, settings):
    """Values at both ends of f32 and a temperature as large: the distance of two is no f32 number, its part of the temperature is a few."""
    rng = np.random.default_rng(n + 1)
    x = (3.3e38 * rng.uniform(-1, 1, (6, n))).astype(np.float32)
    x[:, :2] = [3.3e38, -3.3e38]
    check(dev, x, quant.F32, rng.random(6).astype(np.float32), temperature=np.float32(temperature), **settings)


@pytest.mark.parametrize("settings", [dict(), dict(top_k=6), dict(top_k=70), dict(top_k=700), dict(top_p=0.4), dict(top_p=0.4, min_p=0.2), dict(top_k=90, min_p=1.0),
                                      dict(top_k=90, top_p=0.7, min_p=0.2)], ids=str)
@pytest.mark.parametrize("many", [63, 64, 65, 480, 1024, 1025, 3000])
def test_infinities_by_the_hundred(dev, many, settings):
    """As many equals at the top as a list holds, or fewer or more, which are infinities, or the largest f32, or ones."""
    rng = np.random.default_rng(many)
    x = logits(rng, 6, 5001)
    for r, top in enumerate((np.inf, np.inf, 3.4e38, 3.4e38, 30.0, 30.0)):
        x[r, rng.permutation(5001)[:many]] = top
    check(dev, x, quant.F32, rng.random(6).astype(np.float32), **settings)
