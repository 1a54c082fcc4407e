"""Expert selection (jl_moe_select_dev) at the ends of f32's range, against the f64 statement of it in test_gpu_moe_select: the
difference to a row's largest logit, and the sum of a group's two best choices, where f32 no longer holds them."""
import numpy as np
import pytest

from test_gpu_moe_select import check, form  # noqa: F401

pytestmark = pytest.mark.gpu

LOWEST = np.finfo(np.float32).min


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("n", [2, 5, 64, 70, 128, 200, 384, 1000])
def test_softmax_of_large_logits(dev, form, n, renorm):  # noqa: F811
    """Rows whose largest logit is 2^34 and more in magnitude, where f32 steps are longer than the exponential's range."""
    rng = np.random.default_rng(n)
    rows = []
    for m in (2.0 ** 33, 2.0 ** 34, 2e10, 1e11, 1e20, 3e38):
        for sign in (1, -1):
            rows.append(sign * m * rng.random(n))                                  # all apart
            row = np.zeros(n)
            row[n - 1] = sign * m                                                  # one beside zeros
            rows.append(row)
            row = np.full(n, -m)
            row[rng.permutation(n)[: max(1, n // 3)]] = sign * m / 2                # two values
            rows.append(row)
    rows += [np.full(n, LOWEST), np.full(n, -2e10), np.full(n, 3e38)]              # one value: 1 / n each, and nothing for lanes without an expert
    row = np.full(n, -np.inf)
    row[n // 2:] = LOWEST                                                          # a finite mask over what is in service
    rows.append(row)
    row = np.full(n, LOWEST)
    row[n // 2] = -1e30                                                            # a mask beside a lower one
    rows.append(row)
    with np.errstate(over="ignore"):
        check(dev, np.array(rows).astype(np.float32), min(8, n), renorm=renorm, scale=1.5)


@pytest.mark.parametrize("rows", [1, 3, 20000])
def test_softmax_of_large_logits_by_rows(dev, form, rows):  # noqa: F811
    """The router's own form of a row of two: the larger logit, not the first."""
    logits = np.tile(np.float32([0.0, 2e10]), (rows, 1))
    check(dev, logits, 1)
    check(dev, logits, 2, renorm=False)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("n, n_group, k_group, k", [(16, 4, 2, 6), (256, 8, 4, 8), (256, 8, 8, 16), (63, 7, 3, 9), (160, 8, 3, 16), (384, 4, 2, 8), (1000, 10, 4, 16)])
def test_groups_whose_two_best_pass_the_range(dev, form, n, n_group, k_group, k, score):  # noqa: F811
    """The sum of a group's two best choices is -infinity where a bias is the type's lowest value: such a group is the last that is kept,
    its experts can still be taken.  Sums of +infinity are the first, the lowest of them."""
    rng = np.random.default_rng(n + k_group)
    logits, size = rng.standard_normal((7, n)).astype(np.float32), n // n_group
    low = np.zeros((4, n_group, size), np.float32)
    low[0] = LOWEST                                         # every group
    low[1, 1:] = LOWEST                                     # all but the first
    low[2, : n_group - 1] = LOWEST                          # all but the last
    low[2, 0] = -np.inf                                     # (and the first out of service)
    low[3, n_group // 2:] = -LOWEST
    low[3, 0] = LOWEST
    with np.errstate(over="ignore"):
        for bias in low.reshape(4, n):
            check(dev, logits, k, score=score, bias=bias, n_group=n_group, k_group=k_group, top=2, scale=0.5)
            check(dev, logits, k, score=score, bias=bias, n_group=n_group, k_group=k_group, top=1, renorm=False)
