"""How many bits attention over a paged cache (jl_attend_dev) keeps, over a call as a whole: the distance of its results from the definition in 64 bits, in the 2-norm.

The bars of test_gpu_attend hold element by element, every rounding at its worst; over hundreds of positions they are wide.  Roundings are independent, so over a call they
add up in quadrature.  With u = 2^-24 (half a step of f32), d the width, n the positions, X the largest |score| and S the largest scale * sqrt(sum q^2 k^2):
    a score: d partial sums of no more than X + S or so, rounded once each; q in pieces, two of f16 leaving 2^-22 of each element; some factors
        sqrt(d) u (X + S) + 2^-22 S + 4 u X
    a weight: its argument and the exponential (2 X + 4) u, and its pieces: p = 2^-22 (two of f16), 2^-16 (two of bf16), 2^-24 (three)
    the sums of n weights: sqrt(n) u
and values of either sign add the weights' errors as they add the weights, so that the whole is off by that part of itself; once more for the denominator:
    |out - want| <= 2 (u (sqrt(d) (X + S) + 6 X + 4 + sqrt(n)) + 2^-22 S + p) |want|, and 2^-11 / sqrt(3) |want| where out is f16 (a step's uniform error).
That is 1e-5 to 4e-5 in f32, where a lost piece of q or of the weights is 2e-4 (f16) or 1e-3 (bf16)."""
import numpy as np
import pytest

from jitllm_amd import quant
from test_gpu_attend import reference, run
from test_gpu_attend_edges import causal, way  # noqa: F401
from test_gpu_kv_cache import KINDS, Cache, table_of
from test_gpu_norm_rows import stored, values

pytestmark = pytest.mark.gpu


def bar(c, q, scale, n, pieces, ot):
    d = q.shape[-1]
    k = c.k.astype(np.float64) * c.ks[..., None] if c.t == quant.I8 else values(c.k, c.t)
    k = k.transpose(1, 0, 2, 3).reshape(c.n_kv, -1, d)                                      # every row of the pool
    qh = q.astype(np.float64).reshape(len(q), c.n_kv, -1, d).transpose(1, 0, 2, 3).reshape(c.n_kv, -1, d)
    x = max(np.abs(a @ b.T).max() for a, b in zip(qh, k)) * scale
    s = np.sqrt(max(((a * a) @ (b * b).T).max() for a, b in zip(qh, k))) * scale
    u = 2.0 ** -24
    out = 2 * (u * (np.sqrt(d) * (x + s) + 6 * x + 4 + np.sqrt(n)) + 2.0 ** -22 * s + pieces)
    return out + (2.0 ** -11 / np.sqrt(3) if ot == quant.F16 else 0)


@pytest.mark.parametrize("t, qt, ot", [(quant.F16, quant.F32, quant.F32), (quant.F16, quant.F16, quant.F32), (quant.I8, quant.F32, quant.F32), (quant.I8, quant.BF16, quant.F32),
                                       (quant.BF16, quant.F32, quant.F32), (quant.BF16, quant.BF16, quant.F32), (quant.BF16, quant.BF16, quant.F16)])
@pytest.mark.parametrize("per, group, d, lens", [(1, 4, 64, [1100, 4000]), (1, 8, 128, [3000]), (1, 2, 256, [1500, 900]), (4, 2, 256, [1000, 1300]), (20, 4, 64, [1000, 1700]),
                                                 (48, 2, 128, [1048, 700]), (33, 1, 256, [1033])])
def test_bits_kept(dev, way, t, qt, ot, per, group, d, lens):  # noqa: F811
    rng = np.random.default_rng(d + per)
    table, n_page = table_of(rng, lens, 16)
    c = Cache(t, 2, d, 16, table, n_page)
    seq, length = causal(lens, per)
    q = values(stored(rng.standard_normal((len(seq), 2 * group, d)).astype(np.float32), qt), qt)
    scale = float(np.float32(1 / np.sqrt(d)))
    got, _ = run(dev, c, q, qt, ot, seq, length, scale)
    want = reference(c, q, seq, length, scale)[0]
    pieces = 2.0 ** -22 if t != quant.BF16 else 2.0 ** -16 if qt == quant.BF16 and ot != quant.F32 else 2.0 ** -24
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    most = bar(c, q, scale, max(lens), pieces, ot)
    assert off <= most, (off, most)
