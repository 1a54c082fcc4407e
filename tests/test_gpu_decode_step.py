"""A decode step through its calls, one after the other on one stream: the projections of q, k and v, the rows' norm, the new rows into the cache, attention
over it, the output's projection, the head, and a token of each row.  Every call against the plain statement of it over what the call before left -- the cache
and the token exactly, attention and the norm within their own tests' bars, the projections against the oracle by NMSE 1e-10 -- in a prompt's step, in steps run
eagerly, and in the same steps captured once and replayed."""
import numpy as np
import pytest

import oracle
from conftest import nmse
from jitllm_amd import quant, synth
from jitllm_amd.hipmem import DeviceArray, Graph, Stream
from test_gpu_attend import check as check_attend, reference as attend_reference
from test_gpu_kv_cache import KINDS, Cache, table_of
from test_gpu_norm_rows import check_y, reference as norm_reference
from test_gpu_sample import reference as sample_reference

pytestmark = pytest.mark.gpu
T, WINDOW = quant.Q8_0, 32


class Step:
    """The buffers of `rows` tokens' step over a cache, its calls and its check."""

    def __init__(self, dev, c, rows, weights, e, n_head, n_vocab, window, cap):
        self.dev, self.c, self.rows, self.e, self.nh, self.nv, self.win, self.cap = dev, c, rows, e, n_head, n_vocab, window, cap
        self.w = weights
        f = lambda *s: DeviceArray(np.zeros(s, np.float32))
        u = lambda: DeviceArray(np.zeros(rows, np.uint32))
        self.x, self.y = f(rows, e), f(rows, e)
        self.q, self.k, self.v = f(rows, n_head, c.d), f(rows, c.n_kv, c.d), f(rows, c.n_kv, c.d)
        self.a, self.lse, self.h, self.logits, self.u, self.prob = f(rows, n_head, c.d), f(rows, n_head), f(rows, e), f(rows, n_vocab), f(rows), f(rows)
        self.seq, self.pos, self.len, self.token = u(), u(), u(), u()
        self.temp, self.k_of, self.p_of = DeviceArray(np.full(rows, 0.8, np.float32)), DeviceArray(np.full(rows, 40, np.uint32)), DeviceArray(np.full(rows, 0.95, np.float32))
        self.cache = c.handle(dev)

    def calls(self, s):
        d, c, n, w = self.dev, self.c, self.rows, self.w
        kv, nq = c.n_kv * c.d, self.nh * c.d
        assert d.norm_rows_dev(self.x.ptr, n, self.e, w["norm"][1].ptr, 1e-5, y=self.y.ptr, stream=s)
        for out, name, m in ((self.q, "q", nq), (self.k, "k", kv), (self.v, "v", kv)):
            assert d.matmul_dev(out.ptr, T, w[name][1].ptr, self.y.ptr, m, self.e, n, stream=s)
        assert d.kv_write_dev(self.cache, self.k.ptr, self.v.ptr, quant.F32, self.pos.ptr, n, seq=self.seq.ptr, stream=s)
        assert d.attend_dev(self.cache, self.a.ptr, self.q.ptr, self.nh, self.len.ptr, n, 0.125, seq=self.seq.ptr, window=self.win, softcap=self.cap, lse=self.lse.ptr, stream=s)
        assert d.matmul_dev(self.h.ptr, T, w["o"][1].ptr, self.a.ptr, self.e, nq, n, stream=s)
        assert d.matmul_dev(self.logits.ptr, T, w["head"][1].ptr, self.h.ptr, self.nv, self.e, n, stream=s)
        assert d.sample_dev(self.logits.ptr, n, self.nv, self.u.ptr, self.token.ptr, temperature=self.temp.ptr, top_k=self.k_of.ptr, top_p=self.p_of.ptr, prob=self.prob.ptr,
                            stream=s)

    def put(self, x, seq, pos, u):
        self.x.put(x); self.u.put(u.astype(np.float32))
        self.seq.put(np.array(seq, np.uint32)); self.pos.put(np.array(pos, np.uint32)); self.len.put(np.array(pos, np.uint32) + 1)

    def check(self, x, seq, pos, u):
        c, n, w = self.c, self.rows, self.w
        y = self.y.get()
        check_y(y, norm_reference(x, None, 1.0, w["norm"][0], 1e-5)[1], quant.F32)
        q, k, v, a, h, logits = (b.get() for b in (self.q, self.k, self.v, self.a, self.h, self.logits))
        for got, name, src in ((q, "q", y), (k, "k", y), (v, "v", y), (h, "o", a), (logits, "head", h)):
            src = np.ascontiguousarray(src.reshape(n, -1))
            got = got.reshape(n, -1)
            assert nmse(got, oracle.matmul_q8act_f64(T, w[name][0], src, got.shape[1], src.shape[1], n, WINDOW).reshape(n, -1)) <= 1e-10, name
        c.write(k, v, seq, pos)
        c.check()
        check_attend(a.astype(np.float64), self.lse.get().astype(np.float64), attend_reference(c, q, seq, np.array(pos) + 1, 0.125, self.win, self.cap), quant.F32)
        token, prob = self.token.get(), self.prob.get()
        for r in range(n):
            want = sample_reference(logits[r], u[r].astype(np.float32), 0.8, 40, float(np.float32(0.95)))
            assert token[r] == want[0] and abs(prob[r] - want[1]) <= want[1] * (2.0 ** -24 + self.nv * 2.0 ** -44) + 2.0 ** -43
        return token


@pytest.mark.parametrize("t", KINDS)
@pytest.mark.parametrize("window, cap", [(0, 0.0), (24, 30.0)])
def test_prompt_and_steps(dev, t, window, cap):
    rng = np.random.default_rng(window + t)
    e, n_head, n_kv, d, n_vocab, lens = 256, 8, 2, 64, 1003, [50, 21, 1]
    table, n_page = table_of(rng, [n + 12 for n in lens], 16)
    c = Cache(t, n_kv, d, 16, table, n_page)
    raw = {name: synth.quantized_weights(T, m, k, seed=m + i) for i, (name, m, k) in
           enumerate((("q", n_head * d, e), ("k", n_kv * d, e), ("v", n_kv * d, e), ("o", e, n_head * d), ("head", n_vocab, e)))}
    raw["norm"] = (1 + rng.standard_normal(e) / 10).astype(np.float32)
    weights = {k: (v, DeviceArray(v)) for k, v in raw.items()}
    embed = rng.standard_normal((n_vocab, e)).astype(np.float32)
    st = Stream()
    try:
        # the prompts, all tokens of the three at once
        seq, pos = np.repeat(range(3), lens), np.concatenate([np.arange(n) for n in lens])
        first = Step(dev, c, len(seq), weights, e, n_head, n_vocab, window, cap)
        x, u = embed[rng.integers(0, n_vocab, len(seq))], rng.random(len(seq))
        first.put(x, seq, pos, u)
        first.calls(st.handle)
        st.synchronize()
        token = first.check(x, seq, pos, u)[np.cumsum(lens) - 1]
        # a token of each, step after step
        step = Step(dev, c, 3, weights, e, n_head, n_vocab, window, cap)
        with Graph.capture(st.handle) as g:
            step.calls(st.handle)
        for i in range(8):
            x, u, pos = embed[token], rng.random(3), [n + i for n in lens]
            step.put(x, range(3), pos, u)
            if i % 3 == 1:
                step.calls(st.handle)
            else:
                g.launch()
            st.synchronize()
            token = step.check(x, range(3), pos, u)
    finally:
        st.destroy()
