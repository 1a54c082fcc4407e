"""What stands between a block's projections and behind the last one, as cases to time and to check.

  cache     Device.kv_write_dev / kv_read_dev: rows of keys and values into the pages of a cache (f16, bf16, or int8 with a scale a
            row) and back
  attend    Device.attend_dev: attention of new tokens over such a cache, one token a sequence, a few, or a prompt; windows, soft
            caps, sinks
  sample    Device.sample_dev: a token a row of logits by temperature, top-k, top-p and min-p, from a given random number

With `own` false a pass computes the plain form in elementary torch operations, else it makes the framework's calls.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
CODES = {"f32": 0, "f16": 1, "bf16": 30, "i8": 24}      # ggml type numbers


def listed():
    return [
        # one decoded token's keys and values: the launch is the whole of it
        dict(name="write 1 token f16", op="cache", way="write", ntok=1, n_kv=8, d=128, type="f16", x="f32", to="f32", page=16, nseq=1),
        # a prompt of ragged length quantized into the pages of three requests, and read back for a prefix to be moved
        dict(name="write, read 8191 i8", op="cache", way="both", ntok=8191, n_kv=8, d=128, type="i8", x="f32", to="bf16", page=16, nseq=3),
        # long prefixes read back in full, heads of an uncommon width
        dict(name="read 50001 bf16", op="cache", way="read", ntok=50001, n_kv=4, d=96, type="bf16", x="f32", to="f32", page=64, nseq=7),
        # the first tokens of a single conversation: latency
        dict(name="attend 1 x 777", op="attend", nseq=1, per=1, length=777, n_kv=8, group=4, d=128, type="f16", q="f32", out="f32", page=16,
             window=0, cap=0.0, sinks=False, lse=False),
        # a decode batch of ragged lengths over an int8 cache
        dict(name="attend 64 x 8192 i8", op="attend", nseq=64, per=1, length=8192, n_kv=8, group=4, d=128, type="i8", q="f32", out="f32",
             page=16, window=0, cap=0.0, sinks=False, lse=False),
        # one long document, a token at a time
        dict(name="attend 1 x 131071 bf16", op="attend", nseq=1, per=1, length=131071, n_kv=8, group=8, d=128, type="bf16", q="bf16",
             out="bf16", page=64, window=0, cap=0.0, sinks=False, lse=False),
        # sliding windows with sinks in front of an MXFP4 block, which reads bf16: most of the cache is out of sight
        dict(name="attend 32 window sinks", op="attend", nseq=32, per=1, length=4096, n_kv=8, group=8, d=64, type="bf16", q="f32", out="bf16",
             page=32, window=128, cap=0.0, sinks=True, lse=False),
        # five drafted tokens a request checked at once, wide heads, capped scores
        dict(name="attend 8 x 5 drafted", op="attend", nseq=8, per=5, length=3001, n_kv=4, group=2, d=256, type="f16", q="f32", out="f32",
             page=32, window=0, cap=50.0, sinks=False, lse=True),
        # prompts of three requests behind prefixes that are there already
        dict(name="attend 3 x 683 prompt", op="attend", nseq=3, per=683, length=2048, n_kv=8, group=4, d=128, type="bf16", q="bf16",
             out="bf16", page=16, window=0, cap=0.0, sinks=False, lse=False),
        # one conversation's next token with the usual filters
        dict(name="sample 1 x 131072", op="sample", rows=1, n=131072, type="f32", temp=0.8, k=40, p=0.95, min_p=0.0, mixed=False),
        # a batch of requests, each with settings of its own, some of them greedy
        dict(name="sample 64 x 32000 mixed", op="sample", rows=64, n=32000, type="f32", temp=0.7, k=50, p=0.9, min_p=0.05, mixed=True),
        # a large batch over a large vocabulary of odd length, nothing but a nucleus
        dict(name="sample 256 x 200003", op="sample", rows=256, n=200003, type="f32", temp=1.0, k=0, p=0.95, min_p=0.0, mixed=False),
    ]


# -- drawn cases ---------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["cache", "attend", "attend", "sample"])
    if op == "cache":
        n_kv, d = _log(rng, 1, 16), rng.choice([64, 80, 96, 128, 192, 256])
        t = rng.choice(["f16", "bf16", "i8", "i8"])
        ntok = min(_log(rng, 1, 50000), 50001 * 4 * 96 // (n_kv * d))
        return dict(op=op, way=rng.choice(["both", "read"] if t == "i8" else ["write", "both", "read"]), ntok=ntok, n_kv=n_kv, d=d,
                    type=t, x=rng.choice(["f32", "f32", "bf16", "f16"]), to=rng.choice(["f32", "bf16", "f16"]),
                    page=rng.choice([16, 32, 64, 256]), nseq=min(ntok, rng.randint(1, 9)))
    if op == "attend":
        n_kv, group, d = rng.choice([1, 2, 4, 8, 8, 16]), rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16]), rng.choice([64, 80, 96, 128, 128, 192, 256])
        nseq, per, length = _log(rng, 1, 64), 1, _log(rng, 1, 131071)
        kind = rng.random()
        if kind < 0.2:
            per = rng.randint(2, 8)
        elif kind < 0.4:
            nseq, per = rng.randint(1, 4), _log(rng, 9, 700)
        length = max(per, min(length, 131071 * 8 * 128 // (nseq * n_kv * d), 3 * 683 * 2048 * 32 * 128 // (nseq * per * n_kv * group * d)))
        return dict(op=op, nseq=nseq, per=per, length=length, n_kv=n_kv, group=group, d=d, type=rng.choice(["f16", "bf16", "i8"]),
                    q=rng.choice(["f32", "f32", "bf16", "f16"]), out=rng.choice(["f32", "bf16", "f16"]), page=rng.choice([16, 32, 64, 256]),
                    window=_log(rng, 1, length) if rng.random() < 0.25 else 0, cap=rng.choice([0.0, 0.0, 0.0, 30.0]),
                    sinks=rng.random() < 0.25, lse=rng.random() < 0.3)
    n = _log(rng, 500, 262144)
    rows = max(1, min(_log(rng, 1, 256), 256 * 200003 // n))
    return dict(op=op, rows=rows, n=n, type=rng.choice(["f32", "f32", "bf16", "f16"]), temp=round(rng.uniform(0.2, 1.5), 3),
                k=rng.choice([0, 1, _log(rng, 2, 1000)]), p=rng.choice([1.0, round(rng.uniform(0.1, 0.999), 3)]),
                min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.3), 4)]), mixed=rng.random() < 0.4)


# -- inputs --------------------------------------------------------------------

_program = {}


def _device():
    """The program's one stream and its one device context, kept for its whole run."""
    if "stream" not in _program:
        _program["stream"] = torch.cuda.Stream()
        torch.cuda.synchronize()
    torch.cuda.set_stream(_program["stream"])
    if own and "device" not in _program:
        from jitllm_amd.device import Device
        _program["device"] = Device(device=0, act_window=32)
    return _program.get("device")


def _lengths(case):
    """Positions of each sequence: evenly spaced, the first the longest."""
    if case["op"] == "cache":
        n, k = case["ntok"], case["nseq"]
        return [n // k + (i < n % k) for i in range(k)]
    top, per, k = case["length"], case["per"], case["nseq"]
    return [top - (top - per) * i // k for i in range(k)]


def _inputs(case, seed):
    """The case's tensors, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32)

    s = {}
    if case["op"] == "sample":
        rows, n = case["rows"], case["n"]
        x = 2 * normal(rows, n)
        x.scatter_add_(1, torch.randint(0, n, (rows, 16), generator=g, device="cuda"), 10 * rand(rows, 16))    # a few that stand out
        s["x"], s["u"] = x.to(DTYPES[case["type"]]), rand(rows)
        full = lambda v, t: torch.full((rows,), v, device="cuda", dtype=t)
        s["temp"], s["p"], s["min_p"] = full(case["temp"], torch.float32), full(case["p"], torch.float32), full(case["min_p"], torch.float32)
        s["k"] = full(case["k"], torch.int32)
        if case["mixed"]:      # requests with settings of their own: the filters on and off, every fourth greedy
            on = lambda: torch.rand(rows, generator=g, device="cuda") < 0.5
            s["p"] = torch.where(on(), s["p"], torch.ones_like(s["p"]))
            s["min_p"] = torch.where(on(), s["min_p"], torch.zeros_like(s["min_p"]))
            s["k"] = torch.where(on(), s["k"], torch.zeros_like(s["k"]))
            s["temp"] = torch.where(torch.arange(rows, device="cuda") % 4 == 3, torch.zeros_like(s["temp"]), s["temp"] * (0.5 + rand(rows)))
        return s
    n_kv, d, page, lens = case["n_kv"], case["d"], case["page"], _lengths(case)
    s["lens"] = lens
    need = [-(-n // page) for n in lens]
    n_page = sum(need) + 1                      # one page more than is used
    order = torch.randperm(n_page, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(need), device="cuda", dtype=torch.int32)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k]
        at += k
    s["table"], s["n_page"] = table, n_page
    # what the pages hold already
    shape = (n_page, n_kv, page, d)
    if case["type"] == "i8":
        for name in ("k", "v"):
            s[name] = (40 * normal(*shape)).clamp(-127, 127).round().to(torch.int8)
            s[name + "_scale"] = 0.02 + 0.02 * rand(n_page, n_kv, page)
    else:
        for name in ("k", "v"):
            s[name] = normal(*shape).to(DTYPES[case["type"]])
            s[name + "_scale"] = None
    if case["op"] == "cache":
        ntok = case["ntok"]
        mix = torch.randperm(ntok, generator=g, device="cuda")         # tokens in any order
        s["seq"] = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), torch.tensor(lens, device="cuda"))[mix].to(torch.int32)
        s["pos"] = torch.cat([torch.arange(n, device="cuda") for n in lens])[mix].to(torch.int32)
        for name in ("xk", "xv"):
            s[name] = (normal(ntok, n_kv, d) * (0.5 + rand(1, n_kv, d))).to(DTYPES[case["x"]])
        return s
    nseq, per = case["nseq"], case["per"]
    ntok = nseq * per
    s["q"] = (2 * normal(ntok, n_kv * case["group"], d)).to(DTYPES[case["q"]])
    s["seq"] = torch.arange(nseq, device="cuda").repeat_interleave(per).to(torch.int32)
    j = torch.arange(per, device="cuda")
    s["len"] = (torch.tensor(lens, device="cuda").unsqueeze(1) - per + 1 + j).reshape(-1).to(torch.int32)      # causal among themselves
    s["sink"] = normal(n_kv * case["group"]) if case["sinks"] else None
    return s


def prepare(case, seed):
    dev = _device()
    s = _inputs(case, seed)
    s["case"], s["dev"], s["stream"] = case, dev, _program["stream"].cuda_stream
    # where a program has the results put
    if case["op"] == "sample":
        s["token"] = torch.empty(case["rows"], device="cuda", dtype=torch.int32)
        s["prob"] = torch.empty(case["rows"], device="cuda")
    elif case["op"] == "cache":
        for name in ("yk", "yv"):
            s[name] = torch.empty(case["ntok"], case["n_kv"], case["d"], device="cuda", dtype=DTYPES[case["to"]])
    else:
        s["out"] = torch.empty(s["q"].shape, device="cuda", dtype=DTYPES[case["out"]])
        s["lse"] = torch.empty(s["q"].shape[:2], device="cuda") if case["lse"] else None
    if own and case["op"] != "sample":
        s["cache"] = dev.kv_cache(CODES[case["type"]], case["n_kv"], case["d"], case["page"], s["n_page"], s["k"].data_ptr(), s["v"].data_ptr(),
                                  s["table"].data_ptr(), s["table"].shape[0], s["table"].shape[1], k_scale=_ptr(s["k_scale"]),
                                  v_scale=_ptr(s["v_scale"]))
    torch.cuda.synchronize()
    return s


# -- the plain forms -------------------------------------------------------------

def _quantized(x):
    """int8 rows and their scales: the step is the quotient by 127, halves away from zero."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    step = amax / torch.full_like(amax, 127.0)          # (by a number, torch multiplies by its reciprocal)
    inv = torch.where(step != 0, 1.0 / step, torch.zeros_like(step))
    v = x * inv
    return torch.trunc(v + torch.copysign(torch.full_like(v, 0.5 - 2.0 ** -25), v)).to(torch.int8), step.squeeze(-1)


def _plain_cache(c, s):
    pos, seq = s["pos"].long(), s["seq"].long()
    page, slot = s["table"][seq, pos // c["page"]].long(), pos % c["page"]

    def put(x, pool, scale):
        if scale is None:
            pool[page, :, slot] = x.to(pool.dtype)
        else:
            pool[page, :, slot], scale[page, :, slot] = _quantized(x)

    def get(pool, scale):
        x = pool[page, :, slot].float()
        if scale is not None:
            x = x * scale[page, :, slot].unsqueeze(-1)
        return x.to(DTYPES[c["to"]])

    if c["way"] != "read":
        put(s["xk"], s["k"], s["k_scale"])
        put(s["xv"], s["v"], s["v_scale"])
    if c["way"] == "write":
        return [s["k"], s["v"]]
    return [get(s["k"], s["k_scale"]), get(s["v"], s["v_scale"]), s["k_scale"], s["v_scale"]]


def _plain_attend(c, s):
    nseq, per, n_kv, group, d, top = c["nseq"], c["per"], c["n_kv"], c["group"], c["d"], c["length"]
    pages = s["table"].long()

    def rows(pool, scale):      # [nseq][n_kv][positions][d], all sequences as long as the longest
        x = pool[pages].transpose(1, 2).reshape(nseq, n_kv, -1, d)[:, :, :top].float()
        return x if scale is None else x * scale[pages].transpose(1, 2).reshape(nseq, n_kv, -1)[:, :, :top].unsqueeze(-1)

    q = s["q"].float().view(nseq, per, n_kv, group, d).permute(0, 2, 1, 3, 4).reshape(nseq, n_kv, per * group, d)
    score = q @ rows(s["k"], s["k_scale"]).transpose(2, 3).contiguous() * (1.0 / math.sqrt(d))
    if c["cap"]:
        score = torch.tanh(score / c["cap"]) * c["cap"]
    at, n = torch.arange(top, device="cuda"), s["len"].view(nseq, 1, per, 1, 1)
    seen = at < n
    if c["window"]:
        seen = seen & (at >= n - c["window"])
    score = score.view(nseq, n_kv, per, group, top).masked_fill(~seen, -math.inf)
    m = score.amax(-1, keepdim=True)
    if c["sinks"]:
        sink = s["sink"].view(n_kv, 1, group, 1)
        m = torch.maximum(m, sink)
    w = torch.exp(score - m)
    total = w.sum(-1, keepdim=True)
    if c["sinks"]:
        total = total + torch.exp(sink - m)
    out = w.view(nseq, n_kv, per * group, top) @ rows(s["v"], s["v_scale"])
    out = out.view(nseq, n_kv, per, group, d) / total
    lse = (m + torch.log(total)).permute(0, 2, 1, 3, 4).reshape(nseq * per, n_kv * group) if c["lse"] else None
    return [out.permute(0, 2, 1, 3, 4).reshape(nseq * per, n_kv * group, d).to(DTYPES[c["out"]]), lse]


def _plain_sample(c, s):
    rows, n = c["rows"], c["n"]
    # in 64 bits: a sum next to a border decides which token it is
    x, idx = s["x"].float().sort(dim=-1, descending=True, stable=True)
    temp = s["temp"].double().unsqueeze(1)
    first = torch.arange(n, device="cuda").unsqueeze(0)
    w = torch.where(temp > 0, torch.exp((x.double() - x[:, :1].double()) / temp), (first == 0).double())
    k = torch.where(s["k"] > 0, s["k"], torch.full_like(s["k"], n)).unsqueeze(1)
    w = torch.where(first < k, w, torch.zeros_like(w))
    sums = w.cumsum(-1)
    p = s["p"].double().unsqueeze(1)
    before = torch.where(p < 1, sums - w, torch.full_like(w, -1.0))
    keep = (first == 0) | ((first < k) & (before < p * sums[:, -1:]) & (w >= s["min_p"].double().unsqueeze(1)))
    w = torch.where(keep, w, torch.zeros_like(w))
    at = torch.zeros_like(w).scatter_(1, idx, w)           # in the vocabulary's order again
    sums = at.cumsum(-1)
    token = (sums <= s["u"].double().unsqueeze(1) * sums[:, -1:]).sum(-1, keepdim=True).clamp(max=n - 1)
    return [token.squeeze(1).to(torch.int32), (at.gather(1, token) / sums[:, -1:]).squeeze(1).float()]


# -- a pass ----------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _served(ok):
    if not ok:
        raise RuntimeError("declined")


def run(s):
    c, dev = s["case"], s["dev"]
    if c["op"] == "cache":
        if not own:
            return _plain_cache(c, s)
        if c["way"] != "read":
            _served(dev.kv_write_dev(s["cache"], s["xk"].data_ptr(), s["xv"].data_ptr(), CODES[c["x"]], s["pos"].data_ptr(), c["ntok"],
                                     seq=s["seq"].data_ptr(), stream=s["stream"]))
        if c["way"] == "write":
            return [s["k"], s["v"]]
        _served(dev.kv_read_dev(s["cache"], s["yk"].data_ptr(), s["yv"].data_ptr(), CODES[c["to"]], s["pos"].data_ptr(), c["ntok"],
                                seq=s["seq"].data_ptr(), stream=s["stream"]))
        return [s["yk"], s["yv"], s["k_scale"], s["v_scale"]]
    if c["op"] == "attend":
        if not own:
            return _plain_attend(c, s)
        _served(dev.attend_dev(s["cache"], s["out"].data_ptr(), s["q"].data_ptr(), c["n_kv"] * c["group"], s["len"].data_ptr(), s["len"].shape[0],
                               scale=1.0 / math.sqrt(c["d"]), seq=s["seq"].data_ptr(), q_type=CODES[c["q"]], out_type=CODES[c["out"]],
                               window=c["window"], softcap=c["cap"], sink=_ptr(s["sink"]), lse=_ptr(s["lse"]), stream=s["stream"]))
        return [s["out"], s["lse"]]
    if not own:
        return _plain_sample(c, s)
    _served(dev.sample_dev(s["x"].data_ptr(), c["rows"], c["n"], s["u"].data_ptr(), s["token"].data_ptr(), type=CODES[c["type"]],
                           temperature=s["temp"].data_ptr(), top_k=s["k"].data_ptr(), top_p=s["p"].data_ptr(), min_p=s["min_p"].data_ptr(),
                           prob=s["prob"].data_ptr(), stream=s["stream"]))
    return [s["token"], s["prob"]]


# -- the same from the definitions, in 64 bits -------------------------------------

def _rows_of(s, name, seq, n, page):
    """Rows 0 to n of sequence `seq` in 64 bits, [n_kv][n][d]."""
    used = s["table"][seq, : -(-n // page)].long()
    x = torch.cat([s[name][p] for p in used.tolist()], 1)[:, :n].double() if used.numel() < 64 else \
        s[name].index_select(0, used).permute(1, 0, 2, 3).flatten(1, 2)[:, :n].double()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"].index_select(0, used).permute(1, 0, 2).flatten(1)[:, :n, None].double()
    return x


def _exact_attend(c, s):
    d, group, n_kv, per = c["d"], c["group"], c["n_kv"], c["per"]
    out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    lse = torch.empty(s["q"].shape[:2], device="cuda", dtype=torch.float64)
    for i, n in enumerate(s["lens"]):
        k, v = _rows_of(s, "k", i, n, c["page"]), _rows_of(s, "v", i, n, c["page"])
        mine = slice(i * per, (i + 1) * per)
        end = s["len"][mine].long().unsqueeze(1)
        at = torch.arange(n, device="cuda").unsqueeze(0)
        hidden = (at >= end) | (at < end - c["window"]) if c["window"] else at >= end
        for h in range(n_kv * group):
            e = (s["q"][mine, h].double() @ k[h // group].t()) / math.sqrt(d)
            if c["cap"]:
                e = c["cap"] * torch.tanh(e / c["cap"])
            e = torch.where(hidden, -math.inf, e)
            if c["sinks"]:
                e = torch.cat([e, s["sink"][h].double().expand(per, 1)], 1)
            w = torch.softmax(e, -1)
            out[mine, h] = w[:, :n] @ v[h // group]
            lse[mine, h] = torch.logsumexp(e, -1)
    return [out, lse if c["lse"] else None]


def _exact_cache(c, s):
    if c["type"] == "i8" and c["way"] == "both":
        # the quantizer is defined on 32-bit values and 32-bit quotients
        def through(x):
            x = x.float()
            step = (x.abs().max(-1, keepdim=True).values.double() / 127.0).float()
            v = (x * torch.where(step > 0, step.double().reciprocal().float(), step)).double()
            return torch.sign(v) * torch.floor(v.abs() + 0.5) * step.double(), step.squeeze(-1).double()
        (yk, sk), (yv, sv) = through(s["xk"]), through(s["xv"])
    elif c["way"] == "read":
        yk, yv, sk, sv = torch.empty(s["xk"].shape, device="cuda", dtype=torch.float64), torch.empty(s["xk"].shape, device="cuda", dtype=torch.float64), None, None
        for i, n in enumerate(s["lens"]):
            mine = (s["seq"] == i).nonzero().squeeze(1)
            at = s["pos"][mine].long()
            yk[mine], yv[mine] = _rows_of(s, "k", i, n, c["page"]).permute(1, 0, 2)[at], _rows_of(s, "v", i, n, c["page"]).permute(1, 0, 2)[at]
        return [yk, yv, None if s["k_scale"] is None else s["k_scale"].double(), None if s["v_scale"] is None else s["v_scale"].double()]
    else:
        yk, yv, sk, sv = s["xk"].to(DTYPES[c["type"]]).double(), s["xv"].to(DTYPES[c["type"]]).double(), None, None
    if c["way"] == "both" and sk is None:
        return [yk, yv, None, None]
    pools = [s["k"].double(), s["v"].double()] if c["way"] == "write" else [s["k_scale"].double(), s["v_scale"].double()]
    flat = s["table"].long().flatten()[s["seq"].long() * s["table"].shape[1] + s["pos"].long() // c["page"]] * c["page"] + s["pos"].long() % c["page"]
    for pool, x in zip(pools, (yk, yv) if c["way"] == "write" else (sk, sv)):
        rows = pool.transpose(1, 2).reshape(-1, *((c["n_kv"], c["d"]) if c["way"] == "write" else (c["n_kv"],)))
        rows[flat] = x
        pool.copy_(rows.view(s["n_page"], c["page"], *rows.shape[1:]).transpose(1, 2))
    return pools if c["way"] == "write" else [yk, yv, *pools]


def _exact_sample(c, s):
    x0, n = s["x"].float().cpu().numpy(), c["n"]
    temp, k, p, low, u = (s[a].cpu().numpy() for a in ("temp", "k", "p", "min_p", "u"))
    token, prob = np.empty(c["rows"], np.int32), np.empty(c["rows"])
    for r in range(c["rows"]):
        x = x0[r].astype(np.float64)
        if not temp[r] > 0:
            token[r], prob[r] = x.argmax(), 1.0
            continue
        w = np.exp((x - x.max()) / np.float64(temp[r]))
        keep = k[r] if 0 < k[r] < n else n
        order = np.argpartition(-x, keep - 1)[:keep] if keep < n else np.arange(n)
        if keep < n:           # among equals at the border the lowest come first
            edge = x[order].min()
            above = np.flatnonzero(x > edge)
            order = np.concatenate([above, np.flatnonzero(x == edge)[: keep - above.size]])
        order = order[np.lexsort((order, -x[order]))]
        sums = np.cumsum(w[order])
        if p[r] < 1:
            order = order[: np.searchsorted(sums, np.float64(p[r]) * sums[-1], side="left") + 1]
        order = order[: max(1, int((w[order] >= np.float64(low[r])).sum()))]
        order.sort()
        sums = np.cumsum(w[order])
        at = min(int(np.searchsorted(sums, np.float64(u[r]) * sums[-1], side="right")), order.size - 1)
        token[r], prob[r] = order[at], w[order[at]] / sums[-1]
    return [torch.from_numpy(token), torch.from_numpy(prob)]


def exact(case, seed):
    _device()
    s = _inputs(case, seed)
    return {"cache": _exact_cache, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](case, s)


# -- what a pass cannot do without ----------------------------------------------

_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}


def work(case):
    c = case
    if c["op"] == "cache":
        rows = 2 * c["ntok"] * c["n_kv"]
        held = c["d"] * _SIZE[c["type"]] + (4 if c["type"] == "i8" else 0)
        per = (c["d"] * _SIZE[c["x"]] + held if c["way"] != "read" else 0) + (held + c["d"] * _SIZE[c["to"]] if c["way"] != "write" else 0)
        return {"bytes": rows * per + 8 * c["ntok"], "flops": rows * c["d"] * 4}
    if c["op"] == "attend":
        lens, per, d = _lengths(c), c["per"], c["d"]
        cut = lambda n: min(n, c["window"]) if c["window"] else n
        seen = sum(cut(n - per + 1 + j) for n in lens for j in range(per))
        rows = sum(min(n, c["window"] + per - 1) if c["window"] else n for n in lens) * c["n_kv"] * 2
        heads = c["n_kv"] * c["group"]
        return {"bytes": rows * (d * _SIZE[c["type"]] + (4 if c["type"] == "i8" else 0)) + c["nseq"] * per * heads * d * (_SIZE[c["q"]] + _SIZE[c["out"]]),
                "flops": 4.0 * d * heads * seen}
    return {"bytes": c["rows"] * c["n"] * _SIZE[c["type"]] + 28 * c["rows"], "flops": 8.0 * c["rows"] * c["n"]}
