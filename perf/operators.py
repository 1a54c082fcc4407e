"""The operators that stand around a block's quantized projections, as cases to time and to check.

  norm      Device.norm_rows_dev: residual added, RMSNorm, the normed rows in f32 / f16 / bf16 or in the int8 form
            (values, a scale per 32, a sum per 16) that the quantized matvecs read
  route     Device.moe_select_dev: softmax or sigmoid scores of a mixture's logits, a bias for the selection, groups of
            experts, the k best, renormalised and scaled weights
  adapter   Device.adapter_group_dev: low-rank adapters of many requests beside the projections they share,
            out = base + scale[a] * B[a] (A[a] x), a = the token's adapter

With `own` false a pass computes the plain form in elementary torch operations, else it makes the framework's calls.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 30}      # ggml type numbers
EPS = torch.tensor(1e-5, dtype=torch.float32).item()      # as the call takes it


def listed():
    return [
        # the norm between two blocks of one decoded token: the launch is the whole of it
        dict(name="norm 1x4096", op="norm", rows=1, n=4096, x="f32", y="f32", resid=True, q8=False, window=32),
        # a small decode batch in front of an MXFP4 mixture, which reads bf16
        dict(name="norm 64x2880 bf16", op="norm", rows=64, n=2880, x="bf16", y="bf16", resid=True, q8=False, window=32),
        # a prompt quantized once for the k-quant projections that share it
        dict(name="norm q8 512x4096", op="norm", rows=512, n=4096, x="f32", y=None, resid=True, q8=True, window=256),
        # a batch of long prompts of a ragged length: memory alone
        dict(name="norm q8 4099x7168", op="norm", rows=4099, n=7168, x="f32", y="f32", resid=True, q8=True, window=32),
        # every head of a prompt normed by itself, no residual
        dict(name="norm heads 40003x128", op="norm", rows=40003, n=128, x="f32", y="f32", resid=False, q8=False, window=32),
        # one decoded token of a mixture with a balance bias and limited groups
        dict(name="route 1x256 groups", op="route", rows=1, n_expert=256, k=8, score="sigmoid", bias=True, groups=8, k_group=4, top=2,
             renorm=True, masked=0),
        # a prompt through a softmax router, some experts out of service
        dict(name="route 777x128 softmax", op="route", rows=777, n_expert=128, k=8, score="softmax", bias=True, groups=1, k_group=1,
             top=1, renorm=True, masked=5),
        # a large batch of prompts over many experts
        dict(name="route 16384x384", op="route", rows=16384, n_expert=384, k=8, score="sigmoid", bias=True, groups=1, k_group=1, top=1,
             renorm=True, masked=0),
        # one decoded token with its request's adapter on one projection
        dict(name="adapter 1 token r16", op="adapter", ntok=1, k=4096, rows="4096", rank=16, n_adapter=8, type="f16", x="f32", requests=1,
             mixed=False),
        # a decode batch, every token its own request, beside query, key and value
        dict(name="adapter 64 tokens qkv", op="adapter", ntok=64, k=4096, rows="4096,1024,1024", rank=16, n_adapter=32, type="bf16",
             x="f32", requests=64, mixed=True),
        # prompts of five requests of ragged lengths, an odd rank, adapters kept in f32
        dict(name="adapter 333 tokens r20", op="adapter", ntok=333, k=2880, rows="2880", rank=20, n_adapter=4, type="f32", x="bf16",
             requests=5, mixed=False),
        # long prompts of a few requests beside gate and up
        dict(name="adapter 2048 tokens r64", op="adapter", ntok=2048, k=4096, rows="14336,14336", rank=64, n_adapter=3, type="bf16",
             x="f32", requests=4, mixed=False),
    ]


# -- drawn cases ---------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "route", "adapter"])
    if op == "norm":
        q8 = rng.random() < 0.5
        n = _log(rng, 2, 256) * 32 if q8 else _log(rng, 48, 8192)
        rows = max(1, min(_log(rng, 1, 40000), 4099 * 7168 // n))
        y = rng.choice(["f32", "f16", "bf16"]) if not q8 or rng.random() < 0.3 else None
        return dict(op=op, rows=rows, n=n, x=rng.choice(["f32", "f32", "bf16", "f16"]), y=y, resid=rng.random() < 0.8, q8=q8,
                    window=rng.choice([32, 256]))
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        n = groups * _log(rng, 4, 512 // groups)
        k = min(rng.choice([1, 2, 4, 6, 8, 10]), max(1, n // 4))
        rows = max(1, min(_log(rng, 1, 16384), 16384 * 384 // n))
        bias = rng.random() < 0.7
        return dict(op=op, rows=rows, n_expert=n, k=k, score=rng.choice(["sigmoid", "softmax"]), bias=bias, groups=groups,
                    k_group=max(1, groups // 2), top=rng.choice([1, 2]) if groups > 1 else 1, renorm=rng.random() < 0.8,
                    masked=rng.randint(0, n // 16) if bias else 0)
    k, rank = _log(rng, 16, 256) * 32, _log(rng, 3, 96)
    rows = [_log(rng, 500, 14336) for _ in range(rng.choice([1, 1, 2, 3]))]
    rows = rows if sum(rows) <= 28672 else rows[:1]
    ntok = _log(rng, 1, 2048)
    n_adapter = max(1, min(_log(rng, 1, 64), 30_000_000 // (rank * (len(rows) * k + sum(rows)))))
    ntok = max(1, min(ntok, 2048 * 64 * 36864 // (rank * (len(rows) * k + sum(rows)))))
    return dict(op=op, ntok=ntok, k=k, rows=",".join(map(str, rows)), rank=rank, n_adapter=n_adapter,
                type=rng.choice(["f16", "bf16", "f32"]), x=rng.choice(["f32", "f32", "bf16"]),
                requests=ntok if ntok < 100 or rng.random() < 0.3 else rng.randint(1, 12), mixed=rng.random() < 0.3)


# -- inputs --------------------------------------------------------------------

_program = {}


def _device(window=32):
    """The program's one stream and its one device context a window, kept for its whole run."""
    if "stream" not in _program:
        _program["stream"] = torch.cuda.Stream()
        torch.cuda.synchronize()
    torch.cuda.set_stream(_program["stream"])
    if not own:
        return None
    if window not in _program:
        from jitllm_amd.device import Device
        _program[window] = Device(device=0, act_window=window)
    return _program[window]


def _inputs(case, seed):
    """The case's tensors, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    s = {}
    if case["op"] == "norm":
        rows, n = case["rows"], case["n"]
        s["x"] = normal(rows, n).to(DTYPES[case["x"]])
        s["w"] = 1 + 0.1 * normal(n)
        s["resid"] = 3 * normal(rows, n) if case["resid"] else None
    elif case["op"] == "route":
        n = case["n_expert"]
        s["logits"], s["bias"] = normal(case["rows"], n), None
        if case["bias"]:
            s["bias"] = 0.05 * normal(n)
            if case["masked"]:
                s["bias"][torch.randperm(n, generator=g, device="cuda")[: case["masked"]]] = -math.inf
    else:
        k, rank, na, ntok, t = case["k"], case["rank"], case["n_adapter"], case["ntok"], DTYPES[case["type"]]
        rows = [int(r) for r in case["rows"].split(",")]
        s["x"] = normal(ntok, k).to(DTYPES[case["x"]])
        s["a"] = [(normal(na, rank, k) / math.sqrt(k)).to(t) for _ in rows]
        s["b"] = [(normal(na, r, rank) / math.sqrt(rank)).to(t) for r in rows]
        s["base"] = [normal(ntok, r) for r in rows]
        s["scale"] = 0.5 + torch.rand(na, generator=g, device="cuda")
        # request i carries adapter i modulo (n_adapter + 1), the last of them none; prompts are runs of tokens, a decode
        # batch (a token a request) comes in any order
        req = case["requests"]
        if req == ntok:
            of = torch.randperm(ntok, generator=g, device="cuda")
        else:
            cut = torch.randperm(ntok - 1, generator=g, device="cuda")[: req - 1] + 1
            of = torch.zeros(ntok, dtype=torch.int64, device="cuda")
            of[cut] = 1
            of = of.cumsum(0)
        s["ids"] = (of % (na + 1)).to(torch.int32)
        s["ranks"] = None
        if case["mixed"]:
            s["ranks"] = torch.randint(1, rank + 1, (na,), generator=g, device="cuda", dtype=torch.int32)
    return s


def prepare(case, seed):
    dev = _device(case.get("window", 32))
    s = _inputs(case, seed)
    s["case"], s["op"], s["dev"], s["stream"] = case, case["op"], dev, _program["stream"].cuda_stream
    # where a program has the results put
    if case["op"] == "norm":
        rows, n = case["rows"], case["n"]
        s["h"] = torch.empty(rows, n, device="cuda") if case["resid"] else None
        s["y"] = torch.empty(rows, n, device="cuda", dtype=DTYPES[case["y"]]) if case["y"] else None
        if case["q8"]:
            s["q"] = torch.empty(rows, n, device="cuda", dtype=torch.int8)
            s["as"], s["sum16"] = torch.empty(rows, n // 32, device="cuda"), torch.empty(rows, n // 16, device="cuda")
    elif case["op"] == "route":
        s["sel"] = torch.empty(case["rows"], case["k"], device="cuda", dtype=torch.int32)
        s["wt"] = torch.empty(case["rows"], case["k"], device="cuda")
    else:
        s["out"] = [torch.empty_like(b) for b in s["base"]]
        s["rows"] = [b.shape[1] for b in s["base"]]
        s["ptrs"] = [[t.data_ptr() for t in s[n]] for n in ("out", "base", "a", "b")]
    torch.cuda.synchronize()
    return s


# -- the plain forms -------------------------------------------------------------

def _plain_norm(c, s):
    h = s["resid"] + s["x"].float() if c["resid"] else s["x"].float()
    # in 64 bits: a value next to a border of the 8-bit steps has to fall on the same side
    d = h.double()
    inv = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)
    y = (d * s["w"].double() * inv).float()
    out = [h if c["resid"] else None, y.to(DTYPES[c["y"]]) if c["y"] else None]
    if c["q8"]:
        rows, n, win = c["rows"], c["n"], c["window"]
        pad = -n % win
        amax = torch.nn.functional.pad(y.abs(), (0, pad)).view(rows, -1, win).amax(-1)
        step = amax / torch.full_like(amax, 127.0)      # (by a number, torch multiplies by its reciprocal)
        inv = torch.where(step != 0, 1.0 / step, torch.zeros_like(step))
        of = torch.arange(n, device="cuda") // win
        v = y * inv[:, of]
        q = torch.trunc(v + torch.copysign(torch.full_like(v, 0.5 - 2.0 ** -25), v))    # half away from zero
        scales = step[:, of[::32]]
        out += [q * step[:, of], scales.contiguous(), q.view(rows, -1, 16).sum(-1)]
    return out


def _plain_route(c, s):
    n, rows = c["n_expert"], c["rows"]
    l64 = s["logits"].double()
    # in 64 bits and rounded once: neighbouring scores decide the order
    if c["score"] == "softmax":
        e = torch.exp(l64 - l64.amax(-1, keepdim=True))
        score = (e / e.sum(-1, keepdim=True)).float()
    else:
        score = (1.0 / (1.0 + torch.exp(-l64))).float()
    choice = score + s["bias"] if c["bias"] else score
    if c["groups"] > 1:
        size = n // c["groups"]
        best = choice.view(rows, c["groups"], size).sort(dim=-1, descending=True).values[..., : min(c["top"], size)]
        of = torch.where(best == -math.inf, torch.zeros_like(best), best).sum(-1)
        of = torch.where(best[..., 0] == -math.inf, best[..., 0], of)
        kept = of.sort(dim=-1, descending=True, stable=True).indices[:, : c["k_group"]]
        keep = torch.zeros(rows, c["groups"], dtype=torch.bool, device="cuda").scatter_(1, kept, True)
        choice = torch.where(keep.repeat_interleave(size, 1), choice, torch.full_like(choice, -math.inf))
    top = choice.sort(dim=-1, descending=True, stable=True)
    sel, got = top.indices[:, : c["k"]], top.values[:, : c["k"]] > -math.inf
    w = torch.where(got, score.gather(1, sel), torch.zeros_like(top.values[:, : c["k"]]))
    if c["renorm"]:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    return [torch.where(got, sel, torch.full_like(sel, n)).to(torch.int32), w * 2.5]


def _plain_adapter(c, s):
    # every token against every adapter, its own adapter's part kept: two products a projection
    na, rank, ntok = c["n_adapter"], c["rank"], c["ntok"]
    on = s["ids"].long().unsqueeze(1) == torch.arange(na, device="cuda")                       # [ntok][na]
    on = on.unsqueeze(-1).expand(ntok, na, rank)
    if s["ranks"] is not None:
        on = on & (torch.arange(rank, device="cuda") < s["ranks"].unsqueeze(1))
    x, gain = s["x"].float(), s["scale"].view(1, na, 1)

    def one(a, b, base):
        t = (x @ a.float().view(na * rank, -1).t()).view(ntok, na, rank)
        t = torch.where(on, t * gain, torch.zeros_like(t)).view(ntok, na * rank)
        return base + t @ b.float().transpose(0, 1).reshape(-1, na * rank).t()

    return [one(*p) for p in zip(s["a"], s["b"], s["base"])]


# -- a pass ----------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _served(ok):
    if not ok:
        raise RuntimeError("declined")


def run(s):
    c, op, dev = s["case"], s["op"], s["dev"]
    if op == "norm":
        if not own:
            return _plain_norm(c, s)
        q8 = dict(q=s["q"].data_ptr(), a_s=s["as"].data_ptr(), sum16=s["sum16"].data_ptr()) if c["q8"] else {}
        _served(dev.norm_rows_dev(s["x"].data_ptr(), c["rows"], c["n"], s["w"].data_ptr(), EPS, x_type=CODES[c["x"]],
                                  resid=_ptr(s["resid"]), resid_out=_ptr(s["h"]), y=_ptr(s["y"]),
                                  y_type=CODES[c["y"] or "f32"], stream=s["stream"], **q8))
        if not c["q8"]:
            return [s["h"], s["y"]]
        # the int8 values as what they stand for
        return [s["h"], s["y"], (s["q"].view(c["rows"], -1, 32) * s["as"].unsqueeze(-1)).view(c["rows"], -1), s["as"], s["sum16"]]
    if op == "route":
        if not own:
            return _plain_route(c, s)
        _served(dev.moe_select_dev(s["logits"].data_ptr(), c["rows"], c["n_expert"], c["k"], s["sel"].data_ptr(), c["k"],
                                   s["wt"].data_ptr(), score=1 if c["score"] == "sigmoid" else 0, bias=_ptr(s["bias"]),
                                   n_group=c["groups"], k_group=c["k_group"], group_top=c["top"], renorm=c["renorm"], scale=2.5,
                                   stream=s["stream"]))
        return [s["sel"], s["wt"]]
    if not own:
        return _plain_adapter(c, s)
    out, base, a, b = s["ptrs"]
    _served(dev.adapter_group_dev(out, base, s["rows"], a, b, CODES[c["type"]], c["n_adapter"], c["rank"], s["x"].data_ptr(), c["k"],
                                  s["ids"].data_ptr(), c["ntok"], scale=s["scale"].data_ptr(), ranks=_ptr(s["ranks"]),
                                  x_type=CODES[c["x"]], stream=s["stream"]))
    return s["out"]


# -- the same from the definitions, in 64 bits -------------------------------------

def exact(case, seed):
    _device()
    s, c = _inputs(case, seed), case
    if c["op"] == "norm":
        rows, n = c["rows"], c["n"]
        h = s["x"].double()
        if c["resid"]:
            h = h + s["resid"].double()
        hf = h.float().double()                        # the residual is kept in 32 bits, and normed as kept
        rms = (hf.square().sum(1) / n + EPS).sqrt()
        y = hf / rms.unsqueeze(1) * s["w"].double()
        out = [h if c["resid"] else None, y if c["y"] else None]
        if c["q8"]:
            # the quantizer is defined on 32-bit values and 32-bit quotients
            yf, win, nw = y.float(), c["window"], -(-n // c["window"])
            full = torch.zeros(rows, nw * win, device="cuda")
            full[:, :n] = yf
            parts = full.view(rows, nw, win)
            step = (parts.abs().max(-1, keepdim=True).values.double() / 127.0).float()
            v = (parts * torch.where(step > 0, step.double().reciprocal().float(), step)).double()
            q = torch.sign(v) * torch.floor(v.abs() + 0.5)
            vals = (q * step.double()).view(rows, -1)[:, :n]
            scales = step.expand(rows, nw, win // 32).reshape(rows, -1)[:, : n // 32]
            out += [vals, scales.double(), q.view(rows, -1)[:, :n].unflatten(1, (n // 16, 16)).sum(-1)]
        return out
    if c["op"] == "route":
        n, rows, k = c["n_expert"], c["rows"], c["k"]
        l64 = s["logits"].double()
        p = torch.sigmoid(l64) if c["score"] == "sigmoid" else torch.softmax(l64, -1)
        score = p.float()                               # the order goes by 32-bit scores
        choice = score if s["bias"] is None else score + s["bias"]
        dead = torch.isinf(choice)
        if c["groups"] > 1:
            size = n // c["groups"]
            v = choice.view(rows, c["groups"], size)
            first = v.max(-1)
            total = first.values.clone()
            if c["top"] == 2 and size > 1:
                rest = v.scatter(-1, first.indices.unsqueeze(-1), -math.inf).max(-1).values
                total = total + torch.where(torch.isinf(rest), torch.zeros_like(rest), rest)
            rank_of = (total.unsqueeze(1) > total.unsqueeze(2)).sum(-1)                  # groups strictly better
            order = torch.arange(c["groups"], device="cuda")
            tied = (total.unsqueeze(1) == total.unsqueeze(2)) & (order < order.unsqueeze(1))
            keep = rank_of + tied.sum(-1) < c["k_group"]
            dead = dead | ~keep.repeat_interleave(size, 1)
        live = torch.where(dead, torch.full_like(choice, -math.inf), choice)
        sel = torch.empty(rows, k, dtype=torch.int64, device="cuda")
        w = torch.zeros(rows, k, dtype=torch.float64, device="cuda")
        at = torch.arange(n, device="cuda").expand(rows, n)
        for j in range(k):
            best = live.max(-1, keepdim=True).values
            i = torch.where(live == best, at, n).min(-1, keepdim=True).values
            none = best == -math.inf
            sel[:, j] = torch.where(none, n, i).squeeze(1)
            i = i.clamp(max=n - 1)
            w[:, j] = torch.where(none, 0.0, p.gather(1, i)).squeeze(1)
            live = live.scatter(1, i, -math.inf)
        if c["renorm"]:
            w = w / (w.sum(-1, keepdim=True) + 1e-20)
        return [sel.to(torch.int32), w * 2.5]
    outs = []
    for a, b, base in zip(s["a"], s["b"], s["base"]):
        o = base.double()
        for i in range(c["n_adapter"]):
            of = (s["ids"] == i).nonzero().squeeze(1)
            r = c["rank"] if s["ranks"] is None else int(s["ranks"][i])
            if of.numel():
                t = s["x"][of].double() @ a[i, :r].double().t().contiguous()
                o[of] += s["scale"][i].double() * (t @ b[i, :, :r].double().t().contiguous())
        outs.append(o)
    return outs


# -- what a pass cannot do without ----------------------------------------------

_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def work(case):
    c = case
    if c["op"] == "norm":
        per = _SIZE[c["x"]] + (8 if c["resid"] else 0) + (_SIZE[c["y"]] if c["y"] else 0) + (1 + 4 / 32 + 4 / 16 if c["q8"] else 0)
        return {"bytes": c["rows"] * c["n"] * per + 4 * c["n"], "flops": c["rows"] * c["n"] * (12 if c["q8"] else 6)}
    if c["op"] == "route":
        return {"bytes": c["rows"] * (4 * c["n_expert"] + 8 * c["k"]) + (4 * c["n_expert"] if c["bias"] else 0),
                "flops": c["rows"] * c["n_expert"] * 12}
    rows = [int(r) for r in c["rows"].split(",")]
    na, req, ntok = c["n_adapter"], c["requests"], c["ntok"]
    used = min(req, na)
    share = 1 - (req // (na + 1)) / req                  # of the requests, those that carry an adapter
    rank = c["rank"] * (0.5 if c["mixed"] else 1)        # ranks from 1 up to it, on average
    weights = used * rank * (len(rows) * c["k"] + sum(rows)) * _SIZE[c["type"]]
    return {"bytes": weights + ntok * c["k"] * _SIZE[c["x"]] + 8 * ntok * sum(rows) + 4 * ntok,
            "flops": 2 * share * ntok * rank * (len(rows) * c["k"] + sum(rows))}
