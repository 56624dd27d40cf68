"""Measured cases of a state-space decoder's operators, from a prompt to scored tokens.

* ``causal_conv`` / ``causal_conv_step``: the short depthwise convolution before the scan, over packed prompts and for
  one new token per sequence, with the last inputs kept in a state pool.
* ``selective_scan`` / ``selective_scan_step``: h = exp(delta A) h + delta x B, y = (C h + D x) silu(z), with
  delta = softplus(dt + bias), over packed prompts and for one new token per sequence; f32 state pool.
* ``block_norm``: norm after a block, its gate and residual scale, the residual sum and the next block's norm.
* ``token_logprobs``: log probabilities of given tokens, the rows' entropies and the most likely alternatives.

``run`` computes the plain form in elementary 32-bit torch operations, or, with ``own``, calls ``air_rs.ops``.
"""
import math

import torch

own = False

SCAN_CHUNK = 32                     # tokens per block of the plain form of the scan
MOST_SCAN = 8192 * 8192 * 16        # tokens x channels x states of the largest listed scan
MOST_CONV = 16384 * 8192
MOST_NORM = 6007 * 4096
MOST_LOGITS = 2048 * 128256


# ---------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one long document through the convolution of an inner width of 8192
        {"name": "conv_16384x8192", "op": "conv", "tokens": 16384, "seqs": 1, "dim": 8192, "width": 4, "dtype": "bf16",
         "resume": False, "split": 0},
        # a continuous-batching prefill: ragged prompts packed together, some resuming, channels not a multiple of 8
        {"name": "conv_ragged", "op": "conv", "tokens": 4001, "seqs": 13, "dim": 2050, "width": 3, "dtype": "f32",
         "resume": True, "split": 1},
        # one user generating: latency of a layer's step
        {"name": "conv_step_1", "op": "conv_step", "rows": 1, "dim": 4096, "width": 4, "dtype": "bf16"},
        # a wide decode batch
        {"name": "conv_step_256", "op": "conv_step", "rows": 256, "dim": 8192, "width": 4, "dtype": "bf16"},
        # one long document at an inner width of 8192: few, long recurrences
        {"name": "scan_8192x8192", "op": "scan", "tokens": 8192, "seqs": 1, "dim": 8192, "states": 16, "groups": 1,
         "dtype": "bf16", "resume": False, "gate": True, "split": 0},
        # ragged prompts of a narrow model, some resuming from a cached state
        {"name": "scan_ragged", "op": "scan", "tokens": 6007, "seqs": 13, "dim": 1536, "states": 16, "groups": 1,
         "dtype": "bf16", "resume": True, "gate": True, "split": 1},
        # one user generating
        {"name": "scan_step_1", "op": "scan_step", "rows": 1, "dim": 4096, "states": 16, "groups": 1, "dtype": "bf16",
         "gate": True},
        # a full decode batch
        {"name": "scan_step_128", "op": "scan_step", "rows": 128, "dim": 8192, "states": 16, "groups": 1,
         "dtype": "bf16", "gate": True},
        # one decode row of an 8B-size residual stream: residual sum and the next norm
        {"name": "norm_1x4096", "op": "norm", "rows": 1, "dim": 4096, "dtype": "bf16", "post": False, "gate": "",
         "offset": 0.0, "scale": 1.0},
        # a prefill chunk with everything: norm after the block, gate, residual scale, norm before the next
        {"name": "norm_6007x4096", "op": "norm", "rows": 6007, "dim": 4096, "dtype": "bf16", "post": True,
         "gate": "silu", "offset": 1.0, "scale": 0.22},
        # a generated token's log probability with the most alternatives that an API request may ask for
        {"name": "logprobs_1x128256", "op": "logprobs", "rows": 1, "vocab": 128256, "dtype": "f32", "top": 20},
        # scoring a prompt of 2048 tokens
        {"name": "logprobs_2048x128256", "op": "logprobs", "rows": 2048, "vocab": 128256, "dtype": "bf16", "top": 5},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("conv", "conv_step", "scan", "scan", "scan_step", "norm", "logprobs", "logprobs"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if op in ("conv", "conv_step"):
        dim = _log_int(rng, 64, 12000)
        c = {"op": op, "dim": dim, "width": rng.choice((2, 3, 4, 4)), "dtype": dtype}
        if op == "conv_step":
            return {**c, "rows": _log_int(rng, 1, 400)}
        tokens = _log_int(rng, 1, min(20000, MOST_CONV // dim))
        return {**c, "tokens": tokens, "seqs": _log_int(rng, 1, max(1, min(48, tokens))), "resume": rng.random() < 0.5,
                "split": rng.randrange(1 << 16)}
    if op in ("scan", "scan_step"):
        groups = rng.choice((1, 1, 1, 2, 4))
        dim = groups * _log_int(rng, 32, 8192 // groups)
        states = rng.choice((16, 16, 16, 8, 24, 64))
        c = {"op": op, "dim": dim, "states": states, "groups": groups, "dtype": dtype, "gate": rng.random() < 0.7}
        if op == "scan_step":
            return {**c, "rows": _log_int(rng, 1, min(300, 128 * 8192 * 16 // (dim * states)))}
        tokens = _log_int(rng, 1, min(20000, MOST_SCAN // (dim * states)))
        return {**c, "tokens": tokens, "seqs": _log_int(rng, 1, max(1, min(48, tokens))), "resume": rng.random() < 0.5,
                "split": rng.randrange(1 << 16)}
    if op == "norm":
        dim = rng.choice((8, 1)) * _log_int(rng, 32, 2000)
        return {"op": op, "rows": _log_int(rng, 1, min(20000, MOST_NORM // dim)), "dim": dim, "dtype": dtype,
                "post": rng.random() < 0.5, "gate": rng.choice(("", "silu", "sigmoid")),
                "offset": rng.choice((0.0, 1.0)), "scale": rng.choice((1.0, 0.22))}
    vocab = _log_int(rng, 1000, 160000)
    return {"op": op, "rows": _log_int(rng, 1, MOST_LOGITS // vocab // (2 if dtype == "f32" else 1)), "vocab": vocab,
            "dtype": dtype, "top": rng.choice((0, 1, 5, 20))}


def _lengths(case):
    """Ragged lengths that sum to the case's tokens: cut points of a fixed multiplicative sequence."""
    t, n = case["tokens"], case["seqs"]
    cuts = sorted((1103515245 * (i + 1 + case["split"]) + 12345) % 2147483647 % (t + 1) for i in range(n - 1))
    edges = [0] + cuts + [t]
    return [b - a for a, b in zip(edges, edges[1:])]


# ---------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _batch(case, g, s):
    """Packed sequences (prompts) or one token per sequence (steps) and their state rows."""
    if "tokens" in case:
        lens = _lengths(case)
        edges = [0]
        for x in lens:
            edges.append(edges[-1] + x)
        n = len(lens)
        s["lens"], s["edges"] = lens, edges
        s["cu"] = torch.tensor(edges, dtype=torch.int32, device="cuda")
        s["has_state"] = (_rand(g, n) < (0.7 if case["resume"] else 0.0)).to(torch.int32)
    else:
        n = case["rows"]
    s["slots"] = torch.randperm(n + 3, generator=g, device="cuda")[:n].to(torch.int32)
    return case.get("tokens", case.get("rows")), n + 3


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] in ("conv", "conv_step"):
        t, slots = _batch(case, g, s)
        d, w, dt = case["dim"], case["width"], _dtype(case)
        # x is the first half of a fused projection's rows
        s["x"] = _randn(g, t, 2 * d).to(dt)[:, :d]
        s["w"] = _randn(g, d, w) * w ** -0.5
        s["bias"] = 0.1 * _randn(g, d)
        s["state"] = _randn(g, slots, w - 1, d).to(dt)
        return s
    if case["op"] in ("scan", "scan_step"):
        t, slots = _batch(case, g, s)
        d, n, gr, dt = case["dim"], case["states"], case["groups"], _dtype(case)
        s["x"] = torch.nn.functional.silu(_randn(g, t, d)).to(dt)
        s["dt"] = (0.7 * _randn(g, t, d)).to(dt)
        # one projection holds B and C side by side
        bc = _randn(g, t, 2, gr, n).to(dt)
        s["B"], s["C"] = bc[:, 0], bc[:, 1]
        # states forget within tokens to thousands of tokens: rates 1 .. n, steps of 0.001 to 0.1
        s["A"] = -torch.arange(1, n + 1, device="cuda") * torch.exp(0.2 * _randn(g, d, n))
        step = torch.exp(math.log(0.001) + _rand(g, d) * math.log(100.0))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
        s["D"] = 1.0 + 0.1 * _randn(g, d)
        s["z"] = _randn(g, t, 2 * d).to(dt)[:, d:] if case["gate"] else None
        s["state"] = 0.5 * _randn(g, slots, d, n)
        return s
    if case["op"] == "norm":
        n, d, dt = case["rows"], case["dim"], _dtype(case)
        x = 2.0 * _randn(g, n, d)
        x[:, 7] *= 30.0                   # residual streams have outlier channels
        s.update(resid=x, y=_randn(g, n, d).to(dt), w=1.0 + 0.2 * _randn(g, d) - case["offset"], eps=1e-5,
                 post=1.0 + 0.2 * _randn(g, d) - case["offset"] if case["post"] else None,
                 gate=_randn(g, n, d).to(dt) if case["gate"] else None, resid_out=torch.empty_like(x))
        return s
    n, v = case["rows"], case["vocab"]
    logits = 3.0 * _randn(g, n, v)
    # most rows have a clear favourite; every 16th row is under a grammar that allows a few tokens
    logits[torch.arange(n, device="cuda"), torch.randint(0, v, (n,), generator=g, device="cuda")] += 12.0
    few = torch.randint(0, v, (n, 3), generator=g, device="cuda")
    rows = torch.arange(n, device="cuda")[9::16]
    keep = logits[rows[:, None], few[rows]]
    logits[rows] = -math.inf
    logits[rows[:, None], few[rows]] = keep
    tokens = torch.randint(0, v, (n,), generator=g, device="cuda")
    likely = logits.argmax(-1)
    s["tokens"] = torch.where(_rand(g, n) < 0.5, likely, tokens).to(torch.int32)
    s["logits"] = logits.to(_dtype(case))
    return s


# ---------------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _own_conv(s):
    from air_rs import ops
    out = ops.causal_conv(s["x"], s["w"], s["bias"], state=s["state"], cu_seqlens=s["cu"], slots=s["slots"],
                          has_state=s["has_state"])
    return {"out": out, "state": s["state"]}


def _own_conv_step(s):
    from air_rs import ops
    out = ops.causal_conv_step(s["x"], s["w"], s["state"], s["bias"], slots=s["slots"])
    return {"out": out, "state": s["state"]}


def _own_scan(s):
    from air_rs import ops
    out = ops.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                             state=s["state"], cu_seqlens=s["cu"], slots=s["slots"], has_state=s["has_state"])
    return {"out": out, "state": s["state"]}


def _own_scan_step(s):
    from air_rs import ops
    out = ops.selective_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], D=s["D"], z=s["z"],
                                  dt_bias=s["dt_bias"], slots=s["slots"])
    return {"out": out, "state": s["state"]}


def _own_norm(s):
    from air_rs import ops
    c = s["case"]
    out, resid = ops.block_norm(s["y"], s["w"], s["eps"], residual=s["resid"], post_weight=s["post"], gate=s["gate"],
                                gate_act=c["gate"] or "silu", scale=c["scale"], w_offset=c["offset"],
                                resid_out=s["resid_out"])
    return {"out": out, "resid": resid}


def _own_logprobs(s):
    from air_rs import ops
    r = ops.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    if s["case"]["top"]:
        out.update(top_logprobs=r.top_logprobs, top_ids=r.top_ids)
    return out


_OWN = {"conv": _own_conv, "conv_step": _own_conv_step, "scan": _own_scan, "scan_step": _own_scan_step,
        "norm": _own_norm, "logprobs": _own_logprobs}


def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _plain_conv(s):
    """Every sequence behind its last inputs (or zeros), then the taps as shifted rows."""
    x, w, lens = s["x"].float(), s["w"], torch.tensor(s["lens"], device="cuda")
    h = w.shape[1] - 1
    n, t = len(s["lens"]), x.shape[0]
    seq = torch.repeat_interleave(torch.arange(n, device=x.device), lens, output_size=t)
    at = torch.arange(t, device=x.device) + h * (seq + 1)              # row of each token in the extended rows
    head = s["cu"][:-1].long() + h * torch.arange(n, device=x.device)
    ext = torch.empty(t + n * h, x.shape[1], device=x.device)
    ext[at] = x
    slots = s["slots"].long()
    before = s["state"][slots].float() * (s["has_state"] != 0)[:, None, None]
    j = torch.arange(h, device=x.device)
    ext[head[:, None] + j] = before
    y = s["bias"] + w[:, h] * x
    for i in range(h):
        y = y + w[:, i] * ext[at - h + i]
    s["state"][slots] = ext[(head + lens)[:, None] + j].to(s["state"].dtype)
    return {"out": _silu(y).to(s["x"].dtype), "state": s["state"]}


def _plain_conv_step(s):
    slots = s["slots"].long()
    ext = torch.cat([s["state"][slots], s["x"][:, None]], 1)
    y = s["bias"] + (ext.float() * s["w"].t()).sum(1)
    s["state"][slots] = ext[:, 1:]
    return {"out": _silu(y).to(s["x"].dtype), "state": s["state"]}


def _delta(s):
    v = s["dt"].float() + s["dt_bias"]
    return torch.where(v > 20.0, v, torch.log1p(torch.exp(v.clamp(max=20.0))))


def _plain_scan(s):
    """Blocks of SCAN_CHUNK packed tokens: decays and inputs are combined over spans of 1, 2, 4, .. tokens; a sequence's
    first token takes its initial state and forgets what was before it."""
    t, d = s["x"].shape
    c = s["case"]
    rep = d // c["groups"]
    slots = s["slots"].long()
    init = s["state"][slots] * (s["has_state"] != 0)[:, None, None]
    end = init.clone()
    starts = {e: n for n, e in reversed(list(enumerate(s["edges"][:-1]))) if s["lens"][n]}
    ends = {e - 1: n for n, e in enumerate(s["edges"][1:]) if s["lens"][n]}
    out = torch.empty(t, d, dtype=s["x"].dtype, device=s["x"].device)
    h = torch.zeros(d, c["states"], device=s["x"].device)
    delta, x = _delta(s), s["x"].float()
    for lo in range(0, t, SCAN_CHUNK):
        hi = min(t, lo + SCAN_CHUNK)
        b_, c_ = (s[k][lo:hi].float().repeat_interleave(rep, 1) for k in ("B", "C"))
        a = torch.exp(delta[lo:hi, :, None] * s["A"])
        b = (delta[lo:hi] * x[lo:hi])[..., None] * b_
        for i in range(lo, hi):
            if i in starts:
                b[i - lo] += a[i - lo] * init[starts[i]]
                a[i - lo] = 0.0
        b[0] += a[0] * h
        span = 1
        while span < hi - lo:
            b = torch.cat([b[:span], b[span:] + a[span:] * b[:-span]])
            a = torch.cat([a[:span], a[span:] * a[:-span]])
            span *= 2
        y = (b * c_).sum(-1) + s["D"] * x[lo:hi]
        if s["z"] is not None:
            y = y * _silu(s["z"][lo:hi].float())
        out[lo:hi] = y.to(out.dtype)
        h = b[-1]
        for i in range(lo, hi):
            if i in ends:
                end[ends[i]] = b[i - lo]
    s["state"][slots] = end
    return {"out": out, "state": s["state"]}


def _plain_scan_step(s):
    rep = s["x"].shape[1] // s["case"]["groups"]
    slots = s["slots"].long()
    b, c = (s[k].float().repeat_interleave(rep, 1) for k in ("B", "C"))
    delta, x = _delta(s), s["x"].float()
    h = torch.exp(delta[..., None] * s["A"]) * s["state"][slots] + (delta * x)[..., None] * b
    s["state"][slots] = h
    y = (h * c).sum(-1) + s["D"] * x
    if s["z"] is not None:
        y = y * _silu(s["z"].float())
    return {"out": y.to(s["x"].dtype), "state": s["state"]}


def _rms(x, w, s):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * (w + s["case"]["offset"])


def _plain_norm(s):
    c, h = s["case"], s["y"].float()
    if s["post"] is not None:
        h = _rms(h, s["post"], s)
    if s["gate"] is not None:
        gate = s["gate"].float()
        h = h * (_silu(gate) if c["gate"] == "silu" else 1.0 / (1.0 + torch.exp(-gate)))
    r = s["resid"] + c["scale"] * h
    s["resid_out"].copy_(r)
    return {"out": _rms(r, s["w"], s).to(torch.bfloat16), "resid": s["resid_out"]}


def _plain_logprobs(s):
    outs = []
    rows = max(1, (1 << 26) // s["logits"].shape[1])
    for lo in range(0, s["logits"].shape[0], rows):
        x = s["logits"][lo:lo + rows].float()
        m = x.amax(-1, keepdim=True)
        lp = x - m
        lp = lp - torch.log(torch.exp(lp).sum(-1, keepdim=True))
        p = torch.exp(lp)
        ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
        row = {"logprobs": lp.gather(1, s["tokens"][lo:lo + rows].long()[:, None])[:, 0], "entropy": ent}
        if k := s["case"]["top"]:
            val, ids = torch.sort(x, dim=-1, descending=True, stable=True)
            ids = ids[:, :k]
            row["top_logprobs"] = lp.gather(1, ids)
            row["top_ids"] = torch.where(val[:, :k] == -math.inf, torch.full_like(ids, -1), ids).to(torch.int32)
        outs.append(row)
    return {k: torch.cat([o[k] for o in outs]) for k in outs[0]}


_PLAIN = {"conv": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan, "scan_step": _plain_scan_step,
          "norm": _plain_norm, "logprobs": _plain_logprobs}


# ---------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    op, e = case["op"], 2 if case["dtype"] == "bf16" else 4
    if op in ("conv", "conv_step"):
        d, w = case["dim"], case["width"]
        t, n = (case["tokens"], case["seqs"]) if op == "conv" else (case["rows"], case["rows"])
        kept = n * (w - 1) * d * e * (2 if op == "conv_step" or case["resume"] else 1)
        return {"bytes": 2 * t * d * e + kept + d * (w + 1) * 4, "flops": t * d * (2 * w + 5)}
    if op in ("scan", "scan_step"):
        d, n, g = case["dim"], case["states"], case["groups"]
        t, q = (case["tokens"], case["seqs"]) if op == "scan" else (case["rows"], case["rows"])
        kept = q * d * n * 4 * (2 if op == "scan_step" or case["resume"] else 1)
        rows = t * (d * (4 if case["gate"] else 3) + 2 * g * n) * e
        # decay's product and exponential, decay and add to the state, read it
        return {"bytes": rows + kept + d * (n + 2) * 4, "flops": t * d * (7 * n + 12)}
    if op == "norm":
        n, d = case["rows"], case["dim"]
        return {"bytes": n * d * (e * (2 if case["gate"] else 1) + 4 + 4 + 2) + d * 4 * (2 if case["post"] else 1),
                "flops": n * d * 12}
    n, v = case["rows"], case["vocab"]
    return {"bytes": n * v * e + n * (12 + 8 * case["top"]), "flops": 5 * n * v}


# ---------------------------------------------------------------------------------- 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "conv":                      # sequence by sequence: a correlation of its own rows behind its state's
        pool, w = s["state"].double(), s["w"].double()
        out = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
        for n, slot in enumerate(s["slots"].tolist()):
            lo, hi = s["edges"][n], s["edges"][n + 1]
            old = pool[slot] if int(s["has_state"][n]) else torch.zeros_like(pool[slot])
            ext = torch.cat([old, s["x"][lo:hi].double()])
            if hi > lo:
                for j in range(case["width"]):
                    out[lo:hi] += w[:, j] * ext[j:j + hi - lo]
                v = out[lo:hi] + s["bias"].double()
                out[lo:hi] = v * torch.sigmoid(v)
            pool[slot] = ext[hi - lo:]
        return {"out": out, "state": pool}
    if op == "conv_step":
        pool, out = s["state"].double(), []
        for r, slot in enumerate(s["slots"].tolist()):
            ext = torch.cat([pool[slot], s["x"][r:r + 1].double()])
            v = s["bias"].double() + torch.einsum("jd,dj->d", ext, s["w"].double())
            out.append(v * torch.sigmoid(v))
            pool[slot] = ext[1:]
        return {"out": torch.stack(out), "state": pool}
    if op in ("scan", "scan_step"):       # token by token, all sequences at once, the longest first
        prompt = op == "scan"
        lens = s["lens"] if prompt else [1] * case["rows"]
        if lens and max(lens) * (1 + len(lens) * case["dim"] * case["states"] / 5e7) > 60000:
            return None
        order = sorted(range(len(lens)), key=lambda i: -lens[i])
        lens = [lens[i] for i in order]
        order = torch.tensor(order, device="cuda")
        starts = s["cu"][:-1].long()[order] if prompt else order
        slots = s["slots"].long()[order]
        pool = s["state"].double()
        st = pool[slots]
        if prompt:
            st = st * (s["has_state"][order] != 0).double()[:, None, None]
        a_log, per = s["A"].double(), case["dim"] // case["groups"]
        group = torch.arange(case["dim"], device="cuda") // per
        out = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
        live = len(lens)
        for t in range(lens[0]):
            while lens[live - 1] <= t:
                live -= 1
            at = starts[:live] + t
            u = s["x"][at].double()
            v = s["dt"][at].double() + s["dt_bias"].double()
            step = v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))
            b, c = s["B"][at].double()[:, group], s["C"][at].double()[:, group]
            st[:live] = torch.exp(step[..., None] * a_log) * st[:live] + (step * u)[..., None] * b
            y = torch.einsum("sdn,sdn->sd", st[:live], c) + s["D"].double() * u
            if s["z"] is not None:
                zz = s["z"][at].double()
                y = y * zz * torch.sigmoid(zz)
            out[at] = y
        pool[slots] = st
        return {"out": out, "state": pool}
    if op == "norm":
        h = s["y"].double()
        if s["post"] is not None:
            h = h / (h.square().sum(-1, keepdim=True) / h.shape[1] + s["eps"]).sqrt() * (s["post"].double() + case["offset"])
        if s["gate"] is not None:
            q = s["gate"].double()
            h = h * torch.sigmoid(q) * (q if case["gate"] == "silu" else 1.0)
        r = s["resid"].double() + case["scale"] * h
        n = r / (r.square().sum(-1, keepdim=True) / r.shape[1] + s["eps"]).sqrt() * (s["w"].double() + case["offset"])
        return {"out": n, "resid": r}
    n, k = case["rows"], case["top"]
    lps, ents, tops, ids = [], [], [], []
    step = max(1, (1 << 25) // case["vocab"])
    for lo in range(0, n, step):
        x = s["logits"][lo:lo + step].double()
        lse = torch.logsumexp(x, -1)
        lps.append(x.gather(1, s["tokens"][lo:lo + step].long()[:, None])[:, 0] - lse)
        p = torch.softmax(x, -1)
        ents.append(lse - (p * x.clamp(min=-1e300)).sum(-1))
        if k:
            # the k largest by value, then by index: largest remaining one, k times
            left, idx = x.clone(), torch.arange(x.shape[1], device="cuda")
            top_v, top_i = [], []
            for _ in range(k):
                m = left.amax(-1, keepdim=True)
                i = torch.where(left == m, idx, x.shape[1]).amin(-1)
                gone = m[:, 0] == -math.inf
                top_v.append(m[:, 0] - lse)
                top_i.append(torch.where(gone, -1, i))
                left.scatter_(1, i[:, None], -math.inf)
            tops.append(torch.stack(top_v, 1))
            ids.append(torch.stack(top_i, 1).to(torch.int32))
    out = {"logprobs": torch.cat(lps), "entropy": torch.cat(ents)}
    if k:
        out.update(top_logprobs=torch.cat(tops), top_ids=torch.cat(ids))
    return out
