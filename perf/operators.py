"""Measured cases of the operators of a recurrent (linear-attention) decoder's serving step.

* ``linear_attention``: prompts through S_t = exp(g_t) S_{t-1} + v_t k_t^T, o_t = scale S_t q_t with one decay
  per head (a packed, ragged batch; the state pool is read and updated in place).
* ``linear_attention_step``: the same recurrence for one new token per sequence.
* ``add_rmsnorm_fp8``: residual addition, root-mean-square norm and E4M3 rows with one scale per row, the
  input of the W8A8 projections.
* ``logit_rules``: repetition / frequency / presence penalties, token biases and the grammar mask on logits.

``run`` computes the plain form in elementary 32-bit torch operations, or, with ``own``, calls ``air_rs.ops``.
"""
import math

import torch

own = False

CHUNK = 128                      # tokens per block of the plain form of the prompt recurrence
MOST_TOKENS_HEADS = 16384 * 32   # the largest listed prompt, in tokens x heads


# ---------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one long document through a layer of 32 heads, one fixed decay per head: few, long recurrences
        {"name": "prompt_16k", "op": "prompt", "tokens": 16384, "seqs": 1, "heads": 32, "qk_heads": 32, "dk": 128,
         "dv": 128, "per_token": False, "resume": False, "split": 0},
        # a continuous-batching prefill: ragged prompts packed together, some resuming from a cached state
        {"name": "prompts_ragged", "op": "prompt", "tokens": 8111, "seqs": 13, "heads": 32, "qk_heads": 32, "dk": 128,
         "dv": 128, "per_token": True, "resume": True, "split": 1},
        # state-space layout: queries and keys shared by all the heads of a group, value heads of 64
        {"name": "prompts_grouped", "op": "prompt", "tokens": 4001, "seqs": 4, "heads": 64, "qk_heads": 8, "dk": 128,
         "dv": 64, "per_token": True, "resume": False, "split": 2},
        # one short prompt: latency to the first token
        {"name": "prompt_77", "op": "prompt", "tokens": 77, "seqs": 1, "heads": 16, "qk_heads": 16, "dk": 64,
         "dv": 64, "per_token": True, "resume": False, "split": 3},
        # one user generating: latency of a layer's step
        {"name": "step_1", "op": "step", "rows": 1, "heads": 32, "qk_heads": 32, "dk": 128, "dv": 128,
         "per_token": False, "dtype": "bf16"},
        # a full decode batch
        {"name": "step_64", "op": "step", "rows": 64, "heads": 32, "qk_heads": 32, "dk": 128, "dv": 128,
         "per_token": True, "dtype": "bf16"},
        # a wide decode batch of the grouped layout with fp32 projections
        {"name": "step_251_grouped", "op": "step", "rows": 251, "heads": 64, "qk_heads": 8, "dk": 128, "dv": 64,
         "per_token": True, "dtype": "f32"},
        # one decode row of an 8B-size residual stream
        {"name": "norm_1x4096", "op": "norm", "rows": 1, "dim": 4096, "dtype": "bf16", "offset": 0.0},
        # a decode batch at the 70B hidden size
        {"name": "norm_64x8192", "op": "norm", "rows": 64, "dim": 8192, "dtype": "f32", "offset": 0.0},
        # a prefill chunk
        {"name": "norm_6007x4096", "op": "norm", "rows": 6007, "dim": 4096, "dtype": "bf16", "offset": 1.0},
        # one request with every rule
        {"name": "rules_1x128256", "op": "rules", "rows": 1, "vocab": 128256, "dtype": "f32", "bias": 300,
         "allowed": 0.01},
        # a decode batch, bf16 logits, some rows under a grammar
        {"name": "rules_192x128256", "op": "rules", "rows": 192, "vocab": 128256, "dtype": "bf16", "bias": 40,
         "allowed": 0.3},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("prompt", "prompt", "step", "step", "norm", "rules"))
    if op in ("prompt", "step"):
        heads = rng.choice((4, 8, 16, 32, 64))
        qk = heads // rng.choice((1, 1, 2, 4))
        dk, dv = rng.choice(((128, 128), (128, 128), (128, 64), (64, 128), (64, 64)))
        c = {"op": op, "heads": heads, "qk_heads": qk, "dk": dk, "dv": dv, "per_token": rng.random() < 0.7}
        if op == "prompt":
            tokens = _log_int(rng, 1, min(20000, MOST_TOKENS_HEADS // heads))
            # packed lengths of every kind, empty sequences among them
            seqs = _log_int(rng, 1, max(1, min(48, tokens)))
            return {**c, "tokens": tokens, "seqs": seqs, "resume": rng.random() < 0.5, "split": rng.randrange(1 << 16)}
        return {**c, "rows": _log_int(rng, 1, min(400, 16384 // heads)), "dtype": rng.choice(("bf16", "bf16", "f32"))}
    if op == "norm":
        dim = 128 * _log_int(rng, 1, 128)
        return {"op": op, "rows": _log_int(rng, 1, min(20000, (6007 * 4096) // dim)), "dim": dim,
                "dtype": rng.choice(("bf16", "f32")), "offset": rng.choice((0.0, 1.0))}
    vocab = _log_int(rng, 1000, 160000)
    return {"op": op, "rows": _log_int(rng, 1, min(400, (192 * 128256) // vocab)), "vocab": vocab,
            "dtype": rng.choice(("bf16", "f32")), "bias": rng.choice((0, 1, 40, 300)),
            "allowed": rng.choice((0.01, 0.1, 0.3, 1.0))}


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


def _mixer_inputs(case, g, rows, slots, dtype):
    h, hq, dk, dv = case["heads"], case["qk_heads"], case["dk"], case["dv"]
    q = _randn(g, rows, hq, dk)
    k = torch.nn.functional.normalize(_randn(g, rows, hq, dk), dim=-1)
    v = _randn(g, rows, h, dv)
    # decays: fast heads forget within tens of tokens, slow heads keep thousands
    rate = torch.exp2(-2.0 - 9.0 * torch.arange(h, device="cuda") / h)
    decay = -rate
    if case["per_token"]:
        decay = decay * torch.nn.functional.softplus(_randn(g, rows, h) + 0.5)
    state = _randn(g, slots, h, dv, dk) * 0.5
    return {"case": case, "q": q.to(dtype), "k": k.to(dtype), "v": v.to(dtype), "decay": decay.contiguous(),
            "state": state, "scale": dk ** -0.5}


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "prompt":
        lens = _lengths(case)
        n = len(lens)
        s = _mixer_inputs(case, g, case["tokens"], n + 2, torch.bfloat16)
        cu = [0]
        for x in lens:
            cu.append(cu[-1] + x)
        s["lens"] = lens
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        s["slots"] = torch.randperm(n + 2, generator=g, device="cuda")[:n].to(torch.int32)
        s["has_state"] = (_rand(g, n) < (0.7 if case["resume"] else 0.0)).to(torch.int32)
        return s
    if case["op"] == "step":
        n = case["rows"]
        s = _mixer_inputs(case, g, n, n + 3, torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
        s["slots"] = torch.randperm(n + 3, generator=g, device="cuda")[:n].to(torch.int32)
        return s
    if case["op"] == "norm":
        n, d = case["rows"], case["dim"]
        x = _randn(g, n, d) * 2.0
        x[:, 7] *= 30.0                   # residual streams have outlier channels
        y = _randn(g, n, d).to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
        w = 1.0 + 0.2 * _randn(g, d) - case["offset"]
        return {"case": case, "x": x, "y": y, "w": w, "eps": 1e-5, "resid": torch.empty_like(x)}
    n, v = case["rows"], case["vocab"]
    logits = (_randn(g, n, v) * 3.0).to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
    slots = n + 3
    counts = torch.zeros(slots, v, dtype=torch.uint8, device="cuda")
    seen = torch.randint(0, v, (slots, 512), generator=g, device="cuda")
    counts.scatter_add_(1, seen, torch.randint(1, 9, (slots, 512), generator=g, device="cuda").to(torch.uint8))
    nb = min(case["bias"], v)
    ids = torch.argsort(_rand(g, n, v), dim=1)[:, :nb].to(torch.int32) if nb else torch.zeros(n, 0, dtype=torch.int32, device="cuda")
    words = (v + 31) // 32
    bits = (_rand(g, n, words * 32) < case["allowed"]).view(n, words, 32)
    mask = (bits.to(torch.int64) << torch.arange(32, device="cuda")).sum(-1)
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32)
    mask[1::2] = -1                       # every other row is free of the grammar
    mask[2::16] = 0                       # and a grammar may leave a row nothing
    return {"case": case, "logits": logits, "counts": counts,
            "count_row": torch.randperm(slots, generator=g, device="cuda")[:n].to(torch.int32),
            "repetition": 1.0 + 0.3 * _rand(g, n), "frequency": 0.5 * _rand(g, n), "presence": _rand(g, n) - 0.3,
            "bias_ptr": (torch.arange(n + 1, device="cuda") * nb).to(torch.int32),
            "bias_ids": ids.reshape(-1).contiguous(), "bias_vals": (_randn(g, n * nb) * 5.0).contiguous(),
            "mask": mask, "out": torch.empty(n, v, device="cuda")}


# ---------------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _own_prompt(s):
    from air_rs import ops
    out = ops.linear_attention(s["q"], s["k"], s["v"], s["decay"], state=s["state"], cu_seqlens=s["cu"],
                               slots=s["slots"], has_state=s["has_state"], scale=s["scale"])
    return {"out": out, "state": s["state"]}


def _own_step(s):
    from air_rs import ops
    out = ops.linear_attention_step(s["q"], s["k"], s["v"], s["decay"], s["state"], slots=s["slots"], scale=s["scale"])
    return {"out": out, "state": s["state"]}


def _own_norm(s):
    from air_rs import ops
    xq, xs = ops.add_rmsnorm_fp8(s["x"], s["y"], s["w"], s["eps"], w_offset=s["case"]["offset"], resid_out=s["resid"])
    return {"codes": xq.view(torch.float8_e4m3fn), "scales": xs, "resid": s["resid"]}


def _own_rules(s):
    from air_rs import ops
    return ops.logit_rules(s["logits"], out=s["out"], counts=s["counts"], count_row=s["count_row"],
                           repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                           bias=(s["bias_ptr"], s["bias_ids"], s["bias_vals"]), mask=s["mask"])


_OWN = {"prompt": _own_prompt, "step": _own_step, "norm": _own_norm, "rules": _own_rules}


def _plain_prompt(s):
    """Blocks of CHUNK tokens: masked, decayed scores within a block, the blocks' own states, and each
    block's incoming state as a decayed sum of the earlier ones of its sequence."""
    dev, h = s["q"].device, s["case"]["heads"]
    rep = h // s["q"].shape[1]
    lens = torch.tensor(s["lens"], device=dev)
    starts = s["cu"][:-1].long()
    per = (lens + CHUNK - 1) // CHUNK
    seq = torch.repeat_interleave(torch.arange(len(s["lens"]), device=dev), per)      # sequence of each block
    first = torch.cumsum(per, 0) - per
    block = torch.arange(seq.numel(), device=dev) - first[seq]                        # its index in the sequence
    pos = block[:, None] * CHUNK + torch.arange(CHUNK, device=dev)[None]
    valid = pos < lens[seq][:, None]
    tok = torch.where(valid, starts[seq][:, None] + pos, torch.zeros_like(pos))
    keep = valid[..., None, None]
    q = s["q"].float().repeat_interleave(rep, 1)[tok].mul(s["scale"]).transpose(1, 2)              # [b, h, c, dk]
    k = (s["k"].float().repeat_interleave(rep, 1)[tok] * keep).transpose(1, 2)
    v = (s["v"].float()[tok] * keep).transpose(1, 2)
    g = s["decay"][tok] if s["decay"].dim() == 2 else s["decay"].expand(*tok.shape, h)
    g = (g * valid[..., None]).transpose(1, 2)                                                     # [b, h, c]
    cum = torch.cumsum(g, -1)
    total = cum[..., -1]
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=dev).tril()
    w = torch.exp((cum[..., :, None] - cum[..., None, :]).masked_fill(~low, float("-inf")))
    inner = torch.matmul(torch.matmul(q, k.transpose(-1, -2)) * w, v)
    own_state = torch.matmul((v * torch.exp(total[..., None] - cum)[..., None]).transpose(-1, -2), k)   # [b, h, dv, dk]
    upto = torch.cumsum(total, 0)                                                                  # decay before and in a block
    same = (seq[:, None] == seq[None, :]).tril(-1)
    back = torch.exp(((upto - total)[:, None] - upto[None]).masked_fill(~same[..., None], float("-inf")))   # [b, b, h]
    slots = s["slots"].long()
    init = s["state"][slots] * (s["has_state"] != 0)[:, None, None, None]
    upto_seq = torch.zeros(len(s["lens"]), h, device=dev).index_add_(0, seq, total)
    before = (upto - total) - (upto - total)[first[seq].clamp(max=max(seq.numel() - 1, 0))]        # decay since the sequence began
    into = torch.einsum("abh,bhvk->ahvk", back, own_state) + torch.exp(before)[..., None, None] * init[seq]
    outer = torch.matmul(q * torch.exp(cum)[..., None], into.transpose(-1, -2))
    o = (inner + outer).transpose(1, 2)[valid]
    out = torch.empty(s["q"].shape[0], h, s["case"]["dv"], dtype=s["q"].dtype, device=dev)
    out[tok[valid]] = o.to(out.dtype)
    last = (torch.cumsum(per, 0) - 1).clamp(min=0)
    some = (per > 0)[:, None, None, None]
    at_end = torch.exp(total[last])[..., None, None] * into[last] + own_state[last]
    s["state"][slots] = torch.where(some, at_end, init)
    return {"out": out, "state": s["state"]}


def _plain_step(s):
    h = s["case"]["heads"]
    rep = h // s["q"].shape[1]
    q = s["q"].float().repeat_interleave(rep, 1) * s["scale"]
    k = s["k"].float().repeat_interleave(rep, 1)
    slots = s["slots"].long()
    a = torch.exp(s["decay"]).expand(q.shape[0], h)
    st = s["state"][slots] * a[..., None, None] + s["v"].float()[..., :, None] * k[..., None, :]
    s["state"][slots] = st
    out = (st * q[..., None, :]).sum(-1)
    return {"out": out.to(s["q"].dtype), "state": s["state"]}


def _plain_norm(s):
    r = s["x"] + s["y"].float()
    n = r * torch.rsqrt((r * r).mean(-1, keepdim=True) + s["eps"]) * (s["w"] + s["case"]["offset"])
    amax = n.abs().amax(-1, keepdim=True)
    inv = torch.where(amax > 0, 448.0 / amax, torch.zeros_like(amax))
    codes = (n * inv).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    s["resid"].copy_(r)
    return {"codes": codes, "scales": (amax / 448.0)[:, 0], "resid": s["resid"]}


def _plain_rules(s):
    c = s["counts"][s["count_row"].long()].float()
    x = s["logits"].float()
    f = torch.pow(s["repetition"][:, None], c)
    x = torch.where(c > 0, torch.where(x > 0, x / f, x * f), x)
    x = x - s["frequency"][:, None] * c - s["presence"][:, None] * (c > 0)
    n, v = x.shape
    row = torch.repeat_interleave(torch.arange(n, device=x.device), (s["bias_ptr"][1:] - s["bias_ptr"][:-1]).long(),
                                  output_size=s["bias_ids"].numel())
    x = x.index_put((row, s["bias_ids"].long()), s["bias_vals"], accumulate=True)
    i = torch.arange(v, device=x.device)
    allow = (s["mask"].long()[:, i >> 5] >> (i & 31)) & 1
    s["out"].copy_(x.masked_fill(allow == 0, float("-inf")))
    return s["out"]


_PLAIN = {"prompt": _plain_prompt, "step": _plain_step, "norm": _plain_norm, "rules": _plain_rules}


# ---------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] in ("prompt", "step"):
        h, hq, dk, dv = case["heads"], case["qk_heads"], case["dk"], case["dv"]
        if case["op"] == "prompt":
            t, n, e = case["tokens"], case["seqs"], 2
            state = n * h * dk * dv * 4 * (2 if case["resume"] else 1)
        else:
            t, n, e = case["rows"], case["rows"], 2 if case["dtype"] == "bf16" else 4
            state = n * h * dk * dv * 8
        rows = t * (2 * hq * dk + 2 * h * dv) * e + (t * h * 4 if case["per_token"] else h * 4)
        # the recurrence itself: decay and add to the state, and read it with the query
        return {"bytes": rows + state, "flops": 5 * t * h * dk * dv}
    if case["op"] == "norm":
        n, d, e = case["rows"], case["dim"], 2 if case["dtype"] == "bf16" else 4
        return {"bytes": n * d * (4 + e + 4 + 1) + 4 * n + 4 * d, "flops": 8 * n * d}
    n, v, e = case["rows"], case["vocab"], 2 if case["dtype"] == "bf16" else 4
    return {"bytes": n * v * (e + 1 + 4) + n * ((v + 31) // 32) * 4 + n * case["bias"] * 8, "flops": 4 * n * v}


# ---------------------------------------------------------------------------------- 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prompt":            # token by token, all sequences and heads at once, the longest first
        rep, h = case["heads"] // case["qk_heads"], case["heads"]
        order = sorted(range(len(s["lens"])), key=lambda i: -s["lens"][i])
        lens = [s["lens"][i] for i in order]
        order = torch.tensor(order, device="cuda")
        starts, slots = s["cu"][:-1].long()[order], s["slots"].long()[order]
        pool = s["state"].double()
        st = pool[slots] * (s["has_state"][order] != 0).double()[:, None, None, None]
        out = torch.zeros(case["tokens"], h, case["dv"], dtype=torch.float64, device="cuda")
        live = len(lens)
        for t in range(lens[0]):
            while lens[live - 1] <= t:
                live -= 1
            at = starts[:live] + t
            a = (s["decay"][at] if s["decay"].dim() == 2 else s["decay"].expand(live, h)).double().exp()
            k, q = (s[n][at].double().repeat_interleave(rep, 1) for n in ("k", "q"))
            st[:live].mul_(a[..., None, None]).add_(s["v"][at].double()[..., :, None] * k[..., None, :])
            out[at] = torch.matmul(st[:live], q[..., None])[..., 0] * s["scale"]
        pool[slots] = st
        return {"out": out, "state": pool}
    if case["op"] == "step":
        st, rep = s["state"].double(), case["heads"] // case["qk_heads"]
        out = torch.empty(case["rows"], case["heads"], case["dv"], dtype=torch.float64, device="cuda")
        for r, slot in enumerate(s["slots"].tolist()):
            g = s["decay"][r] if s["decay"].dim() == 2 else s["decay"]
            k, q = (s[n][r].double().repeat_interleave(rep, 0) for n in ("k", "q"))
            st[slot] = st[slot] * g.double().exp()[:, None, None] + torch.einsum("hv,hk->hvk", s["v"][r].double(), k)
            out[r] = torch.einsum("hvk,hk->hv", st[slot], q) * s["scale"]
        return {"out": out, "state": st}
    if case["op"] == "norm":
        r = s["x"].double() + s["y"].double()
        n = r / ((r ** 2).sum(-1, keepdim=True) / r.shape[-1] + s["eps"]).sqrt() * (s["w"].double() + case["offset"])
        scale = n.abs().max(-1).values / 448.0
        # the codes stand for the normalised row over its scale
        return {"codes": n / scale[:, None], "scales": scale, "resid": r}
    x = s["logits"].double()
    for i, slot in enumerate(s["count_row"].tolist()):
        c = s["counts"][slot].long()
        at = c.nonzero()[:, 0]
        n, y = c[at].double(), x[i, at]
        f = s["repetition"][i].double() ** n
        x[i, at] = torch.where(y > 0, y / f, y * f) - s["frequency"][i].double() * n - s["presence"][i].double()
        lo, hi = s["bias_ptr"][i:i + 2].tolist()
        x[i].index_add_(0, s["bias_ids"][lo:hi].long(), s["bias_vals"][lo:hi].double())
        words = s["mask"][i].long() & 0xFFFFFFFF
        bits = torch.stack([(words >> b) & 1 for b in range(32)], 1).reshape(-1)[:x.shape[1]]
        x[i, bits == 0] = -math.inf
    return x
