"""Where the state-space operators round: states that a token forgets, growing states across cuts, rows of logits with one
sure token; and launch forms that only larger calls take.

u = 2^-24. An exponential 2^x is off by at most 4 u relatively; the decay less one of a slow state (|delta A| <= 1/32) by
7.1 u of itself.
"""
import math

import pytest
import torch

from air_rs import ops
from test_state_space_ops import TYPES, U, _dev, _gen, _held, _i32, _scan_inputs, _silu

gpu = pytest.mark.gpu


# ---------------------------------------------------------------------------------- selective scan
def _scan_bound(x, dt, A, B, C, D, z, bias, softplus, lens, init):
    """-> out, its tolerance, states, their tolerance. Every rounding is relative to what is rounded: the old state counts
    as far as the token keeps it, and whole only beside slow decays, where it is added to the token's input first."""
    T, d = x.shape
    per = torch.arange(d) // (d // B.shape[1])
    v = dt.double() + (bias.double() if bias is not None else 0)
    ev = U * (dt.double().abs() + (bias.double().abs() if bias is not None else 0))
    if softplus:
        delta = v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))
        ed = delta * (2 * v.abs() * U + 10 * U) + ev * torch.sigmoid(v) + ev * delta
    else:
        delta, ed = v, ev
    A, x64 = A.double(), x.double()
    out, tol = torch.zeros(T, d, dtype=torch.float64), torch.zeros(T, d, dtype=torch.float64)
    ends, tols, t = [], [], 0
    for n, L in enumerate(lens):
        h, e = init[n].double().clone(), torch.zeros(d, A.shape[1], dtype=torch.float64)
        for _ in range(L):
            g = delta[t][:, None] * A
            a, b, c = torch.exp(g), B[t].double()[per], C[t].double()[per]
            inp = (delta[t] * x64[t])[:, None] * b
            eg = (ed[t] + 3 * U * delta[t].abs())[:, None] * A.abs()
            slow, fast = g.abs() < 0.0313, g.abs() > 0.0312                 # both may hold beside 1/32
            own = torch.maximum(7.1 * U * torch.expm1(g).abs() * slow, (4 * U * a + 2.0 ** -126) * fast)
            e = a * e + (a * eg + own) * h.abs() + U * (h.abs() + inp.abs()) * slow + 3 * U * inp.abs() + \
                (ed[t] * x64[t].abs())[:, None] * b.abs()
            h = a * h + inp
            e = 1.001 * (e + U * h.abs())
            out[t] = (h * c).sum(-1)
            tol[t] = (e * c.abs()).sum(-1) + (A.shape[1] + 3) * U * (h * c).abs().sum(-1)
            t += 1
        ends.append(h)
        tols.append(e)
    if D is not None:
        out, tol = out + D.double() * x64, tol + 2 * U * ((D.double() * x64).abs() + out.abs())
    if z is not None:
        s = _silu(z.double())
        out, tol = out * s, tol * s.abs() * 1.001 + (out * s).abs() * (2 * z.double().abs() + 12) * U
    return out, tol, torch.stack(ends), torch.stack(tols)


FORGETS = [  # lens, channels, states, groups: sequence by sequence, tiles of every width, tiles that cut a sequence, two blocks an SM
    ([3, 1, 4, 5], 32, 16, 1),
    ([9], 12, 130, 1),
    ([40, 17], 32, 8, 1),
    ([40, 17], 33, 16, 1),
    ([19, 40], 32, 24, 2),
    ([40, 17], 24, 64, 1),
    ([700, 60], 64, 16, 1),
    ([300, 230], 37, 8, 1),
    ([300, 230], 40, 32, 1),
    ([300, 230], 32, 64, 2),
    ([260, 300], 24, 40, 1),
    ([25, 14], 5001, 16, 1),
    ([14, 25], 2512, 24, 1),
]


def _forgetting(seed, T, d, n, groups, dtype):
    """Slow steps, and at every seventh token one that forgets all before it: 20 to 60 decay times, with a small input."""
    i = _scan_inputs(seed, T, d, n, groups, dtype)
    i["A"] = -(1 + torch.rand(d, n, generator=_gen(seed)))
    i["dt"] = (0.002 * i["dt"].float().abs()).to(dtype)
    i["dt"][5::7] = (20 + 10 * torch.rand(T, d, generator=_gen(seed + 1)))[5::7].to(dtype)
    i["dt"][0] = 25.0
    i["x"][5::7] = (1e-3 * i["x"].float())[5::7].to(dtype)
    i["x"][0] *= 1e-3
    return i


@gpu
@pytest.mark.parametrize("case", range(len(FORGETS)))
@pytest.mark.parametrize("dtype", TYPES)
def test_scan_forgets_large_states(case, dtype):
    """The state after a token that forgets is as exact as its own input, however large the state was before."""
    lens, d, n, groups = FORGETS[case]
    T, N = sum(lens), len(lens)
    i = _forgetting(case, T, d, n, groups, dtype)
    pool = 1e4 * torch.randn(N, d, n, generator=_gen(90 + case))
    ref, tol, ends, etol = _scan_bound(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], None, None, False, lens, pool)
    st = pool.cuda()
    out = ops.selective_scan(*(i[k].cuda() for k in ("x", "dt", "A", "B", "C")), D=i["D"].cuda(), softplus=False, state=st,
                             has_state=_i32([1] * N), cu_seqlens=_i32([0] + torch.tensor(lens).cumsum(0).tolist()))
    _held(out, ref, tol, dtype == torch.bfloat16)
    _held(st, ends, etol, False)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,n", [(32, 16), (24, 8), (10, 5), (8, 64), (6, 200)])
def test_scan_step_forgets_large_states(dtype, d, n):
    i = _forgetting(d, 8, d, n, 1, dtype)              # rows 0 and 5 forget
    pool = 1e4 * torch.randn(8, d, n, generator=_gen(d))
    ref, tol, ends, etol = _scan_bound(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], None, None, False, [1] * 8, pool)
    st = pool.cuda()
    c = {k: _dev(v) for k, v in i.items()}
    out = ops.selective_scan_step(c["x"], c["dt"], c["A"], c["B"], c["C"], st, D=c["D"], softplus=False)
    _held(out, ref, tol, dtype == torch.bfloat16)
    _held(st, ends, etol, False)


@gpu
@pytest.mark.parametrize("T", [1, 40])
def test_scan_keeps_infinite_states_of_fast_decays(T):
    d, n = 16, 16
    i = {k: _dev(v) for k, v in _scan_inputs(0, T, d, n, 1, torch.float32, gate=False).items()}
    st = torch.full((1, d, n), math.inf, device="cuda")
    ops.selective_scan(i["x"], torch.ones_like(i["dt"]), torch.full_like(i["A"], -1.0), i["B"], i["C"], softplus=False, state=st,
                       has_state=_i32([1]))
    assert bool((st == math.inf).all())


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_growing_states_across_cuts(dtype):
    """Positive rates: a stretch of tokens may multiply a state by more than f32 holds while the state itself fits."""
    T, d, n = 512, 16, 16                              # cut into tiles of 64 tokens
    i = _scan_inputs(0, T, d, n, 1, dtype, gate=False)
    i["A"] = 1.5 + 0.1 * torch.rand(d, n, generator=_gen(1))
    i["x"][:-5] = 0
    tile = torch.arange(T) // 64
    i["dt"] = torch.where(tile % 2 == 0, 1.0, -1.0)[:, None].expand(T, d).contiguous().to(dtype)
    for start in (0.0, 1e-32):                         # at most e^102 times that
        pool = torch.full((1, d, n), start)
        ref, tol, ends, etol = _scan_bound(i["x"], i["dt"], i["A"], i["B"], i["C"], None, None, None, False, [T], pool)
        st = pool.cuda()
        out = ops.selective_scan(*(i[k].cuda() for k in ("x", "dt", "A", "B", "C")), softplus=False, state=st, has_state=_i32([1]))
        _held(out, ref, tol, dtype == torch.bfloat16)
        _held(st, ends, etol, False)
    # rates that no product of f32 holds, and nothing to grow
    i["dt"].fill_(4.0)
    ref, tol, ends, etol = _scan_bound(i["x"], i["dt"], i["A"], i["B"], i["C"], None, None, None, False, [T], torch.zeros(1, d, n))
    st = torch.zeros(1, d, n, device="cuda")
    out = ops.selective_scan(*(i[k].cuda() for k in ("x", "dt", "A", "B", "C")), softplus=False, state=st)
    _held(out, ref, tol, dtype == torch.bfloat16)
    _held(st, ends, etol, False)


# ---------------------------------------------------------------------------------- token log probabilities
@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V", [(12, 97), (12, 70001), (500, 40000)])
def test_entropy_of_rows_with_a_huge_logit(dtype, T, V):
    """One logit so far above the others that it is certain: entropy zero, also where differences pass the type's range."""
    x = 3 * torch.randn(T, V, generator=_gen(T)).cuda()
    top = torch.tensor([torch.finfo(dtype).max, 1e36, 1e35, 3e38], device="cuda")[torch.arange(T, device="cuda") % 4]
    at = torch.randint(0, V, (T,), generator=_gen(V)).cuda()
    x[torch.arange(T, device="cuda"), at] = top
    x[1::3, at[0]] = torch.minimum(x[1::3, at[0]], torch.tensor(torch.finfo(dtype).min, device="cuda"))
    x[torch.arange(T, device="cuda"), at] = top
    r = ops.token_logprobs(x.to(dtype), at.int(), top=2)
    assert bool((r.entropy == 0).all()) and bool((r.logprobs == 0).all())
    assert torch.equal(r.top_ids[:, 0], at.int()) and bool((r.top_logprobs[:, 0] == 0).all())


def _lp_bound(logits, tokens, top):
    """Holds a call against 64 bits, on the device. Exponentials are of d = x - (the largest so far), off by (3 |d| + 4) u,
    but the largest logit's is exactly one: what is relative to the other terms only counts for their share of the sum. R
    counts roundings of the sums: 16 adds of four vectors, one for each of a thread's groups of four (4096 logits a block
    or more) and 16 of the halves, lanes, warps and blocks; where the maximum moves, the terms before it take a factor that is
    off by 4 u, at most once a group and ten times in the joins."""
    r = ops.token_logprobs(logits, tokens, top=top)
    V = logits.shape[1]
    R = 16 + (V / 4096 + 2) + 16
    small = 4 + 4 * (V / 4096 + 12)
    for lo in range(0, logits.shape[0], 256):
        rows = slice(lo, lo + 256)
        x = logits[rows].double()
        m = x.amax(-1, keepdim=True)
        dist = m - x
        s = torch.exp(-dist).sum(-1)
        p, ls = torch.exp(-dist) / s[:, None], torch.log(s)
        spread = (p * dist).sum(-1)
        rel = (3 * spread + small * (p * (dist > 0)).sum(-1) + R) * U
        lp = -dist - ls[:, None]
        near = lambda at, v: rel[:, None] + U * (2 * ls[:, None] + dist.gather(1, at) + v.abs())
        tok = tokens[rows].long()[:, None]
        want = lp.gather(1, tok)
        _held(r.logprobs[rows], want[:, 0].cpu(), near(tok, want)[:, 0].cpu(), False)
        ent = ls + spread
        te = rel * (1 + spread) + (p * dist * (3 * dist + 1 + small)).sum(-1) * U + R * U * spread + U * (2 * ls + 2 * spread + ent)
        _held(r.entropy[rows], ent.cpu(), te.cpu(), False)
        if top:
            order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
            assert torch.equal(r.top_ids[rows].long(), order)
            want = lp.gather(1, order)
            _held(r.top_logprobs[rows], want.cpu(), near(order, want).cpu(), False)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 450])
def test_entropy_of_sure_rows(dtype, T):
    """A favourite 11 to 16 above everything else: its exponential must not swallow the small ones."""
    V = 128000
    x = torch.zeros(T, V)
    x[::2] = torch.randn(len(x[::2]), V, generator=_gen(T))
    at = torch.randint(0, V, (T,), generator=_gen(1))
    x[torch.arange(T), at] = 11 + 4.9 * torch.rand(T, generator=_gen(2))
    _lp_bound(x.to(dtype).cuda(), at.int().cuda(), 1)
    x[:, 0] = 12.0                                     # and one that comes first
    _lp_bound(x.to(dtype).cuda(), at.int().cuda(), 0)


# ---------------------------------------------------------------------------------- the engine's scores
def _engine(device):
    from air_rs.gguf import GGMLType
    from air_rs.models.config import tiny_llama
    from air_rs.models.random_init import random_tensors
    from air_rs.models.reference import OracleModel
    from air_rs.runtime.builder import build_runner
    from air_rs.runtime.engine import Engine
    cfg = tiny_llama()
    recs = list(random_tensors(cfg, GGMLType.Q8_0, seed=0, device="cpu"))
    if device == "cpu":
        return Engine(cfg, None, oracle=OracleModel(cfg, {n: (r, q, s) for n, r, q, s in recs}))
    return Engine(cfg, build_runner(cfg, iter(recs), device="cuda", max_batch=8, max_model_len=256, num_blocks=64))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_engine_scores_no_id_outside_the_vocabulary(device):
    eng = _engine(device)
    V, ids = eng.cfg.vocab_size, [5, 6, 7, 8]
    scores = eng.token_logprobs(ids)
    for bad in (-1, V, V + 100, -V):
        for at in range(len(ids)):
            wrong = ids[:at] + [bad] + ids[at + 1:]
            with pytest.raises(IndexError, match="vocabulary"):
                eng.token_logprobs(wrong)
            with pytest.raises(IndexError, match="vocabulary"):
                eng.token_scores(wrong, top=2)
    with pytest.raises(IndexError, match="vocabulary"):
        eng.token_scores([V], add_bos=False)
    assert eng.token_logprobs(ids) == scores            # nothing is left of the refused calls
    if device == "cuda":
        from air_rs.runtime.engine import SamplingParams
        out = eng.generate_ids([ids], SamplingParams(max_tokens=3, temperature=0.0, ignore_eos=True))
        assert len(out[0]) == 3 and int(eng.runner.err) == 0
        ops.check_errors()
    assert eng.token_logprobs([0, V - 1], add_bos=False)[0] < 0


@gpu
def test_engine_scores_read_the_runners_errors():
    eng = _engine("cuda")
    eng.runner.err.fill_(1)                             # as a kernel of the scored forward would
    with pytest.raises(RuntimeError, match="error code 1"):
        eng.token_scores([5, 6, 7])
    assert len(eng.token_logprobs([5, 6, 7], add_bos=False)) == 2
    assert eng.seqs.allocator.num_used_blocks() == 0


# ---------------------------------------------------------------------------------- causal convolution
@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("step", [False, True])
def test_few_taps_read_whole_rows(dtype, step):
    """Two and three taps take no longer than four: their rows are as whole, and they compute less."""
    d = 8192
    x = torch.randn(4096 if step else 8192, d, device="cuda").to(dtype)
    out = torch.empty_like(x)

    def us(W):
        w, st = torch.randn(d, W, device="cuda"), torch.zeros(x.shape[0], W - 1, d, dtype=dtype, device="cuda")
        times = []
        for _ in range(9):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            ops.causal_conv_step(x, w, st, out=out) if step else ops.causal_conv(x, w, out=out)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b) * 1e3)
        return sorted(times)[4]
    four = us(4)
    for W in (2, 3):
        assert us(W) <= 1.3 * four


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,vectors", [(1100, 640), (1100, 1500), (1000, 1500), (30, 4100), (150, 4100), (300, 4100), (420, 4100), (600, 4100)])
@pytest.mark.parametrize("top", [0, 7])
def test_token_logprobs_blocks_of_every_size(dtype, T, vectors, top):
    """Blocks of 64, 128, 256 and 512 threads and clusters of 8, 4 and 2, rows of odd lengths that start anywhere."""
    V = vectors * (8 if dtype == torch.bfloat16 else 4) - 3
    g = torch.Generator(device="cuda").manual_seed(T + vectors)
    x = (4 * torch.randn(T, V + 5, generator=g, device="cuda")).to(dtype)[:, 2:V + 2]
    tok = torch.randint(0, V, (T,), generator=g, device="cuda").int()
    tok[::3] = x.float().argmax(-1)[::3].int()
    _lp_bound(x, tok, top)


# ---------------------------------------------------------------------------------- forms of larger calls
@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,d,n", [(75, 8192, 16), (21, 8192, 64), (41, 8190, 24), (161, 4096, 8)])
def test_scan_step_with_several_rows_a_thread(dtype, B, d, n):
    i = _scan_inputs(B, B, d, n, 1, dtype)
    g = _gen(B)
    pool = torch.randn(B + 2, d, n, generator=g)
    slots = torch.randperm(B + 2, generator=g)[:B].int()
    slots[2], slots[B - 1] = -1, -1
    live = slots >= 0
    init = pool[slots.long().clamp(min=0)]
    ref, tol, ends, etol = _scan_bound(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], i["z"], i["bias"], True, [1] * B, init)
    c = {k: _dev(v) for k, v in i.items()}
    st = pool.cuda()
    out = ops.selective_scan_step(c["x"], c["dt"], c["A"], c["B"], c["C"], st, D=c["D"], z=c["z"], dt_bias=c["bias"], slots=slots.cuda())
    _held(out[live.cuda()], ref[live], tol[live], dtype == torch.bfloat16)
    assert bool((out[~live.cuda()] == 0).all())
    st = st.cpu()
    _held(st[slots[live].long()], ends[live], etol[live], False)
    free = [s for s in range(B + 2) if s not in slots.tolist()]
    assert torch.equal(st[free], pool[free])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,d,n,groups", [([300, 0, 200, 77], 32, 64, 1), ([150, 400], 37, 40, 1), ([513], 48, 64, 2), ([70, 330], 22, 33, 1)])
def test_scan_cuts_prompts_with_many_states(dtype, lens, d, n, groups):
    """33 to 64 states, sequences that cross the ends of tiles, with and without an initial state, rows at odd places too."""
    T, N = sum(lens), len(lens)
    i = _scan_inputs(T, T, d, n, groups, dtype)
    pool = torch.randn(N, d, n, generator=_gen(T))
    for has in ([1] * N, [k % 2 for k in range(N)]):
        init = pool * torch.tensor(has)[:, None, None]
        ref, tol, ends, etol = _scan_bound(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], i["z"], i["bias"], True, lens, init)
        for pad in (1, 16):
            st, out = pool.cuda(), torch.full((T, d + pad), 7.0, dtype=dtype, device="cuda")
            ops.selective_scan(*(i[k].cuda() for k in ("x", "dt", "A", "B", "C")), D=i["D"].cuda(), z=i["z"].cuda(), dt_bias=i["bias"].cuda(),
                               state=st, has_state=_i32(has), cu_seqlens=_i32([0] + torch.tensor(lens).cumsum(0).tolist()), out=out[:, :d])
            _held(out[:, :d], ref, tol, dtype == torch.bfloat16)
            assert bool((out[:, d:] == 7).all())
            _held(st, ends, etol, False)


# ---------------------------------------------------------------------------------- state rows
@gpu
@pytest.mark.parametrize("T", [2, 40])
def test_rows_of_an_empty_pool_are_reported(T):
    """A pool without rows has no row 0: reported, and as if without a state."""
    d = 16
    i = {k: _dev(v) for k, v in _scan_inputs(0, T, d, 16, 1, torch.float32, gate=False).items()}
    args, w = (i["x"], i["dt"], i["A"], i["B"], i["C"]), torch.randn(d, 4, generator=_gen(0)).cuda()
    none = dict(conv=torch.empty(0, 3, d, device="cuda"), scan=torch.empty(0, d, 16, device="cuda"))
    for slot, code in ((0, 1), (3, 1), (-1, 0)):
        err = torch.zeros(2, dtype=torch.int32, device="cuda")
        kw = dict(slots=_i32([slot]), has_state=_i32([1]))
        assert torch.equal(ops.causal_conv(i["x"], w, state=none["conv"], err=err[:1], **kw), ops.causal_conv(i["x"], w))
        assert torch.equal(ops.selective_scan(*args, state=none["scan"], err=err[1:], **kw), ops.selective_scan(*args))
        assert err.tolist() == [code, code]
