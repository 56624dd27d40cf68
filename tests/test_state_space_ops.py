"""Operators of a state-space decoder against their definitions in 64 bits.

Tolerances count roundings: u = 2^-24 for f32, b = 2^-8 for bf16 outputs (half a step, relative). The kernels' exponential
2^x is off by at most 4 u relatively, exp(x) = 2^(x log2 e) by 4 u + 2 u |x| (the product and its constant), a fast
division by 4 u. So sigmoid and SiLU of v are off by (2 |v| + 10) u relatively. softplus: exp(-|v|) as above, the
logarithm's polynomial 3.0 u with its roundings, the sum dt + bias u (|dt| + |bias|) absolutely, at most so much
relatively in softplus: delta is off by (2 |v| + |dt| + |bias| + 10) u relatively.

The scan's bound is carried along the recurrence, one step's new errors at a time: h' = h + (2^g' - 1) h + delta x B has the
decay's own error (relatively 5 u of 2^g' - 1 for |g| <= 1/10, else 6 u absolutely), the error of g = delta A (relatively that of delta
and 3 u), two roundings of terms of |h| + |b| (each sum is at most that) and those of delta x B.
"""
import math

import pytest
import torch

from air_rs import ops

U, BF = 2.0 ** -24, 2.0 ** -8
gpu = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float32]


def _i32(v, dev="cuda"):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _held(got, ref, tol, rounded):
    """|got - ref| <= tol, plus the rounding of the output's type; NaN and infinities where the reference has them."""
    got, ref = got.detach().double().cpu(), ref.double()
    odd = ~torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(got[odd & ~torch.isnan(ref)], ref[odd & ~torch.isnan(ref)])
    over = (got - ref).abs() - (tol + (BF * 1.01 * (ref.abs() + tol) if rounded else 0) + 1e-37)
    over = over[~odd]
    assert over.numel() == 0 or float(over.max()) <= 0, f"{float(over.max()):.3g} over the bound"


def _silu(v):
    return v * torch.sigmoid(v)


# ---------------------------------------------------------------------------------- causal convolution
def _conv_ref(x, w, bias, lens, init, silu):
    """-> out, tolerance, last inputs; init [N, W - 1, D]."""
    H = w.shape[1] - 1
    outs, mags, ends, t = [], [], [], 0
    for n, L in enumerate(lens):
        ext = torch.cat([init[n].double(), x[t:t + L].double()])
        t += L
        y = torch.zeros(L, x.shape[1], dtype=torch.float64)
        m = torch.zeros_like(y)
        for j in range(H + 1):
            y += w[:, j].double() * ext[j:j + L]
            m += (w[:, j].double() * ext[j:j + L]).abs()
        if bias is not None:
            y, m = y + bias.double(), m + bias.double().abs()
        outs.append(y)
        mags.append(m)
        ends.append(ext[L:].to(x.dtype))
    y, m = torch.cat(outs), torch.cat(mags) * (H + 2) * U
    if silu:                                         # |SiLU'| <= 1.1
        return _silu(y), 1.1 * m + (2 * y.abs() + 10) * U * _silu(y).abs(), torch.stack(ends)
    return y, m, torch.stack(ends)


CONVS = [  # lens, D, W
    ([1], 8, 4),
    ([0, 1, 2, 3, 4, 0, 5, 31, 32, 33, 0], 24, 4),
    ([29, 3, 1, 1, 64], 1032, 4),
    ([40, 0, 1], 513, 3),
    ([2, 100], 7, 2),
    ([300], 1, 4),
    ([1, 1, 1, 1] * 20, 136, 2),
]


@gpu
@pytest.mark.parametrize("case", range(len(CONVS)))
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("silu", [True, False])
def test_conv_matches_the_sum(case, dtype, silu):
    lens, D, W = CONVS[case]
    T, N, g = sum(lens), len(lens), _gen(case)
    x = torch.randn(T, 2 * D, generator=g).to(dtype)
    w = torch.randn(D, W, generator=g)
    bias = torch.randn(D, generator=g) if case % 2 else None
    pool = torch.randn(N + 2, W - 1, D, generator=g).to(dtype)
    slots = torch.randperm(N + 2, generator=g)[:N].int()
    has = (torch.rand(N, generator=g) < 0.5).int()
    if N > 2:
        slots[1] = -1
    init = torch.where((has.bool() & (slots >= 0))[:, None, None], pool[slots.long().clamp(min=0)], torch.zeros((), dtype=dtype))
    ref, tol, ends = _conv_ref(x[:, D:], w, bias, lens, init, silu)
    cu = _i32([0] + torch.tensor(lens).cumsum(0).tolist())
    want = pool.clone()
    for n in range(N):
        if slots[n] >= 0:
            want[slots[n]] = ends[n]
    for pad in (3, 16, 2):                           # rows at odd places, whole 16-byte parts, and pairs
        st = pool.cuda()
        out = torch.full((T + 1, D + pad), 7.0, dtype=dtype, device="cuda")
        ops.causal_conv(x.cuda()[:, D:], w.cuda(), None if bias is None else bias.cuda(), state=st, cu_seqlens=cu,
                        slots=slots.cuda(), has_state=has.cuda(), silu=silu, out=out[:T, :D])
        _held(out[:T, :D], ref, tol, dtype == torch.bfloat16)
        assert bool((out[T:] == 7).all()) and bool((out[:, D:] == 7).all())
        assert torch.equal(st.cpu(), want)
    ops.check_errors()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,W", [(64, 4), (37, 3), (1, 2)])
def test_conv_steps_continue_a_prompt(dtype, D, W):
    g = _gen(D)
    x, w, bias = torch.randn(9, D, generator=g).to(dtype).cuda(), torch.randn(D, W, generator=g).cuda(), torch.randn(D, generator=g).cuda()
    whole = ops.causal_conv(x, w, bias)
    st = torch.zeros(3, W - 1, D, dtype=dtype, device="cuda")
    first = ops.causal_conv(x[:4], w, bias, state=st, slots=_i32([1]))
    pads = st.clone()
    rows = [ops.causal_conv_step(torch.cat([x[i:i + 1], x[:1]]), w, st, bias, slots=_i32([1, -1])) for i in range(4, 9)]
    assert torch.equal(torch.cat([first] + [r[:1] for r in rows]), whole)
    assert all(bool((r[1] == 0).all()) for r in rows)
    assert torch.equal(st[0], pads[0]) and torch.equal(st[2], pads[2])
    assert torch.equal(st[1], x[9 - (W - 1):])


# ---------------------------------------------------------------------------------- selective scan
def _scan_ref(x, dt, A, B, C, D, z, bias, softplus, lens, init):
    """-> out, its tolerance, states [n, d, N], their tolerance (both but for the output's own rounding)."""
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
            b, c = B[t].double()[per], C[t].double()[per]
            inp = (delta[t] * x64[t])[:, None] * b
            eg = (ed[t] + 3 * U * delta[t].abs())[:, None] * A.abs()
            own = torch.where(g.abs() <= 0.0999, 5 * U * torch.expm1(g).abs(), 6 * U * torch.maximum(torch.exp(g), torch.ones(())))
            a = torch.exp(g)
            e = a * e + (a * eg + own) * h.abs() + 2 * U * (2 * h.abs() + inp.abs()) + \
                inp.abs() * 2 * U + (ed[t] * x64[t].abs())[:, None] * b.abs()
            h = a * h + inp
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


SCANS = [  # lens, channels, states, groups
    ([1], 8, 16, 1),
    ([0, 1, 2, 0, 31, 32, 33, 5, 0], 72, 16, 1),
    ([64, 65, 1, 127], 136, 16, 2),
    ([200, 3], 33, 5, 1),
    ([17, 40], 20, 64, 4),
    ([9, 0, 12], 6, 200, 3),
    ([70], 96, 1, 1),
    ([3, 50], 65, 24, 1),
    ([700], 32, 8, 1),
    ([1, 2, 1, 0, 3, 1, 1, 4, 2, 1] * 3, 40, 16, 1),
    ([90, 300, 7, 200], 64, 16, 1),
    ([260, 40], 48, 32, 2),
]


def _scan_inputs(seed, T, d, n, groups, dtype, gate=True):
    g = _gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    A = -torch.arange(1, n + 1) * torch.exp(0.3 * r(d, n))
    step = torch.exp(math.log(1e-3) + torch.rand(d, generator=g) * math.log(300.0))
    return dict(x=r(T, d).to(dtype), dt=r(T, d).to(dtype), A=A, B=r(T, groups, n).to(dtype), C=r(T, groups, n).to(dtype),
                D=r(d), z=r(T, 2 * d).to(dtype)[:, d:] if gate else None, bias=step + torch.log(-torch.expm1(-step)))


def _dev(v):
    return None if v is None else v.cuda()


@gpu
@pytest.mark.parametrize("case", range(len(SCANS)))
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("softplus", [True, False])
def test_scan_matches_the_recurrence(case, dtype, softplus):
    lens, d, n, groups = SCANS[case]
    T, N = sum(lens), len(lens)
    i = _scan_inputs(case, T, d, n, groups, dtype, gate=case % 3 != 1)
    if not softplus:
        i["dt"], i["bias"] = (i["dt"].float().abs() * 0.05).to(dtype), None
    if case % 4 == 3:
        i["D"] = None
    g = _gen(50 + case)
    pool = torch.randn(N + 2, d, n, generator=g)
    slots = torch.randperm(N + 2, generator=g)[:N].int()
    has = (torch.rand(N, generator=g) < 0.6).int()
    if N > 2:
        slots[2] = -1
    init = torch.where((has.bool() & (slots >= 0))[:, None, None], pool[slots.long().clamp(min=0)], torch.zeros(()))
    ref, tol, ends, etol = _scan_ref(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], i["z"], i["bias"], softplus, lens, init)
    b = i["B"][:, 0] if groups == 1 else i["B"]
    free = [s for s in range(N + 2) if s not in slots.tolist()]
    for pad in (1, 16):                              # rows at odd places, and whole 16-byte parts where d allows them
        st, out = pool.cuda(), torch.full((T + 1, d + pad), 7.0, dtype=dtype, device="cuda")
        ops.selective_scan(i["x"].cuda(), i["dt"].cuda(), i["A"].cuda(), b.cuda(), i["C"].cuda(), D=_dev(i["D"]), z=_dev(i["z"]),
                           dt_bias=_dev(i["bias"]), softplus=softplus, state=st, slots=slots.cuda(), has_state=has.cuda(),
                           cu_seqlens=_i32([0] + torch.tensor(lens).cumsum(0).tolist()), out=out[:T, :d])
        _held(out[:T, :d], ref, tol, dtype == torch.bfloat16)
        assert bool((out[T:] == 7).all()) and bool((out[:, d:] == 7).all())
        st = st.cpu()
        for k in range(N):
            if slots[k] >= 0:
                _held(st[slots[k]], ends[k], etol[k], False)
        assert torch.equal(st[free], pool[free])
    ops.check_errors()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,n,groups", [(64, 16, 1), (37, 5, 1), (12, 64, 3), (5, 130, 1)])
def test_scan_steps_continue_a_prompt(dtype, d, n, groups):
    i = _scan_inputs(d, 9, d, n, groups, dtype)
    ref, tol, ends, etol = _scan_ref(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], i["z"], i["bias"], True, [9],
                                     torch.zeros(1, d, n))
    c = {k: v.cuda() for k, v in i.items()}
    kw = dict(D=c["D"], dt_bias=c["bias"])
    st = torch.full((3, d, n), 5.0, device="cuda")
    rows = [ops.selective_scan(c["x"][:4], c["dt"][:4], c["A"], c["B"][:4], c["C"][:4], z=c["z"][:4], state=st, slots=_i32([1]), **kw)]
    for t in range(4, 9):
        two = lambda k: torch.cat([c[k][t:t + 1], c[k][:1]])
        o = ops.selective_scan_step(two("x"), two("dt"), c["A"], two("B"), two("C"), st, z=two("z"), slots=_i32([1, -1]), **kw)
        assert bool((o[1] == 0).all())
        rows.append(o[:1])
    _held(torch.cat(rows), ref, tol, dtype == torch.bfloat16)
    _held(st[1], ends[0], etol[0], False)
    assert bool((st[0] == 5).all()) and bool((st[2] == 5).all())


@gpu
def test_scan_keeps_slow_states():
    """One constant step per channel, so a wrong rate adds up the same way at every token: 4000 tokens of memory."""
    T, d, n = 4000, 16, 4
    i = _scan_inputs(3, T, d, n, 1, torch.float32, gate=False)
    i["A"] = -torch.exp2(-torch.arange(d * n) / 5.0).view(d, n)
    i["dt"] = torch.full((T, d), 1.1e-3)
    ref, tol, ends, etol = _scan_ref(i["x"], i["dt"], i["A"], i["B"], i["C"], None, None, None, False, [T], torch.zeros(1, d, n))
    st = torch.zeros(1, d, n, device="cuda")
    out = ops.selective_scan(*(i[k].cuda() for k in ("x", "dt", "A", "B", "C")), softplus=False, state=st)
    _held(out, ref, tol, False)
    _held(st[0], ends[0], etol[0], False)


# ---------------------------------------------------------------------------------- sequences, streams, graphs
def _calls(T, d, dtype=torch.bfloat16, seed=0):
    """One convolution and one scan over the same batch: -> function of (cu, slots, has, conv state, scan state, out0, out1)."""
    i = {k: _dev(v) for k, v in _scan_inputs(seed, T, d, 16, 1, dtype).items()}
    w = torch.randn(d, 4, generator=_gen(seed + 1)).cuda()

    def run(cu, slots, has, cs, ss, o0=None, o1=None, x=None, err=None):
        x = i["x"] if x is None else x
        a = ops.causal_conv(x, w, state=cs, cu_seqlens=cu, slots=slots, has_state=has, out=o0, err=err)
        b = ops.selective_scan(x, i["dt"], i["A"], i["B"], i["C"], D=i["D"], z=i["z"], dt_bias=i["bias"], state=ss,
                               cu_seqlens=cu, slots=slots, has_state=has, out=o1, err=err)
        return a, b
    run.i = i
    return run


@gpu
def test_bad_offsets_and_rows_are_reported():
    T, d = 100, 40
    run = _calls(T, d)
    whole = [run(_i32([0, 30, 70, 100]), None, None, None, None)][0]
    for cu, slots, ok in (([0, 30, 20, 100], [0, 1, 2], [0]), ([0, 30, 101, 100], [0, 1, 2], [0]), ([0, 30, 70, 200], [0, 1, 2], [0, 1]),
                          ([-5, 30, 70, 100], [0, 1, 2], [1, 2]), ([0, 30, 70, 100], [0, 9, -7], [0, 1, 2])):
        cs, ss = torch.ones(4, 3, d, dtype=torch.bfloat16, device="cuda"), torch.ones(4, d, 16, device="cuda")
        o = [torch.full((T, d), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        run(_i32(cu), _i32(slots), _i32([0, 0, 0]), cs, ss, *o, err=err)
        assert int(err) == 1
        edges = [0, 30, 70, 100]
        for n in ok:                                  # sound sequences are as if alone
            for a, b in zip(o, whole):
                assert torch.equal(a[edges[n]:edges[n + 1]], b[edges[n]:edges[n + 1]])
        assert bool((cs[3] == 1).all()) and bool((ss[3] == 1).all())
        for n in range(3):
            if n not in ok and not (n == 2 and cu[2:] == [20, 100]):
                assert bool((cs[n] == 1).all()) and bool((ss[n] == 1).all())


@gpu
def test_no_sequences_and_no_tokens():
    d = 24
    run = _calls(1, d)
    x0 = torch.empty(0, d, dtype=torch.bfloat16, device="cuda")
    w, A, bc = torch.ones(d, 4, device="cuda"), -torch.ones(d, 16, device="cuda"), torch.empty(0, 16, dtype=torch.bfloat16, device="cuda")
    cs, ss = torch.ones(2, 3, d, dtype=torch.bfloat16, device="cuda"), torch.ones(2, d, 16, device="cuda")
    for cu, has, kept in ((_i32([0]), None, (1, 1)), (_i32([0, 0, 0]), _i32([1, 0]), (1, 0))):
        assert ops.causal_conv(x0, w, state=cs, cu_seqlens=cu, has_state=has).shape == (0, d)
        assert ops.selective_scan(x0, x0, A, bc, bc, state=ss, cu_seqlens=cu, has_state=has).shape == (0, d)
        for st in (cs, ss):                           # an empty sequence keeps its state, or starts it from zeros
            assert [float(r.float().mean()) for r in st] == list(kept)
    assert ops.causal_conv_step(x0, w, cs).shape == (0, d) and ops.selective_scan_step(x0, x0, A, bc, bc, ss).shape == (0, d)
    # tokens outside every sequence are not written
    o = [torch.full((1, d), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    run(_i32([0, 0]), None, None, None, None, *o)
    run(_i32([1, 1]), None, None, None, None, *o)
    assert all(bool((t == 7).all()) for t in o)


@gpu
def test_nan_stays_in_its_sequence_and_after_its_token():
    T, d = 90, 16
    run = _calls(T, d)
    cu = _i32([0, 40, 90])
    clean = run(cu, None, None, None, None)
    x = run.i["x"].clone()
    x[20, 3] = math.nan
    x[60, 5] = math.inf
    cs, ss = torch.zeros(2, 3, d, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, d, 16, device="cuda")
    dirty = run(cu, None, None, cs, ss, x=x)
    for a, b, reach in zip(clean, dirty, (4, 100)):
        same = torch.ones(T, d, dtype=torch.bool, device="cuda")
        same[20:min(40, 20 + reach), 3] = False
        same[60:min(90, 60 + reach), 5] = False
        assert torch.equal(a[same], b[same])
        assert bool(torch.isnan(b[20, 3])) and not bool(torch.isfinite(b[60, 5]))
    assert bool(torch.isnan(ss[0, 3]).all()) and bool(torch.isfinite(ss[0, :3]).all()) and bool(torch.isfinite(ss[1, 6:]).all())


@gpu
def test_other_streams_graphs_and_two_calls_at_once():
    T, d = 1500, 96
    run = _calls(T, d)
    cu, slots, has = _i32([0, 400, 401, 1500]), _i32([2, 0, 1]), _i32([1, 0, 1])
    st = lambda: (torch.ones(3, 3, d, dtype=torch.bfloat16, device="cuda"), torch.ones(3, d, 16, device="cuda"))
    s0 = st()
    want = run(cu, slots, has, *s0)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    s1, s2 = st(), st()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        a = run(cu, slots, has, *s1)
    with torch.cuda.stream(other):
        b = run(cu, slots, has, *s2)
    torch.cuda.synchronize()
    for got, stt in ((a, s1), (b, s2)):
        assert all(torch.equal(p, q) for p, q in zip(got, want)) and all(torch.equal(p, q) for p, q in zip(stt, s0))
    # two graphs that share nothing but the inputs, replayed at once
    graphs, keep = [], []
    for _ in range(2):
        s = st()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o = run(cu, slots, has, *s)
        graphs.append(gr)
        keep.append((s, o))
    torch.cuda.synchronize()
    for gr, stream in zip(graphs, (side, other)):
        with torch.cuda.stream(stream):
            gr.replay()
    torch.cuda.synchronize()
    for s, o in keep:
        assert all(torch.equal(p, q) for p, q in zip(o, want)) and all(torch.equal(p, q) for p, q in zip(s, s0))


def _shifted(t):
    """The same values one element further into a buffer: aligned to single elements only."""
    b = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
    b[1:] = t.reshape(-1)
    return b[1:].view(t.shape)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,d,n,W", [(40, 32, 16, 4), (90, 64, 8, 2), (7, 24, 64, 3)])
def test_operands_at_odd_addresses(dtype, T, d, n, W):
    i = _scan_inputs(T, T, d, n, 1, dtype)
    i["z"] = i["z"].contiguous()
    w, b = torch.randn(d, W, generator=_gen(1)), torch.randn(d, generator=_gen(2))
    zeros = torch.zeros(1, W - 1, d, dtype=dtype)
    ref, tol, ends = _conv_ref(i["x"], w, b, [T], zeros, True)
    sref, stol, sends, setol = _scan_ref(i["x"], i["dt"], i["A"], i["B"], i["C"], i["D"], i["z"], i["bias"], True, [T], torch.zeros(1, d, n))
    c = {k: _shifted(v.cuda()) for k, v in i.items()}
    cs, ss = _shifted(zeros.cuda()), _shifted(torch.zeros(1, d, n, device="cuda"))
    out = ops.causal_conv(c["x"], _shifted(w.cuda()), _shifted(b.cuda()), state=cs)
    _held(out, ref, tol, dtype == torch.bfloat16)
    assert torch.equal(cs.cpu(), ends)
    kw = dict(D=c["D"], z=c["z"], dt_bias=c["bias"])
    out = ops.selective_scan(c["x"], c["dt"], c["A"], c["B"][:, 0], c["C"], state=ss, **kw)
    _held(out, sref, stol, dtype == torch.bfloat16)
    _held(ss[0], sends[0], setol[0], False)
    # the same tokens one by one
    cs.zero_()
    ss.zero_()
    rows = lambda t, k: _shifted(c[k][t:t + 1])
    for t in range(T):
        o = ops.causal_conv_step(rows(t, "x"), _shifted(w.cuda()), cs, _shifted(b.cuda()))
        _held(o, ref[t:t + 1], tol[t:t + 1], dtype == torch.bfloat16)
        kw = dict(D=c["D"], z=rows(t, "z"), dt_bias=c["bias"])
        o = ops.selective_scan_step(rows(t, "x"), rows(t, "dt"), c["A"], rows(t, "B"), rows(t, "C"), ss, **kw)
        _held(o, sref[t:t + 1], stol[t:t + 1], dtype == torch.bfloat16)
    _held(ss[0], sends[0], setol[0], False)
    y, wt = c["x"], _shifted(b.cuda())
    ref, tol, rr, rtol = _norm_ref(i["x"], b, 1e-5, i["z"].float(), b, i["dt"], "silu", 0.5, 1.0)
    res = _shifted(i["z"].float().cuda())
    o, r = ops.block_norm(y, wt, 1e-5, residual=res, post_weight=wt, gate=c["dt"], scale=0.5, w_offset=1.0)
    _held(o, ref, tol, True)
    _held(r, rr, rtol, False)


@gpu
def test_offsets_past_32_bits():
    rows, d, far = 3, 16, (1 << 31) // 2 + 64          # rows 2^30 elements apart: the last one past 2^31
    big = torch.empty(rows * far, dtype=torch.bfloat16, device="cuda")
    i = {k: _dev(v) for k, v in _scan_inputs(0, rows, d, 16, 1, torch.bfloat16).items()}
    w = torch.randn(d, 4, generator=_gen(5)).cuda()
    x = big.as_strided((rows, d), (far, 1))
    x.copy_(i["x"])
    o = big.as_strided((rows, d), (far, 1), 64)
    args = (i["dt"], i["A"], i["B"], i["C"])
    assert torch.equal(ops.causal_conv(x, w, out=o), ops.causal_conv(i["x"], w))
    assert torch.equal(ops.selective_scan(x, *args, out=o), ops.selective_scan(i["x"], *args))
    del big, x, o
    slot = (1 << 31) // (4096 * 16) + 3                # a pool of more than 2^31 states
    pool = torch.zeros(slot + 1, 4096, 16, device="cuda")
    one = {k: _dev(v) for k, v in _scan_inputs(1, 1, 4096, 16, 1, torch.bfloat16).items()}
    small = torch.zeros(1, 4096, 16, device="cuda")
    for s, st in ((slot, pool), (0, small)):
        ops.selective_scan_step(one["x"], one["dt"], one["A"], one["B"], one["C"], st, slots=_i32([s]))
    assert torch.equal(pool[slot], small[0])


# ---------------------------------------------------------------------------------- block norm
def _norm_ref(y, w, eps, resid, post, gate, act, scale, off):
    h, e, K = y.double(), torch.zeros_like(y, dtype=torch.float64), y.shape[1]
    rms = (K / 64 + 24) * U          # relative: a sum in strides and a tree, a fast square root and its product
    if post is not None:
        p = post.double() + off
        h = h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * p
        e = h.abs() * (rms + 4 * U) + U * (h / p).abs() * (post.double().abs() + abs(off))
    if gate is not None:
        q = gate.double()
        f = {"silu": _silu(q), "sigmoid": torch.sigmoid(q), "none": q}[act]
        h, e = h * f, e * f.abs() * 1.001 + (h * f).abs() * ((2 * q.abs() + 12) * U)
    s = scale.double() if isinstance(scale, torch.Tensor) else scale
    r = s * h + (resid.double() if resid is not None else 0)
    er = abs(s) * e + 3 * U * (abs(s) * h.abs() + r.abs())
    if w is None:
        return r, er, r, er
    inv = 1 / (r.square().mean(-1, keepdim=True) + eps).sqrt()
    n = r * inv * (w.double() + off)
    # the norm of r + er: the row's own error and, through 1 / rms, at most the largest relative error of the mean
    through = ((r.abs() * er).mean(-1, keepdim=True) + 1e-300) * inv ** 2
    return n, er * inv * (w.double() + off).abs() + n.abs() * (rms + 6 * U + through) + U * (r * inv).abs() * (w.double().abs() + abs(off)), r, er


NORMS = [  # T, K, residual, post, gate, act, scale, offset, weight
    (1, 4096, torch.float32, False, "", "silu", 1.0, 0.0, True),
    (3, 8, torch.float32, True, "rows", "silu", 0.5, 1.0, True),
    (5, 257, torch.bfloat16, True, "row", "sigmoid", "row", 0.0, True),
    (70, 2048, torch.bfloat16, False, "rows", "none", 0.25, 1.0, True),
    (4, 1000, None, True, "rows", "silu", 1.0, 0.0, False),
    (4, 1000, None, False, "rows", "silu", 1.0, 0.0, True),
    (3, 32768, torch.float32, True, "rows", "sigmoid", 1.0, 1.0, True),
    (3, 12289, torch.float32, True, "", "silu", "row", 1.0, True),
    (6, 1, torch.float32, True, "rows", "silu", 1.0, 0.0, True),
    (3000, 264, torch.float32, False, "", "silu", 1.0, 0.0, True),
    (2, 6000, torch.float32, False, "", "silu", 1.0, 0.0, False),
    (7, 2050, torch.bfloat16, True, "rows", "silu", 0.5, 1.0, True),
    (500, 3000, torch.float32, True, "rows", "silu", "row", 1.0, True),      # more rows than blocks
    (160, 8192, torch.bfloat16, True, "row", "sigmoid", 0.22, 0.0, True),
    (5000, 96, torch.float32, True, "rows", "none", 1.0, 1.0, True),
    (2500, 1000, torch.float32, False, "row", "silu", 1.0, 0.0, True),
    (1300, 2044, torch.float32, True, "", "silu", 0.5, 0.0, False),
]


@gpu
@pytest.mark.parametrize("case", range(len(NORMS)))
@pytest.mark.parametrize("dtype", TYPES)
def test_block_norm(case, dtype):
    T, K, rt, post, gate, act, scale, off, weight = NORMS[case]
    g = _gen(case)
    r = lambda *s: torch.randn(*s, generator=g)
    y = r(T, 2 * K).to(dtype)[:, :K]
    resid = None if rt is None else (3 * r(T, K)).to(rt)
    w, p = (1 + 0.2 * r(K) - off if on else None for on in (weight, post))
    gt = {"": None, "rows": r(T, K).to(dtype), "row": r(K).to(dtype)}[gate]
    sc = r(K) if scale == "row" else scale
    ref, tol, rr, rtol = _norm_ref(y, w, 1e-5, resid, p, gt, act, sc, off)
    store = torch.full((T + 1, K + 5), 7.0, dtype=torch.float32 if case % 2 else torch.bfloat16, device="cuda")
    res = _dev(resid)
    out, ro = ops.block_norm(y.cuda(), _dev(w), 1e-5, residual=res, post_weight=_dev(p), gate=_dev(gt), gate_act=act,
                             scale=_dev(sc) if scale == "row" else scale, w_offset=off, out=store[:T, :K])
    _held(out, ref, tol, out.dtype == torch.bfloat16)
    assert bool((store[T:] == 7).all()) and bool((store[:, K:] == 7).all())
    assert ro is res
    if res is not None:
        _held(res, rr, rtol, rt == torch.bfloat16)
        # into another buffer: the residual stays
        keep, other = _dev(resid), torch.empty(T, K, dtype=rt, device="cuda")
        out, _ = ops.block_norm(y.cuda(), _dev(w), 1e-5, residual=keep, post_weight=_dev(p), gate=_dev(gt), gate_act=act,
                                scale=_dev(sc) if scale == "row" else scale, w_offset=off, resid_out=other)
        assert torch.equal(keep.cpu(), resid)
        _held(other, rr, rtol, rt == torch.bfloat16)
        if weight:
            _held(out, ref, tol, True)


@gpu
def test_block_norm_edges():
    z = torch.zeros(2, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    out, r = ops.block_norm(z, w, 1e-6, residual=z.clone(), post_weight=w)
    assert bool((out == 0).all()) and bool((r == 0).all())
    y = torch.randn(3, 64, generator=_gen(0)).cuda()
    y[1, 5] = math.nan
    out, _ = ops.block_norm(y, w, 1e-6, gate=y)
    assert bool(torch.isnan(out[1]).all()) and bool(torch.isfinite(out[[0, 2]]).all())
    assert ops.block_norm(y[:0], w, 1e-6)[0].shape == (0, 64)
    only, r = ops.block_norm(y[:1], None, 1e-6, residual=torch.ones(1, 64, device="cuda"))
    assert only is None and torch.equal(r, 1 + y[:1])


# ---------------------------------------------------------------------------------- token log probabilities
def _lp_check(logits, tokens, top, **kw):
    """Against 64 bits. u |x| of each logit's distance to the maximum enters its exponential, the log-sum-exp is off by
    that weighted with the probabilities, by the sums and by the logarithm."""
    x = logits.double().cpu()
    T, V = x.shape
    r = ops.token_logprobs(logits, tokens, top=top, **kw)
    m = x.amax(-1, keepdim=True)
    lse = torch.logsumexp(x, -1)
    p = torch.softmax(x, -1)
    dist = (m - x).clamp(max=200)
    dist[x == -math.inf] = 0
    spread = (p * dist).sum(-1)
    rel = (4 * spread + 12 + V / 128) * U                       # of the sum of exponentials
    tl = rel + 4 * U * (lse.abs() + m[:, 0].abs() + 1)
    lpx = x - lse[:, None]
    lpx[x == -math.inf] = -math.inf
    ent = -torch.where(p > 0, p * lpx, torch.zeros(())).sum(-1)
    te = rel * (2 + 2 * ent.abs() + 2 * spread) + tl + (p * dist * (4 * dist + 12 + V / 128) * U).sum(-1)
    empty = (x == -math.inf).all(-1)
    odd = torch.isnan(x).any(-1) | (x == math.inf).any(-1)
    ent[empty], lpx[empty] = 0.0, -math.inf
    ent[odd], lpx[odd] = math.nan, math.nan
    tl[empty | odd], te[empty | odd] = 0.0, 0.0
    tok = torch.full((T,), -1) if tokens is None else tokens.cpu().long()
    want = torch.where((tok >= 0) & (tok < V), lpx.gather(1, tok.clamp(0, V - 1)[:, None])[:, 0], torch.zeros(()).double())
    _held(r.logprobs, want, tl, False)
    _held(r.entropy, ent, te, False)
    assert r.top_ids.shape == r.top_logprobs.shape == (T, top)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    val = x.gather(1, order)
    ids = torch.where((val == -math.inf) | odd[:, None], -1, order)
    ids = torch.cat([ids, torch.full((T, max(0, top - V)), -1)], 1)
    assert torch.equal(r.top_ids.cpu().long(), ids)
    tops = torch.where(ids >= 0, lpx.gather(1, ids.clamp(min=0)), -math.inf)
    tops[odd] = math.nan
    _held(r.top_logprobs, tops, tl[:, None].expand(tops.shape), False)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,top", [(1, 1, 1), (1, 128256, 20), (3, 5, 8), (2, 4099, 32), (40, 50257, 5), (7, 32000, 0), (300, 1031, 20),
                                     (5, 2048, 1), (19, 70001, 32), (2, 262144, 20), (200, 9000, 3)])
def test_token_logprobs(dtype, T, V, top):
    g = _gen(V + T)
    x = (4 * torch.randn(T, V, generator=g)).to(dtype)
    tok = torch.randint(0, V, (T,), generator=g).int()
    tok[::3] = x.float().argmax(-1)[::3].int()
    tok[1::5] = -1
    wide = torch.zeros(T, V + 3, dtype=dtype, device="cuda")     # rows that start anywhere
    wide[:, 1:V + 1] = x.cuda()
    _lp_check(wide[:, 1:V + 1], tok.cuda(), top)
    _lp_check(x.cuda(), tok.cuda(), top)
    ops.check_errors()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [97, 5000, 128256])
def test_token_logprobs_rows_of_every_kind(dtype, V):
    g = _gen(V)
    low = torch.finfo(dtype).min
    x = 3 * torch.randn(16, V, generator=g)
    x[0] = 0.0                                       # all alike
    x[1] = -math.inf                                 # nothing allowed
    x[2, 5:] = -math.inf                             # five tokens left
    x[3, :-1] = low                                  # one, masked by the type's lowest value
    x[4] = low                                       # all of them that low: alike
    x[5, V // 2] = math.nan
    x[6, V - 1] = math.inf
    x[7] = torch.arange(V).float() / V               # rising
    x[8] = -torch.arange(V).float() / V              # falling
    x[9] = torch.randint(0, 2, (V,), generator=g).float()        # two values
    x[10] = -torch.zeros(V)
    x[10, ::2] = 0.0                                 # zeros of both signs are alike
    x[11, 7] = 80.0                                  # certain
    x[12] += 1e4                                     # far from zero
    x[13, ::8] = 50.0                                # every eighth alike and on top
    x[14] = -1e31                                    # huge and negative, one of them less so
    x[14, 3] = -1e30
    x[15, :] = -math.inf
    x[15, V - 1] = -3.0                              # one token
    x = x.to(dtype)
    tok = torch.randint(0, V, (16,), generator=g).int()
    tok[2], tok[11], tok[15], tok[14] = V - 1, 7, V - 1, 3
    for top in (0, 1, 20, 32):
        _lp_check(x.cuda(), tok.cuda(), top)
    _lp_check(x.cuda(), None, 2)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    bad = tok.clone()
    bad[0], bad[9] = V, -2
    _lp_check(x.cuda(), bad.cuda(), 1, err=err)
    assert int(err) == 1


@gpu
def test_token_logprobs_graph_streams_and_far_rows():
    x = torch.randn(33, 30000, generator=_gen(1)).cuda()
    tok = torch.arange(33, dtype=torch.int32, device="cuda")
    want = ops.token_logprobs(x, tok, top=7)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = ops.token_logprobs(x, tok, top=7)
    gr.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    big = torch.zeros(3, (1 << 30) + 8, dtype=torch.bfloat16, device="cuda")
    big[:, :1000] = x[:3, :1000]
    far = ops.token_logprobs(big[:, :1000], tok[:3], top=3)
    near = ops.token_logprobs(big[:, :1000].contiguous(), tok[:3], top=3)
    assert all(torch.equal(a, b) for a, b in zip(far, near))


# ---------------------------------------------------------------------------------- refusals (no GPU needed)
def _meta():
    f, h = torch.zeros(6, 8), torch.zeros(6, 8, dtype=torch.bfloat16)
    return f, h, torch.zeros(8, 4), torch.zeros(8, 16), torch.zeros(6, 16), torch.zeros(6, 3, 8), torch.zeros(6, 8, 16)


F, H, W4, A16, BC, CS, SS = _meta()
I3 = torch.zeros(3, dtype=torch.int32)
REFUSED = {
    "taps": (lambda: ops.causal_conv(F, torch.zeros(8, 5)), "taps"),
    "one tap": (lambda: ops.causal_conv(F, torch.zeros(8, 1)), "taps"),
    "w type": (lambda: ops.causal_conv(F, W4.bfloat16()), "w must"),
    "w channels": (lambda: ops.causal_conv(F, torch.zeros(7, 4)), "w must"),
    "x type": (lambda: ops.causal_conv(F.half(), W4), "x must"),
    "x columns": (lambda: ops.causal_conv(torch.zeros(8, 6).t(), W4), "contiguous"),
    "bias": (lambda: ops.causal_conv(F, W4, torch.zeros(7)), "bias"),
    "conv state type": (lambda: ops.causal_conv(H, W4, state=CS), "state"),
    "conv state rows": (lambda: ops.causal_conv(F, W4, state=CS[:, :2].contiguous()), "state"),
    "slots without state": (lambda: ops.causal_conv(F, W4, slots=I3[:1]), "slots"),
    "slots count": (lambda: ops.causal_conv(F, W4, state=CS, slots=I3), "slots"),
    "slots type": (lambda: ops.causal_conv(F, W4, state=CS, slots=I3[:1].long()), "slots"),
    "too few rows": (lambda: ops.causal_conv(F, W4, state=CS[:1], cu_seqlens=I3), "state rows"),
    "step rows": (lambda: ops.causal_conv_step(F, W4, CS[:5]), "state rows"),
    "out type": (lambda: ops.causal_conv(F, W4, out=H), "out must"),
    "out rows overlap": (lambda: ops.causal_conv(F, W4, out=torch.zeros(8).expand(6, 8)), "overlap"),
    "out is x": (lambda: ops.causal_conv(F, W4, out=F), "shares memory"),
    "out meets x": (lambda x=torch.zeros(6, 12): ops.causal_conv(x[:, :8], W4, out=x[:, 4:]), "shares memory"),
    "out meets x's next row": (lambda x=torch.zeros(8, 12): ops.causal_conv(x[1:7, :8], W4, out=x[:6, 10:].as_strided((6, 8), (12, 1))), "shares memory"),
    "out is the state": (lambda: ops.causal_conv(F, W4, state=CS, out=CS[:, 0]), "shares memory"),
    "conv on CPU": (lambda: ops.causal_conv(F, W4), "CUDA"),
    "parts of one projection": (lambda x=torch.zeros(6, 16): ops.causal_conv(x[:, :8], W4, out=x[:, 8:]), "CUDA"),
    "scan dt type": (lambda: ops.selective_scan(F, H, A16, BC, BC), "dt must"),
    "scan dt shape": (lambda: ops.selective_scan(F, F[:5], A16, BC, BC), "dt must"),
    "A type": (lambda: ops.selective_scan(F, F, A16.bfloat16(), BC, BC), "A must"),
    "states": (lambda: ops.selective_scan(F, F, torch.zeros(8, 257), BC, BC), "states"),
    "B states": (lambda: ops.selective_scan(F, F, A16, BC[:, :8], BC), "B and C"),
    "groups": (lambda: ops.selective_scan(F, F, A16, torch.zeros(6, 3, 16), torch.zeros(6, 3, 16)), "groups"),
    "groups differ": (lambda: ops.selective_scan(F, F, A16, torch.zeros(6, 2, 16), torch.zeros(6, 4, 16)), "groups"),
    "B type": (lambda: ops.selective_scan(F, F, A16, BC.bfloat16(), BC), "B must"),
    "z": (lambda: ops.selective_scan(F, F, A16, BC, BC, z=H), "z must"),
    "skip": (lambda: ops.selective_scan(F, F, A16, BC, BC, D=torch.zeros(9)), "D must"),
    "scan state": (lambda: ops.selective_scan(F, F, A16, BC, BC, state=SS.bfloat16()), "state"),
    "scan out is dt": (lambda d=torch.zeros(6, 8): ops.selective_scan(F, d, A16, BC, BC, out=d), "shares memory"),
    "scan step rows": (lambda: ops.selective_scan_step(F, F, A16, BC, BC, SS[:5]), "state rows"),
    "scan on CPU": (lambda: ops.selective_scan_step(F, F, A16, BC, BC, SS), "CUDA"),
    "norm y": (lambda: ops.block_norm(F[0], None, 1e-5), "y must"),
    "norm columns": (lambda: ops.block_norm(torch.zeros(1, 32769), None, 1e-5), "columns"),
    "norm weight": (lambda: ops.block_norm(F, torch.ones(7), 1e-5), "weight"),
    "norm weight type": (lambda: ops.block_norm(F, torch.ones(8).half(), 1e-5), "weight"),
    "norm gate type": (lambda: ops.block_norm(F, None, 1e-5, gate=H), "gate"),
    "norm gate shape": (lambda: ops.block_norm(F, None, 1e-5, gate=torch.zeros(4)), "gate"),
    "norm residual": (lambda: ops.block_norm(F, None, 1e-5, residual=F[:3]), "residual"),
    "norm out type": (lambda: ops.block_norm(F, None, 1e-5, residual=F, resid_out=torch.zeros(6, 8, dtype=torch.bfloat16)), "resid_out"),
    "norm out is y": (lambda: ops.block_norm(F, torch.ones(8), 1e-5, out=F), "shares memory"),
    "norm out is the residual": (lambda r=torch.zeros(6, 8): ops.block_norm(F, torch.ones(8), 1e-5, residual=r, out=r), "shares memory"),
    "norm residual shifted": (lambda r=torch.zeros(7, 8): ops.block_norm(F, None, 1e-5, residual=r[:6], resid_out=r[1:]), "shares memory"),
    "norm scale": (lambda: ops.block_norm(F, None, 1e-5, scale=torch.ones(3)), "scale"),
    "norm on CPU": (lambda r=torch.zeros(6, 8): ops.block_norm(F, torch.ones(8), 1e-5, residual=r), "CUDA"),
    "alternatives": (lambda: ops.token_logprobs(F, top=33), "alternatives"),
    "fewer than none": (lambda: ops.token_logprobs(F, top=-1), "alternatives"),
    "token type": (lambda: ops.token_logprobs(F, torch.zeros(6, dtype=torch.int64)), "tokens"),
    "token count": (lambda: ops.token_logprobs(F, I3), "tokens"),
    "no vocabulary": (lambda: ops.token_logprobs(torch.zeros(3, 0)), "vocabulary"),
    "logits type": (lambda: ops.token_logprobs(F.double()), "logits must"),
    "logits on CPU": (lambda: ops.token_logprobs(F), "CUDA"),
}


@pytest.mark.parametrize("name", REFUSED)
def test_refused(name):
    if not ops.ext_available():
        pytest.skip("extension not built")
    call, text = REFUSED[name]
    with pytest.raises(RuntimeError, match=text):
        call()


def test_gate_names():
    with pytest.raises(ValueError, match="gate_act"):
        ops.block_norm(F, None, 1e-5, gate_act="tanh")
