"""Operators of a recurrent decoder's serving step against their definitions in 64 bits.

Tolerances. u = 2^-24 is the rounding of f32 (24 significant bits), b = 2^-8 of bf16 (8). A sum of n rounded terms is off by
at most (n + 1) u times the sum of the terms' magnitudes, so outputs are held to a multiple of the
same recurrence run on magnitudes (`mag` below), plus b |o| where the output is rounded to bf16. A
decay product exp(g_1 + ... + g_n) formed from a rounded sum is off by n u |g_1 + ... + g_n|
relatively; terms whose exponent sum passes ln(mag / tiny) vanish, which bounds the sum by 104. The
block form of bf16 prompts rounds the decayed scores and the incoming state once to bf16: 2 b of mag
more on the outputs (not on the state).
"""
import math

import pytest
import torch

from air_rs import ops

U, BF = 2.0 ** -24, 2.0 ** -8
DEV = "cuda"
gpu = pytest.mark.gpu


def _oracle(q, k, v, g, lens, init, scale):
    """q, k [T, Hx, dk], v, g [T, H] -> (out, states) and the same recurrence on magnitudes, f64."""
    H = g.shape[1]
    q, k, v = (x.double().repeat_interleave(H // x.shape[1], 1) for x in (q, k, v))
    out = torch.zeros(q.shape[0], H, v.shape[2], dtype=torch.float64)
    mag = torch.zeros_like(out)
    st, sm = init.double().clone(), init.double().abs()
    t = 0
    for n, L in enumerate(lens):
        for _ in range(L):
            a = g[t].double().exp()[:, None, None]
            st[n] = a * st[n] + v[t][:, :, None] * k[t][:, None, :]
            sm[n] = a * sm[n] + v[t][:, :, None].abs() * k[t][:, None, :].abs()
            out[t] = scale * torch.einsum("hvk,hk->hv", st[n], q[t])
            mag[t] = abs(scale) * torch.einsum("hvk,hk->hv", sm[n], q[t].abs())
            t += 1
    return out, st, mag, sm


def _inputs(seed, T, H, Hq, Hk, Hv, dk, dv, dtype, per_token=True, strong=False):
    r = torch.Generator().manual_seed(seed)
    q = torch.randn(T, Hq, dk, generator=r).to(dtype)
    k = (torch.randn(T, Hk, dk, generator=r) * dk ** -0.5).to(dtype)
    v = torch.randn(T, Hv, dv, generator=r).to(dtype)
    rate = torch.exp2(-6.0 * torch.arange(H) / H) * (3.0 if strong else 0.3)
    g = -rate * torch.rand(T, H, generator=r) if per_token else (-rate).expand(T, H).contiguous()
    return q, k, v, g


def _near(got, ref, mag, c, rounded):
    tol = c * mag + (BF * 1.01 * ref.abs() if rounded else 0) + 1e-30
    over = (got.double().cpu() - ref).abs() - tol
    assert bool((over <= 0).all()), f"{float(over.max()):.3g} over the bound, worst ratio {float(((got.double().cpu() - ref).abs() / tol).max()):.3g}"


def _c(L, dk, blocks):
    """(output, state) multiples of mag for sequences of up to L tokens."""
    base = (2 * L + dk + 16 + 128 * 104) * U
    return (base + (2 * BF * 1.01 if blocks else 0)), base


def _blocks(dtype, dk, dv):
    return dtype == torch.bfloat16 and dk in (64, 128) and dv in (64, 128)


# ---------------------------------------------------------------------------------- prompts
PROMPTS = [  # lens, H, Hq, Hk, Hv, dk, dv
    ([1], 2, 2, 2, 2, 128, 128),
    ([0, 1, 2, 0, 127, 128, 129, 0], 4, 4, 4, 4, 128, 128),
    ([300, 5, 257], 4, 2, 2, 4, 128, 64),
    ([70, 64, 190], 4, 1, 2, 4, 64, 64),
    ([33, 512], 2, 2, 1, 1, 64, 128),
    ([19, 3], 3, 3, 1, 3, 48, 40),
    ([7, 40], 2, 2, 2, 2, 256, 24),
    ([9], 1, 1, 1, 1, 1, 1),
]


@gpu
@pytest.mark.parametrize("case", range(len(PROMPTS)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("per_token", [True, False])
def test_prompts_match_the_recurrence(case, dtype, per_token):
    lens, H, Hq, Hk, Hv, dk, dv = PROMPTS[case]
    T, N = sum(lens), len(lens)
    q, k, v, g = _inputs(case, T, H, Hq, Hk, Hv, dk, dv, dtype, per_token)
    r = torch.Generator().manual_seed(100 + case)
    S = N + 3
    pool = torch.randn(S, H, dv, dk, generator=r)
    slots = torch.randperm(S, generator=r)[:N]
    has = torch.tensor([i % 3 != 0 for i in range(N)])
    init = pool[slots] * has[:, None, None, None]
    scale = dk ** -0.5
    ref, st, mag, sm = _oracle(q, k, v, g, lens, init, scale)
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32)
    dpool = pool.to(DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = ops.linear_attention(q.to(DEV), k.to(DEV), v.to(DEV), (g if per_token else g[0]).to(DEV), state=dpool,
                               cu_seqlens=cu.to(DEV), slots=slots.to(torch.int32).to(DEV),
                               has_state=has.to(torch.int32).to(DEV), err=err)
    assert int(err) == 0 and out.dtype == dtype and out.shape == (T, H, dv)
    co, cs = _c(max(lens), dk, _blocks(dtype, dk, dv))
    _near(out, ref, mag, co, dtype == torch.bfloat16)
    _near(dpool[slots.to(DEV)], st, sm, cs, False)
    rest = torch.ones(S, dtype=torch.bool)
    rest[slots] = False
    assert torch.equal(dpool.cpu()[rest], pool[rest])


@gpu
@pytest.mark.parametrize("N", [32, 33, 70])
def test_many_sequences_in_one_call(N):
    """More sequences than a warp has lanes, empty ones among them, with and without one that is long
    enough to be split."""
    H, d = 3, 64
    r = torch.Generator().manual_seed(N)
    lens = torch.randint(0, 90, (N,), generator=r).tolist()
    lens[5] = lens[-1] = 0
    if N == 70:
        lens[40] = 2900
    T = sum(lens)
    q, k, v, g = _inputs(N, T, H, H, H, H, d, d, torch.bfloat16)
    pool = torch.randn(N, H, d, d, generator=r)
    has = torch.randint(0, 2, (N,), generator=r)
    ref, st, mag, sm = _oracle(q, k, v, g, lens, pool * has[:, None, None, None], 0.125)
    dpool = pool.to(DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=DEV)
    out = ops.linear_attention(q.to(DEV), k.to(DEV), v.to(DEV), g.to(DEV), state=dpool, cu_seqlens=cu,
                               has_state=has.to(torch.int32).to(DEV), err=err)
    assert int(err) == 0
    co, cs = _c(max(lens), d, True)
    _near(out, ref, mag, co, True)
    _near(dpool, st, sm, cs, False)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompt_without_state_and_defaults(dtype):
    q, k, v, g = _inputs(5, 200, 2, 2, 2, 2, 64, 64, dtype)
    ref, _, mag, _ = _oracle(q, k, v, g, [200], torch.zeros(1, 2, 64, 64), 0.125)
    out = ops.linear_attention(q.to(DEV), k.to(DEV), v.to(DEV), g.to(DEV))
    _near(out, ref, mag, _c(200, 64, dtype == torch.bfloat16)[0], dtype == torch.bfloat16)
    # scale and a caller's output rows, with room between the heads
    buf = torch.full((200, 2, 80), 7.0, dtype=dtype, device=DEV)
    ops.linear_attention(q.to(DEV), k.to(DEV), v.to(DEV), g.to(DEV), scale=-2.0, out=buf[..., :64])
    _near(buf[..., :64], ref * -16, mag * 16, _c(200, 64, dtype == torch.bfloat16)[0], dtype == torch.bfloat16)
    assert bool((buf[..., 64:] == 7).all())


@gpu
@pytest.mark.parametrize("offset", [0, 8, 3])
def test_prompt_operands_are_slices_of_one_projection(offset):
    """q | k | v columns of a fused projection, starting at an aligned or unaligned column."""
    T, H, d = 150, 3, 64
    r = torch.Generator().manual_seed(offset)
    fused = torch.randn(T, offset + 3 * H * d + 8, generator=r).to(torch.bfloat16)
    part = lambda f, i: f[:, offset + i * H * d: offset + (i + 1) * H * d].unflatten(1, (H, d))
    _, _, _, g = _inputs(1, T, H, H, H, H, d, d, torch.bfloat16)
    ref, _, mag, _ = _oracle(part(fused, 0), part(fused, 1), part(fused, 2), g, [T], torch.zeros(1, H, d, d), 1.0)
    f = fused.to(DEV)
    gg = torch.randn(T, H + 5, device=DEV)
    gg[:, 2:2 + H] = g.to(DEV)
    out = ops.linear_attention(part(f, 0), part(f, 1), part(f, 2), gg[:, 2:2 + H], scale=1.0)
    _near(out, ref, mag, _c(T, d, True)[0], True)
    # the same operands with the heads outermost in memory
    hm = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)
    out2 = ops.linear_attention(hm(part(f, 0)), hm(part(f, 1)), hm(part(f, 2)), gg[:, 2:2 + H], scale=1.0)
    _near(out2, ref, mag, _c(T, d, True)[0], True)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompt_decay_that_forgets_everything(dtype):
    """-inf and very strong decays in the middle of a block, at its first and last token, and twice
    in a row; the tokens after them have weak decays again."""
    T, H, d = 300, 2, 128
    q, k, v, g = _inputs(2, T, H, H, H, H, d, d, dtype)
    for t in (0, 5, 127, 128, 200, 201, 255):
        g[t, 0] = -math.inf
    g[40:60, 1] = -90.0
    g[130, 1] = -1e4
    init = torch.randn(1, H, d, d)
    ref, st, mag, sm = _oracle(q, k, v, g, [T], init, d ** -0.5)
    pool = init.to(DEV)
    out = ops.linear_attention(q.to(DEV), k.to(DEV), v.to(DEV), g.to(DEV), state=pool,
                               has_state=torch.ones(1, dtype=torch.int32, device=DEV))
    # strong decays: the rounded running sum of a block reaches 128 x 104, whose last place is 2^-11
    co, cs = _c(T, d, dtype == torch.bfloat16)
    _near(out, ref, mag, co + (2.0 ** -10 if dtype == torch.bfloat16 else 0), dtype == torch.bfloat16)
    _near(pool, st, sm, cs, False)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompt_neighbours_and_stale_rows_do_not_leak(dtype):
    """NaN and infinities in the tokens of other sequences, between the sequences, and in the state
    rows of fresh sequences stay there."""
    lens, H, d = [37, 60, 131], 2, 64
    T = sum(lens)
    q, k, v, g = _inputs(3, T, H, H, H, H, d, d, dtype)
    bad = slice(37, 97)
    for x in (q, k, v):
        x[bad] = math.nan
    v[bad][::2] = math.inf
    g[bad] = math.nan
    init = torch.randn(3, H, d, d)
    init[0] = math.nan
    has = torch.tensor([0, 1, 1], dtype=torch.int32)
    use = [0, 2]
    sel = torch.cat([torch.arange(37), torch.arange(97, T)])
    ref, st, mag, sm = _oracle(q[sel], k[sel], v[sel], g[sel], [37, 131],
                               torch.stack([torch.zeros_like(init[0]), init[2]]), d ** -0.5)
    pool = init.to(DEV)
    cu = torch.tensor([0, 37, 97, T], dtype=torch.int32, device=DEV)
    out = ops.linear_attention(q.to(DEV), k.to(DEV), v.to(DEV), g.to(DEV), state=pool, cu_seqlens=cu, has_state=has.to(DEV))
    co, cs = _c(131, d, dtype == torch.bfloat16)
    _near(out[sel.to(DEV)], ref, mag, co, dtype == torch.bfloat16)
    _near(pool[use], st, sm, cs, False)
    # tokens that belong to no sequence: cu skips the bad ones
    out = torch.full((T, H, d), 3.0, dtype=dtype, device=DEV)
    ops.linear_attention(q.to(DEV), k.to(DEV), v.to(DEV), g.to(DEV), out=out,
                         cu_seqlens=torch.tensor([0, 37], dtype=torch.int32, device=DEV))
    _near(out[:37], _oracle(q[:37], k[:37], v[:37], g[:37], [37], torch.zeros(1, H, d, d), d ** -0.5)[0], mag[:37], co,
          dtype == torch.bfloat16)
    assert bool((out[37:] == 3).all())


@gpu
def test_prompt_in_pieces_equals_the_whole():
    """A prompt fed in chunks that resume from the pool, then single tokens."""
    T, H, d = 700, 4, 128
    q, k, v, g = _inputs(4, T, H, H, H, H, d, d, torch.bfloat16)
    ref, st, mag, sm = _oracle(q, k, v, g, [T], torch.zeros(1, H, d, d), d ** -0.5)
    q, k, v, g = (x.to(DEV) for x in (q, k, v, g))
    pool = torch.full((2, H, d, d), math.nan, device=DEV)
    slots = torch.tensor([1], dtype=torch.int32, device=DEV)
    outs, at = [], 0
    for i, n in enumerate((130, 1, 256, 300)):
        s = slice(at, at + n)
        outs.append(ops.linear_attention(q[s], k[s], v[s], g[s], state=pool, slots=slots,
                                         has_state=torch.full((1,), int(i > 0), dtype=torch.int32, device=DEV)))
        at += n
    for t in range(at, T):
        outs.append(ops.linear_attention_step(q[t:t + 1], k[t:t + 1], v[t:t + 1], g[t:t + 1], pool, slots=slots))
    co, cs = _c(T, d, True)
    _near(torch.cat(outs), ref, mag, co, True)
    _near(pool[1:], st, sm, cs, False)
    assert bool(torch.isnan(pool[0]).all())


@gpu
@pytest.mark.parametrize("H,L", [(1, 5000), (2, 4097), (16, 2300)])
def test_long_prompts_split_over_their_length(H, L):
    """Few heads and long sequences (the split over the length), a short neighbour beside them."""
    d = 64
    lens = [L, 3]
    q, k, v, g = _inputs(H, L + 3, H, H, H, H, d, d, torch.bfloat16)
    ref, st, mag, sm = _oracle(q, k, v, g, lens, torch.zeros(2, H, d, d), d ** -0.5)
    pool = torch.zeros(2, H, d, d, device=DEV)
    cu = torch.tensor([0, L, L + 3], dtype=torch.int32, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    args = [x.to(DEV) for x in (q, k, v, g)]
    out = ops.linear_attention(*args, state=pool, cu_seqlens=cu, err=err)
    assert int(err) == 0
    co, cs = _c(L, d, True)
    _near(out, ref, mag, co, True)
    _near(pool, st, sm, cs, False)
    again = ops.linear_attention(*args, state=torch.empty_like(pool), cu_seqlens=cu)
    assert torch.equal(again, out)          # no sum depends on timing


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_slow_decays_keep_the_state_in_32_bits(dtype):
    """A fixed decay a little below 1 over thousands of tokens: a factor rounded the same way at every
    token would drift by 2048 x 2^-25 = 6e-5. Rounding errors of random sign leave sqrt(2048) x 2^-24
    = 2.7e-6 of the largest terms, and less of the whole (2-norm)."""
    T, H, d = 4096, 4, 64
    q, k, v, _ = _inputs(8, T, H, H, H, H, d, d, dtype)
    g = -torch.tensor([3e-4, 7.77e-4, 0.0, 0.11])
    _, st, _, _ = _oracle(q, k, v, g.expand(T, H), [T], torch.zeros(1, H, d, d), 1.0)
    pool = torch.empty(1, H, d, d, device=DEV)
    ops.linear_attention(q.to(DEV), k.to(DEV), v.to(DEV), g.to(DEV), state=pool)
    off = (pool.cpu().double() - st).flatten(2).norm(dim=-1) / st.flatten(2).norm(dim=-1)
    assert float(off.max()) < 2.7e-6, off


@gpu
def test_prompt_is_capturable_and_runs_on_the_callers_stream():
    T, H, d = 260, 4, 128
    q, k, v, g = (x.to(DEV) for x in _inputs(6, T, H, H, H, H, d, d, torch.bfloat16))
    want = ops.linear_attention(q, k, v, g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.linear_attention(q, k, v, g)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(want)
    with torch.cuda.graph(graph):
        ops.linear_attention(q, k, v, g, out=out)
    q.copy_(torch.randn_like(q))
    graph.replay()
    assert torch.equal(out, ops.linear_attention(q, k, v, g))


# ---------------------------------------------------------------------------------- single tokens
@gpu
@pytest.mark.parametrize("B", [1, 5, 64])
@pytest.mark.parametrize("H,Hq,Hk,Hv,dk,dv", [(4, 4, 4, 4, 128, 128), (8, 2, 1, 8, 128, 64), (3, 3, 3, 1, 64, 8),
                                              (2, 2, 2, 2, 64, 128), (2, 2, 2, 2, 96, 20)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_step_matches_the_recurrence(B, H, Hq, Hk, Hv, dk, dv, dtype):
    q, k, v, g = _inputs(B + dk, B, H, Hq, Hk, Hv, dk, dv, dtype, per_token=B != 5)
    r = torch.Generator().manual_seed(B)
    pool = torch.randn(B + 4, H, dv, dk, generator=r)
    slots = torch.randperm(B + 4, generator=r)[:B].to(torch.int32)
    ref, st, mag, sm = _oracle(q, k, v, g, [1] * B, pool[slots.long()], dk ** -0.5)
    dpool, dslots = pool.to(DEV), slots.to(DEV)
    if B > 1:
        dslots[B - 1] = -1                      # a padding row
    out = ops.linear_attention_step(q.to(DEV), k.to(DEV), v.to(DEV), (g[0] if B == 5 else g).to(DEV), dpool, slots=dslots)
    live = B if B == 1 else B - 1
    c = (dk + 16) * U
    _near(out[:live], ref[:live], mag[:live], c, dtype == torch.bfloat16)
    _near(dpool[slots[:live].long().to(DEV)], st[:live], sm[:live], 8 * U, False)
    if B > 1:
        assert not out[B - 1].any() and torch.equal(dpool[int(slots[B - 1])].cpu(), pool[int(slots[B - 1])])


@gpu
def test_step_forgets_at_minus_infinity_and_takes_strided_rows():
    B, H, d = 6, 2, 128
    q, k, v, g = _inputs(9, B, H, H, H, H, d, d, torch.float32)
    g[2] = -math.inf
    pool = torch.randn(B, H, d, d)
    ref, st, mag, sm = _oracle(q, k, v, g, [1] * B, pool, d ** -0.5)
    for pad in (4, 3):                          # rows on and off the 16-byte grid
        f = torch.zeros(B, 3 * H * d + pad, device=DEV)
        parts = [f[:, i * H * d:(i + 1) * H * d].unflatten(1, (H, d)) for i in range(3)]
        for p, x in zip(parts, (q, k, v)):
            p.copy_(x)
        dpool = pool.to(DEV)
        out = ops.linear_attention_step(*parts, g.to(DEV), dpool)
        _near(out, ref, mag, (d + 16) * U, False)
        _near(dpool, st, sm, 8 * U, False)


@gpu
@pytest.mark.parametrize("step", [True, False])
def test_state_pool_beyond_32_bit_offsets(step):
    H, d = 64, 128
    rows = (1 << 31) // (H * d * d) + 2
    if torch.cuda.mem_get_info()[0] < rows * H * d * d * 4 + (2 << 30):
        pytest.skip("needs 11 GB of device memory")
    pool = torch.empty(rows, H, d, d, device=DEV)
    last = torch.tensor([rows - 1], dtype=torch.int32, device=DEV)
    pool[-1] = 0.5
    pool[0] = 0.25
    q, k, v, g = _inputs(1, 1, H, H, H, H, d, d, torch.bfloat16)
    ref, st, mag, sm = _oracle(q, k, v, g, [1], torch.full((1, H, d, d), 0.5), d ** -0.5)
    args = [x.to(DEV) for x in (q, k, v, g)]
    if step:
        out = ops.linear_attention_step(*args, pool, slots=last)
    else:
        out = ops.linear_attention(*args, state=pool, slots=last, has_state=torch.ones_like(last))
    co, cs = _c(1, d, not step)
    _near(out, ref, mag, co, True)
    _near(pool[-1:], st, sm, cs, False)
    assert bool((pool[0] == 0.25).all())


@gpu
def test_device_side_indices_out_of_range_are_reported():
    q, k, v, g = (x.to(DEV) for x in _inputs(1, 40, 2, 2, 2, 2, 64, 64, torch.bfloat16))
    pool = torch.ones(2, 2, 64, 64, device=DEV)
    for kw in ({"slots": [7]}, {"cu": [0, 41]}, {"cu": [-1, 4]}, {"cu": [30, 10]}):
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        cu = torch.tensor(kw.get("cu", [0, 40]), dtype=torch.int32, device=DEV)
        slots = torch.tensor(kw.get("slots", [-1]), dtype=torch.int32, device=DEV)
        ops.linear_attention(q, k, v, g, state=pool, cu_seqlens=cu, slots=slots, err=err)
        assert int(err) == 1, kw
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = ops.linear_attention_step(q[:1], k[:1], v[:1], g[:1], pool, slots=torch.tensor([2], dtype=torch.int32, device=DEV), err=err)
    assert int(err) == 1 and not out.any() and bool((pool == 1).all())


@gpu
def test_linear_attention_refusals():
    q, k, v, g = (x.to(DEV) for x in _inputs(1, 4, 4, 4, 2, 4, 64, 64, torch.bfloat16))
    pool = torch.zeros(4, 4, 64, 64, device=DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    refused = [
        lambda: ops.linear_attention(q.cpu(), k, v, g),
        lambda: ops.linear_attention(q.float(), k, v, g),
        lambda: ops.linear_attention(q.half(), k.half(), v.half(), g),
        lambda: ops.linear_attention(q[:3], k, v, g),
        lambda: ops.linear_attention(q, k[..., :32], v, g),
        lambda: ops.linear_attention(q, k, v, g[:, :3]),
        lambda: ops.linear_attention(q, k, v, g.double()),
        lambda: ops.linear_attention(q, k, v, g.cpu()),
        lambda: ops.linear_attention(q.transpose(1, 2), k, v, g),
        lambda: ops.linear_attention(q, k, v, g, state=pool[:, :2]),
        lambda: ops.linear_attention(q, k, v, g, state=pool.bfloat16()),
        lambda: ops.linear_attention(q, k, v, g, slots=i32(0)),
        lambda: ops.linear_attention(q, k, v, g, state=pool, slots=i32(0, 1)),
        lambda: ops.linear_attention(q, k, v, g, state=pool, cu_seqlens=torch.tensor([0, 4], device=DEV)),
        lambda: ops.linear_attention(q, k, v, g, state=pool[:1], cu_seqlens=i32(0, 2, 4)),
        lambda: ops.linear_attention(q, k, v, g, out=torch.empty(4, 4, 32, dtype=q.dtype, device=DEV)),
        lambda: ops.linear_attention_step(q, k, v, g, pool[:3]),
        lambda: ops.linear_attention_step(q, k, v, g, pool, slots=i32(0, 1)),
    ]
    for i, f in enumerate(refused):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was taken")
    # nothing to do
    e = lambda x: x[:0]
    assert ops.linear_attention(e(q), e(k), e(v), e(g)).shape == (0, 4, 64)
    assert ops.linear_attention_step(e(q), e(k), e(v), e(g), pool).shape == (0, 4, 64)
    ops.linear_attention(q, k, v, g, state=pool, cu_seqlens=i32(0))


# ---------------------------------------------------------------------------------- add + norm + E4M3
def _norm_ref(x, y, w, eps, off):
    r = x.double() + (y.double() if y is not None else 0)
    n = r * (r.square().mean(-1, keepdim=True) + eps).rsqrt() * (w.double() + off)
    return r, n, n.abs().amax(-1) / 448


@gpu
@pytest.mark.parametrize("T,K", [(1, 8), (1, 4096), (3, 136), (5, 2048), (2, 2056), (7, 8192), (2, 16384), (3, 16392),
                                 (1, 32768), (300, 512)])
@pytest.mark.parametrize("ydt", [None, torch.bfloat16, torch.float32])
def test_add_rmsnorm_fp8(T, K, ydt):
    r = torch.Generator().manual_seed(T + K)
    x = torch.randn(T, K, generator=r) * 3
    x[:, K // 2] *= 40
    y = torch.randn(T, K, generator=r).to(ydt) if ydt else None
    w, off, eps = torch.randn(K, generator=r), 0.0 if K % 16 else 1.0, 1e-5
    rr, n, s = _norm_ref(x, y, w, eps, off)
    xd = x.to(DEV)
    nb = torch.empty(T, K, dtype=torch.bfloat16, device=DEV)
    xq, xs = ops.add_rmsnorm_fp8(xd, y.to(DEV) if ydt else None, w.to(DEV), eps, w_offset=off, out_bf16=nb)
    assert torch.equal(xd.cpu(), x + y.float() if ydt else x)            # in place, one f32 addition
    # mean of K squares: (K / threads + 10) roundings; the norm, weight and scale a few more
    c = (K / 64 + 24) * U
    torch.testing.assert_close(xs.cpu().double(), s, rtol=c, atol=0)
    _near(nb, n, n.abs(), c, True)
    # E4M3 has 4 significant bits: half a step is 2^-4 of the value, 2^-10 below the normals
    got = xq.cpu().view(torch.float8_e4m3fn).double()
    want = n / s[:, None]
    assert bool(((got - want).abs() <= want.abs() * (2.0 ** -4 + 2 * c) + 2.0 ** -10).all())
    # away from the rounding boundaries the codes are those of the exact quotient
    lo, hi = ((want * f).clamp(-448, 448).float().to(torch.float8_e4m3fn).double() for f in (1 - 4 * c, 1 + 4 * c))
    assert bool(((got == lo) | (got == hi)).all())


@gpu
@pytest.mark.parametrize("T,K", [(2369, 8), (2368, 256), (2369, 256), (2400, 136), (2400, 264), (2369, 512), (2400, 520)])
@pytest.mark.parametrize("ydt", [None, torch.bfloat16])
def test_add_rmsnorm_fp8_many_narrow_rows(T, K, ydt):
    test_add_rmsnorm_fp8(T, K, ydt)   # blocks of 32 and 64 threads: at most 8 squares a thread, inside K / 64 + 24


@gpu
def test_add_rmsnorm_fp8_special_rows():
    K = 256
    x = torch.randn(6, K, generator=torch.Generator().manual_seed(0))
    x[0] = 0
    x[1, 5] = math.nan
    x[2, 9] = math.inf
    x[3] *= 1e-38
    x[4] *= 1e18
    w = torch.ones(K)
    xq, xs = ops.add_rmsnorm_fp8(x.to(DEV), None, w.to(DEV), 1e-6)
    codes, xs = xq.cpu().view(torch.float8_e4m3fn).float(), xs.cpu()
    assert not codes[0].any() and xs[0] == 0
    for row in (1, 2):                                                    # reported, not swallowed
        assert torch.isnan(codes[row]).any() and not torch.isfinite(xs[row])
    _, n, s = _norm_ref(x, None, w, 1e-6, 0.0)
    for row in (3, 4, 5):
        got = codes[row].double() * xs[row].double()
        step = n[row].abs() * (2.0 ** -4 + 2.0 ** -18) + max(float(s[row]), 2.0 ** -126) * 2.0 ** -10
        assert bool(((got - n[row]).abs() <= step).all()), row


@gpu
def test_add_rmsnorm_fp8_strided_rows_and_out_of_place():
    big = torch.randn(9, 1024, device=DEV)
    x, y = big[:, 256:512], big[:, 512:768]
    keep = big.clone()
    res = torch.zeros(9, 264, device=DEV)[:, :256]
    w = torch.randn(256, device=DEV)
    xq, xs = ops.add_rmsnorm_fp8(x, y, w, 1e-5, resid_out=res)
    assert torch.equal(big, keep) and torch.equal(res, x + y)
    xq2, xs2 = ops.add_rmsnorm_fp8(res.contiguous(), None, w, 1e-5)
    assert torch.equal(xq, xq2) and torch.equal(xs, xs2)
    assert ops.add_rmsnorm_fp8(x[:0], y[:0], w, 1e-5)[0].shape == (0, 256)


@gpu
def test_add_rmsnorm_fp8_feeds_the_fp8_projection():
    from air_rs.gguf import GGMLType
    from air_rs.ops import gemm
    T, K, N = 33, 512, 384
    r = torch.Generator().manual_seed(3)
    codes = (torch.randn(N, K, generator=r) * 2).to(torch.float8_e4m3fn)
    sc = torch.rand(N, K // 128, generator=r) * 0.02 + 0.001
    w = ops.QWeight(ops.FMT_FP8, codes.view(torch.uint8).to(DEV), sc.to(DEV), N, K, GGMLType.FP8_E4M3_B128)
    x, y = torch.randn(T, K, generator=r), torch.randn(T, K, generator=r).bfloat16()
    xq, xs = ops.add_rmsnorm_fp8(x.to(DEV), y.to(DEV), torch.ones(K, device=DEV), 1e-5)
    out = gemm.linear_fp8_rows(xq, xs, w, torch.empty(T, N, device=DEV))
    wd = codes.double() * sc.double().repeat_interleave(128, 1)
    xd = xq.cpu().view(torch.float8_e4m3fn).double() * xs.cpu().double()[:, None]
    ref, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    # the tensor cores' f32 sum keeps at least 2^-13 of the largest term of an accumulation step
    assert bool(((out.double().cpu() - ref).abs() <= 2.0 ** -12 * mag).all())


@gpu
def test_add_rmsnorm_fp8_refusals():
    x, w = torch.randn(4, 256, device=DEV), torch.ones(256, device=DEV)
    for f in (lambda: ops.add_rmsnorm_fp8(x.bfloat16(), None, w, 1e-5), lambda: ops.add_rmsnorm_fp8(x, x[:3], w, 1e-5),
              lambda: ops.add_rmsnorm_fp8(x, x.half(), w, 1e-5), lambda: ops.add_rmsnorm_fp8(x, None, w[:8], 1e-5),
              lambda: ops.add_rmsnorm_fp8(x[:, :252], None, w[:252], 1e-5), lambda: ops.add_rmsnorm_fp8(x.cpu(), None, w, 1e-5),
              lambda: ops.add_rmsnorm_fp8(x[:, 1:9], None, w[:8], 1e-5),
              lambda: ops.add_rmsnorm_fp8(torch.zeros(1, 32776, device=DEV), None, torch.zeros(32776, device=DEV), 1e-5),
              lambda: ops.add_rmsnorm_fp8(x, None, w, 1e-5, xq=torch.empty(4, 128, dtype=torch.uint8, device=DEV))):
        with pytest.raises(RuntimeError):
            f()


# ---------------------------------------------------------------------------------- logit rules
def _rules_ref(lg, counts, rho, fr, pr, bias, allow):
    x = lg.double().clone()
    c = counts.double()
    f = rho.double()[:, None] ** c
    pen = torch.where(x > 0, x / f, x * f)
    x = torch.where((c > 0) & (x != 0), pen, x) - fr.double()[:, None] * c - pr.double()[:, None] * (c > 0)
    for b, row in enumerate(bias):
        for t, val in row:
            x[b, t] += val
    return x.masked_fill(~allow, -math.inf)


@gpu
@pytest.mark.parametrize("B,V", [(1, 1), (3, 31), (2, 2048), (4, 2056), (3, 5003), (2, 128256)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logit_rules(B, V, dtype):
    r = torch.Generator().manual_seed(V)
    lg = (torch.randn(B, V, generator=r) * 4).to(dtype)
    lg[0, 0] = 0.0
    counts = torch.zeros(B + 2, V, dtype=torch.uint8)
    counts[:, torch.randint(0, V, (60,), generator=r)] = torch.randint(1, 6, (60,), generator=r).to(torch.uint8)
    counts[:, V - 1] = 255
    crow = torch.randperm(B + 2, generator=r)[:B].to(torch.int32)
    rho, fr, pr = 1 + torch.rand(B, generator=r), torch.rand(B, generator=r), torch.rand(B, generator=r) - 0.5
    rho[0] = 1.0 if B > 1 else 1.3
    bias = [[(int(t), float(v)) for t, v in zip(torch.randint(0, V, (n,), generator=r), torch.randn(n, generator=r) * 9)]
            for n in ((700, 0, 3, 256)[:B])]                     # repeated tokens add up
    allow = torch.rand(B, V, generator=r) < 0.5
    if B > 1:
        allow[1] = False                                           # a grammar that allows nothing
    bits = torch.nn.functional.pad(allow, (0, -V % 32)).reshape(B, -1, 32).long()
    mask = (bits << torch.arange(32)).sum(-1)
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32)
    ptr = torch.tensor([0] + list(torch.tensor([len(x) for x in bias]).cumsum(0)), dtype=torch.int32)
    ids = torch.tensor([t for x in bias for t, _ in x], dtype=torch.int32)
    vals = torch.tensor([v for x in bias for _, v in x])
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    d = lambda t: t.to(DEV)
    got = ops.logit_rules(d(lg), counts=d(counts), count_row=d(crow), repetition=d(rho), frequency=d(fr), presence=d(pr),
                          bias=(d(ptr), d(ids), d(vals)), mask=d(mask), err=err)
    ref = _rules_ref(lg, counts[crow.long()], rho, fr, pr, bias, allow)
    assert int(err) == 0 and got.dtype == torch.float32
    assert torch.equal(torch.isinf(got.cpu()), torch.isinf(ref) | (ref.abs() > 3.4e38))
    # powf within 4 ulp of an exponent of up to 255, then one rounding per step and per bias entry
    fine = torch.isfinite(got.cpu())
    mag = lg.double().abs() * rho.double()[:, None] ** counts[crow.long()].double() + 300
    for b, row in enumerate(bias):
        for t, val in row:
            mag[b, t] += abs(val)
    assert bool(((got.cpu().double() - ref).abs()[fine] <= (720 * U * mag)[fine]).all())


@gpu
def test_logit_rules_masked_values_and_single_rules():
    V = 100
    lg = torch.randn(3, V)
    lg[0, 3], lg[1, 4], lg[2, 5] = math.nan, math.inf, -math.inf
    d = lg.to(DEV)
    allow = torch.full((3, 4), -1, dtype=torch.int32)
    for b, t in ((0, 3), (1, 4), (2, 5)):
        allow[b, t // 32] &= ~(1 << (t % 32))
    out = torch.empty(3, V, device=DEV)
    ops.logit_rules(d, out=out, mask=allow.to(DEV))
    want = lg.clone()
    want[0, 3] = want[1, 4] = want[2, 5] = -math.inf
    assert torch.equal(out.cpu(), want) and torch.equal(torch.isnan(d.cpu()), torch.isnan(lg))
    # the lowest finite value as a mask of one's own survives penalties without becoming NaN
    low = torch.full((1, 8), torch.finfo(torch.float32).min, device=DEV)
    got = ops.logit_rules(low, counts=torch.full((1, 8), 9, dtype=torch.uint8, device=DEV),
                          repetition=torch.tensor([2.0], device=DEV))
    assert not torch.isnan(got).any() and got.data_ptr() == low.data_ptr()
    # padding row: no counts
    x = torch.ones(2, 8, device=DEV)
    ops.logit_rules(x, counts=torch.ones(2, 8, dtype=torch.uint8, device=DEV), frequency=torch.ones(2, device=DEV),
                    count_row=torch.tensor([-1, 1], dtype=torch.int32, device=DEV))
    assert x.tolist() == [[1.0] * 8, [0.0] * 8]
    b = ops.bias_lists([{5: 2.0}, None], DEV)
    x = torch.zeros(2, 9, device=DEV)[:, 1:]
    ops.logit_rules(x, bias=b)
    assert x[0, 5] == 2.0 and float(x.abs().sum()) == 2.0


@gpu
def test_logit_rules_bad_indices_and_refusals():
    lg = torch.zeros(2, 64, device=DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    f32 = lambda *x: torch.tensor(x, dtype=torch.float32, device=DEV)
    cnt = torch.zeros(2, 64, dtype=torch.uint8, device=DEV)
    for kw in ({"counts": cnt, "count_row": i32(0, 2)}, {"bias": (i32(0, 1, 3), i32(1, 2), f32(1, 1))},
               {"bias": (i32(0, 1, 2), i32(1, 64), f32(1, 1))}, {"bias": (i32(0, 1, 2), i32(-1, 3), f32(1, 1))}):
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        ops.logit_rules(lg.clone(), err=err, **kw)
        assert int(err) == 1, kw
    for f in (lambda: ops.logit_rules(lg.cpu()), lambda: ops.logit_rules(lg.half()), lambda: ops.logit_rules(lg, presence=f32(1, 1)),
              lambda: ops.logit_rules(lg, counts=cnt[:1]), lambda: ops.logit_rules(lg, counts=cnt[:, :32]),
              lambda: ops.logit_rules(lg, counts=cnt, presence=f32(1)), lambda: ops.logit_rules(lg, mask=i32(1, 2)),
              lambda: ops.logit_rules(lg, out=lg.bfloat16()), lambda: ops.logit_rules(lg.t()),
              lambda: ops.logit_rules(lg, bias=(i32(0, 1), i32(0), f32(1)))):
        with pytest.raises(RuntimeError):
            f()
    assert ops.logit_rules(lg[:0]).shape == (0, 64)


def test_bias_lists_and_cpu_tensors_are_refused():
    ptr, ids, vals = ops.bias_lists([{7: 1.5, 2: -1.0}, None, {}, {0: 3.0}], "cpu")
    assert ptr.tolist() == [0, 2, 2, 2, 3] and ids.tolist() == [2, 7, 0] and vals.tolist() == [-1.0, 1.5, 3.0]
    assert ops.bias_lists([None, {}], "cpu") is None
