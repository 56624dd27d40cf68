"""The block form of linear attention where its hand-overs, its split over the length and its state's precision are
at work: long runs of empty sequences between a CTA's blocks, every pair of head sizes, sequences that resume from
the pool and are cut. Definitions, inputs and bounds are those of test_recurrent_ops."""
import pytest
import torch

from air_rs import ops
from test_recurrent_ops import _c, _inputs, _near, _oracle

DEV = "cuda"
gpu = pytest.mark.gpu


def _cu(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------------------------- runs of empty sequences
RUNS = [  # heads, lengths
    # whole items dealt out in turns (more sequences than are sorted): a CTA steps over hundreds of empty ones
    (64, [1000] + [0] * 500 + [1000] + [0] * 500 + [1000]),
    # short prompts around a run of empty slots: turns without work between two blocks of a CTA
    (64, [128] * 30 + [0] * 200 + [100] * 30),
    # one stretch of the list for each SM: a cut sequence, empty ones behind it, a short one at the end
    (2, [2900] + [0] * 500 + [40]),
]


@gpu
@pytest.mark.parametrize("case", range(len(RUNS)))
def test_runs_of_empty_sequences_between_blocks(case):
    """The description of a CTA's next block can be late by many blocks' time; nothing that is waited for meanwhile
    may be missed."""
    H, lens = RUNS[case]
    T, N, d = sum(lens), len(lens), 64
    r = torch.Generator().manual_seed(case)
    q, k, v, g = _inputs(case, T, H, 1, 1, H, d, d, torch.bfloat16)
    has = torch.randint(0, 2, (N,), generator=r)
    full = [n for n in range(N) if lens[n]]
    pool = torch.randn(N, H, d, d, generator=r)
    init = (pool * has[:, None, None, None])[full]
    # an oracle of matrix products, sequence by sequence in blocks of 100 tokens
    out, st, mag, sm = _by_blocks(q, k, v, g, [lens[n] for n in full], init, 0.125)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    dpool = pool.to(DEV)
    args = [x.to(DEV) for x in (q, k, v, g)]
    got = ops.linear_attention(*args, state=dpool, cu_seqlens=_cu(lens), has_state=has.to(torch.int32).to(DEV), err=err)
    assert int(err) == 0
    co, cs = _c(max(lens), d, True)
    _near(got, out, mag, co, True)
    _near(dpool[full], st, sm, cs, False)
    empty = [n for n in range(N) if not lens[n]]
    assert torch.equal(dpool[empty].cpu(), (pool * has[:, None, None, None])[empty])


def _by_blocks(q, k, v, g, lens, init, scale, block=100):
    """_oracle's results by products over blocks of tokens (64 bits), for sequences too long to take token by token."""
    H = g.shape[1]
    q, k, v = (x.double().repeat_interleave(H // x.shape[1], 1).transpose(0, 1) for x in (q, k, v))     # [H, T, d]
    g = g.double().t()
    out = torch.zeros(v.shape, dtype=torch.float64)
    mag = torch.zeros_like(out)
    st, sm = init.double().clone(), init.double().abs()
    t = 0
    for n, L in enumerate(lens):
        for b in range(t, t + L, block):
            e = min(b + block, t + L)
            G = g[:, b:e].cumsum(1)
            w = (G[:, :, None] - G[:, None, :]).masked_fill(~torch.ones(e - b, e - b, dtype=torch.bool).tril(), -float("inf")).exp()
            for x, s, f in ((out, st, lambda z: z), (mag, sm, torch.abs)):
                qb, kb, vb = f(q[:, b:e]), f(k[:, b:e]), f(v[:, b:e])
                x[:, b:e] = abs(scale) * ((qb @ kb.transpose(1, 2) * w) @ vb + (qb * G.exp()[..., None]) @ s[n].transpose(1, 2))
                s[n] = s[n] * G[:, -1].exp()[:, None, None] + (vb * (G[:, -1:] - G).exp()[..., None]).transpose(1, 2) @ kb
        t += L
    if scale < 0:
        out = -out
    return out.transpose(0, 1), st, mag.transpose(0, 1), sm


def test_block_oracle_is_the_recurrence():
    """On the CPU: the oracle by blocks against the one token by token."""
    lens = [250, 3, 101]
    q, k, v, g = _inputs(0, sum(lens), 4, 2, 1, 4, 16, 8, torch.bfloat16, strong=True)
    init = torch.randn(3, 4, 8, 16, generator=torch.Generator().manual_seed(1))
    for a, b in zip(_by_blocks(q, k, v, g, lens, init, -0.3), _oracle(q, k, v, g, lens, init, -0.3)):
        torch.testing.assert_close(a, b, rtol=1e-11, atol=1e-11)


# ---------------------------------------------------------------------------------- malformed offsets
@gpu
@pytest.mark.parametrize("H", [2, 80])
def test_offsets_that_name_more_tokens_than_there_are(H):
    """0, T, 0, T, ...: every second sequence is valid by itself, together they hold T many times over (enough of them
    would pass 32 bits of blocks). The call reports it and writes nothing."""
    T, N, d = 1000, 64, 64
    q, k, v, g = (x.to(DEV) for x in _inputs(1, T, H, 1, 1, 1, d, d, torch.bfloat16))
    pool = torch.ones(N, H, d, d, device=DEV)
    out = torch.full((T, H, d), 3.0, dtype=torch.bfloat16, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, T] * (N // 2) + [0], dtype=torch.int32, device=DEV)
    ops.linear_attention(q, k, v, g, state=pool, cu_seqlens=cu, out=out, has_state=torch.ones(N, dtype=torch.int32, device=DEV),
                         err=err)
    assert int(err) == 1 and bool((out == 3).all()) and bool((pool == 1).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_sequence_with_bad_offsets_keeps_its_state(dtype):
    """Offsets past the tokens, and offsets that go back: those sequences are skipped, fresh or not; the others run."""
    T, H, d = 40, 2, 64
    q, k, v, g = _inputs(1, T, H, H, H, H, d, d, dtype)
    out, st, mag, sm = _oracle(q[:20], k[:20], v[:20], g[:20], [20], torch.zeros(1, H, d, d), 0.125)
    for fresh in (True, False):
        pool = torch.full((4, H, d, d), 2.0, device=DEV)
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        has = torch.tensor([0] + [int(not fresh)] * 3, dtype=torch.int32, device=DEV)
        cu = torch.tensor([0, 20, 50, 40, 40], dtype=torch.int32, device=DEV)
        got = ops.linear_attention(*(x.to(DEV) for x in (q, k, v, g)), state=pool, cu_seqlens=cu, has_state=has, err=err)
        assert int(err) == 1
        co, cs = _c(20, d, dtype == torch.bfloat16)
        _near(got[:20], out, mag, co, dtype == torch.bfloat16)
        _near(pool[:1], st, sm, cs, False)
        assert bool((pool[1:3] == 2).all()) and bool((pool[3] == (0 if fresh else 2)).all())


@gpu
@pytest.mark.parametrize("row", [-2, -2 ** 31, 3, 2 ** 31 - 1])
def test_rows_out_of_range_are_reported_and_count_as_none(row):
    d = 64
    q, k, v, g = (x.to(DEV) for x in _inputs(1, 40, 2, 2, 2, 2, d, d, torch.bfloat16))
    pool = torch.ones(3, 2, d, d, device=DEV)
    at = torch.tensor([row], dtype=torch.int32, device=DEV)
    word = lambda: torch.zeros(1, dtype=torch.int32, device=DEV)
    for T in (40, 3):                       # block form, token by token
        err = word()
        got = ops.linear_attention(q[:T], k[:T], v[:T], g[:T], state=pool, slots=at, err=err)
        assert int(err) == 1 and torch.equal(got, ops.linear_attention(q[:T], k[:T], v[:T], g[:T]))
    err = word()
    assert not ops.linear_attention_step(q[:1], k[:1], v[:1], g[:1], pool, slots=at, err=err).any() and int(err) == 1
    assert bool((pool == 1).all())
    err = word()
    counts = torch.ones(3, 8, dtype=torch.uint8, device=DEV)
    x = ops.logit_rules(torch.ones(1, 8, device=DEV), counts=counts, presence=torch.ones(1, device=DEV), count_row=at, err=err)
    assert int(err) == 1 and bool((x == 1).all())


# ---------------------------------------------------------------------------------- NaN and infinities
def _bad_v(T, Hv, dv, seed):
    """Values with NaN and infinities in single entries, a whole token, and a sequence's first and last tokens, and
    the first such token of each head and column (T: none)."""
    r = torch.Generator().manual_seed(seed)
    bad = torch.zeros(T, Hv, dv)
    put = torch.tensor([float("nan"), float("inf"), -float("inf")])
    for t, h, c in ((T - 1, 0, 3), (T // 2, 0, 5), (T // 2 + 1, 0, 5), (T // 3, Hv - 1, dv - 1), (0, Hv - 1, 9)):
        bad[t, h, c] = put[int(torch.randint(0, 3, (1,), generator=r))]
    bad[(2 * T) // 3, Hv - 1] = float("nan")
    odd = bad != 0
    first = torch.where(odd.any(0), odd.int().argmax(0), torch.full((Hv, dv), T))
    return bad, first


@gpu
@pytest.mark.parametrize("dk,dv", [(128, 128), (128, 64), (64, 128), (64, 64)])
@pytest.mark.parametrize("T", [13, 100, 128, 300, 2600])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nan_and_infinities_in_v_do_not_reach_earlier_tokens(T, dk, dv, dtype):
    """o_t depends on tokens up to t: before a NaN or an infinity of its column it is what the finite values give,
    from it on it is not finite; other columns stay as they are. The state's columns likewise."""
    if dtype == torch.float32 and T > 300:
        pytest.skip("the token-by-token form has no split")
    H = 2
    q, k, v, g = _inputs(T + dk, T, H, H, H, H, dk, dv, dtype)
    bad, first = _bad_v(T, H, dv, T)
    out, st, mag, sm = _by_blocks(q, k, v, g, [T], torch.zeros(1, H, dv, dk), 1.0)
    vb = torch.where(bad != 0, bad, v.float()).to(dtype)
    pool = torch.zeros(1, H, dv, dk, device=DEV)
    got = ops.linear_attention(q.to(DEV), k.to(DEV), vb.to(DEV), g.to(DEV), state=pool, scale=1.0).cpu()
    early = torch.arange(T)[:, None, None] < first[None]
    assert bool(torch.isfinite(got[early]).all()) and not bool(torch.isfinite(got[~early]).any())
    # the sums up to a token hold the finite values alone, those after it are not looked at
    zero = torch.zeros(())
    fine = _by_blocks(q, k, torch.where(bad != 0, zero, v.float()).to(dtype), g, [T], torch.zeros(1, H, dv, dk), 1.0)
    co, cs = _c(T, dk, dtype == torch.bfloat16)
    _near(torch.where(early, got.double(), 0.0), torch.where(early, fine[0], 0.0), mag, co, dtype == torch.bfloat16)
    whole = (first == T)[None, :, :, None].expand_as(st)
    assert not bool(torch.isfinite(pool.cpu()[~whole]).any())
    _near(torch.where(whole, pool.cpu().double(), 0.0), torch.where(whole, st, 0.0), sm, cs, False)


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_nan_in_one_sequence_stays_there(d):
    """Packed sequences that share a CTA's tiles: one with NaN in v between two without."""
    lens, H = [200, 77, 300, 128], 3
    T = sum(lens)
    q, k, v, g = _inputs(d, T, H, H, H, H, d, d, torch.bfloat16)
    out, st, mag, sm = _by_blocks(q, k, v, g, lens, torch.zeros(4, H, d, d), 1.0)
    vb = v.clone()
    vb[210] = float("nan")
    vb[277 + 299, 1, 7] = float("inf")
    pool = torch.zeros(4, H, d, d, device=DEV)
    got = ops.linear_attention(q.to(DEV), k.to(DEV), vb.to(DEV), g.to(DEV), state=pool, cu_seqlens=_cu(lens), scale=1.0).cpu()
    keep = torch.ones(T, H, d, dtype=torch.bool)
    keep[210:277] = False
    keep[576, 1, 7] = False
    assert bool(torch.isnan(got[~keep]).all())
    co, cs = _c(max(lens), d, True)
    _near(torch.where(keep, got.double(), 0.0), torch.where(keep, out, 0.0), mag, co, True)
    _near(pool[[0, 3]], st[[0, 3]], sm[[0, 3]], cs, False)


# ---------------------------------------------------------------------------------- decays
@gpu
def test_decays_after_strong_ones_keep_their_exponents():
    """64 tokens that forget everything, then none that decay: row i's factor for a token of the third 32 is 1. Taken as a
    difference of sums from the block's first token (9200 in log2, steps of 2^-10) it would be off by 2^-11 in the
    exponent wherever the two strong 32s' sum rounds, 3.4e-4 relatively. The scores lie 1.2e-4 (2^-13) on either side of
    the middle of two bf16 numbers, so each output is an exact number."""
    T, H, d = 128, 16, 64
    q, k, v = (torch.zeros(T, H, d) for _ in range(3))
    k[70, :, :3] = torch.tensor([1.0, 2.0 ** -8 - 2.0 ** -13, 2.0 ** -8 + 2.0 ** -13])
    q[:, :, 0] = 1
    q[0::2, :, 1] = q[1::2, :, 2] = 1            # scores 1 + 2^-8 -+ 2^-13
    v[70] = 1
    g = torch.zeros(T, H)
    g[:32] = -100.0 - 0.03 * torch.arange(H)
    g[32:64] = -99.0
    args = [x.to(torch.bfloat16).to(DEV) for x in (q, k, v)]
    got = ops.linear_attention(*args, g.to(DEV), scale=1.0).float().cpu()
    assert not got[:70].any()
    assert bool((got[96::2] == 1).all()) and bool((got[97::2] == 1 + 2.0 ** -7).all())
    assert bool((got[70:96:2] == 1).all()) and bool((got[71:96:2] == 1 + 2.0 ** -7).all())


# ---------------------------------------------------------------------------------- precision and reach
DIMS = [(128, 128), (128, 64), (64, 128), (64, 64)]
# lengths, heads: whole items; two sequences that are cut, with an empty one between and a short one behind
SHAPES = [([300, 129, 5], 4), ([1500, 0, 2100, 7], 3)]


def _slow(T, H):
    """Decays that keep the incoming state for thousands of tokens."""
    return torch.tensor([3e-4, 7.77e-4, 0.0, 1.1e-3])[:H].neg().expand(T, H).contiguous()


@gpu
@pytest.mark.parametrize("dk,dv", DIMS)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("slow", [False, True])
@pytest.mark.parametrize("resume", [False, True])
def test_state_keeps_32_bits(dk, dv, shape, slow, resume):
    """Fresh and resumed sequences, whole and cut, for each pair of head sizes. A block's update is 32 accumulation steps
    (8 times 16 tokens, 4 parts of the keys) that each drop at most 2^-23 of the running sum, half of that in the mean,
    and the sum's size is 2/3 of its last in the mean: 32 x 2^-24 x 2/3 = 1.3e-6 of the state (2-norm). Exponents: 8
    roundings of a sum G weigh G exp(-G) <= 0.37, 8 x 0.37 x 2^-24 = 1.8e-7; the updates of S 2^-24 a block, of random
    sign: 17 blocks 2.5e-7. Without the last part of the decayed keys 3.4e-6 would be missing."""
    lens, H = SHAPES[shape]
    T, N = sum(lens), len(lens)
    q, k, v, g = _inputs(dk + dv + shape, T, H, H, H, H, dk, dv, torch.bfloat16)
    if slow:
        g = _slow(T, H)
    r = torch.Generator().manual_seed(shape)
    pool = torch.randn(N + 2, H, dv, dk, generator=r)
    slots = torch.randperm(N + 2, generator=r)[:N]
    init = pool[slots] * float(resume)
    out, st, mag, sm = _by_blocks(q, k, v, g, lens, init, 1.0)
    dpool = pool.to(DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.linear_attention(*(x.to(DEV) for x in (q, k, v, g)), state=dpool, cu_seqlens=_cu(lens), scale=1.0,
                               slots=slots.to(torch.int32).to(DEV), err=err,
                               has_state=torch.full((N,), int(resume), dtype=torch.int32, device=DEV))
    assert int(err) == 0
    _near(got, out, mag, _c(max(lens), dk, True)[0], True)
    full = [n for n in range(N) if lens[n]]
    off = (dpool.cpu()[slots].double() - st)[full].flatten(2).norm(dim=-1) / st[full].flatten(2).norm(dim=-1)
    assert float(off.max()) < 1.3e-6 + 1.8e-7 + 2.5e-7, off
    empty = [n for n in range(N) if not lens[n]]
    assert torch.equal(dpool.cpu()[slots][empty], init[empty])
    others = torch.ones(N + 2, dtype=torch.bool)
    others[slots] = False
    assert torch.equal(dpool.cpu()[others], pool[others])


@gpu
@pytest.mark.parametrize("H,T", [(64, 40), (2, 2100)])
def test_block_form_with_state_offsets_beyond_32_bits(H, T):
    """The last row of a pool of more than 2^31 numbers, for a whole sequence and for one that is cut."""
    d = 128
    rows = (1 << 31) // (H * d * d) + 2
    if torch.cuda.mem_get_info()[0] < rows * H * d * d * 4 + (3 << 30):
        pytest.skip("needs 12 GB of device memory")
    pool = torch.empty(rows, H, d, d, device=DEV)
    last = torch.tensor([rows - 1], dtype=torch.int32, device=DEV)
    init = torch.randn(1, H, d, d, generator=torch.Generator().manual_seed(H))
    pool[-1:] = init.to(DEV)
    pool[0] = 0.25
    q, k, v, _ = _inputs(H, T, H, 2, 2, 2, d, d, torch.bfloat16)
    g = _slow(T, 2).repeat_interleave(H // 2, 1)
    out, st, mag, sm = _by_blocks(q, k, v, g, [T], init, 1.0)
    got = ops.linear_attention(*(x.to(DEV) for x in (q, k, v, g)), state=pool, slots=last, has_state=torch.ones_like(last), scale=1.0)
    co, cs = _c(T, d, True)
    _near(got, out, mag, co, True)
    _near(pool[-1:], st, sm, cs, False)
    assert bool((pool[0] == 0.25).all())


@gpu
def test_block_form_with_token_offsets_beyond_32_bits():
    """Outputs of more than 2^31 numbers: the last of the packed sequences against the recurrence."""
    T, H, d, L = 140000, 128, 128, 200
    if torch.cuda.mem_get_info()[0] < 4 * T * H * d:
        pytest.skip("needs 9 GB of device memory")
    q, k, v, g = _inputs(3, L, 2, 1, 1, 1, d, d, torch.bfloat16)
    ref, _, mag, _ = _by_blocks(q, k, v, g, [L], torch.zeros(1, 2, d, d), 1.0)
    rows = lambda x: torch.cat([torch.zeros(T - L, *x.shape[1:], dtype=x.dtype, device=DEV), x.to(DEV)])
    lens = [T // 2, T - L - T // 2, L]
    out = ops.linear_attention(rows(q), rows(k), rows(v), rows(g.repeat_interleave(H // 2, 1)), cu_seqlens=_cu(lens), scale=1.0)
    assert not out[: T - L: 997].any() and not out[T - L - 1].any()
    co = _c(L, d, True)[0]
    for h in (0, 63, 64, 127):
        _near(out[T - L:, h], ref[:, h // 64], mag[:, h // 64], co, True)
