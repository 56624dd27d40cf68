"""The state-space decoder runs its operators together: every operator call of a run is recorded and held against its
definition in 64 bits on the inputs that it really got, and the residual stream is followed from call to call."""
import math

import pytest
import torch

from air_rs import ops
from air_rs.models.state_space import StateSpaceConfig, StateSpaceDecoder
from test_state_space_ops import U, _conv_ref, _held, _i32, _norm_ref, _scan_ref

gpu = pytest.mark.gpu


class Recorder:
    """Replaces the operators that the model calls by ones that keep copies of what goes in and out."""
    NAMES = ("causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step", "block_norm")

    def __init__(self, monkeypatch):
        self.calls = []
        for name in self.NAMES:
            monkeypatch.setattr(ops, name, self.wrap(name, getattr(ops, name)))

    def wrap(self, name, fn):
        keep = lambda v: v.detach().cpu().clone() if isinstance(v, torch.Tensor) else v

        def call(*a, **kw):
            before, kb = [keep(x) for x in a], {k: keep(v) for k, v in kw.items()}
            out = fn(*a, **kw)
            pool = a[2] if name == "causal_conv_step" else a[5] if name == "selective_scan_step" else kw.get("state")
            self.calls.append(dict(name=name, a=before, kw=kb, out=[keep(o) for o in (out if isinstance(out, tuple) else (out,))],
                                   after=keep(pool)))
            return out
        return call


def _check(c, lens):
    """Holds one recorded call against its definition."""
    name, a, kw = c["name"], c["a"], c["kw"]
    if name == "block_norm":
        ref, tol, r, rtol = _norm_ref(a[0], a[1], a[2], kw.get("residual"), kw.get("post_weight"), None, "silu",
                                      kw.get("scale", 1.0), 0.0)
        _held(c["out"][0], ref, tol, True)
        if kw.get("residual") is not None:
            _held(c["out"][1], r, rtol, False)
        return
    step, conv = name.endswith("_step"), "conv" in name
    pool = (a[2] if conv else a[5]) if step else kw.get("state")
    slots, has = kw.get("slots"), kw.get("has_state")
    shape = (a[1].shape[1] - 1, a[0].shape[1]) if conv else tuple(a[2].shape)
    init = torch.zeros(len(lens), *shape, dtype=a[0].dtype if conv else torch.float32)
    if pool is not None:
        keep = torch.ones(len(lens), dtype=torch.bool) if step else has != 0 if has is not None else torch.zeros(len(lens), dtype=torch.bool)
        init[keep] = pool[slots.long()][keep]
    if conv:
        ref, tol, ends = _conv_ref(a[0], a[1], a[3] if step else a[2], lens, init, True)
        etol = torch.zeros_like(ends, dtype=torch.float64)
    else:
        ref, tol, ends, etol = _scan_ref(a[0], a[1], a[2], a[3][:, None], a[4][:, None], kw["D"], kw["z"], kw["dt_bias"], True,
                                         lens, init)
    _held(c["out"][0], ref, tol, True)
    if pool is not None:
        _held(c["after"][slots.long()], ends.double(), etol, False)
        others = [i for i in range(pool.shape[0]) if i not in slots.tolist()]
        assert torch.equal(c["after"][others], pool[others])


CONFIGS = [StateSpaceConfig(), StateSpaceConfig(inner_dim=320, state_dim=8, conv_width=3, hidden_dim=192, vocab_size=512),
           StateSpaceConfig(n_layers=3, state_dim=24, post_norm=True, residual_scale=0.22, vocab_size=1000)]


@gpu
@pytest.mark.parametrize("c", range(len(CONFIGS)))
def test_every_call_of_prefill_and_decode(monkeypatch, c):
    cfg = CONFIGS[c]
    m = StateSpaceDecoder.random(cfg, max_seqs=6, seed=c)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (1, 140, 17)]
    slots, one = _i32([4, 0, 2]), _i32([7, 8, 9])
    rec = Recorder(monkeypatch)
    for run, lens in ((lambda: m.prefill(prompts, slots), [1, 140, 17]), (lambda: m.decode(one, slots), [1, 1, 1]),
                      (lambda: m.prefill([[9], [8, 7], [6]], slots, _i32([1, 0, 1])), [1, 2, 1])):
        rec.calls.clear()
        logits = run()
        assert logits.shape == (3, cfg.vocab_size) and bool(torch.isfinite(logits).all())
        assert len(rec.calls) == 1 + 3 * cfg.n_layers
        stream = None
        for call in rec.calls:
            _check(call, lens)
            if call["name"] == "block_norm":
                if stream is not None:
                    assert torch.equal(call["kw"]["residual"], stream)
                stream = call["out"][1] if call["out"][1] is not None else call["a"][0]
    assert int(m.err) == 0


@gpu
def test_prompts_do_not_see_each_other_and_resume():
    """A prompt packed with another and one cut in two reach the same logits and states, to the rounding of bf16
    activations."""
    cfg = StateSpaceConfig()
    m = StateSpaceDecoder.random(cfg, max_seqs=4)
    g = torch.Generator().manual_seed(3)
    a, b = (torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (33, 70))
    whole = m.prefill([a, b], _i32([0, 1]))
    m.prefill([b[:20]], _i32([2]))
    cut = m.prefill([b[20:]], _i32([2]), _i32([1]))
    # bf16 activations through two layers: compare with the spread of the logits
    spread = float(whole[1].max() - whole[1].min())
    assert float((whole[1] - cut[0]).abs().max()) <= 0.05 * spread
    for p in m.states:
        torch.testing.assert_close(p[1], p[2], rtol=0.1, atol=0.02 * float(p[1].abs().max()))


@gpu
def test_generate_and_score():
    cfg = StateSpaceConfig()
    m = StateSpaceDecoder.random(cfg, max_seqs=4)
    prompts = [[5, 6, 7], [11], list(range(40, 90))]
    outs = m.generate(prompts, 5)
    assert [len(o) for o in outs] == [5, 5, 5]
    assert m.generate(prompts, 5) == outs                    # an earlier request leaves nothing behind
    banned = m.generate(prompts, 5, bias=[{outs[0][0]: -1e9}, None, None])
    assert banned[0][0] != outs[0][0] and banned[1] == outs[1]
    states = [s.clone() for s in m.states]
    scores = m.score(prompts, top=4)
    assert all(torch.equal(x, y) for x, y in zip(states, m.states))
    logits = m._prompts(prompts, None, None, every=True).double().cpu()
    at = 0
    for p, s in zip(prompts, scores):
        lp = torch.log_softmax(logits[at:at + len(p) - 1], -1)
        at += len(p)
        assert s.logprobs.shape == (len(p) - 1,) and s.top_ids.shape == (len(p) - 1, 4)
        want = lp.gather(1, torch.tensor(p[1:])[:, None])[:, 0] if len(p) > 1 else torch.empty(0, dtype=torch.float64)
        # a logarithm of a sum of V exponentials, V / 128 of them a lane, in f32
        assert torch.allclose(s.logprobs.double(), want, rtol=0, atol=(cfg.vocab_size / 128 + 64) * U * 32)
        assert torch.equal(s.top_ids.long(), torch.sort(lp, descending=True, stable=True).indices[:, :4])
        ent = -(lp.exp() * lp).sum(-1)
        assert torch.allclose(s.entropy.double(), ent, rtol=0, atol=(cfg.vocab_size / 128 + 64) * U * 64)
    with pytest.raises(RuntimeError, match="index out of range"):
        m.generate([[5], [cfg.vocab_size + 3]], 1)
    with pytest.raises(ValueError):
        m.generate([[1]] * 5, 1)
    with pytest.raises(ValueError):
        m.prefill([[1], []], _i32([0, 1]))
    with pytest.raises(ValueError):
        m.prefill([[1], [2]], _i32([0]))
    assert m.generate([], 3) == [] and m.score([]) == []


def test_engine_token_scores_on_the_oracle(tmp_path):
    from air_rs.gguf import GGMLType
    from air_rs.models.config import tiny_llama
    from air_rs.models.random_init import random_tensors
    from air_rs.models.reference import OracleModel
    from air_rs.runtime.engine import Engine
    cfg = tiny_llama()
    eng = Engine(cfg, None, oracle=OracleModel(cfg, {n: (r, q, s) for n, r, q, s in random_tensors(cfg, GGMLType.Q8_0, seed=0, device="cpu")}))
    ids = [5, 6, 7, 8]
    s = eng.token_scores(ids, top=3)
    assert s.logprobs.tolist() == eng.token_logprobs(ids)
    assert s.top_ids.shape == (len(s.logprobs), 3) and bool((s.top_logprobs[:, 0] >= s.logprobs).all())
    assert bool((s.entropy > 0).all()) and bool((s.entropy <= math.log(cfg.vocab_size) + 1e-4).all())
    assert eng.token_scores([3], add_bos=False, top=2).top_ids.shape == (0, 2)
    with pytest.raises(ValueError):
        eng.token_scores(ids, top=33)


@gpu
def test_engine_token_scores_match_the_oracle():
    from air_rs.gguf import GGMLType
    from air_rs.models.config import tiny_llama
    from air_rs.models.random_init import random_tensors
    from air_rs.models.reference import OracleModel
    from air_rs.runtime.builder import build_runner
    from air_rs.runtime.engine import Engine
    cfg = tiny_llama()
    recs = list(random_tensors(cfg, GGMLType.Q8_0, seed=0, device="cpu"))
    oracle = OracleModel(cfg, {n: (r, q, s) for n, r, q, s in recs})
    eng = Engine(cfg, build_runner(cfg, iter(recs), device="cuda", max_batch=8, max_model_len=256, num_blocks=64))
    ids = torch.randint(0, cfg.vocab_size, (30,), generator=torch.Generator().manual_seed(0)).tolist()
    a, b = eng.token_scores(ids, top=5), Engine(cfg, None, oracle=oracle).token_scores(ids, top=5)
    # the runner's int8 activations against the oracle's: the same tolerance as its log probabilities have elsewhere
    for x, y in zip(a[:3], b[:3]):
        assert x.shape == y.shape
        torch.testing.assert_close(x, y, rtol=0, atol=0.05)
    assert eng.seqs.allocator.num_used_blocks() == 0
