"""The recurrent decoder runs its operators together. E4M3 rows make two models that round apart drift from each
other by percents, so nothing is compared end to end: every operator call of a run is recorded and held against
its definition in 64 bits on the inputs that it really got, and the buffers are followed from call to call."""
import pytest
import torch

from air_rs import ops
from air_rs.models.recurrent import RecurrentConfig, RecurrentDecoder
from air_rs.ops import gemm
from test_recurrent_ops import U, _blocks, _c, _near, _oracle

gpu = pytest.mark.gpu


class Recorder:
    """Replaces the operators that the model calls by ones that keep copies of what goes in and out."""
    NAMES = [(ops, "add_rmsnorm_fp8"), (ops, "linear_attention"), (ops, "linear_attention_step"),
             (gemm, "linear_fp8_rows"), (gemm, "linear_fp8")]

    def __init__(self, monkeypatch):
        self.calls, self.depth = [], 0
        for mod, name in self.NAMES:
            monkeypatch.setattr(mod, name, self.wrap(name, getattr(mod, name)))

    def wrap(self, name, fn):
        keep = lambda v: v.detach().cpu().clone() if isinstance(v, torch.Tensor) else v

        def call(*a, **kw):
            if self.depth:
                return fn(*a, **kw)
            before, kb = [keep(x) for x in a], {k: keep(v) for k, v in kw.items()}
            self.depth += 1
            out = fn(*a, **kw)
            self.depth -= 1
            outs = out if isinstance(out, tuple) else (out,)
            self.calls.append(dict(name=name, a=before, kw=kb, out=[keep(o) for o in outs], live=a, live_out=outs,
                                   after=[keep(x) for x in a]))
            return out
        return call


def _dense(w):
    return w.data.cpu().view(torch.float8_e4m3fn).double() * w.scales.cpu().double().repeat_interleave(128, 1)


def _check_norm(c, eps):
    x, y, w = c["a"][:3]
    r = x.double() + (y.double() if y is not None else 0)
    if y is not None:
        assert torch.equal(c["after"][0], x + y.float())
    n = r / (r.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    s = n.abs().amax(-1) / 448
    k = (x.shape[1] / 64 + 24) * U
    torch.testing.assert_close(c["out"][1].double(), s, rtol=k, atol=0)
    got, want = c["out"][0].view(torch.float8_e4m3fn).double(), n / s[:, None]
    assert bool(((got - want).abs() <= want.abs() * (2.0 ** -4 + 2 * k) + 2.0 ** -10).all())


def _check_rows(c):
    xq, xs, w = c["a"][:3]
    x, wd = xq.view(torch.float8_e4m3fn).double() * xs.double()[:, None], _dense(c["live"][2])
    ref, mag = x @ wd.t(), x.abs() @ wd.abs().t()
    # the tensor cores' f32 sum keeps at least 2^-13 of the largest term of an accumulation step
    _near(c["out"][0], ref, mag, 2.0 ** -12, c["out"][0].dtype == torch.bfloat16)


@gpu
@pytest.mark.parametrize("dims", [(64, 128), (128, 64), (48, 32)])
def test_every_call_of_prefill_and_decode(monkeypatch, dims):
    cfg = RecurrentConfig(key_dim=dims[0], value_dim=dims[1]) if dims[0] != 48 else \
        RecurrentConfig(key_dim=48, value_dim=32, hidden_dim=256, intermediate_dim=256, vocab_size=512)
    m = RecurrentDecoder.random(cfg, max_seqs=6, seed=dims[0])
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (1, 140, 17)]
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    rec = Recorder(monkeypatch)
    one = torch.full((3,), 7, dtype=torch.int32, device="cuda")
    runs = [(lambda: m.prefill(prompts, slots), [len(p) for p in prompts], False),
            (lambda: m.decode(one, slots), [1, 1, 1], True),
            (lambda: m.prefill([[9], [8, 7], [6]], slots, torch.ones_like(slots)), [1, 2, 1], True)]
    for run, lens, resume in runs:
        rec.calls.clear()
        states = [s.clone() for s in m.states]
        logits = run()
        assert int(m.err) == 0
        calls = rec.calls
        mixer = "linear_attention_step" if len(calls[2]["a"]) > 4 else "linear_attention"
        assert [c["name"] for c in calls] == (["add_rmsnorm_fp8", "linear_fp8_rows", mixer, "linear_fp8",
                                               "add_rmsnorm_fp8", "linear_fp8_rows", "linear_fp8"] * cfg.n_layers +
                                              ["add_rmsnorm_fp8", "linear_fp8_rows"])
        assert logits is calls[-1]["live_out"][0] and logits.shape == (3, cfg.vocab_size)
        for i, c in enumerate(calls):
            prev = calls[i - 1] if i else None
            if c["name"] == "add_rmsnorm_fp8":
                _check_norm(c, cfg.eps)
                last = i + 2 == len(calls)
                if prev is None:
                    assert c["a"][1] is None
                elif not last:
                    assert c["live"][1].data_ptr() == prev["live_out"][0].data_ptr()
                    assert c["live"][0].data_ptr() == calls[0]["live"][0].data_ptr()
                else:
                    at = torch.tensor(lens).cumsum(0) - 1
                    assert torch.equal(c["a"][1], prev["out"][0][at]) and c["a"][0].shape[0] == 3
            elif c["name"] == "linear_fp8_rows":
                _check_rows(c)
                assert c["live"][0] is prev["live_out"][0] and c["live"][1] is prev["live_out"][1]
            elif c["name"].startswith("linear_attention"):
                layer = m.layers[i // 7]
                p = prev["out"][0]
                h, dk, dv = cfg.n_heads, cfg.key_dim, cfg.value_dim
                for t, at, d in ((c["a"][0], 0, dk), (c["a"][1], h * dk, dk), (c["a"][2], 2 * h * dk, dv)):
                    assert torch.equal(t.flatten(1), p[:, at:at + h * d])
                gate = p[:, h * (2 * dk + dv):][:, :h].double()
                want = -torch.nn.functional.softplus(gate) * layer.rate.cpu().double()
                torch.testing.assert_close(c["a"][3].double(), want, rtol=1e-5, atol=1e-7)
                pool0 = states[i // 7].cpu()
                init = pool0[slots.cpu().long()] * float(resume)
                ref, st, mag, sm = _oracle(*c["a"][:4], lens, init, c["kw"]["scale"])
                co, cs = _c(max(lens), dk, mixer == "linear_attention" and _blocks(torch.bfloat16, dk, dv))
                _near(c["out"][0], ref, mag, co, True)
                _near(m.states[i // 7][slots.long()], st, sm, cs, False)
                others = [s for s in range(6) if s not in (4, 0, 2)]
                assert torch.equal(m.states[i // 7][others].cpu(), pool0[others])
            else:
                # the output projection takes the mixer's heads side by side, the down projection the gated product
                if prev["name"].startswith("linear_attention"):
                    assert torch.equal(c["a"][0], prev["out"][0].flatten(1))
                else:
                    gu, F = prev["out"][0].double(), cfg.intermediate_dim
                    want = torch.nn.functional.silu(gu[:, :F]) * gu[:, F:]
                    _near(c["a"][0], want, want.abs(), 1e-5, True)
                x = c["a"][0].double()
                s = x.abs().amax(-1, keepdim=True) / 448
                wd = _dense(c["live"][1])
                # the rows' E4M3 rounding (2^-4 of a value, 2^-10 of the scale) against the unrounded product
                slack = (x.abs() * 2.0 ** -4 + s * 2.0 ** -10) @ wd.abs().t()
                _near(c["out"][0], x @ wd.t(), slack, 1.01, True)


@gpu
def test_generate_follows_its_rules():
    cfg = RecurrentConfig()
    m = RecurrentDecoder.random(cfg, max_seqs=4)
    prompts = [[5, 6, 7] * 20, [11], [3] * 300]
    base = m.generate(prompts, 8)
    assert m.generate(prompts, 8) == base and all(len(o) == 8 for o in base)
    # a large bias decides, a strong presence penalty forbids what is there
    assert m.generate(prompts, 3, bias=[{42: 1e4}, None, {9: 1e4}])[0] == [42] * 3
    free = m.generate(prompts, 8, presence=1e4)
    for p, o in zip(prompts, free):
        assert len(set(o)) == 8 and not set(o) & set(p)
    # a grammar that allows one token
    mask = torch.zeros(3, cfg.vocab_size // 32, dtype=torch.int32, device="cuda")
    mask[:, 2] = 1 << 5
    assert m.generate(prompts, 2, mask=mask) == [[69, 69]] * 3
    with pytest.raises(ValueError):
        m.generate([[1]] * 5, 1)
    with pytest.raises(ValueError):
        m.generate([[]], 1)
    with pytest.raises(RuntimeError):
        m.generate([[cfg.vocab_size + 3]], 1)


def test_config_rows_are_whole_16_byte_units():
    for h, dk, dv in ((4, 64, 128), (3, 64, 64), (5, 128, 64)):
        c = RecurrentConfig(n_heads=h, key_dim=dk, value_dim=dv)
        assert c.mixer_rows % 8 == 0 and 0 <= c.mixer_rows - h * (2 * dk + dv + 1) < 8
