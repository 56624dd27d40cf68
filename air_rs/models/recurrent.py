"""A recurrent decoder served in FP8: linear attention with one decay per head in place of softmax
attention, so a sequence's memory is one f32 state per layer and head however long it gets.

A layer is ``add_rmsnorm_fp8`` -> q | k | v | decay projection -> ``linear_attention`` (prompts) or
``linear_attention_step`` (one token per sequence) -> output projection, then ``add_rmsnorm_fp8`` ->
gate | up -> SwiGLU -> down. Every projection is a W8A8 product of block-scaled FP8 weights; the two
norms write its E4M3 rows directly. The logits pass through ``logit_rules`` before the sampler.

    model = RecurrentDecoder.random(RecurrentConfig(), max_seqs=8)
    outs = model.generate([[1, 2, 3], [4, 5]], max_tokens=16, frequency=0.4, bias=[{7: 2.0}, None])
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import ops
from ..gguf import GGMLType
from ..ops import gemm


@dataclass
class RecurrentConfig:
    n_layers: int = 2
    hidden_dim: int = 512
    n_heads: int = 4
    key_dim: int = 64            # per head
    value_dim: int = 128         # per head
    intermediate_dim: int = 1024
    vocab_size: int = 4096
    eps: float = 1e-5

    @property
    def mixer_rows(self) -> int:
        """Rows of the fused projection: q | k | v | decay, rounded up to whole 16-byte rows of bf16."""
        n = self.n_heads * (2 * self.key_dim + self.value_dim + 1)
        return (n + 7) // 8 * 8


@dataclass
class RecurrentLayer:
    mixer_norm: torch.Tensor     # [H] f32
    w_mixer: ops.QWeight         # [mixer_rows, hidden]
    rate: torch.Tensor           # [heads] f32, the decay of a zero projection is -rate ln 2
    w_out: ops.QWeight           # [hidden, heads * value_dim]
    ffn_norm: torch.Tensor
    w_gate_up: ops.QWeight       # [2 * intermediate, hidden]
    w_down: ops.QWeight          # [hidden, intermediate]


class RecurrentDecoder:
    def __init__(self, cfg: RecurrentConfig, embd: ops.QWeight, layers: list[RecurrentLayer], out_norm: torch.Tensor,
                 lm_head: ops.QWeight, max_seqs: int = 64):
        self.cfg, self.embd, self.layers, self.out_norm, self.lm_head = cfg, embd, layers, out_norm, lm_head
        self.device = out_norm.device
        self.max_seqs = max_seqs
        z = lambda *s, dtype: torch.zeros(*s, dtype=dtype, device=self.device)
        self.states = [z(max_seqs, cfg.n_heads, cfg.value_dim, cfg.key_dim, dtype=torch.float32) for _ in layers]
        self.counts = z(max_seqs, cfg.vocab_size, dtype=torch.uint8)
        self.err = z(1, dtype=torch.int32)

    @classmethod
    def random(cls, cfg: RecurrentConfig, max_seqs: int = 64, seed: int = 0, device="cuda") -> "RecurrentDecoder":
        g = torch.Generator().manual_seed(seed)

        def fp8(n, k):
            codes = torch.randn(n, k, generator=g).clamp(-4, 4).to(torch.float8_e4m3fn).view(torch.uint8)
            scales = (0.75 + 0.5 * torch.rand(n, k // 128, generator=g)) * k ** -0.5
            return ops.QWeight(ops.FMT_FP8, codes.to(device), scales.to(device), n, k, GGMLType.FP8_E4M3_B128)

        def norm():
            return (1.0 + 0.1 * torch.randn(cfg.hidden_dim, generator=g)).to(device)

        H, F = cfg.hidden_dim, cfg.intermediate_dim
        table = torch.randn(cfg.vocab_size, H, generator=g).to(torch.bfloat16).to(device)
        embd = ops.QWeight(ops.FMT_BF16, table, None, cfg.vocab_size, H, GGMLType.F16)
        rate = torch.exp2(-1.0 - 6.0 * torch.arange(cfg.n_heads) / cfg.n_heads).to(device)
        layers = [RecurrentLayer(norm(), fp8(cfg.mixer_rows, H), rate, fp8(H, cfg.n_heads * cfg.value_dim), norm(),
                                 fp8(2 * F, H), fp8(H, F)) for _ in range(cfg.n_layers)]
        return cls(cfg, embd, layers, norm(), fp8(cfg.vocab_size, H), max_seqs)

    # ------------------------------------------------------------------ forward
    def _forward(self, ids: torch.Tensor, mixer, last: torch.Tensor | None) -> torch.Tensor:
        """Token ids [T] -> logits f32 of the rows ``last`` (None: all). ``mixer(layer, q, k, v, g)``
        runs the layer's recurrence and returns [T, heads, value_dim] bf16."""
        cfg, T, dev = self.cfg, ids.numel(), self.device
        h, dk, dv, F = cfg.n_heads, cfg.key_dim, cfg.value_dim, cfg.intermediate_dim
        new = lambda n, dtype=torch.bfloat16: torch.empty(T, n, dtype=dtype, device=dev)
        x, y = new(cfg.hidden_dim, torch.float32), None
        ops.embed(self.embd, ids, out_f32=x, err=self.err)
        for i, w in enumerate(self.layers):
            xq, xs = ops.add_rmsnorm_fp8(x, y, w.mixer_norm, cfg.eps)
            p = gemm.linear_fp8_rows(xq, xs, w.w_mixer, new(cfg.mixer_rows), err=self.err)
            q, k, v = (p[:, a:a + h * d].unflatten(1, (h, d)) for a, d in ((0, dk), (h * dk, dk), (2 * h * dk, dv)))
            at = h * (2 * dk + dv)
            g = -torch.nn.functional.softplus(p[:, at:at + h].float()) * w.rate
            o = mixer(i, q, k, v, g)
            y = gemm.linear_fp8(o.view(T, h * dv), w.w_out, new(cfg.hidden_dim), err=self.err)
            xq, xs = ops.add_rmsnorm_fp8(x, y, w.ffn_norm, cfg.eps)
            gu = gemm.linear_fp8_rows(xq, xs, w.w_gate_up, new(2 * F), err=self.err)
            act = new(F)
            ops.swiglu(gu, T, F, out_bf16=act)
            y = gemm.linear_fp8(act, w.w_down, new(cfg.hidden_dim), err=self.err)
        if last is not None:
            x, y = x[last], y[last]
        xq, xs = ops.add_rmsnorm_fp8(x, y, self.out_norm, cfg.eps)
        logits = torch.empty(x.shape[0], cfg.vocab_size, dtype=torch.float32, device=dev)
        return gemm.linear_fp8_rows(xq, xs, self.lm_head, logits, err=self.err)

    def prefill(self, prompts: list[list[int]], slots: torch.Tensor, resume: torch.Tensor | None = None) -> torch.Tensor:
        """Runs the prompts packed together into the state rows ``slots`` (int32); ``resume`` (int32)
        marks those that continue what their row holds, the others start from a zero state and zero
        counts. Returns the logits of each last token."""
        if any(not p for p in prompts):
            raise ValueError("prefill: a prompt has at least one token")
        if slots.shape != (len(prompts),) or (resume is not None and resume.shape != slots.shape):
            raise ValueError(f"prefill: one state row (and resume mark) for each of {len(prompts)} prompts")
        ids = torch.tensor([t for p in prompts for t in p], dtype=torch.int32, device=self.device)
        cu = torch.tensor([0] + [len(p) for p in prompts], dtype=torch.int32, device=self.device).cumsum(0, dtype=torch.int32)
        fresh = torch.ones_like(slots, dtype=torch.bool) if resume is None else resume == 0
        rows = torch.arange(self.max_seqs, device=self.device)
        self.counts.masked_fill_(((rows[:, None] == slots) & fresh).any(1, keepdim=True), 0)
        of_token = torch.tensor([n for n, p in enumerate(prompts) for _ in p], dtype=torch.int64, device=self.device)
        ops.count_tokens(self.counts, ids, count_row=slots[of_token], per_row=1)

        def mixer(i, q, k, v, g):
            return ops.linear_attention(q, k, v, g, state=self.states[i], cu_seqlens=cu, slots=slots, has_state=resume,
                                        scale=1.0 / self.cfg.key_dim, err=self.err)
        return self._forward(ids, mixer, cu[1:].long() - 1)

    def decode(self, ids: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
        """One new token per sequence: ids [B] int32 -> logits [B, V]."""
        def mixer(i, q, k, v, g):
            return ops.linear_attention_step(q, k, v, g, self.states[i], slots=slots, scale=1.0 / self.cfg.key_dim,
                                             err=self.err)
        return self._forward(ids, mixer, None)

    # ------------------------------------------------------------------ generation
    def generate(self, prompts: list[list[int]], max_tokens: int, *, repetition: float = 1.0, frequency: float = 0.0,
                 presence: float = 0.0, bias: list[dict[int, float] | None] | None = None,
                 mask: torch.Tensor | None = None) -> list[list[int]]:
        """Greedy continuation of each prompt under the request's logit rules."""
        B, dev = len(prompts), self.device
        if B > self.max_seqs:
            raise ValueError(f"generate: {B} prompts, {self.max_seqs} state rows")
        if not prompts:
            return []
        slots = torch.arange(B, dtype=torch.int32, device=dev)
        row = lambda v: torch.full((B,), float(v), dtype=torch.float32, device=dev)
        rules = dict(counts=self.counts, count_row=slots, repetition=row(repetition), frequency=row(frequency),
                     presence=row(presence), bias=ops.bias_lists(bias, dev) if bias else None, mask=mask, err=self.err)
        tokens = torch.zeros(B, dtype=torch.int32, device=dev)
        outs = []
        logits = self.prefill(prompts, slots)
        for step in range(max_tokens):
            ops.sample(ops.logit_rules(logits, **rules), tokens)
            ops.count_tokens(self.counts, tokens, count_row=slots)
            outs.append(tokens.clone())
            if step + 1 < max_tokens:
                logits = self.decode(tokens, slots)
        out = torch.stack(outs, 1).tolist() if outs else [[] for _ in prompts]
        if code := int(self.err):
            self.err.zero_()
            raise RuntimeError(f"device kernel reported error code {code} (1=index out of range, 2=wait timed out)")
        return out
