"""A state-space decoder: a selective scan behind a short causal convolution in place of attention and feed-forward, so a
sequence's memory is one f32 state and a few inputs per layer however long it gets (reference src/mamba.rs).

A layer is the norm of the residual stream -> x | z projection -> ``causal_conv`` -> step | B | C projection -> step
projection -> ``selective_scan`` gated by z -> output projection; ``block_norm`` adds the output to the stream
(scaled, and normalised first in models with a norm after each block) and writes the next layer's input in one pass.
``token_logprobs`` scores prompts; the logits of generated tokens pass through ``logit_rules`` before the sampler.

    model = StateSpaceDecoder.random(StateSpaceConfig(), max_seqs=8)
    outs = model.generate([[1, 2, 3], [4, 5]], max_tokens=16)
    scores = model.score([[1, 2, 3, 4]], top=5)
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from .. import ops
from ..gguf import GGMLType
from ..ops import gemm


@dataclass
class StateSpaceConfig:
    n_layers: int = 2
    hidden_dim: int = 512
    inner_dim: int = 1024
    state_dim: int = 16
    step_rank: int = 64
    conv_width: int = 4
    vocab_size: int = 4096
    eps: float = 1e-5
    residual_scale: float = 1.0
    post_norm: bool = False      # a norm after each block, before the sum

    @property
    def selection_rows(self) -> int:
        """Rows of the step | B | C projection, rounded up to whole 16-byte rows of bf16."""
        return (self.step_rank + 2 * self.state_dim + 7) // 8 * 8


@dataclass
class StateSpaceLayer:
    norm: torch.Tensor           # [H] f32
    w_in: ops.QWeight            # [2 inner, H]: x | z
    conv_w: torch.Tensor         # [inner, width] f32
    conv_b: torch.Tensor         # [inner] f32
    w_select: ops.QWeight        # [selection_rows, inner]: step | B | C
    w_step: ops.QWeight          # [inner, step_rank]
    step_bias: torch.Tensor      # [inner] f32
    A: torch.Tensor              # [inner, states] f32, negative
    D: torch.Tensor              # [inner] f32
    w_out: ops.QWeight           # [H, inner]
    post_norm: torch.Tensor | None = None


class StateSpaceDecoder:
    def __init__(self, cfg: StateSpaceConfig, embd: ops.QWeight, layers: list[StateSpaceLayer], out_norm: torch.Tensor,
                 lm_head: ops.QWeight, max_seqs: int = 64):
        self.cfg, self.embd, self.layers, self.out_norm, self.lm_head = cfg, embd, layers, out_norm, lm_head
        self.device = out_norm.device
        self.max_seqs = max_seqs
        z = lambda *s, dtype: torch.zeros(*s, dtype=dtype, device=self.device)
        self.inputs = [z(max_seqs, cfg.conv_width - 1, cfg.inner_dim, dtype=torch.bfloat16) for _ in layers]
        self.states = [z(max_seqs, cfg.inner_dim, cfg.state_dim, dtype=torch.float32) for _ in layers]
        self.err = z(1, dtype=torch.int32)

    @classmethod
    def random(cls, cfg: StateSpaceConfig, max_seqs: int = 64, seed: int = 0, device="cuda") -> "StateSpaceDecoder":
        g = torch.Generator().manual_seed(seed)

        def dense(n, k):
            w = (torch.randn(n, k, generator=g) * k ** -0.5).to(torch.bfloat16).to(device)
            return ops.QWeight(ops.FMT_BF16, w, None, n, k, GGMLType.BF16)

        def norm():
            return (1.0 + 0.1 * torch.randn(cfg.hidden_dim, generator=g)).to(device)

        def layer():
            H, I, N = cfg.hidden_dim, cfg.inner_dim, cfg.state_dim
            # steps between 0.001 and 0.1, rates 1 .. N
            step = torch.exp(math.log(0.001) + torch.rand(I, generator=g) * math.log(100.0))
            return StateSpaceLayer(
                norm(), dense(2 * I, H), (torch.randn(I, cfg.conv_width, generator=g) * cfg.conv_width ** -0.5).to(device),
                (0.1 * torch.randn(I, generator=g)).to(device), dense(cfg.selection_rows, I), dense(I, cfg.step_rank),
                (step + torch.log(-torch.expm1(-step))).to(device), (-torch.arange(1.0, N + 1).expand(I, N)).contiguous().to(device),
                torch.ones(I, device=device), dense(H, I), norm() if cfg.post_norm else None)
        embd = dense(cfg.vocab_size, cfg.hidden_dim)
        return cls(cfg, embd, [layer() for _ in range(cfg.n_layers)], norm(), dense(cfg.vocab_size, cfg.hidden_dim), max_seqs)

    # ------------------------------------------------------------------ forward
    def _forward(self, ids: torch.Tensor, conv, scan, last: torch.Tensor | None) -> torch.Tensor:
        """Token ids [T] -> logits f32 of the rows ``last`` (None: all). ``conv(layer, i, x)`` and ``scan(layer, i, u, dt,
        B, C, z)`` run the i-th layer's convolution and recurrence."""
        cfg, T = self.cfg, ids.numel()
        I, N, R = cfg.inner_dim, cfg.state_dim, cfg.step_rank
        new = lambda n, dtype=torch.bfloat16: torch.empty(T, n, dtype=dtype, device=self.device)
        x = new(cfg.hidden_dim, torch.float32)
        ops.embed(self.embd, ids, out_f32=x, err=self.err)
        n, _ = ops.block_norm(x, self.layers[0].norm if self.layers else self.out_norm, cfg.eps)
        for i, w in enumerate(self.layers):
            xz = gemm.linear(n, w.w_in, new(2 * I), err=self.err)
            u = conv(w, i, xz[:, :I])
            sel = gemm.linear(u, w.w_select, new(cfg.selection_rows), err=self.err)
            dt = gemm.linear(sel[:, :R].contiguous(), w.w_step, new(I), err=self.err)
            y = scan(w, i, u, dt, sel[:, R:R + N], sel[:, R + N:R + 2 * N], xz[:, I:])
            y = gemm.linear(y, w.w_out, new(cfg.hidden_dim), err=self.err)
            after = self.layers[i + 1].norm if i + 1 < len(self.layers) else self.out_norm
            n, x = ops.block_norm(y, after, cfg.eps, residual=x, post_weight=w.post_norm, scale=cfg.residual_scale)
        if last is not None:
            n = n[last]
        logits = torch.empty(n.shape[0], cfg.vocab_size, dtype=torch.float32, device=self.device)
        return gemm.linear(n, self.lm_head, logits, err=self.err)

    def _prompts(self, prompts: list[list[int]], slots: torch.Tensor | None, resume: torch.Tensor | None,
                 every: bool) -> torch.Tensor:
        if any(not p for p in prompts):
            raise ValueError("a prompt has at least one token")
        if slots is not None and (slots.shape != (len(prompts),) or (resume is not None and resume.shape != slots.shape)):
            raise ValueError(f"one state row (and resume mark) for each of {len(prompts)} prompts")
        ids = torch.tensor([t for p in prompts for t in p], dtype=torch.int32, device=self.device)
        if not prompts:
            return torch.empty(0, self.cfg.vocab_size, device=self.device)
        cu = torch.tensor([0] + [len(p) for p in prompts], dtype=torch.int32, device=self.device).cumsum(0, dtype=torch.int32)

        def where(pool):
            return {} if slots is None else dict(state=pool, slots=slots, has_state=resume)

        def conv(w, i, x):
            return ops.causal_conv(x, w.conv_w, w.conv_b, cu_seqlens=cu, err=self.err, **where(self.inputs[i]))

        def scan(w, i, u, dt, B, C, z):
            return ops.selective_scan(u, dt, w.A, B, C, D=w.D, z=z, dt_bias=w.step_bias, cu_seqlens=cu, err=self.err,
                                      **where(self.states[i]))
        return self._forward(ids, conv, scan, None if every else cu[1:].long() - 1)

    def prefill(self, prompts: list[list[int]], slots: torch.Tensor, resume: torch.Tensor | None = None) -> torch.Tensor:
        """Runs the prompts packed together into the state rows ``slots`` (int32); ``resume`` (int32) marks those that
        continue what their row holds. Returns the logits of each last token."""
        return self._prompts(prompts, slots, resume, every=False)

    def decode(self, ids: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
        """One new token per sequence: ids [B] int32 -> logits [B, V]."""
        def conv(w, i, x):
            return ops.causal_conv_step(x, w.conv_w, self.inputs[i], w.conv_b, slots=slots, err=self.err)

        def scan(w, i, u, dt, B, C, z):
            return ops.selective_scan_step(u, dt, w.A, B, C, self.states[i], D=w.D, z=z, dt_bias=w.step_bias,
                                           slots=slots, err=self.err)
        return self._forward(ids, conv, scan, None)

    def _check(self):
        if code := int(self.err):
            self.err.zero_()
            raise RuntimeError(f"device kernel reported error code {code} (1=index out of range, 2=wait timed out)")

    # ------------------------------------------------------------------ generation and scoring
    def generate(self, prompts: list[list[int]], max_tokens: int, *, bias: list[dict[int, float] | None] | None = None,
                 mask: torch.Tensor | None = None) -> list[list[int]]:
        """Greedy continuation of each prompt under the request's biases and grammar mask (``ops.logit_rules``)."""
        B, dev = len(prompts), self.device
        if B > self.max_seqs:
            raise ValueError(f"generate: {B} prompts, {self.max_seqs} state rows")
        if not prompts or max_tokens <= 0:
            return [[] for _ in prompts]
        slots = torch.arange(B, dtype=torch.int32, device=dev)
        rules = dict(bias=ops.bias_lists(bias, dev) if bias else None, mask=mask, err=self.err)
        tokens = torch.zeros(B, dtype=torch.int32, device=dev)
        outs = []
        logits = self.prefill(prompts, slots)
        for step in range(max_tokens):
            ops.sample(ops.logit_rules(logits, **rules), tokens)
            outs.append(tokens.clone())
            if step + 1 < max_tokens:
                logits = self.decode(tokens, slots)
        out = torch.stack(outs, 1).tolist()
        self._check()
        return out

    def score(self, prompts: list[list[int]], top: int = 0) -> list[ops.TokenLogprobs]:
        """Log probabilities of each prompt's tokens after the first, given those before, with the entropies and ``top``
        alternatives (CPU tensors, one set a prompt). Leaves the state rows as they are."""
        if not prompts:
            return []
        logits = self._prompts(prompts, None, None, every=True)
        ids = torch.tensor([t for p in prompts for t in p[1:] + [-1]], dtype=torch.int32, device=self.device)
        r = ops.token_logprobs(logits, ids, top=top, err=self.err)
        r = [t.cpu() for t in r]
        self._check()
        out, at = [], 0
        for p in prompts:
            out.append(ops.TokenLogprobs(*(t[at:at + len(p) - 1] for t in r)))
            at += len(p)
        return out
