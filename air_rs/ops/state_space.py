"""Operators of a state-space decoder: the short causal convolution and the selective scan (for prompts and for single
tokens), the norms around a block with its gate and residual scale, and log probabilities of given tokens.

All take CUDA tensors, run on the current stream without synchronising and can be captured in CUDA graphs. Arguments
that the host can see are checked before the launch (RuntimeError); indices that live on the device are checked in the
kernel, which skips what they name and sets ``err`` (by default the device's shared error word, which
``ops.check_errors`` reads and clears). Outputs whose rows overlap, or that share memory with another operand, are
refused but where in-place use is named.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import count_launch, require_ext
from .recurrent import _err

GATES = {"silu": 0, "sigmoid": 1, "none": 2}


def causal_conv(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, *,
                state: torch.Tensor | None = None, cu_seqlens: torch.Tensor | None = None,
                slots: torch.Tensor | None = None, has_state: torch.Tensor | None = None, silu: bool = True,
                out: torch.Tensor | None = None, err: torch.Tensor | None = None) -> torch.Tensor:
    """Depthwise causal convolution over packed prompts (reference src/gated_deltanet.rs, src/mamba.rs):

        y[t, d] = act(bias[d] + sum_j w[d, j] x[t - W + 1 + j, d])

    x [T, D] bf16 or f32 (any token stride, rows contiguous), w f32 [D, W] with 2 <= W <= 4, bias f32 [D]; act is SiLU
    unless ``silu`` is false. ``cu_seqlens`` int32 [N + 1]: sequence n is tokens cu[n] .. cu[n + 1] - 1, empty ones
    allowed (None: one sequence). ``state`` [S, W - 1, D] of x's type holds the last inputs of each sequence, the newest
    in its last row: sequence n uses row ``slots[n]`` (None: n; -1: starts from zeros and keeps nothing), starts from
    it where ``has_state[n]`` (int32; None: every sequence starts from zeros) and replaces it. Rows of one call are
    distinct. A state row out of range is reported and counts as -1, a sequence with bad offsets is reported and
    skipped, and keeps its state. Tokens outside every sequence are not written. Returns out [T, D] in x's type."""
    out = require_ext().causal_conv(x, w, bias, state, cu_seqlens, slots, has_state, silu, out,
                                    _err(x) if err is None else err)
    count_launch()
    return out


def causal_conv_step(x: torch.Tensor, w: torch.Tensor, state: torch.Tensor, bias: torch.Tensor | None = None, *,
                     slots: torch.Tensor | None = None, silu: bool = True, out: torch.Tensor | None = None,
                     err: torch.Tensor | None = None) -> torch.Tensor:
    """One new token per sequence of :func:`causal_conv`: row n of x [B, D] follows the inputs in state row
    ``slots[n]`` (None: n), which moves on in place. Slot -1 is a padding row: no state, output zero."""
    out = require_ext().causal_conv_step(x, w, state, bias, slots, silu, out, _err(x) if err is None else err)
    count_launch()
    return out


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, *,
                   D: torch.Tensor | None = None, z: torch.Tensor | None = None, dt_bias: torch.Tensor | None = None,
                   softplus: bool = True, state: torch.Tensor | None = None, cu_seqlens: torch.Tensor | None = None,
                   slots: torch.Tensor | None = None, has_state: torch.Tensor | None = None,
                   out: torch.Tensor | None = None, err: torch.Tensor | None = None) -> torch.Tensor:
    """Selective state-space scan over packed prompts (reference src/mamba.rs):

        delta = softplus(dt + dt_bias)          (dt + dt_bias without ``softplus``)
        h_t = exp(delta A) h_{t-1} + delta x B,     y_t = (C . h_t + D x) silu(z)

    x, dt and z [T, D] in bf16 or f32 (one type, any token strides, rows contiguous); A f32 [D, N], N <= 256; B and C
    [T, N] or [T, G, N] of the same type (G divides D, channel d reads group d // (D / G)); D and dt_bias f32 [D].
    ``cu_seqlens``, ``slots``, ``has_state`` and what is reported are those of :func:`causal_conv`; ``state`` is
    f32 [S, D, N], updated in place. h, delta and the sums are f32; y is rounded once, to x's type. A state that holds an
    infinity keeps it where it decays fast and may become NaN where |delta A| <= 1/32. More than 64 states, and calls of
    fewer than six tokens a sequence on average, run token by token (about a microsecond for each token of the longest
    sequence): single tokens that are batched with a long prompt belong in a call of :func:`selective_scan_step`."""
    out = require_ext().selective_scan(x, dt, A, B, C, D, z, dt_bias, softplus, state, cu_seqlens, slots, has_state,
                                       out, _err(x) if err is None else err)
    count_launch()
    return out


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                        state: torch.Tensor, *, D: torch.Tensor | None = None, z: torch.Tensor | None = None,
                        dt_bias: torch.Tensor | None = None, softplus: bool = True,
                        slots: torch.Tensor | None = None, out: torch.Tensor | None = None,
                        err: torch.Tensor | None = None) -> torch.Tensor:
    """One new token per sequence of :func:`selective_scan`: row n of x [B, D], dt, z, B and C advances state row
    ``slots[n]`` (None: n) in place. Slot -1 is a padding row: no state, output zero."""
    out = require_ext().selective_scan_step(x, dt, A, B, C, state, D, z, dt_bias, softplus, slots, out,
                                            _err(x) if err is None else err)
    count_launch()
    return out


def block_norm(y: torch.Tensor, weight: torch.Tensor | None, eps: float, *, residual: torch.Tensor | None = None,
               post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, gate_act: str = "silu",
               scale: float | torch.Tensor = 1.0, w_offset: float = 0.0, out: torch.Tensor | None = None,
               resid_out: torch.Tensor | None = None) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """From a block's output y to the next block's input, every step but the sum optional:

        h = y * rsqrt(mean(y^2) + eps) * (post_weight + w_offset)
        h = h * act(gate)
        r = residual + scale * h
        out = r * rsqrt(mean(r^2) + eps) * (weight + w_offset)

    y [T, K] bf16 or f32, K <= 32768; ``gate`` [T, K] or [K] of y's type through ``gate_act`` "silu", "sigmoid" or
    "none"; ``residual`` [T, K] f32 or bf16; ``scale`` a number or f32 [K]; the weights f32 [K]. Without a residual
    r = scale * h (a gated norm alone: ``post_weight`` for norm before gate, ``weight`` for gate before norm).
    r goes to ``resid_out`` (None: back into ``residual`` when there is one), rounded to the residual's type; out is
    the norm of the unrounded r, in bf16 unless ``out`` is given; with ``weight`` None it is r itself, and written only
    when given or when there is no residual. Rows of any stride, contiguous. Returns (out or None, resid_out or None)."""
    if gate_act not in GATES:
        raise ValueError(f"block_norm: gate_act must be one of {', '.join(GATES)}, not {gate_act!r}")
    if resid_out is None:
        resid_out = residual
    row = scale if isinstance(scale, torch.Tensor) else None
    made, _ = require_ext().block_norm(y, weight, eps, residual, post_weight, gate, GATES[gate_act],
                                       1.0 if row is not None else float(scale), row, w_offset, out,
                                       out is None and (weight is not None or residual is None), resid_out)
    count_launch()
    return made if out is None else out, resid_out


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor        # f32 [T]
    entropy: torch.Tensor         # f32 [T]
    top_logprobs: torch.Tensor    # f32 [T, top]
    top_ids: torch.Tensor         # int32 [T, top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, top: int = 0,
                   err: torch.Tensor | None = None) -> TokenLogprobs:
    """Log probabilities under softmax(logits), logits [T, V] bf16 or f32 (any row stride, rows contiguous): of
    ``tokens`` int32 [T] (None or -1: none, 0 is returned; an id out of range is reported and counts as -1), each row's
    entropy in nats, and the ``top`` <= 32 most likely tokens, the lowest id first among equals.

    Logits of -inf are tokens of probability zero: their log probability is -inf and they are no alternatives, for
    which id -1 and -inf stand where fewer than ``top`` are left. A row of only -inf has entropy 0. A row with NaN or
    +inf gives NaN, and ids of -1."""
    r = require_ext().token_logprobs(logits, tokens, top, _err(logits) if err is None else err)
    count_launch()
    return TokenLogprobs(*r)
