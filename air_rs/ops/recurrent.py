"""Operators of a recurrent (linear-attention) decoder's serving step: linear attention with one
decay per head for prompts and for single tokens, the residual add + RMSNorm that writes the E4M3
rows of the W8A8 projections, and the rules a request puts on its logits.

All take CUDA tensors, run on the current stream without synchronising and can be captured in CUDA
graphs. Arguments that the host can see are checked before the launch (RuntimeError); indices that
live on the device are checked in the kernel, which skips the row and sets ``err`` (by default the
device's shared error word, which ``ops.check_errors`` reads and clears). A state or count row out of range is reported and counts as -1.
Outputs whose rows overlap or interleave in memory are refused; an output shares no memory with other operands
except where in-place use is named.
"""
from __future__ import annotations

import torch

from . import count_launch, require_ext
from .gemm import workspace

_ERR: dict = {}


def _err(t: torch.Tensor) -> torch.Tensor:
    """The shared error word of t's device."""
    e = _ERR.get(t.device)
    if e is None:
        e = _ERR[t.device] = workspace(t.device).err
    return e


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *,
                     state: torch.Tensor | None = None, cu_seqlens: torch.Tensor | None = None,
                     slots: torch.Tensor | None = None, has_state: torch.Tensor | None = None,
                     scale: float | None = None, out: torch.Tensor | None = None,
                     err: torch.Tensor | None = None) -> torch.Tensor:
    """Causal linear attention with a decay per head over packed prompts:

        S_t = exp(g_t) S_{t-1} + v_t k_t^T,    o_t = scale * S_t q_t

    q [T, Hq, dk], k [T, Hk, dk], v [T, Hv, dv] in bf16 or f32 (any token and head strides, last
    dimension contiguous); ``log_decay`` g f32 [H] or [T, H], at most 0 for a decay (-inf forgets
    everything before the token). Hq, Hk and Hv divide H; head h reads head h // (H / Hx). dk <= 256.

    ``cu_seqlens`` int32 [N + 1]: sequence n is tokens cu[n] .. cu[n + 1] - 1, empty ones allowed
    (None: one sequence). ``state`` f32 [S, H, dv, dk] is updated in place: sequence n uses row
    ``slots[n]`` (None: n; -1: starts from zeros and keeps nothing) and starts from that row where
    ``has_state[n]`` (int32; None: every sequence starts from zeros). Rows of one call are distinct.
    Returns out [T, H, dv] in q's type. bf16 prompts with head sizes 64 / 128 run on the tensor
    cores in blocks of 128 tokens, unless there are 12 tokens or fewer or less than 1.5 a sequence
    (empty ones counted), which like all others run token by token. In blocks the decayed scores and
    the state's copy that the queries read are rounded to bf16 (an output error of 2.35e-3 where one
    rounding of exact outputs has 1.66e-3); the state itself stays f32. No token reaches the outputs of
    earlier ones, also where it holds NaN or infinities; in blocks an infinity in k or v may become NaN,
    and in v it makes its column's outputs NaN from its token on. Tokens outside every sequence are not
    written.
    """
    out = require_ext().linear_attention(q, k, v, log_decay, state, cu_seqlens, slots, has_state, scale, out,
                                         _err(q) if err is None else err)
    count_launch()
    return out


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                          state: torch.Tensor, *, slots: torch.Tensor | None = None, scale: float | None = None,
                          out: torch.Tensor | None = None, err: torch.Tensor | None = None) -> torch.Tensor:
    """One new token per sequence of :func:`linear_attention`: row n of q [B, Hq, dk], k, v and
    ``log_decay`` ([H] or [B, H]) advances state row ``slots[n]`` (None: n) in place. Slot -1 is a
    padding row: no state, output zero. Rows of one call are distinct. Returns out [B, H, dv]."""
    out = require_ext().linear_attention_step(q, k, v, log_decay, state, slots, scale, out,
                                              _err(q) if err is None else err)
    count_launch()
    return out


def add_rmsnorm_fp8(x: torch.Tensor, y: torch.Tensor | None, w: torch.Tensor, eps: float, *, w_offset: float = 0.0,
                    resid_out: torch.Tensor | None = None, xq: torch.Tensor | None = None,
                    xs: torch.Tensor | None = None, out_bf16: torch.Tensor | None = None):
    """r = x + y; n = r * rsqrt(mean(r^2) + eps) * (w + w_offset); E4M3 codes of n / s with one scale
    s = max|n| / 448 per row, ready for ``gemm.linear_fp8_rows``.

    x f32 [T, K] is the residual stream, y bf16 / f32 [T, K] (None: nothing is added), K a multiple
    of 8 up to 32768. r goes to ``resid_out`` (None: back into x when there is a y), n also to
    ``out_bf16`` when given. Returns (codes uint8 [T, K], scales f32 [T])."""
    if resid_out is None and y is not None:
        resid_out = x
    codes = require_ext().add_rmsnorm_fp8(x, y, w, eps, w_offset, resid_out, xq, xs, out_bf16)
    count_launch()
    return codes


def logit_rules(logits: torch.Tensor, *, out: torch.Tensor | None = None, counts: torch.Tensor | None = None,
                count_row: torch.Tensor | None = None, repetition: torch.Tensor | None = None,
                frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                bias: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None,
                mask: torch.Tensor | None = None, err: torch.Tensor | None = None) -> torch.Tensor:
    """Penalties, biases and the grammar mask on logits [B, V] (f32 or bf16), in this order:

        x / rho^c if x > 0 else x * rho^c;   x - c * frequency - [c > 0] * presence;
        x + bias[token];   -inf where the allow bit is 0

    c is the token's count in row ``count_row[b]`` (None: b; -1: no counts) of ``counts`` uint8
    [S, V] (the sampler's occurrence counts); ``repetition`` / ``frequency`` / ``presence`` f32 [B];
    ``bias`` (ptr int32 [B + 1], ids int32, values f32) as :func:`bias_lists` builds it, repeated ids
    add up in list order; ``mask`` int32 [B, ceil(V / 32)] allow bits. Writes f32 to ``out`` (None:
    in place for f32 logits, a new tensor for bf16) and returns it. A masked entry is -inf whatever
    its logit was; a row whose mask allows nothing is all -inf. Penalties over different counts
    (repetition over prompt and output, frequency and presence over the output) are two calls."""
    if out is None:
        out = logits if logits.dtype == torch.float32 else torch.empty(logits.shape, dtype=torch.float32, device=logits.device)
    if err is None:
        err = _err(logits)
    ptr, ids, vals = bias if bias is not None else (None, None, None)
    require_ext().logit_rules(logits, out, counts, count_row, repetition, frequency, presence, ptr, ids, vals, mask, err)
    count_launch()
    return out


def bias_lists(rows: list[dict[int, float] | None], device) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None:
    """Per-row {token: bias} maps -> (ptr, ids, values) for :func:`logit_rules`; None when no row has any."""
    ptr, ids, vals = [0], [], []
    for r in rows:
        for t in sorted(r or {}):
            ids.append(int(t))
            vals.append(float(r[t]))
        ptr.append(len(ids))
    if not ids:
        return None
    return (torch.tensor(ptr, dtype=torch.int32, device=device), torch.tensor(ids, dtype=torch.int32, device=device),
            torch.tensor(vals, dtype=torch.float32, device=device))
