"""Outputs whose rows share memory are refused; any other strides are taken."""
import pytest
import torch

from air_rs import ops
from test_recurrent_ops import _inputs

DEV = "cuda"
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("T", [40, 4])
def test_linear_attention_outputs(T):
    H, d = 4, 64
    q, k, v, g = (x.to(DEV) for x in _inputs(1, T, H, H, H, H, d, d, torch.bfloat16))
    want = ops.linear_attention(q, k, v, g)
    new = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)
    for out in (new(H, T, d).transpose(0, 1), new(T, H, 2 * d)[..., :d], new(2 * T, H, d)[::2], new(T, 2 * H, d)[:, ::2]):
        assert ops.linear_attention(q, k, v, g, out=out) is not None and torch.equal(out, want)
    pool = torch.zeros(T, H, d, d, device=DEV)
    for out in (new(1, H, d).expand(T, H, d), new(T, 1, d).expand(T, H, d), new(T * H * d).as_strided((T, H, d), (H * d, d // 2, 1)),
                new(T * H * d).as_strided((T, H, d), (d, d, 1))):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.linear_attention(q, k, v, g, out=out)
        with pytest.raises(RuntimeError, match="overlap"):
            ops.linear_attention_step(q, k, v, g, pool, out=out)
    one = new(1, 1, d).expand(1, 1, d)                       # one row: its strides are never used
    ops.linear_attention(q[:1, :1], k[:1, :1], v[:1, :1], g[:1, :1], out=one)


@gpu
def test_norm_and_rules_outputs():
    x, y, w = torch.randn(1, 256, device=DEV).expand(4, 256), torch.randn(4, 256, device=DEV), torch.ones(256, device=DEV)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.add_rmsnorm_fp8(x, y, w, 1e-5)                   # the sum would go back into x
    with pytest.raises(RuntimeError, match="overlap"):
        ops.add_rmsnorm_fp8(y, None, w, 1e-5, out_bf16=torch.zeros(1, 256, dtype=torch.bfloat16, device=DEV).expand(4, 256))
    res = torch.empty(4, 256, device=DEV)
    a, b = ops.add_rmsnorm_fp8(x, y, w, 1e-5, resid_out=res), ops.add_rmsnorm_fp8(x.contiguous(), y, w, 1e-5)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(res, x + y)
    lg = torch.randn(1, 64, device=DEV).expand(3, 64)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.logit_rules(lg)
    assert torch.equal(ops.logit_rules(lg, out=torch.empty(3, 64, device=DEV)), lg)
    assert ops.logit_rules(lg[:1]).shape == (1, 64)
