"""Operands of linear_fp8_rows: any code and scale rows a caller has are either taken or refused."""
import pytest
import torch

from air_rs import ops
from air_rs.gguf import GGMLType
from air_rs.ops import gemm

DEV = "cuda"
gpu = pytest.mark.gpu


def _weight(N, K, seed=3):
    r = torch.Generator().manual_seed(seed)
    codes = (torch.randn(N, K, generator=r) * 2).to(torch.float8_e4m3fn)
    sc = torch.rand(N, K // 128, generator=r) * 0.02 + 0.001
    w = ops.QWeight(ops.FMT_FP8, codes.view(torch.uint8).to(DEV), sc.to(DEV), N, K, GGMLType.FP8_E4M3_B128)
    return w, codes.double() * sc.double().repeat_interleave(128, 1)


@gpu
@pytest.mark.parametrize("T", [1, 5, 130])
def test_code_rows_of_either_type(T):
    N, K = 200, 256
    w, wd = _weight(N, K)
    r = torch.Generator().manual_seed(T)
    codes = (torch.randn(T, K, generator=r) * 3).to(torch.float8_e4m3fn)
    xs = torch.rand(T, generator=r) + 0.5
    a = gemm.linear_fp8_rows(codes.view(torch.uint8).to(DEV), xs.to(DEV), w, torch.empty(T, N, device=DEV))
    b = gemm.linear_fp8_rows(codes.to(DEV), xs.to(DEV)[:, None], w, torch.empty(T, N + 3, device=DEV)[:, :N])
    x = codes.double() * xs.double()[:, None]
    # the tensor cores' f32 sum keeps at least 2^-13 of the largest term of an accumulation step
    assert bool(((a.cpu().double() - x @ wd.t()).abs() <= 2.0 ** -12 * (x.abs() @ wd.abs().t())).all())
    assert torch.equal(a, b)


@gpu
def test_refusals():
    T, N, K = 4, 200, 256
    w, _ = _weight(N, K)
    xq, xs = torch.zeros(T, K, dtype=torch.uint8, device=DEV), torch.ones(T, device=DEV)
    out = torch.empty(T, N, device=DEV)
    for call in (lambda: gemm.linear_fp8_rows(xq.float(), xs, w, out), lambda: gemm.linear_fp8_rows(xq.int(), xs, w, out),
                 lambda: gemm.linear_fp8_rows(xq[:, :128], xs, w, out), lambda: gemm.linear_fp8_rows(xq, xs.double(), w, out),
                 lambda: gemm.linear_fp8_rows(xq, xs[:3], w, out), lambda: gemm.linear_fp8_rows(xq, xs.cpu(), w, out),
                 lambda: gemm.linear_fp8_rows(xq, xs[:1].expand(T), w, out), lambda: gemm.linear_fp8_rows(xq, xs, w, out.cpu()),
                 lambda: gemm.linear_fp8_rows(xq, torch.ones(T, 2, device=DEV)[:, 0], w, out),
                 lambda: gemm.linear_fp8_rows(xq, xs, w, out[:3]), lambda: gemm.linear_fp8_rows(xq, xs, w, out[0]),
                 lambda: gemm.linear_fp8_rows(xq, xs, w, out[:1].expand(T, N)), lambda: gemm.linear_fp8_rows(xq, xs, w, out.half()),
                 lambda: gemm.linear_fp8_rows(xq, xs, w, out, err=torch.zeros(1, dtype=torch.int32)),
                 lambda: gemm.linear_fp8_rows(xq, xs, w, out, err=torch.zeros(1, device=DEV))):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        gemm.linear_fp8_rows(xq, xs, ops.QWeight(ops.FMT_BF16, out.bfloat16(), None, T, N, GGMLType.F16), out)
    assert gemm.linear_fp8_rows(xq[:0], xs[:0], w, out[:0]).shape == (0, N)
    assert gemm.linear_fp8(torch.empty(0, K, dtype=torch.bfloat16, device=DEV), w, out[:0]).shape == (0, N)


@gpu
def test_a_decoder_takes_no_prompts():
    from air_rs.models.recurrent import RecurrentConfig, RecurrentDecoder
    m = RecurrentDecoder.random(RecurrentConfig(), max_seqs=2)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    assert m.prefill([], none).shape == (0, m.cfg.vocab_size) and m.decode(none, none).shape == (0, m.cfg.vocab_size)
    assert m.generate([], 3) == [] and m.generate([[1]], 0) == [[]]
    assert not m.counts[1].any() and int(m.err) == 0
