"""State rows and token counts of the recurrent decoder's slots."""
import pytest
import torch

from air_rs import ops
from air_rs.models.recurrent import RecurrentConfig, RecurrentDecoder

DEV = "cuda"
gpu = pytest.mark.gpu


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@gpu
def test_count_tokens_skips_rows_and_tokens_out_of_range():
    buf = torch.zeros(4, 8, dtype=torch.uint8, device=DEV)
    ops.count_tokens(buf[:2], _i32(1, 2, 3, 4, 8, -1), count_row=_i32(0, 2, 1, -1, 0, 0))
    want = torch.zeros(4, 8, dtype=torch.uint8)
    want[0, 1] = want[1, 3] = 1
    assert torch.equal(buf.cpu(), want)
    ops.count_tokens(buf[:2], _i32(5, 5, 5))                     # three tokens, two rows
    want[0, 5] = want[1, 5] = 1
    assert torch.equal(buf.cpu(), want)


def _counts(m, prompts):
    want = torch.zeros(m.max_seqs, m.cfg.vocab_size, dtype=torch.int64)
    for slot, ids in prompts.items():
        want[slot] = torch.bincount(torch.tensor(ids), minlength=m.cfg.vocab_size)
    return want.clamp(max=255)


@gpu
def test_a_reused_slot_starts_with_its_own_counts():
    m = RecurrentDecoder.random(RecurrentConfig(), max_seqs=4)
    m.prefill([[1, 2, 2], [5] * 300], _i32(3, 1))
    assert torch.equal(m.counts.cpu().long(), _counts(m, {3: [1, 2, 2], 1: [5] * 300}))
    # slot 3 goes to another request, slot 1 continues, slot 0 is new
    m.prefill([[7, 1], [5, 6], [9]], _i32(3, 1, 0), resume=_i32(0, 1, 0))
    assert torch.equal(m.counts.cpu().long(), _counts(m, {3: [7, 1], 1: [5] * 302 + [6], 0: [9]}))
    # rows out of range change nothing, and are reported
    before = m.counts.clone()
    m.prefill([[2], [3]], _i32(-1, 4))
    assert torch.equal(m.counts, before) and int(m.err) == 1
    for bad in (dict(slots=_i32(0)), dict(slots=_i32(0, 1), resume=_i32(1))):
        with pytest.raises(ValueError):
            m.prefill([[2], [3]], **bad)
    assert torch.equal(m.counts, before)


@gpu
def test_generate_does_not_see_an_earlier_request():
    cfg = RecurrentConfig()
    m = RecurrentDecoder.random(cfg, max_seqs=2)
    prompts = [[5, 6, 7], [11]]
    first = m.generate(prompts, 6, presence=1e4)
    m.generate([[1, 2, 3] * 50], 20, presence=1e4)
    assert m.generate(prompts, 6, presence=1e4) == first


@gpu
def test_errors_without_a_word_of_ones_own_are_raised_once():
    ops.check_errors()
    q = torch.randn(1, 2, 64, device=DEV)
    pool = torch.zeros(2, 2, 64, 64, device=DEV)
    g = torch.zeros(2, device=DEV)
    ops.linear_attention_step(q, q, q, g, pool, slots=_i32(1))
    ops.check_errors(q.device)
    ops.linear_attention_step(q, q, q, g, pool, slots=_i32(2))
    with pytest.raises(RuntimeError, match="code 1"):
        ops.check_errors(q.device)
    ops.check_errors()
    ops.linear_attention_step(q, q, q, g, pool, slots=_i32(2), err=_i32(0))     # a word of one's own
    ops.check_errors("cuda:0")
    ops.linear_attention_step(q, q, q, g, pool, slots=_i32(-3))
    with pytest.raises(RuntimeError):
        ops.check_errors("cuda")
