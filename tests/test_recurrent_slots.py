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
