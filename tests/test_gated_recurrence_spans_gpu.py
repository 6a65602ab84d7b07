"""The gated recurrence on rows that are cut into long spans, against the formulas in 64 bits: in the pass over spans a warp takes more steps than
its ring has stages, so that stages are filled again, and the row's last block, which is short, is the first one backward."""
import pytest
import torch

import test_gated_recurrence_gpu as R

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


# (on 148 SMs: 7 to 18 spans; 7 to 9 steps of 8 tokens a warp, in fp32 14 to 18 of 4; the last warp of the last span takes 5 and more.  The widths are
# whole 16-byte pieces, whole words and neither.)
@pytest.mark.parametrize("T,D", [(3005, 5120), (3005, 5122), (3005, 5121), (10003, 1024), (10001, 1022)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_stages_that_are_filled_again(T, D, dtype):
    R.check(c := R.case(T + D, 1, T, D, dtype), R.train(c))


@pytest.mark.parametrize("rest", range(1, 8))
def test_every_remainder_of_the_last_block(rest):
    """the short block's stage is filled again a few steps later"""
    R.check(c := R.case(rest, 1, 3000 + rest, 5120, BF, gate=rest % 2 == 0), R.train(c))


@pytest.mark.parametrize("T", [1, 2, 3, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 200])
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_lengths_of_rows_that_are_read_as_tiles(T, gate, dtype):
    R.check(c := R.case(T, 2, T, 72, dtype, gate), R.train(c))


def test_the_same_bits_every_time():
    c = R.case(3, 1, 3005, 5120, BF)
    first = R.train(c)
    for _ in range(3):
        for n, t in R.train(c).items():
            assert torch.equal(t, first[n]), n
