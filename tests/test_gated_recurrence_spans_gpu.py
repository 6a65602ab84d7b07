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


def test_gradients_behind_two_to_the_31_elements():
    """the last tokens' gradients are those of a call of their own, from the state before them; the first tokens', whose addresses are small, come last in time"""
    import rwkv_infctx_trainer_b200 as W
    T, D, tail = 33100, 65536, 70
    g = torch.Generator(device="cuda").manual_seed(1)
    n = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=BF)
    x, gy, decay = n(1, T, D), n(1, T, D), torch.rand(D, generator=g, device="cuda") * 4 - 4
    ig, rg = n(1, T, 1).expand(1, T, D), n(1, T, D)
    with torch.no_grad():
        _, before = W.gated_recurrence(x[:, :T - tail], ig[:, :T - tail], rg[:, :T - tail], decay)
        short = [t[:, T - tail:].float().clone() for t in (x, ig, rg)]

    def gradients(x, ig, rg, gy, state):
        x, rg = x.detach().requires_grad_(True), rg.detach().requires_grad_(True)
        y, s = W.gated_recurrence(x, ig, rg, decay, None, state)
        return torch.autograd.grad(y, (x, rg), gy)
    got = gradients(x, ig, rg, gy, None)
    # (in fp32: a bf16 result is off by half a step, and both by their sums: at most 70 terms, 40 + 3 roundings and a decay's 5 a token, of |gy| <= 6 and
    # states <= 8)
    want = gradients(*short, gy[:, T - tail:].float(), before)
    for a, b in zip(got, want):
        a = a[:, T - tail:].float()
        assert float(((a - b).abs() - 2.0 ** -8 * b.abs()).max()) <= (40 + 8 * 70) * R.U * 70 * 6 * 8
    # the same of the first tokens, with what the later ones send back
    head = 70
    with torch.no_grad():
        first = [t[:, :2000].float().clone() for t in (x, ig, rg, gy)]
    # (where softplus(decay) is above 0.1, 1930 tokens leave e^(-0.8 sum of sigmoid(rg)), some e^-770, of what the ones behind them send back)
    want = gradients(*first, None)
    for a, b in zip(got, want):
        a, b = a[:, :head].float(), b[:, :head]
        keep = torch.nn.functional.softplus(decay) > 0.1
        assert float(((a - b).abs() - 2.0 ** -8 * b.abs())[..., keep].max()) <= (40 + 8 * 70) * R.U * 70 * 6 * 8
