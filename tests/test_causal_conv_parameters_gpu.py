"""The short convolution and its single-token call with parameters of every type, with and without a bias, on rows that lie in whole pieces, in words and
anywhere: a bias that is not there is never read."""
import pytest
import torch

import test_causal_conv_gpu as V

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("D", [24, 26, 45])
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("ptype", [BF, HF, F32])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_parameters(dtype, ptype, bias, W, D):
    c = V.case(W + D, 2, 30, D, W, dtype, bias=bias, ptype=ptype)
    V.check(c, V.train(c))


@pytest.mark.parametrize("D", [24, 26, 45])
@pytest.mark.parametrize("ptype", [BF, HF, F32])
def test_single_tokens_without_a_bias(ptype, D):
    import rwkv_infctx_trainer_b200 as W
    c = V.case(D, 2, 12, D, 4, BF, bias=False, ptype=ptype)
    state = c["state"].clone()
    ys = [W.causal_conv_step(c["x"][:, t], state, c["weight"]).unsqueeze(1) for t in range(12)]
    V.check(c, {"y": torch.cat(ys, 1), "state": state}, grads=False)
