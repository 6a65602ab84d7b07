"""The matrix products at sizes that reach every way a product is cut -- tiles of 256 x 256 and 256 x 128 of two CTAs, 128 x 128 and 128 x 64 of one, whole or
with the tiles behind the last full wave cut along the contraction, rows of whole 16-byte pieces or not -- forward and in both gradients, for one matrix and
for a pair; few rows of wide matrices; rows behind 2^31 elements of what the backward pass reads and writes.  (Which sizes reach which way is as on 148 SMs.)"""
import pytest
import torch

import linear_testlib as L

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("rows,K,N", [
    (33, 64, 64), (33, 129, 129), (33, 2056, 2056), (33, 2057, 2057), (4099, 257, 257), (2050, 129, 2056), (2050, 2056, 129), (515, 520, 4104), (515, 4105, 520),
    (3000, 4104, 129), (3000, 129, 4105), (200, 3080, 3080), (2600, 2057, 520), (1500, 4104, 1033), (1500, 3081, 3080), (1500, 3080, 3081), (1500, 64, 64)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_every_cut_of_a_product(rows, K, N, dtype):
    c = L.linear_case(rows + N, rows, K, N, dtype, bias=True, mul=True, residual=True)
    L.check_linear(c, "gelu", L.train_linear(c, "gelu"))


@pytest.mark.parametrize("rows,K,N", [
    (33, 64, 64), (33, 129, 129), (129, 129, 3080), (129, 136, 3081), (2050, 2056, 64), (4099, 2057, 64), (515, 4104, 257), (700, 521, 2056), (1500, 129, 4105),
    (4099, 257, 1032), (4099, 2056, 129), (1029, 4104, 1032), (1029, 3081, 2056), (33, 4104, 1033), (129, 3080, 2057), (1029, 3080, 2057), (1500, 64, 64),
    (1500, 129, 64), (129, 3081, 3080)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_every_cut_of_a_pair(rows, K, N, dtype):
    c = L.gated_case(rows + N, rows, K, N, dtype)
    L.check_gated(c, "silu", L.train_gated(c, "silu"))


# (more CTAs than four an SM: 4 warps each, and 8 warps at the last N of each list)
@pytest.mark.parametrize("rows", [1, 8, 9, 16, 17, 32])
@pytest.mark.parametrize("K,N", [(520, 9504), (521, 9501), (1030, 9473), (520, 9472)])
def test_few_rows_of_a_wide_matrix(rows, K, N):
    for bias in (True, False):
        c = L.linear_case(rows, rows, K, N, BF, bias=bias, mul=bias, residual=bias)
        L.check_linear(c, "silu", L.train_linear(c, "silu"))


@pytest.mark.parametrize("rows", [1, 8, 9, 16, 17, 32])
@pytest.mark.parametrize("K,N", [(520, 4808), (521, 4801), (1030, 4737), (520, 4736)])
def test_few_rows_of_a_wide_pair(rows, K, N):
    c = L.gated_case(rows, rows, K, N, HF)
    L.check_gated(c, "gelu", L.train_gated(c, "gelu"))


@pytest.mark.parametrize("rows", [16, 17, 20, 31, 32, 33])
@pytest.mark.parametrize("K,N", [(4104, 4200), (1025, 17001)])
def test_few_rows_of_more_than_two_to_the_24_elements(rows, K, N):
    c = L.linear_case(rows, rows, K, N, BF, bias=True)
    L.check_linear(c, "relu2", L.train_linear(c, "relu2"))
    c = L.gated_case(rows, rows, K, N // 2, BF)
    L.check_gated(c, "silu", L.train_gated(c, "silu"))


def far(rows, K, N):
    """x and a gradient of y that is zero except in 300 rows at the end and 100 near the 2^31st element: what is added up over rows then has 400 terms"""
    g = torch.Generator(device="cuda").manual_seed(rows + K + N)
    n = lambda *s, std=1.0: (torch.randn(s, generator=g, device="cuda", dtype=BF) * std)
    x, gy = n(rows, K), torch.zeros((rows, N), device="cuda", dtype=BF)
    at = torch.cat([torch.arange(2 ** 31 // max(K, N) - 50, 2 ** 31 // max(K, N) + 50), torch.arange(rows - 300, rows)]).cuda()
    gy[at] = n(400, N)
    return x, [n(N, K, std=K ** -0.5) for _ in range(2)], gy, at


@pytest.mark.parametrize("K,N", [(64, 8200), (8201, 64), (64, 8201)])
def test_rows_behind_two_to_the_31_elements(K, N):
    import rwkv_infctx_trainer_b200 as W
    rows = 265000
    x, (w, _), gy, at = far(rows, K, N)
    bias = torch.randn(N, device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, w, bias)]
    y = W.linear_act(*leaves, "silu")
    gx, gw, gb = torch.autograd.grad(y, leaves, gy)
    want = L.linear_ref(x[at], w, bias, "silu", None, None, gy[at])
    for n, t in (("y", y.detach()[at]), ("gx", gx[at]), ("gweight", gw), ("gbias", gb)):
        L.close(n, t, *want[n])
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert float(gx[rest].abs().max()) == 0.0


@pytest.mark.parametrize("K,N", [(64, 8200), (8201, 64)])
def test_rows_of_a_pair_behind_two_to_the_31_elements(K, N):
    import rwkv_infctx_trainer_b200 as W
    rows = 265000
    x, ws, gy, at = far(rows, K, N)
    leaves = [t.requires_grad_(True) for t in (x, *ws)]
    y = W.gated_linear(*leaves)
    gx, g0, g1 = torch.autograd.grad(y, leaves, gy)
    want = L.gated_ref(x[at], *ws, "silu", gy[at])
    for n, t in (("y", y.detach()[at]), ("gx", gx[at]), ("gw_gate", g0), ("gw_up", g1)):
        L.close(n, t, *want[n])
