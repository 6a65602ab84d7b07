"""Waits of the matrix products that run out in tiles of two CTAs: a block is never loaded by the first of them, so that the second one's copies are ahead
of it; with a limit of one poll others are still on their way.  The call ends, says so, and the next one is right."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


# (on 148 SMs: 256 x 256 whole and cut, 256 x 128 whole and cut, 128 x 128)
@pytest.mark.parametrize("rows,K,N,pair", [(3000, 128, 4104, 0), (1500, 3080, 3080, 0), (2600, 2056, 520, 0), (200, 3080, 3080, 0), (4099, 256, 256, 0),
                                           (1029, 3080, 2056, 1), (4099, 264, 1032, 1)])
@pytest.mark.parametrize("skip", [0, 1, 5])
@pytest.mark.parametrize("limit", [1, 500])
@pytest.mark.parametrize("backward", [0, 1])
def test_a_call_ends_and_the_next_one_is_right(rows, K, N, pair, skip, limit, backward):
    from rwkv_infctx_trainer_b200 import _lib as L
    lib = L.load()
    n = lambda *s: torch.randn(s, device="cuda", dtype=BF)
    t = {"x": n(rows, K), "w0": n(N, K), "y": n(rows, N), "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
    a = L.LinearArgs(rows=rows, K=K, N=N, dtype=1, act=1, pair=pair, x_row=K, w0_row=K, w1_row=K)
    if pair:
        t["w1"] = n(N, K)
    a.saved_bytes = lib.wkv_linear_saved_bytes(ctypes.byref(a))
    t["saved"] = torch.randn(a.saved_bytes // 4, device="cuda")
    outs = ["y"]
    if backward:
        outs = ["gx", "gw0"] + ["gw1"] * pair
        t.update(gy=n(rows, N), gx=n(rows, K), gw0=n(N, K), **({"gw1": n(N, K)} if pair else {}))
    for k, v in t.items():
        setattr(a, k, v.data_ptr())
    size, run = ((lib.wkv_linear_backward_workspace, lib.wkv_linear_backward) if backward else (lib.wkv_linear_forward_workspace, lib.wkv_linear_forward))
    a.workspace_bytes = size(ctypes.byref(a))
    t["workspace"] = torch.empty(max(a.workspace_bytes, 256), dtype=torch.uint8, device="cuda")
    a.workspace = t["workspace"].data_ptr()
    assert run(ctypes.byref(a), L.stream_handle(0)) == 0
    torch.cuda.synchronize()
    assert int(t["status"]) == 0
    want = {k: t[k].clone() for k in outs}
    for _ in range(2):
        # (a block behind the contraction's last is not there to be left out, and of a cut tile every part counts its own)
        assert lib.wkv_linear_selftest_abort(ctypes.byref(a), backward, skip, limit, L.stream_handle(0)) == 0
        torch.cuda.synchronize()
        if skip < 2:
            assert int(t["status"]) == 64
        t["status"].zero_()
        assert run(ctypes.byref(a), L.stream_handle(0)) == 0
        torch.cuda.synchronize()
        assert int(t["status"]) == 0
        for k in outs:
            assert torch.equal(t[k], want[k]), k
