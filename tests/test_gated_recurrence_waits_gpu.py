"""Waits of the gated recurrence that run out on rows of many blocks: the ring's stages would be filled again after it, and must not be.  The stage that is
never loaded counts on bytes that do not come, as a copy that is late would leave it; with a limit of one poll other stages' copies are still on their way."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def args(B, T, D, dtype, backward):
    from rwkv_infctx_trainer_b200 import _lib as L
    lib = L.load()
    n = lambda *s, dt=dtype: torch.randn(s, device="cuda", dtype=dt)
    f32 = torch.float32
    x, ig, rg, z, gy = (n(B, T, D) for _ in range(5))
    t = {"x": x, "input_gate": ig, "decay_gate": rg, "z": z, "decay": n(D, dt=f32), "state_in": n(B, D, dt=f32), "y": torch.empty_like(x),
         "state_out": n(B, D, dt=f32)}
    a = L.GatedRecurrenceArgs(B=B, T=T, D=D, dtype=0 if dtype == f32 else 1, c=8.0)
    for k in "xirz":
        setattr(a, k + "_batch", T * D)
        setattr(a, k + "_token", D)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    a.ckpt_bytes = lib.wkv_gated_recurrence_ckpt_bytes(ctypes.byref(a))
    ckpt = torch.zeros(a.ckpt_bytes, dtype=torch.uint8, device="cuda")
    t.update(ckpt=ckpt, status=status)
    if backward:
        t.update(gy=gy, gx=torch.empty_like(x), ginput_gate=torch.empty_like(x), gdecay_gate=torch.empty_like(x), gz=torch.empty_like(x),
                 gdecay=torch.empty(D, device="cuda"))
    for k, v in t.items():
        setattr(a, k, v.data_ptr())
    size = lib.wkv_gated_recurrence_backward_workspace if backward else lib.wkv_gated_recurrence_forward_workspace
    a.workspace_bytes = size(ctypes.byref(a))
    t["workspace"] = torch.empty(max(a.workspace_bytes, 256), dtype=torch.uint8, device="cuda")
    a.workspace = t["workspace"].data_ptr()
    return a, t


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("skip", [0, 1, 2])
@pytest.mark.parametrize("limit", [1, 500])
@pytest.mark.parametrize("B,T,D,dtype", [(1, 3005, 5120, torch.bfloat16), (8, 700, 2048, torch.bfloat16), (1, 3005, 5120, torch.float32)])
def test_a_call_ends_and_the_next_one_is_right(B, T, D, dtype, limit, skip, backward):
    from rwkv_infctx_trainer_b200 import _lib as L
    lib = L.load()
    a, t = args(B, T, D, dtype, backward)
    run = lib.wkv_gated_recurrence_backward if backward else lib.wkv_gated_recurrence_forward
    outs = [k for k in ("y", "state_out", "gx", "ginput_gate", "gdecay_gate", "gz", "gdecay") if k in t and (backward or not k.startswith("g"))]
    # (backward from states of zero before each block: what it gives is the same every time, which is what is asked)
    assert run(ctypes.byref(a), L.stream_handle(0)) == 0
    torch.cuda.synchronize()
    assert int(t["status"]) == 0
    want = {k: t[k].clone() for k in outs}
    ckpt = t["ckpt"].clone()
    for _ in range(2):
        assert lib.wkv_gated_recurrence_selftest_abort(ctypes.byref(a), backward, skip, limit, L.stream_handle(0)) == 0
        torch.cuda.synchronize()
        assert int(t["status"]) == 128
        t["status"].zero_()
        t["ckpt"].copy_(ckpt)
        assert run(ctypes.byref(a), L.stream_handle(0)) == 0
        torch.cuda.synchronize()
        assert int(t["status"]) == 0
        for k in outs:
            assert torch.equal(t[k], want[k]), k
