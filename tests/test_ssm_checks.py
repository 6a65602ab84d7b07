"""The norm, the short convolution and the selective scan look at their arguments before they launch anything: shapes and
types before devices, so that this runs without a GPU."""
import ctypes
import os
import re

import pytest
import torch

BF, F32 = torch.bfloat16, torch.float32
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def z(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def scan_args(B=2, T=5, D=12, N=16, G=None):
    bc = (B, T, N) if G is None else (B, T, G, N)
    return {"u": z(B, T, D), "delta": z(B, T, D), "A": z(D, N, dtype=F32), "B": z(*bc), "C": z(*bc), "D": z(D, dtype=F32),
            "z": z(B, T, D), "delta_bias": z(D, dtype=F32), "state": z(B, D, N, dtype=F32)}


def scan(a):
    import rwkv_infctx_trainer_b200 as W
    return W.selective_scan(a["u"], a["delta"], a["A"], a["B"], a["C"], a["D"], a["z"], a["delta_bias"], state=a["state"])


def test_right_calls_get_as_far_as_the_device():
    import rwkv_infctx_trainer_b200 as W
    for a in (scan_args(), scan_args(G=3), scan_args(N=64), scan_args(T=0), dict(scan_args(), D=None, z=None, delta_bias=None, state=None)):
        with pytest.raises(RuntimeError, match="CUDA"):
            scan(a)
    with pytest.raises(RuntimeError, match="CUDA"):
        W.causal_conv(z(2, 5, 12), z(12, 4), z(12), z(2, 3, 12))
    with pytest.raises(RuntimeError, match="CUDA"):
        W.causal_conv_step(z(2, 12), z(2, 3, 12), z(12, 1, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        W.rms_norm(z(2, 12), z(12), z(2, 12, dtype=F32))
    with pytest.raises(RuntimeError, match="CUDA"):
        W.rms_norm_q8(z(2, 12), z(12), group=128)


@pytest.mark.parametrize("change", [
    {"delta": z(2, 5, 11)}, {"delta": z(2, 4, 12)}, {"A": z(12, 65, dtype=F32)}, {"A": z(11, 16, dtype=F32)}, {"A": z(12, 0, dtype=F32)},
    {"A": z(12, dtype=F32)}, {"B": z(2, 5, 15)}, {"C": z(2, 5, 17)}, {"B": z(2, 5, 5, 16), "C": z(2, 5, 5, 16)}, {"B": z(2, 5, 0, 16), "C": z(2, 5, 0, 16)},
    {"C": z(2, 5, 1, 16)}, {"B": z(1, 5, 16)}, {"D": z(11, dtype=F32)}, {"z": z(2, 5, 13)}, {"delta_bias": z(1, dtype=F32)},
    {"state": z(2, 12, 15, dtype=F32)}, {"state": z(1, 12, 16, dtype=F32)}, {"u": z(5, 12)}])
def test_scan_of_other_shapes_is_refused(change):
    with pytest.raises(ValueError):
        scan({**scan_args(), **change})


@pytest.mark.parametrize("change", [{"delta": z(2, 5, 12, dtype=F32)}, {"B": z(2, 5, 16, dtype=F32)}, {"C": z(2, 5, 16, dtype=torch.float16)},
                                    {"z": z(2, 5, 12, dtype=F32)}, {"A": z(12, 16, dtype=torch.int32)}, {"state": z(2, 12, 16, dtype=torch.int32)},
                                    {"u": z(2, 5, 12, dtype=torch.float64)}])
def test_scan_of_other_types_is_refused(change):
    with pytest.raises((TypeError, ValueError)):
        scan({**scan_args(), **change})


def test_steps_refuse_what_they_cannot_do_in_place():
    import rwkv_infctx_trainer_b200 as W
    a = scan_args(T=1)
    one = lambda t: t[:, 0]
    step = lambda **k: W.selective_scan_step(*(({"u": one(a["u"]), "delta": one(a["delta"]), "A": a["A"], "B": one(a["B"]), "C": one(a["C"]),
                                                 "state": a["state"]} | k).values()))
    with pytest.raises(RuntimeError, match="CUDA"):
        step()
    with pytest.raises(TypeError):
        step(state=a["state"].to(BF))
    with pytest.raises(ValueError, match="contiguous"):
        step(state=z(12, 2, 16, dtype=F32).transpose(0, 1))
    with pytest.raises(ValueError):
        step(u=a["u"])
    with pytest.raises(ValueError):
        step(B=z(2, 1, 1, 16))
    with pytest.raises(RuntimeError, match="no gradient"):
        step(A=a["A"].clone().requires_grad_(True))
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        step(A=a["A"].clone().requires_grad_(True))
    conv = lambda x=z(2, 12), s=z(2, 3, 12), w=z(12, 4): W.causal_conv_step(x, s, w)
    with pytest.raises(TypeError):
        conv(s=z(2, 3, 12, dtype=F32))
    with pytest.raises(ValueError, match="contiguous"):
        conv(s=z(3, 2, 12).transpose(0, 1))
    with pytest.raises(ValueError):
        conv(x=z(2, 1, 12))
    with pytest.raises(RuntimeError, match="no gradient"):
        conv(w=z(12, 4).requires_grad_(True))


@pytest.mark.parametrize("x,w,b,s", [((2, 5, 12), (11, 4), None, None), ((2, 5, 12), (12, 5), None, None), ((2, 5, 12), (12, 1), None, None),
                                     ((2, 5, 12), (12, 2, 4), None, None), ((2, 5, 12), (12, 4), (11,), None), ((2, 5, 12), (12, 4), None, (2, 4, 12)),
                                     ((2, 5, 12), (12, 4), None, (1, 3, 12)), ((5, 12), (12, 4), None, None)])
def test_convolutions_of_other_shapes_are_refused(x, w, b, s):
    import rwkv_infctx_trainer_b200 as W
    with pytest.raises(ValueError):
        W.causal_conv(z(*x), z(*w), None if b is None else z(*b), None if s is None else z(*s))


def test_norms_of_other_shapes_and_types_are_refused():
    import rwkv_infctx_trainer_b200 as W
    for args in ((z(2, 12), z(11)), (z(2, 12), z(1, 12)), (z(2, 12), z(12), z(1, 12)), (z(2, 0), z(0)), (z(2, 16385), z(16385)), (z(), z(1))):
        with pytest.raises(ValueError):
            W.rms_norm(*args)
    with pytest.raises(TypeError):
        W.rms_norm(z(2, 12), z(12), z(2, 12, dtype=torch.float16))
    with pytest.raises(TypeError):
        W.rms_norm(z(2, 12), torch.zeros(12, dtype=torch.int32))
    with pytest.raises(ValueError):
        W.rms_norm(z(2, 12, dtype=torch.float64), z(12))
    for group in (0, 8, 16, 96, 512, -1):
        with pytest.raises(ValueError, match="group"):
            W.rms_norm_q8(z(2, 12), z(12), group=group)
    with pytest.raises(RuntimeError, match="no gradient"):
        W.rms_norm_q8(z(2, 12), z(12).requires_grad_(True))


def test_argument_structs_have_the_headers_fields():
    import rwkv_infctx_trainer_b200._lib as L
    text = open(os.path.join(ROOT, "include", "wkv_b200.h")).read()
    sizes = {"int": 4, "float": 4, "long long": 8, "size_t": 8}
    for name, cls in (("wkv_rms_norm_args", L.RmsNormArgs), ("wkv_causal_conv_args", L.CausalConvArgs), ("wkv_selective_scan_args", L.SelectiveScanArgs)):
        body = text[text.index("typedef struct %s {" % name):text.index("} %s_t;" % name)].split("{", 1)[1]
        fields = []
        for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
            m = re.match(r"(?:const\s+)?(void|float|int|size_t|long long)\s+(.*)", " ".join(decl.split()))
            if m:
                for n in m.group(2).split(","):
                    n = n.strip()
                    fields.append((n.lstrip("*"), 8 if n.startswith("*") else sizes[m.group(1)]))
        assert fields == [(f[0], ctypes.sizeof(f[1])) for f in cls._fields_], name


def test_error_codes_without_gpu():
    import rwkv_infctx_trainer_b200._lib as L
    lib = L.load()
    buf = (ctypes.c_char * 4096)()
    at = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16
    ref = ctypes.byref
    for fn in ("rms_norm", "causal_conv", "selective_scan"):
        for d in ("forward", "backward"):
            assert getattr(lib, f"wkv_{fn}_{d}")(None, None) == 1
    a = L.RmsNormArgs(rows=1, C=16385, dtype=1, res_dtype=1, weight=at)
    assert lib.wkv_rms_norm_forward(ref(a), None) == 2
    a.C = 64
    a.dtype = 9
    assert lib.wkv_rms_norm_forward(ref(a), None) == 3
    a.dtype, a.res_dtype = 1, 2
    assert lib.wkv_rms_norm_forward(ref(a), None) == 3
    a.res_dtype, a.weight = 1, None
    assert lib.wkv_rms_norm_forward(ref(a), None) == 1
    a.weight = at
    assert lib.wkv_rms_norm_forward(ref(a), None) == 1          # x
    a.x, a.y, a.residual = at, at, at
    assert lib.wkv_rms_norm_forward(ref(a), None) == 1          # h
    a.h, a.scale, a.group = at, at, 48
    assert lib.wkv_rms_norm_forward(ref(a), None) == 2
    a.gweight = at
    assert lib.wkv_rms_norm_backward(ref(a), None) == 5
    a.rows = 0
    a.group, a.gweight = 0, None
    assert lib.wkv_rms_norm_forward(ref(a), None) == 0 and lib.wkv_rms_norm_backward(ref(a), None) == 0

    a = L.CausalConvArgs(B=1, T=20, D=8, W=5, dtype=1, w_dtype=0)
    assert lib.wkv_causal_conv_forward(ref(a), None) == 2
    a.W = 4
    assert lib.wkv_causal_conv_forward(ref(a), None) == 1
    a.weight, a.x, a.y, a.state_in, a.state_out = at, at, at, at, at
    assert lib.wkv_causal_conv_forward(ref(a), None) == 7       # state in place over more than 16 tokens
    a.gweight = at
    assert lib.wkv_causal_conv_backward(ref(a), None) == 5
    a.x_token = -1
    assert lib.wkv_causal_conv_forward(ref(a), None) == 2
    a.x_token, a.D = 8, (1 << 22) + 1
    assert lib.wkv_causal_conv_forward(ref(a), None) == 2
    a.D, a.B, a.T = 8, 1 << 20, 1 << 20
    assert lib.wkv_causal_conv_forward(ref(a), None) == 2
    a = L.CausalConvArgs(W=4)
    assert lib.wkv_causal_conv_forward(ref(a), None) == 0

    a = L.SelectiveScanArgs(B=1, T=300, D=8, N=16, G=3, dtype=1, softplus=1)
    assert lib.wkv_selective_scan_forward(ref(a), None) == 2
    a.G, a.N = 1, 65
    assert lib.wkv_selective_scan_forward(ref(a), None) == 2
    a.N = 16
    assert lib.wkv_selective_scan_forward(ref(a), None) == 1
    for f in ("u", "delta", "Bm", "Cm", "A", "y", "state_in", "state_out"):
        setattr(a, f, at)
    assert lib.wkv_selective_scan_forward(ref(a), None) == 7    # state in place over more than one token
    a.state_out = at + 256
    a.time_groups = 4
    assert lib.wkv_selective_scan_forward(ref(a), None) == 5    # spans need a workspace
    assert lib.wkv_selective_scan_backward(ref(a), None) == 5   # the checkpoints
    assert lib.wkv_selective_scan_ckpt_bytes(ref(a)) == 19 * 8 * 16 * 4
    a.ckpt, a.ckpt_bytes = at, 16
    assert lib.wkv_selective_scan_forward(ref(a), None) == 5
    a.time_groups = -1
    assert lib.wkv_selective_scan_forward(ref(a), None) == 2
    a.time_groups, a.u_token = 0, 1 << 27                       # offsets inside a block of tokens are 32-bit
    assert lib.wkv_selective_scan_forward(ref(a), None) == 2
    a.u_token, a.T, a.B = 8, 1 << 30, 64
    assert lib.wkv_selective_scan_forward(ref(a), None) == 2
    a = L.SelectiveScanArgs(N=16, G=1)
    assert lib.wkv_selective_scan_forward(ref(a), None) == 0


def test_scans_of_more_tokens_than_can_be_numbered_are_refused():
    """(nothing here reaches a launch: the sizes of the checkpoints, and calls that are refused)"""
    import rwkv_infctx_trainer_b200._lib as L
    lib = L.load()
    buf = (ctypes.c_char * 4096)()
    at = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16
    a = L.SelectiveScanArgs(B=1, D=1, N=4, G=1, dtype=1, softplus=1)
    for f in ("u", "delta", "Bm", "Cm", "A", "y", "state_out"):
        setattr(a, f, at)
    a.T = 2 ** 31 - 17
    blocks = (a.T + 15) // 16               # (of 16 bytes each)
    assert lib.wkv_selective_scan_ckpt_bytes(ctypes.byref(a)) == (blocks * 16 + 255) // 256 * 256
    for T in (2 ** 31 - 16, 2 ** 31 - 1):
        a.T = T
        assert lib.wkv_selective_scan_ckpt_bytes(ctypes.byref(a)) == 0
        assert lib.wkv_selective_scan_forward(ctypes.byref(a), None) == 2
        assert lib.wkv_selective_scan_backward(ctypes.byref(a), None) == 2


def test_convolutions_of_more_tokens_than_can_be_numbered_are_refused():
    """(nothing here reaches a launch)"""
    import rwkv_infctx_trainer_b200._lib as L
    lib = L.load()
    buf = (ctypes.c_char * 4096)()
    at = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16
    a = L.CausalConvArgs(B=1, D=1, W=4, dtype=1, x=at, weight=at, y=at, state_out=at, x_batch=1, x_token=1)
    for T in (2 ** 31 - 1, 2 ** 31 - 272):
        a.T = T
        assert lib.wkv_causal_conv_backward_workspace(ctypes.byref(a)) == 0
        assert lib.wkv_causal_conv_forward(ctypes.byref(a), None) == 2
        assert lib.wkv_causal_conv_backward(ctypes.byref(a), None) == 2
    a.T = 2 ** 31 - 273
    assert lib.wkv_causal_conv_backward_workspace(ctypes.byref(a)) > 0
