"""The gated recurrence and the matrix products look at their arguments before they launch anything: shapes and types before
devices, so that this runs without a GPU."""
import ctypes
import os
import re

import pytest
import torch

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def z(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def rec_args(B=2, T=5, D=12):
    return {"x": z(B, T, D), "input_gate": z(B, T, D), "decay_gate": z(B, T, D), "decay": z(D, dtype=F32), "z": z(B, T, D),
            "state": z(B, D, dtype=F32)}


def rec(a, **k):
    import rwkv_infctx_trainer_b200 as W
    return W.gated_recurrence(*a.values(), **k)


def test_right_calls_get_as_far_as_the_device():
    import rwkv_infctx_trainer_b200 as W
    for a in (rec_args(), rec_args(T=0), rec_args(D=1), dict(rec_args(), z=None, state=None), dict(rec_args(), decay=z(12)), dict(rec_args(), state=z(2, 12))):
        with pytest.raises(RuntimeError, match="CUDA"):
            rec(a)
    for call in (lambda: W.linear_act(z(2, 12), z(7, 12)), lambda: W.linear_act(z(12), z(7, 12), z(7, dtype=F32), "gelu", z(7), z(7)),
                 lambda: W.linear_act(z(0, 3, 12), z(7, 12)), lambda: W.gated_linear(z(2, 3, 12, dtype=HF), z(7, 12, dtype=HF), z(7, 12, dtype=HF), "sigmoid")):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("change", [
    {"x": z(5, 12)}, {"x": z(2, 5, 1, 12)}, {"input_gate": z(2, 5, 11)}, {"decay_gate": z(2, 4, 12)}, {"decay_gate": z(1, 5, 12)}, {"decay": z(11, dtype=F32)},
    {"decay": z(1, 12, dtype=F32)}, {"z": z(2, 5, 13)}, {"state": z(2, 11, dtype=F32)}, {"state": z(1, 12, dtype=F32)}, {"state": z(2, 12, 1, dtype=F32)}])
def test_recurrences_of_other_shapes_are_refused(change):
    with pytest.raises(ValueError):
        rec({**rec_args(), **change})


@pytest.mark.parametrize("change", [{"input_gate": z(2, 5, 12, dtype=F32)}, {"decay_gate": z(2, 5, 12, dtype=HF)}, {"z": z(2, 5, 12, dtype=F32)},
                                    {"decay": z(12, dtype=torch.int32)}, {"state": z(2, 12, dtype=torch.int32)}, {"x": z(2, 5, 12, dtype=torch.float64)}])
def test_recurrences_of_other_types_are_refused(change):
    with pytest.raises((TypeError, ValueError)):
        rec({**rec_args(), **change})


@pytest.mark.parametrize("c", [0.0, -1.0, float("nan"), float("inf"), 2e6])
def test_constants_out_of_range_are_refused(c):
    import rwkv_infctx_trainer_b200 as W
    with pytest.raises(ValueError, match="c must be"):
        rec(rec_args(), c=c)
    a = rec_args(T=1)
    with pytest.raises(ValueError, match="c must be"), torch.no_grad():
        W.gated_recurrence_step(a["x"][:, 0], a["input_gate"][:, 0], a["decay_gate"][:, 0], a["decay"], a["state"], c=c)


def test_steps_refuse_what_they_cannot_do_in_place():
    import rwkv_infctx_trainer_b200 as W
    base = {"x": z(2, 12), "input_gate": z(2, 12), "decay_gate": z(2, 12), "decay": z(12, dtype=F32), "state": z(2, 12, dtype=F32), "z": None}
    step = lambda **k: W.gated_recurrence_step(*{**base, **k}.values())
    with pytest.raises(RuntimeError, match="CUDA"):
        step()
    for change in ({"state": z(2, 12)}, {"input_gate": z(2, 12, dtype=F32)}):
        with pytest.raises(TypeError):
            step(**change)
    with pytest.raises(ValueError, match="contiguous"):
        step(state=z(12, 2, dtype=F32).t())
    for change in ({"x": z(2, 1, 12)}, {"decay_gate": z(2, 11)}, {"state": z(3, 12, dtype=F32)}, {"z": z(1, 12)}):
        with pytest.raises(ValueError):
            step(**change)
    for n in ("x", "decay", "state"):
        with pytest.raises(RuntimeError, match="no gradient"):
            step(**{n: base[n].clone().requires_grad_(True)})
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        step(decay=base["decay"].clone().requires_grad_(True))


@pytest.mark.parametrize("x,w,b,mul,res", [((2, 12), (7, 11), None, None, None), ((2, 12), (7,), None, None, None), ((2, 12), (1, 7, 12), None, None, None),
                                           ((2, 12), (0, 12), None, None, None), ((2, 0), (7, 0), None, None, None), ((), (7, 1), None, None, None),
                                           ((2, 12), (7, 12), (6,), None, None), ((2, 12), (7, 12), (1, 7), None, None), ((2, 12), (7, 12), None, (2, 12), None),
                                           ((2, 12), (7, 12), None, (7,), None), ((2, 12), (7, 12), None, None, (1, 7)), ((3, 2, 12), (7, 12), None, None, (6, 7))])
def test_products_of_other_shapes_are_refused(x, w, b, mul, res):
    import rwkv_infctx_trainer_b200 as W
    t = lambda s: None if s is None else z(*s)
    with pytest.raises(ValueError):
        W.linear_act(z(*x), z(*w), t(b), mul=t(mul), residual=t(res))


def test_products_of_other_types_and_activations_are_refused():
    import rwkv_infctx_trainer_b200 as W
    for dt in (F32, torch.float64, torch.int32):
        with pytest.raises(TypeError):
            W.linear_act(z(2, 12, dtype=dt), z(7, 12, dtype=dt))
        with pytest.raises(TypeError):
            W.gated_linear(z(2, 12, dtype=dt), z(7, 12, dtype=dt), z(7, 12, dtype=dt))
    for change in ({"weight": z(7, 12, dtype=HF)}, {"mul": z(2, 7, dtype=F32)}, {"residual": z(2, 7, dtype=F32)}, {"bias": z(7, dtype=torch.int32)}):
        with pytest.raises(TypeError):
            W.linear_act(**{"x": z(2, 12), "weight": z(7, 12), **change})
    with pytest.raises(TypeError):
        W.gated_linear(z(2, 12), z(7, 12), z(7, 12, dtype=HF))
    for a, b in (((7, 12), (8, 12)), ((7, 12), (7, 11)), ((7, 11), (7, 12)), ((7,), (7,))):
        with pytest.raises(ValueError):
            W.gated_linear(z(2, 12), z(*a), z(*b))
    for name in ("relu", "SiLU", "", "swish"):
        with pytest.raises(ValueError, match="activation"):
            W.linear_act(z(2, 12), z(7, 12), activation=name)
        with pytest.raises(ValueError, match="activation"):
            W.gated_linear(z(2, 12), z(7, 12), z(7, 12), name)


def test_argument_structs_have_the_headers_fields():
    import rwkv_infctx_trainer_b200._lib as L
    text = open(os.path.join(ROOT, "include", "wkv_b200.h")).read()
    sizes = {"int": 4, "float": 4, "long long": 8, "size_t": 8}
    for name, cls in (("wkv_gated_recurrence_args", L.GatedRecurrenceArgs), ("wkv_linear_args", L.LinearArgs)):
        body = text[text.index("typedef struct %s {" % name):text.index("} %s_t;" % name)].split("{", 1)[1]
        fields = []
        for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
            m = re.match(r"(?:const\s+)?(void|float|int|size_t|long long)\s+(.*)", " ".join(decl.split()))
            if m:
                for n in m.group(2).split(","):
                    n = n.strip()
                    fields.append((n.lstrip("*"), 8 if n.startswith("*") else sizes[m.group(1)]))
        assert fields == [(f[0], ctypes.sizeof(f[1])) for f in cls._fields_], name


@pytest.fixture
def memory():
    buf = (ctypes.c_char * 4096)()
    yield ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16


def test_error_codes_of_the_recurrence(memory):
    """(nothing here reaches a launch)"""
    import rwkv_infctx_trainer_b200._lib as L
    lib, at, ref = L.load(), memory, ctypes.byref
    fwd, bwd = lib.wkv_gated_recurrence_forward, lib.wkv_gated_recurrence_backward
    assert fwd(None, None) == 1 and bwd(None, None) == 1
    a = L.GatedRecurrenceArgs(B=1, T=300, D=8, dtype=9, c=8.0)
    assert fwd(ref(a), None) == 3 and bwd(ref(a), None) == 3
    a.dtype = 1
    assert fwd(ref(a), None) == 1 and bwd(ref(a), None) == 1
    for f in ("decay", "x", "input_gate", "decay_gate", "y", "state_out"):
        setattr(a, f, at)
    assert bwd(ref(a), None) == 5                               # the states that the forward pass leaves
    a.state_in = at
    assert fwd(ref(a), None) == 7                               # state in place over more than one token
    a.state_in = None
    assert lib.wkv_gated_recurrence_ckpt_bytes(ref(a)) == 5 * 8 * 4        # the state before every 64 tokens
    a.ckpt, a.ckpt_bytes = at, 16
    assert fwd(ref(a), None) == 5 and bwd(ref(a), None) == 5
    a.ckpt_bytes, a.gdecay = 4096, at
    assert bwd(ref(a), None) == 5                               # its workspace
    for field, value in (("c", 0.0), ("c", -1.0), ("c", float("nan")), ("D", (1 << 22) + 1), ("T", 2 ** 31 - 4096), ("x_token", -1), ("r_token", (1 << 26) + 1), ("B", -1),
                         ("T", -1)):
        old = getattr(a, field)
        setattr(a, field, value)
        assert fwd(ref(a), None) == 2 and bwd(ref(a), None) == 2, field
        assert lib.wkv_gated_recurrence_ckpt_bytes(ref(a)) == 0
        setattr(a, field, old)
    a.B, a.D = 2 ** 24, 2 ** 12
    assert fwd(ref(a), None) == 2
    a = L.GatedRecurrenceArgs(c=1.0)
    assert fwd(ref(a), None) == 0 and bwd(ref(a), None) == 0    # no channels, nothing to do
    for limit, skip in ((0, 0), (100001, 0), (5, -1)):
        assert lib.wkv_gated_recurrence_selftest_abort(ref(a), 0, skip, limit, None) == 2


def test_error_codes_of_the_products(memory):
    """(nothing here reaches a launch)"""
    import rwkv_infctx_trainer_b200._lib as L
    lib, at, ref = L.load(), memory, ctypes.byref
    fwd, bwd = lib.wkv_linear_forward, lib.wkv_linear_backward
    assert fwd(None, None) == 1 and bwd(None, None) == 1
    a = L.LinearArgs(rows=40, K=24, N=8, dtype=9, x_row=24, w0_row=24, w1_row=24)
    assert fwd(ref(a), None) == 3
    a.dtype = 0
    assert fwd(ref(a), None) == 7 and bwd(ref(a), None) == 7    # fp32
    a.dtype = 1
    assert fwd(ref(a), None) == 1 and bwd(ref(a), None) == 1
    a.x, a.w0, a.y, a.gy = at, at, at, at
    for field, value in (("rows", -1), ("K", 0), ("N", 0), ("rows", 2 ** 31), ("K", 2 ** 31 - 4095), ("N", 2 ** 31), ("x_row", 23), ("w0_row", -24), ("act", 5), ("act", -1), ("pair", 2)):
        old = getattr(a, field)
        setattr(a, field, value)
        assert fwd(ref(a), None) == 2 and bwd(ref(a), None) == 2, field
        assert lib.wkv_linear_forward_workspace(ref(a)) == 0 and lib.wkv_linear_saved_bytes(ref(a)) == 0
        setattr(a, field, old)
    a.bias, a.bias_dtype = at, 7
    assert fwd(ref(a), None) == 3
    a.bias_dtype = 0
    a.pair = 1
    assert fwd(ref(a), None) == 7                               # a pair has no bias
    a.bias = None
    assert fwd(ref(a), None) == 1                               # its second matrix
    a.w1 = at
    assert lib.wkv_linear_saved_bytes(ref(a)) == 2 * 1280       # [40, 8] of 4 bytes, twice
    a.saved, a.saved_bytes = at, 2500
    assert fwd(ref(a), None) == 5 and bwd(ref(a), None) == 5
    a.saved = None
    assert bwd(ref(a), None) == 5
    a.pair, a.act, a.w1 = 0, 1, None
    assert lib.wkv_linear_saved_bytes(ref(a)) == 1280 and bwd(ref(a), None) == 5
    a.act, a.gw1 = 0, at
    assert lib.wkv_linear_saved_bytes(ref(a)) == 0 and bwd(ref(a), None) == 1
    a.gw1, a.x, a.x_row = None, at + 2, 25                      # rows that are copied first need a workspace
    assert lib.wkv_linear_forward_workspace(ref(a)) >= 40 * 24 * 2 and fwd(ref(a), None) == 5
    a.rows = 0
    assert fwd(ref(a), None) == 0 and bwd(ref(a), None) == 0
    for limit, skip in ((0, 0), (100001, 0), (5, -1)):
        assert lib.wkv_linear_selftest_abort(ref(a), 0, skip, limit, None) == 2
