"""The short causal convolution against its formulas in 64 bits: forward, backward, single tokens, segments."""
import pytest
import torch

import ssm_testlib as S

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def case(seed, B, T, D, W, dtype, bias=True, state=True, strided=False, ptype=F32):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)
    x = n(B, T, 2 * D + 8).to(dtype).cuda()[..., 8:8 + D] if strided else n(B, T, D).to(dtype).cuda()
    return {"x": x, "weight": (n(D, W) * 0.6).to(ptype).cuda(), "bias": n(D).to(ptype).cuda() if bias else None,
            "state": n(B, W - 1, D).to(dtype).cuda() if state else None, "gy": n(B, T, D).to(dtype).cuda(),
            "gs": n(B, W - 1, D).to(dtype).cuda()}


NAMES = dict(zip(("x", "weight", "bias", "state"), ("gx", "gw", "gbias", "gstate")))


def train(c, silu=True):
    import rwkv_infctx_trainer_b200 as W
    leaves = {n: c[n].detach().requires_grad_(True) for n in NAMES if c[n] is not None}
    y, s = W.causal_conv(leaves["x"], leaves["weight"], leaves.get("bias"), leaves.get("state"), silu)
    grads = torch.autograd.grad((y, s), list(leaves.values()), (c["gy"], c["gs"]))
    return {"y": y, "state": s, **{NAMES[n]: g for n, g in zip(leaves, grads)}}


def check(c, got, silu=True, grads=True):
    args = (c["x"], c["weight"], c["bias"], c["state"], silu) + ((c["gy"], c["gs"]) if grads else ())
    want, mag = S.conv_ref(*args), S.conv_ref(*args, mag=True)
    B, T, _ = c["x"].shape
    for n, t in got.items():
        if n == "state":
            assert torch.equal(t.double(), want[n])
        else:
            S.close(n, t, want[n], mag[n].abs(), S.conv_K(n, B, T, c["weight"].shape[-1]))


@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 15, 16, 17, 18, 33, 200])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_lengths_and_widths(W, T, dtype):
    c = case(T, 2, T, 40, W, dtype)
    check(c, train(c))


@pytest.mark.parametrize("D", [1, 2, 3, 4, 6, 7, 8, 33, 66, 100, 130, 2050, 2051])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_channels(D, dtype):
    c = case(D, 3, 37, D, 4, dtype)
    check(c, train(c))


@pytest.mark.parametrize("bias,state,silu", [(False, True, True), (True, False, True), (True, True, False), (False, False, False)])
def test_optional_inputs(bias, state, silu):
    c = case(1, 2, 50, 24, 4, BF, bias, state)
    check(c, train(c, silu), silu)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [48, 45])
def test_views_of_wider_tensors(dtype, D):
    c = case(2, 2, 70, D, 4, dtype, strided=True)
    got = train(c)
    check(c, got)
    for n, t in train(dict(c, x=c["x"].contiguous())).items():
        assert torch.equal(t, got[n]), n
    for n, t in train(dict(c, x=c["x"].transpose(0, 1).contiguous().transpose(0, 1))).items():
        assert torch.equal(t, got[n]), n
    for n, t in train(dict(c, x=c["x"].transpose(1, 2).contiguous().transpose(1, 2))).items():
        assert torch.equal(t, got[n]), n


def test_weights_as_a_depthwise_convolution_has_them():
    import rwkv_infctx_trainer_b200 as W
    for ptype in (BF, HF, F32, torch.float64):
        c = case(3, 2, 30, 24, 4, BF, ptype=ptype)
        got = train(dict(c, weight=c["weight"].unsqueeze(1)))
        assert got["gw"].shape == (24, 1, 4) and got["gw"].dtype == ptype and got["gbias"].dtype == ptype
        check(c, {**got, "gw": got["gw"].squeeze(1), **({"gw": got["gw"].squeeze(1).float(), "gbias": got["gbias"].float()} if ptype == torch.float64 else {})})
    c = case(3, 2, 30, 24, 4, BF, ptype=BF)        # weight and bias of two types
    y, _ = W.causal_conv(c["x"], c["weight"], c["bias"].float(), c["state"])
    assert torch.equal(y, W.causal_conv(c["x"], c["weight"], c["bias"], c["state"])[0])


def test_empty_calls():
    import rwkv_infctx_trainer_b200 as W
    c = case(4, 2, 0, 24, 4, BF)
    got = train(c)
    assert got["y"].shape == (2, 0, 24) and torch.equal(got["state"], c["state"]) and torch.equal(got["gstate"], c["gs"])
    assert float(got["gw"].abs().max()) == 0.0 and float(got["gbias"].abs().max()) == 0.0
    assert float(W.causal_conv(c["x"], c["weight"])[1].abs().max()) == 0.0
    for B, D in ((0, 24), (2, 0)):
        got = train(case(4, B, 5, D, 4, BF))
        assert got["y"].shape == (B, 5, D) and got["state"].shape == (B, 3, D) and float(got["gw"].abs().sum()) == 0.0


@pytest.mark.parametrize("cuts", [[0, 20, 21, 23, 60], [0, 1, 2, 3, 60]])
def test_segments_are_the_unsplit_row(cuts):
    import rwkv_infctx_trainer_b200 as W
    c = case(5, 2, 60, 24, 4, F32)
    leaves = {n: c[n].detach().requires_grad_(True) for n in NAMES}
    s, ys = leaves["state"], []
    for a, b in zip(cuts, cuts[1:]):
        y, s = W.causal_conv(leaves["x"][:, a:b], leaves["weight"], leaves["bias"], s)
        ys.append(y)
    y = torch.cat(ys, 1)
    grads = torch.autograd.grad((y, s), list(leaves.values()), (c["gy"], c["gs"]))
    check(c, {"y": y, "state": s, **{NAMES[n]: g for n, g in zip(leaves, grads)}})


@pytest.mark.parametrize("W_", [2, 3, 4])
@pytest.mark.parametrize("D", [40, 41])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_single_tokens_continue_a_prompt(W_, D, dtype):
    import rwkv_infctx_trainer_b200 as W
    c = case(6, 3, 30, D, W_, dtype)
    y, s = W.causal_conv(c["x"][:, :25], c["weight"], c["bias"], c["state"])
    ys = [y]
    for t in range(25, 30):
        v, at = s._version, s.data_ptr()
        ys.append(W.causal_conv_step(c["x"][:, t], s, c["weight"], c["bias"]).unsqueeze(1))
        assert s._version > v and s.data_ptr() == at
    check(c, {"y": torch.cat(ys, 1), "state": s}, grads=False)


def test_gradients_against_differences():
    c = case(7, 2, 19, 10, 4, F32)
    got = train(c)
    mag = S.conv_ref(c["x"], c["weight"], c["bias"], c["state"], True, c["gy"], c["gs"], mag=True)
    for n, gname in NAMES.items():
        v = torch.randn_like(c[n]).double()

        def loss(e):
            d = dict(c, **{n: c[n].double() + e * v})
            o = S.conv_ref(d["x"], d["weight"], d["bias"], d["state"], True)
            return float((o["y"] * c["gy"].double()).sum() + (o["state"] * c["gs"].double()).sum())

        want = (loss(1e-4) - loss(-1e-4)) / 2e-4
        # (1e-6: the differences' own error, 1e-8 of the third derivative)
        assert abs(float((got[gname].double() * v).sum()) - want) <= (S.conv_K(gname, 2, 19, 4) * S.U + 1e-6) * float((mag[gname] * v.abs()).sum()), n


def test_missing_gradients_and_one_alone():
    import rwkv_infctx_trainer_b200 as W
    c = case(8, 2, 90, 24, 4, BF)
    for use in ("gy", "gs"):
        leaves = {n: c[n].detach().requires_grad_(True) for n in NAMES}
        y, s = W.causal_conv(leaves["x"], leaves["weight"], leaves["bias"], leaves["state"])
        got = torch.autograd.grad(y if use == "gy" else s, list(leaves.values()), c[use])
        other = "gs" if use == "gy" else "gy"
        want = train(dict(c, **{other: torch.zeros_like(c[other])}))
        for n, g in zip(NAMES.values(), got):
            assert torch.equal(g, want[n]), (use, n)
    want = train(c)
    for n in NAMES:
        leaf = c[n].detach().requires_grad_(True)
        d = dict(c, **{n: leaf})
        y, s = W.causal_conv(d["x"], d["weight"], d["bias"], d["state"])
        assert torch.equal(torch.autograd.grad((y, s), leaf, (c["gy"], c["gs"]))[0], want[NAMES[n]]), n


def test_nan_reaches_its_own_window_only():
    import rwkv_infctx_trainer_b200 as W
    c = case(9, 2, 40, 24, 4, F32)
    want = W.causal_conv(c["x"], c["weight"], c["bias"], c["state"])[0]
    for bad in (float("nan"), float("inf")):
        x = c["x"].clone()
        x[1, 7, 3] = bad
        y = W.causal_conv(x, c["weight"], c["bias"], c["state"])[0]
        keep = torch.ones_like(y, dtype=torch.bool)
        keep[1, 7:11, 3] = False
        assert torch.equal(y[keep], want[keep])


# rows and widths for which a thread's strip has more than its 16 tokens at least (about 30, and an odd number of groups in it)
@pytest.mark.parametrize("W,D,dtype", [(4, 2048, BF), (4, 2050, BF), (4, 2051, BF), (4, 2051, F32), (3, 2048, HF), (3, 2051, HF), (2, 2048, BF),
                                       (2, 2050, F32), (2, 2051, BF)])
def test_strips_of_many_tokens(W, D, dtype):
    c = case(D + W, 3, 3001, D, W, dtype)
    check(c, train(c))
