"""The root-mean-square norm against its formula in 64 bits: residual, gradient, outputs in 8 bits."""
import pytest
import torch

import ssm_testlib as S

pytestmark = pytest.mark.gpu
BF, HF, F32, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
TYPES = [(BF, BF), (BF, F32), (BF, None), (HF, HF), (HF, F32), (F32, F32), (F32, None)]
EPS = 1e-6


def case(seed, shape, dtype, rtype, wtype=F32):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)
    c = {"x": n(*shape).to(dtype).cuda(), "weight": (1 + 0.2 * n(shape[-1])).to(wtype).cuda(), "residual": None, "gh": None,
         "gy": n(*shape).to(dtype).cuda()}
    if rtype is not None:
        c["residual"], c["gh"] = (2 * n(*shape)).to(rtype).cuda(), n(*shape).to(rtype).cuda()
    return c


# a sum of C squares over the CTA's threads: C / threads + 16 roundings at most, below C; the root, the quotient and the products 16
def K(name, rows, C):
    k = C + 32
    if name.startswith("g"):
        k = 2 * C + 64
    return k + (rows if name == "gw" else 0)


def train(c):
    import rwkv_infctx_trainer_b200 as W
    leaves = {n: c[n].detach().requires_grad_(True) for n in ("x", "weight", "residual") if c[n] is not None}
    out = W.rms_norm(leaves["x"], leaves["weight"], leaves.get("residual"), EPS)
    out, seeds = (out, (c["gy"], c["gh"])) if isinstance(out, tuple) else ((out,), (c["gy"],))
    grads = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), seeds)))
    got = {"y": out[0], "gx": grads["x"], "gw": grads["weight"]}
    if len(out) == 2:
        got.update(h=out[1], gres=grads["residual"])
    return got


def check(c, got):
    C = c["x"].shape[-1]
    rows = c["x"].numel() // C
    ref = S.norm_ref(c["x"], c["weight"], c["residual"], EPS, c["gy"], c["gh"])
    for n, t in got.items():
        r = "gx" if n == "gres" else n
        S.close(n, t, ref[r], ref[r + "_mag"], K(r, rows, C))


@pytest.mark.parametrize("C", [1, 2, 7, 8, 31, 64, 66, 255, 256, 258, 520, 1000, 2049, 2050, 4096, 5120, 8199, 8200, 8202, 16381, 16382, 16384])
@pytest.mark.parametrize("types", TYPES)
def test_widths(C, types):
    c = case(C, (5, C), *types)
    check(c, train(c))


@pytest.mark.parametrize("shape", [(1, 96), (1, 1, 96), (3, 7, 96), (4001, 64), (2, 3, 5, 8)])
def test_shapes(shape):
    c = case(1, shape, BF, BF)
    got = train(c)
    check(c, got)
    assert got["y"].shape == shape and got["h"].shape == shape


@pytest.mark.parametrize("wtype", [BF, HF, F32, torch.float64])
def test_types_of_the_weight(wtype):
    c = case(2, (30, 160), BF, BF, wtype)
    got = train(c)
    assert got["gw"].dtype == wtype
    check(c, {**got, "gw": got["gw"].float() if wtype == torch.float64 else got["gw"]})


def test_rows_that_are_not_adjacent_and_start_anywhere():
    import rwkv_infctx_trainer_b200 as W
    for rtype in (BF, F32):
        c = case(3, (6, 200), BF, rtype)
        want = train(c)
        for x in (torch.cat((c["x"], c["x"]), 1)[:, :200], c["x"].t().contiguous().t()):
            for n, t in train(dict(c, x=x)).items():
                assert torch.equal(t, want[n]), n
        # (another order of a row's sum)
        for start in (1, 2, 3):
            buf = torch.empty(6 * 200 + 8, dtype=BF, device="cuda")[start:start + 1200].view(6, 200)
            check(dict(c, x=buf.copy_(c["x"])), train(dict(c, x=buf)))


def test_empty_and_zero_rows():
    import rwkv_infctx_trainer_b200 as W
    got = train(case(4, (0, 96), BF, BF))
    assert got["y"].shape == (0, 96) and float(got["gw"].abs().max()) == 0.0
    q, s = W.rms_norm_q8(torch.empty((0, 96), device="cuda"), torch.ones(96, device="cuda"), group=64)
    assert q.shape == (0, 96) and s.shape == (0, 2)
    x = torch.zeros((3, 96), device="cuda")
    assert float(W.rms_norm(x, torch.ones(96, device="cuda")).abs().max()) == 0.0
    q, s = W.rms_norm_q8(x, torch.ones(96, device="cuda"))
    assert float(q.float().abs().max()) == 0.0 and torch.equal(s, torch.ones_like(s))


def test_gradients_against_differences():
    c = case(5, (4, 50), F32, F32)
    got = train(c)
    ref = S.norm_ref(c["x"], c["weight"], c["residual"], EPS, c["gy"], c["gh"])
    for n, g in (("x", "gx"), ("weight", "gw"), ("residual", "gres")):
        v = torch.randn_like(c[n]).double()

        def loss(e):
            d = dict(c, **{n: c[n].double() + e * v})
            o = S.norm_ref(d["x"], d["weight"], d["residual"], EPS)
            return float((o["y"] * c["gy"].double()).sum() + (o["h"] * c["gh"].double()).sum())

        want = (loss(1e-4) - loss(-1e-4)) / 2e-4
        m = float((ref["gx_mag" if g != "gw" else "gw_mag"] * v.abs()).sum())
        # (h was rounded to fp32: another 4 2^-24; the differences' own error 1e-6)
        assert abs(float((got[g].double() * v).sum()) - want) <= ((K("g", 4, 50) + 8) * S.U + 1e-6) * m, n


def test_missing_gradients_and_one_alone():
    import rwkv_infctx_trainer_b200 as W
    for types in ((BF, BF), (BF, F32)):
        c = case(6, (40, 264), *types)
        names = ("x", "weight", "residual")
        for use in ("gy", "gh"):
            leaves = [c[n].detach().requires_grad_(True) for n in names]
            y, h = W.rms_norm(*leaves)
            got = torch.autograd.grad(y if use == "gy" else h, leaves, c[use], allow_unused=True)
            other = "gh" if use == "gy" else "gy"
            want = train(dict(c, **{other: torch.zeros_like(c[other])}))
            for n, g in zip(("gx", "gw", "gres"), got):
                assert torch.equal(g, want[n]), (use, n)
        want = train(c)
        for n, g in zip(names, ("gx", "gw", "gres")):
            leaf = c[n].detach().requires_grad_(True)
            d = dict(c, **{n: leaf})
            out = W.rms_norm(d["x"], d["weight"], d["residual"])
            assert torch.equal(torch.autograd.grad(out, leaf, (c["gy"], c["gh"]))[0], want[g]), n


def test_residual_stream_changed_in_place_is_noticed():
    import rwkv_infctx_trainer_b200 as W
    c = case(7, (4, 64), BF, F32)
    x = c["x"].requires_grad_(True)
    y, h = W.rms_norm(x, c["weight"], c["residual"])
    h.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        (y.float().sum() + h.float().sum()).backward()
    # (a 16-bit h is not what the backward pass starts from)
    c = case(7, (4, 64), BF, BF)
    want = train(c)
    x = c["x"].requires_grad_(True)
    y, h = W.rms_norm(x, c["weight"], c["residual"], EPS)
    h = h.add_(1)
    assert torch.equal(torch.autograd.grad((y, h), x, (c["gy"], c["gh"]))[0], want["gx"])


def test_the_residual_stream_is_not_kept_alive_by_its_own_history():
    import gc
    import weakref

    import rwkv_infctx_trainer_b200 as W
    c = case(8, (4, 64), BF, BF)
    x = c["x"].requires_grad_(True)
    y, h = W.rms_norm(x, c["weight"], c["residual"])
    before = torch.cuda.memory_allocated()
    del y, h
    gc.collect()
    assert torch.cuda.memory_allocated() < before


def grouped(t, group):
    C = t.shape[-1]
    n = -(-C // group)
    return torch.nn.functional.pad(t, (0, n * group - C)).unflatten(-1, (n, group))


@pytest.mark.parametrize("C,group", [(64, None), (1000, None), (1001, None), (5120, None), (16384, None), (96, 32), (512, 128), (1000, 64),
                                     (1001, 128), (8200, 256), (40, 256), (9000, 128),
                                     *((C, g) for C in (1002, 333, 9001) for g in (None, 32, 64, 128, 256)), (2, 32), (1, 256)])
@pytest.mark.parametrize("types", TYPES)
def test_8_bit_output(C, group, types):
    """scale: max|y| / 448 with the norm's fp32 error and two roundings more.  q: half a step of e4m3 (2^-4 of a normal
    value, 2^-10 for values below 2^-6) around y / scale, which the fp32 errors of y and of the scale move before"""
    import rwkv_infctx_trainer_b200 as W
    c = case(C, (6, C), *types)
    out = W.rms_norm_q8(c["x"], c["weight"], c["residual"], EPS, group)
    q, s = out[:2]
    assert q.dtype == F8 and q.shape == c["x"].shape and s.dtype == F32
    ref = S.norm_ref(c["x"], c["weight"], c["residual"], EPS)
    if c["residual"] is not None:
        S.close("h", out[2], ref["h"], ref["h_mag"], 1)
        # the same stream as rms_norm's
        assert torch.equal(out[2], W.rms_norm(c["x"], c["weight"], c["residual"], EPS)[1])
    y = grouped(ref["y"], group or C)
    top = y.abs().amax(-1)
    assert s.shape == top.shape
    k = (K("y", 6, C) + 4 + (0 if c["residual"] is None else 8)) * S.U
    # (h = x + residual: its own cancellation, relative to the larger of the row)
    amp = (grouped(ref["h_mag"], group or C) / grouped(ref["h"].abs(), group or C).clamp_min(1e-30)).clamp(1, 1e6)
    assert ((s.double() - top / 448).abs() <= k * top / 448 * 4).all()
    exact = y / (top / 448).unsqueeze(-1)
    got = grouped(q.double(), group or C)
    err = exact.abs() * (2 * k * amp)
    bound = torch.maximum((exact.abs() + err) * 2.0 ** -4, torch.full_like(exact, 2.0 ** -10)) + err
    assert ((got - exact).abs() <= bound).all()
    assert float(got.abs().amax(-1).min()) == 448.0 or bool((top == 0).any())


def test_8_bit_rows_with_nan_and_infinity():
    """a NaN anywhere in what a scale covers makes the scale and all its values NaN, the other groups keep theirs; an
    infinity has a root-mean-square of infinity: zeros beside it and a NaN in its place, as the formula gives"""
    import rwkv_infctx_trainer_b200 as W
    w = torch.ones(256, device="cuda")
    x = torch.randn((4, 256), device="cuda")
    q0, s0 = W.rms_norm_q8(x, w)
    for bad in (float("nan"), float("inf")):
        z = x.clone()
        z[1, 7] = bad
        q, s = W.rms_norm_q8(z, w)
        assert torch.isnan(s[1]).all() and torch.isnan(q[1].float()).all()
        for r in (0, 2, 3):
            assert torch.equal(q[r].float(), q0[r].float()) and torch.equal(s[r], s0[r])
    z = x.clone()
    z[1, 7] = float("inf")
    q, s = W.rms_norm_q8(z, w, group=64)
    assert torch.isnan(s[1, 0]) and torch.equal(s[1, 1:], torch.ones_like(s[1, 1:])) and float(q[1, 64:].float().abs().max()) == 0.0


# rows beyond what a CTA has on its way: CTAs of all SMs (1024 threads an SM) take nine rows and more each; ways that rows lie, one run and
# two runs a thread
@pytest.mark.parametrize("C", [2048, 2049, 2050, 8192, 12288, 12289, 12290])
@pytest.mark.parametrize("types", [(BF, BF), (BF, F32), (HF, None), (F32, F32)])
def test_rows_that_go_round_a_cta(C, types):
    runs = (C + 7) // 8
    threads = (runs if C <= 8192 else (runs + 1) // 2) + 31 & ~31
    rows = torch.cuda.get_device_properties(0).multi_processor_count * max(1, 1024 // threads) * 9 + 5
    c = case(C, (rows, C), *types)
    got = train(c)
    ref = S.norm_ref(c["x"], c["weight"], c["residual"], EPS, c["gy"], c["gh"])
    for n, t in got.items():
        r = "gx" if n == "gres" else n
        S.close(n, t, ref[r], ref[r + "_mag"], K(r, rows, C))
    # a row's values do not depend on the rows around it: the last ones, alone
    some = {n: (t[-20:] if t is not None and t.dim() > 1 else t) for n, t in c.items()}
    for n, t in train(some).items():
        if n != "gw":
            assert torch.equal(t, got[n][-20:]), n
    # nor does the weight's gradient lose or repeat a row: with gy that is nonzero in one row of each 97 alone, the other rows' share is 0
    thin = dict(c, gy=torch.zeros_like(c["gy"]))
    thin["gy"][::97] = c["gy"][::97]
    few = {n: (t[::97] if t is not None and t.dim() > 1 else t) for n, t in c.items()}
    a, b = train(thin)["gw"].double(), S.norm_ref(few["x"], few["weight"], few["residual"], EPS, few["gy"], few["gh"])
    n = few["x"].shape[0]
    assert ((a - b["gw"]).abs() <= K("gw", n, C) * S.U * b["gw_mag"]).all()


def test_histories_of_the_residual_stream_are_freed():
    """an fp32 residual, of which the node keeps its own output h: without the garbage collector nothing is left of a call whose
    results are dropped, with and without a backward pass"""
    import gc

    import rwkv_infctx_trainer_b200 as W
    for types in ((BF, F32), (F32, F32), (BF, BF)):
        c = case(8, (64, 4096), *types)
        x = c["x"].requires_grad_(True)

        def once(backward):
            y, h = W.rms_norm(x, c["weight"], c["residual"])
            if backward:
                torch.autograd.grad((y, h), x, (c["gy"], c["gh"]))

        gc.collect()
        gc.disable()
        try:
            before = torch.cuda.memory_allocated()
            for backward in (False, True, False, True):
                for _ in range(5):
                    once(backward)
                assert torch.cuda.memory_allocated() == before
        finally:
            gc.enable()
