"""The selective scan against its formulas in 64 bits: forward, backward, single tokens, segments."""
import pytest
import torch

import ssm_testlib as S

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def call(c, softplus=True, **kw):
    import rwkv_infctx_trainer_b200 as W
    a = {n: c[n] for n in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state")}
    a.update(kw)
    return W.selective_scan(a["u"], a["delta"], a["A"], a["B"], a["C"], a["D"], a["z"], a["delta_bias"], softplus, a["state"])


def reference(c, softplus, grads, mag):
    return S.scan_ref(c["u"], c["delta"], c["A"], c["B"], c["C"], c["D"], c["z"], c["delta_bias"], softplus, c["state"],
                      c["gy"] if grads else None, c["gs"] if grads else None, mag)


def check(c, got, softplus=True, grads=True):
    want, mag = reference(c, softplus, grads, False), reference(c, softplus, grads, True)
    B, T, D = c["u"].shape
    N = c["A"].shape[1]
    for n, t in got.items():
        S.close(n, t, want[n], mag[n], S.scan_K(n, B, T, D, N))


def train(c, softplus=True):
    leaves = {n: c[n].detach().requires_grad_(True) for n in S.SCAN_LEAVES if c[n] is not None}
    y, s = call(c, softplus, **leaves)
    grads = torch.autograd.grad((y, s), list(leaves.values()), (c["gy"], c["gs"]))
    names = dict(zip(S.SCAN_LEAVES, S.SCAN_GRADS))
    return {"y": y, "state": s, **{names[n]: g for n, g in zip(leaves, grads)}}


# lengths around a block of 16 tokens and its half, and where a row is cut into spans (128 and up)
@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 15, 16, 17, 31, 33, 130, 300])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_lengths(T, dtype):
    c = S.scan_case(T, 2, T, 37, 16, 1, dtype)
    check(c, train(c))


# states that fill no lane, one lane to sixteen a channel; channels that fill no warp, in one group and in several
@pytest.mark.parametrize("N", [1, 3, 4, 5, 8, 11, 16, 20, 32, 33, 64])
@pytest.mark.parametrize("D,G", [(1, 1), (40, 1), (69, 3), (130, 2)])
def test_states_and_channels(N, D, G):
    c = S.scan_case(N * 100 + D, 2, 21, D, N, G, F32)
    check(c, train(c))


@pytest.mark.parametrize("gate,skip,bias,state,softplus", [(False, True, True, True, True), (True, False, True, True, True),
                                                           (True, True, False, True, True), (True, True, True, False, True),
                                                           (False, False, False, False, True), (True, True, True, True, False)])
@pytest.mark.parametrize("T", [1, 40, 200])
def test_optional_inputs(gate, skip, bias, state, softplus, T):
    c = S.scan_case(T, 3, T, 24, 16, 1, BF, gate, skip, bias, state)
    if not softplus:
        c["delta"] = c["delta"].abs() * 0.2
        if bias:
            c["delta_bias"] = c["delta_bias"].abs() * 0.01
    check(c, train(c, softplus), softplus)


@pytest.mark.parametrize("T", [5, 150])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_views_of_wider_tensors(T, dtype):
    c = S.scan_case(T, 2, T, 48, 16, 2, dtype, strided=True)
    assert not c["u"].is_contiguous() and not c["B"].is_contiguous()
    got = train(c)
    check(c, got)
    # the bits of contiguous copies (odd starts included), channels that are not adjacent are copied
    d = {n: (t.contiguous() if t is not None else None) for n, t in c.items()}
    for n, t in train(d).items():
        assert torch.equal(t, got[n]), n
    turned = dict(d, u=d["u"].transpose(1, 2).contiguous().transpose(1, 2))
    for n, t in train(turned).items():
        assert torch.equal(t, got[n]), n


@pytest.mark.parametrize("offset", [1, 3])
def test_tensors_that_start_anywhere(offset):
    c = S.scan_case(3, 2, 20, 40, 16, 1, BF)
    want = train(c)

    def moved(t):
        buf = torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)
        v = buf[offset:offset + t.numel()].view(t.shape)
        v.copy_(t)
        return v

    for n, t in train({n: (moved(t) if t is not None else None) for n, t in c.items()}).items():
        assert torch.equal(t, want[n]), n


def test_empty_calls():
    import rwkv_infctx_trainer_b200 as W
    c = S.scan_case(1, 2, 0, 24, 16, 1, BF)
    got = train(c)
    assert got["y"].shape == (2, 0, 24) and torch.equal(got["state"], c["state"]) and torch.equal(got["gstate"], c["gs"])
    for n in ("gA", "gD", "gbias"):
        assert float(got[n].abs().max()) == 0.0
    y, s = call(dict(c, state=None))
    assert float(s.abs().max()) == 0.0
    for B, D in ((0, 24), (2, 0)):
        c = S.scan_case(1, B, 3, D, 16, 1, BF)
        got = train(c)
        assert got["y"].shape == (B, 3, D) and got["state"].shape == (B, D, 16)
        assert float(got["gA"].abs().sum()) == 0.0
        assert W.selective_scan_step(c["u"][:, 0], c["delta"][:, 0], c["A"], c["B"][:, 0], c["C"][:, 0], c["state"]).shape == (B, D)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_segments_are_the_unsplit_row(dtype):
    """three segments with the state and its gradient carried: the gradients of one call"""
    T, cuts = 100, [(0, 33), (33, 34), (34, 100)]
    c = S.scan_case(8, 2, T, 20, 16, 1, dtype)
    leaves = {n: c[n].detach().requires_grad_(True) for n in S.SCAN_LEAVES}
    s, ys = leaves["state"], []
    for a, b in cuts:
        seg = {n: leaves[n][:, a:b] for n in ("u", "delta", "B", "C", "z")}
        y, s = call(c, **{**leaves, **seg, "state": s})
        ys.append(y)
    y = torch.cat(ys, 1)
    grads = torch.autograd.grad((y, s), list(leaves.values()), (c["gy"], c["gs"]))
    names = dict(zip(S.SCAN_LEAVES, S.SCAN_GRADS))
    check(c, {"y": y, "state": s, **{names[n]: g for n, g in zip(leaves, grads)}})


@pytest.mark.parametrize("N,G", [(16, 1), (16, 4), (5, 1), (64, 2), (8, 1)])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_single_tokens_continue_a_prompt(N, G, dtype):
    import rwkv_infctx_trainer_b200 as W
    T, P = 40, 33
    c = S.scan_case(N, 3, T, 36, N, G, dtype)
    cut = lambda a, b: {n: (c[n][:, a:b]) for n in ("u", "delta", "B", "C", "z")}
    y, s = call(dict(c, **cut(0, P)))
    ys, address = [y], s.data_ptr()
    for t in range(P, T):
        v = s._version
        ys.append(W.selective_scan_step(c["u"][:, t], c["delta"][:, t], c["A"], c["B"][:, t], c["C"][:, t], s, c["D"], c["z"][:, t],
                                        c["delta_bias"]).unsqueeze(1))
        assert s._version > v and s.data_ptr() == address
    check(c, {"y": torch.cat(ys, 1), "state": s}, grads=False)
    if G == 1:      # B and C without the dimension of the groups
        s2 = s.clone()
        a = W.selective_scan_step(c["u"][:, 0], c["delta"][:, 0], c["A"], c["B"][:, 0, 0], c["C"][:, 0, 0], s)
        b = W.selective_scan_step(c["u"][:, 0], c["delta"][:, 0], c["A"], c["B"][:, 0], c["C"][:, 0], s2)
        assert torch.equal(a, b) and torch.equal(s, s2)


def test_gradients_against_differences():
    """<grad, v> of the fp32 call against central differences of the formulas in 64 bits.  Step 1e-4: the differences are
    off by about 1e-8 of the third derivative, the gradient by K 2^-24 of its terms' magnitude."""
    c = S.scan_case(5, 2, 19, 10, 6, 2, F32)
    got = train(c)
    mag = reference(c, True, True, True)
    for n, gname in zip(S.SCAN_LEAVES, S.SCAN_GRADS):
        v = torch.randn_like(c[n]).double()

        def loss(e):
            o = reference(dict(c, **{n: c[n].double() + e * v}), True, False, False)
            return float((o["y"] * c["gy"].double()).sum() + (o["state"] * c["gs"].double()).sum())

        want = (loss(1e-4) - loss(-1e-4)) / 2e-4
        m = float((mag[gname] * v.abs()).sum())
        assert abs(float((got[gname].double() * v).sum()) - want) <= (S.scan_K(gname, 2, 19, 10, 6) * S.U + 1e-6) * m, n


def test_incoming_gradients_that_are_missing():
    """y alone, and the state alone, have the gradients that zeros in the other's place give"""
    for T in (5, 160):
        c = S.scan_case(2, 2, T, 24, 16, 1, BF)
        for use in ("gy", "gs"):
            leaves = {n: c[n].detach().requires_grad_(True) for n in S.SCAN_LEAVES}
            y, s = call(c, **leaves)
            out = (y, c["gy"]) if use == "gy" else (s, c["gs"])
            got = torch.autograd.grad(out[0], list(leaves.values()), out[1], allow_unused=True)
            z = dict(c, **{("gs" if use == "gy" else "gy"): torch.zeros_like(c["gs" if use == "gy" else "gy"])})
            want = train(z)
            for n, g in zip(S.SCAN_GRADS, got):
                assert torch.equal(g, want[n]), (use, n)


@pytest.mark.parametrize("n", S.SCAN_LEAVES)
def test_one_gradient_alone(n):
    """what is asked for alone has the bits that it has among all"""
    c = S.scan_case(4, 2, 140, 24, 16, 1, BF)
    want = train(c)[dict(zip(S.SCAN_LEAVES, S.SCAN_GRADS))[n]]
    leaf = c[n].detach().requires_grad_(True)
    y, s = call(c, **{n: leaf})
    assert torch.equal(torch.autograd.grad((y, s), leaf, (c["gy"], c["gs"]))[0], want)


def test_repeatable_and_types_of_parameters():
    c = S.scan_case(6, 3, 170, 72, 16, 1, BF)
    a, b = train(c), train(c)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    half = dict(c, **{n: c[n].to(BF) for n in ("A", "D", "delta_bias", "state")})
    got = train(half)
    for n, g in (("A", "gA"), ("D", "gD"), ("delta_bias", "gbias"), ("state", "gstate")):
        assert got[g].dtype == BF, n
    check(half, got)


def test_strong_and_weak_decays():
    """decays that underflow at once and decays of one, steps of up to 30 and as small as 1e-9"""
    c = S.scan_case(7, 1, 64, 32, 8, 1, F32)
    c["A"][:8] *= 200.0
    c["A"][8:16] = 0.0
    c["delta"][:, ::5] += 30.0
    c["delta"][:, 1::5] -= 20.0
    # (an argument of up to 30 in the exponential of softplus and 30 x 1600 in a decay: errors of 30 2^-24 and, in terms that
    # do not underflow, of the exponent they are left with)
    got = train(c)
    want, mag = reference(c, True, True, False), reference(c, True, True, True)
    for n, t in got.items():
        S.close(n, t, want[n], mag[n], S.scan_K(n, 1, 64, 32, 8) + 128)


def test_nan_and_infinity_stay_with_their_channel():
    c = S.scan_case(9, 2, 40, 24, 16, 1, F32)
    want, _ = call(c)
    for bad in (float("nan"), float("inf")):
        d = dict(c, u=c["u"].clone())
        d["u"][0, 10, 5] = bad
        y, s = call(d)
        keep = torch.ones_like(y, dtype=torch.bool)
        keep[0, 10:, 5] = False
        assert torch.equal(y[keep], want[keep])
        assert not torch.isfinite(y[0, 10:, 5]).any()
        assert not torch.isfinite(s[0, 5]).any() and torch.isfinite(s[1]).all()


def test_every_cut_of_a_row_into_spans():
    """the C ABI with each number of spans: the same results up to the re-association of the fold (a fold multiplies a
    span's contribution by one exp of the sum of dt instead of by each token's), and the fixed bits of one span where the
    library would take one"""
    import ctypes
    from rwkv_infctx_trainer_b200 import _lib as L
    lib = L.load()
    B, T, D, N, G = 2, 167, 40, 16, 2
    c = S.scan_case(10, B, T, D, N, G, BF)
    st = torch.cuda.current_stream().cuda_stream
    for groups in (1, 2, 3, 5, 11, 1000):
        a = L.SelectiveScanArgs(B=B, T=T, D=D, N=N, G=G, dtype=L.WKV_BF16, softplus=1, time_groups=groups)
        for n, f in (("u", "u"), ("delta", "delta"), ("B", "Bm"), ("C", "Cm"), ("z", "z")):
            setattr(a, f, c[n].data_ptr())
            setattr(a, n + "_batch", c[n].stride(0))
            setattr(a, n + "_token", c[n].stride(1))
        out = {"y": torch.empty_like(c["u"]), "state": torch.empty_like(c["state"]), "gu": torch.empty_like(c["u"]),
               "gdelta": torch.empty_like(c["u"]), "gz": torch.empty_like(c["u"]), "gB": torch.empty_like(c["B"]),
               "gC": torch.empty_like(c["B"]), "gA": torch.empty_like(c["A"]), "gD": torch.empty_like(c["D"]),
               "gbias": torch.empty_like(c["D"]), "gstate": torch.empty_like(c["state"])}
        for f, t in (("A", c["A"]), ("Dskip", c["D"]), ("delta_bias", c["delta_bias"]), ("state_in", c["state"]), ("gy", c["gy"]),
                     ("gstate_out", c["gs"]), ("y", out["y"]), ("state_out", out["state"]), ("gstate_in", out["gstate"]),
                     *((n, out[n]) for n in ("gu", "gdelta", "gz", "gB", "gC", "gA", "gD", "gbias"))):
            setattr(a, f, t.data_ptr())
        n = lib.wkv_selective_scan_ckpt_bytes(ctypes.byref(a))
        ck = torch.empty(n, dtype=torch.uint8, device="cuda")
        a.ckpt, a.ckpt_bytes = ck.data_ptr(), n
        for fn in ("forward", "backward"):
            n = getattr(lib, f"wkv_selective_scan_{fn}_workspace")(ctypes.byref(a))
            ws = torch.empty(n, dtype=torch.uint8, device="cuda")
            a.workspace, a.workspace_bytes = ws.data_ptr() if n else None, n
            L.check(getattr(lib, f"wkv_selective_scan_{fn}")(ctypes.byref(a), st), fn)
        torch.cuda.synchronize()
        check(c, out)


@pytest.mark.parametrize("softplus", [True, False])
def test_infinite_steps_gates_and_decays(softplus):
    """a step of -inf (softplus: 0) leaves the state, an infinite A forgets it, z of +inf lets an infinity through, one of -87 and
    below closes; a NaN in each reaches its own channel"""
    c = S.scan_case(11, 1, 20, 16, 16, 1, F32)
    if not softplus:
        c["delta"] = c["delta"].abs() * 0.2
        c["delta_bias"] = c["delta_bias"].abs() * 0.01
    want = reference(c, softplus, False, False)
    c["A"][3] = -float("inf")
    c["z"][0, 5, 4] = float("inf")
    c["z"][0, 6, 4] = -200.0
    if softplus:
        c["delta"][0, 7:, 5] = -float("inf")
    for n, at in (("delta", (0, 9, 6)), ("z", (0, 9, 7)), ("u", (0, 9, 8))):
        c[n][at] = float("nan")
    y, s = call(c, softplus)
    for t in (1, 10, 19):       # nothing of the tokens before: C . (dt u B) + D u
        raw = (c["delta"][0, t, 3] + c["delta_bias"][3]).double()
        dt = torch.nn.functional.softplus(raw) if softplus else raw
        u, z = c["u"][0, t, 3].double(), c["z"][0, t, 3].double()
        one = ((c["C"][0, t, 0].double() * c["B"][0, t, 0].double()).sum() * dt * u + c["D"][3].double() * u) * S.silu(z)
        assert abs(float(y[0, t, 3]) - float(one)) <= 1e-4 * (1 + abs(float(one)))
    assert torch.isinf(y[0, 5, 4]) and abs(float(y[0, 6, 4])) < 1e-30
    assert torch.isfinite(s[0, 3]).all() and torch.isfinite(s[0, 4]).all()
    if softplus:
        six = S.scan_ref(*(c[n][:, :7] if n in ("u", "delta", "B", "C", "z") else c[n] for n in S.SCAN_LEAVES[:-1]), True, c["state"])["state"]
        assert float((s[0, 5].double() - six[0, 5]).abs().max()) <= 1e-5 * float(six[0, 5].abs().max())
    for ch, keeps in ((6, False), (8, False), (7, True)):
        assert torch.isnan(y[0, 9, ch]) and bool(torch.isfinite(s[0, ch]).all()) == keeps
    clean = [i for i in range(16) if i not in (3, 4, 5, 6, 7, 8)]
    assert torch.isfinite(y[..., clean]).all() and float((s[0, clean].double() - want["state"][0, clean]).abs().max()) < 1e-4


@pytest.mark.parametrize("N", [3, 8, 16, 33, 64])
@pytest.mark.parametrize("softplus", [True, False])
def test_single_token_with_decays_of_any_size(N, softplus):
    """an A of -inf, or so large that A log2(e) is: a step of zero keeps the state (its bits), any other forgets it; what the call for
    prompts gives, also for more rows than a grid has blocks across"""
    import rwkv_infctx_trainer_b200 as W
    c = S.scan_case(N, 6, 1, 40, N, 1, F32)
    c["A"][3], c["A"][4], c["A"][5, 0] = -float("inf"), -3e38, -float("inf")
    if softplus:
        c["delta"][:3] = -300.0               # (softplus of it is 0)
        c["delta_bias"] = c["delta_bias"].clamp(max=0.0)
    else:
        c["delta"] = c["delta"].abs() * 0.2 + 0.01
        c["delta_bias"].zero_()
        c["delta"][:3] = 0.0
    want_y, want = call(c, softplus, u=c["u"].clone().requires_grad_(True))         # (with a gradient: the kernel for prompts)
    want_y, want = want_y.detach(), want.detach()
    s = c["state"].clone()
    one = lambda n: c[n][:, 0]
    y = W.selective_scan_step(one("u"), one("delta"), c["A"], one("B"), one("C"), s, c["D"], one("z"), c["delta_bias"], softplus)
    assert torch.equal(s[:3], c["state"][:3]) and torch.equal(want[:3], c["state"][:3])
    for a, b in zip(call(c, softplus), (y.unsqueeze(1), s)):
        assert torch.equal(a, b)
    # (two kernels, the same sums in another order: each term of a state passes 4 roundings, of y N + 8 more)
    assert torch.isfinite(s).all() and torch.isfinite(y).all()
    mag = c["state"].abs() + want.abs()
    assert ((s - want).abs() <= 8 * S.U * mag).all()
    ymag = ((mag * one("C").abs()).sum(-1) + (c["D"] * one("u")).abs()) * S.silu(one("z")).abs()
    assert ((y - want_y[:, 0]).abs() <= (N + 64) * S.U * ymag).all()
    ref = reference(c, softplus, False, False)["state"]
    gone = s[3:, 3:5].double()
    assert ((gone - (ref[3:, 3:5])).abs() <= 32 * S.U * ref[3:, 3:5].abs() + 1e-37).all()


# ------------------------------------------------------------------ decays of any size, and rows cut into spans
def train_by_abi(c, groups, softplus=True):
    """forward and backward of one call of the C ABI with `groups` spans a row"""
    import ctypes
    from rwkv_infctx_trainer_b200 import _lib as L
    lib = L.load()
    (B, T, D), (_, N), G = c["u"].shape, c["A"].shape, c["B"].shape[2]
    code = {BF: L.WKV_BF16, HF: L.WKV_F16, F32: L.WKV_F32}[c["u"].dtype]
    a = L.SelectiveScanArgs(B=B, T=T, D=D, N=N, G=G, dtype=code, softplus=int(softplus), time_groups=groups)
    for n, f in (("u", "u"), ("delta", "delta"), ("B", "Bm"), ("C", "Cm"), ("z", "z")):
        setattr(a, f, c[n].data_ptr())
        setattr(a, n + "_batch", c[n].stride(0))
        setattr(a, n + "_token", c[n].stride(1))
    like = {"y": "u", "state": "state", "gu": "u", "gdelta": "u", "gz": "u", "gB": "B", "gC": "B", "gA": "A", "gD": "D", "gbias": "D",
            "gstate": "state"}
    out = {n: torch.empty_like(c[t], memory_format=torch.contiguous_format) for n, t in like.items()}
    for f, t in (("A", c["A"]), ("Dskip", c["D"]), ("delta_bias", c["delta_bias"]), ("state_in", c["state"]), ("gy", c["gy"]),
                 ("gstate_out", c["gs"]), ("state_out", out["state"]), ("gstate_in", out["gstate"]),
                 *((n, out[n]) for n in ("y", "gu", "gdelta", "gz", "gB", "gC", "gA", "gD", "gbias"))):
        setattr(a, f, t.data_ptr())
    n = lib.wkv_selective_scan_ckpt_bytes(ctypes.byref(a))
    ck = torch.empty(n, dtype=torch.uint8, device="cuda")
    a.ckpt, a.ckpt_bytes = ck.data_ptr(), n
    st = torch.cuda.current_stream().cuda_stream
    for fn in ("forward", "backward"):
        n = getattr(lib, f"wkv_selective_scan_{fn}_workspace")(ctypes.byref(a))
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = ws.data_ptr() if n else None, n
        L.check(getattr(lib, f"wkv_selective_scan_{fn}")(ctypes.byref(a), st), fn)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("groups", [1, 2, 4, 13])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N", [8, 16, 20])
def test_growing_states_across_spans(groups, dtype, N):
    """states that grow (A > 0), over a span by more than fp32 holds: what is zero before it stays zero, and what is small enough
    to stay finite does, in every cut of the row as in the uncut one.  One token grows by e^4 at most, the last ten have inputs and the
    first ten outgoing gradients, so that all that the uncut recurrence forms is finite (e^40 of a first-size number).
    A term's exponent is 40 at most, an error of 2^-24 of it (in base 2: 58) in each of two roundings moves it by 2 58 2^-24."""
    T = 208
    c = S.scan_case(20 + N, 2, T, 24, N, 1, dtype)
    c["A"] = c["A"].abs() * 0.5                # up to 4
    c["A"][0] = 4.0
    c["delta"] = torch.ones_like(c["delta"])
    for n in ("delta_bias", "state", "gs"):
        c[n].zero_()
    c["u"][:, :T - 10] = 0
    c["gy"][:, 10:] = 0
    got = train_by_abi(c, groups, softplus=False)
    want, mag = reference(c, False, True, False), reference(c, False, True, True)
    for n, t in got.items():
        S.close(n, t, want[n], mag[n], S.scan_K(n, 2, T, 24, N) + 4 * 58)
    # by the call itself, which chooses the cut
    for n, t in train(c, softplus=False).items():
        S.close(n, t, want[n], mag[n], S.scan_K(n, 2, T, 24, N) + 4 * 58)


@pytest.mark.parametrize("groups", [1, 2, 4])
def test_small_states_that_grow_by_more_than_the_largest_number(groups):
    """1e-37 times e^150 over the first half of a row, steps of zero behind it.  The exponent is 217 in base 2: two roundings of it and of
    its parts move a term by 4 217 2^-24; in the uncut row each of 104 tokens by 8 2^-24 (scan_K)."""
    T, N = 208, 16
    c = S.scan_case(31, 1, T, 24, N, 1, F32)
    c["A"] = torch.full_like(c["A"], 150.0 / 104)
    c["delta"].fill_(1.0)
    c["delta"][:, T // 2:] = 0
    for n in ("delta_bias", "u", "gy"):
        c[n].zero_()
    c["state"] = c["state"].sign() * 1e-37
    c["gs"] = c["gs"].sign() * 1e-37
    got = train_by_abi(c, groups, softplus=False)
    want, mag = reference(c, False, True, False), reference(c, False, True, True)
    for n in ("y", "state", "gstate", "gu", "gA"):
        K = S.scan_K(n, 1, T, 24, N) + 4 * 217
        zeros = 0
        if n in ("y", "gu"):
            zeros = (N + 1) * torch.finfo(F32).tiny * (1 + (S.silu(c["z"].double()).abs() if n == "y" else 0))
        S.close(n, got[n], want[n], mag[n] + zeros / (K * S.U), K)


# (channels of an odd number in two groups: single accesses; state sizes of each number of lanes, and of no multiple of four)
@pytest.mark.parametrize("N", [3, 8, 11, 20, 32, 33, 64])
@pytest.mark.parametrize("D,G", [(48, 2), (50, 2), (37, 1)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_every_state_size_in_spans(N, D, G, dtype):
    c = S.scan_case(N + D, 2, 167, D, N, G, dtype)
    want, mag = reference(c, True, True, False), reference(c, True, True, True)
    for groups in (1, 2, 5, 1000):
        got = train_by_abi(c, groups)
        for n, t in got.items():
            S.close(f"{n} in {groups}", t, want[n], mag[n], S.scan_K(n, 2, 167, D, N))
