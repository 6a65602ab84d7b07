"""The gated linear recurrence against its formulas in 64 bits: forward, backward, single tokens, segments, masks.

The reference carries a bound of the kernel's error beside each value.  In units of 2^-24 (U, half a step of fp32): a sigmoid of x
is off by 2|x| + 8 (the exponent's product 2|x|, ex2 4, the sum and the quotient 4), softplus(p) by 12 + 2.4|p| (a fast exponential
4 + 2.4|p|, the logarithm and the products 8), a decay by |L| times what its exponent is off, and 5 (ex2 4, its mean's constant 1);
1 - a^2 by its argument's error and 8 in the series, by at most 7 decays' and 5 above it; a root by half of that and 4.  Decays below
2^-126 are zero in the kernel: what multiplies a decay is off by 2^-126 of itself on top (FLUSH).  A step adds
3 for its product and sum and what regrouping tokens into segments adds to them, a pass over segments 40 in all.  An output is
rounded once more to its type, by at most half a step."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
FLUSH = 2.0 ** -126
LEAVES = ["x", "input_gate", "decay_gate", "decay", "z", "state"]
GRADS = dict(zip(LEAVES, ["gx", "ginput", "gdecay_gate", "gdecay", "gz", "gstate"]))
INF = float("inf")


def case(seed, B, T, D, dtype, gate=True, state=True, strided=False, ptype=F32, top=None):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, std=1.0: torch.randn(s, generator=g) * std
    wide = lambda: (n(B, T, 2 * D + 8).to(dtype).cuda()[..., 8:8 + D] if strided else n(B, T, D).to(dtype).cuda())
    return {"x": wide(), "input_gate": wide(), "decay_gate": wide(), "z": wide() if gate else None,
            "decay": (torch.rand(D, generator=g) * 6 - 5 if top is None else torch.full((D,), top)).to(ptype).cuda(),
            "state": n(B, D).cuda() if state else None, "gy": n(B, T, D).to(dtype).cuda(), "gs": n(B, D).cuda()}


def ref(c, C=8.0):
    """name -> (value, bound of the error before the last rounding)"""
    d = lambda t: None if t is None else t.detach().double()
    x, ig, rg, p, z, h0, gy, gs = (d(c.get(n)) for n in ("x", "input_gate", "decay_gate", "decay", "z", "state", "gy", "gs"))
    B, T, D = x.shape
    h0 = torch.zeros((B, D), dtype=torch.float64, device=x.device) if h0 is None else h0
    sp = torch.nn.functional.softplus(p)
    r, i = torch.sigmoid(rg), torch.sigmoid(ig)
    L = -C * sp * r
    a, q = torch.exp(L), -torch.expm1(2 * L)
    m = torch.sqrt(q)
    ds = lambda t: (2 * t.abs() + 8) * U
    dk = (12 + 2.4 * p.abs()) * U
    dL = ds(rg) + dk + U
    da = L.abs() * dL + 5 * U
    dm = 0.5 * (ds(rg) + dk + 8 * U) + 3.5 * da + 7 * U
    db = dm + ds(ig) + 3 * U
    b = m * i * x
    h, H, e = h0, h0.abs(), torch.zeros_like(h0)
    hs, Hs, es = [h], [H], [e]
    for t in range(T):
        e = a[:, t] * e + H * (a[:, t] * (da[:, t] + 3 * U) + FLUSH) + b[:, t].abs() * (db[:, t] + 3 * U)
        H = a[:, t] * H + b[:, t].abs()
        h = a[:, t] * h + b[:, t]
        hs.append(h); Hs.append(H); es.append(e)
    h, H = torch.stack(hs, 1), torch.stack(Hs, 1)
    e = torch.stack(es, 1) + (40 * U * H if T else 0)
    s = None if z is None else torch.sigmoid(z)
    gate, dg = (torch.ones_like(x), torch.zeros_like(x)) if z is None else (z * s, ds(z) + 3 * U)
    out = {"y": (h[:, 1:] * gate, (e[:, 1:] + H[:, 1:] * dg) * gate.abs()), "state": (h[:, -1], e[:, -1])}
    if gy is None:
        return out
    dy = gy * gate
    E, Em, eE = gs, gs.abs(), torch.zeros_like(gs)
    rows = []
    for t in range(T - 1, -1, -1):
        G, Gm, eG = dy[:, t] + E, dy[:, t].abs() + Em, eE + dy[:, t].abs() * dg[:, t]
        rows.append((G, Gm, eG))
        E, Em, eE = a[:, t] * G, a[:, t] * Gm, a[:, t] * eG + Gm * (a[:, t] * (da[:, t] + 3 * U) + FLUSH)
    out["gstate"] = (E, eE + (40 * U * Em if T else 0))
    if T == 0:
        zero = torch.zeros_like(x)
        for n in ("gx", "ginput", "gdecay_gate", "gz"):
            out[n] = (zero, zero)
        out["gdecay"] = (torch.zeros_like(p),) * 2
        return out
    G, Gm, eG = (torch.stack(v[::-1], 1) for v in zip(*rows))
    eG = eG + 40 * U * Gm
    mi, emi = m * i, eG * m * i + Gm * m * i * (dm + ds(ig) + 3 * U)
    out["gx"] = (G * mi, emi)
    out["ginput"] = (G * mi * x * (1 - i), emi * x.abs() * (1 - i) + Gm * mi * x.abs() * (i * ds(ig) + 2 * U))
    slope = torch.where(q > 0, L / torch.where(q > 0, m, 1.0), 0.0)
    t1, t2 = h[:, :-1] * a * L, -i * x * a * a * slope
    m1, m2 = H[:, :-1] * a * L.abs(), t2.abs()
    gLL = G * (t1 + t2)
    egLL = (eG * (m1 + m2) + Gm * a * L.abs() * e[:, :-1] + Gm * L.abs() * H[:, :-1] * FLUSH + Gm * (m1 * (da + dL + 4 * U) + m2 * (2 * da + dL + dm + ds(ig) + 6 * U)))
    out["gdecay_gate"] = (gLL * (1 - r), egLL * (1 - r) + Gm * (m1 + m2) * (r * ds(rg) + 2 * U))
    ratio = torch.sigmoid(p) / sp
    out["gdecay"] = (gLL.sum((0, 1)) * ratio,
                     (egLL.sum((0, 1)) + (Gm * (m1 + m2)).sum((0, 1)) * (2 * dk + (B * T + 4) * U)) * ratio)
    if z is not None:
        dgate = s * (1 + z * (1 - s))
        out["gz"] = (gy * h[:, 1:] * dgate, gy.abs() * (e[:, 1:] * dgate.abs() + H[:, 1:] * s * (1 + z.abs()) * (2 * ds(z) + 8 * U)))
    return out


def close(name, got, want, err):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), name
    half, tiny = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).tiny
    bound = half * (want.abs() + err) + err + tiny
    over = (got.detach().double() - want).abs() / bound
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3f} of the bound at {int(over.argmax())} of {tuple(got.shape)}"


def infer(c, C=8.0):
    import rwkv_infctx_trainer_b200 as W
    y, s = W.gated_recurrence(c["x"], c["input_gate"], c["decay_gate"], c["decay"], c["z"], c["state"], C)
    return {"y": y, "state": s}


def train(c, C=8.0):
    import rwkv_infctx_trainer_b200 as W
    leaves = {n: c[n].detach().requires_grad_(True) for n in LEAVES if c[n] is not None}
    y, s = W.gated_recurrence(leaves["x"], leaves["input_gate"], leaves["decay_gate"], leaves["decay"], leaves.get("z"), leaves.get("state"), C)
    grads = torch.autograd.grad((y, s), list(leaves.values()), (c["gy"], c["gs"]))
    return {"y": y, "state": s, **{GRADS[n]: g for n, g in zip(leaves, grads)}}


def check(c, got, C=8.0):
    want = ref(c, C)
    for n, t in got.items():
        close(n, t, *want[n])


@pytest.mark.parametrize("T", [1, 2, 3, 7, 8, 9, 31, 32, 33, 63, 64, 65, 128, 200])
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_lengths(T, gate, dtype):
    check(c := case(T, 2, T, 70, dtype, gate), train(c))


@pytest.mark.parametrize("D", [1, 2, 3, 4, 6, 7, 8, 31, 63, 64, 65, 66, 72, 130, 1531])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_channels(D, dtype):
    check(c := case(D, 3, 37, D, dtype), train(c))


@pytest.mark.parametrize("B,T,D", [(1, 1100, 64), (1, 513, 40), (2, 700, 1000), (1, 300, 5121), (9, 140, 2048), (40, 65, 520), (1, 4099, 9)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_cut_into_spans(B, T, D, dtype):
    check(c := case(B, B, T, D, dtype), train(c))


@pytest.mark.parametrize("gate,state", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("C", [0.5, 8.0, 50.0])
def test_optional_inputs_and_constants(gate, state, C):
    c = case(1, 2, 90, 50, F32, gate, state)
    got = train(c, C)
    check(c, got, C)
    for n, t in infer(c, C).items():
        assert torch.equal(t, got[n])


@pytest.mark.parametrize("top", [-30.0, -12.0, 0.0, 8.0, 60.0])
def test_decays_from_almost_one_to_zero(top):
    check(c := case(2, 2, 100, 40, F32, top=top), train(c))


@pytest.mark.parametrize("D", [48, 45])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_views_of_wider_tensors(D, dtype):
    c = case(3, 2, 70, D, dtype, strided=True)
    got = train(c)
    check(c, got)
    for lay in (lambda t: t.contiguous(), lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):
        for n, t in train({k: lay(v) if k in LEAVES and k not in ("decay", "state") else v for k, v in c.items()}).items():
            assert torch.equal(t, got[n]), n


def test_a_row_for_all_and_one_token_for_all():
    c = case(4, 1, 50, 40, F32)
    for sizes in ((3, 50, 40),):
        wide = {n: c[n].expand(sizes) if n in ("x", "input_gate", "decay_gate", "z", "gy") else c[n] for n in c}
        wide["state"], wide["gs"] = c["state"].expand(3, 40), c["gs"].expand(3, 40)
        check(wide, train(wide))
    one = dict(c, decay_gate=c["decay_gate"][:, :1].expand(1, 50, 40))
    check(one, train(one))


def test_parameters_of_every_float_type():
    for pt in (BF, HF, F32, torch.float64):
        c = case(5, 2, 40, 24, BF, ptype=pt)
        got = train(c)
        assert got["gdecay"].dtype == pt
        check(c, got)


def test_empty_calls():
    c = case(6, 2, 0, 24, BF)
    got = train(c)
    assert got["y"].shape == (2, 0, 24) and torch.equal(got["state"], c["state"]) and torch.equal(got["gstate"], c["gs"])
    assert float(got["gdecay"].abs().max()) == 0.0
    assert float(infer(dict(c, state=None))["state"].abs().max()) == 0.0
    for B, D in ((0, 24), (2, 0)):
        got = train(case(6, B, 5, D, BF))
        assert got["y"].shape == (B, 5, D) and got["state"].shape == (B, D) and float(got["gdecay"].abs().sum()) == 0.0


@pytest.mark.parametrize("cuts", [[0, 20, 21, 23, 150], [0, 64, 128, 129, 150], [0, 0, 150]])
def test_segments_are_the_unsplit_row(cuts):
    import rwkv_infctx_trainer_b200 as W
    c = case(7, 2, 150, 24, F32)
    leaves = {n: c[n].detach().requires_grad_(True) for n in LEAVES}
    s, ys = leaves["state"], []
    for a, b in zip(cuts, cuts[1:]):
        y, s = W.gated_recurrence(*(leaves[n][:, a:b] for n in ("x", "input_gate", "decay_gate")), leaves["decay"], leaves["z"][:, a:b], s)
        ys.append(y)
    y = torch.cat(ys, 1)
    grads = torch.autograd.grad((y, s), list(leaves.values()), (c["gy"], c["gs"]))
    check(c, {"y": y, "state": s, **{GRADS[n]: g for n, g in zip(leaves, grads)}})


@pytest.mark.parametrize("D", [64, 41, 2, 1])
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_single_tokens_continue_a_prompt(D, gate, dtype):
    import rwkv_infctx_trainer_b200 as W
    c = case(8, 3, 30, D, dtype, gate, strided=True)
    want = ref({**c, "gy": None})
    state = infer({n: t[:, :20] if t is not None and t.dim() == 3 else t for n, t in c.items()})["state"]
    for t in range(20, 30):
        one = lambda n: None if c[n] is None else c[n][:, t]
        kept = state
        y = W.gated_recurrence_step(one("x"), one("input_gate"), one("decay_gate"), c["decay"], state, one("z"))
        assert kept is state
        close("y", y, want["y"][0][:, t], want["y"][1][:, t])
    close("state", state, *want["state"])


def test_a_step_of_many_rows():
    import rwkv_infctx_trainer_b200 as W
    c = case(9, 70001, 1, 6, F32)
    want, state = ref({**c, "gy": None}), c["state"].clone()
    y = W.gated_recurrence_step(c["x"][:, 0], c["input_gate"][:, 0], c["decay_gate"][:, 0], c["decay"], state, c["z"][:, 0])
    close("y", y, want["y"][0][:, 0], want["y"][1][:, 0])
    close("state", state, *want["state"])
    check(c, train(c))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_closed_gates_keep_the_state(dtype):
    """masked tokens (a decay gate of minus infinity) leave the state as it is and have no gradient"""
    c = case(10, 2, 90, 40, dtype)
    mask = torch.zeros(2, 90, dtype=torch.bool)
    mask[0, 30:], mask[1, :17], mask[1, 50:60] = True, True, True
    mask = mask.cuda()
    c["decay_gate"] = c["decay_gate"].masked_fill(mask.unsqueeze(-1), -INF)
    c["x"] = c["x"].masked_fill(mask.unsqueeze(-1), torch.finfo(dtype).min / 4)
    got = train(c)
    assert torch.isfinite(got["gdecay"]).all()
    for n in ("gx", "ginput", "gdecay_gate"):
        assert float(got[n].masked_fill(~mask.unsqueeze(-1), 0).abs().max()) == 0.0, n
    short = infer({n: t[:1, :30] if t is not None and t.dim() == 3 else t[:1] if n in ("state", "gs") else t for n, t in c.items()})
    # (30 tokens and 90 may be divided among CTAs otherwise: 40 U each of the sum of the magnitudes, 30 inputs and a state below 4)
    assert float((short["state"] - got["state"][:1]).detach().abs().max()) <= 2 * 40 * U * 31 * 4
    everything = dict(c, decay_gate=torch.full_like(c["decay_gate"], -INF))
    got = train(everything)
    assert torch.equal(got["state"], c["state"])


def test_infinities_and_nans_stay_in_their_channel_and_behind_their_token():
    for name, value in (("x", INF), ("x", float("nan")), ("input_gate", float("nan")), ("decay_gate", float("nan")), ("z", float("nan"))):
        c = case(11, 2, 70, 10, F32)
        clean = infer(c)
        c[name] = c[name].clone()
        c[name][1, 33, 4] = value
        got = infer(c)
        assert torch.equal(got["y"][0], clean["y"][0]) and torch.equal(got["y"][1, :33], clean["y"][1, :33])
        keep = [k for k in range(10) if k != 4]
        assert torch.equal(got["y"][..., keep], clean["y"][..., keep])
        assert not torch.isfinite(got["y"][1, 33, 4])
    c = case(11, 2, 70, 10, F32)
    for gate, value in ((INF, 1.0), (-INF, 0.0)):                 # gates that are wide open or closed
        d = dict(c, input_gate=torch.full_like(c["input_gate"], gate), decay=torch.full_like(c["decay"], INF if gate > 0 else -2.0))
        got = train(d)
        assert torch.isfinite(got["y"]).all() and torch.isfinite(got["gx"]).all()
        if value == 0.0:
            assert float(got["gx"].abs().max()) == 0.0


def test_the_same_bits_every_time_and_only_the_gradients_asked_for():
    import rwkv_infctx_trainer_b200 as W
    c = case(12, 2, 300, 200, BF)
    first = train(c)
    for n, t in train(c).items():
        assert torch.equal(t, first[n])
    for name in LEAVES:
        leaf = c[name].detach().requires_grad_(True)
        y, s = W.gated_recurrence(*(leaf if n == name else c[n] for n in LEAVES))
        g, = torch.autograd.grad((y, s), leaf, (c["gy"], c["gs"]))
        assert torch.equal(g, first[GRADS[name]]), name
    leaf = c["x"].detach().requires_grad_(True)
    for pick in (0, 1):                                           # a gradient on one of the two outputs
        out = W.gated_recurrence(leaf, *(c[n] for n in LEAVES[1:]))
        g, = torch.autograd.grad(out[pick], leaf, (c["gy"], c["gs"])[pick])
        want = ref({**c, "gy": c["gy"] if pick == 0 else torch.zeros_like(c["gy"]), "gs": c["gs"] if pick == 1 else torch.zeros_like(c["gs"])})["gx"]
        close("gx", g, *want)


def test_gradients_against_differences():
    """the gradient in a direction against (f(+) - f(-)) / 2e of the formulas in 64 bits, e = 1e-5: its own error is e^2 f''' and
    2^-53 f / e, both below 1e-9 of the sums"""
    c = case(13, 2, 40, 20, F32)
    got = train(c)
    g = torch.Generator(device="cuda").manual_seed(1)
    for n in LEAVES:
        v = torch.randn(c[n].shape, generator=g, device="cuda", dtype=torch.float64)
        f = []
        for e in (1e-5, -1e-5):
            o = ref({**c, n: c[n].double() + e * v, "gy": None})
            f.append(float((o["y"][0] * c["gy"].double()).sum() + (o["state"][0] * c["gs"].double()).sum()))
        want = (f[0] - f[1]) / 2e-5
        bound = ref(c)[GRADS[n]][1]
        slack = float((bound * v.abs()).sum() + U * (got[GRADS[n]].double() * v).abs().sum()) + 1e-6 * max(1.0, abs(want))
        assert abs(float((got[GRADS[n]].double() * v).sum()) - want) <= slack, n


def test_captured_and_replayed_and_on_another_stream():
    import rwkv_infctx_trainer_b200 as W
    c = case(14, 2, 130, 66, BF)
    want = train(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = train(c)
    side.synchronize()
    for n in want:
        assert torch.equal(got[n], want[n]), n
    static = {n: t.clone() for n, t in c.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = train(static)
    for seed in (15, 16):
        new = case(seed, 2, 130, 66, BF)
        for n in static:
            static[n].copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        for n, t in train(new).items():
            assert torch.equal(out[n], t), n


def test_more_than_two_to_the_31_elements():
    """the last tokens of a tensor of 2^31 elements and more: from the state before them they are a call of their own"""
    import rwkv_infctx_trainer_b200 as W
    T, D, tail = 33100, 65536, 70
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((1, T, D), generator=g, device="cuda", dtype=BF)
    decay = torch.randn(D, generator=g, device="cuda")
    y, s = W.gated_recurrence(x, x, x, decay)
    _, before = W.gated_recurrence(x[:, :T - tail], x[:, :T - tail], x[:, :T - tail], decay)
    y2, s2 = W.gated_recurrence(x[:, T - tail:], x[:, T - tail:], x[:, T - tail:], decay, state=before)
    # (tokens fall into segments otherwise: each of 70 steps may round differently, 4 U a step of states that add up to below 70)
    assert float((s - s2).abs().max()) <= 4 * 70 * U * 70
    assert float((y[:, T - tail:].float() - y2.float()).abs().max()) <= 2.0 ** -8 * float(y2.float().abs().max())
