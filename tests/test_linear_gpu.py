"""The matrix products with their epilogue against their formulas in 64 bits: every way a product is cut, every activation, odd
sizes, strides and alignments, few rows, both 16-bit types."""
import pytest
import torch

import linear_testlib as L

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("rows,K,N", [(128, 64, 128), (17, 64, 128), (300, 128, 256), (129, 192, 136), (256, 1024, 264)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_forward(rows, K, N, dtype):
    import rwkv_infctx_trainer_b200 as W
    c = L.linear_case(rows, rows, K, N, dtype)
    L.close("y", W.linear_act(c["x"], c["weight"]), *L.linear_ref(c["x"], c["weight"], None, "none", None, None)["y"])


@pytest.mark.parametrize("rows,K,N", [(17, 64, 64), (128, 64, 128), (129, 72, 136), (256, 512, 256), (300, 1000, 520), (1000, 200, 1032), (64, 4096, 128),
                                      (2000, 64, 64), (64, 64, 2000)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_gradients(rows, K, N, dtype):
    L.check_linear(c := L.linear_case(rows, rows, K, N, dtype), "none", L.train_linear(c, "none"))


@pytest.mark.parametrize("name", L.ACTS)
@pytest.mark.parametrize("rows", [3, 12, 70, 400])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_activations_with_everything(name, rows, dtype):
    c = L.linear_case(1, rows, 136, 264, dtype, bias=True, mul=True, residual=True)
    L.check_linear(c, name, L.train_linear(c, name))


@pytest.mark.parametrize("bias,mul,residual", [(True, False, False), (False, True, False), (False, False, True), (True, False, True), (False, True, True)])
@pytest.mark.parametrize("name", ["none", "gelu"])
@pytest.mark.parametrize("rows", [5, 200])
def test_optional_inputs(bias, mul, residual, name, rows):
    c = L.linear_case(2, rows, 100, 90, BF, bias, mul, residual)
    L.check_linear(c, name, L.train_linear(c, name))


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 15, 16, 17, 31, 127, 128, 129, 255, 256, 257])
@pytest.mark.parametrize("K,N", [(72, 40), (65, 33)])
def test_rows(rows, K, N):
    c = L.linear_case(rows, rows, K, N, BF, bias=True)
    L.check_linear(c, "silu", L.train_linear(c, "silu"))


@pytest.mark.parametrize("K", [1, 2, 7, 8, 9, 31, 63, 64, 65, 127, 129, 511, 513, 1531])
@pytest.mark.parametrize("rows", [4, 40])
def test_contraction_lengths(K, rows):
    c = L.linear_case(K, rows, K, 72, HF)
    L.check_linear(c, "sigmoid", L.train_linear(c, "sigmoid"))


@pytest.mark.parametrize("N", [1, 2, 7, 8, 9, 15, 16, 17, 63, 64, 65, 127, 129, 255, 257, 1001])
@pytest.mark.parametrize("rows", [4, 40])
def test_columns(N, rows):
    c = L.linear_case(N, rows, 80, N, BF, bias=True, mul=True, residual=True)
    L.check_linear(c, "relu2", L.train_linear(c, "relu2"))


@pytest.mark.parametrize("rows,K,N", [(4096, 520, 3080), (300, 8192, 264), (8200, 264, 300), (2049, 129, 4100)])
def test_many_tiles_and_long_contractions(rows, K, N):
    c = L.linear_case(3, rows, K, N, BF, bias=True, residual=True)
    L.check_linear(c, "gelu", L.train_linear(c, "gelu"))


@pytest.mark.parametrize("rows,K,N", [(1, 64, 8), (8, 520, 40), (16, 136, 24), (17, 64, 64), (130, 200, 72), (300, 264, 520), (5, 33, 9), (50, 65, 33), (4100, 264, 1100),
                                      (8, 2560, 1000)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_gated_pairs(rows, K, N, dtype):
    L.check_gated(c := L.gated_case(rows, rows, K, N, dtype), "silu", L.train_gated(c, "silu"))


@pytest.mark.parametrize("name", L.ACTS)
@pytest.mark.parametrize("rows", [6, 140])
def test_gated_activations(name, rows):
    L.check_gated(c := L.gated_case(4, rows, 200, 136, BF), name, L.train_gated(c, name))


@pytest.mark.parametrize("rows", [6, 140])
def test_leading_dimensions_views_and_strides(rows):
    """the same numbers wherever they lie: the same bits"""
    import rwkv_infctx_trainer_b200 as W
    K, N = 136, 72
    c = L.linear_case(5, rows, K, N, BF, bias=True, mul=True, residual=True)
    want = L.train_linear(c, "silu")
    wide = lambda t, at: torch.cat((torch.ones_like(t[:, :at]), t, torch.ones_like(t)), 1)[:, at:at + t.shape[1]]
    off = lambda t: torch.cat((t.new_ones(1), t.reshape(-1)))[1:].view(t.shape)          # two bytes off
    for lay in (lambda t: wide(t, 8), lambda t: wide(t, 3), off, lambda t: t.t().contiguous().t(), lambda t: torch.stack((t, t), 1)[:, 1]):
        got = L.train_linear({n: lay(t) if t is not None and t.dim() == 2 else t for n, t in c.items()}, "silu")
        for n in want:
            assert torch.equal(got[n], want[n]), n
    up = lambda t: t.view(2, rows // 2, t.shape[1])
    y = W.linear_act(up(c["x"]), c["weight"], c["bias"], "silu", up(c["mul"]), up(c["residual"]))
    assert y.shape == (2, rows // 2, N) and torch.equal(y.view(rows, N), want["y"])
    y = W.linear_act(up(c["x"]).transpose(0, 1), c["weight"], c["bias"], "silu", up(c["mul"]).transpose(0, 1), up(c["residual"]).transpose(0, 1))
    assert torch.equal(y.transpose(0, 1).reshape(rows, N), want["y"])
    assert torch.equal(W.linear_act(c["x"][0], c["weight"]), W.linear_act(c["x"][:1], c["weight"])[0])
    g = L.gated_case(5, rows, K, N, BF)
    want = L.train_gated(g, "gelu")
    for lay in (lambda t: wide(t, 8), lambda t: wide(t, 3), off, lambda t: t.t().contiguous().t()):
        got = L.train_gated({n: lay(t) for n, t in g.items()}, "gelu")
        for n in want:
            assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("rows", [4, 60])
def test_one_row_for_all_and_gradients_that_are_broadcast(rows):
    import rwkv_infctx_trainer_b200 as W
    c = L.linear_case(6, rows, 72, 48, BF)
    x = c["x"][:1].clone().requires_grad_(True)
    y = W.linear_act(x.expand(rows, 72), c["weight"], None, "silu")
    assert torch.equal(y, W.linear_act(c["x"][:1].repeat(rows, 1), c["weight"], None, "silu"))
    g, = torch.autograd.grad(y.sum(), x)
    d = dict(c, x=c["x"][:1].repeat(rows, 1), gy=torch.ones_like(c["gy"]))
    want, err = L.linear_ref(d["x"], d["weight"], None, "silu", None, None, d["gy"])["gx"]
    # (autograd adds the rows' rounded gradients in the type: half a step of each and of every partial sum)
    h = L.half(BF)
    bound = (err + h * want.abs()).sum(0) + rows * h * want.abs().sum(0) * 2
    assert bool(((g[0].double() - want.sum(0)).abs() <= bound).all())


def test_bias_of_every_float_type():
    for bt in (BF, HF, F32, torch.float64):
        c = L.linear_case(7, 90, 64, 40, BF, bias=True, btype=bt)
        got = L.train_linear(c, "none")
        assert got["gbias"].dtype == bt
        L.check_linear(c, "none", got)


def test_empty_calls():
    import rwkv_infctx_trainer_b200 as W
    c = L.linear_case(8, 0, 24, 40, BF, bias=True, mul=True, residual=True)
    got = L.train_linear(c, "gelu")
    assert got["y"].shape == (0, 40) and got["gx"].shape == (0, 24)
    assert float(got["gweight"].abs().max()) == 0.0 and float(got["gbias"].abs().max()) == 0.0
    got = L.train_gated(L.gated_case(8, 0, 24, 40, HF), "silu")
    assert got["y"].shape == (0, 40) and float(got["gw_gate"].abs().max()) == 0.0 and float(got["gw_up"].abs().max()) == 0.0
    assert W.linear_act(c["x"].view(3, 0, 24), c["weight"]).shape == (3, 0, 40)


@pytest.mark.parametrize("rows", [6, 200])
def test_infinities_and_nans_stay_in_their_rows(rows):
    import rwkv_infctx_trainer_b200 as W
    c = L.linear_case(9, rows, 72, 48, BF)
    clean = W.linear_act(c["x"], c["weight"], None, "silu")
    x = c["x"].clone()
    x[1, 5], x[3, 70] = float("nan"), float("inf")
    got = W.linear_act(x, c["weight"], None, "silu")
    keep = [r for r in range(rows) if r not in (1, 3)]
    assert torch.equal(got[keep], clean[keep]) and torch.isnan(got[1]).all()
    for name in L.ACTS:                                           # a NaN pre-activation is a NaN
        assert torch.isnan(W.linear_act(x, c["weight"], None, name)[1]).all(), name
        assert torch.isnan(W.gated_linear(x, c["weight"], c["weight"], name)[1]).all(), name
    big = torch.full_like(c["weight"], 300.0)                     # pre-activations far out
    for name, want in (("sigmoid", 1.0), ("gelu", None), ("silu", None)):
        y = W.linear_act(torch.full_like(c["x"], 3.0), big, None, name)
        assert torch.equal(y, torch.full_like(y, 300.0 * 3.0 * 72 if want is None else want)), name
        y = W.linear_act(torch.full_like(c["x"], -3.0), big, None, name)
        assert float(y.abs().max()) == 0.0, name


def test_the_same_bits_every_time_and_only_the_gradients_asked_for():
    import rwkv_infctx_trainer_b200 as W
    c = L.linear_case(10, 300, 200, 136, BF, bias=True, mul=True, residual=True)
    first = L.train_linear(c, "gelu")
    for n, t in L.train_linear(c, "gelu").items():
        assert torch.equal(t, first[n])
    for name in L.LINEAR:
        leaf = c[name].detach().requires_grad_(True)
        a = {n: leaf if n == name else c[n] for n in L.LINEAR}
        y = W.linear_act(a["x"], a["weight"], a["bias"], "gelu", a["mul"], a["residual"])
        assert torch.equal(torch.autograd.grad(y, leaf, c["gy"])[0], first["g" + name]), name
    g = L.gated_case(10, 300, 200, 136, BF)
    first = L.train_gated(g, "silu")
    for name in L.GATED:
        leaf = g[name].detach().requires_grad_(True)
        a = {n: leaf if n == name else g[n] for n in L.GATED}
        y = W.gated_linear(a["x"], a["w_gate"], a["w_up"])
        assert torch.equal(torch.autograd.grad(y, leaf, g["gy"])[0], first["g" + name]), name
    with torch.no_grad():
        assert torch.equal(W.gated_linear(g["x"], g["w_gate"], g["w_up"]), first["y"])


def test_gradients_against_differences():
    """(f(+) - f(-)) / 2e of the formulas in 64 bits against the gradient's product with the direction"""
    c = L.linear_case(11, 40, 48, 32, HF, bias=True, mul=True, residual=True)
    got = L.train_linear(c, "gelu")
    want = L.linear_ref(c["x"], c["weight"], c["bias"], "gelu", c["mul"], c["residual"], c["gy"])
    g = torch.Generator(device="cuda").manual_seed(1)
    d = {n: c[n].double() for n in L.LINEAR}
    for n in L.LINEAR:
        v = torch.randn(c[n].shape, generator=g, device="cuda", dtype=torch.float64)
        f = []
        for e in (1e-5, -1e-5):
            p = {**d, n: d[n] + e * v}
            z = p["x"] @ p["weight"].t() + p["bias"]
            f.append(float(((L.act("gelu", z)[0] * p["mul"] + p["residual"]) * c["gy"].double()).sum()))
        diff, grad = (f[0] - f[1]) / 2e-5, got["g" + n].double()
        err = want["g" + n][1] if n != "residual" else torch.zeros_like(v)
        slack = float(((err + L.half(HF) * grad.abs() + L.least(HF)) * v.abs()).sum()) + 1e-6 * max(1.0, abs(diff))
        assert abs(float((grad * v).sum()) - diff) <= slack, n


def test_captured_and_replayed_and_on_another_stream():
    for rows in (5, 300):
        c = L.linear_case(12, rows, 136, 72, BF, bias=True, mul=True)
        want = L.train_linear(c, "gelu")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = L.train_linear(c, "gelu")
        side.synchronize()
        for n in want:
            assert torch.equal(got[n], want[n]), n
        static = {n: None if t is None else t.clone() for n, t in c.items()}
        graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = L.train_linear(static, "gelu")
        with torch.cuda.graph(second):
            out2 = L.train_gated({"x": static["x"], "w_gate": static["weight"], "w_up": static["weight"], "gy": static["gy"]}, "silu")
        for seed in (13, 14):
            new = L.linear_case(seed, rows, 136, 72, BF, bias=True, mul=True)
            for n in static:
                if static[n] is not None:
                    static[n].copy_(new[n])
            graph.replay()
            second.replay()
            torch.cuda.synchronize()
            for n, t in L.train_linear(new, "gelu").items():
                assert torch.equal(out[n], t), n
            for n, t in L.train_gated({"x": new["x"], "w_gate": new["weight"], "w_up": new["weight"], "gy": new["gy"]}, "silu").items():
                assert torch.equal(out2[n], t), n


def test_two_streams_at_once():
    cases = [L.linear_case(20 + i, 300, 264, 520, BF, bias=True) for i in range(2)]
    want = [L.train_linear(c, "silu") for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(L.train_linear(cases[i], "silu"))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for n in want[i]:
                assert torch.equal(r[n], want[i][n]), n


def test_more_than_two_to_the_31_elements():
    """rows behind 2^31 elements of x and of y (a call of fewer rows may add up its sums in another order: against 64 bits)"""
    import rwkv_infctx_trainer_b200 as W
    rows, K, N = 265000, 8192, 8200
    w = torch.randn((N, K), device="cuda", dtype=BF) * K ** -0.5
    x = torch.randn((rows, K), device="cuda", dtype=BF)
    y = W.linear_act(x, w)
    for at in (0, 262143, rows - 300):
        L.close(f"y {at}", y[at:at + 256], *L.linear_ref(x[at:at + 256], w, None, "none", None, None)["y"])
