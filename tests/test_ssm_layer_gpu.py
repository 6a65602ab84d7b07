"""The norm, the convolution and the scan together, as a layer uses them -- norm with the residual, projection, convolution,
projection, scan, projection -- and what a program does around them: prompts and decoded tokens, segments, graphs, streams,
threads, tensors of more than 2^31 elements."""
import threading

import pytest
import torch
import torch.nn.functional as F

import ssm_testlib as S

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
C, D, N, R, W4 = 48, 96, 16, 8, 4


def params(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, std=1.0: (torch.randn(s, generator=g) * std)
    p = {"norm": 1 + 0.1 * n(C), "in_proj": n(2 * D, C, std=C ** -0.5), "conv": n(D, W4, std=0.5), "conv_bias": 0.1 * n(D),
         "x_proj": n(R + 2 * N, D, std=D ** -0.5), "dt_proj": n(D, R, std=R ** -0.5), "dt_bias": n(D) - 3,
         "A": -torch.exp(n(D, N, std=0.5)), "D": 1 + 0.1 * n(D), "out_proj": n(C, D, std=D ** -0.5)}
    big = ("in_proj", "x_proj", "dt_proj", "out_proj")
    return {k: v.to(dtype if k in big else F32).cuda() for k, v in p.items()}


def layer(p, x, res, conv_state, state):
    import rwkv_infctx_trainer_b200 as W
    y, h = W.rms_norm(x, p["norm"], res)
    u, z = F.linear(y, p["in_proj"]).chunk(2, -1)
    u, conv_state = W.causal_conv(u, p["conv"], p["conv_bias"], conv_state)
    dt, B, Cm = F.linear(u, p["x_proj"]).split((R, N, N), -1)
    y, state = W.selective_scan(u, F.linear(dt, p["dt_proj"]), p["A"], B, Cm, p["D"], z, p["dt_bias"], state=state)
    return F.linear(y, p["out_proj"]), h, conv_state, state


def step(p, x, res, conv_state, state):
    import rwkv_infctx_trainer_b200 as W
    y, h = W.rms_norm(x, p["norm"], res)
    u, z = F.linear(y, p["in_proj"]).chunk(2, -1)
    u = W.causal_conv_step(u, conv_state, p["conv"], p["conv_bias"])
    dt, B, Cm = F.linear(u, p["x_proj"]).split((R, N, N), -1)
    y = W.selective_scan_step(u, F.linear(dt, p["dt_proj"]), p["A"], B, Cm, state, p["D"], z, p["dt_bias"])
    return F.linear(y, p["out_proj"]), h


def layer64(p, x, res, conv_state, state):
    h = x + res
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6) * p["norm"]
    u, z = F.linear(y, p["in_proj"]).chunk(2, -1)
    xs = torch.cat((conv_state, u), 1)
    u = F.silu(sum(xs[:, j:j + x.shape[1]] * p["conv"][:, j] for j in range(W4)) + p["conv_bias"])
    dt, B, Cm = F.linear(u, p["x_proj"]).split((R, N, N), -1)
    dt = F.softplus(F.linear(dt, p["dt_proj"]) + p["dt_bias"])
    ys = []
    for t in range(x.shape[1]):
        state = torch.exp(dt[:, t].unsqueeze(-1) * p["A"]) * state + (dt[:, t] * u[:, t]).unsqueeze(-1) * B[:, t].unsqueeze(1)
        ys.append((state * Cm[:, t].unsqueeze(1)).sum(-1))
    y = (torch.stack(ys, 1) + p["D"] * u) * F.silu(z)
    return F.linear(y, p["out_proj"]), h, xs[:, x.shape[1]:], state


def inputs(B, T, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)
    return (n(B, T, C).to(dtype).cuda(), n(B, T, C).to(dtype).cuda(), n(B, W4 - 1, D).to(dtype).cuda(), n(B, D, N).cuda())


def rel(a, b):
    return float((a.double() - b).norm() / b.norm())


@pytest.mark.parametrize("cuts", [[0, 24], [0, 9, 10, 24]])
def test_layer_in_fp32_and_its_gradients(cuts):
    """against the layer in 64 bits, in one call and in segments with both states and their gradients carried.  Tolerance of the
    2-norm: ten operations forward and ten back, none of which adds more than 1100 roundings of 2^-24 to a term (the scan:
    16 T + 300 = 700, the projections: their width, at most 96, the parameters' sums: B T = 48 more), each amplified by at most 4
    (the norm of a projection's matrix, about 2; the gates' slopes, 1.1; softplus' exponent 16 2^-24 of its argument): 20 * 1100 * 4 * 2^-24
    would be 5e-3, were all of them of one sign; 1e-4, a fiftieth of it, is held to"""
    torch.backends.cuda.matmul.allow_tf32 = False
    p = params(F32)
    x, res, cs, st = inputs(2, 24, F32)
    leaves = {**p, "x": x, "res": res, "cs": cs, "st": st}
    leaves = {k: v.detach().requires_grad_(True) for k, v in leaves.items()}
    c, s, ys, hs = leaves["cs"], leaves["st"], [], []
    for a, b in zip(cuts, cuts[1:]):
        y, h, c, s = layer(leaves, leaves["x"][:, a:b], leaves["res"][:, a:b], c, s)
        ys.append(y)
        hs.append(h)
    out = [torch.cat(ys, 1), torch.cat(hs, 1), c, s]
    d = {k: v.detach().double().requires_grad_(True) for k, v in leaves.items()}
    want = layer64(d, d["x"], d["res"], d["cs"], d["st"])
    seeds = [torch.randn_like(o) for o in out]
    got_g = torch.autograd.grad(out, list(leaves.values()), seeds)
    want_g = torch.autograd.grad(want, list(d.values()), [t.double() for t in seeds])
    for n, a, b in [*zip(("y", "h", "conv_state", "state"), out, want), *zip(leaves, got_g, want_g)]:
        assert rel(a.detach(), b.detach()) <= 1e-4, (n, rel(a.detach(), b.detach()))


def test_decoded_tokens_follow_a_prompt():
    """a bf16 layer token by token against the layer over the whole row.  The same operations on the same values but for the
    projections (a library product may add up in another order for one row) and the scan (the same sums): outputs differ by
    roundings of bf16, 2^-8 of a value, of which a term passes six"""
    p = params(BF)
    x, res, cs, st = inputs(3, 30, BF)
    with torch.no_grad():
        want, wh, wc, ws = layer(p, x, res, cs, st)
        y, h, c, s = layer(p, x[:, :22], res[:, :22], cs, st)
        ys = [y]
        for t in range(22, 30):
            y, h = step(p, x[:, t], res[:, t], c, s)
            assert torch.equal(h, wh[:, t])
            ys.append(y.unsqueeze(1))
    assert rel(torch.cat(ys, 1), want.double()) <= 6 * 2.0 ** -8
    assert rel(c, wc.double()) <= 6 * 2.0 ** -8 and rel(s, ws.double()) <= 6 * 2.0 ** -8


def test_decode_step_in_a_graph():
    """captured once, replayed with new inputs in the same places: what plain calls give, state after state"""
    p = params(BF)
    x, res, cs, st = inputs(4, 12, BF)
    with torch.no_grad():
        c0, s0 = cs.clone(), st.clone()
        want = [step(p, x[:, t].contiguous(), res[:, t].contiguous(), c0, s0)[0] for t in range(12)]
        bx, br, c, s = x[:, 0].clone(), res[:, 0].clone(), cs.clone(), st.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(p, bx, br, c.clone(), s.clone())          # (the library's products set themselves up)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                y, _ = step(p, bx, br, c, s)
        torch.cuda.current_stream().wait_stream(side)
        for t in range(12):
            bx.copy_(x[:, t])
            br.copy_(res[:, t])
            graph.replay()
            assert rel(y, want[t].double()) <= 6 * 2.0 ** -8
        assert rel(c, c0.double()) <= 6 * 2.0 ** -8 and rel(s, s0.double()) <= 6 * 2.0 ** -8


@pytest.mark.parametrize("T", [20, 200])
def test_training_in_graphs_beside_an_eager_graph(T):
    """forward and backward captured, twice, while an eager graph of the same leaves lives: replays of either, in either order,
    give the eager call's bits (each has its own workspaces).  (The eager graph is one of the capturing stream: the leaves' nodes keep
    the stream of the graph that made them, and torch refuses to capture across the default stream.)"""
    import rwkv_infctx_trainer_b200 as W
    c = S.scan_case(T, 2, T, 40, 16, 1, BF)
    leaves = [c[n].requires_grad_(True) for n in S.SCAN_LEAVES]
    cw, cb = torch.randn((40, 4), device="cuda", requires_grad=True), torch.randn(40, device="cuda", requires_grad=True)
    nw = torch.rand(40, device="cuda", requires_grad=True)
    leaves += [cw, cb, nw]

    def run():
        u, h = W.rms_norm(c["u"], nw, c["z"])
        u, cs = W.causal_conv(u, cw, cb)
        y, s = W.selective_scan(u, c["delta"], c["A"], c["B"], c["C"], c["D"], h, c["delta_bias"], state=c["state"])
        return [y, s], [cs]

    def train():
        out, more = run()
        return [t.detach() for t in out + more] + list(torch.autograd.grad(out, leaves, (c["gy"], c["gs"])))

    want = [t.clone() for t in train()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        alive, _ = run()                                   # an eager graph of the same leaves
        train()
        side.synchronize()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs = train()
            graphs.append((g, outs))
    torch.cuda.current_stream().wait_stream(side)
    for k in (0, 1, 1, 0):
        for t in graphs[k][1]:
            t.zero_()
        graphs[k][0].replay()
        for a, b in zip(graphs[k][1], want):
            assert torch.equal(a, b)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = torch.autograd.grad(alive, leaves, (c["gy"], c["gs"]))
    side.synchronize()
    for a, b in zip(got, want[3:]):
        assert torch.equal(a, b)


def test_on_another_stream_and_on_a_new_thread():
    import rwkv_infctx_trainer_b200 as W
    c = S.scan_case(3, 2, 150, 40, 16, 1, BF)
    call = lambda: W.selective_scan(c["u"], c["delta"], c["A"], c["B"], c["C"], c["D"], c["z"], c["delta_bias"], state=c["state"])
    want = call()
    torch.cuda.synchronize()
    got = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got.append(call())
        s.synchronize()

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 4
    for y, s in got:
        assert torch.equal(y, want[0]) and torch.equal(s, want[1])


def test_the_same_tensor_in_several_places():
    """u, delta and z one tensor, x and residual one tensor: the gradients add up"""
    import rwkv_infctx_trainer_b200 as W
    c = S.scan_case(4, 2, 30, 40, 16, 1, F32)
    x = c["u"].requires_grad_(True)
    y, _ = W.selective_scan(x, x, c["A"], c["B"], c["C"], None, x)
    a, b, d = (x.detach().clone().requires_grad_(True) for _ in range(3))
    y2, _ = W.selective_scan(a, b, c["A"], c["B"], c["C"], None, d)
    one = torch.autograd.grad(y, x, c["gy"])[0]
    three = torch.autograd.grad(y2, (a, b, d), c["gy"])
    # (three roundings of a sum)
    assert float((one - sum(three)).abs().max()) <= 4 * S.U * float(sum(t.abs() for t in three).max())
    w = torch.ones(40, device="cuda")
    y, h = W.rms_norm(x, w, x)
    assert torch.equal(h, 2 * x)
    # d/dx of 2x: twice each gradient that reaches it
    y2, h2 = W.rms_norm(a, w, b)
    g = torch.autograd.grad((y2, h2), (a, b), (c["gy"], c["gy"]))
    assert torch.equal(torch.autograd.grad((y, h), x, (c["gy"], c["gy"]))[0], g[0] + g[1])


def test_saved_tensors_that_went_to_the_host():
    import rwkv_infctx_trainer_b200 as W
    c = S.scan_case(5, 2, 50, 40, 16, 1, BF, strided=True)
    leaves = [c[n].requires_grad_(True) for n in S.SCAN_LEAVES]
    cw, nw = torch.randn((40, 4), device="cuda", requires_grad=True), torch.rand(40, device="cuda", requires_grad=True)

    def run():
        u, h = W.rms_norm(c["u"], nw, c["z"])
        u, _ = W.causal_conv(u, cw)
        y, s = W.selective_scan(u, c["delta"], c["A"], c["B"], c["C"], c["D"], h, c["delta_bias"], state=c["state"])
        return torch.autograd.grad((y, s), leaves + [cw, nw], (c["gy"], c["gs"]))

    want = run()
    with torch.autograd.graph.save_on_cpu():
        got = run()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_offsets_that_pass_32_bits():
    """views of a tensor of more than 2^31 elements, and outputs of as many"""
    import rwkv_infctx_trainer_b200 as W
    T, wide, d = 66000, 33000, 64
    big = torch.empty((1, T, wide), dtype=BF, device="cuda")
    assert big.numel() > 2 ** 31
    view = big[..., wide - d:]
    view.normal_()
    bc = big[..., :32]
    bc.normal_()
    delta = torch.randn((1, T, d), device="cuda").to(BF)
    A = -torch.rand((d, 16), device="cuda") - 0.1
    Bm, Cm = bc[..., :16], bc[..., 16:]
    for keep in (False, True):
        with torch.set_grad_enabled(keep):
            a = view.detach().requires_grad_(keep)
            b = view.contiguous().detach().requires_grad_(keep)
            (y1, s1), (y2, s2) = (W.selective_scan(t, delta, A, Bm, Cm, z=t) for t in (a, b))
            (c1, _), (c2, _) = (W.causal_conv(t, A[:, :4].contiguous()) for t in (a, b))
            assert torch.equal(y1, y2) and torch.equal(s1, s2) and torch.equal(c1, c2)
            if keep:
                g1, g2 = (torch.autograd.grad((y, c), t, (delta, delta))[0] for y, c, t in ((y1, c1, a), (y2, c2, b)))
                assert torch.equal(g1, g2)
    del big, view, bc
    rows, c = 262200, 8200
    x = torch.randn((rows, c), device="cuda", dtype=BF)
    assert x.numel() > 2 ** 31
    w = torch.rand(c, device="cuda")
    with torch.no_grad():
        y = W.rms_norm(x, w)
        assert torch.equal(y[-3:], W.rms_norm(x[-3:].clone(), w))
        q, s = W.rms_norm_q8(x, w, group=128)
        q3, s3 = W.rms_norm_q8(x[-3:].clone(), w, group=128)
        assert torch.equal(q[-3:].float(), q3.float()) and torch.equal(s[-3:], s3)
        del q, s, y
        y, _ = W.causal_conv(x.unsqueeze(0), w.unsqueeze(1).expand(c, 4).contiguous())
        tail, _ = W.causal_conv(x[-200:].unsqueeze(0), w.unsqueeze(1).expand(c, 4).contiguous())
        assert torch.equal(y[0, -150:], tail[0, -150:])


def test_inference_mode_and_many_rows():
    import rwkv_infctx_trainer_b200 as W
    p = params(BF)
    with torch.inference_mode():
        x, res, cs, st = inputs(2, 3, BF)
        y, _ = step(p, x[:, 0], res[:, 0], cs, st)
    plain = st.clone(), cs.clone()                     # (of inference tensors, outside)
    with torch.inference_mode():
        step(p, x[:, 1], res[:, 1], plain[1], plain[0])
        step(p, x[:, 1], res[:, 1], cs, st)
    assert torch.equal(plain[0], st) and torch.equal(plain[1], cs)
    # more rows than a grid has blocks across
    B, d, n = 70000, 4, 4
    c = S.scan_case(1, B, 1, d, n, 1, BF)
    state = c["state"].clone()
    one = lambda k, rows=slice(None): c[k][rows, 0]
    y = W.selective_scan_step(one("u"), one("delta"), c["A"], one("B"), one("C"), state, c["D"], one("z"), c["delta_bias"])
    few, r = c["state"][-500:].clone(), slice(-500, None)
    y2 = W.selective_scan_step(one("u", r), one("delta", r), c["A"], one("B", r), one("C", r), few, c["D"], one("z", r), c["delta_bias"])
    # (two kernels, the same formulas: another order of two sums)
    assert float((state[-500:] - few).abs().max()) <= 4 * S.U * float(few.abs().max())
    assert float((y[-500:].float() - y2.float()).abs().max()) <= 2.0 ** -7 * float(y2.float().abs().max())
    xs, w = torch.randn((B, 8), device="cuda").to(BF), torch.randn((8, 4), device="cuda")
    s0 = torch.randn((B, 3, 8), device="cuda").to(BF)
    s1 = s0[-7:].clone()
    y = W.causal_conv_step(xs, s0, w)
    assert torch.equal(y[-7:], W.causal_conv_step(xs[-7:], s1, w)) and torch.equal(s0[-7:], s1)


def _all_ops(c, x, res, w, cw, cb):
    """the three operators in training, and every gradient (twice from one graph)"""
    import rwkv_infctx_trainer_b200 as W
    scan = {n: t for n, t in c.items() if n in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state")}
    ins = [*scan.values(), x, res, w, cw, cb]
    s = list(W.selective_scan(scan["u"], scan["delta"], scan["A"], scan["B"], scan["C"], scan["D"], scan["z"], scan["delta_bias"], True, scan["state"]))
    outs = [*s, *W.causal_conv(x, cw, cb), *W.rms_norm(x, w, res)]
    grads = [torch.autograd.grad(outs, ins, [torch.ones_like(o) for o in outs], retain_graph=True) for _ in range(2)]
    for a, b in zip(*grads):
        assert torch.equal(a, b)
    return [o.detach() for o in outs] + list(grads[0])


def _layer_inputs(seed, B=3, T=37, D=24, N=16):
    g = torch.Generator("cuda").manual_seed(seed)
    def r(*s, dtype=torch.bfloat16): return torch.randn(s, device="cuda", generator=g).to(dtype)
    f = torch.float32
    scan = dict(u=r(B, T, D), delta=r(B, T, D), A=-r(D, N, dtype=f).abs(), B=r(B, T, N), C=r(B, T, N), D=r(D, dtype=f), z=r(B, T, D),
                delta_bias=r(D, dtype=f), state=r(B, D, N, dtype=f))
    return scan, r(B, T, D), r(B, T, D), r(D, dtype=f), r(D, 4, dtype=f), r(D, dtype=f)


# what of each tensor is one value for all: rows (0) or tokens (1)
@pytest.mark.parametrize("dim", [0, 1])
def test_broadcast_inputs_and_their_gradients(dim):
    """the same bits as from copies, and as gradient their sum over what was broadcast"""
    scan, x, res, w, cw, cb = _layer_inputs(dim)
    names = ("u", "delta", "B", "C", "z") if dim else ("u", "delta", "B", "C", "z", "state")
    small = {n: scan[n].narrow(dim, 0, 1).clone().requires_grad_(True) for n in names}
    small["x"], small["res"] = (t.narrow(dim, 0, 1).clone().requires_grad_(True) for t in (x, res))
    rest = [t.clone().requires_grad_(True) for t in (w, cw, cb)]
    others = {n: t.clone().requires_grad_(True) for n, t in scan.items() if n not in names}

    def run(copies):
        wide = {}
        for n, t in small.items():
            v = t.detach().expand((scan[n] if n in scan else x).shape)
            wide[n] = (v.contiguous() if copies else v).requires_grad_(True)
        return _all_ops({**{n: wide.get(n, others.get(n)) for n in scan}}, wide["x"], wide["res"], *rest)
    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)

    # through the expansion itself
    import rwkv_infctx_trainer_b200 as W
    full = {n: t.expand((scan[n] if n in scan else x).shape) for n, t in small.items()}
    y, h = W.rms_norm(full["x"], rest[0], full["res"])
    got = torch.autograd.grad((y, h), (small["x"], small["res"]), (x, res))
    leaf = [full[n].detach().contiguous().requires_grad_(True) for n in ("x", "res")]
    y, h = W.rms_norm(leaf[0], rest[0], leaf[1])
    for g, each in zip(got, torch.autograd.grad((y, h), leaf, (x, res))):
        assert torch.equal(g, each.sum(dim, keepdim=True))


def test_calls_at_once_on_two_streams():
    """each with its own workspaces: the bits of the calls made alone"""
    # (lengths that are cut into spans, so that workspaces are used forward as well)
    sets = [_layer_inputs(seed, 2, 700, 130, 16) for seed in (5, 6)]
    for scan, *others in sets:
        for t in (*scan.values(), *others):
            t.requires_grad_(True)
    alone = [_all_ops(*s) for s in sets]
    torch.cuda.synchronize()
    streams, out = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                out[i].append(_all_ops(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for got in out[i]:
            for a, b in zip(got, alone[i]):
                assert torch.equal(a, b)


def test_states_made_in_inference_mode_are_not_touched_outside():
    """torch refuses in-place changes of such tensors outside inference mode; the refusal comes before the token is taken in"""
    import rwkv_infctx_trainer_b200 as W
    p = params(BF)
    with torch.inference_mode():
        x, res, cs, st = inputs(2, 3, BF)
    c = S.scan_case(1, 2, 1, D, N, 1, BF)
    with torch.inference_mode():
        keep = cs.clone(), st.clone()
    for grad in (True, False):
        with torch.set_grad_enabled(grad):
            with pytest.raises(RuntimeError, match="[Ii]nference"):
                W.causal_conv_step(c["u"][:, 0], cs, p["conv"].detach(), p["conv_bias"].detach())
            with pytest.raises(RuntimeError, match="[Ii]nference"):
                W.selective_scan_step(c["u"][:, 0], c["delta"][:, 0], p["A"], c["B"][:, 0], c["C"][:, 0], st)
            assert torch.equal(cs, keep[0]) and torch.equal(st, keep[1])
