"""The operators of a recurrent layer together, as a layer and its feed-forward block use them -- norm, projections, convolution, gated
recurrence, projection with the residual, norm, gated pair, projection with the residual; the channel mix of the WKV models -- and what a
program does around them: segments, prompts and decoded tokens, graphs, threads, waits that run out, derivatives that do not exist."""
import ctypes
import threading

import pytest
import torch
import torch.autograd.forward_ad as fwAD
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
C, D, FF, W4 = 48, 96, 136, 4


def params(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, std=1.0: (torch.randn(s, generator=g) * std)
    p = {"norm1": 1 + 0.1 * n(C), "w_in": n(D, C, std=C ** -0.5), "w_z": n(D, C, std=C ** -0.5), "b_z": 0.1 * n(D), "conv": n(D, W4, std=0.5),
         "conv_bias": 0.1 * n(D), "w_gates": n(2 * D, D, std=D ** -0.5), "b_gates": 0.5 * n(2 * D), "decay": n(D) - 3, "w_out": n(C, D, std=D ** -0.5),
         "norm2": 1 + 0.1 * n(C), "w_gate": n(FF, C, std=C ** -0.5), "w_up": n(FF, C, std=C ** -0.5), "w_down": n(C, FF, std=FF ** -0.5)}
    return {k: v.to(dtype if k.startswith("w_") else F32).cuda() for k, v in p.items()}


def layer(p, x, conv_state, state, one=False):
    import rwkv_infctx_trainer_b200 as W
    y = W.rms_norm(x, p["norm1"])
    u = W.linear_act(y, p["w_in"])
    z = W.linear_act(y, p["w_z"], p["b_z"])
    if one:
        u = W.causal_conv_step(u, conv_state, p["conv"], p["conv_bias"])
    else:
        u, conv_state = W.causal_conv(u, p["conv"], p["conv_bias"], conv_state)
    ig, rg = W.linear_act(u, p["w_gates"], p["b_gates"]).chunk(2, -1)
    if one:
        y = W.gated_recurrence_step(u, ig, rg, p["decay"], state, z)
    else:
        y, state = W.gated_recurrence(u, ig, rg, p["decay"], z, state)
    x = W.linear_act(y, p["w_out"], residual=x)
    h = W.gated_linear(W.rms_norm(x, p["norm2"]), p["w_gate"], p["w_up"], "gelu")
    return W.linear_act(h, p["w_down"], residual=x), conv_state, state


def layer64(p, x, conv_state, state):
    norm = lambda t, w: t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w
    y = norm(x, p["norm1"])
    u, z = F.linear(y, p["w_in"]), F.linear(y, p["w_z"], p["b_z"])
    xs = torch.cat((conv_state, u), 1)
    u = F.silu(sum(xs[:, j:j + x.shape[1]] * p["conv"][:, j] for j in range(W4)) + p["conv_bias"])
    ig, rg = F.linear(u, p["w_gates"], p["b_gates"]).chunk(2, -1)
    a = torch.exp(-8.0 * F.softplus(p["decay"]) * torch.sigmoid(rg))
    b = torch.sqrt(1 - a * a) * torch.sigmoid(ig) * u
    ys = []
    for t in range(x.shape[1]):
        state = a[:, t] * state + b[:, t]
        ys.append(state)
    x = x + F.linear(torch.stack(ys, 1) * F.silu(z), p["w_out"])
    y = norm(x, p["norm2"])
    return x + F.linear(F.gelu(F.linear(y, p["w_gate"])) * F.linear(y, p["w_up"]), p["w_down"]), xs[:, x.shape[1]:], state


def inputs(B, T, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)
    return n(B, T, C).to(dtype).cuda(), n(B, W4 - 1, D).to(dtype).cuda(), n(B, D).cuda()


def rel(a, b):
    return float((a.double() - b).norm() / b.norm())


# A term passes 10 roundings to the type on its way forward (the outputs of ten operators) and 16 on the way back (their gradients, the kept
# pre-activations and the gradients of those), each of at most half a step of a value.  Their relative 2-norm is at most that half step, and is
# carried on with factors (the projections' norms of about 2, the norms' division by the root mean square) that are 1 in the mean of a
# random projection and are taken as 2: 26 * 2 half steps, were all of one sign.
ROUNDINGS = 26 * 2


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,T,cuts", [(2, 24, [0, 24]), (2, 24, [0, 9, 10, 24]), (1, 5, [0, 5]), (3, 150, [0, 64, 150])])
def test_layer_and_its_gradients(B, T, cuts, dtype):
    """against the layer in 64 bits, in one call and in segments with both states and their gradients carried"""
    p = params(dtype)
    x, cs, st = inputs(B, T, dtype)
    leaves = {k: v.detach().requires_grad_(True) for k, v in {**p, "x": x, "cs": cs, "st": st}.items()}
    c, s, ys = leaves["cs"], leaves["st"], []
    for a, b in zip(cuts, cuts[1:]):
        y, c, s = layer(leaves, leaves["x"][:, a:b], c, s)
        ys.append(y)
    out = [torch.cat(ys, 1), c, s]
    d = {k: v.detach().double().requires_grad_(True) for k, v in leaves.items()}
    want = layer64(d, d["x"], d["cs"], d["st"])
    seeds = [torch.randn_like(o) for o in out]
    got_g = torch.autograd.grad(out, list(leaves.values()), seeds)
    want_g = torch.autograd.grad(want, list(d.values()), [t.double() for t in seeds])
    bound = ROUNDINGS * torch.finfo(dtype).eps / 2
    for n, a, b in [*zip(("y", "conv_state", "state"), out, want), *zip(leaves, got_g, want_g)]:
        assert rel(a.detach(), b.detach()) <= bound, (n, rel(a.detach(), b.detach()))


@pytest.mark.parametrize("B", [1, 3, 20])
def test_decoded_tokens_follow_a_prompt(B):
    """token by token against the whole row: the same operations on the same values, whose sums are added up in another order for few rows.
    Outputs differ where a rounding falls the other way, by steps of bf16, on the way of a term at most ten"""
    p = params(BF)
    x, cs, st = inputs(B, 30, BF)
    with torch.no_grad():
        want, wc, ws = layer(p, x, cs, st)
        y, c, s = layer(p, x[:, :22], cs, st)
        ys = [y]
        for t in range(22, 30):
            y, c, s = layer(p, x[:, t], c, s, one=True)
            ys.append(y.unsqueeze(1))
        got = torch.cat(ys, 1)
    for a, b in ((got, want), (c, wc), (s, ws)):
        assert rel(a, b.double()) <= 10 * torch.finfo(BF).eps


@pytest.mark.parametrize("dtype", [BF, HF])
def test_channel_mix(dtype):
    """sigmoid(xr Wr^T) * (relu(xk Wk^T)^2 Wv^T) and its gradients: 3 roundings forward and 9 back on a term's way"""
    import rwkv_infctx_trainer_b200 as W
    g = torch.Generator().manual_seed(3)
    n = lambda *s, std=1.0: (torch.randn(s, generator=g) * std).to(dtype).cuda().requires_grad_(True)
    ins = [n(2, 70, C), n(2, 70, C), n(FF, C, std=C ** -0.5), n(C, FF, std=FF ** -0.5), n(C, C, std=C ** -0.5)]

    def mix(xk, xr, wk, wv, wr):
        kv = W.linear_act(W.linear_act(xk, wk, activation="relu2"), wv)
        return W.linear_act(xr, wr, activation="sigmoid", mul=kv)
    y = mix(*ins)
    d = [t.detach().double().requires_grad_(True) for t in ins]
    want = torch.sigmoid(F.linear(d[1], d[4])) * F.linear(F.relu(F.linear(d[0], d[2])).square(), d[3])
    gy = torch.randn_like(y)
    bound = 12 * 2 * torch.finfo(dtype).eps / 2
    assert rel(y.detach(), want.detach()) <= bound
    for a, b in zip(torch.autograd.grad(y, ins, gy), torch.autograd.grad(want, d, gy.double())):
        assert rel(a, b) <= bound


def test_a_decode_step_and_a_training_step_in_a_graph():
    """captured, replayed with other inputs in place; a backward pass is captured with leaves of its own"""
    p = params(BF)
    x, cs, st = inputs(4, 40, BF)
    with torch.no_grad():
        one = [x[:, 0].clone(), cs.clone(), st.clone()]
        layer(p, *[t.clone() for t in one], one=True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, _, _ = layer(p, *one, one=True)
        one[1].copy_(cs)
        one[2].copy_(st)
        c, s = cs.clone(), st.clone()
        for t in range(5):
            one[0].copy_(x[:, t])
            graph.replay()
            w, c, s = layer(p, x[:, t], c, s, one=True)
            assert torch.equal(y, w) and torch.equal(one[1], c) and torch.equal(one[2], s)

    def training(p, x, cs, st):
        leaves = {k: v.detach().requires_grad_(True) for k, v in {**p, "x": x, "cs": cs, "st": st}.items()}
        out = layer(leaves, leaves["x"], leaves["cs"], leaves["st"])
        return torch.autograd.grad([o.float().square().sum() for o in out], list(leaves.values()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    static = [t.clone() for t in (x, cs, st)]
    with torch.cuda.stream(side):
        training(p, *static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = training(p, *static)
    for seed in (5, 6):
        new = inputs(4, 40, BF, seed)
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        for a, b in zip(got, training(p, *new)):
            assert torch.equal(a, b)


def test_the_first_call_of_a_process_inside_a_capture():
    import os
    import subprocess
    import sys
    code = """
import torch, rwkv_infctx_trainer_b200 as W
n = lambda *s: torch.randn(s, device="cuda", dtype=torch.bfloat16)
x, w, z = n(40, 64), n(72, 64), n(1, 40, 64)
decay = torch.zeros(64, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.no_grad(), torch.cuda.graph(g):
    y = W.linear_act(x, w, activation="gelu")
    r, s = W.gated_recurrence(z, z, z, decay)
g.replay()
torch.cuda.synchronize()
with torch.no_grad():
    assert torch.equal(y, W.linear_act(x, w, activation="gelu")) and torch.equal(r, W.gated_recurrence(z, z, z, decay)[0])
print("same")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "same" in out.stdout, out.stderr[-2000:]


def test_threads():
    p = params(BF)
    rows = [inputs(2, 33, BF, seed) for seed in range(4)]
    run = lambda t: layer(p, *t)[0]
    with torch.no_grad():
        want = [run(t) for t in rows]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.no_grad(), torch.cuda.stream(stream):
            for _ in range(10):
                y = run(rows[i])
                stream.synchronize()
                if not torch.equal(y, want[i]):
                    bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def calls():
    """name -> (call, inputs that are all differentiable)"""
    import rwkv_infctx_trainer_b200 as W
    g = torch.Generator().manual_seed(9)
    n = lambda *s, dtype=BF: torch.randn(s, generator=g).to(dtype).cuda()
    r = lambda: n(2, 20, C)
    return {"gated_recurrence": (lambda x, i, d, p, z, s: W.gated_recurrence(x, i, d, p, z, s), [r(), r(), r(), n(C, dtype=F32), r(), n(2, C, dtype=F32)]),
            "linear_act": (lambda x, w, b, m, q: (W.linear_act(x, w, b, "silu", m, q),), [r(), n(24, C), n(24), n(2, 20, 24), n(2, 20, 24)]),
            "gated_linear": (lambda x, a, b: (W.gated_linear(x, a, b),), [r(), n(24, C), n(24, C)])}


@pytest.mark.parametrize("name", ["gated_recurrence", "linear_act", "gated_linear"])
def test_derivatives_that_do_not_exist_are_refused(name):
    call, ins = calls()[name]
    leaves = [t.requires_grad_(True) for t in ins]
    out = list(call(*leaves))
    seeds = [torch.randn_like(o) for o in out]
    want = torch.autograd.grad(out, leaves, seeds, retain_graph=True)
    got = torch.autograd.grad(out, leaves, seeds, create_graph=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b) and a.requires_grad
    for a in got:
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(a.float().square().sum() + leaves[0].float().sum(), leaves[0], retain_graph=True)
    for grad in (True, False):
        for i, t in enumerate(ins):
            with torch.set_grad_enabled(grad), fwAD.dual_level():
                duals = [x.detach().clone() for x in ins]
                duals[i] = fwAD.make_dual(duals[i], torch.ones_like(t))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*duals)


@pytest.mark.parametrize("name", ["gated_recurrence", "linear_act", "gated_linear"])
def test_inputs_changed_before_the_backward_pass_are_noticed(name):
    call, ins = calls()[name]
    leaves = [t.requires_grad_(True) for t in ins]
    out = list(call(*leaves))
    with torch.no_grad():
        leaves[0].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaves, [torch.randn_like(o) for o in out])


def test_inference_mode():
    import rwkv_infctx_trainer_b200 as W
    p = params(BF)
    x, cs, st = inputs(2, 12, BF)
    with torch.no_grad():
        want = layer(p, x, cs, st)
    with torch.inference_mode():
        got = layer(p, x, cs, st)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        _, c, s = got
        layer(p, x[:, 0], c, s, one=True)
    before = s.clone()
    with torch.no_grad(), pytest.raises(RuntimeError, match="inference"):
        W.gated_recurrence_step(*(torch.randn(2, D, device="cuda", dtype=BF) for _ in range(3)), p["decay"], s)
    assert torch.equal(s, before)


def aligned(n):
    return torch.empty(max(int(n), 256), dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("skip", [0, 1, 3])
@pytest.mark.parametrize("rows,K,N,pair", [(256, 512, 512, 0), (600, 520, 1000, 0), (200, 300 * 8, 200, 0), (300, 256, 136, 1)])
def test_waits_of_a_product_run_out(rows, K, N, pair, skip, backward):
    """a block of every CTA's first tile that is never loaded: the call ends, says so, and the next one is as ever"""
    import rwkv_infctx_trainer_b200 as W
    from rwkv_infctx_trainer_b200 import _lib as L
    lib = L.load()
    n = lambda *s: torch.randn(s, device="cuda", dtype=BF)
    x, w0, w1, gy = n(rows, K), n(N, K), n(N, K), n(rows, N)
    y, gx, g0, g1, status = torch.empty_like(gy), torch.empty_like(x), torch.empty_like(w0), torch.empty_like(w1), torch.zeros(1, dtype=torch.int32, device="cuda")
    a = L.LinearArgs(rows=rows, K=K, N=N, dtype=1, act=1, pair=pair, x=x.data_ptr(), w0=w0.data_ptr(), w1=w1.data_ptr() if pair else None, x_row=K, w0_row=K, w1_row=K,
                     y=y.data_ptr(), status=status.data_ptr())
    a.saved_bytes = lib.wkv_linear_saved_bytes(ctypes.byref(a))
    saved = torch.zeros(max(a.saved_bytes, 256), dtype=torch.uint8, device="cuda")
    a.saved = saved.data_ptr()
    if backward:
        a.gy, a.gx, a.gw0, a.gw1 = gy.data_ptr(), gx.data_ptr(), g0.data_ptr(), g1.data_ptr() if pair else None
    size = lib.wkv_linear_backward_workspace if backward else lib.wkv_linear_forward_workspace
    a.workspace_bytes = size(ctypes.byref(a))
    ws = aligned(a.workspace_bytes)
    a.workspace = ws.data_ptr()
    assert lib.wkv_linear_selftest_abort(ctypes.byref(a), backward, skip, 500, L.stream_handle(0)) == 0
    torch.cuda.synchronize()
    assert int(status) == 64
    status.zero_()
    run = lib.wkv_linear_backward if backward else lib.wkv_linear_forward
    assert run(ctypes.byref(a), L.stream_handle(0)) == 0
    torch.cuda.synchronize()
    assert int(status) == 0
    if not backward:
        assert torch.equal(y, W.gated_linear(x, w0, w1) if pair else W.linear_act(x, w0, activation="silu"))


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("skip", [0, 1])
@pytest.mark.parametrize("B,T,channels", [(1, 400, 64), (2, 100, 200), (8, 130, 2048)])
def test_waits_of_a_recurrence_run_out(B, T, channels, skip, backward):
    import rwkv_infctx_trainer_b200 as W
    from rwkv_infctx_trainer_b200 import _lib as L
    lib = L.load()
    n = lambda *s, dtype=BF: torch.randn(s, device="cuda", dtype=dtype)
    x, ig, rg, z, gy = (n(B, T, channels) for _ in range(5))
    decay, st = n(channels, dtype=F32), n(B, channels, dtype=F32)
    outs = [torch.empty_like(x) for _ in range(5)]
    so, gd, status = torch.empty_like(st), torch.empty_like(decay), torch.zeros(1, dtype=torch.int32, device="cuda")
    a = L.GatedRecurrenceArgs(B=B, T=T, D=channels, dtype=1, c=8.0, x=x.data_ptr(), input_gate=ig.data_ptr(), decay_gate=rg.data_ptr(), z=z.data_ptr(),
                              decay=decay.data_ptr(), state_in=st.data_ptr(), y=outs[0].data_ptr(), state_out=so.data_ptr(), status=status.data_ptr())
    for k in "xirz":
        setattr(a, k + "_batch", T * channels)
        setattr(a, k + "_token", channels)
    a.ckpt_bytes = lib.wkv_gated_recurrence_ckpt_bytes(ctypes.byref(a))
    ckpt = torch.zeros(a.ckpt_bytes, dtype=torch.uint8, device="cuda")
    a.ckpt = ckpt.data_ptr()
    if backward:
        a.gy, a.gx, a.ginput_gate, a.gdecay_gate, a.gz, a.gdecay = (t.data_ptr() for t in (gy, *outs[1:], gd))
    size = lib.wkv_gated_recurrence_backward_workspace if backward else lib.wkv_gated_recurrence_forward_workspace
    a.workspace_bytes = size(ctypes.byref(a))
    ws = aligned(a.workspace_bytes)
    a.workspace = ws.data_ptr()
    assert lib.wkv_gated_recurrence_selftest_abort(ctypes.byref(a), backward, skip, 500, L.stream_handle(0)) == 0
    torch.cuda.synchronize()
    assert int(status) == 128
    status.zero_()
    run = lib.wkv_gated_recurrence_backward if backward else lib.wkv_gated_recurrence_forward
    assert run(ctypes.byref(a), L.stream_handle(0)) == 0
    torch.cuda.synchronize()
    assert int(status) == 0
    if not backward:
        y, s = W.gated_recurrence(x, ig, rg, decay, z, st)
        assert torch.equal(y, outs[0]) and torch.equal(s, so)


def test_a_wait_that_ran_out_is_reported_by_the_next_call():
    """the kernels write one word per device in mapped host memory; this test writes it in their place"""
    import rwkv_infctx_trainer_b200 as W
    from rwkv_infctx_trainer_b200 import _lib as L
    call, ins = calls()["linear_act"]
    rec, rins = calls()["gated_recurrence"]
    call(*ins), rec(*rins)
    torch.cuda.synchronize()
    word = ctypes.c_int.from_address(L.native().status_word(0))
    for bit, look in ((64, lambda: call(*ins)), (128, lambda: rec(*rins)), (64, lambda: W.gated_linear(ins[0], ins[1], ins[1]))):
        word.value = bit
        with pytest.raises(RuntimeError, match=rf"device-side wait ran out \(status {bit}\)"):
            look()
        assert word.value == 0
        look()
