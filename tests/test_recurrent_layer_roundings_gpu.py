"""The recurrent layer and the channel mix against the same layers in 64 bits that are rounded where the operators round: each output, each gradient of an input, and the
gradient of a pre-activation as an operand of its products.  What is left are the operators' own errors in fp32: they make a value round the other way here and there.

A value's error before it is rounded is at most 2^-17 of its size (sums of up to 136 terms at a few roundings each, a gate's and a decay's errors).  Of values a step
eps apart (relative, between eps / 2 and eps) at most 2^-17 / (eps / 2) round the other way, by a step: a relative 2-norm of sqrt(2^-16 / eps) eps a rounding.  A term
passes 10 of them forward and 16 back, each carried on with a factor of up to 2, were all of one sign: 52 times that, 2 % in bf16 and 0.6 % in fp16."""
import pytest
import torch
import torch.nn.functional as F

import test_recurrent_layer_gpu as R

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


class Round(torch.autograd.Function):
    """forward to the type f, backward to the type b (None: as it is)"""

    @staticmethod
    def forward(ctx, x, f, b):
        ctx.b = b
        return x if f is None else x.to(f).to(x.dtype)

    @staticmethod
    def backward(ctx, g):
        return g if ctx.b is None else g.to(ctx.b).to(g.dtype), None, None


def bound(dtype, n=52):
    eps = torch.finfo(dtype).eps
    return n * (2.0 ** -16 / eps) ** 0.5 * eps


def product(x, w, dt, bias=None, act=None, mul=None, residual=None):
    """act(x w^T + bias) mul + residual as linear_act rounds it (a product without an activation and a mul takes gy as it is, in the type already)"""
    z = Round.apply(F.linear(Round.apply(x, None, dt), Round.apply(w, None, dt)), None, dt)
    z = z if bias is None else z + bias
    y = z if act is None else act(z)
    y = y if mul is None else y * Round.apply(mul, None, dt)
    y = y if residual is None else y + residual
    return Round.apply(y, dt, None)


def pair(x, wg, wu, dt, act):
    x = Round.apply(x, None, dt)
    g, u = (Round.apply(F.linear(x, Round.apply(w, None, dt)), None, dt) for w in (wg, wu))
    return Round.apply(act(g) * u, dt, None)


def norm(x, w, dt):
    x = Round.apply(x, None, dt)
    return Round.apply(x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w, dt, None)


def layer(p, x, conv_state, state, dt):
    y = norm(x, p["norm1"], dt)
    u, z = product(y, p["w_in"], dt), product(y, p["w_z"], dt, p["b_z"])
    xs = torch.cat((Round.apply(conv_state, None, dt), Round.apply(u, None, dt)), 1)
    u = Round.apply(F.silu(sum(xs[:, j:j + x.shape[1]] * p["conv"][:, j] for j in range(R.W4)) + p["conv_bias"]), dt, None)
    ig, rg = product(u, p["w_gates"], dt, p["b_gates"]).chunk(2, -1)
    ur, ig, rg, z = (Round.apply(t, None, dt) for t in (u, ig, rg, z))
    a = torch.exp(-8.0 * F.softplus(p["decay"]) * torch.sigmoid(rg))
    b = torch.sqrt(1 - a * a) * torch.sigmoid(ig) * ur
    ys = []
    for t in range(x.shape[1]):
        state = a[:, t] * state + b[:, t]
        ys.append(state)
    x = product(Round.apply(torch.stack(ys, 1) * F.silu(z), dt, None), p["w_out"], dt, residual=x)
    h = pair(norm(x, p["norm2"], dt), p["w_gate"], p["w_up"], dt, F.gelu)
    return product(h, p["w_down"], dt, residual=x), xs[:, x.shape[1]:], state


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,T", [(2, 24), (3, 150)])
def test_layer_and_its_gradients(B, T, dtype):
    p = R.params(dtype)
    x, cs, st = R.inputs(B, T, dtype)
    leaves = {k: v.detach().requires_grad_(True) for k, v in {**p, "x": x, "cs": cs, "st": st}.items()}
    out = R.layer(leaves, leaves["x"], leaves["cs"], leaves["st"])
    d = {k: v.detach().double().requires_grad_(True) for k, v in leaves.items()}
    want = layer(d, d["x"], d["cs"], d["st"], dtype)
    seeds = [torch.randn_like(o) for o in out]
    got_g = torch.autograd.grad(out, list(leaves.values()), seeds)
    want_g = torch.autograd.grad(want, list(d.values()), [t.double() for t in seeds])
    # (a gradient in the type is rounded once more than the reference's: half a step)
    for n, a, b in [*zip(("y", "conv_state", "state"), out, want), *zip(leaves, got_g, want_g)]:
        e = R.rel(a.detach(), b.detach())
        assert e <= bound(dtype) + torch.finfo(dtype).eps / 2, (n, e)


@pytest.mark.parametrize("B", [1, 3, 20])
def test_decoded_tokens(B):
    """a prompt and tokens after it: ten roundings, no gradient"""
    p = R.params(BF)
    x, cs, st = R.inputs(B, 30, BF)
    with torch.no_grad():
        want = layer({k: v.double() for k, v in p.items()}, x.double(), cs.double(), st.double(), BF)
        y, c, s = R.layer(p, x[:, :22], cs, st)
        ys = [y]
        for t in range(22, 30):
            y, c, s = R.layer(p, x[:, t], c, s, one=True)
            ys.append(y.unsqueeze(1))
    for n, a, b in zip(("y", "conv_state", "state"), (torch.cat(ys, 1), c, s), want):
        assert R.rel(a, b) <= bound(BF, 20), (n, R.rel(a, b))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_channel_mix(dtype):
    """three roundings forward and nine back"""
    import rwkv_infctx_trainer_b200 as W
    g = torch.Generator().manual_seed(3)
    n = lambda *s, std=1.0: (torch.randn(s, generator=g) * std).to(dtype).cuda().requires_grad_(True)
    ins = [n(2, 70, R.C), n(2, 70, R.C), n(R.FF, R.C, std=R.C ** -0.5), n(R.C, R.FF, std=R.FF ** -0.5), n(R.C, R.C, std=R.C ** -0.5)]
    xk, xr, wk, wv, wr = ins
    y = W.linear_act(xr, wr, activation="sigmoid", mul=W.linear_act(W.linear_act(xk, wk, activation="relu2"), wv))
    d = [t.detach().double().requires_grad_(True) for t in ins]
    kv = product(product(d[0], d[2], dtype, act=lambda z: F.relu(z).square()), d[3], dtype)
    want = product(d[1], d[4], dtype, act=torch.sigmoid, mul=kv)
    gy = torch.randn_like(y)
    limit = bound(dtype, 24) + torch.finfo(dtype).eps / 2
    assert R.rel(y.detach(), want.detach()) <= limit
    for a, b in zip(torch.autograd.grad(y, ins, gy), torch.autograd.grad(want, d, gy.double())):
        assert R.rel(a, b) <= limit
