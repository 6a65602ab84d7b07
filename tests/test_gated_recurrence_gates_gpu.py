"""The gradients of the gated recurrence where a gate is wide open or almost closed: sigmoids there are near 1 or near 0, and what is left of them
has digits of its own.  Against the formulas in 64 bits; inputs whose terms are all of one sign (but for the decay gate's two), so that errors
are relative.

In units of 2^-24 (U): a sigmoid of x and its complement, sigmoid(-x), are off by 4|x| + 16 relative to themselves (an exponential by 2|x| + 4, the
sum and the quotient by 4, their product by 1), a decay a = e^L by |L| times the error of L, and 5, the root m of 1 - a^2 by half of the error of
1 - a^2: its series by 8 and by the error of L, above it 7 decays' and 5.  G adds one decay and 3 a token, and 40 for what regrouping tokens
into segments changes.  What a normal fp32 number cannot hold is flushed to zero: a sigmoid r below 2^-126 makes 1 - a^2 too small by up to 2 c
softplus(p) 2^-126, one of 1 - a^2 below it by up to 2^-126, and m by no more than the root of that (`lost`); i x a^2 L / m is then i x m / 2, and half as
much is missing of it; a flushed L is missing in h a L."""
import pytest
import torch

from test_gated_recurrence_gpu import close

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
C = 8.0


def ds(t):
    return (4 * t.abs() + 16) * U


def gradients(x, ig, rg, p, h0, gy, z=None):
    import rwkv_infctx_trainer_b200 as W
    leaves = [t.detach().requires_grad_(True) for t in (x, ig, rg, p, h0) + (() if z is None else (z,))]
    y, s = W.gated_recurrence(*leaves[:4], leaves[5] if z is not None else None, leaves[4], C)
    g = torch.autograd.grad((y, s), leaves, (gy, torch.zeros_like(s)))
    return {"y": y, **dict(zip(("gx", "ginput", "gdecay_gate", "gdecay", "gstate", "gz"), g))}


def ref(x, ig, rg, p, h0, gy):
    """name -> (value, bound of the error before the last rounding), without an output gate; x, h0 and gy are positive"""
    x, ig, rg, p, h0, gy = (t.double() for t in (x, ig, rg, p, h0, gy))
    T = x.shape[1]
    r, i = torch.sigmoid(rg), torch.sigmoid(ig)
    L = -C * torch.nn.functional.softplus(p) * r
    a, q = torch.exp(L), -torch.expm1(2 * L)
    m = torch.sqrt(q)
    dL = ds(rg) + (13 + 2.4 * p.abs()) * U
    da = L.abs() * dL + 5 * U
    dm = 0.5 * (dL + 8 * U) + 3.5 * da + 7 * U
    sp = torch.nn.functional.softplus(p)
    lost = torch.where((r < 2.0 ** -126) | (q < 2.0 ** -126), (2 * C * sp).clamp_min(1.0).sqrt() * 2.0 ** -63, 0.0)
    hs, h = [h0], h0
    for t in range(T):
        h = a[:, t] * h + m[:, t] * i[:, t] * x[:, t]
        hs.append(h)
    h = torch.stack(hs, 1)
    G, E = [], torch.zeros_like(h0)
    for t in range(T - 1, -1, -1):
        G.append(gy[:, t] + E)
        E = a[:, t] * G[-1]
    G = torch.stack(G[::-1], 1)
    dG = T * (float(da.max()) + 3 * U) + 40 * U
    dh = T * (da + dm + ds(ig) + 6 * U).amax(1, keepdim=True) + 40 * U
    gx = G * m * i
    dgx = dG + dm + ds(ig) + 4 * U
    gi = gx * x * torch.sigmoid(-ig)
    t1, t2 = h[:, :-1] * a * L, -i * x * a * a * torch.where(q > 0, L / torch.where(q > 0, m, 1.0), 0.0)
    gLL = G * (t1 + t2)
    egLL = G * (t1.abs() * (dG + dh + da + dL + 4 * U) + t2.abs() * (dG + 2 * da + dL + dm + ds(ig) + 10 * U)) + G * (t1.abs() + t2.abs()) * U
    gr = torch.sigmoid(-rg)
    egLL = egLL + G * i * x * lost / 2 + G * h[:, :-1] * (C * sp).clamp_min(1.0) * 2.0 ** -126 * (lost > 0)
    return {"gx": (gx, gx * dgx + G * i * lost), "ginput": (gi, gi * (dgx + ds(ig) + 2 * U) + G * i * x * torch.sigmoid(-ig) * lost),
            "gdecay_gate": (gLL * gr, gr * (egLL + gLL.abs() * (ds(rg) + 2 * U)))}


def inputs(seed, T, D, dtype, low=-1.0, high=1.0):
    g = torch.Generator().manual_seed(seed)
    u = lambda *s: torch.rand(s, generator=g)
    return {"x": (u(2, T, D) + 0.5).to(dtype).cuda(), "ig": (4 * u(2, T, D) - 2).to(dtype).cuda(), "rg": (4 * u(2, T, D) - 2).to(dtype).cuda(),
            "p": (u(D) * (high - low) + low).cuda(), "h0": (u(2, D) + 0.5).cuda(), "gy": (u(2, T, D) + 0.5).to(dtype).cuda()}


@pytest.mark.parametrize("gate", ["ig", "rg"])
@pytest.mark.parametrize("T,D", [(1, 72), (9, 72), (9, 70), (9, 71), (70, 64)])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_open_and_closed_gates(gate, T, D, dtype):
    c = inputs(T + D, T, D, dtype, -9.0, -3.0)
    # (a sigmoid's gate, from -25 to 25 along the channels)
    c[gate] = torch.linspace(-25, 25, D).expand(2, T, D).to(dtype).cuda().contiguous()
    got, want = gradients(**c), ref(**c)
    for n in want:
        close(n, got[n], *want[n])


@pytest.mark.parametrize("value", [-200.0, -95.0, -60.0, 60.0, 95.0, 200.0])
@pytest.mark.parametrize("gate", ["ig", "rg"])
def test_gates_far_out(gate, value):
    c = inputs(1, 9, 72, F32, -9.0, -3.0)
    c[gate] = torch.full_like(c[gate], value)
    got, want = gradients(**c), ref(**c)
    for n in want:
        close(n, got[n], *want[n])


@pytest.mark.parametrize("D", [72, 71])
def test_decays_next_to_one(D):
    """1 - a^2 from the smallest normal number on: its root is that of the forward pass"""
    c = inputs(2, 1, D, F32)
    c["p"] = torch.full_like(c["p"], -5.07)                       # 2 c softplus(p) = 0.1
    c["rg"] = torch.linspace(-84.8, -80.0, D).expand(2, 1, D).contiguous().cuda()
    q = -torch.expm1(-2 * C * torch.nn.functional.softplus(c["p"].double()) * torch.sigmoid(c["rg"].double()))
    assert 2.0 ** -126 * (1 + 400 * U) < float(q.min()) < 2e-38
    got, want = gradients(**c), ref(**c)
    for n in want:
        close(n, got[n], *want[n])


@pytest.mark.parametrize("D", [68, 69])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_output_gates_far_out(D, dtype):
    """the gradient of z, gy h s (1 + z (1 - s)): off by the errors of h, of s and of 1 - s, the latter where z carries them"""
    c = inputs(3, 9, D, dtype)
    z = [-3e38, -100.0, -30.0, -5.0, -1.5, 0.0, 0.5, 3.0, 8.0, 12.0, 20.0, 50.0, 90.0, 1e3, 1e4, 1e6, 1e20, 3e38]
    z = torch.tensor((z * 4)[:D]).expand(2, 9, D).contiguous().to(dtype).cuda()
    got = gradients(**c, z=z)["gz"]
    x, ig, rg, p, h, gy, z = (t.double() for t in (c["x"], c["ig"], c["rg"], c["p"], c["h0"], c["gy"], z))
    L = -C * torch.nn.functional.softplus(p) * torch.sigmoid(rg)
    a, m = torch.exp(L), torch.sqrt(-torch.expm1(2 * L))
    da = L.abs() * (ds(rg) + (13 + 2.4 * p.abs()) * U) + 5 * U
    hs = []
    for t in range(9):
        h = a[:, t] * h + m[:, t] * torch.sigmoid(ig[:, t]) * x[:, t]
        hs.append(h)
    h = torch.stack(hs, 1)
    dh = 9 * (da + 0.5 * ds(rg) + 3.5 * da + ds(ig) + (0.5 * (21 + 2.4 * p.abs()) + 13) * U).amax(1, keepdim=True) + 40 * U
    s, rest = torch.sigmoid(z), torch.sigmoid(-z)
    want = gy * h * s * (1 + z * rest)
    err = gy * h * s * (1 + z.abs() * rest) * (dh + 2 * ds(z).clamp_max(1.0) + 4 * U)
    close("gz", got, want, err)
