"""The matrix products with their epilogue in 64 bits, written from their formulas, with a bound of the kernel's error beside each value.

In units of 2^-24 (U, half a step of fp32).  A sum of K products in fp32 is off by K + 4 additions, each at most 2 U (the tensor
core cuts off where it does not round) of the terms' absolute values.  A sigmoid of z is off by 2|z| + 16 relative to itself (the
exponent's product 2|z|, the exponential, the sum, the quotient and the products behind it 16), Phi(z) through erfc by z^2 + 2|z| + 24
(erfc 8 steps and its argument's rounding, which its slope carries z^2 times).  An error of z moves an activation by at most its largest
slope (1.13 for gelu, 1.1 for silu, 1/4 for the sigmoid, 2|z| for the squared ReLU), its derivative by at most its largest curvature
(0.8, 0.5, 0.1 and 2).  The pre-activation is kept in fp32; the gradient of it that the products take and every output are rounded to
the type: half a step of it, and half the smallest subnormal."""
import math

import torch
import torch.nn.functional as F

U = 2.0 ** -24
ACTS = ["none", "silu", "gelu", "relu2", "sigmoid"]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def act(name, z):
    """value, derivative"""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu2":
        return F.relu(z).square(), 2 * F.relu(z)
    if name == "gelu":
        phi = 0.5 * torch.erfc(-z * math.sqrt(0.5))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(z)
    return (s, s * (1 - s)) if name == "sigmoid" else (z * s, s * (1 + z * (1 - s)))


def slopes(name, z, e):
    """largest slope and curvature near z, and the relative error of the function"""
    rel = {"none": 0 * z, "relu2": 4 + 0 * z, "gelu": z * z + 2 * z.abs() + 24}.get(name, 2 * z.abs() + 16) * U
    s1 = {"none": 1.0, "silu": 1.1, "gelu": 1.13, "sigmoid": 0.25}.get(name, 2 * (z.abs() + e))
    s2 = {"none": 0.0, "silu": 0.5, "gelu": 0.8, "sigmoid": 0.1, "relu2": 2.0}[name]
    return s1, s2, rel


def dot(a, b, ea=None):
    """a b^T, and its error: of the sums, and of a where `ea` bounds it"""
    mag = a.abs() @ b.abs().t()
    e = (a.shape[1] + 4) * 2 * U * mag
    return a @ b.t(), e if ea is None else e + ea @ b.abs().t()


def values(name, z, ez):
    v, _ = act(name, z)
    s1, _, rel = slopes(name, z, ez)
    return v, s1 * ez + rel * v.abs()


def linear_ref(x, w, bias, name, mul, res, gy=None):
    """name -> (value, bound of the error before its rounding); x, mul, res, gy of two dimensions"""
    dt, h = x.dtype, half(x.dtype)
    d = lambda t: None if t is None else t.detach().double()
    x, w, bias, mul, res, gy = (d(t) for t in (x, w, bias, mul, res, gy))
    z, ez = dot(x, w)
    if bias is not None:
        z, ez = z + bias, ez + 2 * U * (z.abs() + bias.abs())
    a, ea = values(name, z, ez)
    m = 1.0 if mul is None else mul
    y, ey = a * m, ea * abs(m) + 2 * U * (a * m).abs()
    if res is not None:
        y, ey = y + res, ey + 2 * U * (y.abs() + res.abs())
    out = {"y": (y, ey)}
    if gy is None:
        return out
    kept = name != "none" or mul is not None
    dz = ez if kept else 0 * z
    _, da = act(name, z)
    _, s2, rel = slopes(name, z, dz)
    gz = gy * m * da
    # (the derivative is a sum of terms of up to 1 + |z|, each off as the function is)
    egz = (gy * m).abs() * (s2 * dz + (rel + 4 * U) * (1 + z.abs()) * (0 if name == "none" else 1)) + 2 * U * gz.abs()
    rounded = egz + (h * (gz.abs() + egz) + least(dt) if kept else 0)
    out["gx"] = dot(gz, w.t(), rounded)
    out["gweight"] = dot(gz.t(), x.t(), rounded.t())
    out["gbias"] = (gz.sum(0), egz.sum(0) + (len(gz) + 4) * U * gz.abs().sum(0))
    a2, e2 = values(name, z, dz)
    out["gmul"] = (gy * a2, gy.abs() * e2 + 2 * U * (gy * a2).abs())
    return out


def gated_ref(x, wg, wu, name, gy=None):
    dt, h = x.dtype, half(x.dtype)
    x, wg, wu = (t.detach().double() for t in (x, wg, wu))
    gy = None if gy is None else gy.detach().double()
    (g, eg), (u, eu) = dot(x, wg), dot(x, wu)
    a, ea = values(name, g, eg)
    out = {"y": (a * u, ea * (u.abs() + eu) + a.abs() * eu + 2 * U * (a * u).abs())}
    if gy is None:
        return out
    dg, du = eg, eu
    a, ea = values(name, g, dg)
    _, da = act(name, g)
    _, s2, rel = slopes(name, g, dg)
    eda = s2 * dg + (rel + 4 * U) * (1 + g.abs()) * (0 if name == "none" else 1)
    gu, egu = gy * a, gy.abs() * ea + 2 * U * (gy * a).abs()
    gg = gy * u * da
    egg = gy.abs() * (eda * (u.abs() + du) + da.abs() * du) + 4 * U * gg.abs()
    rg, ru = egg + h * (gg.abs() + egg) + least(dt), egu + h * (gu.abs() + egu) + least(dt)
    p, q = dot(gg, wg.t(), rg), dot(gu, wu.t(), ru)
    # (one sum over both: the additions of each also act on the other's terms)
    both = 2 * U * ((gg.shape[1] + 4) * (gg.abs() @ wg.abs() + gu.abs() @ wu.abs()))
    out["gx"] = (p[0] + q[0], p[1] + q[1] + both)
    out["gw_gate"], out["gw_up"] = dot(gg.t(), x.t(), rg.t()), dot(gu.t(), x.t(), ru.t())
    return out


def close(name, got, want, err):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), name
    bound = half(got.dtype) * (want.abs() + err) + err + least(got.dtype)
    over = (got.detach().double() - want).abs() / bound
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3f} of the bound at {int(over.argmax())} of {tuple(got.shape)}"


def linear_case(seed, rows, K, N, dtype, bias=False, mul=False, residual=False, btype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, std=1.0: torch.randn(s, generator=g) * std
    return {"x": n(rows, K).to(dtype).cuda(), "weight": n(N, K, std=K ** -0.5).to(dtype).cuda(),
            "bias": n(N, std=0.5).to(btype).cuda() if bias else None, "mul": n(rows, N).to(dtype).cuda() if mul else None,
            "residual": n(rows, N, std=2.0).to(dtype).cuda() if residual else None, "gy": n(rows, N).to(dtype).cuda()}


def gated_case(seed, rows, K, N, dtype):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, std=1.0: torch.randn(s, generator=g) * std
    return {"x": n(rows, K).to(dtype).cuda(), "w_gate": n(N, K, std=K ** -0.5).to(dtype).cuda(), "w_up": n(N, K, std=K ** -0.5).to(dtype).cuda(),
            "gy": n(rows, N).to(dtype).cuda()}


LINEAR, GATED = ["x", "weight", "bias", "mul", "residual"], ["x", "w_gate", "w_up"]


def train_linear(c, name):
    import rwkv_infctx_trainer_b200 as W
    leaves = {n: c[n].detach().requires_grad_(True) for n in LINEAR if c[n] is not None}
    y = W.linear_act(leaves["x"], leaves["weight"], leaves.get("bias"), name, leaves.get("mul"), leaves.get("residual"))
    grads = torch.autograd.grad(y, list(leaves.values()), c["gy"])
    return {"y": y, **{"g" + n: g for n, g in zip(leaves, grads)}}


def check_linear(c, name, got):
    want = linear_ref(c["x"], c["weight"], c["bias"], name, c["mul"], c["residual"], c["gy"])
    for n, t in got.items():
        if n == "gresidual":
            assert torch.equal(t, c["gy"])
        else:
            close(n, t, *want[n])


def train_gated(c, name):
    import rwkv_infctx_trainer_b200 as W
    leaves = {n: c[n].detach().requires_grad_(True) for n in GATED}
    y = W.gated_linear(leaves["x"], leaves["w_gate"], leaves["w_up"], name)
    return {"y": y, **{"g" + n: g for n, g in zip(leaves, torch.autograd.grad(y, list(leaves.values()), c["gy"]))}}


def check_gated(c, name, got):
    want = gated_ref(c["x"], c["w_gate"], c["w_up"], name, c["gy"])
    for n, t in got.items():
        close(n, t, *want[n])
