"""The norm, the short convolution and the selective scan in 64 bits, written from their formulas, with the magnitudes that
fp32 errors are measured against.

Every reference takes ``mag``: the same sums with every term's absolute value.  A kernel that adds in fp32 is off by at most
K 2^-24 of that sum, where K counts the roundings a term passes through; a result in a type of half-step ``eps / 2`` is then
rounded once.  ``close`` holds a result to exactly that."""
import torch

U = 2.0 ** -24          # half a step of fp32


def close(name, got, want, mag, K):
    """|got - want| <= eps / 2 |want| + K 2^-24 mag (1 + eps), element by element; smallest normal numbers aside"""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny
    got, err = got.detach().double(), K * U * mag
    assert torch.isfinite(got).all(), name
    bound = half * (want.abs() + err) + err + tiny
    over = (got - want).abs() / bound
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3f} of the bound at {int(over.argmax())}"


def silu(x):
    return x * torch.sigmoid(x)


def silu_grad(x, mag=False):
    # (the sum 1 + x (1 - s) cancels near x = -1.28: its roundings are 2^-24 of 1 + |x| (1 - s))
    s = torch.sigmoid(x)
    return s * (1 + (x.abs() if mag else x) * (1 - s))


# ---------------------------------------------------------------------------------------- selective scan
def scan_ref(u, delta, A, B, C, D, z, bias, softplus, state, gy=None, gs=None, mag=False):
    """dict of y, state and (with gy, gs) the gradients; B, C [B,T,G,N]"""
    d = lambda t: None if t is None else t.detach().double()
    u, delta, A, B, C, D, z, bias, state, gy, gs = (d(t) for t in (u, delta, A, B, C, D, z, bias, state, gy, gs))
    nb, T, nd = u.shape
    N, G = A.shape[1], B.shape[2]
    raw = delta if bias is None else delta + bias
    dt, sig = (torch.nn.functional.softplus(raw), torch.sigmoid(raw)) if softplus else (raw, torch.ones_like(raw))
    gate, dgate = (torch.ones_like(u), None) if z is None else (silu(z), silu_grad(z, mag))
    h = torch.zeros((nb, nd, N), dtype=torch.float64, device=u.device) if state is None else state
    D = torch.zeros(nd, dtype=torch.float64, device=u.device) if D is None else D
    dec = torch.exp(dt.unsqueeze(-1) * A)
    w = lambda t: t.abs() if mag else t
    u, B, C, D, gate, h, dt_, A_ = w(u), w(B), w(C), w(D), w(gate), w(h), w(dt), w(A)
    wide = lambda t: t.repeat_interleave(nd // G, 2)          # [B,T,D,N]
    Bw, Cw = wide(B), wide(C)
    hs = [h]
    for t in range(T):
        hs.append(dec[:, t] * hs[-1] + (dt_[:, t] * u[:, t]).unsqueeze(-1) * Bw[:, t])
    H = torch.stack(hs, 1)                                       # state before token t; the last behind all
    y0 = (H[:, 1:] * Cw).sum(-1) + D * u
    out = {"y": y0 * gate, "state": H[:, -1]}
    if gy is None and gs is None:
        return out
    gy = torch.zeros_like(u) if gy is None else w(gy)
    E = torch.zeros_like(out["state"]) if gs is None else w(gs)
    dy = gy * gate
    rows = []
    for t in range(T - 1, -1, -1):
        g = Cw[:, t] * dy[:, t].unsqueeze(-1) + E
        E = dec[:, t] * g
        rows.append(g)
    g = torch.stack(rows[::-1], 1) if rows else torch.zeros_like(Bw)
    ga = g * dec * H[:, :-1]
    gin = (g * Bw).sum(-1)
    graw = (u * gin + (ga * A_).sum(-1)) * sig
    by_group = lambda t: t.unflatten(2, (G, nd // G)).sum(3)
    out.update(gu=dt_ * gin + D * dy, gdelta=graw, gA=(ga * dt_.unsqueeze(-1)).sum((0, 1)), gB=by_group(g * (dt_ * u).unsqueeze(-1)),
               gC=by_group(H[:, 1:] * dy.unsqueeze(-1)), gD=(dy * u).sum((0, 1)), gbias=graw.sum((0, 1)), gstate=E)
    if z is not None:
        out["gz"] = gy * y0 * dgate
    return out


def scan_K(name, B, T, D, N):
    """roundings a term of an output passes through, counted in 2^-24:
    a decay 8 (exp2 2 ulp = 4, its argument's two roundings 2, the product and the sum 2) for each of at most T tokens, in
    each direction for a gradient; dt 16 (exp of an argument below 16: 8, log1p and the sums 8), entering a term twice and
    the exponents once more (an error x of the exponent X moves e^-X by X e^-X x < 0.4 x); gates 16 each; the sum over the
    states N, over the channels D (16-bit sums over CTAs included), over the tokens B T"""
    k = 8 * T + 64 + N
    if name.startswith("g"):
        k += 8 * T + 64 + 16
    if name in ("gB", "gC"):
        k += D
    if name in ("gA", "gD", "gbias"):
        k += B * T
    return k


def scan_case(seed, B, T, D, N, G, dtype, gate=True, skip=True, bias=True, state=True, device="cuda", strided=False):
    g = torch.Generator(device="cpu").manual_seed(seed)
    n = lambda *s, std=1.0: torch.randn(s, generator=g) * std
    wide = lambda *s, std=1.0: (n(*s[:-1], 2 * s[-1] + 8, std=std).to(dtype).to(device)[..., 8:8 + s[-1]] if strided
                                else n(*s, std=std).to(dtype).to(device))
    c = {"u": wide(B, T, D), "delta": wide(B, T, D, std=0.7), "B": wide(B, T, G * N, std=0.7).unflatten(-1, (G, N)),
         "C": wide(B, T, G * N, std=0.7).unflatten(-1, (G, N)), "z": wide(B, T, D) if gate else None,
         "A": (-torch.rand((D, N), generator=g) * 8 - 0.01).to(device), "D": n(D).to(device) if skip else None,
         "delta_bias": (torch.rand(D, generator=g) * 4 - 5).to(device) if bias else None,
         "state": n(B, D, N).to(device) if state else None, "gy": n(B, T, D).to(dtype).to(device), "gs": n(B, D, N).to(device)}
    return c


SCAN_LEAVES = ["u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state"]
SCAN_GRADS = ["gu", "gdelta", "gA", "gB", "gC", "gD", "gz", "gbias", "gstate"]


# ---------------------------------------------------------------------------------------- convolution
def conv_ref(x, w, bias, state, act, gy=None, gs=None, mag=False):
    d = lambda t: None if t is None else t.detach().double()
    x, w, bias, state, gy, gs = (d(t) for t in (x, w, bias, state, gy, gs))
    B, T, D = x.shape
    W = w.shape[-1]
    state = torch.zeros((B, W - 1, D), dtype=torch.float64, device=x.device) if state is None else state
    xs = torch.cat((state, x), 1)
    pre = sum(xs[:, j:j + T] * w[:, j] for j in range(W)) + (0 if bias is None else bias)
    ab = lambda t: t.abs() if mag else t
    pm = sum(ab(xs[:, j:j + T] * w[:, j]) for j in range(W)) + (0 if bias is None else ab(bias)) if mag else pre
    # (d silu(s) / d s is at most 1.1 in size, and |silu(s)| <= |s|)
    out = {"y": (1.1 * pm if mag else silu(pre)) if act else pm, "state": xs[:, T:]}
    if gy is None:
        return out
    dp = silu_grad(pre) if act else torch.ones_like(pre)
    # an error of s moves silu'(s) by at most 0.5 of it
    g = ab(gy) * (dp.abs() + 0.5 * pm) if mag else gy * dp
    gxs = sum(torch.nn.functional.pad(g * ab(w[:, j]), (0, 0, j, W - 1 - j)) for j in range(W))
    if gs is not None:
        gxs = gxs + torch.nn.functional.pad(ab(gs), (0, 0, T, 0))
    out.update(gx=gxs[:, W - 1:], gstate=gxs[:, :W - 1], gbias=g.sum((0, 1)),
               gw=torch.stack([(g * ab(xs[:, j:j + T])).sum((0, 1)) for j in range(W)], -1))
    return out


# s: W products and sums; the sigmoid 16 (exp of an argument below 16: 8, the sum, the quotient, the products)
def conv_K(name, B, T, W):
    k = 2 * W + 32
    if name.startswith("g"):
        k += 2 * W + 32
    if name in ("gw", "gbias"):
        k += B * T
    return k


# ---------------------------------------------------------------------------------------- norm
def norm_ref(x, w, res, eps, gy=None, gh=None):
    d = lambda t: None if t is None else t.detach().double()
    x, w, res, gy, gh = (d(t) for t in (x, w, res, gy, gh))
    out = {}
    h = x if res is None else x + res
    r = torch.rsqrt((h * h).mean(-1, keepdim=True) + eps)
    out["y"], out["h"] = h * r * w, h
    out["y_mag"], out["h_mag"] = out["y"].abs(), x.abs() + (0 if res is None else res.abs())
    if gy is None and gh is None:
        return out
    gy = torch.zeros_like(x) if gy is None else gy
    gh = torch.zeros_like(x) if gh is None else gh
    xh, gn = h * r, gy * w
    out["gx"] = gh + r * (gn - xh * (gn * xh).mean(-1, keepdim=True))
    out["gx_mag"] = gh.abs() + r * (gn.abs() + xh.abs() * (gn * xh).abs().mean(-1, keepdim=True))
    dims = tuple(range(x.dim() - 1))
    out["gw"], out["gw_mag"] = (gy * xh).sum(dims), (gy * xh).abs().sum(dims)
    return out
