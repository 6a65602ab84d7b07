"""Selective state space scan, short causal convolution and root-mean-square norm: the work whose speed is
measured, with a plain form of each operator.

A case is one call of an operator, as a layer norm -> projection -> convolution -> scan makes it:

  op      "scan"   selective_scan / selective_scan_step   (B rows, T tokens, D channels, N states, G groups of B and C)
          "conv"   causal_conv / causal_conv_step         (B, T, D, width W)
          "norm"   rms_norm                               (rows, C; residual in the activations' type or in fp32)
          "q8"     rms_norm_q8                            (rows, C; group 0: one scale a row)
  mode    "train"  forward and the gradients of everything that has one
          "infer"  forward alone, state carried (a prompt)
          "step"   one token, state updated in place
  dtype   of the activations (parameters and the scan's state are fp32)

Tensors that a layer cuts out of a wider projection (x and z, B and C) are such views here too.
"""
import math

import torch
import torch.nn.functional as F

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
F8 = torch.float8_e4m3fn


def _scan(name, mode, B, T, D, N=16, G=1, dtype="bf16", gate=True):
    c = {"op": "scan", "mode": mode, "B": B, "T": T, "D": D, "N": N, "G": G, "dtype": dtype, "gate": gate}
    return {"name": name, **c} if name else c


def _conv(name, mode, B, T, D, W=4, dtype="bf16", silu=True):
    c = {"op": "conv", "mode": mode, "B": B, "T": T, "D": D, "W": W, "dtype": dtype, "silu": silu}
    return {"name": name, **c} if name else c


def _norm(name, op, mode, rows, C, dtype="bf16", residual="same", group=0):
    c = {"op": op, "mode": mode, "rows": rows, "C": C, "dtype": dtype, "residual": residual, "group": group}
    return {"name": name, **c} if name else c


def listed():
    return [
        # a training segment at the 7B shape's width: 4 rows of 4096 tokens
        _scan("scan_train_7b", "train", 4, 4096, 4096),
        # rows and widths that fit no tile, B and C shared by two groups of channels, no gate
        _scan("scan_train_ragged", "train", 3, 1001, 1530, G=2, gate=False),
        # the small fp32 job that numerics are checked on
        _scan("scan_train_fp32_small", "train", 2, 509, 256, N=8, dtype="fp32"),
        # a long prompt of one row
        _scan("scan_prefill", "infer", 1, 8191, 5120),
        # one decoded token for a large batch: the state alone is 34 MB
        _scan("scan_decode", "step", 64, 1, 8192),
        # one decoded token of one row: latency
        _scan("scan_decode_one_row", "step", 1, 1, 2560),
        # the convolution in front of scan_train_7b
        _conv("conv_train_7b", "train", 4, 4096, 4096),
        # a prompt of two rows, odd sizes, width 3
        _conv("conv_prefill_ragged", "infer", 2, 1999, 1531, W=3),
        # the convolution of a decoded token, 8 rows
        _conv("conv_decode", "step", 8, 1, 5120),
        # the norm in front of a training layer, residual stream in the activations' type
        _norm("norm_train_7b", "norm", "train", 16384, 4096),
        # a prompt's norm with an 8-bit output for the projection behind it, a scale per 128 channels
        _norm("norm_q8_prefill", "q8", "infer", 1999, 5120, residual="fp32", group=128),
        # the same for 8 decoded rows, one scale a row
        _norm("norm_q8_decode", "q8", "step", 8, 2560),
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["scan", "scan", "scan", "conv", "conv", "norm", "q8"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    if op in ("norm", "q8"):
        C = spread(64, 8192)
        rows = spread(1, min(20000, (1 << 26) // C))
        residual = rng.choice(["same", "same", "fp32", "none"])
        if op == "norm":
            return _norm(None, op, rng.choice(["train", "train", "infer"]), rows, C, dtype, residual)
        return _norm(None, op, "infer", rows, C, dtype, residual, rng.choice([0, 64, 128]))
    mode = rng.choice(["train", "train", "infer", "step"])
    if mode == "step":
        B, T, D = spread(1, 64), 1, spread(64, 8192)
    else:
        B, T = rng.randint(1, 8), spread(2, 8192)
        D = spread(64, max(64, min(8192, (1 << 26) // (B * T))))
    if op == "conv":
        return _conv(None, mode, B, T, D, rng.choice([2, 3, 4, 4]), dtype, rng.random() < 0.8)
    N, G = rng.choice([8, 16, 16, 16, 32]), rng.choice([1, 1, 2, 4])
    if mode != "step":
        D = max(64, min(D, (1 << 30) // (B * T * N)))
    return _scan(None, mode, B, T, D // G * G, N, G, dtype, rng.random() < 0.7)


# ---------------------------------------------------------------------------------------------
# inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, train = DTYPES[case["dtype"]], case["mode"] == "train"
    f32 = torch.float32

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return torch.randn(shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)

    def uniform(*shape, lo, hi):
        return torch.rand(shape, generator=g, device="cuda").mul_(hi - lo).add_(lo)

    s = {"case": case}
    if case["op"] in ("norm", "q8"):
        rows, C = case["rows"], case["C"]
        s["x"] = normal(rows, C)
        s["weight"] = normal(C, std=0.1, mean=1.0, dtype=f32)
        s["residual"] = None
        if case["residual"] != "none":
            s["residual"] = normal(rows, C, std=2.0, dtype=f32 if case["residual"] == "fp32" else dt)
        names = ["x", "weight", "residual"]
        if train:
            s["gy"] = normal(rows, C)
            if s["residual"] is not None:
                s["gh"] = normal(rows, C, dtype=s["residual"].dtype)
    elif case["op"] == "conv":
        B, T, D, W = case["B"], case["T"], case["D"], case["W"]
        s["x"] = normal(B, T, 2 * D)[..., :D]                 # the half of a projection that the gate leaves
        s["weight"] = uniform(D, W, lo=-1.0, hi=1.0) * W ** -0.5
        s["bias"] = uniform(D, lo=-0.5, hi=0.5)
        s["state"] = normal(B, W - 1, D)
        names = ["x", "weight", "bias", "state"]
        if train:
            s["gy"], s["gs"] = normal(B, T, D), normal(B, W - 1, D)
    else:
        B, T, D, N, G = (case[k] for k in "BTDNG")
        rank = 8 * max(1, D // 128)
        s["u"] = F.silu(normal(B, T, D, dtype=f32)).to(dt)    # what the convolution gives
        s["delta"] = normal(B, T, D, std=0.5)
        wide = normal(B, T, rank + 2 * G * N, std=0.7)        # one projection gives delta's factor, B and C
        s["B"] = wide[..., rank:rank + G * N].unflatten(-1, (G, N))
        s["C"] = wide[..., rank + G * N:].unflatten(-1, (G, N))
        s["z"] = normal(B, T, 2 * D)[..., D:] if case["gate"] else None
        # A: -1 .. -N as such layers start, moved by training; step sizes from 0.001 to 0.1
        s["A"] = -torch.arange(1, N + 1, device="cuda", dtype=f32) * torch.exp(normal(D, N, std=0.1, dtype=f32))
        step = torch.exp(uniform(D, lo=math.log(1e-3), hi=math.log(0.1)))
        s["delta_bias"] = step + torch.log(-torch.expm1(-step))
        s["D"] = normal(D, std=0.1, mean=1.0, dtype=f32)
        s["state"] = normal(B, D, N, std=0.3, dtype=f32)
        names = ["u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state"]
        if train:
            s["gy"], s["gs"] = normal(B, T, D), normal(B, D, N, std=0.3, dtype=f32)
    s["names"] = [n for n in names if s[n] is not None]
    if train:
        for n in s["names"]:
            s[n] = s[n].detach().requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------------
# one pass

def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    with torch.no_grad():
        if case["op"] == "norm":
            return _plain_norm(s, case)
        if case["op"] == "q8":
            return _plain_q8(s, case)
        if case["op"] == "conv":
            return _plain_conv(s, case)
        return _plain_scan(s, case)


def _own(s, case):
    import rwkv_infctx_trainer_b200 as W

    if case["op"] == "norm":
        with torch.set_grad_enabled(case["mode"] == "train"):
            out = W.rms_norm(s["x"], s["weight"], s["residual"])
        out = out if isinstance(out, tuple) else (out,)
        seeds = [s[n] for n in ("gy", "gh") if n in s]
    elif case["op"] == "q8":
        return W.rms_norm_q8(s["x"], s["weight"], s["residual"], group=case["group"] or None)
    elif case["op"] == "conv":
        if case["mode"] == "step":
            y = W.causal_conv_step(s["x"][:, 0], s["state"], s["weight"], s["bias"], silu=case["silu"])
            return y, s["state"]
        with torch.set_grad_enabled(case["mode"] == "train"):
            out = W.causal_conv(s["x"], s["weight"], s["bias"], s["state"], silu=case["silu"])
        seeds = [s[n] for n in ("gy", "gs") if n in s]
    else:
        if case["mode"] == "step":
            y = W.selective_scan_step(s["u"][:, 0], s["delta"][:, 0], s["A"], s["B"][:, 0], s["C"][:, 0], s["state"], s["D"],
                                      None if s["z"] is None else s["z"][:, 0], s["delta_bias"])
            return y, s["state"]
        with torch.set_grad_enabled(case["mode"] == "train"):
            out = W.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], s["D"], s["z"], s["delta_bias"], state=s["state"])
        seeds = [s[n] for n in ("gy", "gs") if n in s]
    if case["mode"] != "train":
        return out
    grads = torch.autograd.grad(out, [s[n] for n in s["names"]], seeds)
    return [t.detach() for t in out], list(grads)


def _f32(t):
    return None if t is None else t.float()


def _plain_norm_parts(s):
    x, res = s["x"].float(), s["residual"]
    h = x if res is None else x + res.float()
    return h, torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6)


def _plain_norm(s, case):
    h, r = _plain_norm_parts(s)
    w, res = s["weight"].float(), s["residual"]
    out = [(h * r * w).to(s["x"].dtype)] + ([] if res is None else [h.to(res.dtype)])
    if case["mode"] != "train":
        return tuple(out) if res is not None else (out[0],)
    gn = s["gy"].float() * w
    xh = h * r
    gx = r * (gn - xh * (gn * xh).mean(-1, keepdim=True))
    if res is not None:
        gx = gx + s["gh"].float()
    grads = [gx.to(s["x"].dtype), (s["gy"].float() * xh).sum(0)] + ([] if res is None else [gx.to(res.dtype)])
    return out, grads


def _plain_q8(s, case):
    h, r = _plain_norm_parts(s)
    y, res, (rows, C) = h * r * s["weight"].float(), s["residual"], s["x"].shape
    group = case["group"] or C
    n = -(-C // group)
    parts = F.pad(y, (0, n * group - C)).view(rows, n, group)
    top = parts.abs().amax(-1, keepdim=True)
    scale = torch.where(top == 0, torch.ones_like(top), top / 448.0)
    q = (parts / scale).clamp(-448.0, 448.0).to(F8).view(rows, n * group)[:, :C].contiguous()
    return (q, scale.squeeze(-1)) + (() if res is None else (h.to(res.dtype),))


def _plain_conv(s, case):
    x, w, b, st, T, W = s["x"].float(), s["weight"].float(), s["bias"].float(), s["state"].float(), case["T"], case["W"]
    xs = torch.cat((st, x), 1)                                                    # [B, W-1+T, D]
    pre = sum(xs[:, j:j + T] * w[:, j] for j in range(W)) + b
    sig = torch.sigmoid(pre)
    dt = s["x"].dtype
    y, new = (pre * sig if case["silu"] else pre).to(dt), xs[:, T:].to(dt)
    if case["mode"] == "step":
        s["state"].copy_(new)
        return y[:, 0], s["state"]
    if case["mode"] != "train":
        return y, new
    gp = s["gy"].float()
    if case["silu"]:
        gp = gp * sig * (1 + pre * (1 - sig))
    gxs = sum(F.pad(gp * w[:, j], (0, 0, j, W - 1 - j)) for j in range(W))
    gxs = gxs + F.pad(s["gs"].float(), (0, 0, T, 0))
    gw = torch.stack([(gp * xs[:, j:j + T]).sum((0, 1)) for j in range(W)], -1)
    return [y, new], [gxs[:, W - 1:].to(dt), gw, gp.sum((0, 1)), gxs[:, :W - 1].to(dt)]


def _recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, from h = 0: what a span of tokens does, spans doubled log2(T) times."""
    k = 1
    while k < b.shape[1]:
        b = torch.cat((b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]), 1)
        a = torch.cat((a[:, :k], a[:, k:] * a[:, :-k]), 1)
        k *= 2
    return b


def _plain_scan(s, case):
    B, T, D, N, G = (case[k] for k in "BTDNG")
    u, A, Dv, z = s["u"].float(), s["A"].float(), s["D"].float(), _f32(s["z"])
    raw = s["delta"].float() + s["delta_bias"].float()
    dt = F.softplus(raw)
    # [B, T, D, N]: groups of D / G channels share a row of B and of C
    Bm, Cm = (s[n].float().repeat_interleave(D // G, 2) for n in "BC")
    a = torch.exp(dt.unsqueeze(-1) * A)
    b = (dt * u).unsqueeze(-1) * Bm
    b[:, 0] += a[:, 0] * s["state"]
    h = _recurrence(a, b)
    del b
    y0 = (h * Cm).sum(-1) + Dv * u
    gate = None if z is None else z * torch.sigmoid(z)
    kind = s["u"].dtype
    y, new = (y0 if z is None else y0 * gate).to(kind), h[:, -1].contiguous()
    if case["mode"] == "step":
        s["state"].copy_(new)
        return y[:, 0], s["state"]
    if case["mode"] != "train":
        return y, new
    gy = s["gy"].float()
    dy = gy if z is None else gy * gate
    c = dy.unsqueeze(-1) * Cm
    c[:, -1] += s["gs"]
    later = torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), 1)
    gh = _recurrence(later.flip(1), c.flip(1)).flip(1)
    del c, later
    before = torch.cat((s["state"].unsqueeze(1), h[:, :-1]), 1)
    gdec = gh * a * before                              # the gradient at dt A
    gB = (gh * (dt * u).unsqueeze(-1)).unflatten(2, (G, D // G)).sum(3)
    gC = (h * dy.unsqueeze(-1)).unflatten(2, (G, D // G)).sum(3)
    gin = (gh * Bm).sum(-1)
    graw = (u * gin + (gdec * A).sum(-1)) * torch.sigmoid(raw)
    grads = {"u": (dt * gin + Dv * dy).to(kind), "delta": graw.to(kind), "A": (gdec * dt.unsqueeze(-1)).sum((0, 1)),
             "B": gB.to(kind), "C": gC.to(kind), "D": (dy * u).sum((0, 1)), "delta_bias": graw.sum((0, 1)),
             "state": gh[:, 0] * a[:, 0]}
    if z is not None:
        sig = torch.sigmoid(z)
        grads["z"] = (gy * y0 * sig * (1 + z * (1 - sig))).to(kind)
    return [y, new], [grads[n] for n in s["names"]]


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    train = case["mode"] == "train"
    if case["op"] == "scan":
        return _exact_scan(s, case, train)
    d = {n: s[n].detach().double().requires_grad_(train) for n in s["names"]}
    if case["op"] == "conv":
        B, T, D, W = (case[k] for k in "BTDW")
        xs = torch.cat((d["state"], d["x"]), 1)
        y = F.conv1d(xs.transpose(1, 2), d["weight"].unsqueeze(1), d["bias"], groups=D).transpose(1, 2)
        y = F.silu(y) if case["silu"] else y
        out = [y, xs[:, T:]]
        if case["mode"] == "step":
            return y[:, 0], out[1]
        seeds = [s["gy"].double(), s["gs"].double()] if train else None
    else:
        h = d["x"] if s["residual"] is None else d["x"] + d["residual"]
        y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * d["weight"]
        if case["op"] == "q8":
            C, group = case["C"], case["group"] or case["C"]
            scale = torch.stack([p.abs().amax(-1) for p in y.split(group, -1)], -1) / 448.0
            q = torch.cat([p / scale[:, i:i + 1] for i, p in enumerate(y.split(group, -1))], -1)
            return (q, scale) + (() if s["residual"] is None else (h,))
        out = [y] + ([] if s["residual"] is None else [h])
        seeds = [s[n].double() for n in ("gy", "gh") if n in s]
    if not train:
        return tuple(out)
    grads = torch.autograd.grad(out, [d[n] for n in s["names"]], seeds)
    return [t.detach() for t in out], list(grads)


def _exact_scan(s, case, train):
    """The recurrence token by token and automatic differentiation, a block of channels after the other."""
    B, T, D, N, G = (case[k] for k in "BTDNG")
    d = {n: s[n].detach().double().requires_grad_(train) for n in s["names"]}
    per = D // G
    width = max(1, min(per, (1 << 31) // (B * T * N * 8) if train else per))
    ys, new, grads = [], [], {n: torch.zeros_like(d[n]) for n in d}
    for grp in range(G):
        for c0 in range(grp * per, (grp + 1) * per, width):
            c1 = min(c0 + width, (grp + 1) * per)
            with torch.set_grad_enabled(train):
                dt = F.softplus(d["delta"][..., c0:c1] + d["delta_bias"][c0:c1])
                A, Bm, Cm = d["A"][c0:c1], d["B"][:, :, grp], d["C"][:, :, grp]
                dtu = dt * d["u"][..., c0:c1]
                h, rows = d["state"][:, c0:c1], []
                for step, inp, bt, ct in zip(dt.unbind(1), dtu.unbind(1), Bm.unbind(1), Cm.unbind(1)):
                    h = torch.exp(step.unsqueeze(-1) * A) * h + inp.unsqueeze(-1) * bt.unsqueeze(1)
                    rows.append(torch.einsum("bcn,bn->bc", h, ct))
                y = torch.stack(rows, 1) + d["D"][c0:c1] * d["u"][..., c0:c1]
                if "z" in d:
                    y = y * F.silu(d["z"][..., c0:c1])
            if train:
                got = torch.autograd.grad([y, h], [d[n] for n in s["names"]], [s["gy"][..., c0:c1].double(), s["gs"][:, c0:c1].double()])
                for n, t in zip(s["names"], got):
                    grads[n] += t
            ys.append(y.detach())
            new.append(h.detach())
    y, new = torch.cat(ys, -1), torch.cat(new, 1)
    if case["mode"] == "step":
        return y[:, 0], new
    return ([y, new], [grads[n] for n in s["names"]]) if train else (y, new)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    """Bytes: the forward pass reads its inputs and writes its outputs once; the backward pass reads the inputs and the
    incoming gradients and writes the gradients once.  Operations: multiplications, additions and exponentials."""
    size, train = DTYPES[case["dtype"]].itemsize, case["mode"] == "train"
    if case["op"] in ("norm", "q8"):
        n, C = case["rows"] * case["C"], case["C"]
        res = {"none": 0, "same": size, "fp32": 4}[case["residual"]]
        if case["op"] == "q8":
            groups = -(-C // (case["group"] or C))
            return {"bytes": n * (size + 2 * res + 1) + 4 * (C + case["rows"] * groups), "flops": 6 * n}
        fwd, bwd = n * (2 * size + 2 * res) + 4 * C, n * (size + max(res, size) + res + size + (res if res != size else 0)) + 8 * C
        return {"bytes": fwd + (bwd if train else 0), "flops": n * (5 + (10 if train else 0))}
    B, T, D = case["B"], case["T"], case["D"]
    n = B * T * D
    if case["op"] == "conv":
        W = case["W"]
        params, state = 4 * D * (W + 1), B * (W - 1) * D * size
        fwd, bwd = 2 * n * size + params + 2 * state, 3 * n * size + 2 * params + 3 * state
        return {"bytes": fwd + (bwd if train else 0), "flops": n * (2 * W + 4 + (4 * W + 8 if train else 0))}
    N, G, z = case["N"], case["G"], int(case["gate"])
    params, state, bc = 4 * D * (N + 2), 4 * B * D * N, B * T * G * N * size
    fwd = (3 + z) * n * size + 2 * bc + params + 2 * state
    bwd = (5 + 2 * z) * n * size + 4 * bc + 2 * params + 3 * state
    return {"bytes": fwd + (bwd if train else 0), "flops": n * (N * (7 + (20 if train else 0)) + 12)}
