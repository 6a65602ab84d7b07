"""Gated linear recurrence, matrix product with its epilogue, gated pair of matrix products: the work whose speed is
measured, with a plain form of each operator.

A case is one call of an operator, as a recurrent layer and its feed-forward block make it
(norm -> projections -> convolution -> recurrence -> projection + residual, norm -> gated pair -> projection + residual):

  op      "rec"     gated_recurrence / gated_recurrence_step       (B rows, T tokens, D channels; gate: the output gate z)
          "linear"  linear_act: act(x W^T + bias) * mul + residual  (rows, K -> N)
          "gated"   gated_linear: act(x Wg^T) * (x Wu^T)            (rows, K -> N)
  mode    "train"   forward and the gradients of everything that has one
          "infer"   forward alone (the recurrence: state carried, a prompt)
          "step"    "rec" only: one token, state updated in place
  dtype   of the activations and the matrices (the recurrence's parameter and its state are fp32)
"""
import math

import torch
import torch.nn.functional as F

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DECAY = 8.0             # the recurrence's constant c


def _rec(name, mode, B, T, D, dtype="bf16", gate=True):
    c = {"op": "rec", "mode": mode, "B": B, "T": T, "D": D, "dtype": dtype, "gate": gate}
    return {"name": name, **c} if name else c


def _linear(name, mode, rows, K, N, act="none", dtype="bf16", bias=False, mul=False, residual=False):
    c = {"op": "linear", "mode": mode, "rows": rows, "K": K, "N": N, "act": act, "dtype": dtype, "bias": bias, "mul": mul,
         "residual": residual}
    return {"name": name, **c} if name else c


def _gated(name, mode, rows, K, N, act="silu", dtype="bf16"):
    c = {"op": "gated", "mode": mode, "rows": rows, "K": K, "N": N, "act": act, "dtype": dtype}
    return {"name": name, **c} if name else c


def listed():
    return [
        # a training segment at the 7B shape's width: 4 rows of 4096 tokens
        _rec("rec_train_7b", "train", 4, 4096, 4096),
        # rows and widths that fit no tile, no output gate
        _rec("rec_train_ragged", "train", 3, 1001, 1531, gate=False),
        # the small fp32 job that numerics are checked on
        _rec("rec_train_fp32_small", "train", 2, 509, 256, dtype="fp32"),
        # a long prompt of one row
        _rec("rec_prefill", "infer", 1, 8191, 5120),
        # one decoded token for a large batch
        _rec("rec_decode", "step", 64, 1, 8192),
        # a layer's output projection in training, the residual added in its epilogue
        _linear("linear_train_7b", "train", 16384, 4096, 4096, residual=True),
        # sizes that fit no tile, fp16, bias and GELU
        _linear("linear_train_ragged", "train", 3003, 1531, 2049, act="gelu", dtype="fp16", bias=True),
        # a channel mix's receptance for a prompt: sigmoid(x W^T) times the values
        _linear("linear_prefill", "infer", 1999, 2560, 2560, act="sigmoid", mul=True),
        # a channel mix's squared-ReLU key for 8 decoded rows: the matrix is read once
        _linear("linear_decode", "infer", 8, 4096, 14336, act="relu2"),
        # the gated pair of a feed-forward block in training
        _gated("gated_train_7b", "train", 8192, 4096, 14336),
        # the same for a prompt of the 3B shape's width
        _gated("gated_prefill", "infer", 1999, 2560, 8960),
        # one decoded row: two matrices read once
        _gated("gated_decode", "infer", 1, 2560, 8960),
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["rec", "rec", "linear", "linear", "gated"])
    if op == "rec":
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        mode = rng.choice(["train", "train", "infer", "step"])
        if mode == "step":
            B, T, D = spread(1, 64), 1, spread(64, 8192)
        else:
            B, T = rng.randint(1, 8), spread(2, 16384)
            D = spread(64, max(64, min(8192, (1 << 26) // (B * T * (2 if dtype == "fp32" else 1)))))
        return _rec(None, mode, B, T, D, dtype, rng.random() < 0.6)
    dtype, mode = rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["train", "train", "infer"])
    rows, K = spread(1, 16384), spread(64, 8192)
    most = (16384 * 4096 * 4096 if op == "linear" else 8192 * 4096 * 14336) // (rows * K)
    N = spread(64, max(64, min(14336, most)))
    if rng.random() < 0.6:                                    # widths of models are multiples of 64
        K, N = (K + 63) // 64 * 64, max(64, N // 64 * 64)
    if op == "gated":
        return _gated(None, mode, rows, K, N, rng.choice(["silu", "silu", "gelu", "sigmoid", "relu2", "none"]), dtype)
    return _linear(None, mode, rows, K, N, rng.choice(["none", "none", "silu", "gelu", "sigmoid", "relu2"]), dtype,
                   rng.random() < 0.4, rng.random() < 0.25, rng.random() < 0.4)


# ---------------------------------------------------------------------------------------------
# inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, train = DTYPES[case["dtype"]], case["mode"] == "train"
    f32 = torch.float32

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return torch.randn(shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)

    s = {"case": case}
    if case["op"] == "rec":
        B, T, D = (case[k] for k in "BTD")
        s["x"] = normal(B, T, D)                              # what the convolution gives
        gates = normal(B, T, 2 * D)                           # one projection gives both gates
        s["input_gate"], s["decay_gate"] = gates[..., :D], gates[..., D:]
        # the decay where the gate is fully open: 0.9 to 0.999, as such layers start
        top = torch.rand(D, generator=g, device="cuda").mul_(0.099).add_(0.9)
        s["decay"] = torch.log(torch.expm1(-torch.log(top) / DECAY))
        s["z"] = normal(B, T, 2 * D)[..., D:] if case["gate"] else None
        s["state"] = normal(B, D, std=0.5, dtype=f32)
        names = ["x", "input_gate", "decay_gate", "decay", "z", "state"]
        if train:
            s["gy"], s["gs"] = normal(B, T, D), normal(B, D, std=0.5, dtype=f32)
    else:
        rows, K, N = (case[k] for k in ("rows", "K", "N"))
        s["x"] = normal(rows, K)                              # what the norm in front gives
        if case["op"] == "gated":
            s["w_gate"], s["w_up"] = normal(N, K, std=K ** -0.5), normal(N, K, std=K ** -0.5)
            names = ["x", "w_gate", "w_up"]
        else:
            s["weight"] = normal(N, K, std=K ** -0.5)
            s["bias"] = normal(N, std=0.1, dtype=f32) if case["bias"] else None
            s["mul"] = normal(rows, N) if case["mul"] else None
            s["residual"] = normal(rows, N, std=2.0) if case["residual"] else None
            names = ["x", "weight", "bias", "mul", "residual"]
        if train:
            s["gy"] = normal(rows, N)
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
        return {"rec": _plain_rec, "linear": _plain_linear, "gated": _plain_gated}[case["op"]](s, case)


def _own(s, case):
    import rwkv_infctx_trainer_b200 as W

    train = case["mode"] == "train"
    if case["op"] == "rec":
        if case["mode"] == "step":
            y = W.gated_recurrence_step(s["x"][:, 0], s["input_gate"][:, 0], s["decay_gate"][:, 0], s["decay"], s["state"],
                                        None if s["z"] is None else s["z"][:, 0], c=DECAY)
            return y, s["state"]
        with torch.set_grad_enabled(train):
            out = W.gated_recurrence(s["x"], s["input_gate"], s["decay_gate"], s["decay"], s["z"], state=s["state"], c=DECAY)
        seeds = [s[n] for n in ("gy", "gs") if n in s]
    else:
        with torch.set_grad_enabled(train):
            if case["op"] == "gated":
                out = (W.gated_linear(s["x"], s["w_gate"], s["w_up"], activation=case["act"]),)
            else:
                out = (W.linear_act(s["x"], s["weight"], s["bias"], activation=case["act"], mul=s["mul"], residual=s["residual"]),)
        seeds = [s[n] for n in ("gy",) if n in s]
    if not train:
        return out
    grads = torch.autograd.grad(out, [s[n] for n in s["names"]], seeds)
    return [t.detach() for t in out], list(grads)


def _act(name, z):
    """the activation and its derivative"""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu2":
        p = z.clamp_min(0)
        return p * p, 2 * p
    if name == "gelu":                                        # z Phi(z)
        phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    sig = torch.sigmoid(z)
    if name == "sigmoid":
        return sig, sig * (1 - sig)
    return z * sig, sig * (1 + z * (1 - sig))                 # silu


def _plain_linear(s, case):
    x, w, dt = s["x"].float(), s["weight"].float(), s["x"].dtype
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    a, da = _act(case["act"], z)
    y = a if s["mul"] is None else a * s["mul"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    y = y.to(dt)
    if case["mode"] != "train":
        return (y,)
    gy = s["gy"].float()
    gz = (gy if s["mul"] is None else gy * s["mul"].float()) * da
    grads = {"x": (gz @ w).to(dt), "weight": (gz.t() @ x).to(dt), "bias": gz.sum(0), "mul": (gy * a).to(dt), "residual": s["gy"].detach()}
    return [y], [grads[n] for n in s["names"]]


def _plain_gated(s, case):
    x, wg, wu, dt = s["x"].float(), s["w_gate"].float(), s["w_up"].float(), s["x"].dtype
    u = x @ wu.t()
    a, da = _act(case["act"], x @ wg.t())
    y = (a * u).to(dt)
    if case["mode"] != "train":
        return (y,)
    gy = s["gy"].float()
    gu, gg = gy * a, gy * u * da
    return [y], [(gg @ wg + gu @ wu).to(dt), (gg.t() @ x).to(dt), (gu.t() @ x).to(dt)]


def _recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, from h = 0: what a span of tokens does, spans doubled log2(T) times."""
    k = 1
    while k < b.shape[1]:
        b = torch.cat((b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]), 1)
        a = torch.cat((a[:, :k], a[:, k:] * a[:, :-k]), 1)
        k *= 2
    return b


def _plain_rec(s, case):
    x, p = s["x"].float(), s["decay"].float()
    i, r = torch.sigmoid(s["input_gate"].float()), torch.sigmoid(s["decay_gate"].float())
    kind = s["x"].dtype
    rate = -DECAY * F.softplus(p)
    L = rate * r                                              # log of the decay
    a, q = torch.exp(L), -torch.expm1(2 * L)
    m = torch.sqrt(q)
    b = m * i * x
    b[:, 0] += a[:, 0] * s["state"]
    h = _recurrence(a, b)
    z = None if s["z"] is None else s["z"].float()
    gate, dgate = (None, None) if z is None else _act("silu", z)
    y, new = (h if z is None else h * gate).to(kind), h[:, -1].contiguous()
    if case["mode"] == "step":
        s["state"].copy_(new)
        return y[:, 0], s["state"]
    if case["mode"] != "train":
        return y, new
    gy = s["gy"].float()
    c = gy.clone() if z is None else gy * gate
    c[:, -1] += s["gs"]
    later = torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), 1)
    gh = _recurrence(later.flip(1), c.flip(1)).flip(1)
    before = torch.cat((s["state"].unsqueeze(1), h[:, :-1]), 1)
    slope = torch.where(q > 0, L / torch.where(q > 0, m, 1), 0)          # L dm/dL = -a^2 L / m
    gLL = gh * (a * L * before - i * x * a * a * slope)       # the gradient at L, times L
    grads = {"x": (gh * m * i).to(kind), "input_gate": (gh * m * x * i * (1 - i)).to(kind), "decay_gate": (gLL * (1 - r)).to(kind),
             "decay": gLL.sum((0, 1)) * torch.sigmoid(p) / F.softplus(p), "state": gh[:, 0] * a[:, 0]}
    if z is not None:
        grads["z"] = (gy * h * dgate).to(kind)
    return [y, new], [grads[n] for n in s["names"]]


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits, gradients by automatic differentiation

def exact(case, seed):
    s = prepare(case, seed)
    train = case["mode"] == "train"
    d = {n: s[n].detach().double().requires_grad_(train) for n in s["names"]}
    if case["op"] == "rec":
        with torch.set_grad_enabled(train):
            a = torch.exp(-DECAY * F.softplus(d["decay"]) * torch.sigmoid(d["decay_gate"]))
            b = torch.sqrt((1 - a) * (1 + a)) * torch.sigmoid(d["input_gate"]) * d["x"]
            h, rows = d["state"], []
            for at, bt in zip(a.unbind(1), b.unbind(1)):
                h = at * h + bt
                rows.append(h)
            y = torch.stack(rows, 1)
            if "z" in d:
                y = y * F.silu(d["z"])
        if case["mode"] == "step":
            return y[:, 0], h
        out, seeds = [y, h], [s[n].double() for n in ("gy", "gs") if n in s]
    else:
        fns = {"none": lambda t: t, "silu": F.silu, "gelu": F.gelu, "sigmoid": torch.sigmoid, "relu2": lambda t: F.relu(t).square()}
        act = fns[case["act"]]
        with torch.set_grad_enabled(train):
            if case["op"] == "gated":
                y = act(F.linear(d["x"], d["w_gate"])) * F.linear(d["x"], d["w_up"])
            else:
                y = act(F.linear(d["x"], d["weight"], d.get("bias")))
                y = y * d["mul"] if "mul" in d else y
                y = y + d["residual"] if "residual" in d else y
        out, seeds = [y], [s[n].double() for n in ("gy",) if n in s]
    if not train:
        return tuple(out)
    grads = torch.autograd.grad(out, [d[n] for n in s["names"]], seeds)
    return [t.detach() for t in out], list(grads)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    """Bytes: the forward pass reads its inputs and writes its outputs once; the backward pass reads the inputs and the
    incoming gradients and writes the gradients once.  Operations: multiplications and additions, and for the recurrence
    exponentials, roots and quotients."""
    size, train = DTYPES[case["dtype"]].itemsize, case["mode"] == "train"
    if case["op"] == "rec":
        B, T, D = (case[k] for k in "BTD")
        n, z, state = B * T * D, int(case["gate"]), 4 * B * D
        fwd, bwd = (4 + z) * n * size + 2 * state + 4 * D, (7 + 2 * z) * n * size + 3 * state + 8 * D
        return {"bytes": fwd + (bwd if train else 0), "flops": n * ((18 + 6 * z) + (40 + 10 * z if train else 0))}
    rows, K, N = (case[k] for k in ("rows", "K", "N"))
    pair = 2 if case["op"] == "gated" else 1
    x, w, y = rows * K * size, pair * N * K * size, rows * N * size
    bias = 4 * N if case.get("bias") else 0
    mul, res = (y if case.get(k) else 0 for k in ("mul", "residual"))
    fwd, bwd = x + w + y + bias + mul + res, 2 * x + 2 * w + y + 2 * bias + 2 * mul
    return {"bytes": fwd + (bwd if train else 0), "flops": 2 * rows * pair * N * K * (3 if train else 1)}
