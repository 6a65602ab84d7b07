"""What the matrix products keep for the backward pass: nothing that the wanted gradients do not need."""
import itertools

import pytest
import torch

import linear_testlib as L

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
MB = 2 ** 20


def call(c, leaves, name):
    import rwkv_infctx_trainer_b200 as W
    a = {n: leaves.get(n, c[n]) for n in L.LINEAR}
    return W.linear_act(a["x"], a["weight"], a["bias"], name, a["mul"], a["residual"])


@pytest.mark.parametrize("name", ["none", "gelu"])
@pytest.mark.parametrize("mul", [True, False])
@pytest.mark.parametrize("rows", [5, 200])
def test_every_choice_of_gradients(rows, mul, name):
    """the same bits whichever others are wanted"""
    c = L.linear_case(1, rows, 72, 48, BF, bias=True, mul=mul, residual=True)
    names = [n for n in L.LINEAR if c[n] is not None]
    want = L.train_linear(c, name)
    for k in range(1, len(names) + 1):
        for some in itertools.combinations(names, k):
            leaves = {n: c[n].detach().requires_grad_(True) for n in some}
            y = call(c, leaves, name)
            assert torch.equal(y, want["y"])
            for n, g in zip(some, torch.autograd.grad(y, list(leaves.values()), c["gy"])):
                assert torch.equal(g, want["g" + n]), (some, n)


@pytest.mark.parametrize("name", ["silu", "none"])
def test_every_choice_of_gradients_of_a_pair(name):
    import rwkv_infctx_trainer_b200 as W
    c = L.gated_case(2, 60, 72, 48, BF)
    want = L.train_gated(c, name)
    for k in (1, 2, 3):
        for some in itertools.combinations(L.GATED, k):
            leaves = {n: c[n].detach().requires_grad_(True) for n in some}
            y = W.gated_linear(*(leaves.get(n, c[n]) for n in L.GATED), name)
            for n, g in zip(some, torch.autograd.grad(y, list(leaves.values()), c["gy"])):
                assert torch.equal(g, want["g" + n]), (some, n)


def held(make):
    """bytes that a call keeps beside its output"""
    make()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = make()
    return torch.cuda.memory_allocated() - before - y.numel() * y.element_size()


def test_what_is_kept():
    import rwkv_infctx_trainer_b200 as W
    rows, K, N = 4096, 1024, 2048                                 # x 8 MB, the matrix 4, y 16, its pre-activations 32
    c = L.linear_case(3, rows, K, N, BF, mul=True, residual=True)
    grad = lambda t: t.detach().requires_grad_(True)
    x, w, m, r = grad(c["x"]), grad(c["weight"]), grad(c["mul"]), grad(c["residual"])
    of = lambda t: t * 1                                          # an activation of its own: gone if the call does not keep it
    near = lambda n, mb: abs(n - mb * MB) < MB / 4
    with torch.no_grad():
        fx, fm, fr = of(c["x"]), of(c["mul"]), of(c["residual"])
    assert near(held(lambda: W.linear_act(of(x), c["weight"])), 0)                              # a frozen matrix: not its x
    assert near(held(lambda: W.linear_act(of(x), w)), 8)
    assert near(held(lambda: W.linear_act(of(x), c["weight"], None, "silu")), 32)
    assert near(held(lambda: W.linear_act(fx, w, None, "silu")), 32)
    assert near(held(lambda: W.linear_act(fx, c["weight"], None, "silu", fm, of(r))), 0)        # the residual alone
    assert near(held(lambda: W.linear_act(fx, c["weight"], None, "silu", of(m), fr)), 48)       # mul and the pre-activations
    assert near(held(lambda: W.gated_linear(of(x), c["weight"], c["weight"])), 64)
    assert near(held(lambda: W.gated_linear(of(x), w, c["weight"])), 72)


def test_what_is_not_kept_may_change():
    import rwkv_infctx_trainer_b200 as W
    c = L.linear_case(4, 60, 72, 48, BF)
    want = L.train_linear(c, "silu")
    x = c["x"].detach().requires_grad_(True)
    h = x * 1
    y = W.linear_act(h, c["weight"], None, "silu")
    with torch.no_grad():
        h.zero_()
    assert torch.equal(torch.autograd.grad(y, x, c["gy"])[0], want["gx"])
    h, w = c["x"].clone(), c["weight"].detach().requires_grad_(True)
    y = W.linear_act(h, w, None, "silu")
    h.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, w, c["gy"])


def test_saved_on_the_host_and_formed_again():
    """what is kept goes through the hooks for saved tensors, and a call may be made again in the backward pass"""
    import rwkv_infctx_trainer_b200 as W
    from torch.utils.checkpoint import checkpoint
    c, g = L.linear_case(5, 70, 72, 48, BF, bias=True, mul=True, residual=True), L.gated_case(5, 70, 72, 48, BF)
    want, pair = L.train_linear(c, "gelu"), L.train_gated(g, "silu")
    n = lambda *s: torch.randn(s, device="cuda", dtype=BF)
    rec = [n(2, 70, 48), n(2, 70, 48), n(2, 70, 48), torch.randn(48, device="cuda"), n(2, 70, 48), torch.randn(2, 48, device="cuda")]
    seeds = (n(2, 70, 48), torch.randn(2, 48, device="cuda"))

    def recurrence(call):
        leaves = [t.detach().requires_grad_(True) for t in rec]
        return torch.autograd.grad(call(*leaves), leaves, seeds)
    plain = recurrence(W.gated_recurrence)
    again = lambda f: lambda *a: checkpoint(f, *a, use_reentrant=False)
    with torch.autograd.graph.save_on_cpu():
        got, got_pair, got_rec = L.train_linear(c, "gelu"), L.train_gated(g, "silu"), recurrence(W.gated_recurrence)
    for a, b in ((got, want), (got_pair, pair), (dict(enumerate(got_rec)), dict(enumerate(plain))), (dict(enumerate(recurrence(again(W.gated_recurrence)))), dict(enumerate(plain)))):
        for k in b:
            assert torch.equal(a[k], b[k]), k
    leaves = {k: c[k].detach().requires_grad_(True) for k in L.LINEAR}
    y = checkpoint(lambda *a: call(c, dict(zip(L.LINEAR, a)), "gelu"), *leaves.values(), use_reentrant=False)
    for k, t in zip(L.LINEAR, torch.autograd.grad(y, list(leaves.values()), c["gy"])):
        assert torch.equal(t, want["g" + k]), k
