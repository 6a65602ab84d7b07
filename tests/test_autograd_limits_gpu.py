"""What the operators' autograd nodes do not have, second derivatives and forward-mode derivatives, is refused: nothing is
dropped in silence."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
B, T, C, N = 2, 20, 64, 16


def n(*shape, dtype=BF, seed=[0]):
    seed[0] += 1
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed[0])).to(dtype).cuda()


def time_mix(version):
    import rwkv_infctx_trainer_b200 as W
    torch.manual_seed(version)
    if version == 4:
        m = W.RWKV_TimeMix_v4(0, 2, C, C).cuda().to(BF)
        return lambda x, shift, state: (lambda o: (o[0], o[1].shift_state, o[1].wkv_state))(m(x, W.TimeMixState(shift, state)))
    m = (W.RWKV_TimeMix if version == 5 else W.RWKV_TimeMix6_0)(0, 2, C, 1, 64, C).cuda().to(BF)
    return lambda x, shift, state: (lambda o: (o[0], *o[1]))(m(x, (shift, state)))


def ops():
    """name -> (call, inputs that are all differentiable)"""
    import rwkv_infctx_trainer_b200 as W
    rows = lambda k: [n(B, T, C) for _ in range(k)]
    s64 = n(B, 1, 64, 64, dtype=F32)
    return {
        "rms_norm": (lambda x, w, r: W.rms_norm(x, w, r), [n(B, T, C), n(C, dtype=F32), n(B, T, C)]),
        "rms_norm, no residual": (lambda x, w: (W.rms_norm(x, w),), [n(B, T, C), n(C, dtype=F32)]),
        "causal_conv": (lambda x, w, b, s: W.causal_conv(x, w, b, s), [n(B, T, C), n(C, 4, dtype=F32), n(C, dtype=F32), n(B, 3, C)]),
        "selective_scan": (lambda u, d, A, b, c, D, z, s: W.selective_scan(u, d, -A.abs(), b, c, D, z, state=s),
                           [*rows(2), n(C, N, dtype=F32), n(B, T, N), n(B, T, N), n(C, dtype=F32), n(B, T, C), n(B, C, N, dtype=F32)]),
        "WKV6": (lambda r, k, v, w, u, s: W.wkv6(r, k, v, w, u, s), [*rows(4), n(1, 64), s64]),
        "WKV5": (lambda r, k, v, w, u, s: W.wkv5(r, k, v, w, u, s), [*rows(3), torch.rand(C).cuda() * 0.9 + 0.05, n(1, 64), s64]),
        "WKV6STATE_CUDA": (lambda r, k, v, w, u, s: (W.WKV6STATE_CUDA.apply(B, T, C, 1, r, k, v, w, u, s.clone()),), [*rows(4), n(1, 64), s64]),
        "wkv (v4)": (lambda w, u, k, v, s: W.wkv(w, u, k, v, s), [n(C, dtype=F32), n(C), *rows(2), n(B, C, 3, dtype=F32)]),
        "lnx_gate": (lambda y, g, w, b: (W.lnx_gate(y, g, w, b, 1e-5, 1),), [*rows(2), n(C), n(C)]),
        "ddlerp": (lambda x, s, m, d: (W.ddlerp(x, s, m, d),), [n(B, T, C), n(B, C), n(3, C), n(3, B, T, C)]),
        "time mix v4": (time_mix(4), [n(B, T, C), n(B, C), n(B, C, 3, dtype=F32)]),
        "time mix v5": (time_mix(5), [n(B, T, C), n(B, C), s64]),
        "time mix v6": (time_mix(6), [n(B, T, C), n(B, C), s64]),
    }


NAMES = ["rms_norm", "rms_norm, no residual", "causal_conv", "selective_scan", "WKV6", "WKV5", "WKV6STATE_CUDA", "wkv (v4)", "lnx_gate",
         "ddlerp", "time mix v4", "time mix v5", "time mix v6"]


@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives_are_refused(name):
    """a graph of the gradients is made on demand, with the bits that the gradients have without; whoever differentiates it is told"""
    call, ins = ops()[name]
    leaves = [t.requires_grad_(True) for t in ins]
    out = [o for o in call(*leaves) if o.requires_grad]
    seeds = [torch.randn_like(o) for o in out]
    used = torch.autograd.grad(out, leaves, seeds, retain_graph=True, allow_unused=True)
    want = [g for g in used if g is not None]
    leaves = [t for t, g in zip(leaves, used) if g is not None]
    got = torch.autograd.grad(out, leaves, seeds, create_graph=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b) and a.requires_grad
    # a penalty on a gradient beside another term, for each gradient and each leaf
    for g in got:
        for leaf in leaves:
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad(g.float().square().sum() + leaf.float().sum(), leaf, retain_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            (g.float().square().sum() + leaves[0].float().sum()).backward(retain_graph=True)
    # through the incoming gradient alone
    gy = [s.clone().requires_grad_(True) for s in seeds]
    g = torch.autograd.grad(out, leaves, gy, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(g.float().sum() + gy[0].float().sum(), gy[0])


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name):
    call, ins = ops()[name]
    for grad in (True, False):
        for i, t in enumerate(ins):
            with torch.set_grad_enabled(grad), fwAD.dual_level():
                duals = [x.detach().clone() for x in ins]
                duals[i] = fwAD.make_dual(duals[i], torch.ones_like(t))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*duals)
    call(*ins)


def test_forward_mode_is_refused_by_calls_without_gradients():
    import rwkv_infctx_trainer_b200 as W
    with torch.no_grad(), fwAD.dual_level():
        x, s, w = n(B, C), n(B, 3, C), n(C, 4, dtype=F32)
        dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))
        with pytest.raises(RuntimeError, match="forward-mode"):
            W.causal_conv_step(dual(x), s, w)
        with pytest.raises(RuntimeError, match="forward-mode"):
            W.rms_norm_q8(dual(x), n(C, dtype=F32))
        with pytest.raises(RuntimeError, match="forward-mode"):
            W.selective_scan_step(x, dual(n(B, C)), n(C, N, dtype=F32), n(B, N), n(B, N), n(B, C, N, dtype=F32))


def test_parameters_of_a_block_in_forward_mode():
    import rwkv_infctx_trainer_b200 as W
    m = W.RWKV_TimeMix6_0(0, 2, C, 1, 64, C).cuda().to(BF)
    with fwAD.dual_level():
        p = fwAD.make_dual(m.time_maa_k.detach().clone(), torch.ones_like(m.time_maa_k))
        del m.time_maa_k
        m.time_maa_k = p
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                m(n(B, T, C), (n(B, C), n(B, 1, 64, 64, dtype=F32)))
