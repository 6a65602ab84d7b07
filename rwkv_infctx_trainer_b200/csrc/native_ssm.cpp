// PyTorch binding of the norm, the short causal convolution and the selective scan (see rms_norm.cu, causal_conv.cu,
// selective_scan.cu): argument checks, allocation, autograd nodes.
#include "native_ops.h"

namespace wkv_native {
namespace {

Tensor opt(const OptTensor &t) { return t.has_value() ? *t : Tensor(); }

int small(int64_t n, const char *what) {
    TORCH_CHECK_VALUE(n <= std::numeric_limits<int>::max(), what, " is too large: ", n);
    return (int)n;
}
void check_type(const Tensor &t, at::ScalarType dt, const char *name) {
    TORCH_CHECK_TYPE(!t.defined() || t.scalar_type() == dt, name, " must be ", dt, ", got ", t.scalar_type());
}
void check_param(const Tensor &t, const char *name) {
    TORCH_CHECK_TYPE(!t.defined() || at::isFloatingType(t.scalar_type()), name, " must be a floating point tensor");
}
void check_sizes(const Tensor &t, at::IntArrayRef want, const char *name) {
    TORCH_CHECK_VALUE(!t.defined() || t.sizes() == want, name, " must have shape ", want, ", got ", t.sizes());
}
// the calls that update a state in place have no backward pass
void refuse_grad(std::initializer_list<const Tensor *> ts, const char *call, const char *other) {
    TORCH_CHECK(!wants_grad(ts), call, " updates the state in place and has no gradient: call it under torch.no_grad(), or ", other);
}
void check_in_place(const Tensor &state, const char *call) {
    TORCH_CHECK_VALUE(state.is_contiguous(), call, ": the state is updated in place and must be contiguous");
}
// Before the launch: torch refuses this for a tensor made in inference mode, outside of it, and then nothing may have changed.
void changes_in_place(const Tensor &state) { torch::autograd::impl::bump_version(state); }

// Rows of adjacent channels with any stride between rows and between tokens, as the kernels take them: a view of a wider
// tensor stays one, anything else is copied.
struct Rows {
    Tensor t;
    int64_t batch = 0, token = 0;
};
// t: [B, T, ...], or [B, ...] for one token, with everything behind one run of `n` elements
Rows rows_of(const Tensor &t, int64_t n, bool one_token) {
    if (!t.defined()) return {};
    const int64_t lead = one_token ? 1 : 2;
    const auto sizes = t.sizes(), strides = t.strides();
    int64_t run = 1;
    bool packed = true;
    for (int64_t i = t.dim() - 1; i >= lead; i--) {
        if (sizes[i] != 1 && strides[i] != run) packed = false;
        run *= sizes[i];
    }
    // (offsets inside a block of tokens are 32-bit, and a dimension of one element may have any stride)
    if (!one_token && sizes[1] > 1 && strides[1] > (1 << 26)) packed = false;
    const Tensor c = packed ? t : t.contiguous();
    const int64_t token = one_token || c.size(1) <= 1 ? n : c.stride(1);
    return {c, c.size(0) > 1 ? c.stride(0) : token, token};
}

// ------------------------------------------------------------------------------ norm
struct NormCall {
    Tensor x, residual, weight;
    wkv_rms_norm_args_t a = {};
};
void check_norm(const Tensor &x, const Tensor &weight, const Tensor &residual) {
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 16384, "x must be [..., C] with 1 <= C <= 16384, got ", x.sizes());
    dtype_code(x.scalar_type());
    check_param(weight, "weight");
    check_sizes(weight, {x.size(-1)}, "weight");
    check_sizes(residual, x.sizes(), "residual");
    TORCH_CHECK_TYPE(!residual.defined() || residual.scalar_type() == x.scalar_type() || residual.scalar_type() == at::kFloat,
                     "residual must be float32 or of x's type");
}
NormCall norm_call(const Tensor &x, const Tensor &weight, const Tensor &residual, double eps) {
    NormCall c;
    c.x = contig(x);
    c.weight = as_contig(weight, param_type(weight));
    if (residual.defined()) c.residual = contig(residual);
    c.a.C = (int)x.size(-1);
    c.a.rows = x.numel() / x.size(-1);
    c.a.dtype = dtype_code(x.scalar_type());
    c.a.res_dtype = residual.defined() ? dtype_code(residual.scalar_type()) : c.a.dtype;
    c.a.w_dtype = dtype_code(c.weight.scalar_type());
    c.a.eps = (float)eps;
    c.a.x = ptr(c.x); c.a.residual = ptr(c.residual); c.a.weight = ptr(c.weight);
    return c;
}

struct RmsNormBackward : OpNode {
    bool has_residual;
    double eps;
    at::ScalarType x_type, w_type;
    std::string name() const override { return "RmsNormBackward"; }
    variable_list gradients(variable_list &&grads) override {
        at::AutoDispatchBelowADInplaceOrView below;
        const variable_list st = unpack();
        // (a saved-tensor hook may hand back another layout)
        auto again = [](const Tensor &t) { return t.defined() ? contig(t) : t; };
        const Tensor weight = again(st[0]), x = again(st[1]), residual = again(st[2]), kept = again(st[3]);
        const Tensor &h = kept.defined() ? kept : residual.defined() ? residual : x;      // (of h's size and type)
        c10::cuda::OptionalCUDAGuard guard(h.device());
        const Tensor gy = grads[0].defined() ? as_contig(grads[0], x_type) : Tensor();
        const Tensor gh = has_residual && grads[1].defined() ? as_contig(grads[1], h.scalar_type()) : Tensor();
        const bool want_x = task_should_compute_output(0), want_w = task_should_compute_output(1),
                   want_r = has_residual && task_should_compute_output(2), shared = h.scalar_type() == x_type;
        Tensor gx, gres, gw, ws;
        if (want_x || (want_r && shared)) gx = fresh(h.sizes(), x_type, h);
        if (want_r && !shared) gres = fresh_like(h);
        if (want_w) gw = fresh(weight.sizes(), weight.scalar_type(), weight);
        wkv_rms_norm_args_t a = {};
        a.C = (int)h.size(-1);
        a.rows = h.numel() / h.size(-1);
        a.dtype = dtype_code(x_type); a.res_dtype = dtype_code(h.scalar_type()); a.w_dtype = dtype_code(weight.scalar_type());
        a.eps = (float)eps;
        a.weight = ptr(weight); a.x = ptr(x); a.residual = ptr(residual); a.h = ptr(kept); a.gy = ptr(gy); a.gh = ptr(gh);
        a.gx = ptr(gx); a.gresidual = ptr(gres); a.gweight = ptr(gw);
        if (want_w) {
            a.workspace_bytes = wkv_rms_norm_backward_workspace(&a);
            ws = bytes_like(h, a.workspace_bytes);
            a.workspace = ptr(ws);
        }
        check(wkv_rms_norm_backward(&a, stream_of(h)), "wkv_rms_norm_backward");
        // (of one type, the two are the same values: one tensor, as for an addition)
        return {want_x ? gx : Tensor(), want_w ? as_input(gw, w_type, weight.sizes()) : gw, want_r && shared ? gx : gres};
    }
};

variable_list rms_norm(const Tensor &x, const Tensor &weight, const OptTensor &residual_, double eps) {
    const Tensor residual = opt(residual_);
    check_norm(x, weight, residual);
    require_cuda({&x, &weight, &residual});
    c10::cuda::OptionalCUDAGuard guard(x.device());
    const bool save = wants_grad({&x, &weight, &residual});
    std::shared_ptr<RmsNormBackward> node;
    if (save) {
        node = make_node<RmsNormBackward>({x, weight, residual});
        node->has_residual = residual.defined();
        node->eps = eps;
        node->x_type = x.scalar_type();
        node->w_type = weight.scalar_type();
    }
    Tensor y, h;
    NormCall c;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        c = norm_call(x, weight, residual, eps);
        y = fresh_like(c.x);
        if (residual.defined()) h = fresh_like(c.residual);
        c.a.y = ptr(y); c.a.h = ptr(h);
        check(wkv_rms_norm_forward(&c.a, stream_of(x)), "wkv_rms_norm_forward");
    }
    if (save) {
        // An fp32 h serves the backward pass as well as its terms; it is an output of the node: kept as an alias that has no
        // history (and whose in-place changes are noticed).
        if (h.defined() && h.scalar_type() == at::kFloat) node->keep({c.weight, Tensor(), Tensor(), h.detach()});
        else node->keep({c.weight, c.x, c.residual, Tensor()});
        torch::autograd::set_history(y, node);
        if (h.defined()) torch::autograd::set_history(h, node);
    }
    if (h.defined()) return {y, h};
    return {y};
}

variable_list rms_norm_q8(const Tensor &x, const Tensor &weight, const OptTensor &residual_, double eps, c10::optional<int64_t> group) {
    const Tensor residual = opt(residual_);
    check_norm(x, weight, residual);
    const int64_t gr = group.value_or(0);
    TORCH_CHECK_VALUE(!group.has_value() || gr == 32 || gr == 64 || gr == 128 || gr == 256, "group must be None, 32, 64, 128 or 256, got ", gr);
    TORCH_CHECK(!wants_grad({&x, &weight, &residual}), "rms_norm_q8 has no gradient: call it under torch.no_grad(), or rms_norm");
    require_cuda({&x, &weight, &residual});
    c10::cuda::OptionalCUDAGuard guard(x.device());
    NormCall c = norm_call(x, weight, residual, eps);
    Tensor q = fresh(x.sizes(), at::kFloat8_e4m3fn, x), h;
    auto sizes = x.sizes().vec();
    sizes.back() = gr ? (c.a.C + gr - 1) / gr : 1;
    Tensor scale = fresh(sizes, at::kFloat, x);
    if (residual.defined()) h = fresh_like(c.residual);
    c.a.y = ptr(q); c.a.h = ptr(h); c.a.scale = (float *)ptr(scale);
    c.a.group = (int)gr;
    if (c.a.rows > 0) check(wkv_rms_norm_forward(&c.a, stream_of(x)), "wkv_rms_norm_forward");
    if (h.defined()) return {q, scale, h};
    return {q, scale};
}

// ------------------------------------------------------------------------------ convolution
struct ConvCall {
    Rows x;
    Tensor weight, bias, state;
    wkv_causal_conv_args_t a = {};
};
// x [B,T,D], weight [D,W] (or [D,1,W], as a depthwise nn.Conv1d has it), bias [D], state [B,W-1,D]
void check_conv(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &state, int64_t B, int64_t D) {
    dtype_code(x.scalar_type());
    check_param(weight, "weight");
    check_param(bias, "bias");
    TORCH_CHECK_VALUE((weight.dim() == 2 || (weight.dim() == 3 && weight.size(1) == 1)) && weight.size(0) == D && weight.size(-1) >= 2 && weight.size(-1) <= 4,
                      "weight must be [D,W] or [D,1,W] with D = ", D, " and W = 2, 3 or 4, got ", weight.sizes());
    check_sizes(bias, {D}, "bias");
    check_sizes(state, {B, weight.size(-1) - 1, D}, "state");
}
// sizes: [B,T,D], or [B,D] for one token
ConvCall conv_call(const Rows &x, at::IntArrayRef sizes, const Tensor &weight, const Tensor &bias, const Tensor &state, bool silu) {
    ConvCall c;
    c.x = x;
    const auto pt = bias.defined() && bias.scalar_type() != weight.scalar_type() ? at::kFloat : param_type(weight);
    c.weight = as_contig(weight, pt);
    if (bias.defined()) c.bias = as_contig(bias, pt);
    if (state.defined()) c.state = as_contig(state, x.t.scalar_type());
    c.a.B = small(sizes[0], "B"); c.a.T = sizes.size() == 2 ? 1 : small(sizes[1], "T"); c.a.D = small(sizes.back(), "D");
    c.a.W = (int)weight.size(-1);
    c.a.dtype = dtype_code(x.t.scalar_type()); c.a.w_dtype = dtype_code(pt);
    c.a.silu = silu;
    c.a.x_batch = x.batch; c.a.x_token = x.token;
    c.a.x = ptr(x.t); c.a.weight = ptr(c.weight); c.a.bias = ptr(c.bias); c.a.state_in = ptr(c.state);
    return c;
}

struct CausalConvBackward : OpNode {
    bool silu;
    at::ScalarType w_type, b_type, s_type;
    std::vector<int64_t> w_shape;
    std::string name() const override { return "CausalConvBackward"; }
    variable_list gradients(variable_list &&grads) override {
        at::AutoDispatchBelowADInplaceOrView below;
        const variable_list st = unpack();
        const Tensor &x = st[0];
        c10::cuda::OptionalCUDAGuard guard(x.device());
        ConvCall c = conv_call(rows_of(x, x.size(2), false), x.sizes(), st[1], st[2], st[3], silu);
        const auto dt = x.scalar_type(), pt = c.weight.scalar_type();
        const int64_t B = x.size(0), D = x.size(2), W = c.a.W;
        const Tensor gy = grads[0].defined() ? as_contig(grads[0], dt) : Tensor(), gs = grads[1].defined() ? as_contig(grads[1], dt) : Tensor();
        Tensor gx, gw, gb, gs_in, ws;
        if (task_should_compute_output(0)) gx = fresh(x.sizes(), dt, x);
        if (task_should_compute_output(1)) gw = fresh({D, W}, pt, x);
        if (task_should_compute_output(2)) gb = fresh({D}, pt, x);
        if (task_should_compute_output(3)) gs_in = fresh({B, W - 1, D}, dt, x);
        c.a.gy = ptr(gy); c.a.gstate_out = ptr(gs);
        c.a.gx = ptr(gx); c.a.gweight = ptr(gw); c.a.gbias = ptr(gb); c.a.gstate_in = ptr(gs_in);
        if (gw.defined() || gb.defined()) {
            c.a.workspace_bytes = wkv_causal_conv_backward_workspace(&c.a);
            ws = bytes_like(x, c.a.workspace_bytes);
            c.a.workspace = ptr(ws);
        }
        check(wkv_causal_conv_backward(&c.a, stream_of(x)), "wkv_causal_conv_backward");
        return {gx, as_input(gw, w_type, w_shape), as_input(gb, b_type, {D}), gs_in.defined() ? gs_in.to(s_type) : gs_in};
    }
};

std::tuple<Tensor, Tensor> causal_conv(const Tensor &x, const Tensor &weight, const OptTensor &bias_, const OptTensor &state_, bool silu) {
    const Tensor bias = opt(bias_), state = opt(state_);
    TORCH_CHECK_VALUE(x.dim() == 3, "x must be [B,T,D], got ", x.sizes());
    check_conv(x, weight, bias, state, x.size(0), x.size(2));
    if (state.defined()) dtype_code(state.scalar_type());
    require_cuda({&x, &weight, &bias, &state});
    c10::cuda::OptionalCUDAGuard guard(x.device());
    const bool save = wants_grad({&x, &weight, &bias, &state});
    std::shared_ptr<CausalConvBackward> node;
    if (save) {
        node = make_node<CausalConvBackward>({x, weight, bias, state});
        node->silu = silu;
        node->w_type = weight.scalar_type();
        node->b_type = bias.defined() ? bias.scalar_type() : weight.scalar_type();
        node->s_type = state.defined() ? state.scalar_type() : x.scalar_type();
        node->w_shape = weight.sizes().vec();
    }
    Tensor y, s;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        ConvCall c = conv_call(rows_of(x, x.size(2), false), x.sizes(), weight, bias, state, silu);
        y = fresh(x.sizes(), x.scalar_type(), x);
        s = fresh({x.size(0), c.a.W - 1, x.size(2)}, x.scalar_type(), x);
        c.a.y = ptr(y); c.a.state_out = ptr(s);
        check(wkv_causal_conv_forward(&c.a, stream_of(x)), "wkv_causal_conv_forward");
        if (save) node->keep({c.x.t, c.weight, c.bias, c.state});
    }
    if (save) {
        torch::autograd::set_history(y, node);
        torch::autograd::set_history(s, node);
    }
    return {y, s};
}

Tensor causal_conv_step(const Tensor &x, const Tensor &state, const Tensor &weight, const OptTensor &bias_, bool silu) {
    const Tensor bias = opt(bias_);
    TORCH_CHECK_VALUE(x.dim() == 2, "x must be [B,D], got ", x.sizes());
    check_conv(x, weight, bias, state, x.size(0), x.size(1));
    check_type(state, x.scalar_type(), "state");
    check_in_place(state, "causal_conv_step");
    refuse_grad({&x, &state, &weight, &bias}, "causal_conv_step", "causal_conv");
    require_cuda({&x, &state, &weight, &bias});
    c10::cuda::OptionalCUDAGuard guard(x.device());
    ConvCall c = conv_call(rows_of(x, x.size(1), true), x.sizes(), weight, bias, state, silu);
    Tensor y = fresh(x.sizes(), x.scalar_type(), x);
    c.a.y = ptr(y); c.a.state_out = ptr(state);
    changes_in_place(state);
    check(wkv_causal_conv_forward(&c.a, stream_of(x)), "wkv_causal_conv_forward");
    return y;
}

// ------------------------------------------------------------------------------ selective scan
struct ScanCall {
    Rows u, delta, B, C, z;
    Tensor A, D, bias, state;
    wkv_selective_scan_args_t a = {};
};
// u, delta, z [B,T,D]; A [D,N]; B, C [B,T,N] or [B,T,G,N]; D, delta_bias [D]; state [B,D,N]; for one token without T
void check_scan(const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &Bm, const Tensor &Cm, const Tensor &D, const Tensor &z,
                const Tensor &bias, const Tensor &state) {
    const auto dt = u.scalar_type();
    dtype_code(dt);
    for (auto [t, name] : {std::pair<const Tensor *, const char *>{&delta, "delta"}, {&Bm, "B"}, {&Cm, "C"}, {&z, "z"}}) check_type(*t, dt, name);
    for (auto [t, name] : {std::pair<const Tensor *, const char *>{&A, "A"}, {&D, "D"}, {&bias, "delta_bias"}, {&state, "state"}}) check_param(*t, name);
    const bool one = u.dim() == 2;
    const int64_t B = u.size(0), T = one ? 1 : u.size(1), d = u.size(-1);
    TORCH_CHECK_VALUE(A.dim() == 2 && A.size(0) == d && A.size(1) >= 1 && A.size(1) <= 64, "A must be [D,N] with D = ", d, " and 1 <= N <= 64, got ", A.sizes());
    const int64_t N = A.size(1);
    check_sizes(delta, u.sizes(), "delta");
    check_sizes(z, u.sizes(), "z");
    check_sizes(D, {d}, "D");
    check_sizes(bias, {d}, "delta_bias");
    check_sizes(state, {B, d, N}, "state");
    const int64_t lead = one ? 1 : 2, G = Bm.dim() == lead + 2 ? Bm.size(lead) : 1;
    TORCH_CHECK_VALUE(G >= 1 && d % G == 0, "the groups of B must divide the channels: ", G, " of ", d);
    TORCH_CHECK_VALUE((Bm.dim() == lead + 1 || Bm.dim() == lead + 2) && Bm.size(0) == B && (one || Bm.size(1) == T) && Bm.size(-1) == N,
                      one ? "B must be [B,N] or [B,G,N], got " : "B must be [B,T,N] or [B,T,G,N], got ", Bm.sizes());
    check_sizes(Cm, Bm.sizes(), "C");
    require_cuda({&u, &delta, &A, &Bm, &Cm, &D, &z, &bias, &state});
}
ScanCall scan_call(const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &Bm, const Tensor &Cm, const Tensor &D, const Tensor &z,
                   const Tensor &bias, const Tensor &state, bool softplus) {
    ScanCall c;
    const bool one = u.dim() == 2;
    const int64_t lead = one ? 1 : 2, d = u.size(-1), N = A.size(1), G = Bm.dim() == lead + 2 ? Bm.size(lead) : 1;
    c.u = rows_of(u, d, one); c.delta = rows_of(delta, d, one); c.z = rows_of(z, d, one);
    c.B = rows_of(Bm, G * N, one); c.C = rows_of(Cm, G * N, one);
    c.A = as_contig(A, at::kFloat);
    if (D.defined()) c.D = as_contig(D, at::kFloat);
    if (bias.defined()) c.bias = as_contig(bias, at::kFloat);
    if (state.defined()) c.state = as_contig(state, at::kFloat);
    wkv_selective_scan_args_t &a = c.a;
    a.B = small(u.size(0), "B"); a.T = one ? 1 : small(u.size(1), "T"); a.D = small(d, "D"); a.N = (int)N; a.G = (int)G;
    a.dtype = dtype_code(u.scalar_type()); a.softplus = softplus;
    a.u = ptr(c.u.t); a.delta = ptr(c.delta.t); a.Bm = ptr(c.B.t); a.Cm = ptr(c.C.t); a.z = ptr(c.z.t);
    a.u_batch = c.u.batch; a.u_token = c.u.token; a.delta_batch = c.delta.batch; a.delta_token = c.delta.token;
    a.B_batch = c.B.batch; a.B_token = c.B.token; a.C_batch = c.C.batch; a.C_token = c.C.token;
    a.z_batch = c.z.batch; a.z_token = c.z.token;
    a.A = (const float *)ptr(c.A); a.Dskip = (const float *)ptr(c.D); a.delta_bias = (const float *)ptr(c.bias);
    a.state_in = (const float *)ptr(c.state);
    return c;
}

struct SelectiveScanBackward : OpNode {
    bool softplus;
    at::ScalarType A_type, D_type, bias_type, s_type;
    std::string name() const override { return "SelectiveScanBackward"; }
    variable_list gradients(variable_list &&grads) override {
        at::AutoDispatchBelowADInplaceOrView below;
        const variable_list st = unpack();
        const Tensor &u = st[0], &A = st[2], &Bm = st[3];
        const Tensor ckpt = st[8].defined() ? contig(st[8]) : st[8];
        c10::cuda::OptionalCUDAGuard guard(u.device());
        ScanCall c = scan_call(u, st[1], A, Bm, st[4], st[5], st[6], st[7], Tensor(), softplus);
        const auto dt = u.scalar_type();
        const int64_t B = u.size(0), D = u.size(2), N = A.size(1);
        const Tensor gy = grads[0].defined() ? as_contig(grads[0], dt) : Tensor(), gs = grads[1].defined() ? as_contig(grads[1], at::kFloat) : Tensor();
        auto want = [&](size_t i, at::IntArrayRef sizes, at::ScalarType t) { return task_should_compute_output(i) ? fresh(sizes, t, u) : Tensor(); };
        Tensor gu = want(0, u.sizes(), dt), gdelta = want(1, u.sizes(), dt), gA = want(2, {D, N}, at::kFloat), gB = want(3, Bm.sizes(), dt),
               gC = want(4, Bm.sizes(), dt), gD = want(5, {D}, at::kFloat), gz = want(6, u.sizes(), dt), gbias = want(7, {D}, at::kFloat),
               gstate = want(8, {B, D, N}, at::kFloat);
        wkv_selective_scan_args_t &a = c.a;
        a.gy = ptr(gy); a.gstate_out = (const float *)ptr(gs);
        a.gu = ptr(gu); a.gdelta = ptr(gdelta); a.gz = ptr(gz); a.gB = ptr(gB); a.gC = ptr(gC);
        a.gA = (float *)ptr(gA); a.gD = (float *)ptr(gD); a.gbias = (float *)ptr(gbias); a.gstate_in = (float *)ptr(gstate);
        a.ckpt = ptr(ckpt);
        a.ckpt_bytes = ckpt.defined() ? (size_t)ckpt.numel() : 0;
        a.workspace_bytes = wkv_selective_scan_backward_workspace(&a);
        Tensor ws = bytes_like(u, a.workspace_bytes);
        a.workspace = ptr(ws);
        check(wkv_selective_scan_backward(&a, stream_of(u)), "wkv_selective_scan_backward");
        auto as = [](const Tensor &g, at::ScalarType t) { return g.defined() ? g.to(t) : g; };
        return {gu, gdelta, as(gA, A_type), gB, gC, as(gD, D_type), gz, as(gbias, bias_type), as(gstate, s_type)};
    }
};

std::tuple<Tensor, Tensor> selective_scan(const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &Bm, const Tensor &Cm,
                                          const OptTensor &D_, const OptTensor &z_, const OptTensor &bias_, bool softplus,
                                          const OptTensor &state_) {
    const Tensor D = opt(D_), z = opt(z_), bias = opt(bias_), state = opt(state_);
    TORCH_CHECK_VALUE(u.dim() == 3, "u must be [B,T,D], got ", u.sizes());
    check_scan(u, delta, A, Bm, Cm, D, z, bias, state);
    c10::cuda::OptionalCUDAGuard guard(u.device());
    const bool save = wants_grad({&u, &delta, &A, &Bm, &Cm, &D, &z, &bias, &state});
    std::shared_ptr<SelectiveScanBackward> node;
    if (save) {
        node = make_node<SelectiveScanBackward>({u, delta, A, Bm, Cm, D, z, bias, state});
        node->softplus = softplus;
        auto type_of = [](const Tensor &t) { return t.defined() ? t.scalar_type() : at::kFloat; };
        node->A_type = type_of(A); node->D_type = type_of(D); node->bias_type = type_of(bias); node->s_type = type_of(state);
    }
    Tensor y, s;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        ScanCall c = scan_call(u, delta, A, Bm, Cm, D, z, bias, state, softplus);
        y = fresh(u.sizes(), u.scalar_type(), u);
        s = fresh({u.size(0), u.size(2), A.size(1)}, at::kFloat, u);
        c.a.y = ptr(y); c.a.state_out = (float *)ptr(s);
        Tensor ckpt;
        if (save) {
            c.a.ckpt_bytes = wkv_selective_scan_ckpt_bytes(&c.a);
            ckpt = bytes_like(u, c.a.ckpt_bytes);
            c.a.ckpt = ptr(ckpt);
        }
        c.a.workspace_bytes = wkv_selective_scan_forward_workspace(&c.a);
        Tensor ws = bytes_like(u, c.a.workspace_bytes);
        c.a.workspace = ptr(ws);
        check(wkv_selective_scan_forward(&c.a, stream_of(u)), "wkv_selective_scan_forward");
        if (save) node->keep({c.u.t, c.delta.t, c.A, c.B.t, c.C.t, c.D, c.z.t, c.bias, ckpt});
    }
    if (save) {
        torch::autograd::set_history(y, node);
        torch::autograd::set_history(s, node);
    }
    return {y, s};
}

Tensor selective_scan_step(const Tensor &u, const Tensor &delta, const Tensor &A, const Tensor &Bm, const Tensor &Cm, const Tensor &state,
                           const OptTensor &D_, const OptTensor &z_, const OptTensor &bias_, bool softplus) {
    const Tensor D = opt(D_), z = opt(z_), bias = opt(bias_);
    TORCH_CHECK_VALUE(u.dim() == 2, "u must be [B,D], got ", u.sizes());
    refuse_grad({&u, &delta, &A, &Bm, &Cm, &D, &z, &bias, &state}, "selective_scan_step", "selective_scan");
    check_type(state, at::kFloat, "state");
    check_in_place(state, "selective_scan_step");
    check_scan(u, delta, A, Bm, Cm, D, z, bias, state);
    c10::cuda::OptionalCUDAGuard guard(u.device());
    ScanCall c = scan_call(u, delta, A, Bm, Cm, D, z, bias, state, softplus);
    Tensor y = fresh(u.sizes(), u.scalar_type(), u);
    c.a.y = ptr(y); c.a.state_out = (float *)ptr(state);
    changes_in_place(state);
    check(wkv_selective_scan_forward(&c.a, stream_of(u)), "wkv_selective_scan_forward");
    return y;
}

}  // namespace
}  // namespace wkv_native

void bind_ssm(py::module_ &m) {
    using namespace wkv_native;
    m.def("rms_norm", &rms_norm);
    m.def("rms_norm_q8", &rms_norm_q8);
    m.def("causal_conv", &causal_conv);
    m.def("causal_conv_step", &causal_conv_step);
    m.def("selective_scan", &selective_scan);
    m.def("selective_scan_step", &selective_scan_step);
}
