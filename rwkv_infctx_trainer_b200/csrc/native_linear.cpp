// PyTorch binding of the matrix products with their epilogue (linear.cu): argument checks, allocation, autograd nodes.
#include "native_args.h"

namespace wkv_native {
namespace {

int act_code(const std::string &name) {
    if (name == "none") return WKV_ACT_NONE;
    if (name == "silu") return WKV_ACT_SILU;
    if (name == "gelu") return WKV_ACT_GELU;
    if (name == "relu2") return WKV_ACT_RELU2;
    if (name == "sigmoid") return WKV_ACT_SIGMOID;
    TORCH_CHECK_VALUE(false, "activation must be 'none', 'silu', 'gelu', 'relu2' or 'sigmoid', got '", name, "'");
    return -1;
}

// Rows of adjacent elements a fixed stride apart, as the kernels take them; anything else is copied.
struct Mat {
    Tensor t;
    int64_t rows = 0, row = 0;
};
Mat matrix_of(const Tensor &t) {
    const int64_t C = t.size(-1);
    const auto sizes = t.sizes(), strides = t.strides();
    Mat m;
    m.rows = C ? t.numel() / C : 0;
    bool ok = C <= 1 || strides[t.dim() - 1] == 1;
    int64_t row = -1, run = 1;                       // the stride between rows, and rows of the dimensions looked at
    for (int64_t i = t.dim() - 2; ok && i >= 0; i--) {
        if (sizes[i] == 1) continue;
        if (row < 0) row = strides[i];
        else ok = strides[i] == row * run;
        run *= sizes[i];
    }
    if (row < 0) row = C;
    ok = ok && (row >= C || m.rows <= 1);            // (rows that overlap, one row for all: a copy)
    m.t = ok ? t : t.contiguous();
    m.row = ok ? row : C;
    return m;
}

struct LinearCall {
    Mat x, w0, w1;
    Tensor bias, mul, residual;
    wkv_linear_args_t a = {};
};
void check_matrix(const Tensor &w, const Tensor &x, const char *name) {
    check_type(w, x.scalar_type(), name);
    TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) >= 1 && w.size(1) == x.size(-1), name, " must be [N,K] with K = ", x.size(-1), ", got ", w.sizes());
}
void check_x(const Tensor &x) {
    TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "x must be bfloat16 or float16, got ", x.scalar_type());
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must be [..., K] with K >= 1, got ", x.sizes());
}
std::vector<int64_t> out_sizes(const Tensor &x, int64_t N) {
    auto s = x.sizes().vec();
    s.back() = N;
    return s;
}
LinearCall linear_call(const Tensor &x, const Tensor &w0, const Tensor &w1, const Tensor &bias, const Tensor &mul, const Tensor &residual, int act) {
    LinearCall c;
    c.x = matrix_of(x);
    c.w0 = matrix_of(w0);
    if (w1.defined()) c.w1 = matrix_of(w1);
    if (bias.defined()) c.bias = as_contig(bias, param_type(bias));
    if (mul.defined()) c.mul = contig(mul);
    if (residual.defined()) c.residual = contig(residual);
    wkv_linear_args_t &a = c.a;
    a.rows = c.x.rows; a.K = x.size(-1); a.N = w0.size(0);
    a.dtype = dtype_code(x.scalar_type()); a.bias_dtype = bias.defined() ? dtype_code(c.bias.scalar_type()) : a.dtype;
    a.act = act; a.pair = w1.defined();
    a.x = ptr(c.x.t); a.w0 = ptr(c.w0.t); a.w1 = ptr(c.w1.t); a.bias = ptr(c.bias); a.mul = ptr(c.mul); a.residual = ptr(c.residual);
    a.x_row = c.x.row; a.w0_row = c.w0.row; a.w1_row = c.w1.row;
    a.status = status_word(x.device().index());
    return c;
}

// What is kept depends on which gradients are wanted: x for those of the matrices, the matrices for that of x, mul and the pre-activations for any but the
// residual's.  (A frozen matrix' x may go, or change, before the backward pass.)
struct LinearBackward : OpNode {
    int act;
    bool pair;
    int64_t rows, K, N;
    std::vector<int64_t> x_sizes;
    at::ScalarType b_type, b_kept;
    std::string name() const override { return pair ? "GatedLinearBackward" : "LinearActBackward"; }
    // inputs: x, w0, then of a pair w1, else bias, mul, residual
    variable_list gradients(variable_list &&grads) override {
        at::AutoDispatchBelowADInplaceOrView below;
        const variable_list st = unpack();
        if (!grads[0].defined()) return variable_list(pair ? 3 : 5);
        const Tensor gy = contig(grads[0]);
        auto want = [&](size_t i) { return task_should_compute_output(i); };
        auto matrix = [&](const Tensor &t) { return t.defined() ? matrix_of(t) : Mat(); };
        const Mat x = matrix(st[0]), w0 = matrix(st[1]), w1 = matrix(st[2]);
        const Tensor mul = st[3].defined() ? contig(st[3]) : st[3], saved = st[4].defined() ? contig(st[4]) : st[4];
        const auto dt = gy.scalar_type();
        c10::cuda::OptionalCUDAGuard guard(gy.device());
        poll_status(gy.device().index(), false);
        Tensor gx, gw0, gw1, gb, gm;
        if (want(0)) gx = fresh(x_sizes, dt, gy);
        if (want(1)) gw0 = fresh({N, K}, dt, gy);
        if (pair && want(2)) gw1 = fresh({N, K}, dt, gy);
        if (!pair && want(2)) gb = fresh({N}, b_kept, gy);
        if (!pair && want(3)) gm = fresh(gy.sizes(), dt, gy);
        wkv_linear_args_t a = {};
        a.rows = rows; a.K = K; a.N = N;
        a.dtype = dtype_code(dt); a.bias_dtype = dtype_code(b_kept);
        a.act = act; a.pair = pair;
        a.x = ptr(x.t); a.w0 = ptr(w0.t); a.w1 = ptr(w1.t); a.mul = ptr(mul);
        a.x_row = x.row; a.w0_row = w0.row; a.w1_row = w1.row;
        a.status = status_word(gy.device().index());
        a.gy = ptr(gy); a.gx = ptr(gx); a.gw0 = ptr(gw0); a.gw1 = ptr(gw1); a.gbias = ptr(gb); a.gmul = ptr(gm);
        a.saved = ptr(saved);
        a.saved_bytes = saved.defined() ? (size_t)saved.numel() : 0;
        if (gx.defined() || gw0.defined() || gw1.defined() || gb.defined() || gm.defined()) {
            a.workspace_bytes = wkv_linear_backward_workspace(&a);
            Tensor ws = bytes_like(gy, a.workspace_bytes);
            a.workspace = ptr(ws);
            check(wkv_linear_backward(&a, stream_of(gy)), "wkv_linear_backward");
        }
        if (pair) return {gx, gw0, gw1};
        return {gx, gw0, gb.defined() ? gb.to(b_type) : gb, gm, want(4) ? grads[0] : Tensor()};
    }
};

Tensor linear_forward(const Tensor &x, const Tensor &w0, const Tensor &w1, const Tensor &bias, const Tensor &mul, const Tensor &residual, int act) {
    require_cuda({&x, &w0, &w1, &bias, &mul, &residual});
    c10::cuda::OptionalCUDAGuard guard(x.device());
    poll_status(x.device().index(), false);
    const bool save = wants_grad({&x, &w0, &w1, &bias, &mul, &residual});
    std::shared_ptr<LinearBackward> node;
    if (save) {
        if (w1.defined()) node = make_node<LinearBackward>({x, w0, w1});
        else node = make_node<LinearBackward>({x, w0, bias, mul, residual});
        node->act = act;
        node->pair = w1.defined();
        node->b_type = node->b_kept = at::kFloat;
        if (bias.defined()) {
            node->b_type = bias.scalar_type();
            node->b_kept = param_type(bias);
        }
    }
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        LinearCall c = linear_call(x, w0, w1, bias, mul, residual, act);
        wkv_linear_args_t &a = c.a;
        y = fresh(out_sizes(x, a.N), x.scalar_type(), x);
        a.y = ptr(y);
        const auto grad = [&](const Tensor &t) { return save && t.defined() && t.requires_grad(); };
        const bool of_x = grad(x), of_w = grad(w0) || grad(w1), any = of_x || of_w || grad(bias) || grad(mul);
        Tensor saved;
        if (any) {
            a.saved_bytes = wkv_linear_saved_bytes(&a);
            saved = bytes_like(x, a.saved_bytes);
            a.saved = ptr(saved);
        }
        a.workspace_bytes = wkv_linear_forward_workspace(&a);
        Tensor ws = bytes_like(x, a.workspace_bytes);
        a.workspace = ptr(ws);
        check(wkv_linear_forward(&a, stream_of(x)), "wkv_linear_forward");
        if (save) {
            node->rows = a.rows; node->K = a.K; node->N = a.N;
            node->x_sizes = x.sizes().vec();
            const Tensor none;
            node->keep({of_w ? c.x.t : none, of_x ? c.w0.t : none, of_x ? c.w1.t : none, any ? c.mul : none, saved});
        }
    }
    if (save) torch::autograd::set_history(y, node);
    return y;
}

Tensor linear_act(const Tensor &x, const Tensor &weight, const OptTensor &bias_, const std::string &activation, const OptTensor &mul_,
                  const OptTensor &residual_) {
    const Tensor bias = opt(bias_), mul = opt(mul_), residual = opt(residual_);
    const int act = act_code(activation);
    check_x(x);
    check_matrix(weight, x, "weight");
    const auto sizes = out_sizes(x, weight.size(0));
    check_param(bias, "bias");
    check_sizes(bias, {weight.size(0)}, "bias");
    for (auto [t, name] : {std::pair<const Tensor *, const char *>{&mul, "mul"}, {&residual, "residual"}}) {
        check_type(*t, x.scalar_type(), name);
        check_sizes(*t, sizes, name);
    }
    return linear_forward(x, weight, Tensor(), bias, mul, residual, act);
}

Tensor gated_linear(const Tensor &x, const Tensor &w_gate, const Tensor &w_up, const std::string &activation) {
    const int act = act_code(activation);
    check_x(x);
    check_matrix(w_gate, x, "w_gate");
    check_matrix(w_up, x, "w_up");
    check_sizes(w_up, w_gate.sizes(), "w_up");
    return linear_forward(x, w_gate, w_up, Tensor(), Tensor(), Tensor(), act);
}

}  // namespace
}  // namespace wkv_native

void bind_linear(py::module_ &m) {
    using namespace wkv_native;
    m.def("linear_act", &linear_act);
    m.def("gated_linear", &gated_linear);
}
