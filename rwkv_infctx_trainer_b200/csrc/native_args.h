// Checks of arguments and views of activations, shared by the bindings of the operators beside the WKV ops.
#pragma once
#include "native_ops.h"

namespace wkv_native {

inline Tensor opt(const OptTensor &t) { return t.has_value() ? *t : Tensor(); }

inline int small(int64_t n, const char *what) {
    TORCH_CHECK_VALUE(n <= std::numeric_limits<int>::max(), what, " is too large: ", n);
    return (int)n;
}
inline void check_type(const Tensor &t, at::ScalarType dt, const char *name) {
    TORCH_CHECK_TYPE(!t.defined() || t.scalar_type() == dt, name, " must be ", dt, ", got ", t.scalar_type());
}
inline void check_param(const Tensor &t, const char *name) {
    TORCH_CHECK_TYPE(!t.defined() || at::isFloatingType(t.scalar_type()), name, " must be a floating point tensor");
}
inline void check_sizes(const Tensor &t, at::IntArrayRef want, const char *name) {
    TORCH_CHECK_VALUE(!t.defined() || t.sizes() == want, name, " must have shape ", want, ", got ", t.sizes());
}
// the calls that update a state in place have no backward pass
inline void refuse_grad(std::initializer_list<const Tensor *> ts, const char *call, const char *other) {
    TORCH_CHECK(!wants_grad(ts), call, " updates the state in place and has no gradient: call it under torch.no_grad(), or ", other);
}
inline void check_in_place(const Tensor &state, const char *call) {
    TORCH_CHECK_VALUE(state.is_contiguous(), call, ": the state is updated in place and must be contiguous");
}
// Before the launch: torch refuses this for a tensor made in inference mode, outside of it, and then nothing may have changed.
inline void changes_in_place(const Tensor &state) { torch::autograd::impl::bump_version(state); }

// Rows of adjacent channels with any stride between rows and between tokens, as the kernels take them: a view of a wider
// tensor stays one, anything else is copied.
struct Rows {
    Tensor t;
    int64_t batch = 0, token = 0;
};
// t: [B, T, ...], or [B, ...] for one token, with everything behind one run of `n` elements
inline Rows rows_of(const Tensor &t, int64_t n, bool one_token) {
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

}  // namespace wkv_native
