// Short causal convolution over time, one filter per channel, with the last W-1 inputs as its carried state:
//
//   s_t = bias + sum_j weight[d,j] x_{t-W+1+j},   y_t = silu(s_t)  or  s_t          (x of negative time: the state)
//   state_out = the last W-1 inputs
//
//   backward: ds = gy silu'(s),  gx_t = sum_j weight[d,j] ds_{t+W-1-j},  gweight[d,j] = sum_t ds_t x_{t-W+1+j},  gbias = sum ds;
//   what reaches inputs of negative time is the state's gradient.
//
// Bound by HBM.  A thread owns a few neighbouring channels and walks a strip of tokens with the last W-1 inputs in
// registers; neighbouring strips read W-1 tokens twice (from L2).  Nothing is kept for the backward pass: s is formed again.
#include "elem_io.cuh"
#include "wkv_internal.h"

namespace wkv {
namespace {

constexpr int MAX_W = 4;

struct ConvArgs {
    int B, T, D, w_dtype, silu;
    long long x_batch, x_token;          // strides of x in elements
    const void *x, *w, *bias, *state_in;
    void *y, *state_out;
    const void *gy, *gs_out;
    void *gx, *gs_in;
    float *part;                         // [B * strips of a row, D * (W + 1)]
    int strip, nstrip, vec;
};

__device__ __forceinline__ float silu_grad(float s) {
    const float sg = sigmoidf(s);
    return sg * (1.f + s * (1.f - sg));
}

// inputs of the row at time t: from the state below zero (zeros without one)
template <typename F, int V, int W>
__device__ __forceinline__ void input_at(const ConvArgs &a, int b, int c, int n, int t, Raw<F, V> &r) {
    if (t >= 0) r.load((const F *)a.x + (size_t)b * a.x_batch + (size_t)t * a.x_token + c, a.vec, n);
    else if (a.state_in) r.load((const F *)a.state_in + ((size_t)b * (W - 1) + (W - 1 + t)) * a.D + c, a.vec, n);
    else r.zero();
}

// V channels per thread: 16 bytes of them.  blockIdx.x: (row, strip), blockIdx.y: 256 runs of channels
template <typename F, int W>
__global__ void __launch_bounds__(256) k_conv_fwd(ConvArgs a) {
    pdl_wait();
    pdl_trigger();
    constexpr int V = 16 / (int)sizeof(F), AHEAD = 4;
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * V;
    if (c >= a.D) return;
    const int n = min(V, a.D - c), b = blockIdx.x / a.nstrip, t0 = (blockIdx.x - b * a.nstrip) * a.strip;
    const int t1 = min(t0 + a.strip, a.T);
    Raw<F, V> in[W - 1 + AHEAD];
#pragma unroll
    for (int j = 0; j < W - 1; j++) input_at<F, V, W>(a, b, c, n, t0 - (W - 1) + j, in[j]);
    float w[V][W], bias[V];
#pragma unroll
    for (int q = 0; q < V; q++) {
        bias[q] = a.bias && q < n ? param_at(a.bias, a.w_dtype, c + q) : 0.f;
#pragma unroll
        for (int j = 0; j < W; j++) w[q][j] = q < n ? param_at(a.w, a.w_dtype, (size_t)(c + q) * W + j) : 0.f;
    }
    F *y = (F *)a.y + ((size_t)b * a.T) * a.D + c;
    for (int t = t0; t < t1; t += AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (t + i < t1) input_at<F, V, W>(a, b, c, n, t + i, in[W - 1 + i]);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (t + i < t1) {
                float s[V];
#pragma unroll
                for (int q = 0; q < V; q++) s[q] = bias[q];
#pragma unroll
                for (int j = 0; j < W; j++) {
                    float f[V];
                    in[i + j].get(f);
#pragma unroll
                    for (int q = 0; q < V; q++) s[q] += w[q][j] * f[q];
                }
                if (a.silu) {
#pragma unroll
                    for (int q = 0; q < V; q++) s[q] *= sigmoidf(s[q]);
                }
                Raw<F, V> o;
                o.put(s);
                o.store(y + (size_t)(t + i) * a.D, a.vec, n);
            }
        }
        // the last W-1 inputs that exist move to the front
        const int k = min(AHEAD, t1 - t);
        Raw<F, V> last[W - 1];
#pragma unroll
        for (int j = 0; j < W - 1; j++)
#pragma unroll
            for (int i = 1; i <= AHEAD; i++)
                if (i == k) last[j] = in[i + j];
#pragma unroll
        for (int j = 0; j < W - 1; j++) in[j] = last[j];
    }
    if (t1 == a.T && a.state_out) {
#pragma unroll
        for (int j = 0; j < W - 1; j++) in[j].store((F *)a.state_out + ((size_t)b * (W - 1) + j) * a.D + c, a.vec, n);
    }
}

// A thread walks its strip forward, W-1 tokens past its end: at token t it forms s_t and ds_t, adds to the sums of the
// parameters' gradients where t is its own, and hands out gx of token t-W+1, which is complete then.
template <typename F, int W>
__global__ void __launch_bounds__(256) k_conv_bwd(ConvArgs a) {
    pdl_wait();
    pdl_trigger();
    constexpr int V = 4;
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * V;
    if (c >= a.D) return;
    const int n = min(V, a.D - c), b = blockIdx.x / a.nstrip, t0 = (blockIdx.x - b * a.nstrip) * a.strip;
    const int t1 = min(t0 + a.strip, a.T);
    float w[V][W], bias[V], gw[V][W], gb[V];
#pragma unroll
    for (int q = 0; q < V; q++) {
        bias[q] = a.bias && q < n ? param_at(a.bias, a.w_dtype, c + q) : 0.f;
        gb[q] = 0.f;
#pragma unroll
        for (int j = 0; j < W; j++) {
            w[q][j] = q < n ? param_at(a.w, a.w_dtype, (size_t)(c + q) * W + j) : 0.f;
            gw[q][j] = 0.f;
        }
    }
    float x[V][W], g[V][W];              // x_{t-W+1} .. x_t;  sums for gx_{t-W+1} .. gx_t
#pragma unroll
    for (int j = 0; j < W - 1; j++) {
        Raw<F, V> r;
        float f[V];
        input_at<F, V, W>(a, b, c, n, t0 - (W - 1) + j, r);
        r.get(f);
#pragma unroll
        for (int q = 0; q < V; q++) x[q][j] = f[q];
    }
#pragma unroll
    for (int q = 0; q < V; q++)
#pragma unroll
        for (int j = 0; j < W; j++) g[q][j] = 0.f;
    const F *gy = a.gy ? (const F *)a.gy + ((size_t)b * a.T) * a.D + c : nullptr;
    // (of the tokens before the strip only the first strip's, the state, are its own)
    const int first = t0 == 0 ? -(W - 1) : t0;
    for (int t = t0; t < t1 + W - 1; t++) {
        float ds[V];
#pragma unroll
        for (int q = 0; q < V; q++) ds[q] = 0.f;
        if (t < a.T) {
            Raw<F, V> rx, rg;
            float f[V];
            input_at<F, V, W>(a, b, c, n, t, rx);
            rg.zero();
            if (gy) rg.load(gy + (size_t)t * a.D, a.vec, n);
            rx.get(f);
            rg.get(ds);
#pragma unroll
            for (int q = 0; q < V; q++) {
                x[q][W - 1] = f[q];
                if (a.silu) {
                    float s = bias[q];
#pragma unroll
                    for (int j = 0; j < W; j++) s += w[q][j] * x[q][j];
                    ds[q] *= silu_grad(s);
                }
                if (t < t1) {
                    gb[q] += ds[q];
#pragma unroll
                    for (int j = 0; j < W; j++) gw[q][j] += ds[q] * x[q][j];
                }
            }
        }
        const int to = t - (W - 1);       // the token whose gradient is complete
        float o[V];
#pragma unroll
        for (int q = 0; q < V; q++) {
#pragma unroll
            for (int j = 0; j < W; j++) g[q][j] += w[q][j] * ds[q];
            o[q] = g[q][0];
        }
        if (to >= first && to < t1) {
            if (a.gs_out && to >= a.T - (W - 1)) {        // a token that is part of the state handed on
                Raw<F, V> r;
                float f[V];
                r.load((const F *)a.gs_out + ((size_t)b * (W - 1) + (to - (a.T - (W - 1)))) * a.D + c, a.vec, n);
                r.get(f);
#pragma unroll
                for (int q = 0; q < V; q++) o[q] += f[q];
            }
            Raw<F, V> r;
            r.put(o);
            if (to >= 0) {
                if (a.gx) r.store((F *)a.gx + ((size_t)b * a.T + to) * a.D + c, a.vec, n);
            } else if (a.gs_in) {
                r.store((F *)a.gs_in + ((size_t)b * (W - 1) + (W - 1 + to)) * a.D + c, a.vec, n);
            }
        }
#pragma unroll
        for (int q = 0; q < V; q++) {
#pragma unroll
            for (int j = 0; j < W - 1; j++) { x[q][j] = x[q][j + 1]; g[q][j] = g[q][j + 1]; }
            g[q][W - 1] = 0.f;
        }
    }
    if (a.part) {
        float *p = a.part + (size_t)blockIdx.x * ((size_t)a.D * (W + 1));
#pragma unroll
        for (int q = 0; q < V; q++) {
            if (q < n) {
#pragma unroll
                for (int j = 0; j < W; j++) p[(size_t)(c + q) * W + j] = gw[q][j];
                p[(size_t)a.D * W + c + q] = gb[q];
            }
        }
    }
}

int check_conv(const wkv_causal_conv_args_t *a) {
    if (!a) return WKV_ERR_NULL;
    if (a->B < 0 || a->T < 0 || a->D < 0 || a->W < 2 || a->W > MAX_W) return WKV_ERR_SHAPE;
    if (!known_dtype(a->dtype) || !known_dtype(a->w_dtype)) return WKV_ERR_DTYPE;
    if (a->x_batch < 0 || a->x_token < 0) return WKV_ERR_SHAPE;
    if (a->B > 0 && a->D > 0 && !a->weight) return WKV_ERR_NULL;
    if (a->B > 0 && a->D > 0 && a->T > 0 && !a->x) return WKV_ERR_NULL;
    return WKV_OK;
}

// tokens of a strip: so long that the W-1 tokens read twice do not count, and so short that the GPU is full
int strip_for(int B, int T, int D, int per_thread, int longest) {
    const long long across = (long long)B * ((D + per_thread - 1) / per_thread), want = (long long)device_sm_count() * 1536;
    long long strip = across * T / want;
    strip = strip < 16 ? 16 : strip > longest ? longest : strip;
    return (int)strip;
}

ConvArgs conv_args(const wkv_causal_conv_args_t *a) {
    ConvArgs k = {};
    k.B = a->B; k.T = a->T; k.D = a->D; k.w_dtype = a->w_dtype; k.silu = a->silu != 0;
    k.x_batch = a->x_batch; k.x_token = a->x_token;
    k.x = a->x; k.w = a->weight; k.bias = a->bias; k.state_in = a->state_in;
    return k;
}
// whether every row of every tensor starts at a multiple of 16 bytes
bool conv_vec(const wkv_causal_conv_args_t *a, std::initializer_list<const void *> ptrs) {
    const int v = 16 / elem_size(a->dtype);
    return a->D % v == 0 && a->x_token % v == 0 && a->x_batch % v == 0 && all_aligned(ptrs);
}

template <class Fn>
int by_width(int W, Fn f) {
    switch (W) {
        case 2: return f(std::integral_constant<int, 2>{});
        case 3: return f(std::integral_constant<int, 3>{});
        default: return f(std::integral_constant<int, 4>{});
    }
}

constexpr int BWD_V = 4;

}  // namespace
}  // namespace wkv

using namespace wkv;

extern "C" int wkv_causal_conv_forward(const wkv_causal_conv_args_t *a, void *stream) {
    int e = check_conv(a);
    if (e != WKV_OK) return e;
    if (a->B == 0 || a->D == 0) return WKV_OK;
    if (a->T > 0 && !a->y) return WKV_ERR_NULL;
    // (a thread of the first strip reads the state after one of the last strip has written it)
    if (a->T > 16 && a->state_in && a->state_in == a->state_out) return WKV_ERR_UNSUPPORTED;
    ConvArgs k = conv_args(a);
    k.y = a->y; k.state_out = a->state_out;
    k.vec = conv_vec(a, {a->x, a->state_in, a->y, a->state_out});
    const int per = 16 / elem_size(a->dtype);
    k.strip = strip_for(a->B, a->T, a->D, per, 64);
    k.nstrip = a->T > 0 ? (a->T + k.strip - 1) / k.strip : 1;
    const int runs = (a->D + per - 1) / per, nt = runs >= 256 ? 256 : (runs + 31) / 32 * 32;
    return by_dtype(a->dtype, [&](auto f) {
        using F = decltype(f);
        return by_width(a->W, [&](auto w) {
            return launch_chained(k_conv_fwd<F, decltype(w)::value>, dim3(a->B * k.nstrip, (runs + nt - 1) / nt), dim3(nt), 0,
                                  (cudaStream_t)stream, k);
        });
    });
}

extern "C" size_t wkv_causal_conv_backward_workspace(const wkv_causal_conv_args_t *a) {
    if (check_conv(a) != WKV_OK || a->B == 0 || a->D == 0 || a->T == 0) return 0;
    const int strip = strip_for(a->B, a->T, a->D, BWD_V, 256);
    return align256((size_t)a->B * ((a->T + strip - 1) / strip) * a->D * (a->W + 1) * 4);
}

extern "C" int wkv_causal_conv_backward(const wkv_causal_conv_args_t *a, void *stream) {
    int e = check_conv(a);
    if (e != WKV_OK) return e;
    cudaStream_t s = (cudaStream_t)stream;
    const bool params = a->gweight || a->gbias, empty = a->B == 0 || a->D == 0;
    if (a->D == 0) return WKV_OK;
    int rows = 0;
    if (!empty) {
        ConvArgs k = conv_args(a);
        k.gy = a->gy; k.gs_out = a->gstate_out; k.gx = a->gx; k.gs_in = a->gstate_in;
        k.vec = conv_vec(a, {a->x, a->state_in, a->gy, a->gstate_out, a->gx, a->gstate_in});
        k.strip = strip_for(a->B, a->T, a->D, BWD_V, 256);
        k.nstrip = a->T > 0 ? (a->T + k.strip - 1) / k.strip : 1;
        if (params && a->T > 0) {
            if (!a->workspace || a->workspace_bytes < wkv_causal_conv_backward_workspace(a)) return WKV_ERR_WORKSPACE;
            if (!aligned16(a->workspace)) return WKV_ERR_ALIGN;
            k.part = (float *)a->workspace;
            rows = a->B * k.nstrip;
        }
        const int runs = (a->D + BWD_V - 1) / BWD_V, nt = runs >= 256 ? 256 : (runs + 31) / 32 * 32;
        e = by_dtype(a->dtype, [&](auto f) {
            using F = decltype(f);
            return by_width(a->W, [&](auto w) {
                return launch_chained(k_conv_bwd<F, decltype(w)::value>, dim3(a->B * k.nstrip, (runs + nt - 1) / nt), dim3(nt), 0, s, k);
            });
        });
        if (e != WKV_OK) return e;
    }
    if (!params) return WKV_OK;
    FoldOut f = {};
    const long long nw = (long long)a->D * a->W;
    f.p[0] = a->gweight; f.dtype[0] = a->w_dtype;
    f.p[1] = a->gbias; f.dtype[1] = a->w_dtype;
    f.start[1] = nw;
    for (int i = 2; i < 5; i++) f.start[i] = nw + a->D;
    return fold_params((const float *)a->workspace, rows, nw + a->D, f, s);
}
