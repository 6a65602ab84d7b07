// Short causal convolution over time, one filter per channel, with the last W-1 inputs as its carried state:
//
//   s_t = bias + sum_j weight[d,j] x_{t-W+1+j},   y_t = silu(s_t)  or  s_t          (x of negative time: the state)
//   state_out = the last W-1 inputs
//
//   backward: ds = gy silu'(s),  gx_t = sum_j weight[d,j] ds_{t+W-1-j},  gweight[d,j] = sum_t ds_t x_{t-W+1+j},  gbias = sum ds;
//   what reaches inputs of negative time is the state's gradient.
//
// Bound by HBM forward.  A thread owns four neighbouring channels and walks a strip of tokens with the last W-1 inputs in
// registers, on packed arithmetic; neighbouring strips read W-1 tokens twice (from L2).  Nothing is kept for the backward pass: s is formed again.
// 4 rows of 4096 tokens and bf16 channels, W = 4: 51 us forward (5.2 TB/s), 117 backward with the fold of the parameters' gradients
// (3.5 TB/s).  Backward neither HBM nor issue (0.49 a cycle) is the limit: 126 to 128 registers leave 512 threads an SM, half of those that
// a strip's length is chosen for, to hide the latency of what a token needs.
#include "elem_io.cuh"
#include "wkv_internal.h"

namespace wkv {
namespace {

constexpr int MAX_W = 4, MAX_D = 1 << 22, SHORTEST = 16, LONGEST = 256;            // (tokens of a strip, at least and at most)
// (token numbers up to the end of the last strip, and a few behind it, are 32-bit)
constexpr int MAX_T = 0x7FFFFFFF - LONGEST - 16;
constexpr int V = 4;                     // channels of a thread
// Tokens of a group and groups on their way (us forward, 4 rows of 4096 tokens and channels: 6 x 3 63, 4 x 4 59, 4 x 3 57, 2 x 8 59;
// backward: 6 x 2 140, 3 x 6 124, 3 x 4 122, 3 x 3 120): small groups leave registers for more threads.
constexpr int FWD_GT = 4, FWD_AHEAD = 3, BWD_GT = 3, BWD_AHEAD = 3;

struct ConvArgs {
    int B, T, D, w_dtype, silu;
    long long x_batch, x_token;          // strides of x in elements
    const void *x, *w, *bias, *state_in;
    void *y, *state_out;
    const void *gy, *gs_out;
    void *gx, *gs_in;
    float *part;                         // [B * strips of a row, D * (W + 1)]
    int strip, nstrip, vec_w;
};

// How rows lie, and a thread's four channels.  RUNS: rows start at multiples of four elements, the channels are neighbours.
// WORDS: at multiples of 4 bytes, the channels are 4-byte words (two of 16 bits, or one of 32) that are 32 words apart.  ONES: 16-bit
// rows that start anywhere, single channels 32 apart.  In each a warp's access is one piece of a row.
enum { RUNS, WORDS, ONES };
template <typename F, int MODE>
struct Lie {
    static constexpr int UNIT = MODE == RUNS ? V : MODE == WORDS ? 4 / (int)sizeof(F) : 1, APART = MODE == RUNS ? V : 32 * UNIT;
    static __device__ __forceinline__ int first() {
        const int i = blockIdx.y * blockDim.x + threadIdx.x;
        return MODE == RUNS ? i * V : (i >> 5) * (32 * V) + (i & 31) * UNIT;
    }
    // how many of the channels from c on exist
    static __device__ __forceinline__ int left(int D, int c) { return MODE == RUNS ? V : min(V, (D - c + APART - 1) / APART * UNIT); }
    static __device__ __forceinline__ int channel(int c, int q) { return c + q / UNIT * APART + q % UNIT; }
    static __device__ __forceinline__ void load(Raw<F, V> &r, const F *p, int n) {
        if constexpr (MODE == RUNS) r.load(p, true, V);
        else if constexpr (MODE == ONES) r.template gather<32>(p, n);
        else {
#pragma unroll
            for (int i = 0; i < Raw<F, V>::WORDS; i++) r.w[i] = i * UNIT < n ? *reinterpret_cast<const uint32_t *>(p + i * APART) : 0u;
        }
    }
    static __device__ __forceinline__ void store(const Raw<F, V> &r, F *p, int n) {
        if constexpr (MODE == RUNS) r.store(p, true, V);
        else if constexpr (MODE == ONES) r.template scatter<32>(p, n);
        else {
#pragma unroll
            for (int i = 0; i < Raw<F, V>::WORDS; i++)
                if (i * UNIT < n) *reinterpret_cast<uint32_t *>(p + i * APART) = r.w[i];
        }
    }
    // into shared memory without passing through registers (RUNS, WORDS)
    static __device__ __forceinline__ void load_async(Raw<F, V> &to, const F *p, int n) {
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(&to);
        if constexpr (MODE == RUNS) {
            if constexpr (sizeof(to) == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(p) : "memory");
            else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(p) : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < Raw<F, V>::WORDS; i++)
                if (i * UNIT < n) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + 4 * i), "l"(p + i * APART) : "memory");
        }
    }
};

// inputs of the row at time t: from the state below zero (zeros without one)
template <typename F, int W, int MODE>
__device__ __forceinline__ void input_at(const ConvArgs &a, int b, int c, int n, int t, Raw<F, V> &r) {
    if (t >= 0) Lie<F, MODE>::load(r, (const F *)a.x + (size_t)b * a.x_batch + (size_t)t * a.x_token + c, n);
    else if (a.state_in) Lie<F, MODE>::load(r, (const F *)a.state_in + ((size_t)b * (W - 1) + (W - 1 + t)) * a.D + c, n);
    else r.zero();
}

// the parameters of a thread's channels: two pairs of channels per tap
template <typename F, int W, int MODE>
__device__ __forceinline__ void load_params(const ConvArgs &a, int c, int n, f2 (&w)[W][2], f2 (&bias)[2]) {
    float t[V][W], bb[V];
#pragma unroll
    for (int q = 0; q < V; q++) {
        bb[q] = a.bias && q < n ? param_at(a.bias, a.w_dtype, Lie<F, MODE>::channel(c, q)) : 0.f;
        if (W == 4 && a.vec_w) {
            const float4 v = q < n ? __ldg(reinterpret_cast<const float4 *>((const float *)a.w + (size_t)Lie<F, MODE>::channel(c, q) * W)) : make_float4(0.f, 0.f, 0.f, 0.f);
            t[q][0] = v.x; t[q][1] = v.y; t[q][2 % W] = v.z; t[q][3 % W] = v.w;
        } else {
#pragma unroll
            for (int j = 0; j < W; j++) t[q][j] = q < n ? param_at(a.w, a.w_dtype, (size_t)Lie<F, MODE>::channel(c, q) * W + j) : 0.f;
        }
    }
#pragma unroll
    for (int p = 0; p < 2; p++) {
        bias[p] = make_float2(bb[2 * p], bb[2 * p + 1]);
#pragma unroll
        for (int j = 0; j < W; j++) w[j][p] = make_float2(t[2 * p][j], t[2 * p + 1][j]);
    }
}
template <typename F>
__device__ __forceinline__ void get_pairs(const Raw<F, V> &r, f2 (&v)[2]) {
    float f[V];
    r.get(f);
    v[0] = make_float2(f[0], f[1]);
    v[1] = make_float2(f[2], f[3]);
}
template <typename F>
__device__ __forceinline__ Raw<F, V> put_pairs(const f2 (&v)[2]) {
    const float f[V] = {v[0].x, v[0].y, v[1].x, v[1].y};
    Raw<F, V> r;
    r.put(f);
    return r;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ f2 sigmoid2(f2 x) {
    const f2 t = mul2(x, both(-1.4426950408889634f)), d = add2(make_float2(ex2(t.x), ex2(t.y)), both(1.f));
    return make_float2(rcp(d.x), rcp(d.y));
}

// A thread's inputs on their way: a ring of AHEAD groups of GT tokens of N tensors in shared memory, a place of its own for
// each thread (nobody else reads it: no barriers).  Held in registers instead, two groups were as many as fit: 4 rows of 4096 tokens
// and channels took 78 us forward and 218 backward, with the ring 66 and 149.  Most groups are whole and inside the strip: those
// run without a look at each token, and the ways that rows lie are compiled apart: 57 and 120 us.  (There are no copies of 2 bytes:
// ONES has one group on its way, in registers.)
template <typename F, int GT, int N, int AHEAD, int MODE>
struct Ring {
    Raw<F, V> *mine;                     // [AHEAD][GT][N][threads]
    int threads, n, in = 0, out = 0;     // the groups to be filled and to be read
    Raw<F, V> held[MODE != ONES ? 1 : GT * N];   // ONES: one group, in registers
    __device__ __forceinline__ Raw<F, V> &at(int group, int i, int k) const { return mine[((group * GT + i) * N + k) * threads]; }
    __device__ __forceinline__ void load(int i, int k, const F *p) {
        if constexpr (MODE != ONES) Lie<F, MODE>::load_async(at(in, i, k), p, n);
        else Lie<F, MODE>::load(held[i * N + k], p, n);
    }
    __device__ __forceinline__ const Raw<F, V> &read(int i, int k) const { return MODE != ONES ? at(out, i, k) : held[MODE != ONES ? 0 : i * N + k]; }
    __device__ __forceinline__ void commit() {
        if (MODE == ONES) return;
        asm volatile("cp.async.commit_group;" ::: "memory");
        in = in + 1 == AHEAD ? 0 : in + 1;
    }
    // the next group to be read has arrived
    __device__ __forceinline__ void wait() {
        if (MODE != ONES) asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
    }
    // the group has been read (before anything is copied to its place)
    __device__ __forceinline__ void next() {
        __syncwarp(__activemask());
        out = out + 1 == AHEAD ? 0 : out + 1;
    }
};
template <typename F, int MODE>
using FwdRing = Ring<F, FWD_GT, 1, FWD_AHEAD, MODE>;
template <typename F, int MODE>
using BwdRing = Ring<F, BWD_GT, 2, BWD_AHEAD, MODE>;

// blockIdx.x: (row, strip), blockIdx.y: runs of channels
template <typename F, int W, int MODE>
__global__ void __launch_bounds__(256) k_conv_fwd(ConvArgs a) {
    pdl_wait();
    pdl_trigger();
    constexpr int GT = FWD_GT;
    extern __shared__ __align__(16) char smem_raw[];
    const int c = Lie<F, MODE>::first();
    if (c >= a.D) return;
    const int n = Lie<F, MODE>::left(a.D, c), b = blockIdx.x / a.nstrip, t0 = (blockIdx.x - b * a.nstrip) * a.strip;
    const int t1 = min(t0 + a.strip, a.T);
    FwdRing<F, MODE> ring = {reinterpret_cast<Raw<F, V> *>(smem_raw) + threadIdx.x, (int)blockDim.x, n};
    const F *px = (const F *)a.x + (size_t)b * a.x_batch + (size_t)t0 * a.x_token + c;
    int left = t1 - t0;                  // tokens that are still to be fetched
    auto fetch = [&]() {
        if (left >= GT) {
#pragma unroll
            for (int i = 0; i < GT; i++) ring.load(i, 0, px + i * a.x_token);
        } else {
#pragma unroll
            for (int i = 0; i < GT; i++)
                if (i < left) ring.load(i, 0, px + i * a.x_token);
        }
        ring.commit();
        px += GT * a.x_token;
        left -= GT;
    };
#pragma unroll
    for (int g = 0; g < (MODE != ONES ? FWD_AHEAD : 1); g++) fetch();
    f2 w[W][2], bias[2], x[W - 1 + GT][2];
    load_params<F, W, MODE>(a, c, n, w, bias);
#pragma unroll
    for (int j = 0; j < W - 1; j++) {
        Raw<F, V> r;
        input_at<F, W, MODE>(a, b, c, n, t0 - (W - 1) + j, r);
        get_pairs(r, x[j]);
    }
    F *y = (F *)a.y + ((size_t)b * a.T + t0) * a.D + c;
    auto group = [&](auto whole, int count) {
        ring.wait();
#pragma unroll
        for (int i = 0; i < GT; i++) get_pairs(ring.read(i, 0), x[W - 1 + i]);
        ring.next();
        fetch();
#pragma unroll
        for (int i = 0; i < GT; i++) {
            f2 s[2] = {bias[0], bias[1]};
#pragma unroll
            for (int j = 0; j < W; j++)
#pragma unroll
                for (int p = 0; p < 2; p++) s[p] = fma2(w[j][p], x[i + j][p], s[p]);
            if (a.silu) {
#pragma unroll
                for (int p = 0; p < 2; p++) s[p] = mul2(s[p], sigmoid2(s[p]));
            }
            if (decltype(whole)::value || i < count) Lie<F, MODE>::store(put_pairs<F>(s), y + (size_t)i * a.D, n);
        }
        y += (size_t)GT * a.D;
        // the last W-1 inputs that exist move to the front
#pragma unroll
        for (int j = 0; j < W - 1; j++) {
            f2 l[2] = {x[GT + j][0], x[GT + j][1]};
            if (!decltype(whole)::value) {
#pragma unroll
                for (int i = 1; i < GT; i++)
                    if (i == count) { l[0] = x[i + j][0]; l[1] = x[i + j][1]; }
            }
            x[j][0] = l[0];
            x[j][1] = l[1];
        }
    };
    int t = t0;
    for (; t + GT <= t1; t += GT) group(std::true_type{}, GT);
    if (t < t1) group(std::false_type{}, t1 - t);
    if (t1 == a.T && a.state_out) {
#pragma unroll
        for (int j = 0; j < W - 1; j++) Lie<F, MODE>::store(put_pairs<F>(x[j]), (F *)a.state_out + ((size_t)b * (W - 1) + j) * a.D + c, n);
    }
}

// A thread walks its strip forward, W-1 tokens past its end, in groups: it forms s and ds of a group's tokens, adds to the sums
// of the parameters' gradients where they are its own, and hands out gx of the tokens W-1 earlier, which is complete then.
template <typename F, int W, int MODE>
__global__ void __launch_bounds__(256) k_conv_bwd(ConvArgs a) {
    pdl_wait();
    pdl_trigger();
    constexpr int GT = BWD_GT;
    extern __shared__ __align__(16) char smem_raw[];
    const int c = Lie<F, MODE>::first();
    if (c >= a.D) return;
    const int n = Lie<F, MODE>::left(a.D, c), b = blockIdx.x / a.nstrip, t0 = (blockIdx.x - b * a.nstrip) * a.strip;
    const int t1 = min(t0 + a.strip, a.T), stop = t1 + W - 1;
    BwdRing<F, MODE> ring = {reinterpret_cast<Raw<F, V> *>(smem_raw) + threadIdx.x, (int)blockDim.x, n};
    const F *px = (const F *)a.x + (size_t)b * a.x_batch + (size_t)t0 * a.x_token + c, *gy = (const F *)a.gy + ((size_t)b * a.T + t0) * a.D + c;
    int left = min(stop, a.T) - t0;
    auto fetch = [&]() {
        if (left >= GT) {
#pragma unroll
            for (int i = 0; i < GT; i++) ring.load(i, 0, px + i * a.x_token);
            if (a.gy) {
#pragma unroll
                for (int i = 0; i < GT; i++) ring.load(i, 1, gy + (size_t)i * a.D);
            }
        } else {
#pragma unroll
            for (int i = 0; i < GT; i++) {
                if (i < left) {
                    ring.load(i, 0, px + i * a.x_token);
                    if (a.gy) ring.load(i, 1, gy + (size_t)i * a.D);
                }
            }
        }
        ring.commit();
        px += GT * a.x_token;
        gy += (size_t)GT * a.D;
        left -= GT;
    };
#pragma unroll
    for (int g = 0; g < (MODE != ONES ? BWD_AHEAD : 1); g++) fetch();
    f2 w[W][2], bias[2], gw[W][2], gb[2] = {both(0.f), both(0.f)};
    f2 x[W - 1 + GT][2], ds[W - 1 + GT][2];              // of tokens t-W+1 .. t+GT-1
    load_params<F, W, MODE>(a, c, n, w, bias);
#pragma unroll
    for (int j = 0; j < W; j++) gw[j][0] = gw[j][1] = both(0.f);
#pragma unroll
    for (int j = 0; j < W - 1; j++) {
        Raw<F, V> r;
        input_at<F, W, MODE>(a, b, c, n, t0 - (W - 1) + j, r);
        get_pairs(r, x[j]);
        ds[j][0] = ds[j][1] = both(0.f);
    }
    // (of the tokens before the strip only the first strip's, the state, are its own)
    const int first = t0 == 0 ? -(W - 1) : t0;
    F *gx = (F *)a.gx + ((size_t)b * a.T + t0) * a.D + c - (long long)(W - 1) * a.D;      // of token t-W+1
    // inside: the group's tokens are the strip's own, and so are those W-1 earlier
    auto group = [&](auto inside, int t) {
        constexpr bool IN = decltype(inside)::value;
        ring.wait();
#pragma unroll
        for (int i = 0; i < GT; i++) {
            get_pairs(ring.read(i, 0), x[W - 1 + i]);
            if (a.gy) get_pairs(ring.read(i, 1), ds[W - 1 + i]);
            else ds[W - 1 + i][0] = ds[W - 1 + i][1] = both(0.f);
        }
        ring.next();
        fetch();
        if (a.silu) {
#pragma unroll
            for (int i = 0; i < GT; i++)
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    f2 s = bias[p];
#pragma unroll
                    for (int j = 0; j < W; j++) s = fma2(w[j][p], x[i + j][p], s);
                    const f2 sg = sigmoid2(s);
                    // silu'(s) = sg (1 + s (1 - sg)) = sg + s sg - s sg^2
                    ds[W - 1 + i][p] = mul2(ds[W - 1 + i][p], mul2(sg, fma2(s, sub2(both(1.f), sg), both(1.f))));
                }
        }
#pragma unroll
        for (int i = 0; i < GT; i++) {
            f2(&d)[2] = ds[W - 1 + i];
            // behind the row there is no gradient (zero times what is formed from no inputs may be a NaN)
            if (!IN && t + i >= a.T) d[0] = d[1] = both(0.f);
            if (IN || t + i < t1) {
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    gb[p] = add2(gb[p], d[p]);
#pragma unroll
                    for (int j = 0; j < W; j++) gw[j][p] = fma2(d[p], x[i + j][p], gw[j][p]);
                }
            }
            const int to = t + i - (W - 1);       // the token whose gradient is complete
            if (IN || (to >= first && to < t1)) {
                f2 o[2];
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    o[p] = mul2(w[0][p], ds[W - 1 + i][p]);
#pragma unroll
                    for (int j = 1; j < W; j++) o[p] = fma2(w[j][p], ds[W - 1 + i - j][p], o[p]);
                }
                if (!IN && a.gs_out && to >= a.T - (W - 1)) {        // a token that is part of the state handed on
                    Raw<F, V> r;
                    f2 f[2];
                    Lie<F, MODE>::load(r, (const F *)a.gs_out + ((size_t)b * (W - 1) + (to - (a.T - (W - 1)))) * a.D + c, n);
                    get_pairs(r, f);
                    o[0] = add2(o[0], f[0]);
                    o[1] = add2(o[1], f[1]);
                }
                if (IN || to >= 0) {
                    if (a.gx) Lie<F, MODE>::store(put_pairs<F>(o), gx + (size_t)i * a.D, n);
                } else if (a.gs_in) {
                    Lie<F, MODE>::store(put_pairs<F>(o), (F *)a.gs_in + ((size_t)b * (W - 1) + (W - 1 + to)) * a.D + c, n);
                }
            }
        }
        gx += (size_t)GT * a.D;
#pragma unroll
        for (int j = 0; j < W - 1; j++)
#pragma unroll
            for (int p = 0; p < 2; p++) {
                x[j][p] = x[GT + j][p];
                ds[j][p] = ds[GT + j][p];
            }
    };
    int t = t0;
    for (; t < stop && t - (W - 1) < t0; t += GT) group(std::false_type{}, t);
    for (; t + GT <= t1; t += GT) group(std::true_type{}, t);
    for (; t < stop; t += GT) group(std::false_type{}, t);
    if (a.part) {
        float *p = a.part + (size_t)blockIdx.x * ((size_t)a.D * (W + 1));
#pragma unroll
        for (int q = 0; q < V; q++) {
            if (q < n) {
#pragma unroll
                for (int j = 0; j < W; j++) p[(size_t)Lie<F, MODE>::channel(c, q) * W + j] = q & 1 ? gw[j][q / 2].y : gw[j][q / 2].x;
                p[(size_t)a.D * W + Lie<F, MODE>::channel(c, q)] = q & 1 ? gb[q / 2].y : gb[q / 2].x;
            }
        }
    }
}

int check_conv(const wkv_causal_conv_args_t *a) {
    if (!a) return WKV_ERR_NULL;
    if (a->B < 0 || a->T < 0 || a->D < 0 || a->W < 2 || a->W > MAX_W || a->D > MAX_D || a->T > MAX_T) return WKV_ERR_SHAPE;
    if ((long long)a->B * (a->T / SHORTEST + 1) > 0x7FFFFFFF) return WKV_ERR_SHAPE;       // (more strips than a grid has blocks)
    if (!known_dtype(a->dtype) || !known_dtype(a->w_dtype)) return WKV_ERR_DTYPE;
    if (a->x_batch < 0 || a->x_token < 0) return WKV_ERR_SHAPE;
    if (a->B > 0 && a->D > 0 && !a->weight) return WKV_ERR_NULL;
    if (a->B > 0 && a->D > 0 && a->T > 0 && !a->x) return WKV_ERR_NULL;
    return WKV_OK;
}

// Tokens of a strip: so many strips that the GPU has `threads` an SM, `longest` tokens at most: short ones leave little to hide a
// load behind, long ones few threads (us with the ring alone: forward 64 tokens 66, 128 80, 32 76; backward 110 tokens 149, 220 171, 64 167).
// (Of these threads an SM holds 768 forward and 512 backward with W = 4: the numbers set the strips, not the occupancy.)
constexpr int FWD_THREADS = 1536, FWD_LONGEST = 64, BWD_THREADS = 1024, BWD_LONGEST = LONGEST;
int strip_for(int B, int T, int D, int threads, int longest) {
    const long long across = (long long)B * ((D + V - 1) / V), want = (long long)device_sm_count() * threads;
    const long long strip = across * T / want;
    return (int)(strip < SHORTEST ? SHORTEST : strip > longest ? longest : strip);
}

ConvArgs conv_args(const wkv_causal_conv_args_t *a) {
    ConvArgs k = {};
    k.B = a->B; k.T = a->T; k.D = a->D; k.w_dtype = a->w_dtype; k.silu = a->silu != 0;
    k.x_batch = a->x_batch; k.x_token = a->x_token;
    k.vec_w = a->w_dtype == WKV_F32 && aligned16(a->weight);
    k.x = a->x; k.w = a->weight; k.bias = a->bias; k.state_in = a->state_in;
    return k;
}
// how the rows of all the tensors lie
int lie_of(const wkv_causal_conv_args_t *a, std::initializer_list<const void *> ptrs) {
    const int size = elem_size(a->dtype);
    auto multiples = [&](int elements) {
        for (const void *p : ptrs)
            if (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(elements * size - 1)) return false;
        return a->D % elements == 0 && a->x_token % elements == 0 && a->x_batch % elements == 0;
    };
    return multiples(V) ? RUNS : multiples(4 / size) ? WORDS : ONES;
}

// f is called with the way the rows lie (fp32 rows always start at multiples of 4 bytes)
template <typename F, class Fn>
int by_lie(int lie, Fn f) {
    if (lie == RUNS) return f(std::integral_constant<int, RUNS>{});
    if (lie == WORDS || sizeof(F) == 4) return f(std::integral_constant<int, WORDS>{});
    return f(std::integral_constant<int, sizeof(F) == 4 ? WORDS : ONES>{});
}

template <class Fn>
int by_width(int W, Fn f) {
    switch (W) {
        case 2: return f(std::integral_constant<int, 2>{});
        case 3: return f(std::integral_constant<int, 3>{});
        default: return f(std::integral_constant<int, 4>{});
    }
}

// threads of a CTA: few of them where that gives every SM one
int threads_for(int runs, long long strips) {
    int nt = 256;
    while (nt > 32 && (runs + nt - 1) / nt * strips < device_sm_count()) nt /= 2;
    return nt;
}

}  // namespace
}  // namespace wkv

using namespace wkv;

extern "C" int wkv_causal_conv_forward(const wkv_causal_conv_args_t *a, void *stream) {
    int e = check_conv(a);
    if (e != WKV_OK) return e;
    if (a->B == 0 || a->D == 0) return WKV_OK;
    if (a->T > 0 && !a->y) return WKV_ERR_NULL;
    // (a thread of the first strip reads the state after one of the last strip has written it)
    if (a->T > SHORTEST && a->state_in && a->state_in == a->state_out) return WKV_ERR_UNSUPPORTED;
    ConvArgs k = conv_args(a);
    k.y = a->y; k.state_out = a->state_out;
    const int lie = lie_of(a, {a->x, a->state_in, a->y, a->state_out});
    k.strip = strip_for(a->B, a->T, a->D, FWD_THREADS, FWD_LONGEST);
    k.nstrip = a->T > 0 ? (a->T + k.strip - 1) / k.strip : 1;
    const int runs = lie == RUNS ? a->D / V : (a->D + 32 * V - 1) / (32 * V) * 32, nt = threads_for(runs, (long long)a->B * k.nstrip);
    return by_dtype(a->dtype, [&](auto f) {
        using F = decltype(f);
        return by_width(a->W, [&](auto w) {
            return by_lie<F>(lie, [&](auto m) {
                constexpr auto kern = k_conv_fwd<F, decltype(w)::value, decltype(m)::value>;
                constexpr int BYTES = FWD_AHEAD * FWD_GT * (int)sizeof(Raw<F, V>);       // a thread's ring
                static unsigned char done[64];
                if (!set_max_smem_once(kern, 256 * BYTES, done)) return (int)WKV_ERR_LAUNCH;
                return launch_chained(kern, dim3(a->B * k.nstrip, (runs + nt - 1) / nt), dim3(nt), nt * BYTES, (cudaStream_t)stream, k);
            });
        });
    });
}

extern "C" size_t wkv_causal_conv_backward_workspace(const wkv_causal_conv_args_t *a) {
    if (check_conv(a) != WKV_OK || a->B == 0 || a->D == 0 || a->T == 0) return 0;
    const int strip = strip_for(a->B, a->T, a->D, BWD_THREADS, BWD_LONGEST);
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
        const int lie = lie_of(a, {a->x, a->state_in, a->gy, a->gstate_out, a->gx, a->gstate_in});
        k.strip = strip_for(a->B, a->T, a->D, BWD_THREADS, BWD_LONGEST);
        k.nstrip = a->T > 0 ? (a->T + k.strip - 1) / k.strip : 1;
        if (params && a->T > 0) {
            if (!a->workspace || a->workspace_bytes < wkv_causal_conv_backward_workspace(a)) return WKV_ERR_WORKSPACE;
            if (!aligned16(a->workspace)) return WKV_ERR_ALIGN;
            k.part = (float *)a->workspace;
            rows = a->B * k.nstrip;
        }
        const int runs = lie == RUNS ? a->D / V : (a->D + 32 * V - 1) / (32 * V) * 32, nt = threads_for(runs, (long long)a->B * k.nstrip);
        e = by_dtype(a->dtype, [&](auto f) {
            using F = decltype(f);
            return by_width(a->W, [&](auto w) {
                return by_lie<F>(lie, [&](auto m) {
                    constexpr auto kern = k_conv_bwd<F, decltype(w)::value, decltype(m)::value>;
                    constexpr int BYTES = BWD_AHEAD * BWD_GT * 2 * (int)sizeof(Raw<F, V>);       // a thread's ring
                    static unsigned char done[64];
                    if (!set_max_smem_once(kern, 256 * BYTES, done)) return (int)WKV_ERR_LAUNCH;
                    return launch_chained(kern, dim3(a->B * k.nstrip, (runs + nt - 1) / nt), dim3(nt), nt * BYTES, s, k);
                });
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
