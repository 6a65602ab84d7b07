// Gated linear recurrence, forward and backward: one state per channel, its decay and its input behind gates.
//
//   r_t = sigmoid(decay_gate_t),  i_t = sigmoid(input_gate_t),  L_t = -c softplus(decay) r_t,  a_t = exp(L_t),
//   m_t = sqrt(1 - a_t^2),  h_t = a_t h_{t-1} + m_t i_t x_t,  y_t = h_t silu(z_t)      (without z: y_t = h_t)
//
//   backward, with d = gy silu(z) and E_t = a_t G_t what token t sends to h_{t-1}:
//   G_t = d_t + E_{t+1},  gx = G m i,  ginput_gate = G m x i (1 - i),  gz = gy h silu'(z)
//   gL L = G (h_{t-1} a L - i x a^2 L / m),  gdecay_gate = gL L (1 - r),  gdecay = sum_t gL L  sigmoid(decay) / softplus(decay)
//   (dm/dL = -a^2 / m has no bound where a is near 1; L dm/dL goes to zero there, and only that product is formed)
//
// Bound by HBM: five elements a token and channel forward (two fewer... none are read twice), nine and four backward.  A CTA
// owns 64 channels of a row (two a lane) and walks over its tokens in blocks of 8 warps x S tokens.  A warp's S tokens are a
// segment: from zero its state is hl and its decay P = prod a; the eight segments' (P, hl) meet in shared memory, every thread
// folds them in order (one barrier a block) and runs its segment again from the state that it then knows, its a and m i x still
// in registers.  So the serial chain is 8 + S steps a block, and the gates, which are most of the work, are formed once.
// A warp's inputs come through a ring of its own in shared memory (cp.async), the blocks behind on their way meanwhile.
//
// Few chains: the CTAs of a cluster take neighbouring blocks of one row and exchange their folds through distributed shared
// memory (one cluster barrier a step); nothing is read twice and nothing is waited for in global memory.
//
// Backward: blocks in reverse.  The forward pass leaves the state before each block (4 bytes a channel per 8 S tokens); hl and
// P are formed again, and with them the segment's E from zero, so that one exchange serves both directions.
//
// 1 - a^2 is -expm1(2L): its series below 1/4 (2^-24 of it are left out there), 1 - a a above.
#include <cooperative_groups.h>

#include "elem_io.cuh"
#include "wkv_internal.h"

namespace cg = cooperative_groups;

namespace wkv {
namespace {

constexpr int CH = 64, NW = 8, MAX_CL = 8;
constexpr float LOG2E_ = 1.4426950408889634f, LN2_ = 0.6931471805599453f;
// the mean error of ex2 over exponents from -0.5 to -0.01, made good in its argument (selective_scan.cu)
constexpr float EX2_MEAN_ = 1.8e-8f;

__device__ __forceinline__ float ex2a(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcpa(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rsqrta(float x) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float sig(float x) { return rcpa(1.f + ex2a(-LOG2E_ * x)); }

struct RecArgs {
    int T, D, slabs, cl, nsteps;          // slabs of CH channels; cl: CTAs of a cluster, nsteps: blocks of a row / cl, rounded up
    float c;
    const void *x, *ig, *rg, *z;
    long long x_batch, x_token, ig_batch, ig_token, rg_batch, rg_token, z_batch, z_token;
    const float *decay, *state_in;
    void *y;
    float *state_out, *ckpt;              // ckpt [B, nsteps * cl, D]
    const void *gy;
    const float *gs_out;
    void *gx, *gig, *grg, *gz;
    float *gs_in, *part;                  // part [B * cl, D]
};

// Tokens of a warp in a block, and shared memory, for two CTAs an SM.
template <typename F>
struct Geo {
    static constexpr int S = sizeof(F) == 2 ? 8 : 4, BT = NW * S, SLOT = BT * CH;        // SLOT: elements of one tensor's block
    static constexpr int FWD_STAGES = 3, BWD_STAGES = 2;
    static constexpr int fwd_ring(bool z) { return FWD_STAGES * (3 + z) * SLOT * (int)sizeof(F); }
    static constexpr int bwd_ring(bool z) { return BWD_STAGES * (4 + z) * SLOT * (int)sizeof(F); }
};

// softplus(p) and its derivative over it, once per CTA and channel
struct Rate {
    float rate2, x2, ratio;               // L log2(e) = rate2 r;  -2 L = x2 r;  sigmoid(p) / softplus(p)
};
__device__ __forceinline__ Rate rate_of(float p, float c) {
    const float t = expf(-fabsf(p)), s = fmaxf(p, 0.f) + log1pf(t), sg = p >= 0.f ? 1.f / (1.f + t) : t / (1.f + t);
    Rate r;
    // (an infinite rate becomes the largest one: a decay gate of zero then keeps the state; a NaN stays)
    float k = c * s;
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(k) : "f"(1.1e38f));
    r.rate2 = -k * LOG2E_;
    r.x2 = 2.f * k;
    r.ratio = s > 1e-30f ? sg / s : (s == s ? 1.f : s);
    return r;
}

// the gates of a token: decay a, 1 - a^2
__device__ __forceinline__ float one_minus_square(float a, float x2) {
    float p = fmaf(x2, -1.f / 720.f, 1.f / 120.f);
    p = fmaf(x2, p, -1.f / 24.f);
    p = fmaf(x2, p, 1.f / 6.f);
    p = fmaf(x2, p, -0.5f);
    p = fmaf(x2, p, 1.f) * x2;
    return x2 < 0.25f ? p : fmaf(-a, a, 1.f);
}

template <int BYTES>
__device__ __forceinline__ void cp_async(void *smem, const void *g, int valid) {
    const uint32_t s = (uint32_t)__cvta_generic_to_shared(smem);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s), "l"(g), "r"(valid) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(s), "l"(g), "r"(valid) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// How rows lie: pieces of 16 bytes, words, or (two-byte elements) anywhere.
enum { PIECES = 0, WORDS = 1, ANYWHERE = 2 };

// A warp's S tokens of one tensor -> its slot [S][CH] of the ring.  Tokens from `n` on and channels from D on become zeros.
template <typename F, int MODE>
__device__ __forceinline__ void fill(F *slot, const F *row, long long token, int n, int ch0, int D, int lane) {
    constexpr int S = Geo<F>::S;
    if constexpr (MODE == PIECES) {
        constexpr int PER = 16 / sizeof(F), ROWP = CH / PER;
#pragma unroll
        for (int k = 0; k < S * ROWP / 32; k++) {
            const int i = lane + 32 * k, s = i / ROWP, e = (i % ROWP) * PER;
            const bool ok = s < n && ch0 + e < D;
            cp_async<16>(slot + s * CH + e, ok ? row + s * token + e : row, ok ? 16 : 0);
        }
    } else if constexpr (MODE == WORDS) {
#pragma unroll
        for (int s = 0; s < S; s++) {
            const int e = 2 * lane, left = D - ch0 - e;
            const bool ok = s < n && left > 0;
            const F *p = ok ? row + s * token + e : row;
            if constexpr (sizeof(F) == 2) {
                cp_async<4>(slot + s * CH + e, p, ok ? min(left, 2) * 2 : 0);
            } else {
                cp_async<4>(slot + s * CH + e, p, ok ? 4 : 0);
                cp_async<4>(slot + s * CH + e + 1, ok && left > 1 ? p + 1 : row, ok && left > 1 ? 4 : 0);
            }
        }
    } else {
        uint32_t w[S];
#pragma unroll
        for (int s = 0; s < S; s++) {
            const int e = 2 * lane, left = D - ch0 - e;
            const uint16_t *p = reinterpret_cast<const uint16_t *>(row + s * token + e);
            w[s] = 0;
            if (s < n && left > 0) w[s] = p[0];
            if (s < n && left > 1) w[s] |= (uint32_t)p[1] << 16;
        }
#pragma unroll
        for (int s = 0; s < S; s++) *reinterpret_cast<uint32_t *>(slot + s * CH + 2 * lane) = w[s];
    }
}
template <typename F>
__device__ __forceinline__ f2 pair_at(const F *slot, int s, int lane) {
    Raw<F, 2> r;
    r.load(slot + s * CH + 2 * lane, true, 2);
    float f[2];
    r.get(f);
    return make_float2(f[0], f[1]);
}
// The state before a token, in the places of its two gates (which are in registers by then): a lane's own.
template <typename F>
__device__ __forceinline__ void keep_state(F *slot, int next, int s, int lane, f2 h) {
    if constexpr (sizeof(F) == 4) {
        *reinterpret_cast<f2 *>(slot + s * CH + 2 * lane) = h;
    } else {
        *reinterpret_cast<float *>(slot + s * CH + 2 * lane) = h.x;
        *reinterpret_cast<float *>(slot + next + s * CH + 2 * lane) = h.y;
    }
}
template <typename F>
__device__ __forceinline__ f2 kept_state(const F *slot, int next, int s, int lane) {
    if constexpr (sizeof(F) == 4) return *reinterpret_cast<const f2 *>(slot + s * CH + 2 * lane);
    else return make_float2(*reinterpret_cast<const float *>(slot + s * CH + 2 * lane), *reinterpret_cast<const float *>(slot + next + s * CH + 2 * lane));
}
// decay gates of minus infinity for the tokens behind the row's last: they keep the state (x is zero there)
template <typename F>
__device__ __forceinline__ void close_gates(F *slot, int n, int lane) {
    for (int s = max(n, 0); s < Geo<F>::S; s++) {
        const float f[2] = {-INFINITY, -INFINITY};
        Raw<F, 2> r;
        r.put(f);
        r.store(slot + s * CH + 2 * lane, true, 2);
    }
}
template <typename F>
__device__ __forceinline__ void store_out(F *p, f2 v, bool pair, int left) {
    const float f[2] = {v.x, v.y};
    Raw<F, 2> r;
    r.put(f);
    r.store(p, pair, left);
}

// what a segment does to the state (and to E): [side][segment][channel pair]
struct Exchange {
    float4 seg[2][NW][32];                // P, hl of two channels
    float4 cta[2][MAX_CL][32];            // the same of the cluster's CTAs
};
struct ExchangeBack {
    float4 seg[2][NW][32];                // P, hl
    f2 segE[2][NW][32];                   // E from zero
    float4 cta[2][MAX_CL][32];            // P, E of the cluster's CTAs
    f2 sum[NW][32];
};

template <typename F, bool Z, int MODE>
__global__ void __launch_bounds__(256, 2) k_rec_fwd(const RecArgs g) {
    pdl_wait();
    pdl_trigger();
    constexpr int S = Geo<F>::S, BT = Geo<F>::BT, SLOT = Geo<F>::SLOT, NT = 3 + Z, ST = Geo<F>::FWD_STAGES, RING = ST * NT * SLOT * (int)sizeof(F);
    extern __shared__ __align__(16) unsigned char smem[];
    Exchange &ex = *reinterpret_cast<Exchange *>(smem + RING);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = blockIdx.x % g.cl, chain = blockIdx.x / g.cl, b = chain / g.slabs, ch0 = (chain - b * g.slabs) * CH, ch = ch0 + 2 * lane;
    F *ring = reinterpret_cast<F *>(smem) + warp * S * CH;          // [stage][tensor][warp][S][CH]

    const Rate k0 = rate_of(ch < g.D ? g.decay[ch] : 0.f, g.c), k1 = rate_of(ch + 1 < g.D ? g.decay[ch + 1] : 0.f, g.c);
    f2 h = make_float2(0.f, 0.f);
    if (g.state_in != nullptr) {
        if (ch < g.D) h.x = g.state_in[(size_t)b * g.D + ch];
        if (ch + 1 < g.D) h.y = g.state_in[(size_t)b * g.D + ch + 1];
    }
    auto start = [&](int step) {
        const long long t0 = ((long long)step * g.cl + rank) * BT + warp * S;
        const int n = (int)max(0ll, min((long long)S, g.T - t0));
        const long long at = n > 0 ? t0 : 0;
        F *slot = ring + (step % ST) * NT * SLOT;
        fill<F, MODE>(slot, (const F *)g.rg + b * g.rg_batch + at * g.rg_token + ch0, g.rg_token, n, ch0, g.D, lane);
        fill<F, MODE>(slot + SLOT, (const F *)g.ig + b * g.ig_batch + at * g.ig_token + ch0, g.ig_token, n, ch0, g.D, lane);
        fill<F, MODE>(slot + 2 * SLOT, (const F *)g.x + b * g.x_batch + at * g.x_token + ch0, g.x_token, n, ch0, g.D, lane);
        if (Z) fill<F, MODE>(slot + 3 * SLOT, (const F *)g.z + b * g.z_batch + at * g.z_token + ch0, g.z_token, n, ch0, g.D, lane);
    };
#pragma unroll
    for (int p = 0; p < ST - 1; p++) {
        if (p < g.nsteps) start(p);
        cp_commit();
    }
    const bool pair = (g.D & 1) == 0;
    for (int step = 0; step < g.nsteps; step++) {
        __syncwarp();                                               // (all lanes are done with the slot that is filled now)
        if (step + ST - 1 < g.nsteps) start(step + ST - 1);
        cp_commit();
        cp_wait<ST - 1>();
        __syncwarp();
        F *slot = ring + (step % ST) * NT * SLOT;
        const long long blk = (long long)step * g.cl + rank, t0 = blk * BT + warp * S;
        const int n = (int)max(0ll, min((long long)S, g.T - t0));
        if (n < S) close_gates(slot, n, lane);
        f2 a[S], v[S], P = both(1.f), hl = both(0.f);
#pragma unroll
        for (int s = 0; s < S; s++) {
            const f2 rg = pair_at(slot, s, lane), ig = pair_at(slot + SLOT, s, lane), x = pair_at(slot + 2 * SLOT, s, lane);
            const float r0 = sig(rg.x), r1 = sig(rg.y);
            a[s] = make_float2(ex2a(fmaf(r0, k0.rate2, EX2_MEAN_)), ex2a(fmaf(r1, k1.rate2, EX2_MEAN_)));
            const f2 m = make_float2(sqrtf(one_minus_square(a[s].x, r0 * k0.x2)), sqrtf(one_minus_square(a[s].y, r1 * k1.x2)));
            v[s] = mul2(mul2(m, make_float2(sig(ig.x), sig(ig.y))), x);
            hl = fma2(a[s], hl, v[s]);
            P = mul2(P, a[s]);
        }
        const int side = step & 1;
        ex.seg[side][warp][lane] = make_float4(P.x, P.y, hl.x, hl.y);
        __syncthreads();
        f2 hs = h;                                                  // before this warp's segment
        if (g.cl == 1) {
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const float4 q = ex.seg[side][w][lane];
                if (w == warp) hs = h;
                h = fma2(make_float2(q.x, q.y), h, make_float2(q.z, q.w));
            }
            if (g.ckpt != nullptr && warp == 0) {
                float *c = g.ckpt + ((size_t)b * g.nsteps + blk) * g.D + ch;
                if (ch < g.D) c[0] = hs.x;
                if (ch + 1 < g.D) c[1] = hs.y;
            }
        } else {
            f2 Pc = both(1.f), hc = both(0.f), Pw = both(1.f), hw = both(0.f);
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const float4 q = ex.seg[side][w][lane];
                if (w == warp) { Pw = Pc; hw = hc; }
                hc = fma2(make_float2(q.x, q.y), hc, make_float2(q.z, q.w));
                Pc = mul2(Pc, make_float2(q.x, q.y));
            }
            cg::cluster_group cl = cg::this_cluster();
            if (warp < g.cl) {
                Exchange *to = cl.map_shared_rank(&ex, warp);
                to->cta[side][rank][lane] = make_float4(Pc.x, Pc.y, hc.x, hc.y);
            }
            cl.sync();
            f2 hr = h;
            for (int q = 0; q < g.cl; q++) {
                const float4 e = ex.cta[side][q][lane];
                if (q == rank) hr = h;
                h = fma2(make_float2(e.x, e.y), h, make_float2(e.z, e.w));
            }
            hs = fma2(Pw, hr, hw);
            if (g.ckpt != nullptr && warp == 0) {
                float *c = g.ckpt + ((size_t)b * g.nsteps * g.cl + blk) * g.D + ch;
                if (ch < g.D) c[0] = hr.x;
                if (ch + 1 < g.D) c[1] = hr.y;
            }
        }
        if (ch < g.D) {
            F *y = (F *)g.y + ((size_t)b * g.T + t0) * g.D + ch;
#pragma unroll
            for (int s = 0; s < S; s++) {
                hs = fma2(a[s], hs, v[s]);
                f2 o = hs;
                if (Z) {
                    const f2 z = pair_at(slot + 3 * SLOT, s, lane);
                    o = mul2(o, mul2(z, make_float2(sig(z.x), sig(z.y))));
                }
                if (s < n) store_out(y + (size_t)s * g.D, o, pair, g.D - ch);
            }
        }
    }
    if (g.cl > 1) cg::this_cluster().sync();                        // (no CTA leaves while another may write to it)
    if (g.state_out != nullptr && warp == 0 && rank == 0) {
        if (ch < g.D) g.state_out[(size_t)b * g.D + ch] = h.x;
        if (ch + 1 < g.D) g.state_out[(size_t)b * g.D + ch + 1] = h.y;
    }
}

template <typename F, bool Z, int MODE>
__global__ void __launch_bounds__(256, 2) k_rec_bwd(const RecArgs g) {
    pdl_wait();
    pdl_trigger();
    constexpr int S = Geo<F>::S, BT = Geo<F>::BT, SLOT = Geo<F>::SLOT, NT = 4 + Z, ST = Geo<F>::BWD_STAGES, RING = ST * NT * SLOT * (int)sizeof(F);
    extern __shared__ __align__(16) unsigned char smem[];
    ExchangeBack &ex = *reinterpret_cast<ExchangeBack *>(smem + RING);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rank = blockIdx.x % g.cl, chain = blockIdx.x / g.cl, b = chain / g.slabs, ch0 = (chain - b * g.slabs) * CH, ch = ch0 + 2 * lane;
    F *ring = reinterpret_cast<F *>(smem) + warp * S * CH;

    const Rate k0 = rate_of(ch < g.D ? g.decay[ch] : 0.f, g.c), k1 = rate_of(ch + 1 < g.D ? g.decay[ch + 1] : 0.f, g.c);
    const f2 rate = make_float2(k0.rate2, k1.rate2);
    f2 E = make_float2(0.f, 0.f), total = make_float2(0.f, 0.f);
    if (g.gs_out != nullptr) {
        if (ch < g.D) E.x = g.gs_out[(size_t)b * g.D + ch];
        if (ch + 1 < g.D) E.y = g.gs_out[(size_t)b * g.D + ch + 1];
    }
    // (k counts the steps in the order of the walk)
    auto start = [&](int k) {
        const int step = g.nsteps - 1 - k;
        const long long t0 = ((long long)step * g.cl + rank) * BT + warp * S;
        const int n = (int)max(0ll, min((long long)S, g.T - t0));
        const long long at = n > 0 ? t0 : 0;
        F *slot = ring + (k % ST) * NT * SLOT;
        fill<F, MODE>(slot, (const F *)g.rg + b * g.rg_batch + at * g.rg_token + ch0, g.rg_token, n, ch0, g.D, lane);
        fill<F, MODE>(slot + SLOT, (const F *)g.ig + b * g.ig_batch + at * g.ig_token + ch0, g.ig_token, n, ch0, g.D, lane);
        fill<F, MODE>(slot + 2 * SLOT, (const F *)g.x + b * g.x_batch + at * g.x_token + ch0, g.x_token, n, ch0, g.D, lane);
        // (no incoming gradient: zeros)
        fill<F, MODE>(slot + 3 * SLOT, g.gy != nullptr ? (const F *)g.gy + ((size_t)b * g.T + at) * g.D + ch0 : (const F *)g.x, g.D,
                      g.gy != nullptr ? n : 0, ch0, g.D, lane);
        if (Z) fill<F, MODE>(slot + 4 * SLOT, (const F *)g.z + b * g.z_batch + at * g.z_token + ch0, g.z_token, n, ch0, g.D, lane);
    };
#pragma unroll
    for (int p = 0; p < ST - 1; p++) {
        if (p < g.nsteps) start(p);
        cp_commit();
    }
    const bool pair = (g.D & 1) == 0;
    for (int k = 0; k < g.nsteps; k++) {
        __syncwarp();
        if (k + ST - 1 < g.nsteps) start(k + ST - 1);
        cp_commit();
        const int step = g.nsteps - 1 - k;
        const long long blk = (long long)step * g.cl + rank, t0 = blk * BT + warp * S;
        f2 h = make_float2(0.f, 0.f);                               // before the block
        {
            const float *c = g.ckpt + ((size_t)b * g.nsteps * g.cl + blk) * g.D + ch;
            if (ch < g.D) h.x = c[0];
            if (ch + 1 < g.D) h.y = c[1];
        }
        cp_wait<ST - 1>();
        __syncwarp();
        F *slot = ring + (k % ST) * NT * SLOT;
        const int n = (int)max(0ll, min((long long)S, g.T - t0));
        if (n < S) close_gates(slot, n, lane);
        f2 a[S], r[S], in[S], rs[S], P = both(1.f), hl = both(0.f), El = both(0.f);
#pragma unroll
        for (int s = 0; s < S; s++) {
            const f2 rg = pair_at(slot, s, lane), ig = pair_at(slot + SLOT, s, lane), x = pair_at(slot + 2 * SLOT, s, lane);
            r[s] = make_float2(sig(rg.x), sig(rg.y));
            in[s] = make_float2(sig(ig.x), sig(ig.y));
            a[s] = make_float2(ex2a(fmaf(r[s].x, k0.rate2, EX2_MEAN_)), ex2a(fmaf(r[s].y, k1.rate2, EX2_MEAN_)));
            const f2 q = make_float2(one_minus_square(a[s].x, r[s].x * k0.x2), one_minus_square(a[s].y, r[s].y * k1.x2));
            // 1 / m; where m is zero, so are L and m / that
            rs[s] = make_float2(rsqrta(q.x > 1e-37f ? q.x : (q.x == q.x ? 1e-37f : q.x)), rsqrta(q.y > 1e-37f ? q.y : (q.y == q.y ? 1e-37f : q.y)));
            hl = fma2(a[s], hl, mul2(mul2(mul2(q, rs[s]), in[s]), x));
            P = mul2(P, a[s]);
        }
        f2 sz[Z ? S : 1];
#pragma unroll
        for (int s = S - 1; s >= 0; s--) {
            f2 d = pair_at(slot + 3 * SLOT, s, lane);
            if (Z) {
                const f2 z = pair_at(slot + 4 * SLOT, s, lane);
                sz[s] = make_float2(sig(z.x), sig(z.y));
                d = mul2(d, mul2(z, sz[s]));
            }
            El = mul2(a[s], add2(d, El));
        }
        const int side = k & 1;
        ex.seg[side][warp][lane] = make_float4(P.x, P.y, hl.x, hl.y);
        ex.segE[side][warp][lane] = El;
        __syncthreads();
        f2 Es = E;                                                  // behind this warp's segment
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float4 q = ex.seg[side][w][lane];
            if (w < warp) h = fma2(make_float2(q.x, q.y), h, make_float2(q.z, q.w));
        }
        if (g.cl == 1) {
#pragma unroll
            for (int w = NW - 1; w >= 0; w--) {
                const float4 q = ex.seg[side][w][lane];
                if (w == warp) Es = E;
                E = fma2(make_float2(q.x, q.y), E, ex.segE[side][w][lane]);
            }
        } else {
            f2 Pc = both(1.f), Ec = both(0.f), Pw = both(1.f), Ew = both(0.f);
#pragma unroll
            for (int w = NW - 1; w >= 0; w--) {
                const float4 q = ex.seg[side][w][lane];
                if (w == warp) { Pw = Pc; Ew = Ec; }
                Ec = fma2(make_float2(q.x, q.y), Ec, ex.segE[side][w][lane]);
                Pc = mul2(Pc, make_float2(q.x, q.y));
            }
            cg::cluster_group cl = cg::this_cluster();
            if (warp < g.cl) {
                ExchangeBack *to = cl.map_shared_rank(&ex, warp);
                to->cta[side][rank][lane] = make_float4(Pc.x, Pc.y, Ec.x, Ec.y);
            }
            cl.sync();
            f2 Er = E;
            for (int q = g.cl - 1; q >= 0; q--) {
                const float4 e = ex.cta[side][q][lane];
                if (q == rank) Er = E;
                E = fma2(make_float2(e.x, e.y), E, make_float2(e.z, e.w));
            }
            Es = fma2(Pw, Er, Ew);
        }
#pragma unroll
        for (int s = 0; s < S; s++) {
            keep_state(slot, SLOT, s, lane, h);
            const f2 x = pair_at(slot + 2 * SLOT, s, lane);
            const f2 q = make_float2(one_minus_square(a[s].x, r[s].x * k0.x2), one_minus_square(a[s].y, r[s].y * k1.x2));
            h = fma2(a[s], h, mul2(mul2(mul2(q, rs[s]), in[s]), x));
        }
#pragma unroll
        for (int s = S - 1; s >= 0; s--) {
            const f2 x = pair_at(slot + 2 * SLOT, s, lane), gy = pair_at(slot + 3 * SLOT, s, lane), hb = kept_state(slot, SLOT, s, lane);
            const f2 q = make_float2(one_minus_square(a[s].x, r[s].x * k0.x2), one_minus_square(a[s].y, r[s].y * k1.x2));
            const f2 m = mul2(q, rs[s]), ix = mul2(in[s], x), mi = mul2(m, in[s]), L = mul2(r[s], rate);
            f2 d = gy, gz = both(0.f);
            if (Z) {
                const f2 z = pair_at(slot + 4 * SLOT, s, lane);
                const f2 hn = fma2(a[s], hb, mul2(m, ix));
                d = mul2(d, mul2(z, sz[s]));
                // silu' = s (1 + z (1 - s))
                gz = mul2(mul2(gy, hn), mul2(sz[s], fma2(z, sub2(both(1.f), sz[s]), both(1.f))));
            }
            const f2 G = add2(d, Es), aL = mul2(a[s], L);
            Es = mul2(a[s], G);
            const f2 gx = mul2(G, mi), gi = mul2(mul2(mul2(G, m), ix), sub2(both(1.f), in[s]));
            // G (h a L - i x a^2 L / m)
            const f2 gLL = mul2(G, sub2(mul2(hb, aL), mul2(ix, mul2(mul2(a[s], aL), rs[s]))));
            total = add2(total, gLL);
            const f2 gr = mul2(mul2(gLL, both(LN2_)), sub2(both(1.f), r[s]));
            if (s < n && ch < g.D) {
                const size_t at = ((size_t)b * g.T + t0 + s) * g.D + ch;
                if (g.gx != nullptr) store_out((F *)g.gx + at, gx, pair, g.D - ch);
                if (g.gig != nullptr) store_out((F *)g.gig + at, gi, pair, g.D - ch);
                if (g.grg != nullptr) store_out((F *)g.grg + at, gr, pair, g.D - ch);
                if (Z && g.gz != nullptr) store_out((F *)g.gz + at, gz, pair, g.D - ch);
            }
        }
    }
    if (g.cl > 1) cg::this_cluster().sync();
    if (g.gs_in != nullptr && warp == 0 && rank == 0) {
        if (ch < g.D) g.gs_in[(size_t)b * g.D + ch] = E.x;
        if (ch + 1 < g.D) g.gs_in[(size_t)b * g.D + ch + 1] = E.y;
    }
    if (g.part != nullptr) {
        ex.sum[warp][lane] = total;
        __syncthreads();
        if (warp == 0) {
#pragma unroll
            for (int w = 1; w < NW; w++) total = add2(total, ex.sum[w][lane]);
            float *p = g.part + ((size_t)b * g.cl + rank) * g.D + ch;
            if (ch < g.D) p[0] = total.x * (LN2_ * k0.ratio);
            if (ch + 1 < g.D) p[1] = total.y * (LN2_ * k1.ratio);
        }
    }
}

// One token: a thread takes two channels, the state is updated in place.
template <typename F>
__global__ void __launch_bounds__(128) k_rec_step(const RecArgs g, long long pairs, int row_pairs, bool vec) {
    pdl_wait();
    pdl_trigger();
    const long long i = (long long)blockIdx.x * 128 + threadIdx.x;
    if (i >= pairs) return;
    const int b = (int)(i / row_pairs), ch = 2 * (int)(i % row_pairs), n = min(2, g.D - ch);
    auto in = [&](const void *p, long long batch) {
        Raw<F, 2> r;
        r.load((const F *)p + b * batch + ch, vec, n);
        float f[2];
        r.get(f);
        return make_float2(f[0], f[1]);
    };
    const f2 x = in(g.x, g.x_batch), ig = in(g.ig, g.ig_batch), rg = in(g.rg, g.rg_batch);
    f2 z = both(0.f);
    if (g.z != nullptr) z = in(g.z, g.z_batch);
    const size_t at = (size_t)b * g.D + ch;
    f2 h = both(0.f);
    if (g.state_in != nullptr) h = make_float2(g.state_in[at], n > 1 ? g.state_in[at + 1] : 0.f);
    auto one = [&](float h, float x, float ig, float rg, float p) {
        const Rate k = rate_of(p, g.c);
        const float r = sig(rg), a = ex2a(fmaf(r, k.rate2, EX2_MEAN_)), m = sqrtf(one_minus_square(a, r * k.x2));
        return fmaf(a, h, m * sig(ig) * x);
    };
    h = make_float2(one(h.x, x.x, ig.x, rg.x, g.decay[ch]), n > 1 ? one(h.y, x.y, ig.y, rg.y, g.decay[ch + 1]) : 0.f);
    g.state_out[at] = h.x;
    if (n > 1) g.state_out[at + 1] = h.y;
    if (g.z != nullptr) h = mul2(h, mul2(z, make_float2(sig(z.x), sig(z.y))));
    store_out((F *)g.y + at, h, (g.D & 1) == 0 && ((uintptr_t)g.y & (2 * sizeof(F) - 1)) == 0, n);
}

template <typename F> bool lies_in(const wkv_gated_recurrence_args_t *a, size_t bytes, bool back) {
    const long long e = (long long)(bytes / sizeof(F));
    bool ok = true;
    auto look = [&](const void *p, long long batch, long long token) {
        if (p != nullptr) ok = ok && (reinterpret_cast<uintptr_t>(p) % bytes) == 0 && batch % e == 0 && token % e == 0;
    };
    look(a->x, a->x_batch, a->x_token);
    look(a->input_gate, a->i_batch, a->i_token);
    look(a->decay_gate, a->r_batch, a->r_token);
    look(a->z, a->z_batch, a->z_token);
    if (back) look(a->gy, (long long)a->T * a->D, a->D);
    return ok && (bytes == 4 || a->D % e == 0);
}

// CTAs of a cluster: as many as there are places for (two CTAs an SM) and blocks of tokens to take
int cluster_size(const wkv_gated_recurrence_args_t *a) {
    const int bt = a->dtype == WKV_F32 ? Geo<float>::BT : Geo<__half>::BT;
    const long long chains = (long long)a->B * ((a->D + CH - 1) / CH), places = 2ll * device_sm_count(), blocks = ((long long)a->T + bt - 1) / bt;
    int cl = 1;
    while (cl < MAX_CL && chains * cl * 2 <= places && cl * 2 <= blocks) cl *= 2;
    return cl;
}

bool sizes_ok(const wkv_gated_recurrence_args_t *a) {
    return a->B >= 0 && a->T >= 0 && a->D >= 0 && a->D <= (1 << 22) && a->T <= 2147483647 - 4096 && known_dtype(a->dtype) &&
           (long long)a->B * ((a->D + CH - 1) / CH) <= 2147483647 / MAX_CL && (long long)a->B * a->D <= 1ll << 34 && a->c > 0.f;
}
RecArgs args_of(const wkv_gated_recurrence_args_t *a) {
    RecArgs g = {};
    const int bt = a->dtype == WKV_F32 ? Geo<float>::BT : Geo<__half>::BT;
    g.T = a->T; g.D = a->D; g.slabs = (a->D + CH - 1) / CH; g.cl = cluster_size(a);
    g.nsteps = (int)(((long long)a->T + (long long)bt * g.cl - 1) / ((long long)bt * g.cl));
    g.c = a->c;
    g.x = a->x; g.ig = a->input_gate; g.rg = a->decay_gate; g.z = a->z;
    g.x_batch = a->x_batch; g.x_token = a->x_token; g.ig_batch = a->i_batch; g.ig_token = a->i_token;
    g.rg_batch = a->r_batch; g.rg_token = a->r_token; g.z_batch = a->z_batch; g.z_token = a->z_token;
    g.decay = a->decay; g.state_in = a->state_in; g.y = a->y; g.state_out = a->state_out; g.ckpt = (float *)a->ckpt;
    g.gy = a->gy; g.gs_out = a->gstate_out; g.gx = a->gx; g.gig = a->ginput_gate; g.grg = a->gdecay_gate; g.gz = a->gz;
    g.gs_in = a->gstate_in; g.part = (float *)a->workspace;
    return g;
}
size_t ckpt_need(const wkv_gated_recurrence_args_t *a) {
    const RecArgs g = args_of(a);
    return (size_t)a->B * g.nsteps * g.cl * a->D * 4;
}

template <class K>
int launch_rec(K kern, const RecArgs &g, int B, int smem, unsigned char (&done)[64], cudaStream_t s) {
    if (!set_max_smem_once(kern, smem, done)) return WKV_ERR_LAUNCH;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(B * g.slabs * g.cl));
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = g.cl; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g.cl > 1 ? 2 : 1;
    launch_count.fetch_add(1, std::memory_order_relaxed);
    return cudaLaunchKernelEx(&cfg, kern, g) == cudaSuccess ? WKV_OK : WKV_ERR_LAUNCH;
}
template <typename F, bool Z, int MODE, bool BACK>
int launch_as(const RecArgs &g, int B, cudaStream_t s) {
    static unsigned char done[64];
    if constexpr (BACK) return launch_rec(k_rec_bwd<F, Z, MODE>, g, B, Geo<F>::bwd_ring(Z) + (int)sizeof(ExchangeBack), done, s);
    else return launch_rec(k_rec_fwd<F, Z, MODE>, g, B, Geo<F>::fwd_ring(Z) + (int)sizeof(Exchange), done, s);
}
template <bool BACK>
int launch_by(const wkv_gated_recurrence_args_t *a, const RecArgs &g, cudaStream_t s) {
    return by_dtype(a->dtype, [&](auto f) {
        using F = decltype(f);
        const int mode = lies_in<F>(a, 16, BACK) ? PIECES : sizeof(F) == 4 || lies_in<F>(a, 4, BACK) ? WORDS : ANYWHERE;
        auto go = [&](auto zc) {
            constexpr bool Z = decltype(zc)::value;
            if (mode == PIECES) return launch_as<F, Z, PIECES, BACK>(g, a->B, s);
            if constexpr (sizeof(F) == 2) {
                if (mode == ANYWHERE) return launch_as<F, Z, ANYWHERE, BACK>(g, a->B, s);
            }
            return launch_as<F, Z, WORDS, BACK>(g, a->B, s);
        };
        return a->z != nullptr ? go(std::true_type{}) : go(std::false_type{});
    });
}

}  // namespace
}  // namespace wkv

using namespace wkv;

extern "C" size_t wkv_gated_recurrence_ckpt_bytes(const wkv_gated_recurrence_args_t *a) { return a != nullptr && sizes_ok(a) ? ckpt_need(a) : 0; }

extern "C" int wkv_gated_recurrence_forward(const wkv_gated_recurrence_args_t *a, void *stream) {
    if (a == nullptr) return WKV_ERR_NULL;
    if (!known_dtype(a->dtype)) return WKV_ERR_DTYPE;
    if (!sizes_ok(a)) return WKV_ERR_SHAPE;
    if ((long long)a->B * a->D == 0) return WKV_OK;
    if (a->decay == nullptr || a->state_out == nullptr) return WKV_ERR_NULL;
    if (a->T > 0 && (a->x == nullptr || a->input_gate == nullptr || a->decay_gate == nullptr || a->y == nullptr)) return WKV_ERR_NULL;
    RecArgs g = args_of(a);
    const cudaStream_t s = (cudaStream_t)stream;
    if (a->T == 1 && a->ckpt == nullptr) {
        const int row = (a->D + 1) / 2;
        const long long pairs = (long long)a->B * row;
        return by_dtype(a->dtype, [&](auto f) {
            using F = decltype(f);
            return launch_chained(k_rec_step<F>, dim3((unsigned)((pairs + 127) / 128)), dim3(128), 0, s, g, pairs, row,
                                  lies_in<F>(a, 2 * sizeof(F), false) && a->D % 2 == 0);
        });
    }
    if (a->ckpt != nullptr && a->ckpt_bytes < ckpt_need(a)) return WKV_ERR_WORKSPACE;
    return launch_by<false>(a, g, s);
}

extern "C" size_t wkv_gated_recurrence_backward_workspace(const wkv_gated_recurrence_args_t *a) {
    return a != nullptr && sizes_ok(a) && a->gdecay != nullptr ? (size_t)a->B * cluster_size(a) * a->D * 4 : 0;
}

extern "C" int wkv_gated_recurrence_backward(const wkv_gated_recurrence_args_t *a, void *stream) {
    if (a == nullptr) return WKV_ERR_NULL;
    if (!known_dtype(a->dtype)) return WKV_ERR_DTYPE;
    if (!sizes_ok(a)) return WKV_ERR_SHAPE;
    const cudaStream_t s = (cudaStream_t)stream;
    FoldOut out = {};
    out.p[0] = a->gdecay; out.dtype[0] = WKV_F32;
    for (int i = 1; i < 5; i++) out.start[i] = a->D;
    if ((long long)a->B * a->D == 0) return a->gdecay != nullptr && a->D > 0 ? fold_params(nullptr, 0, a->D, out, s) : WKV_OK;
    if (a->decay == nullptr || (a->T > 0 && (a->x == nullptr || a->input_gate == nullptr || a->decay_gate == nullptr))) return WKV_ERR_NULL;
    if (a->T > 0 && (a->ckpt == nullptr || a->ckpt_bytes < ckpt_need(a))) return WKV_ERR_WORKSPACE;
    if (a->gdecay != nullptr && (a->workspace == nullptr || a->workspace_bytes < wkv_gated_recurrence_backward_workspace(a))) return WKV_ERR_WORKSPACE;
    RecArgs g = args_of(a);
    if (a->gdecay == nullptr) g.part = nullptr;
    const int rc = launch_by<true>(a, g, s);
    if (rc != WKV_OK || a->gdecay == nullptr) return rc;
    return fold_params(g.part, a->B * g.cl, a->D, out, s);
}
