// Selective state space scan, forward and backward.  Per channel d and state n, with a row of B and C for each group of
// channels:
//
//   dt_t = softplus(delta_t + bias),  a_t = exp(dt_t A),  h_t = a_t h_{t-1} + dt_t u_t B_t,
//   y_t = (sum_n C_t h_t + D u_t) silu(z_t)
//
//   backward, with dy = gy silu(z) and E_t = a_t G_t what token t sends to h_{t-1}:
//   G_t = C_t dy_t + E_{t+1}
//   gC_t = sum_d h_t dy_t,  gB_t = sum_d G_t dt_t u_t,  gu_t = dt_t (G_t . B_t) + D dy_t
//   gdt_t = u_t (G_t . B_t) + sum_n G_t A a_t h_{t-1},  gA = sum_t G_t dt_t a_t h_{t-1}
//   gz_t = gy_t y_t silu'(z_t)  (y before the gate),  gD = sum dy u,  gdelta = gdt sigmoid(delta + bias)
//
// A thread owns four states of a channel and keeps them in fp32 registers; LPC lanes share a channel (N <= 4 LPC, padded
// states have A = B = C = 0 and stay zero), a warp 32/LPC channels.  Tokens come in blocks of 16: what is per token and
// channel (softplus, gates, loads, stores) is divided among the channel's lanes, lane q taking the tokens that are q mod LPC;
// sums over n are exchanged so that each lane ends with those of its own tokens.  Warps do not wait for one another in the
// forward pass.
//
// Few chains (B x D): the tokens of a row are cut into spans that run in parallel.  The decay over a span is exp(A sum dt),
// so a first pass leaves each span's contribution from zero and sum dt, and the full pass starts from their fold.
//
// The backward pass needs h_t at every token: the forward pass leaves the state before every 16th token (4 N / 16 bytes a
// token and channel), a block is run again from there.
#include "elem_io.cuh"
#include "wkv_internal.h"

namespace wkv {
namespace {

constexpr int TB = 16;               // tokens of a block
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr unsigned FULL_MASK = 0xffffffffu;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct ScanArgs {
    int B, T, D, N, G, Dg, softplus;
    int ncb, nspan, span_blocks, nblk;           // channel blocks per group, spans of a row, their length, blocks of a row
    int vec_b, vec_c;
    const void *u, *delta, *Bm, *Cm, *z;
    long long u_batch, u_token, delta_batch, delta_token, B_batch, B_token, C_batch, C_token, z_batch, z_token;
    const float *A, *Dskip, *bias, *state_in;
    void *y;
    float *state_out, *ckpt;
    float *span_state, *span_dt;                 // [B, nspan, D, N], [B, nspan, D]: a span from zero, its sum of dt
    const void *gy;
    const float *gs_out;
    void *gu, *gdelta, *gz;
    float *gs_in;
    float *part_bc, *part;                       // [ncb, B, T, G, 8 LPC]; [B * nspan, D (N + 2)]
};

// softplus(x) and its derivative sigmoid(x), for any x: with t = e^-|x| no term overflows and log1p keeps small steps exact
__device__ __forceinline__ float softplus(float x, float &sig) {
    const float t = __expf(-fabsf(x)), r = __fdividef(1.f, 1.f + t);
    sig = x >= 0.f ? r : t * r;
    // (fmaxf drops a NaN, log1pf brings it back)
    return fmaxf(x, 0.f) + log1pf(t);
}

// What a warp works on: LPC lanes a channel, lane = c * LPC + q.
template <int LPC>
struct Geo {
    static constexpr int CPW = 32 / LPC;         // channels of a warp
    static constexpr int PT = TB / LPC;          // tokens of a block that are a lane's own
    static constexpr int NP = 4 * LPC;           // states with padding
    static constexpr int NI = (TB * LPC + 31) / 32;      // runs of four of a B or C block that a lane loads
};

// the values of a block that a lane brings in, on their way while the block before is worked on
template <typename F, int LPC>
struct BlockBC {
    Raw<F, 4> b[Geo<LPC>::NI], c[Geo<LPC>::NI];
    __device__ __forceinline__ void load(const ScanArgs &a, int batch, int grp, int t0, int t_end, int lane) {
#pragma unroll
        for (int k = 0; k < Geo<LPC>::NI; k++) {
            const int i = lane + 32 * k, t = t0 + i / LPC, n0 = 4 * (i % LPC), n = min(4, a.N - n0);
            b[k].zero();
            c[k].zero();
            if (i < TB * LPC && t < t_end && n > 0) {
                b[k].load((const F *)a.Bm + (size_t)batch * a.B_batch + (size_t)t * a.B_token + (size_t)grp * a.N + n0, a.vec_b, n);
                c[k].load((const F *)a.Cm + (size_t)batch * a.C_batch + (size_t)t * a.C_token + (size_t)grp * a.N + n0, a.vec_c, n);
            }
        }
    }
    // sB, sC: [TB][NP]
    __device__ __forceinline__ void put(float *sB, float *sC, int lane) const {
#pragma unroll
        for (int k = 0; k < Geo<LPC>::NI; k++) {
            const int i = lane + 32 * k;
            if (i < TB * LPC) {
                float f[4];
                b[k].get(f);
                *reinterpret_cast<float4 *>(sB + 4 * i) = make_float4(f[0], f[1], f[2], f[3]);
                c[k].get(f);
                *reinterpret_cast<float4 *>(sC + 4 * i) = make_float4(f[0], f[1], f[2], f[3]);
            }
        }
    }
};

// v[j] summed over a channel's lanes, for NB tokens j: every lane gets the sum of token q mod NB
template <int LPC, int NB>
__device__ __forceinline__ float sum_tokens(float (&v)[NB], int q) {
#pragma unroll
    for (int m = NB / 2; m > 0; m >>= 1) {
        const bool up = q & m;
#pragma unroll
        for (int j = 0; j < m; j++) {
            const float send = up ? v[j] : v[j + m], keep = up ? v[j + m] : v[j];
            v[j] = keep + __shfl_xor_sync(FULL_MASK, send, m);
        }
    }
    float s = v[0];
#pragma unroll
    for (int m = NB; m < LPC; m <<= 1) s += __shfl_xor_sync(FULL_MASK, s, m);
    return s;
}

__device__ __forceinline__ void load_states(const float *p, size_t at, int n0, int N, float *h) {
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = p != nullptr && n0 + i < N ? p[at + n0 + i] : 0.f;
}
__device__ __forceinline__ void store_states(float *p, size_t at, int n0, int N, const float *h) {
    if (N % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
        if (n0 < N) *reinterpret_cast<float4 *>(p + at + n0) = make_float4(h[0], h[1], h[2], h[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (n0 + i < N) p[at + n0 + i] = h[i];
    }
}

// Forward.  SUMMARY: only the span's contribution from zero and its sum of dt.
template <typename F, int LPC, bool SUMMARY>
__global__ void __launch_bounds__(128) k_scan_fwd(ScanArgs a) {
    pdl_wait();
    pdl_trigger();
    using P = Geo<LPC>;
    __shared__ __align__(16) float2 s_dt[4][TB][P::CPW];
    __shared__ __align__(16) float s_b[4][TB * P::NP], s_c[4][TB * P::NP];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane / LPC, q = lane % LPC;
    // unit = ((batch * spans + span) * G + group) * ncb + channel block
    long long unit = (long long)blockIdx.x * 4 + warp;
    const int cb = (int)(unit % a.ncb);
    unit /= a.ncb;
    const int grp = (int)(unit % a.G);
    unit /= a.G;
    const int nspan = SUMMARY ? a.nspan - 1 : a.nspan;       // (nobody asks for the last span's contribution)
    const int span = (int)(unit % nspan), b = (int)(unit / nspan);
    if (b >= a.B) return;
    const int cg = cb * P::CPW + c, ch = grp * a.Dg + cg, n0 = 4 * q;
    const bool live = cg < a.Dg;
    const size_t row = ((size_t)b * a.D + ch) * a.N;         // of [B, D, N]
    float A2[4], h[4];
    load_states(live ? a.A : nullptr, (size_t)ch * a.N, n0, a.N, A2);
#pragma unroll
    for (int i = 0; i < 4; i++) A2[i] *= LOG2E;
    if (SUMMARY) {
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = 0.f;
    } else {
        load_states(live ? a.state_in : nullptr, row, n0, a.N, h);
        for (int j = 0; j < span; j++) {
            const size_t at = ((size_t)b * a.nspan + j) * a.D + ch;
            float U[4];
            load_states(live ? a.span_state : nullptr, at * a.N, n0, a.N, U);
            const float s = live ? a.span_dt[at] : 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) h[i] = ex2(A2[i] * s) * h[i] + U[i];
        }
    }
    const float bias = live && a.bias ? a.bias[ch] : 0.f, dskip = live && a.Dskip ? a.Dskip[ch] : 0.f;
    const int blk1 = min((span + 1) * a.span_blocks, a.nblk);
    const F *pu = (const F *)a.u + (size_t)b * a.u_batch + ch, *pd = (const F *)a.delta + (size_t)b * a.delta_batch + ch;
    const F *pz = a.z ? (const F *)a.z + (size_t)b * a.z_batch + ch : nullptr;

    F ru[P::PT], rd[P::PT], rz[P::PT];
    BlockBC<F, LPC> bc;
    auto fetch = [&](int blk) {
        if (blk >= blk1) return;
#pragma unroll
        for (int i = 0; i < P::PT; i++) {
            const int t = blk * TB + q + LPC * i;
            if (live && t < a.T) {
                ru[i] = pu[(size_t)t * a.u_token];
                rd[i] = pd[(size_t)t * a.delta_token];
                if (!SUMMARY && pz) rz[i] = pz[(size_t)t * a.z_token];
            }
        }
        bc.load(a, b, grp, blk * TB, a.T, lane);
    };
    fetch(span * a.span_blocks);
    float total = 0.f;                   // SUMMARY: the lane's part of sum dt
    for (int blk = span * a.span_blocks; blk < blk1; blk++) {
        if (!SUMMARY && a.ckpt && live) store_states(a.ckpt, (((size_t)b * a.nblk + blk) * a.D + ch) * a.N, n0, a.N, h);
        float u[P::PT], z[P::PT];
        __syncwarp();                    // (the block before has been read)
#pragma unroll
        for (int i = 0; i < P::PT; i++) {
            const int t = q + LPC * i;
            float dt = 0.f;
            u[i] = 0.f;
            z[i] = 0.f;
            if (live && blk * TB + t < a.T) {
                u[i] = Elem<F>::ld(&ru[i]);
                dt = Elem<F>::ld(&rd[i]) + bias;
                float sig;
                if (a.softplus) dt = softplus(dt, sig);
                if (!SUMMARY && pz) z[i] = Elem<F>::ld(&rz[i]);
            }
            s_dt[warp][t][c] = make_float2(dt, dt * u[i]);
            total += dt;
        }
        bc.put(s_b[warp], s_c[warp], lane);
        __syncwarp();
        fetch(blk + 1);
#pragma unroll
        for (int i = 0; i < P::PT; i++) {
            float yv[LPC];
#pragma unroll
            for (int j = 0; j < LPC; j++) {
                const int t = i * LPC + j;
                const float2 d = s_dt[warp][t][c];
                const float4 Bv = *reinterpret_cast<const float4 *>(&s_b[warp][t * P::NP + n0]);
                h[0] = ex2(d.x * A2[0]) * h[0] + d.y * Bv.x;
                h[1] = ex2(d.x * A2[1]) * h[1] + d.y * Bv.y;
                h[2] = ex2(d.x * A2[2]) * h[2] + d.y * Bv.z;
                h[3] = ex2(d.x * A2[3]) * h[3] + d.y * Bv.w;
                if (!SUMMARY) {
                    const float4 Cv = *reinterpret_cast<const float4 *>(&s_c[warp][t * P::NP + n0]);
                    yv[j] = (Cv.x * h[0] + Cv.y * h[1]) + (Cv.z * h[2] + Cv.w * h[3]);
                }
            }
            if (!SUMMARY) {
                float y = sum_tokens<LPC, LPC>(yv, q) + dskip * u[i];
                if (pz) y *= z[i] * sigmoidf(z[i]);
                const int t = blk * TB + i * LPC + q;
                if (live && t < a.T) Elem<F>::st((F *)a.y + ((size_t)b * a.T + t) * a.D + ch, y);
            }
        }
    }
    if (SUMMARY) {
#pragma unroll
        for (int m = 1; m < LPC; m <<= 1) total += __shfl_xor_sync(FULL_MASK, total, m);
        const size_t at = ((size_t)b * a.nspan + span) * a.D + ch;
        if (live) store_states(a.span_state, at * a.N, n0, a.N, h);
        if (live && q == 0) a.span_dt[at] = total;
    } else if (span == a.nspan - 1 && a.state_out && live) {
        store_states(a.state_out, row, n0, a.N, h);
    }
}

// One token: a thread for four states; state_out may be state_in (each thread reads its own before it writes).
template <typename F, int LPC>
__global__ void __launch_bounds__(256) k_scan_step(ScanArgs a) {
    pdl_wait();
    pdl_trigger();
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) / LPC;
    const int q = threadIdx.x % LPC, n0 = 4 * q;
    const bool live = i < (long long)a.B * a.D;
    const int b = live ? (int)(i / a.D) : 0, ch = live ? (int)(i - (long long)b * a.D) : 0, grp = ch / a.Dg;
    const size_t row = ((size_t)b * a.D + ch) * a.N;
    float h[4], A2[4], Bv[4], Cv[4];
    load_states(live ? a.state_in : nullptr, row, n0, a.N, h);
    load_states(a.A, (size_t)ch * a.N, n0, a.N, A2);
    const F *pB = (const F *)a.Bm + (size_t)b * a.B_batch + (size_t)grp * a.N, *pC = (const F *)a.Cm + (size_t)b * a.C_batch + (size_t)grp * a.N;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        Bv[k] = n0 + k < a.N ? Elem<F>::ld(pB + n0 + k) : 0.f;
        Cv[k] = n0 + k < a.N ? Elem<F>::ld(pC + n0 + k) : 0.f;
    }
    const float u = Elem<F>::ld((const F *)a.u + (size_t)b * a.u_batch + ch);
    float dt = Elem<F>::ld((const F *)a.delta + (size_t)b * a.delta_batch + ch) + (a.bias ? a.bias[ch] : 0.f), sig;
    if (a.softplus) dt = softplus(dt, sig);
    float y = 0.f;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        h[k] = ex2(dt * (A2[k] * LOG2E)) * h[k] + dt * u * Bv[k];
        y += Cv[k] * h[k];
    }
#pragma unroll
    for (int m = 1; m < LPC; m <<= 1) y += __shfl_xor_sync(FULL_MASK, y, m);
    if (!live) return;
    if (a.state_out) store_states(a.state_out, row, n0, a.N, h);
    if (q == 0) {
        if (a.Dskip) y += a.Dskip[ch] * u;
        if (a.z) {
            const float z = Elem<F>::ld((const F *)a.z + (size_t)b * a.z_batch + ch);
            y *= z * sigmoidf(z);
        }
        Elem<F>::st((F *)a.y + (size_t)b * a.D + ch, y);
    }
}

// Backward, summary: what a span sends to the state before it, from zero behind it, and its sum of dt.
template <typename F, int LPC>
__global__ void __launch_bounds__(128) k_scan_bwd_summary(ScanArgs a) {
    pdl_wait();
    pdl_trigger();
    using P = Geo<LPC>;
    __shared__ __align__(16) float2 s_dt[4][TB][P::CPW];
    __shared__ __align__(16) float s_b[4][TB * P::NP], s_c[4][TB * P::NP];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane / LPC, q = lane % LPC;
    long long unit = (long long)blockIdx.x * 4 + warp;
    const int cb = (int)(unit % a.ncb);
    unit /= a.ncb;
    const int grp = (int)(unit % a.G);
    unit /= a.G;
    const int span = 1 + (int)(unit % (a.nspan - 1)), b = (int)(unit / (a.nspan - 1));       // (nobody asks for the first's)
    if (b >= a.B) return;
    const int cg = cb * P::CPW + c, ch = grp * a.Dg + cg, n0 = 4 * q;
    const bool live = cg < a.Dg;
    float A2[4], E[4];
    load_states(live ? a.A : nullptr, (size_t)ch * a.N, n0, a.N, A2);
#pragma unroll
    for (int i = 0; i < 4; i++) { A2[i] *= LOG2E; E[i] = 0.f; }
    const float bias = live && a.bias ? a.bias[ch] : 0.f;
    const F *pd = (const F *)a.delta + (size_t)b * a.delta_batch + ch;
    const F *pg = a.gy ? (const F *)a.gy + (size_t)b * a.T * a.D + ch : nullptr;
    const F *pz = a.z ? (const F *)a.z + (size_t)b * a.z_batch + ch : nullptr;
    const int blk0 = span * a.span_blocks, blk1 = min(blk0 + a.span_blocks, a.nblk);
    F rg[P::PT], rd[P::PT], rz[P::PT];
    BlockBC<F, LPC> bc;
    auto fetch = [&](int blk) {
        if (blk < blk0) return;
#pragma unroll
        for (int i = 0; i < P::PT; i++) {
            const int t = blk * TB + q + LPC * i;
            if (live && t < a.T) {
                if (pg) rg[i] = pg[(size_t)t * a.D];
                rd[i] = pd[(size_t)t * a.delta_token];
                if (pz) rz[i] = pz[(size_t)t * a.z_token];
            }
        }
        bc.load(a, b, grp, blk * TB, a.T, lane);
    };
    fetch(blk1 - 1);
    float total = 0.f;
    for (int blk = blk1 - 1; blk >= blk0; blk--) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < P::PT; i++) {
            const int t = q + LPC * i;
            float dt = 0.f, dy = 0.f;
            if (live && blk * TB + t < a.T) {
                if (pg) dy = Elem<F>::ld(&rg[i]);
                dt = Elem<F>::ld(&rd[i]) + bias;
                float sig;
                if (a.softplus) dt = softplus(dt, sig);
                if (pz) {
                    const float z = Elem<F>::ld(&rz[i]);
                    dy *= z * sigmoidf(z);
                }
            }
            s_dt[warp][t][c] = make_float2(dt, dy);
            total += dt;
        }
        bc.put(s_b[warp], s_c[warp], lane);
        __syncwarp();
        fetch(blk - 1);
#pragma unroll
        for (int t = TB - 1; t >= 0; t--) {
            const float2 d = s_dt[warp][t][c];
            const float4 Cv = *reinterpret_cast<const float4 *>(&s_c[warp][t * P::NP + n0]);
            E[0] = ex2(d.x * A2[0]) * (Cv.x * d.y + E[0]);
            E[1] = ex2(d.x * A2[1]) * (Cv.y * d.y + E[1]);
            E[2] = ex2(d.x * A2[2]) * (Cv.z * d.y + E[2]);
            E[3] = ex2(d.x * A2[3]) * (Cv.w * d.y + E[3]);
        }
    }
#pragma unroll
    for (int m = 1; m < LPC; m <<= 1) total += __shfl_xor_sync(FULL_MASK, total, m);
    const size_t at = ((size_t)b * a.nspan + span) * a.D + ch;
    if (live) store_states(a.span_state, at * a.N, n0, a.N, E);
    if (live && q == 0) a.span_dt[at] = total;
}

// Backward.  The warps of a CTA hold neighbouring channels of one group and one span; they meet once a block to add up what
// they have for gB and gC.
template <int LPC>
struct BwdGeo {
    static constexpr int WARPS = LPC >= 8 ? 4 : 8;
    static constexpr int CH = WARPS * Geo<LPC>::CPW;             // channels of a CTA
    static constexpr int VALUES = 8 * LPC;                       // gB and gC of a token: [8][LPC], state 4 q + (i & 3)
    struct Warp {
        float4 d[TB][Geo<LPC>::CPW];                             // dt, dt u, dy, -
        float b[TB * Geo<LPC>::NP], c[TB * Geo<LPC>::NP];
        float sum[2][TB * VALUES];
    };
    static constexpr int SMEM = WARPS * (int)sizeof(Warp);
};

// the eight values of a lane summed over the warp's channels: what is left, `first` on, is given to put(i, value)
template <int LPC, class Put>
__device__ __forceinline__ void sum_channels(float (&v)[8], int lane, Put put) {
    int first = 0;
    int left = 8;
#pragma unroll
    for (int m = 16, k = 4; m >= LPC; m >>= 1, k >>= 1) {
        if (k >= 1) {
            const bool up = lane & m;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (j < k) {
                    const float send = up ? v[j] : v[j + k], keep = up ? v[j + k] : v[j];
                    v[j] = keep + __shfl_xor_sync(FULL_MASK, send, m);
                }
            }
            first += up ? k : 0;
            left = k;
        } else {
            v[0] += __shfl_xor_sync(FULL_MASK, v[0], m);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (j < left) put(first + j, v[j]);
}

template <typename F, int LPC>
__global__ void __launch_bounds__(32 * BwdGeo<LPC>::WARPS) k_scan_bwd(ScanArgs a) {
    pdl_wait();
    pdl_trigger();
    using P = Geo<LPC>;
    using Q = BwdGeo<LPC>;
    constexpr int HALF = TB / 2, NB = LPC < 8 ? LPC : 8;
    extern __shared__ __align__(16) char smem_raw[];
    typename Q::Warp *all = reinterpret_cast<typename Q::Warp *>(smem_raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane / LPC, q = lane % LPC;
    typename Q::Warp &my = all[warp];
    long long unit = blockIdx.x;
    const int cb = (int)(unit % a.ncb);
    unit /= a.ncb;
    const int grp = (int)(unit % a.G);
    unit /= a.G;
    const int span = (int)(unit % a.nspan), b = (int)(unit / a.nspan);
    const int cg = cb * Q::CH + warp * P::CPW + c, ch = grp * a.Dg + cg, n0 = 4 * q;
    const bool live = cg < a.Dg;
    const size_t row = ((size_t)b * a.D + ch) * a.N;
    float A2[4], E[4], gA[4];
    load_states(live ? a.A : nullptr, (size_t)ch * a.N, n0, a.N, A2);
    load_states(live ? a.gs_out : nullptr, row, n0, a.N, E);
#pragma unroll
    for (int i = 0; i < 4; i++) { A2[i] *= LOG2E; gA[i] = 0.f; }
    for (int j = a.nspan - 1; j > span; j--) {
        const size_t at = ((size_t)b * a.nspan + j) * a.D + ch;
        float V[4];
        load_states(live ? a.span_state : nullptr, at * a.N, n0, a.N, V);
        const float s = live ? a.span_dt[at] : 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) E[i] = ex2(A2[i] * s) * E[i] + V[i];
    }
    const float bias = live && a.bias ? a.bias[ch] : 0.f, dskip = live && a.Dskip ? a.Dskip[ch] : 0.f;
    float gD = 0.f, gbias = 0.f;
    const int blk0 = span * a.span_blocks, blk1 = min(blk0 + a.span_blocks, a.nblk);
    const F *pu = (const F *)a.u + (size_t)b * a.u_batch + ch, *pd = (const F *)a.delta + (size_t)b * a.delta_batch + ch;
    const F *pz = a.z ? (const F *)a.z + (size_t)b * a.z_batch + ch : nullptr;
    const F *pg = a.gy ? (const F *)a.gy + (size_t)b * a.T * a.D + ch : nullptr;

    F ru[P::PT], rd[P::PT], rz[P::PT], rg[P::PT];
    float rh[4];
    BlockBC<F, LPC> bc;
    auto fetch = [&](int blk) {
        if (blk < blk0) return;
#pragma unroll
        for (int i = 0; i < P::PT; i++) {
            const int t = blk * TB + q + LPC * i;
            if (live && t < a.T) {
                ru[i] = pu[(size_t)t * a.u_token];
                rd[i] = pd[(size_t)t * a.delta_token];
                if (pz) rz[i] = pz[(size_t)t * a.z_token];
                if (pg) rg[i] = pg[(size_t)t * a.D];
            }
        }
        load_states(live ? a.ckpt : nullptr, (((size_t)b * a.nblk + blk) * a.D + ch) * a.N, n0, a.N, rh);
        bc.load(a, b, grp, blk * TB, a.T, lane);
    };
    fetch(blk1 - 1);
    for (int blk = blk1 - 1; blk >= blk0; blk--) {
        const int buf = blk & 1;
        float u[P::PT], sg[P::PT], z[P::PT], g[P::PT], h0[4], mid[4];
#pragma unroll
        for (int i = 0; i < 4; i++) { h0[i] = rh[i]; mid[i] = rh[i]; }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < P::PT; i++) {
            const int t = q + LPC * i;
            float dt = 0.f, dy = 0.f;
            u[i] = 0.f; sg[i] = 0.f; z[i] = 0.f; g[i] = 0.f;
            if (live && blk * TB + t < a.T) {
                u[i] = Elem<F>::ld(&ru[i]);
                dt = Elem<F>::ld(&rd[i]) + bias;
                sg[i] = 1.f;
                if (a.softplus) dt = softplus(dt, sg[i]);
                if (pg) g[i] = Elem<F>::ld(&rg[i]);
                dy = g[i];
                if (pz) {
                    z[i] = Elem<F>::ld(&rz[i]);
                    dy *= z[i] * sigmoidf(z[i]);
                }
            }
            my.d[t][c] = make_float4(dt, dt * u[i], dy, 0.f);
        }
        bc.put(my.b, my.c, lane);
        __syncwarp();
        fetch(blk - 1);
        // the state before token HALF
#pragma unroll
        for (int t = 0; t < HALF; t++) {
            const float4 d = my.d[t][c], Bv = *reinterpret_cast<const float4 *>(&my.b[t * P::NP + n0]);
            mid[0] = ex2(d.x * A2[0]) * mid[0] + d.y * Bv.x;
            mid[1] = ex2(d.x * A2[1]) * mid[1] + d.y * Bv.y;
            mid[2] = ex2(d.x * A2[2]) * mid[2] + d.y * Bv.z;
            mid[3] = ex2(d.x * A2[3]) * mid[3] + d.y * Bv.w;
        }
#pragma unroll 1
        for (int half = 1; half >= 0; half--) {
            const int tb = half * HALF;
            float dec[HALF][4], h[HALF + 1][4];          // a_t; the state before token t
#pragma unroll
            for (int i = 0; i < 4; i++) h[0][i] = half ? mid[i] : h0[i];
#pragma unroll
            for (int t = 0; t < HALF; t++) {
                const float4 d = my.d[tb + t][c], Bv = *reinterpret_cast<const float4 *>(&my.b[(tb + t) * P::NP + n0]);
                const float Bf[4] = {Bv.x, Bv.y, Bv.z, Bv.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    dec[t][i] = ex2(d.x * A2[i]);
                    h[t + 1][i] = dec[t][i] * h[t][i] + d.y * Bf[i];
                }
            }
#pragma unroll
            for (int nb = HALF / NB - 1; nb >= 0; nb--) {
                float gin[NB], gdec[NB], yv[NB];
#pragma unroll
                for (int j = NB - 1; j >= 0; j--) {
                    const int t = nb * NB + j;
                    const float4 d = my.d[tb + t][c], Bv = *reinterpret_cast<const float4 *>(&my.b[(tb + t) * P::NP + n0]),
                                 Cv = *reinterpret_cast<const float4 *>(&my.c[(tb + t) * P::NP + n0]);
                    const float Bf[4] = {Bv.x, Bv.y, Bv.z, Bv.w}, Cf[4] = {Cv.x, Cv.y, Cv.z, Cv.w};
                    float v[8], s0 = 0.f, s1 = 0.f, s2 = 0.f;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float G = Cf[i] * d.z + E[i], ga = G * (dec[t][i] * h[t][i]);
                        v[i] = G * d.y;
                        v[4 + i] = h[t + 1][i] * d.z;
                        s0 += G * Bf[i];
                        s1 += ga * A2[i];
                        s2 += Cf[i] * h[t + 1][i];
                        gA[i] += ga * d.x;
                        E[i] = dec[t][i] * G;
                    }
                    gin[j] = s0; gdec[j] = s1; yv[j] = s2;
                    float *out = &my.sum[buf][(tb + t) * Q::VALUES + q];
                    sum_channels<LPC>(v, lane, [&](int i, float x) { out[i * LPC] = x; });
                }
                const float gi = sum_tokens<LPC, NB>(gin, q), gd = sum_tokens<LPC, NB>(gdec, q) * LN2, y0 = sum_tokens<LPC, NB>(yv, q);
                // the lane's own token: NB < LPC when a channel has more lanes than a half has tokens
                const int t = tb + nb * NB + q % NB;
                if (t % LPC == q && live && blk * TB + t < a.T) {
                    constexpr int P2 = P::PT > 1 ? P::PT / 2 : 0;
                    const int lo = P::PT > 1 ? nb : 0;
                    const float uu = half ? u[P2 + lo] : u[lo], sv = half ? sg[P2 + lo] : sg[lo], zz = half ? z[P2 + lo] : z[lo],
                                gg = half ? g[P2 + lo] : g[lo];
                    const float4 d = my.d[t][c];
                    const float graw = (uu * gi + gd) * sv;
                    gD += d.z * uu;
                    gbias += graw;
                    const size_t at = ((size_t)b * a.T + blk * TB + t) * a.D + ch;
                    if (a.gu) Elem<F>::st((F *)a.gu + at, d.x * gi + dskip * d.z);
                    if (a.gdelta) Elem<F>::st((F *)a.gdelta + at, graw);
                    if (a.gz) {
                        const float s = sigmoidf(zz);
                        Elem<F>::st((F *)a.gz + at, gg * (y0 + dskip * uu) * (s * (1.f + zz * (1.f - s))));
                    }
                }
            }
        }
        if (a.part_bc) {
            // (two buffers: a warp that is a block ahead writes the other one)
            __syncthreads();
            for (int e = threadIdx.x; e < TB * Q::VALUES; e += 32 * Q::WARPS) {
                const int t = blk * TB + e / Q::VALUES;
                float s = all[0].sum[buf][e];
#pragma unroll
                for (int w = 1; w < Q::WARPS; w++) s += all[w].sum[buf][e];
                if (t < a.T)
                    a.part_bc[((((size_t)cb * a.B + b) * a.T + t) * a.G + grp) * Q::VALUES + e % Q::VALUES] = s;
            }
        }
    }
#pragma unroll
    for (int m = 1; m < LPC; m <<= 1) {
        gD += __shfl_xor_sync(FULL_MASK, gD, m);
        gbias += __shfl_xor_sync(FULL_MASK, gbias, m);
    }
    if (live) {
        if (span == 0 && a.gs_in) store_states(a.gs_in, row, n0, a.N, E);
        if (a.part) {
            float *p = a.part + ((size_t)b * a.nspan + span) * ((size_t)a.D * (a.N + 2));
            store_states(p, (size_t)ch * a.N, n0, a.N, gA);
            if (q == 0) {
                p[(size_t)a.D * a.N + ch] = gD;
                p[(size_t)a.D * (a.N + 1) + ch] = gbias;
            }
        }
    }
}

// gB, gC: the sums of the CTAs of a row's channels, in a fixed order
template <typename F>
__global__ void __launch_bounds__(256) k_scan_fold_bc(const float *__restrict__ part, int ncb, long long rows, int lpc, int N, F *gB, F *gC) {
    pdl_wait();
    pdl_trigger();
    const int values = 8 * lpc;
    const long long total = rows * values, i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    float s = 0.f;
#pragma unroll 8
    for (int k = 0; k < ncb; k++) s += part[(size_t)k * total + i];
    const long long row = i / values;
    const int e = (int)(i - row * values), v = e / lpc, n = 4 * (e % lpc) + (v & 3);
    F *g = v < 4 ? gB : gC;
    if (g != nullptr && n < N) Elem<F>::st(g + row * N + n, s);
}

// ------------------------------------------------------------------------------------------------ host side
int lanes_for(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

int check_scan(const wkv_selective_scan_args_t *a) {
    if (!a) return WKV_ERR_NULL;
    if (a->B < 0 || a->T < 0 || a->D < 0 || a->N < 1 || a->N > 64 || a->G < 1 || a->D % a->G != 0 || a->time_groups < 0) return WKV_ERR_SHAPE;
    if (!known_dtype(a->dtype)) return WKV_ERR_DTYPE;
    for (long long s : {a->u_batch, a->u_token, a->delta_batch, a->delta_token, a->B_batch, a->B_token, a->C_batch, a->C_token, a->z_batch, a->z_token})
        if (s < 0) return WKV_ERR_SHAPE;
    if (a->B == 0 || a->D == 0) return WKV_OK;
    if (!a->A || (a->T > 0 && (!a->u || !a->delta || !a->Bm || !a->Cm))) return WKV_ERR_NULL;
    return WKV_OK;
}

// spans of a row: enough for the GPU, of four blocks at least
int plan_spans(const wkv_selective_scan_args_t *a) {
    const int lpc = lanes_for(a->N), cpw = 32 / lpc, nblk = (a->T + TB - 1) / TB;
    const long long warps = (long long)a->B * a->G * ((a->D / a->G + cpw - 1) / cpw);
    long long n = a->time_groups;
    if (n == 0) {
        const long long want = (long long)device_sm_count() * 12;
        n = warps * 2 > want ? 1 : want / warps;
        if (n > 32) n = 32;
        if (n > nblk / 4) n = nblk / 4;
    }
    if (n > nblk) n = nblk;
    if (n < 1) n = 1;
    const long long len = (nblk + n - 1) / n;
    return len > 0 ? (int)((nblk + len - 1) / len) : 1;         // (no span is empty)
}

ScanArgs scan_args(const wkv_selective_scan_args_t *a) {
    ScanArgs k = {};
    k.B = a->B; k.T = a->T; k.D = a->D; k.N = a->N; k.G = a->G; k.Dg = a->D / a->G; k.softplus = a->softplus != 0;
    k.nblk = (a->T + TB - 1) / TB;
    k.nspan = plan_spans(a);
    k.span_blocks = (k.nblk + k.nspan - 1) / k.nspan;
    k.u = a->u; k.delta = a->delta; k.Bm = a->Bm; k.Cm = a->Cm; k.z = a->z;
    k.u_batch = a->u_batch; k.u_token = a->u_token; k.delta_batch = a->delta_batch; k.delta_token = a->delta_token;
    k.B_batch = a->B_batch; k.B_token = a->B_token; k.C_batch = a->C_batch; k.C_token = a->C_token;
    k.z_batch = a->z_batch; k.z_token = a->z_token;
    k.A = a->A; k.Dskip = a->Dskip; k.bias = a->delta_bias; k.state_in = a->state_in;
    const uintptr_t run = 4 * (uintptr_t)elem_size(a->dtype) - 1;
    auto fits = [&](const void *p, long long batch, long long token) {
        return a->N % 4 == 0 && batch % 4 == 0 && token % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & run) == 0;
    };
    k.vec_b = fits(a->Bm, a->B_batch, a->B_token);
    k.vec_c = fits(a->Cm, a->C_batch, a->C_token);
    return k;
}

template <class Fn>
int by_lanes(int lpc, Fn f) {
    switch (lpc) {
        case 1: return f(std::integral_constant<int, 1>{});
        case 2: return f(std::integral_constant<int, 2>{});
        case 4: return f(std::integral_constant<int, 4>{});
        case 8: return f(std::integral_constant<int, 8>{});
        default: return f(std::integral_constant<int, 16>{});
    }
}
int warps_of_cta(int lpc) { return lpc >= 8 ? 4 : 8; }

size_t span_bytes(const wkv_selective_scan_args_t *a, int nspan) {
    if (nspan < 2) return 0;
    const size_t n = (size_t)a->B * nspan * a->D;
    return align256(n * a->N * 4) + align256(n * 4);
}
void place_spans(const wkv_selective_scan_args_t *a, ScanArgs &k, char *ws) {
    k.span_state = (float *)ws;
    k.span_dt = (float *)(ws + align256((size_t)a->B * k.nspan * a->D * a->N * 4));
}
int bwd_channel_blocks(const wkv_selective_scan_args_t *a) {
    const int lpc = lanes_for(a->N), per = warps_of_cta(lpc) * (32 / lpc);
    return (a->D / a->G + per - 1) / per;
}
struct BwdLayout {
    size_t spans, bc, params, total;
};
BwdLayout bwd_layout(const wkv_selective_scan_args_t *a) {
    const int nspan = plan_spans(a);
    BwdLayout l;
    l.spans = span_bytes(a, nspan);
    l.bc = align256((size_t)bwd_channel_blocks(a) * a->B * a->T * a->G * 8 * lanes_for(a->N) * 4);
    l.params = align256((size_t)a->B * nspan * a->D * (a->N + 2) * 4);
    l.total = l.spans + l.bc + l.params;
    return l;
}
bool nothing(const wkv_selective_scan_args_t *a) { return a->B == 0 || a->D == 0 || a->T == 0; }

}  // namespace
}  // namespace wkv

using namespace wkv;

extern "C" size_t wkv_selective_scan_ckpt_bytes(const wkv_selective_scan_args_t *a) {
    if (check_scan(a) != WKV_OK || nothing(a)) return 0;
    return align256((size_t)a->B * ((a->T + TB - 1) / TB) * a->D * a->N * 4);
}

extern "C" size_t wkv_selective_scan_forward_workspace(const wkv_selective_scan_args_t *a) {
    if (check_scan(a) != WKV_OK || nothing(a)) return 0;
    return span_bytes(a, plan_spans(a));
}

extern "C" int wkv_selective_scan_forward(const wkv_selective_scan_args_t *a, void *stream) {
    int e = check_scan(a);
    if (e != WKV_OK) return e;
    cudaStream_t s = (cudaStream_t)stream;
    if (a->B == 0 || a->D == 0) return WKV_OK;
    if (a->T == 0) {
        if (!a->state_out || a->state_out == a->state_in) return WKV_OK;
        const size_t n = (size_t)a->B * a->D * a->N * 4;
        const cudaError_t r = a->state_in ? cudaMemcpyAsync(a->state_out, a->state_in, n, cudaMemcpyDeviceToDevice, s)
                                          : cudaMemsetAsync(a->state_out, 0, n, s);
        return r == cudaSuccess ? WKV_OK : WKV_ERR_LAUNCH;
    }
    if (!a->y) return WKV_ERR_NULL;
    if (a->T > 1 && a->state_in && a->state_in == a->state_out) return WKV_ERR_UNSUPPORTED;
    ScanArgs k = scan_args(a);
    k.y = a->y; k.state_out = a->state_out;
    const int lpc = lanes_for(a->N), cpw = 32 / lpc;
    if (a->T == 1 && !a->ckpt) {
        const long long threads = (long long)a->B * a->D * lpc;
        return by_dtype(a->dtype, [&](auto f) {
            return by_lanes(lpc, [&](auto l) {
                return launch_chained(k_scan_step<decltype(f), decltype(l)::value>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, k);
            });
        });
    }
    if (a->ckpt) {
        if (a->ckpt_bytes < wkv_selective_scan_ckpt_bytes(a)) return WKV_ERR_WORKSPACE;
        if (!aligned16(a->ckpt)) return WKV_ERR_ALIGN;
        k.ckpt = (float *)a->ckpt;
    }
    const size_t need = span_bytes(a, k.nspan);
    if (need) {
        if (!a->workspace || a->workspace_bytes < need) return WKV_ERR_WORKSPACE;
        if (!aligned16(a->workspace)) return WKV_ERR_ALIGN;
        place_spans(a, k, (char *)a->workspace);
    }
    k.ncb = (k.Dg + cpw - 1) / cpw;
    const long long per_span = (long long)k.ncb * a->G * a->B;
    return by_dtype(a->dtype, [&](auto f) {
        return by_lanes(lpc, [&](auto l) {
            using F = decltype(f);
            constexpr int LPC = decltype(l)::value;
            if (k.nspan > 1) {
                const int r = launch_chained(k_scan_fwd<F, LPC, true>, dim3((unsigned)((per_span * (k.nspan - 1) + 3) / 4)), dim3(128), 0, s, k);
                if (r != WKV_OK) return r;
            }
            return launch_chained(k_scan_fwd<F, LPC, false>, dim3((unsigned)((per_span * k.nspan + 3) / 4)), dim3(128), 0, s, k);
        });
    });
}

extern "C" size_t wkv_selective_scan_backward_workspace(const wkv_selective_scan_args_t *a) {
    if (check_scan(a) != WKV_OK || nothing(a)) return 0;
    return bwd_layout(a).total;
}

extern "C" int wkv_selective_scan_backward(const wkv_selective_scan_args_t *a, void *stream) {
    int e = check_scan(a);
    if (e != WKV_OK) return e;
    cudaStream_t s = (cudaStream_t)stream;
    if (a->D == 0) return WKV_OK;
    const long long np = (long long)a->D * (a->N + 2);
    FoldOut fo = {};
    fo.p[0] = a->gA; fo.p[1] = a->gD; fo.p[2] = a->gbias;
    fo.start[1] = (long long)a->D * a->N;
    fo.start[2] = fo.start[1] + a->D;
    fo.start[3] = fo.start[4] = np;
    const bool params = a->gA || a->gD || a->gbias;
    if (nothing(a)) {
        if (a->B > 0 && a->gstate_in) {
            const size_t n = (size_t)a->B * a->D * a->N * 4;
            const cudaError_t r = a->gstate_out ? cudaMemcpyAsync(a->gstate_in, a->gstate_out, n, cudaMemcpyDeviceToDevice, s)
                                                : cudaMemsetAsync(a->gstate_in, 0, n, s);
            if (r != cudaSuccess) return WKV_ERR_LAUNCH;
        }
        return params ? fold_params(nullptr, 0, np, fo, s) : WKV_OK;
    }
    const BwdLayout l = bwd_layout(a);
    if (!a->ckpt || a->ckpt_bytes < wkv_selective_scan_ckpt_bytes(a)) return WKV_ERR_WORKSPACE;
    if (!a->workspace || a->workspace_bytes < l.total) return WKV_ERR_WORKSPACE;
    if (!aligned16(a->workspace) || !aligned16(a->ckpt)) return WKV_ERR_ALIGN;
    ScanArgs k = scan_args(a);
    char *ws = (char *)a->workspace;
    if (l.spans) place_spans(a, k, ws);
    k.ckpt = (float *)a->ckpt;
    k.gy = a->gy; k.gs_out = a->gstate_out; k.gu = a->gu; k.gdelta = a->gdelta; k.gz = a->z ? a->gz : nullptr; k.gs_in = a->gstate_in;
    k.part_bc = a->gB || a->gC ? (float *)(ws + l.spans) : nullptr;
    k.part = params ? (float *)(ws + l.spans + l.bc) : nullptr;
    const int lpc = lanes_for(a->N), cpw = 32 / lpc;
    const int ncb = bwd_channel_blocks(a);
    e = by_dtype(a->dtype, [&](auto f) {
        return by_lanes(lpc, [&](auto l_) {
            using F = decltype(f);
            constexpr int LPC = decltype(l_)::value;
            if (k.nspan > 1) {
                ScanArgs m = k;
                m.ncb = (k.Dg + cpw - 1) / cpw;
                const long long units = (long long)m.ncb * a->G * (k.nspan - 1) * a->B;
                const int r = launch_chained(k_scan_bwd_summary<F, LPC>, dim3((unsigned)((units + 3) / 4)), dim3(128), 0, s, m);
                if (r != WKV_OK) return r;
            }
            k.ncb = ncb;
            static unsigned char done[64];
            if (!set_max_smem_once(k_scan_bwd<F, LPC>, BwdGeo<LPC>::SMEM, done)) return (int)WKV_ERR_LAUNCH;
            const int r = launch_chained(k_scan_bwd<F, LPC>, dim3((unsigned)((long long)ncb * a->G * k.nspan * a->B)),
                                         dim3(32 * BwdGeo<LPC>::WARPS), BwdGeo<LPC>::SMEM, s, k);
            if (r != WKV_OK || !k.part_bc) return r;
            const long long rows = (long long)a->B * a->T * a->G;
            return launch_chained(k_scan_fold_bc<F>, dim3((unsigned)((rows * 8 * LPC + 255) / 256)), dim3(256), 0, s, k.part_bc, ncb, rows,
                                  LPC, a->N, (F *)a->gB, (F *)a->gC);
        });
    });
    if (e != WKV_OK || !params) return e;
    return fold_params(k.part, a->B * k.nspan, np, fo, s);
}
