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
// A thread owns four states of each of two neighbouring channels and keeps them in fp32 registers (pairs of states, on packed
// instructions); LPC lanes share the two channels (N <= 4 LPC, padded states have A = B = C = 0 and stay zero), a warp has
// 64 / LPC channels.  Two channels, because what bounded a thread with one was the shared memory's path to the registers:
// B and C of a token are 32 bytes a lane, 8 of the 12 cycles that a warp's loads took per token.  Tokens come in blocks of 16:
// what is per token and channel (softplus, gates, loads, stores) is divided among the channels' lanes, lane q taking the
// tokens that are q mod LPC; sums over n are exchanged so that each lane ends with those of its own tokens.
// Warps do not wait for one another in the forward pass.
//
// Few chains (B x D): the tokens of a row are cut into spans that run in parallel.  The decay over a span is exp(A sum dt),
// so a first pass leaves each span's contribution from zero and sum dt, and the full pass starts from their fold.
//
// The backward pass needs h_t at every token: the forward pass leaves the state before every 16th token (4 N / 16 bytes a
// token and channel), a block is run again from there.
//
// Not bound by HBM: 4 rows of 4096 tokens and channels, 16 states, take 605 us forward and 1700 backward, of which
// their bytes would take 83 and 147.  (Forward calls that follow one another take 780: the next one's CTAs are placed while this one's
// run, 256 of them for 444 places, and end up uneven on the SMs.  With ordinary launches 570.)  Per token and eight channels an SM that is full takes 18 and 54 cycles; of
// these 10 and 17 are exponentials on the special function unit (a state's decay is formed once forward, 1.75 times backward), 9 and 29
// the shared memory's path (B, C, steps, and the exchanges of the sums), 9 and 25 the issue of 37 and 101 instructions, with 7 warps an
// SM.  None of these is a limit: what is left is latency, with few warps to hide it.  More warps did not help (their
// states and decays do not fit: 12 warps of 165 registers 1785 us a pass where 8 of 254 took 1680), nor did a quarter of the
// exponentials on the multiply-add pipe (prompts 2 % faster, nothing else).
#include "elem_io.cuh"
#include "wkv_internal.h"

namespace wkv {
namespace {

constexpr int TB = 16;               // tokens of a block
// (log2(e) as the sum of two floats)
constexpr float LOG2E = 1.4426950408889634f, LOG2E_LOW = 1.9259629911266175e-8f, LN2 = 0.6931471805599453f, EX2_MEAN = 1.8e-8f;
constexpr unsigned FULL_MASK = 0xffffffffu;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct ScanArgs {
    int B, T, D, N, G, Dg, softplus;
    int ncb, nspan, span_blocks, nblk;           // channel blocks per group, spans of a row, their length, blocks of a row
    int vec_b, vec_c, vec_a, vec_s;
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

__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// e^x for x from -126 to 0: the rounding of the exponent x log2(e), up to 2^-24 of it, is made good, and so is the mean error of ex2,
// -5e-8 over exponents below -1 (above them it is -2e-8 and less: 3e-8 too much is added there, half a rounding)
__device__ __forceinline__ float exp_near(float x) {
    const float e = LOG2E * x, lo = fmaf(LOG2E, x, -e) + LOG2E_LOW * x, t = ex2(e);
    return fmaf(t, fmaf(lo, LN2, 5e-8f), t);
}
__device__ __forceinline__ float sigm(float x) { return rcp(1.f + ex2(-LOG2E * x)); }

// softplus(x) = max(x, 0) + log(1 + t), t = e^-|x|, and with SIG its derivative sigmoid(x), for any x: no term overflows.
// log(1 + t) = 2 artanh(s), s = t / (2 + t) <= 1/3: its power series up to s^13 is short of it by less than 2 s^15 / (15 (1 - s^2)), at
// most 1.05e-8 or a relative 1.5e-8, and keeps the digits of small steps (log of a rounded 1 + t does not).
template <bool SIG>
__device__ __forceinline__ float softplus(float x, float &sig) {
    float ax = -fabsf(x), s;
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(ax) : "f"(-126.f));        // (infinities; a NaN stays)
    const float t = exp_near(ax);
    if (SIG) {
        const float w = rcp((1.f + t) * (2.f + t)), r = (2.f + t) * w;       // r = 1 / (1 + t)
        s = t * (1.f + t) * w;
        sig = x >= 0.f ? r : t * r;
    } else {
        s = t * rcp(2.f + t);
    }
    const float s2 = s * s;
    float p = 1.f / 13.f;
    p = p * s2 + 1.f / 11.f;
    p = p * s2 + 1.f / 9.f;
    p = p * s2 + 1.f / 7.f;
    p = p * s2 + 1.f / 5.f;
    p = p * s2 + 1.f / 3.f;
    p = p * s2 + 1.f;
    // (fmaxf drops a NaN, s brings it back)
    return fmaxf(x, 0.f) + 2.f * s * p;
}

template <bool SIG, int PT>
__device__ __forceinline__ void softplus_all(f2 (&x)[PT], f2 (&sig)[PT]) {
#pragma unroll
    for (int i = 0; i < PT; i++) {
        f2 g;
        x[i] = make_float2(softplus<SIG>(x[i].x, g.x), softplus<SIG>(x[i].y, g.y));
        if (SIG) sig[i] = g;
    }
}

// What a warp works on: LPC lanes for two channels, lane = c * LPC + q.
template <int LPC>
struct Geo {
    static constexpr int CL = 32 / LPC;          // pairs of channels of a warp
    static constexpr int CPW = 2 * CL;           // channels of a warp
    static constexpr int PT = TB / LPC;          // tokens of a block that are a lane's own
    static constexpr int NP = 4 * LPC;           // states with padding
    static constexpr int NI = (TB * LPC + 31) / 32;      // runs of four of a B or C block that a lane loads
    // rows of what a warp keeps per token and pair of channels, padded so that lanes that write neighbouring tokens use
    // different banks (16 and 8 bytes an element)
    static constexpr int ROW16 = CL + (LPC == 2 ? 4 : LPC == 4 ? 2 : 1);
    static constexpr int ROW8 = CL + (LPC == 2 ? 8 : LPC == 4 ? 4 : LPC == 8 ? 2 : 1);
};

// A lane's own tokens of a block in one tensor: token q + LPC i of the block, 64-bit block address, 32-bit offsets inside
// (the host checks the strides).  Tokens behind the row's last are read as the last one, without a branch around the loads,
// and made zero later; rows of B and C behind it are zeros at once.
//
// FAST: the two channels are one aligned access in every tensor, and so are runs of four of B and C; else the second channel
// is `second` elements on (0 where there is none).  Compiled apart: a branch at each access keeps the compiler from moving
// work across it, and with one or two warps on a scheduler that is what a token's time was (forward 94 us of 4 x 512 tokens of
// 4096 channels with the branches).
template <typename F, int LPC, bool FAST>
struct Own {
    Raw<F, 2> v[Geo<LPC>::PT];
    __device__ __forceinline__ void load(const F *block, int token_stride, int q, int last, int second) {
#pragma unroll
        for (int i = 0; i < Geo<LPC>::PT; i++) {
            const F *p = block + (long long)min(q + LPC * i, last) * token_stride;
            if (FAST) {
                v[i].load(p, true, 2);
            } else {
                alignas(8) const F two[2] = {p[0], p[second]};
                v[i] = *reinterpret_cast<const Raw<F, 2> *>(two);
            }
        }
    }
    __device__ __forceinline__ f2 get(int i) const {
        float f[2];
        v[i].get(f);
        return make_float2(f[0], f[1]);
    }
};
template <typename F>
__device__ __forceinline__ f2 pair_of(const Raw<F, 2> &r) {
    float f[2];
    r.get(f);
    return make_float2(f[0], f[1]);
}
template <bool FAST, typename F>
__device__ __forceinline__ void store_pair(F *p, bool second, f2 v) {
    const float f[2] = {v.x, v.y};
    if (FAST) {
        Raw<F, 2> r;
        r.put(f);
        r.store(p, true, 2);
    } else {
        Elem<F>::st(p, v.x);
        if (second) Elem<F>::st(p + 1, v.y);
    }
}

// the rows of B or C of a block, on their way while the block before is worked on
template <typename F, int LPC, bool FAST>
struct BlockRows {
    Raw<F, 4> r[Geo<LPC>::NI];
    // p: row of the block's first token, state 0
    __device__ __forceinline__ void load(const F *p, int token_stride, bool vec, int N, int last, int lane) {
#pragma unroll
        for (int k = 0; k < Geo<LPC>::NI; k++) {
            const int i = lane + 32 * k, n0 = 4 * (i % LPC), n = min(4, N - n0);
            r[k].zero();
            if (n > 0 && i / LPC <= min(last, TB - 1)) r[k].load(p + (long long)(i / LPC) * token_stride + n0, FAST || vec, n);
        }
    }
    // to: [TB][NP]
    __device__ __forceinline__ void put(float *to, int lane) const {
#pragma unroll
        for (int k = 0; k < Geo<LPC>::NI; k++) {
            const int i = lane + 32 * k;
            float f[4];
            r[k].get(f);
            if (TB * LPC >= 32 || i < TB * LPC) *reinterpret_cast<float4 *>(to + 4 * i) = make_float4(f[0], f[1], f[2], f[3]);
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

// four neighbouring states as two pairs; `swap`: the second pair first
__device__ __forceinline__ void load_states(const float *p, size_t at, int n0, int N, f2 (&h)[2], bool swap = false) {
    float f[4];
    if (p != nullptr && N % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
        const float4 v = n0 < N ? *reinterpret_cast<const float4 *>(p + at + n0) : make_float4(0.f, 0.f, 0.f, 0.f);
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = p != nullptr && n0 + i < N ? p[at + n0 + i] : 0.f;
    }
    const f2 a = make_float2(f[0], f[1]), b = make_float2(f[2], f[3]);
    h[0] = swap ? b : a;
    h[1] = swap ? a : b;
}
__device__ __forceinline__ void store_states(float *p, size_t at, int n0, int N, const f2 (&h)[2], bool swap = false) {
    const f2 a = swap ? h[1] : h[0], b = swap ? h[0] : h[1];
    const float f[4] = {a.x, a.y, b.x, b.y};
    if (N % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0) {
        if (n0 < N) *reinterpret_cast<float4 *>(p + at + n0) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (n0 + i < N) p[at + n0 + i] = f[i];
    }
}
// A log2(e).  An infinite A (the exponential of a large parameter), or one whose product is, becomes the largest number: its decay
// is zero all the same (for steps above 1e-36), and a step of zero keeps the state.
__device__ __forceinline__ float decay_rate(float A) {
    float x = A * LOG2E;
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-3.4e38f));        // (a NaN stays)
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(3.4e38f));
    return x;
}
// the same of four states
__device__ __forceinline__ void load_decays(const float *A, size_t at, int n0, int N, f2 (&A2)[2], bool swap = false) {
    load_states(A, at, n0, N, A2, swap);
#pragma unroll
    for (int i = 0; i < 2; i++) A2[i] = make_float2(decay_rate(A2[i].x), decay_rate(A2[i].y));
}
__device__ __forceinline__ f2 ex2(f2 x) { return make_float2(ex2(x.x), ex2(x.y)); }
// The exponent of a token's decay, dt A log2(e), and a little: ex2 gives too little on average, by 1.9e-8 of it for exponents from
// -0.5 to -0.01 and by 0.6e-8 from -0.001 to 0 (by 5e-8 below -1, where a state is soon forgotten), which over the memory of a state
// adds up.  1.8e-8 more in the exponent, 1.25e-8 of the power, leaves -0.7e-8 and 0.7e-8, and ex2 of it alone is 1 (tokens behind a row's
// end, with a step of zero, keep the state).  Errors of the gradients of A, the bias and the
// state against 64 bits halve (2 x 500 tokens, 512 channels: 1.06, 1.02, 0.75 -> 0.52, 0.51, 0.40 e-6).
__device__ __forceinline__ f2 exponent(float dt, f2 A2) { return fma2(both(dt), A2, both(EX2_MEAN)); }
// What a span with decay rates A2, sum of steps `s` and contribution U from zero does to the state before it: h = 2^(A2 s) h + U.
// A growing state's power may be above the largest number, and then a state of zero has to stay zero and a small one to become what it
// grows to, as without spans.  ANY power is taken as two factors, of at most 2^127 and 2^127.9 (the second is 1 for powers up to
// 2^127: the same bits); decaying states need one.
template <bool ANY>
__device__ __forceinline__ void over_span(const f2 (&A2)[2], float s, f2 (&h)[2], const f2 (&U)[2], float &least) {
    if (!ANY) least = fminf(least, s);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const f2 e = mul2(A2[i], both(s));
        if (ANY) {
            auto first = [](float x) { return ex2(x > 127.f ? 127.f : x); };       // (a NaN stays)
            auto rest = [](float x) { return ex2(fminf(fmaxf(x - 127.f, 0.f), 127.9f)); };
            h[i] = fma2(make_float2(first(e.x), first(e.y)), mul2(make_float2(rest(e.x), rest(e.y)), h[i]), U[i]);
        } else {
            h[i] = fma2(ex2(e), h[i], U[i]);
        }
    }
}
// Whether a state of the warp may have grown over a span: a rate above zero, or a sum of steps below.  Only then is the fold taken
// again with two factors (with them at once, the 512 spans of 1 x 65536 tokens of 64 channels: 249 us a pass instead of 215).
__device__ __forceinline__ bool may_grow(const f2 (&A2)[2][2], float least) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) most = fmaxf(most, fmaxf(A2[i / 2][i & 1].x, A2[i / 2][i & 1].y));
    return __any_sync(FULL_MASK, most > 0.f || least < 0.f);
}
// two pairs of floats in shared memory
__device__ __forceinline__ void pairs_at(const float *p, f2 &a, f2 &b) {
    const float4 v = *reinterpret_cast<const float4 *>(p);
    a = make_float2(v.x, v.y);
    b = make_float2(v.z, v.w);
}

// The unit of a warp of the forward and the summary kernels: ((batch * spans + span) * G + group) * ncb + channel block.
struct Unit {
    int cb, grp, span, b;
    __device__ __forceinline__ Unit(const ScanArgs &a, long long i, int nspan) {
        cb = (int)(i % a.ncb);
        i /= a.ncb;
        grp = (int)(i % a.G);
        i /= a.G;
        span = (int)(i % nspan);
        b = (int)(i / nspan);
    }
};

// Forward.  SUMMARY: only the span's contribution from zero and its sum of dt.
template <typename F, int LPC, bool SUMMARY, bool FAST>
__global__ void __launch_bounds__(128, SUMMARY ? 4 : 3) k_scan_fwd(ScanArgs a) {
    pdl_wait();
    pdl_trigger();
    using P = Geo<LPC>;
    __shared__ __align__(16) float4 s_dt[4][TB][P::ROW16];              // dt, dt u of the first channel, of the second
    __shared__ __align__(16) float s_b[4][TB * P::NP], s_c[SUMMARY ? 1 : 4][TB * P::NP];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane / LPC, q = lane % LPC;
    const Unit un(a, (long long)blockIdx.x * 4 + warp, SUMMARY ? a.nspan - 1 : a.nspan);     // (nobody asks for the last span's contribution)
    if (un.b >= a.B) return;
    const int b = un.b, grp = un.grp, cg = un.cb * P::CPW + 2 * c, n0 = 4 * q;
    const bool live = cg < a.Dg, live2 = cg + 1 < a.Dg;
    const int ch = grp * a.Dg + (live ? cg : 0), second = live2 ? 1 : 0;    // (lanes without a channel read another's, and write nothing)
    const size_t row = ((size_t)b * a.D + ch) * a.N;         // of [B, D, N]
    const int up = second * a.N;                              // to the second channel's states
    f2 A2[2][2], h[2][2];
    load_decays(a.A, (size_t)ch * a.N, n0, a.N, A2[0]);
    load_decays(a.A, (size_t)ch * a.N + up, n0, a.N, A2[1]);
    if (SUMMARY) {
        h[0][0] = h[0][1] = h[1][0] = h[1][1] = both(0.f);
    } else {
        float least = 0.f;
        auto from_spans = [&](auto any) {
            load_states(a.state_in, row, n0, a.N, h[0]);
            load_states(a.state_in, row + up, n0, a.N, h[1]);
            for (int j = 0; j < un.span; j++) {
                const size_t at = ((size_t)b * a.nspan + j) * a.D + ch;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    f2 U[2];
                    load_states(a.span_state, at * a.N + k * up, n0, a.N, U);
                    over_span<decltype(any)::value>(A2[k], a.span_dt[at + k * second], h[k], U, least);
                }
            }
        };
        from_spans(std::false_type{});
        if (un.span > 0 && may_grow(A2, least)) from_spans(std::true_type{});
    }
    const f2 bias = a.bias ? make_float2(a.bias[ch], a.bias[ch + second]) : both(0.f);
    const f2 dskip = a.Dskip ? make_float2(a.Dskip[ch], a.Dskip[ch + second]) : both(0.f);
    const int blk0 = un.span * a.span_blocks, blk1 = min(blk0 + a.span_blocks, a.nblk), t0 = blk0 * TB;
    const int su = (int)a.u_token, sd = (int)a.delta_token, sz = (int)a.z_token, sB = (int)a.B_token, sC = (int)a.C_token;
    const F *pu = (const F *)a.u + (size_t)b * a.u_batch + (size_t)t0 * a.u_token + ch;
    const F *pd = (const F *)a.delta + (size_t)b * a.delta_batch + (size_t)t0 * a.delta_token + ch;
    const F *pz = (const F *)a.z + (size_t)b * a.z_batch + (size_t)t0 * a.z_token + ch;
    const F *pB = (const F *)a.Bm + (size_t)b * a.B_batch + (size_t)t0 * a.B_token + (size_t)grp * a.N;
    const F *pC = (const F *)a.Cm + (size_t)b * a.C_batch + (size_t)t0 * a.C_token + (size_t)grp * a.N;
    F *py = SUMMARY ? nullptr : (F *)a.y + ((size_t)b * a.T + t0 + q) * a.D + ch;
    float *ck = !SUMMARY && a.ckpt && live ? a.ckpt + (((size_t)b * a.nblk + blk0) * a.D + ch) * a.N : nullptr;
    const bool gated = !SUMMARY && a.z != nullptr;

    Own<F, LPC, FAST> ru, rd, rz;
    BlockRows<F, LPC, FAST> rB, rC;
    int last = a.T - 1 - t0;             // the row's last token, counted from the block to be fetched
    auto fetch = [&]() {
        ru.load(pu, su, q, last, second);
        rd.load(pd, sd, q, last, second);
        if (gated) rz.load(pz, sz, q, last, second);
        rB.load(pB, sB, a.vec_b, a.N, last, lane);
        if (!SUMMARY) rC.load(pC, sC, a.vec_c, a.N, last, lane);
        pu += (long long)su * TB; pd += (long long)sd * TB; pz += (long long)sz * TB;
        pB += (long long)sB * TB; pC += (long long)sC * TB;
    };
    fetch();
    f2 total = both(0.f);                // SUMMARY: the lane's part of sum dt
    for (int blk = blk0; blk < blk1; blk++) {
        if (ck) {
            store_states(ck, 0, n0, a.N, h[0]);
            if (live2) store_states(ck, a.N, n0, a.N, h[1]);
            ck += (size_t)a.D * a.N;
        }
        f2 u[P::PT], z[P::PT], y[P::PT], step[P::PT];
        __syncwarp();                    // (the block before has been read)
#pragma unroll
        for (int i = 0; i < P::PT; i++) {
            u[i] = ru.get(i);
            step[i] = add2(rd.get(i), bias);
            z[i] = rz.get(i);            // (not used without a gate)
        }
        if (a.softplus) softplus_all<false>(step, step);
#pragma unroll
        for (int i = 0; i < P::PT; i++) {
            f2 dt = step[i];
            if (q + LPC * i > last) dt = u[i] = both(0.f);    // behind the row: a = 1, nothing is added
            s_dt[warp][q + LPC * i][c] = make_float4(dt.x, dt.x * u[i].x, dt.y, dt.y * u[i].y);
            if (SUMMARY) total = add2(total, dt);
        }
        rB.put(s_b[warp], lane);
        if (!SUMMARY) rC.put(s_c[warp], lane);
        __syncwarp();
        const int end = last;
        last -= TB;
        if (blk + 1 < blk1) fetch();
#pragma unroll
        for (int i = 0; i < P::PT; i++) {
            float y0[LPC], y1[LPC];
            constexpr int GT = LPC < 4 ? LPC : 4;
#pragma unroll
            for (int j0 = 0; j0 < LPC; j0 += GT) {
                f2 dec[GT][2][2], in[GT][2][2];
#pragma unroll
                for (int j = 0; j < GT; j++) {
                    const int t = i * LPC + j0 + j;
                    const float4 d = s_dt[warp][t][c];
                    f2 B[2];
                    pairs_at(&s_b[warp][t * P::NP + n0], B[0], B[1]);
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        dec[j][0][m] = exponent(d.x, A2[0][m]);
                        dec[j][1][m] = exponent(d.z, A2[1][m]);
                        in[j][0][m] = mul2(both(d.y), B[m]);
                        in[j][1][m] = mul2(both(d.w), B[m]);
                    }
                }
#pragma unroll
                for (int j = 0; j < GT; j++)
#pragma unroll
                    for (int m = 0; m < 2; m++) { dec[j][0][m] = ex2(dec[j][0][m]); dec[j][1][m] = ex2(dec[j][1][m]); }
#pragma unroll
                for (int j = 0; j < GT; j++) {
                    const int t = i * LPC + j0 + j;
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        h[0][m] = fma2(dec[j][0][m], h[0][m], in[j][0][m]);
                        h[1][m] = fma2(dec[j][1][m], h[1][m], in[j][1][m]);
                    }
                    if (!SUMMARY) {
                        f2 C[2];
                        pairs_at(&s_c[warp][t * P::NP + n0], C[0], C[1]);
                        const f2 s0 = fma2(C[1], h[0][1], mul2(C[0], h[0][0])), s1 = fma2(C[1], h[1][1], mul2(C[0], h[1][0]));
                        y0[j0 + j] = s0.x + s0.y;
                        y1[j0 + j] = s1.x + s1.y;
                    }
                }
            }
            if (!SUMMARY) y[i] = make_float2(sum_tokens<LPC, LPC>(y0, q), sum_tokens<LPC, LPC>(y1, q));
        }
        if (!SUMMARY) {
#pragma unroll
            for (int i = 0; i < P::PT; i++) y[i] = fma2(dskip, u[i], y[i]);
            if (gated) {
#pragma unroll
                for (int i = 0; i < P::PT; i++) y[i] = mul2(y[i], make_float2(z[i].x * sigm(z[i].x), z[i].y * sigm(z[i].y)));
            }
            if (live) {
#pragma unroll
                for (int i = 0; i < P::PT; i++)
                    if (q + LPC * i <= end) store_pair<FAST>(py + (long long)(LPC * i) * a.D, live2, y[i]);
            }
            py += (long long)TB * a.D;
        }
    }
    if (SUMMARY) {
#pragma unroll
        for (int m = 1; m < LPC; m <<= 1)
            total = add2(total, make_float2(__shfl_xor_sync(FULL_MASK, total.x, m), __shfl_xor_sync(FULL_MASK, total.y, m)));
        const size_t at = ((size_t)b * a.nspan + un.span) * a.D + ch;
        if (live) {
            store_states(a.span_state, at * a.N, n0, a.N, h[0]);
            if (q == 0) a.span_dt[at] = total.x;
        }
        if (live2) {
            store_states(a.span_state, (at + 1) * a.N, n0, a.N, h[1]);
            if (q == 0) a.span_dt[at + 1] = total.y;
        }
    } else if (un.span == a.nspan - 1 && a.state_out) {
        if (live) store_states(a.state_out, row, n0, a.N, h[0]);
        if (live2) store_states(a.state_out, row + a.N, n0, a.N, h[1]);
    }
}

// One token: a thread for eight states of a channel, in two runs of four that are LANES runs apart (the lanes of a channel read
// whole sectors); state_out may be state_in (each thread reads its own before it writes).  N <= 8 LANES.
// Bound by HBM where rows are many, then by a thread's other loads, most of 2 and 4 bytes (64 rows of 8192 channels with 16 states,
// from HBM: one run a thread 27 us, two 20, four 28; two rows a thread 29, four 37; 256 rows 59: 4.5 TB/s).  The limit of the decay
// rates costs 0.3 us of 16 there.
template <typename F, int LANES>
__global__ void __launch_bounds__(256) k_scan_step(ScanArgs a) {
    pdl_wait();
    pdl_trigger();
    const int i = (blockIdx.x * 256 + threadIdx.x) / LANES, q = threadIdx.x % LANES, b = blockIdx.y;
    const bool live = i < a.D;
    const int ch = live ? i : 0, grp = ch / a.Dg;
    const size_t row = ((size_t)b * a.D + ch) * a.N;
    const F *pB = (const F *)a.Bm + (size_t)b * a.B_batch + (size_t)grp * a.N, *pC = (const F *)a.Cm + (size_t)b * a.C_batch + (size_t)grp * a.N;
    Raw<float, 4> rA[2], rh[2];
    Raw<F, 4> rB[2], rC[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int n0 = 4 * (q + j * LANES), n = a.N - n0;
        rh[j].zero();
        rA[j].zero();
        rB[j].zero();
        rC[j].zero();
        if (n > 0) {
            if (a.state_in) rh[j].load(a.state_in + row + n0, a.vec_s, n);
            rA[j].load(a.A + (size_t)ch * a.N + n0, a.vec_a, n);
            rB[j].load(pB + n0, a.vec_b, n);
            rC[j].load(pC + n0, a.vec_c, n);
        }
    }
    const float u = Elem<F>::ld((const F *)a.u + (size_t)b * a.u_batch + ch);
    float dt = Elem<F>::ld((const F *)a.delta + (size_t)b * a.delta_batch + ch) + (a.bias ? a.bias[ch] : 0.f), sig, y = 0.f;
    const float z = a.z ? Elem<F>::ld((const F *)a.z + (size_t)b * a.z_batch + ch) : 0.f, dskip = a.Dskip ? a.Dskip[ch] : 0.f;
    if (a.softplus) dt = softplus<false>(dt, sig);
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const int n0 = 4 * (q + j * LANES), n = a.N - n0;
        float h[4], A[4], B[4], C[4];
        rh[j].get(h);
        rA[j].get(A);
        rB[j].get(B);
        rC[j].get(C);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            h[k] = ex2(fmaf(dt, decay_rate(A[k]), EX2_MEAN)) * h[k] + dt * u * B[k];
            y += C[k] * h[k];
        }
        if (live && a.state_out && n > 0) {
            rh[j].put(h);
            rh[j].store(a.state_out + row + n0, a.vec_s, n);
        }
    }
#pragma unroll
    for (int m = 1; m < LANES; m <<= 1) y += __shfl_xor_sync(FULL_MASK, y, m);
    if (live && q == 0) {
        y += dskip * u;
        if (a.z) y *= z * sigm(z);
        Elem<F>::st((F *)a.y + (size_t)b * a.D + ch, y);
    }
}

// Backward, summary: what a span sends to the state before it, from zero behind it, and its sum of dt.
template <typename F, int LPC, bool FAST>
__global__ void __launch_bounds__(128) k_scan_bwd_summary(ScanArgs a) {
    pdl_wait();
    pdl_trigger();
    using P = Geo<LPC>;
    __shared__ __align__(16) float4 s_dt[4][TB][P::ROW16];              // dt, dy of the first channel, of the second
    __shared__ __align__(16) float s_c[4][TB * P::NP];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane / LPC, q = lane % LPC;
    const Unit un(a, (long long)blockIdx.x * 4 + warp, a.nspan - 1);
    if (un.b >= a.B) return;
    const int b = un.b, grp = un.grp, span = un.span + 1, cg = un.cb * P::CPW + 2 * c, n0 = 4 * q;      // (nobody asks for the first span's)
    const bool live = cg < a.Dg, live2 = cg + 1 < a.Dg;
    const int ch = grp * a.Dg + (live ? cg : 0), second = live2 ? 1 : 0;
    f2 A2[2][2], E[2][2];
    load_decays(a.A, (size_t)ch * a.N, n0, a.N, A2[0]);
    load_decays(a.A, (size_t)(ch + second) * a.N, n0, a.N, A2[1]);
    E[0][0] = E[0][1] = E[1][0] = E[1][1] = both(0.f);
    const f2 bias = a.bias ? make_float2(a.bias[ch], a.bias[ch + second]) : both(0.f);
    const int blk0 = span * a.span_blocks, blk1 = min(blk0 + a.span_blocks, a.nblk), t0 = (blk1 - 1) * TB;
    const int sd = (int)a.delta_token, sz = (int)a.z_token, sC = (int)a.C_token;
    const F *pd = (const F *)a.delta + (size_t)b * a.delta_batch + (size_t)t0 * a.delta_token + ch;
    const F *pz = (const F *)a.z + (size_t)b * a.z_batch + (size_t)t0 * a.z_token + ch;
    const F *pg = (const F *)a.gy + ((size_t)b * a.T + t0) * a.D + ch;
    const F *pC = (const F *)a.Cm + (size_t)b * a.C_batch + (size_t)t0 * a.C_token + (size_t)grp * a.N;
    Own<F, LPC, FAST> rd, rz, rg;
    BlockRows<F, LPC, FAST> rC;
    int last = a.T - 1 - t0;
    auto fetch = [&]() {
        rd.load(pd, sd, q, last, second);
        if (a.gy) rg.load(pg, a.D, q, last, second);
        if (a.z) rz.load(pz, sz, q, last, second);
        rC.load(pC, sC, a.vec_c, a.N, last, lane);
        pd -= (long long)sd * TB; pz -= (long long)sz * TB; pg -= (long long)a.D * TB; pC -= (long long)sC * TB;
    };
    fetch();
    f2 total = both(0.f);
    for (int blk = blk1 - 1; blk >= blk0; blk--) {
        __syncwarp();
        f2 step[P::PT], g[P::PT];
#pragma unroll
        for (int i = 0; i < P::PT; i++) {
            step[i] = add2(rd.get(i), bias);
            g[i] = a.gy ? rg.get(i) : both(0.f);
        }
        if (a.softplus) softplus_all<false>(step, step);
        if (a.z) {
#pragma unroll
            for (int i = 0; i < P::PT; i++) {
                const f2 z = rz.get(i);
                g[i] = mul2(g[i], make_float2(z.x * sigm(z.x), z.y * sigm(z.y)));
            }
        }
#pragma unroll
        for (int i = 0; i < P::PT; i++) {
            f2 dt = step[i], dy = g[i];
            if (q + LPC * i > last) dt = dy = both(0.f);
            s_dt[warp][q + LPC * i][c] = make_float4(dt.x, dy.x, dt.y, dy.y);
            total = add2(total, dt);
        }
        rC.put(s_c[warp], lane);
        __syncwarp();
        last += TB;
        if (blk > blk0) fetch();
#pragma unroll
        for (int t = TB - 1; t >= 0; t--) {
            const float4 d = s_dt[warp][t][c];
            f2 C[2];
            pairs_at(&s_c[warp][t * P::NP + n0], C[0], C[1]);
#pragma unroll
            for (int m = 0; m < 2; m++) {
                E[0][m] = mul2(ex2(exponent(d.x, A2[0][m])), fma2(C[m], both(d.y), E[0][m]));
                E[1][m] = mul2(ex2(exponent(d.z, A2[1][m])), fma2(C[m], both(d.w), E[1][m]));
            }
        }
    }
#pragma unroll
    for (int m = 1; m < LPC; m <<= 1)
        total = add2(total, make_float2(__shfl_xor_sync(FULL_MASK, total.x, m), __shfl_xor_sync(FULL_MASK, total.y, m)));
    const size_t at = ((size_t)b * a.nspan + span) * a.D + ch;
    if (live) {
        store_states(a.span_state, at * a.N, n0, a.N, E[0]);
        if (q == 0) a.span_dt[at] = total.x;
    }
    if (live2) {
        store_states(a.span_state, (at + 1) * a.N, n0, a.N, E[1]);
        if (q == 0) a.span_dt[at + 1] = total.y;
    }
}

// Backward.  The warps of a CTA hold neighbouring channels of one group and one span.  They share the rows of B and C, and
// once a block add up what they have for gB and gC; one barrier a block serves both (two buffers of each).
//
// A block is run forward once more from the state the forward pass left, which leaves the states before its quarters in
// shared memory; then quarter by quarter from the last, forward again with decays and states in registers and back.
//
// gB and gC are sums over the channels, of a CTA here and of all CTAs in k_scan_fold_bc (which costs a workspace of LPC^2 / 8 bytes a
// token and channel: 0.5, 2, 8 and 32 for up to 8, 16, 32 and 64 states).  A thread adds up its two, then eight values a lane and token are exchanged.  Each
// exchange halves the values: lanes 16 apart hold their two pairs of states in opposite order, so that the first one needs
// no selects.
//
// Shared memory of a CTA, KB for 16-bit inputs and fp32: 152 and 168 for up to 8 states, 104 and 112 up to 16, 98 and 102 up to 32, 133 and
// 135 up to 64.
template <typename F, int LPC>
struct BwdGeo {
    static constexpr int WARPS = 4;
    static constexpr int CH = WARPS * Geo<LPC>::CPW;             // channels of a CTA
    static constexpr int VALUES = 8 * LPC;                       // gB and gC of a token: [8][LPC], state 4 q + (i & 3)
    static constexpr int RUNS = TB * LPC;                        // runs of four of a block's rows of B (or C)
    struct Warp {
        float4 d[TB][Geo<LPC>::ROW16];                              // dt, dt u of the first channel, of the second
        float4 own[2][TB][Geo<LPC>::ROW16];                         // u, sigmoid(delta + bias), z, gy
        float4 res[TB][Geo<LPC>::ROW16];                            // sums over the states: G . B of the two channels, G A a h of the two
        float2 res_y[TB][Geo<LPC>::ROW8];                          // C . h
        float4 state[2][4][32];                                  // before tokens 0, 4, 8, 12
        float4 ckpt[2][32];                                      // the next block's: states before it; u, delta, z, gy
        Raw<F, 2> in[4][TB][Geo<LPC>::CL];
        float2 dy[TB][Geo<LPC>::ROW8];                             // of the two channels
        float sum[2][TB * VALUES];
    };
    struct Cta {
        float4 b[2][2][RUNS], c[2][2][RUNS];                     // [buffer][as it is, pairs swapped]
        Warp w[WARPS];
    };
    static constexpr int SMEM = (int)sizeof(Cta);
};

// sizeof(R) bytes (4, 8 or 16) into shared memory without passing through registers; to be waited for by the same thread
template <typename R>
__device__ __forceinline__ void copy_async(R *to, const void *from) {
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
    if constexpr (sizeof(R) == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(from), "n"(sizeof(R)) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// a lane's values for gB (vb) and gC (vc) summed over the warp's channels: put(kind, state & 3, sum) for each that is left
template <int LPC, class Put>
__device__ __forceinline__ void sum_channels(f2 (&vb)[2], f2 (&vc)[2], int lane, Put put) {
    const int hi = lane & 16 ? 2 : 0;
    f2 b = add2(vb[0], make_float2(__shfl_xor_sync(FULL_MASK, vb[1].x, 16), __shfl_xor_sync(FULL_MASK, vb[1].y, 16)));
    f2 c = add2(vc[0], make_float2(__shfl_xor_sync(FULL_MASK, vc[1].x, 16), __shfl_xor_sync(FULL_MASK, vc[1].y, 16)));
    if (LPC == 16) {
        put(0, hi, b.x); put(0, hi + 1, b.y);
        put(1, hi, c.x); put(1, hi + 1, c.y);
        return;
    }
    const bool up8 = lane & 8;
    const int n = hi + (up8 ? 1 : 0);
    const float sb = (up8 ? b.y : b.x) + __shfl_xor_sync(FULL_MASK, up8 ? b.x : b.y, 8);
    const float sc = (up8 ? c.y : c.x) + __shfl_xor_sync(FULL_MASK, up8 ? c.x : c.y, 8);
    if (LPC == 8) {
        put(0, n, sb);
        put(1, n, sc);
        return;
    }
    const bool up4 = lane & 4;
    float s = (up4 ? sc : sb) + __shfl_xor_sync(FULL_MASK, up4 ? sb : sc, 4);
#pragma unroll
    for (int m = 2; m >= LPC; m >>= 1) s += __shfl_xor_sync(FULL_MASK, s, m);
    put(up4 ? 1 : 0, n, s);
}

template <typename F, int LPC, bool FAST>
__global__ void __launch_bounds__(32 * BwdGeo<F, LPC>::WARPS, 2) k_scan_bwd(ScanArgs a) {
    pdl_wait();
    pdl_trigger();
    using P = Geo<LPC>;
    using Q = BwdGeo<F, LPC>;
    constexpr int QT = 4, NB = LPC < QT ? LPC : QT, THREADS = 32 * Q::WARPS, RL = (2 * Q::RUNS + THREADS - 1) / THREADS;
    extern __shared__ __align__(16) char smem_raw[];
    typename Q::Cta &cta = *reinterpret_cast<typename Q::Cta *>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, c = lane / LPC, q = lane % LPC;
    typename Q::Warp &my = cta.w[warp];
    const Unit un(a, blockIdx.x, a.nspan);
    const int b = un.b, grp = un.grp, span = un.span, cg = un.cb * Q::CH + warp * P::CPW + 2 * c, n0 = 4 * q;
    const bool live = cg < a.Dg, live2 = cg + 1 < a.Dg, swap = lane & 16;
    const int ch = grp * a.Dg + (live ? cg : 0), second = live2 ? 1 : 0;
    const size_t row = ((size_t)b * a.D + ch) * a.N;
    f2 A2[2][2], E[2][2], gA[2][2];
    load_decays(a.A, (size_t)ch * a.N, n0, a.N, A2[0], swap);
    load_decays(a.A, (size_t)(ch + second) * a.N, n0, a.N, A2[1], swap);
    gA[0][0] = gA[0][1] = gA[1][0] = gA[1][1] = both(0.f);
    float least = 0.f;
    auto from_spans = [&](auto any) {
        load_states(live ? a.gs_out : nullptr, row, n0, a.N, E[0], swap);
        load_states(live2 ? a.gs_out : nullptr, row + a.N, n0, a.N, E[1], swap);
        for (int j = a.nspan - 1; j > span; j--) {
            const size_t at = ((size_t)b * a.nspan + j) * a.D + ch;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                f2 V[2];
                load_states((k ? live2 : live) ? a.span_state : nullptr, (at + k) * a.N, n0, a.N, V, swap);
                over_span<decltype(any)::value>(A2[k], a.span_dt[at + k * second], E[k], V, least);
            }
        }
    };
    from_spans(std::false_type{});
    if (span + 1 < a.nspan && may_grow(A2, least)) from_spans(std::true_type{});
    const f2 bias = a.bias ? make_float2(a.bias[ch], a.bias[ch + second]) : both(0.f);
    const f2 dskip = a.Dskip ? make_float2(a.Dskip[ch], a.Dskip[ch + second]) : both(0.f);
    f2 gD = both(0.f), gbias = both(0.f);
    const int blk0 = span * a.span_blocks, blk1 = min(blk0 + a.span_blocks, a.nblk), t0 = (blk1 - 1) * TB;
    const int su = (int)a.u_token, sd = (int)a.delta_token, sz = (int)a.z_token;
    const F *pu = (const F *)a.u + (size_t)b * a.u_batch + (size_t)t0 * a.u_token + ch;
    const F *pd = (const F *)a.delta + (size_t)b * a.delta_batch + (size_t)t0 * a.delta_token + ch;
    const F *pz = (const F *)a.z + (size_t)b * a.z_batch + (size_t)t0 * a.z_token + ch;
    const F *pg = (const F *)a.gy + ((size_t)b * a.T + t0) * a.D + ch;
    const float *ck = a.ckpt + (((size_t)b * a.nblk + (blk1 - 1)) * a.D + ch) * a.N;
    size_t out = ((size_t)b * a.T + t0 + q) * a.D + ch;           // of gu, gdelta, gz

    // the CTA's threads bring in a block's rows of B (the first RUNS items) and of C
    Raw<F, 4> rbc[RL];
    auto fetch_rows = [&](int blk, int last) {
#pragma unroll
        for (int k = 0; k < RL; k++) {
            const int i = tid + k * THREADS, run = i % Q::RUNS, m0 = 4 * (run % LPC), n = min(4, a.N - m0);
            const bool isC = i >= Q::RUNS;
            const long long token = isC ? a.C_token : a.B_token;
            const F *p = isC ? (const F *)a.Cm + (size_t)b * a.C_batch : (const F *)a.Bm + (size_t)b * a.B_batch;
            rbc[k].zero();
            if (i < 2 * Q::RUNS && n > 0 && run / LPC <= last)
                rbc[k].load(p + (long long)(blk * TB + run / LPC) * token + (size_t)grp * a.N + m0, FAST || (isC ? a.vec_c : a.vec_b), n);
        }
    };
    auto put_rows = [&](int buf) {
#pragma unroll
        for (int k = 0; k < RL; k++) {
            const int i = tid + k * THREADS, run = i % Q::RUNS;
            float f[4];
            rbc[k].get(f);
            if (i < 2 * Q::RUNS) {
                float4(&to)[2][Q::RUNS] = i >= Q::RUNS ? cta.c[buf] : cta.b[buf];
                to[0][run] = make_float4(f[0], f[1], f[2], f[3]);
                to[1][run] = make_float4(f[2], f[3], f[0], f[1]);
            }
        }
    };
    int last = a.T - 1 - t0;
    // a lane's own tokens of the next block, and the states before it: copied into shared memory (FAST), else held in registers
    Own<F, LPC, FAST> held[FAST ? 1 : 4];
    f2 held_state[FAST ? 1 : 2][2];
    auto own_tokens = [&](int k, const F *block, int token_stride) {
        if constexpr (FAST) {
#pragma unroll
            for (int i = 0; i < P::PT; i++) copy_async(&my.in[k][q + LPC * i][c], block + (long long)min(q + LPC * i, last) * token_stride);
        } else {
            held[k].load(block, token_stride, q, last, second);
        }
    };
    auto fetch = [&]() {
        own_tokens(0, pu, su);
        own_tokens(1, pd, sd);
        if (a.z) own_tokens(2, pz, sz);
        if (a.gy) own_tokens(3, pg, a.D);
#pragma unroll
        for (int k = 0; k < 2; k++) {
            if constexpr (FAST) {
                if (n0 < a.N) copy_async(&my.ckpt[k][lane], ck + k * second * a.N + n0);
            } else {
                load_states(ck, (size_t)(k * second) * a.N, n0, a.N, held_state[k]);
            }
        }
        pu -= (long long)su * TB; pd -= (long long)sd * TB; pz -= (long long)sz * TB; pg -= (long long)a.D * TB;
        ck -= (size_t)a.D * a.N;
    };
#pragma unroll
    for (int k = 0; k < 2; k++)
        if (n0 >= a.N) my.ckpt[k][lane] = make_float4(0.f, 0.f, 0.f, 0.f);       // (lanes of padded states: nothing is copied there)
    fetch();
    fetch_rows(blk1 - 1, last);
    put_rows((blk1 - 1) & 1);
    __syncthreads();
    for (int blk = blk1 - 1; blk >= blk0; blk--) {
        const int buf = blk & 1, end = last;
        const float4 *sB = cta.b[buf][swap ? 1 : 0] + q, *sC = cta.c[buf][swap ? 1 : 0] + q;
        if constexpr (FAST) {
            copies_done();
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int i = 0; i < P::PT; i++) my.in[k][q + LPC * i][c] = held[k].v[i];
#pragma unroll
            for (int k = 0; k < 2; k++)
                my.ckpt[k][lane] = make_float4(held_state[k][0].x, held_state[k][0].y, held_state[k][1].x, held_state[k][1].y);
        }
        f2 x[2][2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const float4 v = my.ckpt[k][lane];
            const f2 v0 = make_float2(v.x, v.y), v1 = make_float2(v.z, v.w);
            x[k][0] = (k ? live2 : live) ? (swap ? v1 : v0) : both(0.f);
            x[k][1] = (k ? live2 : live) ? (swap ? v0 : v1) : both(0.f);
            my.state[k][0][lane] = make_float4(x[k][0].x, x[k][0].y, x[k][1].x, x[k][1].y);
        }
        __syncwarp();
        {
            f2 dt[P::PT], sig[P::PT], dy[P::PT], z[P::PT];
#pragma unroll
            for (int i = 0; i < P::PT; i++) {
                const int t = q + LPC * i;
                dt[i] = add2(pair_of(my.in[1][t][c]), bias);
                sig[i] = both(1.f);
                dy[i] = a.gy ? pair_of(my.in[3][t][c]) : both(0.f);
                z[i] = a.z ? pair_of(my.in[2][t][c]) : both(0.f);
            }
            if (a.softplus) softplus_all<true>(dt, sig);
#pragma unroll
            for (int i = 0; i < P::PT; i++) {
                const int t = q + LPC * i;
                f2 u = pair_of(my.in[0][t][c]);
                const f2 g = dy[i];
                if (a.z) dy[i] = mul2(g, make_float2(z[i].x * sigm(z[i].x), z[i].y * sigm(z[i].y)));
                if (!live || t > end) dt[i].x = dy[i].x = u.x = 0.f;
                if (!live2 || t > end) dt[i].y = dy[i].y = u.y = 0.f;
                my.d[t][c] = make_float4(dt[i].x, dt[i].x * u.x, dt[i].y, dt[i].y * u.y);
                my.dy[t][c] = dy[i];
                my.own[0][t][c] = make_float4(u.x, sig[i].x, z[i].x, g.x);
                my.own[1][t][c] = make_float4(u.y, sig[i].y, z[i].y, g.y);
            }
        }
        __syncwarp();
        last += TB;
        if (blk > blk0) {
            fetch();
            fetch_rows(blk - 1, TB - 1);
        }
        // the states before the quarters
#pragma unroll
        for (int g = 0; g < TB / QT - 1; g++) {
            f2 dec[QT][2][2], in[QT][2][2];
#pragma unroll
            for (int t = 0; t < QT; t++) {
                const float4 d = my.d[g * QT + t][c];
                f2 B[2];
                pairs_at(&sB[(g * QT + t) * LPC].x, B[0], B[1]);
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        dec[t][k][m] = exponent(k ? d.z : d.x, A2[k][m]);
                        in[t][k][m] = mul2(both(k ? d.w : d.y), B[m]);
                    }
            }
#pragma unroll
            for (int t = 0; t < QT; t++)
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int m = 0; m < 2; m++) dec[t][k][m] = ex2(dec[t][k][m]);
#pragma unroll
            for (int t = 0; t < QT; t++)
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int m = 0; m < 2; m++) x[k][m] = fma2(dec[t][k][m], x[k][m], in[t][k][m]);
            my.state[0][g + 1][lane] = make_float4(x[0][0].x, x[0][0].y, x[0][1].x, x[0][1].y);
            my.state[1][g + 1][lane] = make_float4(x[1][0].x, x[1][0].y, x[1][1].x, x[1][1].y);
        }
#pragma unroll 1
        for (int quarter = TB / QT - 1; quarter >= 0; quarter--) {
            const int tb = quarter * QT;
            f2 G[QT][2][2], ah[QT][2][2], h[QT][2][2];             // [token][channel][pair]: a_t, later G_t; a_t h_{t-1}; h_t
            {
                f2 x0[2][2];
#pragma unroll
                for (int k = 0; k < 2; k++) pairs_at(&my.state[k][quarter][lane].x, x0[k][0], x0[k][1]);
                f2 in[QT][2][2];
#pragma unroll
                for (int t = 0; t < QT; t++) {
                    const float4 d = my.d[tb + t][c];
                    f2 B[2];
                    pairs_at(&sB[(tb + t) * LPC].x, B[0], B[1]);
#pragma unroll
                    for (int k = 0; k < 2; k++)
#pragma unroll
                        for (int m = 0; m < 2; m++) {
                            G[t][k][m] = exponent(k ? d.z : d.x, A2[k][m]);
                            in[t][k][m] = mul2(both(k ? d.w : d.y), B[m]);
                        }
                }
#pragma unroll
                for (int t = 0; t < QT; t++)
#pragma unroll
                    for (int k = 0; k < 2; k++)
#pragma unroll
                        for (int m = 0; m < 2; m++) G[t][k][m] = ex2(G[t][k][m]);
#pragma unroll
                for (int t = 0; t < QT; t++)
#pragma unroll
                    for (int k = 0; k < 2; k++)
#pragma unroll
                        for (int m = 0; m < 2; m++) {
                            ah[t][k][m] = mul2(G[t][k][m], t ? h[t - 1][k][m] : x0[k][m]);
                            h[t][k][m] = add2(ah[t][k][m], in[t][k][m]);
                        }
            }
#pragma unroll
            for (int t = QT - 1; t >= 0; t--) {
                const float2 dy = my.dy[tb + t][c];
                f2 C[2];
                pairs_at(&sC[(tb + t) * LPC].x, C[0], C[1]);
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        const f2 g = fma2(C[m], both(k ? dy.y : dy.x), E[k][m]);
                        E[k][m] = mul2(G[t][k][m], g);
                        G[t][k][m] = g;
                    }
            }
#pragma unroll
            for (int nb = QT / NB - 1; nb >= 0; nb--) {
                float gin[2][NB], gdec[2][NB], yv[2][NB];
#pragma unroll
                for (int j = NB - 1; j >= 0; j--) {
                    const int t = nb * NB + j;
                    const float4 d = my.d[tb + t][c];
                    const float2 dy = my.dy[tb + t][c];
                    f2 B[2], C[2], vb[2], vc[2];
                    pairs_at(&sB[(tb + t) * LPC].x, B[0], B[1]);
                    pairs_at(&sC[(tb + t) * LPC].x, C[0], C[1]);
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const f2 dt = both(k ? d.z : d.x), du = both(k ? d.w : d.y), g = both(k ? dy.y : dy.x);
                        f2 s0, s1, s2;
#pragma unroll
                        for (int m = 0; m < 2; m++) {
                            const f2 ga = mul2(G[t][k][m], ah[t][k][m]);
                            vb[m] = k ? fma2(G[t][k][m], du, vb[m]) : mul2(G[t][k][m], du);
                            vc[m] = k ? fma2(h[t][k][m], g, vc[m]) : mul2(h[t][k][m], g);
                            s0 = m ? fma2(G[t][k][m], B[m], s0) : mul2(G[t][k][m], B[m]);
                            s1 = m ? fma2(ga, A2[k][m], s1) : mul2(ga, A2[k][m]);
                            s2 = m ? fma2(C[m], h[t][k][m], s2) : mul2(C[m], h[t][k][m]);
                            gA[k][m] = fma2(ga, dt, gA[k][m]);
                        }
                        gin[k][j] = s0.x + s0.y; gdec[k][j] = s1.x + s1.y; yv[k][j] = s2.x + s2.y;
                    }
                    float *to = &my.sum[buf][(tb + t) * Q::VALUES + q];
                    sum_channels<LPC>(vb, vc, lane, [&](int kind, int n, float v) { to[(4 * kind + n) * LPC] = v; });
                }
                const f2 gi = make_float2(sum_tokens<LPC, NB>(gin[0], q), sum_tokens<LPC, NB>(gin[1], q));
                const f2 gd = make_float2(sum_tokens<LPC, NB>(gdec[0], q), sum_tokens<LPC, NB>(gdec[1], q));
                const f2 y0 = make_float2(sum_tokens<LPC, NB>(yv[0], q), sum_tokens<LPC, NB>(yv[1], q));
                // (of channels with more lanes than a batch has tokens several hold the same)
                const int t = tb + nb * NB + q % NB;
                my.res[t][c] = make_float4(gi.x, gi.y, gd.x, gd.y);
                my.res_y[t][c] = y0;
            }
        }
        __syncwarp();
        // the lane's own tokens
#pragma unroll
        for (int i = 0; i < P::PT; i++) {
            const int t = q + LPC * i;
            const float4 o0 = my.own[0][t][c], o1 = my.own[1][t][c], d = my.d[t][c], r = my.res[t][c];
            const f2 dy = my.dy[t][c], u = make_float2(o0.x, o1.x), gi = make_float2(r.x, r.y), gd = make_float2(r.z, r.w);
            const f2 graw = mul2(fma2(u, gi, mul2(gd, both(LN2))), make_float2(o0.y, o1.y));
            if (live && t <= end) {
                gD = fma2(dy, u, gD);
                gbias = add2(gbias, graw);
                const size_t at = out + (size_t)(LPC * i) * a.D;
                if (a.gu) store_pair<FAST>((F *)a.gu + at, live2, fma2(make_float2(d.x, d.z), gi, mul2(dskip, dy)));
                if (a.gdelta) store_pair<FAST>((F *)a.gdelta + at, live2, graw);
                if (a.gz) {
                    const float sx = sigm(o0.z), sy = sigm(o1.z);
                    const f2 dz = make_float2(sx * (1.f + o0.z * (1.f - sx)), sy * (1.f + o1.z * (1.f - sy)));
                    store_pair<FAST>((F *)a.gz + at, live2, mul2(mul2(make_float2(o0.w, o1.w), fma2(dskip, u, my.res_y[t][c])), dz));
                }
            }
        }
        out -= (size_t)TB * a.D;
        if (blk > blk0) put_rows(buf ^ 1);
        __syncthreads();
        if (a.part_bc) {
            for (int e = tid; e < TB * Q::VALUES; e += THREADS) {
                float s = cta.w[0].sum[buf][e];
#pragma unroll
                for (int w = 1; w < Q::WARPS; w++) s += cta.w[w].sum[buf][e];
                if (e / Q::VALUES <= end)
                    a.part_bc[((((size_t)un.cb * a.B + b) * a.T + blk * TB + e / Q::VALUES) * a.G + grp) * Q::VALUES + e % Q::VALUES] = s;
            }
        }
    }
#pragma unroll
    for (int m = 1; m < LPC; m <<= 1) {
        gD = add2(gD, make_float2(__shfl_xor_sync(FULL_MASK, gD.x, m), __shfl_xor_sync(FULL_MASK, gD.y, m)));
        gbias = add2(gbias, make_float2(__shfl_xor_sync(FULL_MASK, gbias.x, m), __shfl_xor_sync(FULL_MASK, gbias.y, m)));
    }
    float *p = a.part + ((size_t)b * a.nspan + span) * ((size_t)a.D * (a.N + 2));
#pragma unroll
    for (int k = 0; k < 2; k++) {
        if (k ? live2 : live) {
            if (span == 0 && a.gs_in) store_states(a.gs_in, row + k * a.N, n0, a.N, E[k], swap);
            if (a.part) {
                store_states(p, (size_t)(ch + k) * a.N, n0, a.N, gA[k], swap);
                if (q == 0) {
                    p[(size_t)a.D * a.N + ch + k] = k ? gD.y : gD.x;
                    p[(size_t)a.D * (a.N + 1) + ch + k] = k ? gbias.y : gbias.x;
                }
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
constexpr long long MAX_STRIDE = 1 << 26, MAX_BLOCKS = 0x7FFFFFFF, MAX_T = 0x7FFFFFFF - TB;
// (fewer than 5 states are padded to 8: one lane for four states and twice 64 channels a warp would need 255 registers and spill)
int lanes_for(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

int check_scan(const wkv_selective_scan_args_t *a) {
    if (!a) return WKV_ERR_NULL;
    if (a->B < 0 || a->T < 0 || a->D < 0 || a->N < 1 || a->N > 64 || a->G < 1 || a->D % a->G != 0 || a->time_groups < 0) return WKV_ERR_SHAPE;
    if (!known_dtype(a->dtype)) return WKV_ERR_DTYPE;
    for (long long s : {a->u_batch, a->u_token, a->delta_batch, a->delta_token, a->B_batch, a->B_token, a->C_batch, a->C_token, a->z_batch, a->z_token})
        if (s < 0) return WKV_ERR_SHAPE;
    // (the offsets inside a block of 16 tokens are 32-bit)
    for (long long s : {(long long)a->D, a->u_token, a->delta_token, a->B_token, a->C_token, a->z_token})
        if (s > MAX_STRIDE) return WKV_ERR_SHAPE;
    // (blocks of a grid: at most a warp's worth for each block of tokens, and the fold of gB and gC)
    if ((long long)a->B * a->D * (a->T / TB + 1) > MAX_BLOCKS || (long long)a->B * a->T * a->G > MAX_BLOCKS) return WKV_ERR_SHAPE;
    // (token numbers up to the end of the last block are 32-bit)
    if (a->T > MAX_T) return WKV_ERR_SHAPE;
    if (a->B == 0 || a->D == 0) return WKV_OK;
    if (!a->A || (a->T > 0 && (!a->u || !a->delta || !a->Bm || !a->Cm))) return WKV_ERR_NULL;
    return WKV_OK;
}

// n spans of whole blocks, none of them empty
int whole_spans(long long n, int nblk) {
    if (n > nblk) n = nblk;
    if (n < 1) n = 1;
    const long long len = (nblk + n - 1) / n;
    return len > 0 ? (int)((nblk + len - 1) / len) : 1;
}
int bwd_channel_blocks(const wkv_selective_scan_args_t *a) {
    const int lpc = lanes_for(a->N), per = 4 * (64 / lpc);
    return (a->D / a->G + per - 1) / per;
}
// Spans of a row, forward: none where one warp a scheduler or nearly that many are there without (512 warps: 59 us uncut, 67
// in two spans; 320 warps: 754 us uncut, 500 in twelve); else so many that a few CTAs queue for every place, of eight blocks at
// least, or of two while there are fewer warps than schedulers (2 rows of 509 tokens and 256 channels: 69 us uncut, 23 in 16).
int plan_forward(const wkv_selective_scan_args_t *a) {
    const int cpw = 64 / lanes_for(a->N), nblk = (a->T + TB - 1) / TB;
    const long long warps = (long long)a->B * a->G * ((a->D / a->G + cpw - 1) / cpw), sms = device_sm_count();
    long long n = a->time_groups;
    if (n == 0) {
        if (warps * 14 >= sms * 40) return 1;
        long long most = nblk / 2 < sms * 4 / warps ? nblk / 2 : sms * 4 / warps;
        if (nblk / 8 > most) most = nblk / 8;
        n = sms * 24 / warps < most ? sms * 24 / warps : most;
    }
    return whole_spans(n, nblk);
}

// Backward: the number of spans that a simple account of the time finds best.  A full pass of a block takes 1 with two CTAs on
// an SM and 0.77 with one (932 and 715 us for 2048 tokens); a span starts up in 1.5 blocks; the summary pass takes 0.27 of a
// full pass for the work that fills the GPU.  Against measurements of 1 to 32 spans (us: chosen, uncut, best of those tried): 4 rows of
// 4096 tokens and channels 1684, 1684, 1684; 1 of 8191 x 5120 1230, 2399, 1219; 8 of 512 x 1024 145, 166, 145.
// All of that is of 9 to 16 states.  Two CTAs fit on an SM for 9 to 32; with fewer states a CTA's shared memory is 152 KB (fp32 168), with
// more 133 (135), and an SM has one: there the account is off by up to a wave, and the choice has not been measured.  Nor are more
// than 32 spans tried: 1 x 65536 tokens of 64 channels run on 32 CTAs (790 us backward).
int plan_backward(const wkv_selective_scan_args_t *a) {
    const int nblk = (a->T + TB - 1) / TB;
    if (a->time_groups) return whole_spans(a->time_groups, nblk);
    const long long ctas = (long long)a->B * a->G * bwd_channel_blocks(a), sms = device_sm_count();
    int best = 1;
    double least = 0;
    for (int n = 1; n <= 32 && (n == 1 || 2 * n <= nblk); n++) {
        const long long x = ctas * n, rest = x % (2 * sms);
        const int len = (nblk + n - 1) / n;
        const double waves = (double)(x / (2 * sms)) + (rest == 0 ? 0.0 : rest <= sms ? 0.77 : 1.0);
        const double t = waves * (len + 1.5) + 0.27 * (double)ctas / (double)(2 * sms) * (n - 1) * (len + 1);
        if (n == 1 || t < least) { least = t; best = n; }
    }
    return whole_spans(best, nblk);
}

ScanArgs scan_args(const wkv_selective_scan_args_t *a, int nspan, bool &fast) {
    ScanArgs k = {};
    k.B = a->B; k.T = a->T; k.D = a->D; k.N = a->N; k.G = a->G; k.Dg = a->D / a->G; k.softplus = a->softplus != 0;
    k.nblk = (a->T + TB - 1) / TB;
    k.nspan = nspan;
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
    // two neighbouring channels in one access: in every tensor
    const uintptr_t two = 2 * (uintptr_t)elem_size(a->dtype) - 1;
    auto even = [&](const void *p, long long batch, long long token) {
        return p == nullptr || (batch % 2 == 0 && token % 2 == 0 && (reinterpret_cast<uintptr_t>(p) & two) == 0);
    };
    const bool pairs = k.Dg % 2 == 0 && even(a->u, a->u_batch, a->u_token) && even(a->delta, a->delta_batch, a->delta_token) &&
              even(a->z, a->z_batch, a->z_token) && even(a->y, 0, 0) && even(a->gy, 0, 0) && even(a->gu, 0, 0) && even(a->gdelta, 0, 0) &&
              even(a->gz, 0, 0);
    fast = pairs && k.vec_b && k.vec_c;
    return k;
}

template <class Fn>
int by_lanes(int lpc, Fn f) {
    switch (lpc) {
        case 2: return f(std::integral_constant<int, 2>{});
        case 4: return f(std::integral_constant<int, 4>{});
        case 8: return f(std::integral_constant<int, 8>{});
        default: return f(std::integral_constant<int, 16>{});
    }
}

size_t span_bytes(const wkv_selective_scan_args_t *a, int nspan) {
    if (nspan < 2) return 0;
    const size_t n = (size_t)a->B * nspan * a->D;
    return align256(n * a->N * 4) + align256(n * 4);
}
void place_spans(const wkv_selective_scan_args_t *a, ScanArgs &k, char *ws) {
    k.span_state = (float *)ws;
    k.span_dt = (float *)(ws + align256((size_t)a->B * k.nspan * a->D * a->N * 4));
}
struct BwdLayout {
    size_t spans, bc, params, total;
};
BwdLayout bwd_layout(const wkv_selective_scan_args_t *a) {
    const int nspan = plan_backward(a);
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
    return span_bytes(a, plan_forward(a));
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
    bool fast;
    ScanArgs k = scan_args(a, plan_forward(a), fast);
    k.y = a->y; k.state_out = a->state_out;
    const int lpc = lanes_for(a->N), cpw = 64 / lpc;
    // (more rows than a grid has blocks across go through the kernel for prompts, where a thread too reads its states before it writes)
    if (a->T == 1 && !a->ckpt && a->B <= 65535) {
        k.vec_a = a->N % 4 == 0 && aligned16(a->A);
        k.vec_s = a->N % 4 == 0 && all_aligned({a->state_in, a->state_out});
        return by_dtype(a->dtype, [&](auto f) {
            return by_lanes(lpc, [&](auto l) {
                constexpr int LANES = decltype(l)::value / 2;
                const long long threads = (long long)a->D * LANES;
                return launch_chained(k_scan_step<decltype(f), LANES>, dim3((unsigned)((threads + 255) / 256), a->B), dim3(256), 0, s, k);
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
                const int r = launch_chained(fast ? k_scan_fwd<F, LPC, true, true> : k_scan_fwd<F, LPC, true, false>,
                                             dim3((unsigned)((per_span * (k.nspan - 1) + 3) / 4)), dim3(128), 0, s, k);
                if (r != WKV_OK) return r;
            }
            return launch_chained(fast ? k_scan_fwd<F, LPC, false, true> : k_scan_fwd<F, LPC, false, false>,
                                  dim3((unsigned)((per_span * k.nspan + 3) / 4)), dim3(128), 0, s, k);
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
    bool fast;
    ScanArgs k = scan_args(a, plan_backward(a), fast);
    char *ws = (char *)a->workspace;
    if (l.spans) place_spans(a, k, ws);
    k.ckpt = (float *)a->ckpt;
    k.gy = a->gy; k.gs_out = a->gstate_out; k.gu = a->gu; k.gdelta = a->gdelta; k.gz = a->z ? a->gz : nullptr; k.gs_in = a->gstate_in;
    k.part_bc = a->gB || a->gC ? (float *)(ws + l.spans) : nullptr;
    k.part = params ? (float *)(ws + l.spans + l.bc) : nullptr;
    const int lpc = lanes_for(a->N), cpw = 64 / lpc;
    const int ncb = bwd_channel_blocks(a);
    e = by_dtype(a->dtype, [&](auto f) {
        return by_lanes(lpc, [&](auto l_) {
            using F = decltype(f);
            constexpr int LPC = decltype(l_)::value;
            if (k.nspan > 1) {
                ScanArgs m = k;
                m.ncb = (k.Dg + cpw - 1) / cpw;
                const long long units = (long long)m.ncb * a->G * (k.nspan - 1) * a->B;
                const int r = launch_chained(fast ? k_scan_bwd_summary<F, LPC, true> : k_scan_bwd_summary<F, LPC, false>, dim3((unsigned)((units + 3) / 4)), dim3(128), 0, s, m);
                if (r != WKV_OK) return r;
            }
            k.ncb = ncb;
            static unsigned char done[2][64];
            const auto kern = fast ? k_scan_bwd<F, LPC, true> : k_scan_bwd<F, LPC, false>;
            if (!set_max_smem_once(kern, BwdGeo<F, LPC>::SMEM, done[fast])) return (int)WKV_ERR_LAUNCH;
            const int r = launch_chained(kern, dim3((unsigned)((long long)ncb * a->G * k.nspan * a->B)),
                                         dim3(32 * BwdGeo<F, LPC>::WARPS), BwdGeo<F, LPC>::SMEM, s, k);
            if (r != WKV_OK || !k.part_bc) return r;
            const long long rows = (long long)a->B * a->T * a->G;
            return launch_chained(k_scan_fold_bc<F>, dim3((unsigned)((rows * 8 * LPC + 255) / 256)), dim3(256), 0, s, k.part_bc, ncb, rows,
                                  LPC, a->N, (F *)a->gB, (F *)a->gC);
        });
    });
    if (e != WKV_OK || !params) return e;
    return fold_params(k.part, a->B * k.nspan, np, fo, s);
}
