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
// A CTA owns 64 channels of a row (two a lane) and walks over its tokens in blocks of 8 warps x S tokens.  A warp's S tokens are a
// segment: from zero its state is hl and its decay P = prod a; the eight segments' (P, hl) meet in shared memory, every thread
// folds them in order (one barrier a block) and runs its segment again from the state that it then knows, its a and m i x still
// in registers.  So the serial chain is 8 + S steps a block, the gates, which are most of the work, are formed once, and every input
// is read once.  TMA brings a block's tile of each tensor into a ring in shared memory, blocks ahead, and takes the outputs from there, from the places of
// inputs that are in registers by then; rows that are not made of 16-byte pieces are copied by their warps (cp.async, in words).
//
// What bounds it (4 x 4096 x 4096 in bf16 with z, two CTAs of 256 threads an SM): forward 166 us (4.0 TB/s; the bytes take 103 at the copy
// rate), backward 297 (4.0; 185).  No single resource: special functions are busy for 63 % of the time on an SM with two CTAs (6 a token and
// channel: 4 exponentials, a root, and one reciprocal for the three sigmoids; one each took 217 us), issue 55 %, HBM 62 %; 256 CTAs are 1.73 an SM.
// Segments of 4 tokens instead of 8: 185 and, of 284 then, 306 (folds and barriers twice as often).  Registers are what limits the segment: what does not
// fit waits for L2 (forward 475 us with 40 bytes a thread of that), so that backward d and e go to shared memory, into the places of the gates, and
// 1 - i beside the ring.
//
// What is left of an open gate, 1 - i and 1 - r, has digits of its own: e^-x times the sigmoid, not a difference (which was 12 % off at a gate of 12).
// Backward 297 us, 284 with the differences; 324 with the smaller of r and 1 - r in a register, 1 - i in another, and L / (1 - a^2) formed again.
//
// Few chains: a row is cut into spans that run in parallel.  A first pass leaves what a span does to the state (its decay and its state
// from zero; backward: to E), without a barrier: its warps take an eighth of a span each.  The full pass starts from the fold of the
// spans before it.  (A cluster's CTAs on neighbouring blocks of a row, their folds exchanged through distributed shared memory at
// every step, read nothing twice, and took 2 us a step more: 4 x 4096 x 4096 forward 258 us with two CTAs a cluster, 165 without.)
//
// Backward: blocks in reverse.  The forward pass leaves the state before each block (4 bytes a channel per 64 tokens, of fp32 32); hl and
// P are formed again, and with them the segment's E from zero, so that one exchange serves both directions.
//
// 1 - a^2 is -expm1(2L): its series below 1/4 (2^-24 of it are left out there), 1 - a a above.
#include "elem_io.cuh"
#include "elem_math.cuh"
#include "sm100_primitives.cuh"
#include "tma_host.cuh"
#include "wkv_internal.h"

namespace wkv {
namespace {

constexpr int CH = 64, NW = 8, MAX_SPANS = 256;
__device__ __forceinline__ float rsqrta(float x) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr unsigned WAIT_LIMIT = 4000000u;
// (what a self-test changes in the calls of its thread)
thread_local int t_skip = -1;
thread_local unsigned t_limit = WAIT_LIMIT;

struct RecArgs {
    CUtensorMap in_spans[5];              // as `in`, the tiles of a warp
    CUtensorMap in[5], out[4];            // TILES: decay gate, input gate, x, (gy,) z; y, or gx, ginput_gate, gdecay_gate, gz
    int T, D, slabs, nspan, span;         // slabs of CH channels; spans of a row, tokens of a span (a multiple of a block)
    float c;
    const void *x, *ig, *rg, *z;
    long long x_batch, x_token, ig_batch, ig_token, rg_batch, rg_token, z_batch, z_token;
    const float *decay, *state_in;
    void *y;
    float *state_out, *ckpt;              // ckpt [B, nkept, D]: the state before every ckpt_tokens()
    int *status;
    unsigned limit;                       // polls of a wait
    int skip;                             // self-test: the block whose tiles are never loaded (-1)
    int nkept, pair;                      // pair: two neighbouring channels are one access in every output
    const void *gy;
    const float *gs_out;
    void *gx, *gig, *grg, *gz;
    float *gs_in, *part;                  // part [B * nspan, D]
    float2 *spans;                        // [B, nspan, D]: a span's decay, and its state (backward: E) from zero
};

// How rows lie: pieces of 16 bytes (TMA brings a block's tile of each tensor, and takes the outputs' away), words, or (two-byte
// elements) anywhere: a warp fetches its own tokens.
enum { TILES = 0, WORDS = 1, ANYWHERE = 2 };
// elements of a token's row in the ring: CH channels, and where rows start at any element one more word, because they are copied from the word that
// their first element is in (which is of the same allocation: those start and end at words)
__host__ __device__ constexpr int row_of(int mode) { return mode == ANYWHERE ? CH + 2 : CH; }

// Tokens of a warp in a block (S), for two CTAs an SM: what a thread keeps of its tokens has to fit in 128 registers, because what
// does not would wait for L2 (shared memory leaves no L1).
template <typename F, bool BACK>
struct Geo {
    static constexpr int S = sizeof(F) == 2 ? 8 : 4, BT = NW * S;
    static __host__ __device__ constexpr int slot(int mode) { return BT * row_of(mode); }                             // elements of one tensor's block
    static constexpr int STAGES = BACK ? 2 : 3, KEPT = BT * 32 * 8;                      // KEPT (backward): 1 - i of a block, two channels a lane
    static constexpr int ring(bool z, int mode) { return STAGES * (3 + BACK + z) * slot(mode) * (int)sizeof(F); }
};
// tokens between two states that are kept: a block of the backward pass
__host__ __device__ constexpr int ckpt_tokens(int elem) { return elem == 2 ? 64 : 32; }

// softplus(p) and its derivative over it, once per CTA and channel
struct Rate {
    float rate2, x2, ratio;               // L log2(e) = rate2 r;  -2 L = x2 r;  sigmoid(p) / softplus(p)
};
__device__ __forceinline__ Rate rate_of(float p, float c) {
    float sg;
    const float s = softplus<true>(p, sg);
    Rate r;
    // (an infinite rate becomes the largest one: a decay gate of zero then keeps the state; a NaN stays)
    float k = c * s;
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(k) : "f"(1.1e38f));
    r.rate2 = -k * LOG2E;
    r.x2 = 2.f * k;
    r.ratio = s > 1e-30f ? sg / s : (s == s ? 1.f : s);
    return r;
}

// Sigmoids of two channels' gates (Z: and of the output gate): one reciprocal for a channel's two or three, of the product of their
// 1 + e^-x, because special functions are what bounds the forward pass.  `range` adds up the products: while it is below 2^125 none
// of them has left the range; else (gates below -28 or so, infinities, NaNs, which would spread from one gate to the others) the
// caller takes the segment again with FAST = false: a reciprocal for each there, and the same bits for all others.
constexpr float RANGE = 4.2535296e37f;
// REST: and e^-x of the decay gate (at most 3e38, whose sigmoid is zero), from which r and 1 - r follow, and 1 - i as e^-x times the sigmoid: the
// difference would have no digits where a gate is open.
template <bool Z, bool FAST, bool REST>
__device__ __forceinline__ void sigmoids(f2 rg, f2 ig, f2 z, f2 &r, f2 &i, f2 &s, f2 &range, f2 &exp_r, f2 &rest_i) {
    // (a zero that the compiler does not know: it would keep what both ways have in common in registers, for all tokens)
    f2 zero = both(0.f);
    if (!FAST) asm volatile("mov.b32 %0, 0;" : "=f"(zero.x));
    auto exp_of = [&](f2 x) { return ex2(FAST ? mul2(x, both(-LOG2E)) : mul2(add2(x, both(zero.x)), both(-LOG2E))); };
    const f2 er = exp_of(rg), ei = exp_of(ig), pr = add2(er, both(1.f)), pi = add2(ei, both(1.f)), ri = mul2(pr, pi);
    f2 d = ri;
    if (Z) {
        const f2 pz = add2(exp_of(z), both(1.f));
        d = mul2(ri, pz);
        const f2 inv = make_float2(rcp(d.x), rcp(d.y)), iz = mul2(inv, pz);
        r = mul2(iz, pi);
        i = mul2(iz, pr);
        s = mul2(inv, ri);
    } else {
        const f2 inv = make_float2(rcp(d.x), rcp(d.y));
        r = mul2(inv, pi);
        i = mul2(inv, pr);
    }
    if (REST) {
        exp_r = er;
        rest_i = mul2(ei, i);
    }
    range = add2(range, d);
    if (!FAST) {
        if (REST) {
            asm("min.NaN.f32 %0, %0, %1;" : "+f"(exp_r.x) : "f"(3e38f));
            asm("min.NaN.f32 %0, %0, %1;" : "+f"(exp_r.y) : "f"(3e38f));
        }
        if (!(d.x < RANGE)) {
            r.x = sigm(rg.x);
            i.x = sigm(ig.x);
            if (Z) s.x = sigm(z.x);
            if (REST) rest_i.x = sigm(-ig.x);
        }
        if (!(d.y < RANGE)) {
            r.y = sigm(rg.y);
            i.y = sigm(ig.y);
            if (Z) s.y = sigm(z.y);
            if (REST) rest_i.y = sigm(-ig.y);
        }
    }
}
template <bool Z, bool FAST>
__device__ __forceinline__ void sigmoids(f2 rg, f2 ig, f2 z, f2 &r, f2 &i, f2 &s, f2 &range) {
    f2 exp_r, rest_i;
    sigmoids<Z, FAST, false>(rg, ig, z, r, i, s, range, exp_r, rest_i);
}
__device__ __forceinline__ bool in_range(f2 range) { return __all_sync(0xffffffffu, range.x + range.y < RANGE); }
// Decays a of two channels and q = 1 - a^2; x = -2 L.  EXACT (fp32 tensors): below x = 1/4 the decay is its power series, too (y^7 / 5040 is left
// out, 1e-10): rounded once, where ex2 is off by up to three roundings, which over the memory of a state add up.
template <bool EXACT>
__device__ __forceinline__ void decays(f2 r, f2 rate, f2 x2, f2 &a, f2 &q) {
    const f2 e = fma2(r, rate, both(EX2_MEAN)), x = mul2(r, x2);
    a = make_float2(ex2(e.x), ex2(e.y));
    if (EXACT) {
        const f2 y = mul2(x, both(0.5f));
        f2 t = fma2(y, both(1.f / 720.f), both(-1.f / 120.f));
        t = fma2(y, t, both(1.f / 24.f));
        t = fma2(y, t, both(-1.f / 6.f));
        t = fma2(y, t, both(0.5f));
        t = fma2(y, t, both(-1.f));
        t = fma2(y, t, both(1.f));
        a = make_float2(x.x < 0.25f ? t.x : a.x, x.y < 0.25f ? t.y : a.y);
    }
    f2 p = fma2(x, both(-1.f / 720.f), both(1.f / 120.f));
    p = fma2(x, p, both(-1.f / 24.f));
    p = fma2(x, p, both(1.f / 6.f));
    p = fma2(x, p, both(-0.5f));
    p = mul2(fma2(x, p, both(1.f)), x);
    const f2 d = fma2(neg2(a), a, both(1.f));
    q = make_float2(x.x < 0.25f ? p.x : d.x, x.y < 0.25f ? p.y : d.y);
}

__device__ __forceinline__ void cp_async4(void *smem, const void *g, int valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(sm100::smem_u32(smem)), "l"(g), "r"(valid) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }


// A warp's S tokens of one tensor -> its slot of the ring.  block: the CTA's first token; token: stride.  Tokens from `n` on and channels
// from D on become zeros (ANYWHERE: a channel behind the last may become anything).  Offsets inside a block are 32-bit (the host checks the strides).
template <typename F, int MODE, int S>
__device__ __forceinline__ void fill(F *slot, const F *block, int token, int warp, int n, int left, int lane) {
    constexpr int ROW = row_of(MODE);
    const uint32_t at = (uint32_t)(warp * S) * (uint32_t)token;
    if constexpr (MODE == WORDS) {
        left -= 2 * lane;
#pragma unroll
        for (int s = 0; s < S; s++) {
            const bool ok = s < n && left > 0;
            const F *p = block + (ok ? at + 2 * lane + (uint32_t)s * (uint32_t)token : 0u);
            if constexpr (sizeof(F) == 2) {
                cp_async4(slot + s * ROW + 2 * lane, p, ok ? min(left, 2) * 2 : 0);
            } else {
                cp_async4(slot + s * ROW + 2 * lane, p, ok ? 4 : 0);
                cp_async4(slot + s * ROW + 2 * lane + 1, ok && left > 1 ? p + 1 : block, ok && left > 1 ? 4 : 0);
            }
        }
    } else {
        auto word = [&](int s, int w) {
            const uintptr_t row = reinterpret_cast<uintptr_t>(block + (at + (uint32_t)s * (uint32_t)token));
            const int odd = (int)(row >> 1) & 1;
            const bool ok = s < n && 2 * w - odd < left;
            cp_async4(slot + s * ROW + 2 * w, reinterpret_cast<const void *>(((ok ? row : reinterpret_cast<uintptr_t>(block)) & ~(uintptr_t)3) + (ok ? 4 * w : 0)),
                      ok ? 4 : 0);
        };
#pragma unroll
        for (int s = 0; s < S; s++) word(s, lane);
        if (lane < S) word(lane, 32);
    }
}
// bit s: whether the row of a warp's token s starts in the second half of a word (the same for every block: their tokens are even in number)
template <typename F, int MODE, int S>
__device__ __forceinline__ uint32_t odd_rows(const void *p, long long at, long long token, int warp) {
    uint32_t m = 0;
    if constexpr (MODE == ANYWHERE) {
        const long long first = (long long)(reinterpret_cast<uintptr_t>(p) >> 1) + at + (long long)warp * S * token;
#pragma unroll
        for (int s = 0; s < S; s++) m |= (uint32_t)((first + s * token) & 1) << s;
    }
    return m;
}
template <typename F, int MODE>
__device__ __forceinline__ f2 pair_at(const F *slot, int s, int lane, uint32_t odd) {
    Raw<F, 2> r;
    const F *p = slot + s * row_of(MODE) + 2 * lane;
    r.load(p, true, 2);
    if constexpr (MODE == ANYWHERE) {
        const uint32_t next = *reinterpret_cast<const uint32_t *>(p + 2);
        r.w[0] = odd >> s & 1 ? __funnelshift_r(r.w[0], next, 16) : r.w[0];
    }
    float f[2];
    r.get(f);
    return make_float2(f[0], f[1]);
}
// Two fp32 values of a lane in the places of two tensors' pairs that it no longer needs.
template <typename F, int MODE>
__device__ __forceinline__ void keep_pair(F *slot, F *other, int s, int lane, f2 v) {
    const int at = s * row_of(MODE) + 2 * lane;
    if constexpr (sizeof(F) == 4) {
        *reinterpret_cast<f2 *>(slot + at) = v;
    } else {
        *reinterpret_cast<float *>(slot + at) = v.x;
        *reinterpret_cast<float *>(other + at) = v.y;
    }
}
template <typename F, int MODE>
__device__ __forceinline__ f2 kept_pair(const F *slot, const F *other, int s, int lane) {
    const int at = s * row_of(MODE) + 2 * lane;
    if constexpr (sizeof(F) == 4) return *reinterpret_cast<const f2 *>(slot + at);
    else return make_float2(*reinterpret_cast<const float *>(slot + at), *reinterpret_cast<const float *>(other + at));
}
// decay gates of minus infinity for the tokens behind the row's last: they keep the state (x is zero there)
template <typename F, int MODE, int S>
__device__ __forceinline__ void close_gates(F *slot, int n, int lane) {
    __syncwarp();                         // (ANYWHERE: a neighbour's word is written)
    for (int s = n; s < S; s++) {
        const float f[2] = {-INFINITY, -INFINITY};
        Raw<F, 2> r;
        r.put(f);
        r.store(slot + s * row_of(MODE) + 2 * lane, true, 2);
        if (MODE == ANYWHERE && lane == 0) r.store(slot + s * row_of(MODE) + CH, true, 2);
    }
    __syncwarp();
}
// two channels of a block's output, `at` elements from its first; left: channels there are
template <typename F>
__device__ __forceinline__ void store_out(F *block, uint32_t at, f2 v, bool pair, int left) {
    const float f[2] = {v.x, v.y};
    Raw<F, 2> r;
    r.put(f);
    r.store(block + at, pair, left);
}
// the same into a slot of the ring, from where TMA takes it (a lane's own place)
template <typename F>
__device__ __forceinline__ void put_pair(F *slot, int s, int lane, f2 v) {
    store_out<F>(slot, s * CH + 2 * lane, v, true, 2);
}

// What the thread that fills a ring keeps of it, in shared memory: blocks 0 .. asked - 1 were asked for; lost: the first one whose wait it gave up.
// A stage whose barrier still counts bytes must not be armed again: nothing is asked for once a wait has run out, so that block k's phase stays
// (k / ST) & 1.
struct Filled {
    int asked, lost;
};
constexpr int NEVER = 0x7fffffff;
// what a segment does to the state (and to E): [side][segment][channel pair]
struct Exchange {
    float4 seg[2][NW][32];                // P, hl of two channels
    uint64_t full[4];
    int abort;
    Filled filled;
};
struct alignas(16) ExchangeBack {
    float4 seg[2][NW][32];                // P, hl
    f2 segE[2][NW][32];                   // E from zero
    f2 sum[NW][32];
    uint64_t full[4];
    int abort;
    Filled filled;
};

// The ring's blocks: TILES: one thread has TMA bring the block's tile of each tensor, all wait on the stage's barrier (bounded: a wait
// that runs out is reported, the others of the CTA end at once, and the call's results are invalid; no stage is filled after it).
template <int ST, class X>
__device__ __forceinline__ void init_tiles(X &ex) {
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) sm100::mbar_init(ex.full + i, 1);
        ex.abort = 0;
        ex.filled = {0, NEVER};
        sm100::fence_mbar_init();
    }
    __syncthreads();
}
// bar: of block k; fills: whether this thread fills the ring
__device__ __forceinline__ void await_tile(uint64_t *bar, int parity, int k, int *abort, Filled *f, bool fills, const RecArgs &g) {
    if (sm100::mbar_wait_or_abort(bar, parity, abort, g.limit)) return;
    *(volatile int *)abort = 1;
    if (g.status != nullptr) atomicOr(g.status, WKV_RECURRENCE_TIMEOUT);
    if (fills) f->lost = min(f->lost, k);
}
__device__ __forceinline__ bool given_up(const int *abort) { return *(volatile const int *)abort != 0; }
// Before the CTA's shared memory may go: what was asked for and not waited for has landed (bounded).
template <int ST>
__device__ __forceinline__ void let_tiles_land(uint64_t *bars, const Filled &f, unsigned limit) {
    for (int k = f.lost; k < f.asked; k++) sm100::mbar_wait_landed(bars + k % ST, (k / ST) & 1, limit);
}
// two channels' state (or E) behind the spans from `first` up to `last`
__device__ __forceinline__ f2 fold_spans(const RecArgs &g, int b, int first, int last, int dir, int ch, f2 h) {
    const float2 *p = g.spans + (size_t)b * g.nspan * g.D + ch;
#pragma unroll 4
    for (int i = first; i != last; i += dir) {
        if (ch < g.D) {
            const float2 q = p[(size_t)i * g.D];
            h.x = fmaf(q.x, h.x, q.y);
        }
        if (ch + 1 < g.D) {
            const float2 q = p[(size_t)i * g.D + 1];
            h.y = fmaf(q.x, h.y, q.y);
        }
    }
    return h;
}

template <typename F, bool Z, int MODE>
__global__ void __launch_bounds__(256, 2) k_rec_fwd(const __grid_constant__ RecArgs g) {
    pdl_wait();
    pdl_trigger();
    using G = Geo<F, false>;
    constexpr int S = G::S, BT = G::BT, ROW = row_of(MODE), SLOT = G::slot(MODE), NT = 3 + Z, ST = G::STAGES, RING = ST * NT * SLOT * (int)sizeof(F);
    extern __shared__ __align__(128) unsigned char smem[];
    Exchange &ex = *reinterpret_cast<Exchange *>(smem + RING);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int span = blockIdx.x % g.nspan, chain = blockIdx.x / g.nspan, b = chain / g.slabs, ch0 = (chain - b * g.slabs) * CH, ch = ch0 + 2 * lane;
    const long long begin = (long long)span * g.span;
    const int nsteps = (int)((min((long long)g.T, begin + g.span) - begin + BT - 1) / BT);
    F *ring = reinterpret_cast<F *>(smem);                          // [stage][tensor][warp][S][CH]

    const Rate k0 = rate_of(ch < g.D ? g.decay[ch] : 0.f, g.c), k1 = rate_of(ch + 1 < g.D ? g.decay[ch + 1] : 0.f, g.c);
    const f2 rate = make_float2(k0.rate2, k1.rate2), x2 = make_float2(k0.x2, k1.x2);
    f2 h = make_float2(0.f, 0.f);
    if (g.state_in != nullptr) {
        if (ch < g.D) h.x = g.state_in[(size_t)b * g.D + ch];
        if (ch + 1 < g.D) h.y = g.state_in[(size_t)b * g.D + ch + 1];
    }
    if (span > 0) h = fold_spans(g, b, 0, span, 1, ch, h);
    const uint32_t odd_r = odd_rows<F, MODE, S>(g.rg, b * g.rg_batch + begin * g.rg_token + ch0, g.rg_token, warp),
                   odd_i = odd_rows<F, MODE, S>(g.ig, b * g.ig_batch + begin * g.ig_token + ch0, g.ig_token, warp),
                   odd_x = odd_rows<F, MODE, S>(g.x, b * g.x_batch + begin * g.x_token + ch0, g.x_token, warp),
                   odd_z = Z ? odd_rows<F, MODE, S>(g.z, b * g.z_batch + begin * g.z_token + ch0, g.z_token, warp) : 0u;
    auto start = [&](int step) {
        const long long t0 = begin + (long long)step * BT;
        F *slot = ring + (step % ST) * NT * SLOT;
        if constexpr (MODE == TILES) {
            sm100::mbar_expect_tx(ex.full + step % ST, NT * SLOT * sizeof(F));
            ex.filled.asked++;
            if (step == g.skip) return;
#pragma unroll
            for (int i = 0; i < NT; i++) sm100::tma_load_3d(slot + i * SLOT, g.in + i, ex.full + step % ST, ch0, (int)t0, b);
        } else {
            const int n = (int)max(0ll, min((long long)S, g.T - (t0 + warp * S))), left = g.D - ch0;
            slot += warp * S * ROW;
            fill<F, MODE, S>(slot, (const F *)g.rg + (b * g.rg_batch + t0 * g.rg_token + ch0), (int)g.rg_token, warp, n, left, lane);
            fill<F, MODE, S>(slot + SLOT, (const F *)g.ig + (b * g.ig_batch + t0 * g.ig_token + ch0), (int)g.ig_token, warp, n, left, lane);
            fill<F, MODE, S>(slot + 2 * SLOT, (const F *)g.x + (b * g.x_batch + t0 * g.x_token + ch0), (int)g.x_token, warp, n, left, lane);
            if (Z) fill<F, MODE, S>(slot + 3 * SLOT, (const F *)g.z + (b * g.z_batch + t0 * g.z_token + ch0), (int)g.z_token, warp, n, left, lane);
        }
    };
    if constexpr (MODE == TILES) {
        init_tiles<ST>(ex);
        if (threadIdx.x == 0) {
            for (int p = 0; p < min(ST, nsteps); p++) start(p);
        }
    } else {
#pragma unroll
        for (int p = 0; p < ST - 1; p++) {
            if (p < nsteps) start(p);
            cp_commit();
        }
    }
    for (int step = 0; step < nsteps; step++) {
        if constexpr (MODE == TILES) {
            await_tile(ex.full + step % ST, (step / ST) & 1, step, &ex.abort, &ex.filled, threadIdx.x == 0, g);
        } else {
            __syncwarp();                                           // (all lanes are done with the slot that is filled now)
            if (step + ST - 1 < nsteps) start(step + ST - 1);
            cp_commit();
            cp_wait<ST - 1>();
            __syncwarp();
        }
        F *slot = ring + (step % ST) * NT * SLOT + warp * S * ROW;
        const long long t0 = begin + (long long)step * BT;
        const int n = (int)max(0ll, min((long long)S, g.T - (t0 + warp * S)));          // this warp's tokens of the block
        if (n < S) close_gates<F, MODE, S>(slot, n, lane);
        f2 a[S], v[S], gate[Z ? S : 1], P, hl;
        auto segment = [&](auto fast) {
            f2 range = both(0.f);
            P = both(1.f);
            hl = both(0.f);
#pragma unroll
            for (int s = 0; s < S; s++) {
                const f2 x = pair_at<F, MODE>(slot + 2 * SLOT, s, lane, odd_x), z = Z ? pair_at<F, MODE>(slot + 3 * SLOT, s, lane, odd_z) : both(0.f);
                f2 r, in, sz;
                sigmoids<Z, decltype(fast)::value>(pair_at<F, MODE>(slot, s, lane, odd_r), pair_at<F, MODE>(slot + SLOT, s, lane, odd_i), z, r, in, sz, range);
                f2 q;
                decays<sizeof(F) == 4>(r, rate, x2, a[s], q);
                v[s] = mul2(mul2(make_float2(sqrtf(q.x), sqrtf(q.y)), in), x);
                if (Z) gate[s] = mul2(z, sz);
                hl = fma2(a[s], hl, v[s]);
                P = mul2(P, a[s]);
            }
            return in_range(range);
        };
        if (!segment(std::true_type{})) segment(std::false_type{});
        const int side = step & 1;
        ex.seg[side][warp][lane] = make_float4(P.x, P.y, hl.x, hl.y);
        if (MODE == TILES && lane == 0) sm100::tma_store_wait_read();                   // (of the block before: its stage is filled next)
        __syncthreads();
        if (MODE == TILES && threadIdx.x == 0 && step > 0 && step + ST - 1 < nsteps && !given_up(&ex.abort)) start(step + ST - 1);
        f2 hs = h;                                                  // before this warp's segment
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float4 q = ex.seg[side][w][lane];
            if (w == warp) hs = h;
            h = fma2(make_float2(q.x, q.y), h, make_float2(q.z, q.w));
        }
        constexpr int CKPT = ckpt_tokens(sizeof(F));
        static_assert(BT == CKPT, "the state before a block is kept");
        if (g.ckpt != nullptr && warp == 0) {
            float *c = g.ckpt + ((size_t)b * g.nkept + t0 / CKPT) * g.D + ch;
            if (ch < g.D) c[0] = hs.x;
            if (ch + 1 < g.D) c[1] = hs.y;
        }
        if constexpr (MODE == TILES) {
#pragma unroll
            for (int s = 0; s < S; s++) {
                hs = fma2(a[s], hs, v[s]);
                put_pair(slot + 2 * SLOT, s, lane, Z ? mul2(hs, gate[s]) : hs);
            }
            sm100::fence_async_smem();
            __syncwarp();
            if (lane == 0 && n > 0) {
                sm100::tma_store_3d(g.out, slot + 2 * SLOT, ch0, (int)t0 + warp * S, b);
                sm100::tma_store_commit();
            }
        } else {
            const int m = ch < g.D ? n : 0;
            F *y = (F *)g.y + (((size_t)b * g.T + t0) * g.D + ch0);
#pragma unroll
            for (int s = 0; s < S; s++) {
                hs = fma2(a[s], hs, v[s]);
                if (s < m) store_out(y, (uint32_t)(warp * S + s) * (uint32_t)g.D + 2 * lane, Z ? mul2(hs, gate[s]) : hs, g.pair, g.D - ch);
            }
        }
    }
    if (MODE == TILES && lane == 0) sm100::tma_store_wait_all();
    if (MODE == TILES && threadIdx.x == 0) let_tiles_land<ST>(ex.full, ex.filled, g.limit);
    if (g.state_out != nullptr && warp == 0 && span == g.nspan - 1) {
        if (ch < g.D) g.state_out[(size_t)b * g.D + ch] = h.x;
        if (ch + 1 < g.D) g.state_out[(size_t)b * g.D + ch + 1] = h.y;
    }
}

template <typename F, bool Z, int MODE>
__global__ void __launch_bounds__(256, 2) k_rec_bwd(const __grid_constant__ RecArgs g) {
    pdl_wait();
    pdl_trigger();
    using G = Geo<F, true>;
    constexpr int S = G::S, BT = G::BT, ROW = row_of(MODE), SLOT = G::slot(MODE), NT = 4 + Z, ST = G::STAGES, RING = ST * NT * SLOT * (int)sizeof(F);
    constexpr int CKPT = ckpt_tokens(sizeof(F));
    static_assert(BT == CKPT, "a block starts from a state that is kept");
    extern __shared__ __align__(128) unsigned char smem[];
    ExchangeBack &ex = *reinterpret_cast<ExchangeBack *>(smem + RING);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int span = blockIdx.x % g.nspan, chain = blockIdx.x / g.nspan, b = chain / g.slabs, ch0 = (chain - b * g.slabs) * CH, ch = ch0 + 2 * lane;
    const long long begin = (long long)span * g.span;
    const int nsteps = (int)((min((long long)g.T, begin + g.span) - begin + BT - 1) / BT);
    F *ring = reinterpret_cast<F *>(smem);

    const Rate k0 = rate_of(ch < g.D ? g.decay[ch] : 0.f, g.c), k1 = rate_of(ch + 1 < g.D ? g.decay[ch + 1] : 0.f, g.c);
    const f2 rate = make_float2(k0.rate2, k1.rate2), x2 = make_float2(k0.x2, k1.x2);
    const f2 rate_e = mul2(x2, both(-0.5f));                        // L = rate_e r
    f2 *kept = reinterpret_cast<f2 *>(smem + RING + sizeof(ExchangeBack)) + warp * S * 32 + lane;       // [warp][S][lane]: 1 - i
    f2 E = make_float2(0.f, 0.f), total = make_float2(0.f, 0.f);
    if (g.gs_out != nullptr) {
        if (ch < g.D) E.x = g.gs_out[(size_t)b * g.D + ch];
        if (ch + 1 < g.D) E.y = g.gs_out[(size_t)b * g.D + ch + 1];
    }
    const uint32_t odd_r = odd_rows<F, MODE, S>(g.rg, b * g.rg_batch + begin * g.rg_token + ch0, g.rg_token, warp),
                   odd_i = odd_rows<F, MODE, S>(g.ig, b * g.ig_batch + begin * g.ig_token + ch0, g.ig_token, warp),
                   odd_x = odd_rows<F, MODE, S>(g.x, b * g.x_batch + begin * g.x_token + ch0, g.x_token, warp),
                   odd_z = Z ? odd_rows<F, MODE, S>(g.z, b * g.z_batch + begin * g.z_token + ch0, g.z_token, warp) : 0u,
                   odd_g = odd_rows<F, MODE, S>(g.gy, ((long long)b * g.T + begin) * g.D + ch0, g.D, warp);
    // (k counts the steps in the order of the walk)
    if (span < g.nspan - 1) E = fold_spans(g, b, g.nspan - 1, span, -1, ch, E);
    auto start = [&](int k) {
        const long long t0 = begin + (long long)(nsteps - 1 - k) * BT;
        F *slot = ring + (k % ST) * NT * SLOT;
        if constexpr (MODE == TILES) {
            sm100::mbar_expect_tx(ex.full + k % ST, NT * SLOT * sizeof(F));
            ex.filled.asked++;
            if (k == g.skip) return;
#pragma unroll
            for (int i = 0; i < NT; i++) sm100::tma_load_3d(slot + i * SLOT, g.in + i, ex.full + k % ST, ch0, (int)t0, b);
        } else {
            const int n = (int)max(0ll, min((long long)S, g.T - (t0 + warp * S))), left = g.D - ch0;
            slot += warp * S * ROW;
            fill<F, MODE, S>(slot, (const F *)g.rg + (b * g.rg_batch + t0 * g.rg_token + ch0), (int)g.rg_token, warp, n, left, lane);
            fill<F, MODE, S>(slot + SLOT, (const F *)g.ig + (b * g.ig_batch + t0 * g.ig_token + ch0), (int)g.ig_token, warp, n, left, lane);
            fill<F, MODE, S>(slot + 2 * SLOT, (const F *)g.x + (b * g.x_batch + t0 * g.x_token + ch0), (int)g.x_token, warp, n, left, lane);
            if (g.gy != nullptr) fill<F, MODE, S>(slot + 3 * SLOT, (const F *)g.gy + (((size_t)b * g.T + t0) * g.D + ch0), g.D, warp, n, left, lane);
            else fill<F, MODE, S>(slot + 3 * SLOT, (const F *)g.x, 0, warp, 0, left, lane);         // (no incoming gradient: zeros)
            if (Z) fill<F, MODE, S>(slot + 4 * SLOT, (const F *)g.z + (b * g.z_batch + t0 * g.z_token + ch0), (int)g.z_token, warp, n, left, lane);
        }
    };
    if constexpr (MODE == TILES) {
        init_tiles<ST>(ex);
        if (threadIdx.x == 0) {
            for (int p = 0; p < min(ST, nsteps); p++) start(p);
        }
    } else {
#pragma unroll
        for (int p = 0; p < ST - 1; p++) {
            if (p < nsteps) start(p);
            cp_commit();
        }
    }
    for (int k = 0; k < nsteps; k++) {
        const long long t0 = begin + (long long)(nsteps - 1 - k) * BT;
        f2 h = make_float2(0.f, 0.f);                               // before the block
        {
            const float *c = g.ckpt + ((size_t)b * g.nkept + t0 / CKPT) * g.D + ch;
            if (ch < g.D) h.x = c[0];
            if (ch + 1 < g.D) h.y = c[1];
        }
        if constexpr (MODE == TILES) {
            await_tile(ex.full + k % ST, (k / ST) & 1, k, &ex.abort, &ex.filled, threadIdx.x == 0, g);
        } else {
            __syncwarp();
            if (k + ST - 1 < nsteps) start(k + ST - 1);
            cp_commit();
            cp_wait<ST - 1>();
            __syncwarp();
        }
        F *slot = ring + (k % ST) * NT * SLOT + warp * S * ROW;
        const int n = (int)max(0ll, min((long long)S, g.T - (t0 + warp * S)));
        if (n < S) close_gates<F, MODE, S>(slot, n, lane);
        // er: e^-x of the decay gate.  i is m i / m, and 1 / (1 - a^2) the square of 1 / m.
        f2 a[S], er[S], mi[S], rs[S], sz[Z ? S : 1], P, hl, El = both(0.f);
        auto segment = [&](auto fast) {
            f2 range = both(0.f);
            P = both(1.f);
            hl = both(0.f);
#pragma unroll
            for (int s = 0; s < S; s++) {
                // (loads of all tokens at once would need registers that there are not: 200 bytes a thread went to L2)
                if (s % 2 == 0) __syncwarp();
                const f2 z = Z ? pair_at<F, MODE>(slot + 4 * SLOT, s, lane, odd_z) : both(0.f);
                f2 r, in, rest, q;
                sigmoids<Z, decltype(fast)::value, true>(pair_at<F, MODE>(slot, s, lane, odd_r), pair_at<F, MODE>(slot + SLOT, s, lane, odd_i), z, r, in, sz[Z ? s : 0], range, er[s], rest);
                kept[s * 32] = rest;
                decays<sizeof(F) == 4>(r, rate, x2, a[s], q);
                // (where 1 - a^2 is zero, so are L and m: any factor does; the smallest normal number keeps its root, a NaN stays)
                f2 low = q;
                asm("max.NaN.f32 %0, %0, %1;" : "+f"(low.x) : "f"(1.17549435e-38f));
                asm("max.NaN.f32 %0, %0, %1;" : "+f"(low.y) : "f"(1.17549435e-38f));
                rs[s] = make_float2(rsqrta(low.x), rsqrta(low.y));
                mi[s] = mul2(mul2(q, rs[s]), in);
                hl = fma2(a[s], hl, mul2(mi[s], pair_at<F, MODE>(slot + 2 * SLOT, s, lane, odd_x)));
                P = mul2(P, a[s]);
            }
            return in_range(range);
        };
        if (!segment(std::true_type{})) segment(std::false_type{});
        __syncwarp();
        // d = gy silu(z), and e, what is left of gz without h, go where the gates, gy and z were
#pragma unroll
        for (int s = S - 1; s >= 0; s--) {
            __syncwarp();             // (ANYWHERE: a neighbour reads this lane's words.  All: loads moved up would need registers that there are not)
            f2 d = pair_at<F, MODE>(slot + 3 * SLOT, s, lane, odd_g);
            if (Z) {
                // silu' = sz (1 + z (1 - sz)).  From 17 on z (1 - sz) is below 7e-7, and the difference is made of sz's roundings: with 17 in place of a
                // larger z they stay below 3e-6.
                const f2 z = pair_at<F, MODE>(slot + 4 * SLOT, s, lane, odd_z), gs = mul2(d, sz[Z ? s : 0]), zc = make_float2(fminf(z.x, 17.f), fminf(z.y, 17.f));
                d = mul2(gs, z);
                if (MODE == ANYWHERE) __syncwarp();
                keep_pair<F, MODE>(slot + 4 * SLOT, slot + 3 * SLOT, s, lane, mul2(gs, fma2(zc, sub2(both(1.f), sz[Z ? s : 0]), both(1.f))));
            }
            keep_pair<F, MODE>(slot, slot + SLOT, s, lane, d);
            El = mul2(a[s], add2(d, El));
        }
        const int side = k & 1;
        ex.seg[side][warp][lane] = make_float4(P.x, P.y, hl.x, hl.y);
        ex.segE[side][warp][lane] = El;
        if (MODE == TILES && lane == 0) sm100::tma_store_wait_read();
        __syncthreads();
        if (MODE == TILES && threadIdx.x == 0 && k > 0 && k + ST - 1 < nsteps && !given_up(&ex.abort)) start(k + ST - 1);
        f2 Es = E;                                                  // behind this warp's segment
#pragma unroll
        for (int w = NW - 1; w > 0; w--)
            if (w > warp) {
                const float4 q = ex.seg[side][w][lane];
                Es = fma2(make_float2(q.x, q.y), Es, ex.segE[side][w][lane]);
            }
        E = fma2(P, Es, El);
#pragma unroll
        for (int w = NW - 2; w >= 0; w--)
            if (w < warp) {
                const float4 q = ex.seg[side][w][lane];
                E = fma2(make_float2(q.x, q.y), E, ex.segE[side][w][lane]);
            }
#pragma unroll
        for (int w = 0; w < NW - 1; w++)
            if (w < warp) {
                const float4 q = ex.seg[side][w][lane];
                h = fma2(make_float2(q.x, q.y), h, make_float2(q.z, q.w));
            }
        f2 hb[S + 1];                                               // the states before the tokens
        hb[0] = h;
#pragma unroll
        for (int s = 0; s < S; s++) hb[s + 1] = fma2(a[s], hb[s], mul2(mi[s], pair_at<F, MODE>(slot + 2 * SLOT, s, lane, odd_x)));
        const int m = ch < g.D ? n : 0;
        const size_t block = ((size_t)b * g.T + t0) * g.D + ch0;
#pragma unroll
        for (int s = S - 1; s >= 0; s--) {
            const f2 v = mul2(mi[s], pair_at<F, MODE>(slot + 2 * SLOT, s, lane, odd_x));
            const f2 p1 = add2(er[s], both(1.f)), r = make_float2(rcp(p1.x), rcp(p1.y)), rest = mul2(er[s], r);
            const f2 ar = mul2(a[s], rate_e), Gs = add2(kept_pair<F, MODE>(slot, slot + SLOT, s, lane), Es);
            Es = mul2(a[s], Gs);
            const f2 gx = mul2(Gs, mi[s]), gi = mul2(mul2(Gs, v), kept[s * 32]);
            // G (h a L - i x a^2 L / m), i / m = m i / m^2; r first, which alone may be as small as 1 / m^2 is large
            const f2 gLL = mul2(Gs, sub2(mul2(hb[s], mul2(ar, r)), mul2(mul2(mul2(mul2(mul2(v, rs[s]), rs[s]), r), a[s]), ar)));
            total = add2(total, gLL);
            const f2 gr = mul2(gLL, rest);
            const f2 gz = Z ? mul2(kept_pair<F, MODE>(slot + 4 * SLOT, slot + 3 * SLOT, s, lane), hb[s + 1]) : both(0.f);
            if constexpr (MODE == TILES) {
                put_pair(slot, s, lane, gr);
                put_pair(slot + SLOT, s, lane, gi);
                put_pair(slot + 2 * SLOT, s, lane, gx);
                if (Z) put_pair(slot + 3 * SLOT, s, lane, gz);
            } else if (s < m) {
                const uint32_t at = (uint32_t)(warp * S + s) * (uint32_t)g.D + 2 * lane;
                if (g.gx != nullptr) store_out((F *)g.gx + block, at, gx, g.pair, g.D - ch);
                if (g.gig != nullptr) store_out((F *)g.gig + block, at, gi, g.pair, g.D - ch);
                if (g.grg != nullptr) store_out((F *)g.grg + block, at, gr, g.pair, g.D - ch);
                if (Z && g.gz != nullptr) store_out((F *)g.gz + block, at, gz, g.pair, g.D - ch);
            }
        }
        if constexpr (MODE == TILES) {
            sm100::fence_async_smem();
            __syncwarp();
            if (lane == 0 && n > 0) {
                const int t = (int)t0 + warp * S;
                if (g.grg != nullptr) sm100::tma_store_3d(g.out + 2, slot, ch0, t, b);
                if (g.gig != nullptr) sm100::tma_store_3d(g.out + 1, slot + SLOT, ch0, t, b);
                if (g.gx != nullptr) sm100::tma_store_3d(g.out, slot + 2 * SLOT, ch0, t, b);
                if (Z && g.gz != nullptr) sm100::tma_store_3d(g.out + 3, slot + 3 * SLOT, ch0, t, b);
                sm100::tma_store_commit();
            }
        }
    }
    if (MODE == TILES && lane == 0) sm100::tma_store_wait_all();
    if (MODE == TILES && threadIdx.x == 0) let_tiles_land<ST>(ex.full, ex.filled, g.limit);
    if (g.gs_in != nullptr && warp == 0 && span == 0) {
        if (ch < g.D) g.gs_in[(size_t)b * g.D + ch] = E.x;
        if (ch + 1 < g.D) g.gs_in[(size_t)b * g.D + ch + 1] = E.y;
    }
    if (g.part != nullptr) {
        ex.sum[warp][lane] = total;
        __syncthreads();
        if (warp == 0) {
#pragma unroll
            for (int w = 1; w < NW; w++) total = add2(total, ex.sum[w][lane]);
            float *p = g.part + ((size_t)b * g.nspan + span) * g.D + ch;
            if (ch < g.D) p[0] = total.x * k0.ratio;
            if (ch + 1 < g.D) p[1] = total.y * k1.ratio;
        }
    }
}

// What a span does to the state, or (BACK) to E: its warps take an eighth of its tokens each, with a ring each, and meet at its end.
template <typename F, bool Z, int MODE, bool BACK>
__global__ void __launch_bounds__(256, 2) k_rec_spans(const __grid_constant__ RecArgs g) {
    pdl_wait();
    pdl_trigger();
    constexpr int S = Geo<F, BACK>::S, NT = BACK ? 2 + Z : 3, ST = 4, SLOT = S * row_of(MODE);
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float4 seg[NW][32];
    __shared__ uint64_t bars[NW][ST];
    __shared__ int abort;
    __shared__ Filled filled[NW];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // (the last span forward and the first one backward are not needed)
    const int n1 = g.nspan - 1, span = blockIdx.x % n1 + BACK, chain = blockIdx.x / n1, b = chain / g.slabs, ch0 = (chain - b * g.slabs) * CH, ch = ch0 + 2 * lane;
    F *ring = reinterpret_cast<F *>(smem) + warp * ST * NT * SLOT;
    const Rate k0 = rate_of(ch < g.D ? g.decay[ch] : 0.f, g.c), k1 = rate_of(ch + 1 < g.D ? g.decay[ch + 1] : 0.f, g.c);
    const f2 rate = make_float2(k0.rate2, k1.rate2), x2 = make_float2(k0.x2, k1.x2);
    // this warp's tokens
    const long long begin = (long long)span * g.span, end = min((long long)g.T, begin + g.span), part = g.span / NW;
    const long long from = min(end, begin + warp * part), to = min(end, from + part);
    const int nsteps = (int)((to - from + S - 1) / S);
    const uint32_t odd_r = odd_rows<F, MODE, S>(g.rg, b * g.rg_batch + from * g.rg_token + ch0, g.rg_token, 0),
                   odd_i = odd_rows<F, MODE, S>(g.ig, b * g.ig_batch + from * g.ig_token + ch0, g.ig_token, 0),
                   odd_x = odd_rows<F, MODE, S>(g.x, b * g.x_batch + from * g.x_token + ch0, g.x_token, 0),
                   odd_z = Z ? odd_rows<F, MODE, S>(g.z, b * g.z_batch + from * g.z_token + ch0, g.z_token, 0) : 0u,
                   odd_g = odd_rows<F, MODE, S>(g.gy, ((long long)b * g.T + from) * g.D + ch0, g.D, 0);
    auto at_step = [&](int k) { return from + (long long)(BACK ? nsteps - 1 - k : k) * S; };
    auto start = [&](int k) {
        const long long t0 = at_step(k);
        F *slot = ring + (k % ST) * NT * SLOT;
        if constexpr (MODE == TILES) {
            if (lane == 0) {
                uint64_t *bar = &bars[warp][k % ST];
                sm100::mbar_expect_tx(bar, NT * SLOT * sizeof(F));
                filled[warp].asked++;
                if (k == g.skip) return;
                sm100::tma_load_3d(slot, g.in_spans, bar, ch0, (int)t0, b);
                sm100::tma_load_3d(slot + SLOT, g.in_spans + (BACK ? 3 : 1), bar, ch0, (int)t0, b);
                if (!BACK || Z) sm100::tma_load_3d(slot + 2 * SLOT, g.in_spans + (BACK ? 4 : 2), bar, ch0, (int)t0, b);
            }
        } else {
            const int n = (int)min((long long)S, to - t0), left = g.D - ch0;
            fill<F, MODE, S>(slot, (const F *)g.rg + (b * g.rg_batch + t0 * g.rg_token + ch0), (int)g.rg_token, 0, n, left, lane);
            if (!BACK) {
                fill<F, MODE, S>(slot + SLOT, (const F *)g.ig + (b * g.ig_batch + t0 * g.ig_token + ch0), (int)g.ig_token, 0, n, left, lane);
                fill<F, MODE, S>(slot + 2 * SLOT, (const F *)g.x + (b * g.x_batch + t0 * g.x_token + ch0), (int)g.x_token, 0, n, left, lane);
            } else {
                if (g.gy != nullptr) fill<F, MODE, S>(slot + SLOT, (const F *)g.gy + (((size_t)b * g.T + t0) * g.D + ch0), g.D, 0, n, left, lane);
                else fill<F, MODE, S>(slot + SLOT, (const F *)g.x, 0, 0, 0, left, lane);
                if (Z) fill<F, MODE, S>(slot + 2 * SLOT, (const F *)g.z + (b * g.z_batch + t0 * g.z_token + ch0), (int)g.z_token, 0, n, left, lane);
            }
        }
    };
    if constexpr (MODE == TILES) {
        if (lane == 0) {
            for (int i = 0; i < ST; i++) sm100::mbar_init(&bars[warp][i], 1);
            filled[warp] = {0, NEVER};
            sm100::fence_mbar_init();
        }
        if (threadIdx.x == 0) abort = 0;
        __syncthreads();
    }
#pragma unroll
    for (int p = 0; p < ST - 1; p++) {
        if (p < nsteps) start(p);
        if (MODE != TILES) cp_commit();
    }
    f2 P = both(1.f), h = both(0.f);
    for (int k = 0; k < nsteps; k++) {
        __syncwarp();
        if (k + ST - 1 < nsteps && (MODE != TILES || !given_up(&abort))) start(k + ST - 1);
        if constexpr (MODE == TILES) {
            await_tile(&bars[warp][k % ST], (k / ST) & 1, k, &abort, filled + warp, lane == 0, g);
        } else {
            cp_commit();
            cp_wait<ST - 1>();
            __syncwarp();
        }
        F *slot = ring + (k % ST) * NT * SLOT;
        const int n = (int)min((long long)S, to - at_step(k));
        if (n < S) {
            close_gates<F, MODE, S>(slot, n, lane);
            // (backward it is the first step, and TMA fills the stage again: ordered behind these stores by the fence, and by the warp's barrier
            // that every refill stands behind)
            if (MODE == TILES) sm100::fence_async_smem();
        }
        f2 a[S], v[S];
        auto gates = [&](auto fast) {
            f2 range = both(0.f);
#pragma unroll
            for (int s = 0; s < S; s++) {
                f2 r, in, sz;
                if (!BACK) {
                    sigmoids<false, decltype(fast)::value>(pair_at<F, MODE>(slot, s, lane, odd_r), pair_at<F, MODE>(slot + SLOT, s, lane, odd_i), both(0.f), r, in, sz, range);
                    f2 q;
                    decays<sizeof(F) == 4>(r, rate, x2, a[s], q);
                    v[s] = mul2(mul2(make_float2(sqrtf(q.x), sqrtf(q.y)), in), pair_at<F, MODE>(slot + 2 * SLOT, s, lane, odd_x));
                } else {
                    const f2 z = Z ? pair_at<F, MODE>(slot + 2 * SLOT, s, lane, odd_z) : both(0.f);
                    sigmoids<false, decltype(fast)::value>(pair_at<F, MODE>(slot, s, lane, odd_r), z, both(0.f), r, sz, in, range);
                    f2 q;
                    decays<sizeof(F) == 4>(r, rate, x2, a[s], q);
                    v[s] = pair_at<F, MODE>(slot + SLOT, s, lane, odd_g);
                    if (Z) v[s] = mul2(v[s], mul2(z, sz));
                }
            }
            return in_range(range);
        };
        if (!gates(std::true_type{})) gates(std::false_type{});
#pragma unroll
        for (int i = 0; i < S; i++) {
            const int s = BACK ? S - 1 - i : i;
            h = BACK ? mul2(a[s], add2(v[s], h)) : fma2(a[s], h, v[s]);
            P = mul2(P, a[s]);
        }
    }
    if constexpr (MODE == TILES) {
        if (lane == 0) let_tiles_land<ST>(bars[warp], filled[warp], g.limit);
    }
    seg[warp][lane] = make_float4(P.x, P.y, h.x, h.y);
    __syncthreads();
    if (warp == 0) {
        P = both(1.f);
        h = both(0.f);
#pragma unroll
        for (int i = 0; i < NW; i++) {
            const float4 q = seg[BACK ? NW - 1 - i : i][lane];
            h = fma2(make_float2(q.x, q.y), h, make_float2(q.z, q.w));
            P = mul2(P, make_float2(q.x, q.y));
        }
        float2 *o = g.spans + ((size_t)b * g.nspan + span) * g.D + ch;
        if (ch < g.D) o[0] = make_float2(P.x, h.x);
        if (ch + 1 < g.D) o[1] = make_float2(P.y, h.y);
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
        f2 a, q;
        decays<sizeof(F) == 4>(both(sigm(rg)), both(k.rate2), both(k.x2), a, q);
        return fmaf(a.x, h, sqrtf(q.x) * sigm(ig) * x);
    };
    h = make_float2(one(h.x, x.x, ig.x, rg.x, g.decay[ch]), n > 1 ? one(h.y, x.y, ig.y, rg.y, g.decay[ch + 1]) : 0.f);
    g.state_out[at] = h.x;
    if (n > 1) g.state_out[at + 1] = h.y;
    if (g.z != nullptr) h = mul2(h, mul2(z, make_float2(sigm(z.x), sigm(z.y))));
    store_out((F *)g.y + at, 0u, h, vec, n);
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
    if (back) {
        for (const void *p : {a->gy, (const void *)a->gx, (const void *)a->ginput_gate, (const void *)a->gdecay_gate, (const void *)a->gz})
            look(p, (long long)a->T * a->D, a->D);
    } else {
        look(a->y, (long long)a->T * a->D, a->D);
    }
    return ok && (bytes < 16 || a->D % e == 0);
}

int block_tokens(const wkv_gated_recurrence_args_t *a, bool back) {
    if (back) return a->dtype == WKV_F32 ? Geo<float, true>::BT : Geo<__half, true>::BT;
    return a->dtype == WKV_F32 ? Geo<float, false>::BT : Geo<__half, false>::BT;
}

// Spans of a row and their length.  A full pass takes a CTA 40 ns a token where two share an SM, 27 where it is alone (4 x 4096 x 4096
// forward 165 us, 1 x 8192 x 5120 in one span 215), the first pass over spans about half of that.
struct Spans {
    int n, tokens;
};
Spans count_spans(const wkv_gated_recurrence_args_t *a, bool back) {
    const long long unit = block_tokens(a, back), chains = (long long)a->B * ((a->D + CH - 1) / CH), sms = device_sm_count();
    const long long blocks = (a->T + unit - 1) / unit;
    auto time = [&](long long ctas, long long tokens) {                  // CTAs of so many tokens, two at most on an SM
        const long long full = ctas / (2 * sms), rest = ctas - full * 2 * sms;
        return (double)tokens * (full * 40.0 + (rest == 0 ? 0.0 : rest <= sms ? 27.0 : 40.0));
    };
    Spans best = {1, (int)std::max(unit, blocks * unit)};
    double t_best = time(chains, a->T);
    for (long long n = 2; n <= MAX_SPANS && n * 2 <= blocks && (n - 1) * chains <= 8 * sms; n++) {
        const long long len = (blocks + n - 1) / n * unit, used = (a->T + len - 1) / len;
        if (used != n) continue;
        const double t = time(chains * n, len) + 0.5 * time(chains * (n - 1), len) + 4000.0 + 100.0 * n;
        if (t < t_best) { best = {(int)n, (int)len}; t_best = t; }
    }
    return best;
}
// (the search takes up to 25 us and a call asks several times: the last answers of a thread are remembered by their sizes)
Spans spans_for(const wkv_gated_recurrence_args_t *a, bool back) {
    struct Entry {
        int B, T, D, dtype, sms;
        Spans s;
    };
    static thread_local Entry last[2][16];
    const int sms = device_sm_count();
    Entry &e = last[back][((unsigned)a->B * 7u + (unsigned)a->T * 5u + (unsigned)a->D * 3u) >> 2 & 15u];
    if (e.s.n == 0 || e.B != a->B || e.T != a->T || e.D != a->D || e.dtype != a->dtype || e.sms != sms)
        e = {a->B, a->T, a->D, a->dtype, sms, count_spans(a, back)};
    return e.s;
}
size_t spans_bytes(const wkv_gated_recurrence_args_t *a, bool back) {
    const int n = spans_for(a, back).n;
    return n > 1 ? align256((size_t)a->B * n * a->D * sizeof(float2)) : 0;
}

bool strides_ok(const wkv_gated_recurrence_args_t *a) {
    for (long long t : {a->x_token, a->i_token, a->r_token, a->z != nullptr ? a->z_token : 0})
        if (a->T > 1 && (t < 0 || t > 1 << 26)) return false;
    return true;
}
bool sizes_ok(const wkv_gated_recurrence_args_t *a) {
    return a->B >= 0 && a->T >= 0 && a->D >= 0 && a->D <= (1 << 22) && a->T <= 2147483647 - 4096 && known_dtype(a->dtype) &&
           (long long)a->B * ((a->D + CH - 1) / CH) <= 2147483647 / MAX_SPANS && (long long)a->B * a->D <= 1ll << 34 && a->c > 0.f &&
           strides_ok(a);
}
long long kept_states(const wkv_gated_recurrence_args_t *a) {
    const int t = ckpt_tokens(elem_size(a->dtype));
    return ((long long)a->T + t - 1) / t;
}
RecArgs args_of(const wkv_gated_recurrence_args_t *a, bool back) {
    RecArgs g = {};
    const Spans sp = spans_for(a, back);
    g.T = a->T; g.D = a->D; g.slabs = (a->D + CH - 1) / CH; g.nspan = sp.n; g.span = sp.tokens;
    g.nkept = (int)kept_states(a);
    g.c = a->c;
    g.x = a->x; g.ig = a->input_gate; g.rg = a->decay_gate; g.z = a->z;
    g.x_batch = a->x_batch; g.x_token = a->x_token; g.ig_batch = a->i_batch; g.ig_token = a->i_token;
    g.rg_batch = a->r_batch; g.rg_token = a->r_token; g.z_batch = a->z_batch; g.z_token = a->z_token;
    g.decay = a->decay; g.state_in = a->state_in; g.y = a->y; g.state_out = a->state_out; g.ckpt = (float *)a->ckpt;
    g.gy = a->gy; g.gs_out = a->gstate_out; g.gx = a->gx; g.gig = a->ginput_gate; g.grg = a->gdecay_gate; g.gz = a->gz;
    g.gs_in = a->gstate_in;
    g.spans = (float2 *)a->workspace;
    g.part = (float *)((char *)a->workspace + (back ? spans_bytes(a, true) : 0));
    g.status = a->status; g.limit = t_limit; g.skip = t_skip;
    return g;
}
size_t ckpt_need(const wkv_gated_recurrence_args_t *a) { return (size_t)a->B * kept_states(a) * a->D * 4; }

template <class K>
int launch_rec(K kern, const RecArgs &g, long long ctas, int smem, unsigned char (&done)[64], cudaStream_t s) {
    if (!set_max_smem_once(kern, smem, done)) return WKV_ERR_LAUNCH;
    return launch_chained(kern, dim3((unsigned)ctas), dim3(256), smem, s, g);
}
template <typename F, bool Z, int MODE, bool BACK>
int launch_as(const RecArgs &g, int B, cudaStream_t s) {
    static unsigned char done[2][64];
    const long long chains = (long long)B * g.slabs;
    if (g.nspan > 1) {
        const int smem = NW * 4 * (BACK ? 2 + Z : 3) * Geo<F, BACK>::S * row_of(MODE) * (int)sizeof(F);
        const int rc = launch_rec(k_rec_spans<F, Z, MODE, BACK>, g, chains * (g.nspan - 1), smem, done[1], s);
        if (rc != WKV_OK) return rc;
    }
    if constexpr (BACK) return launch_rec(k_rec_bwd<F, Z, MODE>, g, chains * g.nspan, Geo<F, true>::ring(Z, MODE) + (int)sizeof(ExchangeBack) + Geo<F, true>::KEPT, done[0], s);
    else return launch_rec(k_rec_fwd<F, Z, MODE>, g, chains * g.nspan, Geo<F, false>::ring(Z, MODE) + (int)sizeof(Exchange), done[0], s);
}
// the tiles' maps; false: TMA cannot read or write these rows
template <typename F, bool BACK>
bool make_maps(const wkv_gated_recurrence_args_t *a, RecArgs &g) {
    using G = Geo<F, BACK>;
    const long long yt = a->D, yb = (long long)a->T * a->D;
    const int z = a->z != nullptr;
    struct { const void *p; long long batch, token; } in[5] = {{a->decay_gate, a->r_batch, a->r_token}, {a->input_gate, a->i_batch, a->i_token}, {a->x, a->x_batch, a->x_token}};
    in[3 + BACK] = {a->z, a->z_batch, a->z_token};
    if (BACK) in[3] = {a->gy, yb, yt};
    for (int i = 0; i < 3 + BACK + z; i++) {
        // (a dimension of one element may have any stride)
        const long long token = a->T > 1 ? in[i].token : yt, batch = a->B > 1 ? in[i].batch : token * a->T;
        if (in[i].p == nullptr || !make_tile_map(&g.in[i], in[i].p, sizeof(F), a->B, a->T, a->D, batch, token, CH, G::BT)) return false;
        const bool first = BACK ? i == 0 || i >= 3 : i < 3;               // what the pass over spans reads
        if (g.nspan > 1 && first && !make_tile_map(&g.in_spans[i], in[i].p, sizeof(F), a->B, a->T, a->D, batch, token, CH, G::S)) return false;
    }
    void *out[4] = {BACK ? a->gx : a->y, a->ginput_gate, a->gdecay_gate, a->gz};
    for (int i = 0; i < (BACK ? 3 + z : 1); i++)
        if (out[i] != nullptr && !make_tile_map(&g.out[i], out[i], sizeof(F), a->B, a->T, a->D, yb, yt, CH, G::S)) return false;
    return true;
}

template <bool BACK>
int launch_by(const wkv_gated_recurrence_args_t *a, RecArgs &g, cudaStream_t s) {
    return by_dtype(a->dtype, [&](auto f) {
        using F = decltype(f);
        g.pair = a->D % 2 == 0 && lies_in<F>(a, 2 * sizeof(F), BACK);
        const int mode = a->T > 0 && lies_in<F>(a, 16, BACK) && make_maps<F, BACK>(a, g) ? TILES : sizeof(F) == 4 || lies_in<F>(a, 4, BACK) ? WORDS : ANYWHERE;
        auto go = [&](auto zc) {
            constexpr bool Z = decltype(zc)::value;
            if (mode == TILES) return launch_as<F, Z, TILES, BACK>(g, a->B, s);
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

extern "C" size_t wkv_gated_recurrence_forward_workspace(const wkv_gated_recurrence_args_t *a) {
    return a != nullptr && sizes_ok(a) && a->T > 1 ? spans_bytes(a, false) : 0;
}

extern "C" int wkv_gated_recurrence_forward(const wkv_gated_recurrence_args_t *a, void *stream) {
    if (a == nullptr) return WKV_ERR_NULL;
    if (!known_dtype(a->dtype)) return WKV_ERR_DTYPE;
    if (!sizes_ok(a)) return WKV_ERR_SHAPE;
    if ((long long)a->B * a->D == 0) return WKV_OK;
    if (a->decay == nullptr || a->state_out == nullptr) return WKV_ERR_NULL;
    if (a->T > 0 && (a->x == nullptr || a->input_gate == nullptr || a->decay_gate == nullptr || a->y == nullptr)) return WKV_ERR_NULL;
    RecArgs g = args_of(a, false);
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
    if (a->T > 1 && a->state_out == a->state_in) return WKV_ERR_UNSUPPORTED;        // (spans of a row start from it at any time)
    if (a->ckpt != nullptr && a->ckpt_bytes < ckpt_need(a)) return WKV_ERR_WORKSPACE;
    const size_t need = wkv_gated_recurrence_forward_workspace(a);
    if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need)) return WKV_ERR_WORKSPACE;
    if (!aligned16(a->workspace)) return WKV_ERR_ALIGN;
    return launch_by<false>(a, g, s);
}

extern "C" size_t wkv_gated_recurrence_backward_workspace(const wkv_gated_recurrence_args_t *a) {
    if (a == nullptr || !sizes_ok(a)) return 0;
    return spans_bytes(a, true) + (a->gdecay != nullptr ? (size_t)a->B * spans_for(a, true).n * a->D * 4 : 0);
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
    const size_t need = wkv_gated_recurrence_backward_workspace(a);
    if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need)) return WKV_ERR_WORKSPACE;
    if (!aligned16(a->workspace)) return WKV_ERR_ALIGN;
    RecArgs g = args_of(a, true);
    if (a->gdecay == nullptr) g.part = nullptr;
    const int rc = launch_by<true>(a, g, s);
    if (rc != WKV_OK || a->gdecay == nullptr) return rc;
    return fold_params(g.part, a->B * g.nspan, a->D, out, s);
}

extern "C" int wkv_gated_recurrence_selftest_abort(const wkv_gated_recurrence_args_t *a, int backward_call, int skip_block, unsigned limit, void *stream) {
    if (skip_block < 0 || limit < 1 || limit > 100000) return WKV_ERR_SHAPE;
    t_skip = skip_block;
    t_limit = limit;
    const int rc = backward_call ? wkv_gated_recurrence_backward(a, stream) : wkv_gated_recurrence_forward(a, stream);
    t_skip = -1;
    t_limit = WAIT_LIMIT;
    return rc;
}
