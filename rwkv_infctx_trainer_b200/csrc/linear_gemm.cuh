// Matrix products D[m,n] = sum_k A[m,k] B[n,k] of 16-bit operands on the 5th generation tensor cores, with an epilogue: the tile
// kernel of linear.cu.
//
// Each operand lies with its contraction dimension contiguous (x and W forward) or with the other one contiguous (W for the
// gradient of x; the gradient of y and x for the gradient of W): no operand is ever transposed in memory, the instruction
// descriptor says how the tile lies.  TMA brings 64 contraction steps of a tile a stage, in the 128-byte swizzle; contraction-major
// tiles as one box of rows, the others as boxes of 64 columns x 64 steps.
//
// A pair of CTAs (CG = 2) computes 256 x 256 on both SMs' tensor cores (tcgen05 cta_group::2, M = 256, N = 256): each brings its own
// 128 rows of A and half of the rows of B, 32 KB a stage where a lone CTA would bring 48 for its 128 x 256.  What an SM can take in, about 60 bytes a cycle,
// is as near a bound as the products: at 256 x 256 both are met, the smaller tiles (256 x 128 of a pair, 128 x 128 and 128 x 64 of a lone CTA) wait for
// their operands.  Persistent: a CTA walks over its tiles; two accumulators in tensor memory, so that the
// epilogue of a tile runs under the products of the next.
//
// Measured: 16384 x 4096 -> 4096 346 us (1588 TFLOP/s; a library product without an epilogue 340), 8192 x 4096 -> 14336 590 (1631; 641); tensor pipe busy for 94 %
// of the cycles, 82 % in a pair's forward pass that leaves two fp32 pre-activations.  A launch's first loads and last epilogue take 4.5 to 6 us.
//
// Warps: 8 of the epilogue (quarter w % 4 of the accumulator's rows, half w / 4 of its columns), one that loads, one that issues.
// Epilogue: 32 columns from tensor memory (a thread has a row), turned through shared memory, then whole 16-byte pieces of
// rows are finished in fp32 -- bias, activation, product, residual -- and rounded once.
//
// Every wait is bounded: a warp that gives up sets the abort flag (of both CTAs of a pair, in the end) and the status word, loads in flight are
// waited for, tensor memory is freed, and the kernel returns.
#pragma once
#include <cuda.h>

#include "elem_io.cuh"
#include "sm100_primitives.cuh"

namespace wkv {
namespace linear {

enum { ACT_NONE = 0, ACT_SILU = 1, ACT_GELU = 2, ACT_RELU2 = 3, ACT_SIGMOID = 4, ACT_COUNT = 5 };

constexpr int EPI_WARPS = 8, THREADS = 32 * (EPI_WARPS + 2), KB = 64, ACC = 2;
enum { EPI_LINEAR = 0, EPI_GATED = 1, EPI_PLAIN = 2 };         // (PLAIN: the sums alone, of the gradients)

__device__ __forceinline__ float sigmoid_of(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }
// Phi(z), and g = e^(-z^2 / 2).  For t = |z| the tail is g R(t), R(t) = erfcx(t / sqrt 2) / 2, a smooth function that falls from 1/2 as 0.4 / t:
// w P(w) in w = 1 / (1 + 0.35 t), P of degree 8 fitted for the least largest relative error (with its rounded coefficients 3.7e-8 below t = 1, 5.7e-8 at 13).
// A small tail keeps digits, which 1 + erf does not: g's exponent is rounded, so that in all it is off by 4e-7 of itself below t = 1, 2e-6 at 6 and 8e-6
// at 13, 1/500 of half a step of bf16.  (Through erfcf the epilogue of 1999 x 2560 -> 8960 took 128 us of a
// product's 78.)
__device__ __forceinline__ float phi_of(float z, float &g) {
    const float t = fabsf(z), w = __fdividef(1.f, fmaf(0.35f, t, 1.f));
    float p = -0.029164928942918777f;
    p = fmaf(p, w, 0.1440657675266266f);
    p = fmaf(p, w, -0.25591233372688293f);
    p = fmaf(p, w, 0.1594051569700241f);
    p = fmaf(p, w, -0.023272467777132988f);
    p = fmaf(p, w, 0.10557854920625687f);
    p = fmaf(p, w, 0.11981452256441116f);
    p = fmaf(p, w, 0.1398644745349884f);
    p = fmaf(p, w, 0.13962124288082123f);
    g = exp2f(-0.7213475204444817f * t * t);
    const float q = g * (p * w);
    return z >= 0.f ? 1.f - q : q;
}

template <int R, int N>
__device__ __forceinline__ void act_values(int act, float (&z)[R][N]) {
    auto each = [&](auto f) {
#pragma unroll
        for (int k = 0; k < R; k++)
#pragma unroll
            for (int i = 0; i < N; i++) z[k][i] = f(z[k][i]);
    };
    switch (act) {
        case ACT_SILU: each([](float z) { return z * sigmoid_of(z); }); break;
        case ACT_GELU:
            each([](float z) {
                float g;
                return z * phi_of(z, g);
            });
            break;
        case ACT_RELU2:
            each([](float z) {
                const float p = z > 0.f ? z : (z == z ? 0.f : z);
                return p * p;
            });
            break;
        case ACT_SIGMOID: each([](float z) { return sigmoid_of(z); }); break;
        default: break;
    }
}

struct Epi {
    int act, vec;                     // vec: y, mul and residual are rows of whole 16-byte pieces
    const void *bias;                 // [N]
    int bias_dtype;
    const void *mul, *residual;       // [M,N]
    void *y[2];                       // [M,N] of each source of rows (the second: the gradient of a second matrix)
    long long y_row;                  // their row stride, and that of mul and residual
    float *z[2];                      // pre-activations (or NULL)
    long long z_row;
    float *part;                      // sums of parts of a contraction: [tile][part][row of the tile][column of the tile]
};

// Element i of the bias, 0 without one.  Plain loads: the compiler may move the 16-bit forms of __ldg, and did, out of a loop and in front of the
// check.
__device__ __forceinline__ float bias_at(const Epi &e, int i) {
    if (e.bias == nullptr) return 0.f;
    if (e.bias_dtype == WKV_F32) return Elem<float>::ld((const float *)e.bias + i);
    if (e.bias_dtype == WKV_BF16) return Elem<__nv_bfloat16>::ld((const __nv_bfloat16 *)e.bias + i);
    return Elem<__half>::ld((const __half *)e.bias + i);
}

struct GemmArgs {
    CUtensorMap a[2], b[2];
    int M, N;                         // of one source
    int m_tiles, n_tiles;             // m_tiles: of all sources
    int m_tiles0;                     // tiles of A's first source (rows of the second one after them); m_tiles where there is one
    int kb, kb0;                      // contraction blocks of 64, of all sources and of the first one
    int main, rest;                   // tiles that are computed whole, and those behind them whose contraction is cut
    int splits, kb_split;             // into so many parts of so many blocks: a wave of CTAs that the rest alone would not fill
    int group;                        // tiles of M that are walked together
    int *status;
    unsigned limit;                   // polls of a wait
    int skip;                         // self-test: the block of a CTA's first tile that is never loaded (-1)
    Epi e;
};

// ------------------------------------------------------------------------------------------ PTX of a pair of CTAs
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// address, in the cluster's window, of the same place in the shared memory of CTA `rank`
__device__ __forceinline__ uint32_t map_rank(const void *p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(sm100::smem_u32(p)), "r"(rank));
    return r;
}
// (what it orders are reads of tensor memory, which tcgen05's fence has ordered: with .release.cluster it waited for the outputs' stores, 0.15 of the
// epilogue's time)
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void store_remote(uint32_t at, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <int CG>
__device__ __forceinline__ void tma_2d(void *dst, const void *map, uint32_t bar, int c0, int c1) {
    if constexpr (CG == 2)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     ::"r"(sm100::smem_u32(dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     ::"r"(sm100::smem_u32(dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    if constexpr (CG == 2)
        asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
    else
        sm100::mma_ss(d, a, b, idesc, accumulate);
}
// arrive on the barrier (of both CTAs of a pair) when all products issued so far are done
template <int CG>
__device__ __forceinline__ void commit(uint64_t *bar) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(sm100::smem_u32(bar)), "h"((uint16_t)3) : "memory");
    else
        sm100::mma_commit(bar);
}
template <int CG>
__device__ __forceinline__ void tmem_get(uint32_t *result, uint32_t cols) {
    if constexpr (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm100::smem_u32(result)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        sm100::tmem_alloc(result, cols);
        sm100::tmem_relinquish();
    }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
    else sm100::tmem_dealloc(addr, cols);
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float *v) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
}

template <typename F>
__host__ __device__ constexpr uint32_t instruction(int M, int N, bool a_mn, bool b_mn) {
    constexpr uint32_t kind = std::is_same<F, __nv_bfloat16>::value ? 1u : 0u;      // bf16 or fp16, both operands alike
    return (1u << 4) | (kind << 7) | (kind << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}
// A swizzled tile: contraction-major rows of 128 bytes, 8 of them 1024 apart; else blocks of 64 columns x 64 steps, `LEAD` bytes apart.
constexpr int BLOCK_BYTES = 64 * 128;
template <bool MN>
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr) {
    uint64_t d = (uint64_t)((addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(MN ? BLOCK_BYTES >> 4 : 1) << 16;       // leading dimension: from one block of 64 columns to the next
    d |= (uint64_t)(1024 >> 4) << 32;                       // stride dimension: from 8 rows to the next 8
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// the start of 16 contraction steps within a stage's tile
template <bool MN> __device__ __forceinline__ uint32_t k16_offset(int k) { return MN ? k * 16 * 128 : k * 32; }

// ------------------------------------------------------------------------------------------ layout
template <int CG, int BN>
struct Tile {
    static constexpr int BM = 128 * CG, B_ROWS = BN / CG;                                    // B_ROWS: of one CTA
    static constexpr int A_BYTES = 128 * 128, B_BYTES = B_ROWS * 128, STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = (STAGE * 6 <= 196608) ? (196608 / STAGE > 8 ? 8 : 196608 / STAGE) : 5;
    static constexpr int TURN = EPI_WARPS * 4096;                                            // epilogue: 32 x 32 floats a warp
    static constexpr int BARS = STAGES * STAGE + TURN;
    static constexpr int SMEM = BARS + (2 * STAGES + 2 * ACC) * 8 + 16 + 1024;                // (16: four words; 1024: alignment of the stages)
    static constexpr uint32_t COLS = ACC * BN;
};

struct Item {
    int m, n, part, kb, kb_end;       // part: index of the sums that are left, -1 where the tile is finished
};
__device__ __forceinline__ void tile_at(const GemmArgs &g, int i, int &m, int &n) {
    const int per = g.group * g.n_tiles, grp = i / per, first = grp * g.group, rows = min(g.group, g.m_tiles - first);
    i -= grp * per;
    n = i / rows;
    m = first + i - n * rows;
}
__device__ __forceinline__ Item item_at(const GemmArgs &g, int i) {
    Item t;
    t.part = -1;
    t.kb = 0;
    t.kb_end = g.kb;
    if (i >= g.main) {
        const int j = i - g.main, split = j / g.rest, r = j - split * g.rest;
        i = g.main + r;
        if (g.splits > 1) {
            t.part = r * g.splits + split;
            t.kb = split * g.kb_split;
            t.kb_end = min(g.kb, t.kb + g.kb_split);
        }
    }
    tile_at(g, i, t.m, t.n);
    return t;
}

// R pieces of W columns each (accumulators f; EPI_GATED: u in `u`), `rows` apart from row `row` on -> their outputs.  What is read for them is
// asked for first; the activation is chosen once for all of them.  ok: whether a piece's row exists; n: columns of a piece that exist (W at least
// where VEC: one access of 16 bytes each).
template <typename F, int EPI, int R, int W, bool VEC>
struct Finish {
    Raw<F, VEC ? 8 : 2> mul[R], res[R];

    __device__ __forceinline__ void ask(const Epi &e, long long row, int rows, int col, int n, const bool (&ok)[R]) {
        if (EPI != EPI_LINEAR) return;
        auto get = [&](const void *p, Raw<F, VEC ? 8 : 2> (&to)[R]) {
#pragma unroll
            for (int k = 0; k < R; k++) {
                to[k].zero();
                const F *q = (const F *)p + (row + k * rows) * e.y_row + col;
                if (ok[k] && n > 0) to[k].load(q, VEC, n);
            }
        };
        if (e.mul != nullptr) get(e.mul, mul);
        if (e.residual != nullptr) get(e.residual, res);
    }
    __device__ __forceinline__ void put(void *p, long long at, const float (&f)[W], bool ok, int n) const {
        if constexpr (W == 8) {
            Raw<F, 8> r;
            r.put(f);
            if (ok && n > 0) r.store((F *)p + at, true, 8);
        } else {
            if (ok && n > 0) Elem<F>::st((F *)p + at, f[0]);
        }
    }
    __device__ __forceinline__ void keep(float *p, const float (&f)[W], bool ok, int n) const {
        if (!ok || n <= 0) return;
        if constexpr (W == 8) {
            *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4 *>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
        } else {
            *p = f[0];
        }
    }
    __device__ __forceinline__ void finish(const Epi &e, int src, long long row, int rows, int col, int n, const bool (&ok)[R], float (&f)[R][W],
                                           const float (&u)[R][W], const float (&bias)[W]) {
        if (EPI == EPI_LINEAR && e.bias != nullptr) {
#pragma unroll
            for (int k = 0; k < R; k++)
#pragma unroll
                for (int i = 0; i < W; i++) f[k][i] += bias[i];
        }
        if (EPI != EPI_PLAIN && e.z[0] != nullptr) {
#pragma unroll
            for (int k = 0; k < R; k++) {
                const long long at = (row + k * rows) * e.z_row + col;
                keep(e.z[0] + at, f[k], ok[k], n);
                if (EPI == EPI_GATED) keep(e.z[1] + at, u[k], ok[k], n);
            }
        }
        if (EPI != EPI_PLAIN) act_values(e.act, f);
        if (EPI == EPI_GATED) {
#pragma unroll
            for (int k = 0; k < R; k++)
#pragma unroll
                for (int i = 0; i < W; i++) f[k][i] *= u[k][i];
        }
        if (EPI == EPI_LINEAR && e.mul != nullptr) {
#pragma unroll
            for (int k = 0; k < R; k++) {
                float m[VEC ? 8 : 2];
                mul[k].get(m);
#pragma unroll
                for (int i = 0; i < W; i++) f[k][i] *= m[i];
            }
        }
        if (EPI == EPI_LINEAR && e.residual != nullptr) {
#pragma unroll
            for (int k = 0; k < R; k++) {
                float m[VEC ? 8 : 2];
                res[k].get(m);
#pragma unroll
                for (int i = 0; i < W; i++) f[k][i] += m[i];
            }
        }
        void *y = src ? e.y[1] : e.y[0];
#pragma unroll
        for (int k = 0; k < R; k++) put(y, (row + k * rows) * e.y_row + col, f[k], ok[k], n);
    }
};

template <typename F, int CG, int BN, bool A_MN, bool B_MN, int EPI>
__global__ void __launch_bounds__(THREADS, 1) k_gemm(const __grid_constant__ GemmArgs g) {
    using T = Tile<CG, BN>;
    constexpr int ST = T::STAGES;
    constexpr bool PAIR_B = EPI == EPI_GATED;              // the tile's columns: half of them of each of B's sources
    extern __shared__ unsigned char raw[];
    unsigned char *smem = raw + ((1024 - (sm100::smem_u32(raw) & 1023)) & 1023);
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + T::BARS), *empty = full + ST, *acc_full = empty + ST, *acc_empty = acc_full + ACC;
    uint32_t *tmem = reinterpret_cast<uint32_t *>(acc_empty + ACC);
    volatile int *abort = reinterpret_cast<int *>(tmem + 1), *asked = abort + 1;             // asked: stages each CTA of the pair has asked for (of the first CTA)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;
    const int first = blockIdx.x / CG, step = gridDim.x / CG, items = g.main + g.rest * g.splits;

    // (before pdl_wait: shared memory alone, and the tensor maps, which are arguments)
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) {
            sm100::mbar_init(full + i, 1);
            sm100::mbar_init(empty + i, 1);
        }
        for (int i = 0; i < ACC; i++) {
            sm100::mbar_init(acc_full + i, 1);
            sm100::mbar_init(acc_empty + i, CG * EPI_WARPS);
        }
        *abort = 0;
        asked[0] = asked[1] = 0;
        sm100::fence_mbar_init();
        sm100::prefetch_tmap(g.a);
        sm100::prefetch_tmap(g.b);
    }
    __syncwarp();
    pdl_wait();
    pdl_trigger();
    if (warp == EPI_WARPS + 1) tmem_get<CG>(tmem, T::COLS);
    sm100::tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync();
    sm100::tc_fence_after();
    const uint32_t acc0 = *reinterpret_cast<volatile uint32_t *>(tmem);
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        const bool ok = sm100::mbar_wait_or_abort(bar, parity, const_cast<const int *>(abort), g.limit);
        if (!ok) {
            *abort = 1;
            if (g.status != nullptr) atomicOr(g.status, WKV_LINEAR_TIMEOUT);
        }
        return ok;
    };

    if (warp == EPI_WARPS) {
        // ---- loads: this CTA's rows of A and of B; the pair's bytes are counted by the first CTA's barrier
        if (sm100::elect_one()) {
            int st = 0;
            uint32_t parity = 0;
            unsigned issued = 0;
            bool ok = true;
            for (int i = first; ok && i < items; i += step) {
                const Item t = item_at(g, i);
                const int src = t.m >= g.m_tiles0, m0 = (t.m - (src ? g.m_tiles0 : 0)) * T::BM + (int)rank * 128;
                // B: a CTA of a pair holds half of the tile's columns
                const int bsrc = PAIR_B && CG == 2 ? (int)rank : 0;
                const int n0 = PAIR_B ? t.n * (BN / 2) : t.n * BN + (int)rank * T::B_ROWS;
                for (int kb = t.kb; kb < t.kb_end; kb++) {
                    ok = wait(empty + st, parity ^ 1);
                    if (!ok) break;
                    issued++;
                    if (kb == g.skip && i == first && rank == 0) {
                        if (++st == ST) { st = 0; parity ^= 1; }
                        continue;
                    }
                    unsigned char *a = smem + st * T::STAGE, *b = a + T::A_BYTES;
                    const uint32_t bar = CG == 2 ? map_rank(full + st, 0) : sm100::smem_u32(full + st);
                    if (rank == 0) sm100::mbar_expect_tx(full + st, CG * T::STAGE);
                    const int ks = kb >= g.kb0, k0 = (kb - (ks ? g.kb0 : 0)) * KB;
                    const CUtensorMap *ma = g.a + (src | ks), *mb = g.b + (PAIR_B ? bsrc : ks);
                    if (A_MN) {
#pragma unroll
                        for (int j = 0; j < 2; j++) tma_2d<CG>(a + j * BLOCK_BYTES, ma, bar, m0 + 64 * j, k0);
                    } else {
                        tma_2d<CG>(a, ma, bar, k0, m0);
                    }
                    if (B_MN) {
#pragma unroll
                        for (int j = 0; j < T::B_ROWS / 64; j++) tma_2d<CG>(b + j * BLOCK_BYTES, mb, bar, n0 + 64 * j, k0);
                    } else if (PAIR_B && CG == 1) {
                        tma_2d<CG>(b, g.b, bar, k0, n0);
                        tma_2d<CG>(b + T::B_BYTES / 2, g.b + 1, bar, k0, n0);
                    } else {
                        tma_2d<CG>(b, mb, bar, k0, n0);
                    }
                    if (++st == ST) { st = 0; parity ^= 1; }
                }
            }
            // Before this CTA's shared memory may go: all stages read, and after an abort (below) at least written.
            for (int k = 0; k < ST && issued > 0; k++) {
                if (ok && (unsigned)k < issued) {
                    const unsigned last = issued - 1 - k;
                    ok = wait(empty + last % ST, (last / ST) & 1);
                }
            }
            if (!ok) {
                if (rank == 0) asked[0] = (int)issued;
                else store_remote(map_rank(const_cast<int *>(asked) + 1, 0), issued);
            }
        }
        __syncwarp();
    } else if (warp == EPI_WARPS + 1) {
        // ---- products: one thread of the pair
        if (rank == 0 && sm100::elect_one()) {
            constexpr uint32_t idesc = instruction<F>(T::BM, BN, A_MN, B_MN);
            int st = 0, buf = 0;
            uint32_t parity = 0, acc_parity = 0;
            bool ok = true;
            for (int i = first; ok && i < items; i += step) {
                const Item t = item_at(g, i);
                ok = wait(acc_empty + buf, acc_parity ^ 1);
                if (!ok) break;
                sm100::tc_fence_after();
                const uint32_t d = acc0 + buf * BN;
                for (int kb = t.kb; kb < t.kb_end; kb++) {
                    ok = wait(full + st, parity);
                    if (!ok) break;
                    sm100::tc_fence_after();
                    const uint32_t a = sm100::smem_u32(smem + st * T::STAGE), b = a + T::A_BYTES;
#pragma unroll
                    for (int k = 0; k < KB / 16; k++)
                        mma<CG>(d, tile_desc<A_MN>(a + k16_offset<A_MN>(k)), tile_desc<B_MN>(b + k16_offset<B_MN>(k)), idesc, kb > t.kb || k > 0);
                    commit<CG>(empty + st);
                    if (++st == ST) { st = 0; parity ^= 1; }
                }
                if (!ok) break;
                commit<CG>(acc_full + buf);
                if (++buf == ACC) { buf = 0; acc_parity ^= 1; }
            }
            if (!ok) {
                // (products in flight read this shared memory and write this tensor memory)
                commit<CG>(acc_full + buf);
                sm100::mbar_wait_landed(acc_full + buf, acc_parity, g.limit);
            }
        }
        __syncwarp();
    } else {
        // ---- epilogue
        const int quarter = warp & 3, half = warp >> 2;
        float *turn = reinterpret_cast<float *>(smem + ST * T::STAGE) + warp * 1024;
        const Epi &e = g.e;
        const uint32_t turn_w = sm100::smem_u32(turn) + lane * 128;
        int buf = 0;
        uint32_t acc_parity = 0;
        for (int i = first; i < items; i += step) {
            const Item t = item_at(g, i);
            const int src = t.m >= g.m_tiles0;
            const long long row0 = (long long)(t.m - (src ? g.m_tiles0 : 0)) * T::BM + rank * 128 + quarter * 32;
            if (!__all_sync(0xffffffffu, wait(acc_full + buf, acc_parity))) break;
            sm100::tc_fence_after();
            const uint32_t lanes = acc0 + buf * BN + ((uint32_t)(quarter * 32) << 16);
            // columns of the output that a tile has, a pass takes, and this warp's half of them
            constexpr int OUT = EPI == EPI_GATED ? BN / 2 : BN, PASS = EPI == EPI_GATED ? 16 : 32, PASSES = OUT / 2 / PASS;
#pragma unroll 1
            for (int p = 0; p < PASSES; p++) {
                const int c = half * (OUT / 2) + p * PASS, col0 = t.n * OUT + c;
                auto turn_in = [&] {
                    float v[32];
                    if (EPI == EPI_GATED) {
                        sm100::tmem_ld16(lanes + c, v);
                        sm100::tmem_ld16(lanes + OUT + c, v + 16);
                    } else {
                        tmem_ld32(lanes + c, v);
                    }
                    sm100::tmem_ld_wait();
                    if (p == PASSES - 1) {
                        // (the accumulator is in registers: the next tile's products may have it)
                        sm100::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            if (CG == 2) arrive_remote(map_rank(acc_empty + buf, 0));
                            else sm100::mbar_arrive(acc_empty + buf);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(turn_w + ((j ^ (lane & 7)) << 4)), "f"(v[4 * j]),
                                     "f"(v[4 * j + 1]), "f"(v[4 * j + 2]), "f"(v[4 * j + 3]) : "memory");
                    __syncwarp();
                };
                auto at = [&](int r, int chunk) { return *reinterpret_cast<const float4 *>(turn + r * 32 + ((chunk ^ (r & 7)) << 2)); };
                auto get8 = [&](int r, int chunk, float (&f)[8]) {
                    const float4 x = at(r, chunk), y = at(r, chunk + 1);
                    f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w; f[4] = y.x; f[5] = y.y; f[6] = y.z; f[7] = y.w;
                };
                if (t.part >= 0) {
                    turn_in();
                    // (of a pair: 16 columns of each half)
                    const int cc = (lane & 7) * 4, pc = EPI == EPI_GATED ? (cc < 16 ? c + cc : OUT + c + cc - 16) : c + cc;
                    float *out = e.part + ((size_t)t.part * T::BM + rank * 128 + quarter * 32) * BN + pc;
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const int r = k * 4 + (lane >> 3);
                        if (row0 + r < g.M) *reinterpret_cast<float4 *>(out + (size_t)r * BN) = at(r, lane & 7);
                    }
                } else if (e.vec) {
                    constexpr int LANES = PASS / 8, ROWS = 32 / LANES, R = 32 / ROWS;        // lanes of a row, rows of an access, accesses
                    const int cc = (lane % LANES) * 8, col = col0 + cc, n = g.N - col, r0 = lane / LANES;
                    Finish<F, EPI, R, 8, true> out;
                    bool ok[R];
#pragma unroll
                    for (int k = 0; k < R; k++) ok[k] = row0 + r0 + k * ROWS < g.M;
                    out.ask(e, row0 + r0, ROWS, col, n, ok);
                    float bias[8], f[R][8], u[R][8];
                    if (EPI == EPI_LINEAR && e.bias != nullptr) {
#pragma unroll
                        for (int k = 0; k < 8; k++) bias[k] = k < n ? bias_at(e, col + k) : 0.f;
                    }
                    turn_in();
#pragma unroll
                    for (int k = 0; k < R; k++) {
                        get8(r0 + k * ROWS, cc / 4, f[k]);
                        if (EPI == EPI_GATED) get8(r0 + k * ROWS, 4 + cc / 4, u[k]);
                    }
                    out.finish(e, src, row0 + r0, ROWS, col, n, ok, f, u, bias);
                } else {
                    constexpr int ROWS = 32 / PASS, R = 8;
                    const int cc = lane % PASS, col = col0 + cc, n = g.N - col;
                    float bias[1] = {EPI == EPI_LINEAR && n > 0 ? bias_at(e, col) : 0.f};
                    turn_in();
#pragma unroll 1
                    for (int r0 = lane / PASS; r0 < 32; r0 += R * ROWS) {
                        Finish<F, EPI, R, 1, false> out;
                        bool ok[R];
                        float f[R][1], u[R][1];
#pragma unroll
                        for (int k = 0; k < R; k++) ok[k] = row0 + r0 + k * ROWS < g.M;
                        out.ask(e, row0 + r0, ROWS, col, min(n, 1), ok);
#pragma unroll
                        for (int k = 0; k < R; k++) {
                            const int r = r0 + k * ROWS;
                            f[k][0] = turn[r * 32 + (((cc >> 2) ^ (r & 7)) << 2) + (cc & 3)];
                            if (EPI == EPI_GATED) u[k][0] = turn[r * 32 + (((4 + (cc >> 2)) ^ (r & 7)) << 2) + (cc & 3)];
                        }
                        out.finish(e, src, row0 + r0, ROWS, col, n, ok, f, u, bias);
                    }
                }
                __syncwarp();
            }
            if (++buf == ACC) { buf = 0; acc_parity ^= 1; }
        }
    }
    sm100::tc_fence_before();
    __syncthreads();
    if (CG == 2) {
        if (threadIdx.x == 0 && *abort) store_remote(map_rank(const_cast<int *>(abort), rank ^ 1), 1);
        __syncwarp();
        cluster_sync();
    }
    if (*abort) {
        // (the same for both CTAs of a pair.)  Copies on their way: of the last ST stages that were asked for.  The second CTA's bytes are counted here, and where it was
        // ahead nothing waits for them yet.
        if (threadIdx.x == 0 && rank == 0) {
            const int n0 = asked[0], n1 = CG == 2 ? asked[1] : 0, n = max(n0, n1);
            for (int k = n0; n0 > 0 && k < n1; k++) sm100::mbar_expect_tx(full + k % ST, T::STAGE);
            for (int k = max(0, n - ST); k < n; k++) sm100::mbar_wait_landed(full + k % ST, (k / ST) & 1, g.limit);
        }
        __syncwarp();
        if (CG == 2) cluster_sync();
    }
    sm100::tc_fence_after();
    if (warp == EPI_WARPS + 1) tmem_free<CG>(acc0, T::COLS);
}

// The sums of the parts of the tiles behind `main`, in order, then the epilogue: a thread has 8 columns of a row.
template <typename F, int EPI, int BM, int BN>
__global__ void __launch_bounds__(256) k_fold_parts(const __grid_constant__ GemmArgs g) {
    pdl_wait();
    pdl_trigger();
    constexpr int OUT = EPI == EPI_GATED ? BN / 2 : BN, PIECES = OUT / 8, CTAS = BM * PIECES / 256;      // CTAs of a tile
    const int r = blockIdx.x / CTAS, i = (blockIdx.x - r * CTAS) * 256 + threadIdx.x, y = i / PIECES, c = (i - y * PIECES) * 8;
    int tm, tn;
    tile_at(g, g.main + r, tm, tn);
    const int src = tm >= g.m_tiles0, col = tn * OUT + c, n = g.N - col;
    const long long row = (long long)(tm - (src ? g.m_tiles0 : 0)) * BM + y;
    if (row >= g.M || n <= 0) return;
    float f[1][8], u[1][8], bias[8];
#pragma unroll
    for (int k = 0; k < 8; k++) f[0][k] = u[0][k] = 0.f;
    const float *p = g.e.part + ((size_t)r * g.splits * BM + y) * BN + c;
    auto add = [&](const float *q, float (&to)[8]) {
        const float4 a = *reinterpret_cast<const float4 *>(q), b = *reinterpret_cast<const float4 *>(q + 4);
        to[0] += a.x; to[1] += a.y; to[2] += a.z; to[3] += a.w; to[4] += b.x; to[5] += b.y; to[6] += b.z; to[7] += b.w;
    };
#pragma unroll 4
    for (int s = 0; s < g.splits; s++) {
        add(p + (size_t)s * BM * BN, f[0]);
        if (EPI == EPI_GATED) add(p + (size_t)s * BM * BN + OUT, u[0]);
    }
    const bool ok[1] = {true};
    if (g.e.vec) {
        Finish<F, EPI, 1, 8, true> out;
        out.ask(g.e, row, 1, col, n, ok);
#pragma unroll
        for (int k = 0; k < 8; k++) bias[k] = EPI == EPI_LINEAR ? bias_at(g.e, col + k) : 0.f;
        out.finish(g.e, src, row, 1, col, n, ok, f, u, bias);
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (k >= n) break;
            Finish<F, EPI, 1, 1, false> out;
            float v[1][1] = {{f[0][k]}};
            const float w[1][1] = {{u[0][k]}}, b[1] = {EPI == EPI_LINEAR ? bias_at(g.e, col + k) : 0.f};
            out.ask(g.e, row, 1, col + k, 1, ok);
            out.finish(g.e, src, row, 1, col + k, 1, ok, v, w, b);
        }
    }
}

}  // namespace linear
}  // namespace wkv
