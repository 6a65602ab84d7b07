// Matrix products with their epilogue, forward and backward:
//
//   linear_act    y = act(z) mul + residual,  z = x W^T + bias
//       backward  gz = gy mul act'(z),  gx = gz W,  gW = gz^T x,  gbias = sum gz,  gmul = gy act(z),  gresidual = gy
//   gated_linear  y = act(g) u,  g = x Wg^T,  u = x Wu^T
//       backward  gu = gy act(g),  gg = gy u act'(g),  gx = gg Wg + gu Wu,  gWg = gg^T x,  gWu = gu^T x
//
// The products run on the tile kernel of linear_gemm.cuh.  The pair's forward pass is one product whose tile of 256 columns is half
// of each matrix (a CTA of the pair brings the rows of one), so that g and u of an element end up in one thread; its gradient of x
// is one product over both contractions, and that of the matrices one over the rows of both.  Few rows (decoded tokens) are bound
// by reading the matrix: k_few_rows streams it through registers once.
//
// What the forward pass keeps: the pre-activations, in fp32.  (In the activations' type the gradients of the matrices were 0.0031 off
// instead of 0.0023, the 2-norm of 8192 x 4096 -> a pair of 14336, and that of the bias 3e-4; the pass over them takes 240 us instead of 197.)
#include <algorithm>

#include "linear_gemm.cuh"
#include "tma_host.cuh"
#include "wkv_internal.h"

namespace wkv {
namespace linear {
namespace {

constexpr unsigned WAIT_LIMIT = 4000000u;
// (what a self-test changes in the calls of its thread)
thread_local int t_skip = -1;
thread_local unsigned t_limit = WAIT_LIMIT;

inline long long up8(long long n) { return (n + 7) & ~7ll; }

// 8 elements from any address (the first n of them): in words, which lie in the allocation of the elements that are in them
template <typename F>
__device__ __forceinline__ void load_any(Raw<F, 8> &r, const F *p, int n) {
    if (n < 8) {
        r.load(p, false, n);
        return;
    }
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const uint32_t *q = reinterpret_cast<const uint32_t *>(at & ~(uintptr_t)3);
    uint32_t w[5];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = q[i];
    const bool odd = at & 2;
    w[4] = odd ? q[4] : 0u;
#pragma unroll
    for (int i = 0; i < 4; i++) r.w[i] = odd ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
}
template <bool VEC, typename F>
__device__ __forceinline__ void load_piece(Raw<F, 8> &r, const F *p, int n) {
    if (VEC) r.load(p, true, 8);
    else load_any(r, p, n);
}

// ------------------------------------------------------------------------------------------ few rows
// A CTA has 16 rows of the matrix (of a pair: 8 of each), its 4 or 8 warps runs of 256 contraction steps (for 32 rows of x 128) in turn; the warps' sums meet
// in shared memory in a fixed order.  mma.sync with the matrix as the 16-row operand and the rows of x as the 8 columns: the
// contraction steps may be numbered in any order that both operands share, so that a lane's 16-byte piece (8 steps of one row) is
// its part of two instructions as it is, without a turn through shared memory.  (The tensor core's rate does not matter here.)
template <typename F>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<F, __nv_bfloat16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}


struct FewArgs {
    int M, K, N;                       // M: rows of x
    const void *x, *w[2];
    long long x_row, w_row[2];
    Epi e;
};

// VEC: every row of x and of the matrices is made of whole 16-byte pieces
template <typename F, int TOKENS, bool PAIR, bool VEC, int FEW_WARPS>
__global__ void __launch_bounds__(32 * FEW_WARPS) k_few_rows(const FewArgs g) {
    pdl_wait();
    pdl_trigger();
    constexpr int NT = TOKENS / 8, OUT = PAIR ? 8 : 16, UNROLL = TOKENS == 32 ? 2 : 4;
    __shared__ float part[FEW_WARPS][16][TOKENS + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, q = lane >> 2, c = lane & 3;
    const int row0 = blockIdx.x * OUT;
    // this lane's two rows of the matrix: q and q + 8 of the tile (of a pair: row q of each)
    const int r0 = row0 + q, r1 = PAIR ? row0 + q : row0 + q + 8;
    const F *w0 = (const F *)g.w[0] + (size_t)min(r0, g.N - 1) * g.w_row[0];
    const F *w1 = PAIR ? (const F *)g.w[1] + (size_t)min(r1, g.N - 1) * g.w_row[1] : (const F *)g.w[0] + (size_t)min(r1, g.N - 1) * g.w_row[0];
    const F *x[NT];
    bool live[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        live[j] = 8 * j + q < g.M;
        x[j] = (const F *)g.x + (size_t)(live[j] ? 8 * j + q : 0) * g.x_row;
    }
    float d[NT][4];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) d[j][i] = 0.f;
    auto run = [&](int k0, auto all) {
        constexpr bool whole = decltype(all)::value;
        Raw<F, 8> a[UNROLL][2][2], b[UNROLL][NT][2];
#pragma unroll
        for (int s = 0; s < UNROLL; s++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int k = k0 + s * 64 + h * 32 + c * 8, n = whole ? 8 : min(8, g.K - k);
                if (whole || n > 0) {
                    load_piece<VEC>(a[s][0][h], w0 + k, n);
                    load_piece<VEC>(a[s][1][h], w1 + k, n);
                } else {
                    a[s][0][h].zero();
                    a[s][1][h].zero();
                }
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    if (live[j] && (whole || n > 0)) load_piece<VEC>(b[s][j][h], x[j] + k, n);
                    else b[s][j][h].zero();
                }
            }
        }
#pragma unroll
        for (int s = 0; s < UNROLL; s++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    mma16<F>(d[j], a[s][0][h].w[0], a[s][1][h].w[0], a[s][0][h].w[1], a[s][1][h].w[1], b[s][j][h].w[0], b[s][j][h].w[1]);
                    mma16<F>(d[j], a[s][0][h].w[2], a[s][1][h].w[2], a[s][0][h].w[3], a[s][1][h].w[3], b[s][j][h].w[2], b[s][j][h].w[3]);
                }
    };
    int k0 = warp * 64 * UNROLL;
    for (; k0 + 64 * UNROLL <= g.K; k0 += UNROLL * 64 * FEW_WARPS) run(k0, std::true_type{});
    if (k0 < g.K) run(k0, std::false_type{});
#pragma unroll
    for (int j = 0; j < NT; j++) {
        part[warp][q][8 * j + 2 * c] = d[j][0];
        part[warp][q][8 * j + 2 * c + 1] = d[j][1];
        part[warp][q + 8][8 * j + 2 * c] = d[j][2];
        part[warp][q + 8][8 * j + 2 * c + 1] = d[j][3];
    }
    __syncthreads();
    // neighbouring threads take neighbouring columns of y
    for (int i = threadIdx.x; i < OUT * TOKENS; i += 32 * FEW_WARPS) {
        const int o = i % OUT, t = i / OUT, col = row0 + o;
        if (t < g.M && col < g.N) {
            float f = 0.f, u = 0.f;
#pragma unroll
            for (int w = 0; w < FEW_WARPS; w++) {
                f += part[w][o][t];
                if (PAIR) u += part[w][o + 8][t];
            }
            Finish<F, PAIR ? EPI_GATED : EPI_LINEAR, 1, 1, false> out;
            const bool ok[1] = {true};
            float v[1][1] = {{f}};
            const float w[1][1] = {{u}}, bias[1] = {PAIR ? 0.f : bias_at(g.e, col)};
            out.ask(g.e, t, 1, col, 1, ok);
            out.finish(g.e, 0, t, 1, col, 1, ok, v, w, bias);
        }
    }
}

// ------------------------------------------------------------------------------------------ gradient of the pre-activation
struct GradArgs {
    long long rows;
    int N, act, rows_per;
    const void *gy, *mul;
    const float *z[2];
    long long z_row;
    void *gz[2], *gmul;
    long long gz_row;
    float *part;                        // [gridDim.y, N] sums of gz over a CTA's rows
};

// act(z) and its derivative, of N elements: the activation is chosen once
template <int N>
__device__ __forceinline__ void act_both(int act, const float (&z)[N], float (&v)[N], float (&d)[N]) {
    auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < N; i++) f(z[i], v[i], d[i]);
    };
    // sigmoid(z) and sigmoid(-z) from one exponential: both keep their digits
    auto sigmoids = [](float z, float &s, float &n) {
        const float e = __expf(-fabsf(z)), r = __fdividef(1.f, 1.f + e), q = e * r;
        s = z >= 0.f ? r : q;
        n = z >= 0.f ? q : r;
    };
    switch (act) {
        case ACT_SILU:
            each([&](float z, float &v, float &d) {
                float s, n;
                sigmoids(z, s, n);
                v = z * s;
                d = s * fmaf(z, n, 1.f);
            });
            break;
        case ACT_SIGMOID:
            each([&](float z, float &v, float &d) {
                float n;
                sigmoids(z, v, n);
                d = v * n;
            });
            break;
        case ACT_GELU:
            each([&](float z, float &v, float &d) {
                float g;
                const float phi = phi_of(z, g);
                v = z * phi;
                d = fmaf(z, 0.3989422804014327f * g, phi);
            });
            break;
        case ACT_RELU2:
            each([&](float z, float &v, float &d) {
                const float p = z > 0.f ? z : (z == z ? 0.f : z);
                v = p * p;
                d = 2.f * p;
            });
            break;
        default:
            each([&](float z, float &v, float &d) {
                v = z;
                d = 1.f;
            });
    }
}

// A warp walks down rows of 256 columns, 8 a lane.  Bound by HBM: 8192 x 14336 of a pair 240 us (1.64 GB), 16384 x 4096 for the bias alone 41 (3.3
// TB/s of one tensor), with gelu 92; two rows at a time and half the warps an SM took 235, 51 and 106.  VEC: gy, mul and gmul are rows of whole pieces (z and
// gz always are).
template <typename F, bool PAIR, bool VEC>
__global__ void __launch_bounds__(256, 4) k_grad_act(const GradArgs g) {
    pdl_wait();
    pdl_trigger();
    __shared__ float red[8][256];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 256 + lane * 8, n = g.N - col;
    const bool whole = VEC || n >= 8;
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const long long r0 = (long long)blockIdx.y * g.rows_per, r1 = min(g.rows, r0 + g.rows_per);
    if (n > 0) {
#pragma unroll 1
        for (long long row = r0 + warp; row < r1; row += 8) {
            Raw<F, 8> ry, rm;
            Raw<float, 8> rz, ru;
            rz.zero();
            load_piece<VEC>(ry, (const F *)g.gy + row * g.N + col, n);
            if (g.z[0] != nullptr) rz.load(g.z[0] + row * g.z_row + col, whole, n);
            if (PAIR) ru.load(g.z[1] + row * g.z_row + col, whole, n);
            else if (g.mul != nullptr) load_piece<VEC>(rm, (const F *)g.mul + row * g.N + col, n);
            float gy[8], z[8], m[8], v[8], d[8];
            ry.get(gy);
            rz.get(z);
            act_both(g.act, z, v, d);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                v[i] *= gy[i];
                d[i] *= gy[i];
            }
            if (PAIR || g.mul != nullptr) {
                if (PAIR) ru.get(m);
                else rm.get(m);
#pragma unroll
                for (int i = 0; i < 8; i++) d[i] *= m[i];
            }
#pragma unroll
            for (int i = 0; i < 8; i++) sum[i] += d[i];
            if (g.gz[0] != nullptr) {
                ry.put(d);
                ry.store((F *)g.gz[0] + row * g.gz_row + col, whole, n);
            }
            if (PAIR) {
                ry.put(v);
                ry.store((F *)g.gz[1] + row * g.gz_row + col, whole, n);
            } else if (g.gmul != nullptr) {
                ry.put(v);
                ry.store((F *)g.gmul + row * g.N + col, VEC, n);
            }
        }
    }
    if (g.part == nullptr) return;
#pragma unroll
    for (int i = 0; i < 8; i++) red[warp][lane * 8 + i] = sum[i];
    __syncthreads();
    const int mine = blockIdx.x * 256 + threadIdx.x;
    if (mine < g.N) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 8; w++) s += red[w][threadIdx.x];
        g.part[(size_t)blockIdx.y * g.N + mine] = s;
    }
}

// rows that do not lie in whole 16-byte pieces -> rows that do; up to three matrices (blockIdx.y)
struct RepackArgs {
    struct One {
        const void *from;
        void *to;
        long long rows, cols, from_row, to_row;
    } m[3];
};
template <typename F>
__global__ void __launch_bounds__(256) k_repack(const RepackArgs g) {
    pdl_wait();
    pdl_trigger();
    const RepackArgs::One &m = g.m[blockIdx.y];
    const long long pieces = (m.cols + 7) / 8, total = m.rows * pieces;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long row = i / pieces, col = (i - row * pieces) * 8;
        Raw<F, 8> r;
        load_any(r, (const F *)m.from + row * m.from_row + col, (int)min(8ll, m.cols - col));
        r.store((F *)m.to + row * m.to_row + col, true, 8);
    }
}

// ------------------------------------------------------------------------------------------ host side
struct Matrix {
    const void *p;
    long long rows, cols, pitch;
};
inline bool tma_ready(const void *p, long long pitch) { return aligned16(p) && pitch % 8 == 0 && pitch < (1ll << 38); }

// Scratch, handed out in order; with a NULL base only counted.
struct Scratch {
    char *base;
    size_t used = 0;
    void *take(size_t bytes) {
        const size_t at = used;
        used += align256(bytes);
        return base ? base + at : nullptr;
    }
};

// How a product is cut: the tile, and the tiles behind the last full wave whose contraction is cut (Item in linear_gemm.cuh).
struct Cut {
    int cg, bn, m_tiles0, m_tiles, n_tiles, main, rest, splits, kb_split;
    size_t part_bytes() const { return splits > 1 ? (size_t)rest * splits * (128 * cg) * bn * 4 : 0; }
};
// The cut that takes least by this estimate, in us, fitted to one B200 (`first`: a launch with its first and its last tile's latency; `block`: 64
// contraction steps of a tile on every SM).  256 x 256 of two CTAs runs at the tensor cores' rate (4.2 million multiply-adds of a pair in 0.365 us); the other tiles are bound by
// their operands' way into an SM, about 60 bytes a cycle: 24 KB a block for 256 x 128 of two and 128 x 64 of one, 32 KB for 128 x 128 of one.  Cut
// contractions cost a launch and their sums' way through L2.  (2048 x 2560 -> 2560, 80 tiles on 74 pairs: 28 us with the last 6 cut in four, 31 without;
// 1500 x 8192 -> 1000, 24 tiles: 25 cut in three, 44 without.)
Cut find_cut(long long m, long long n, int sources, int kb, bool pair) {
    struct { int cg, bn; double first, block; } tiles[4] = {{2, 256, 6.2, 0.365}, {2, 128, 5.7, 0.222}, {1, 128, 4.7, 0.272}, {1, 64, 4.5, 0.228}};
    const int sms = device_sm_count();
    Cut best = {};
    double t_best = 1e30;
    for (const auto &t : tiles) {
        const long long bm = 128 * t.cg, out = pair ? t.bn / 2 : t.bn, m0 = (m + bm - 1) / bm, nt = (n + out - 1) / out, all = sources * m0 * nt;
        if (all > 1 << 29) continue;
        const int places = sms / t.cg;
        const long long waves = all / places, rest = all - waves * places;
        for (int s = 1; s <= 16 && s <= std::max(1, kb / 2); s++) {
            if (s > 1 && (rest == 0 || rest * (s - 1) >= places)) break;
            const int len = (kb + s - 1) / s, used = (kb + len - 1) / len;
            if (used != s) continue;
            double us = t.first + waves * kb * t.block + (rest ? (double)((rest * s + places - 1) / places) * len * t.block : 0.0);
            if (s > 1) us += 2.0 + 0.4 * s + (double)rest * s * bm * t.bn * 8 / 3e7;
            if (us < t_best) {
                t_best = us;
                best = {t.cg, t.bn, (int)m0, (int)(sources * m0), (int)nt, (int)(all - rest), (int)rest, s, len};
            }
        }
    }
    return best;
}

// (a call asks three times: the last answers of a thread are remembered by their sizes)
Cut cut_for(long long m, long long n, int sources, int kb, bool pair) {
    struct Entry {
        long long m, n;
        int sources, kb, pair, sms;
        Cut cut;
    };
    static thread_local Entry last[64];
    const int sms = device_sm_count();
    Entry &e = last[((unsigned long long)m * 31u + (unsigned long long)n * 7u + (unsigned)kb * 3u + sources) >> 2 & 63u];
    if (e.sms != sms || e.m != m || e.n != n || e.sources != sources || e.kb != kb || e.pair != (int)pair) e = {m, n, sources, kb, pair, sms, find_cut(m, n, sources, kb, pair)};
    return e.cut;
}

template <typename F, int CG, int BN, bool A_MN, bool B_MN, int EPI>
int launch_gemm(const GemmArgs &g, cudaStream_t s) {
    using T = Tile<CG, BN>;
    static unsigned char done[64];
    const auto kern = k_gemm<F, CG, BN, A_MN, B_MN, EPI>;
    if (!set_max_smem_once(kern, T::SMEM, done)) return WKV_ERR_LAUNCH;
    const long long items = g.main + (long long)g.rest * g.splits;
    const int places = device_sm_count() / CG, grid = (int)std::min<long long>(items, places) * CG;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = T::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CG; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CG > 1 ? 2 : 1;
    launch_count.fetch_add(1, std::memory_order_relaxed);
    if (cudaLaunchKernelEx(&cfg, kern, g) != cudaSuccess) return WKV_ERR_LAUNCH;
    if (g.splits == 1) return WKV_OK;
    constexpr int CTAS = T::BM * (EPI == EPI_GATED ? BN / 2 : BN) / 8 / 256;
    return launch_chained(k_fold_parts<F, EPI, T::BM, BN>, dim3((unsigned)(g.rest * CTAS)), dim3(256), 0, s, g);
}

// D = A B^T.  a, b: one or two sources.  How two are taken: with one B the rows of D are those of both (A's second source below the
// first), else the contraction runs over both; a pair's forward pass has one A and two B.
template <typename F, bool A_MN, bool B_MN, int EPI>
int product(const Matrix (&a)[2], const Matrix (&b)[2], int a_sources, int b_sources, long long m, long long n, long long k, const Cut &cut, const Epi &e,
            void *part, int *status, cudaStream_t s) {
    constexpr bool PAIR = EPI == EPI_GATED;
    if (cut.cg == 0) return WKV_ERR_SHAPE;
    GemmArgs g = {};
    g.M = (int)m; g.N = (int)n;
    g.m_tiles0 = cut.m_tiles0; g.m_tiles = cut.m_tiles; g.n_tiles = cut.n_tiles;
    g.kb0 = (int)((k + KB - 1) / KB);
    g.kb = g.kb0 * (a_sources == 2 && b_sources == 2 ? 2 : 1);
    g.main = cut.main; g.rest = cut.rest; g.splits = cut.splits; g.kb_split = cut.kb_split;
    g.group = 8;
    g.status = status; g.limit = t_limit; g.skip = t_skip;
    g.e = e;
    g.e.part = (float *)part;
    const int b_box = PAIR ? cut.bn / 2 : cut.bn / cut.cg;
    for (int i = 0; i < a_sources; i++)
        if (!make_matrix_map(&g.a[i], a[i].p, a[i].rows, a[i].cols, a[i].pitch, A_MN ? 64 : 128)) return WKV_ERR_LAUNCH;
    for (int i = 0; i < b_sources; i++)
        if (!make_matrix_map(&g.b[i], b[i].p, b[i].rows, b[i].cols, b[i].pitch, B_MN ? 64 : b_box)) return WKV_ERR_LAUNCH;
    if (cut.cg == 2) return cut.bn == 256 ? launch_gemm<F, 2, 256, A_MN, B_MN, EPI>(g, s) : launch_gemm<F, 2, 128, A_MN, B_MN, EPI>(g, s);
    return cut.bn == 128 ? launch_gemm<F, 1, 128, A_MN, B_MN, EPI>(g, s) : launch_gemm<F, 1, 64, A_MN, B_MN, EPI>(g, s);
}

int check_args(const wkv_linear_args_t *a) {
    if (a == nullptr) return WKV_ERR_NULL;
    if (a->dtype != WKV_BF16 && a->dtype != WKV_F16) return known_dtype(a->dtype) ? WKV_ERR_UNSUPPORTED : WKV_ERR_DTYPE;
    if (a->bias != nullptr && !known_dtype(a->bias_dtype)) return WKV_ERR_DTYPE;
    const long long most = (1ll << 31) - 4096;         // (numbers of rows and columns, and what loops add to them, are 32-bit)
    if (a->rows < 0 || a->K < 1 || a->N < 1 || a->rows > most || a->K > most || a->N > most) return WKV_ERR_SHAPE;
    if ((a->x != nullptr && a->rows > 1 && a->x_row < a->K) || (a->w0 != nullptr && a->N > 1 && a->w0_row < a->K) ||
        (a->pair && a->w1 != nullptr && a->N > 1 && a->w1_row < a->K))
        return WKV_ERR_SHAPE;
    if (a->act < 0 || a->act >= ACT_COUNT || a->pair < 0 || a->pair > 1) return WKV_ERR_SHAPE;
    if (a->pair && (a->bias != nullptr || a->mul != nullptr || a->residual != nullptr || a->gbias != nullptr || a->gmul != nullptr)) return WKV_ERR_UNSUPPORTED;
    return WKV_OK;
}
bool keeps(const wkv_linear_args_t *a) { return a->pair || a->act != ACT_NONE || a->mul != nullptr; }
size_t saved_one(const wkv_linear_args_t *a) { return align256((size_t)a->rows * up8(a->N) * 4); }
// Up to 16 rows, and up to 32 of matrices of up to 2^24 elements, where starting and ending the tile kernel counts (us, streamed and in tiles: 32 rows of
// 2560 -> 2560 8.1 and 12, of 4096 -> 4096 12 and 13.5, of 4096 -> 14336 39 and 27: the rows of x come from L1 for every 16 of the matrix).
bool few(const wkv_linear_args_t *a) { return a->rows <= 16 || (a->rows <= 32 && (1 + a->pair) * a->N <= (1 << 24) / a->K); }
Matrix x_of(const wkv_linear_args_t *a) { return {a->x, a->rows, a->K, a->x_row}; }
Matrix w_of(const wkv_linear_args_t *a, int i) { return {i ? a->w1 : a->w0, a->N, a->K, i ? a->w1_row : a->w0_row}; }

// The matrices where TMA can read them, else copies in the scratch.
template <typename F>
int ready(std::initializer_list<Matrix *> ms, Scratch &ws, cudaStream_t s) {
    RepackArgs r = {};
    int n = 0;
    long long most = 0;
    for (Matrix *m : ms) {
        if (tma_ready(m->p, m->pitch)) continue;
        const long long pitch = up8(m->cols);
        void *to = ws.take((size_t)m->rows * pitch * 2);
        r.m[n++] = {m->p, to, m->rows, m->cols, m->pitch, pitch};
        most = std::max(most, m->rows * (pitch / 8));
        if (ws.base == nullptr) continue;
        m->p = to;
        m->pitch = pitch;
    }
    if (n == 0 || ws.base == nullptr) return WKV_OK;
    return launch_chained(k_repack<F>, dim3((unsigned)std::min<long long>((most + 255) / 256, 148 * 16), (unsigned)n), dim3(256), 0, s, r);
}

Epi epilogue_of(const wkv_linear_args_t *a) {
    Epi e = {};
    e.act = a->act;
    e.vec = a->N % 8 == 0 && all_aligned({a->y, a->mul, a->residual});
    e.bias = a->bias; e.bias_dtype = a->bias_dtype; e.mul = a->mul; e.residual = a->residual;
    e.y[0] = a->y; e.y_row = a->N;
    if (a->saved != nullptr && keeps(a)) {
        e.z[0] = (float *)a->saved;
        e.z[1] = a->pair ? (float *)((char *)a->saved + saved_one(a)) : nullptr;
        e.z_row = up8(a->N);
    }
    return e;
}

template <typename F>
int forward(const wkv_linear_args_t *a, Scratch ws, size_t *need, cudaStream_t s) {
    Matrix x = x_of(a), w[2] = {w_of(a, 0), w_of(a, a->pair)};
    Epi e = epilogue_of(a);
    const bool count = need != nullptr;
    if (few(a)) {
        if (count) { *need = 0; return WKV_OK; }
        FewArgs g = {};
        g.M = (int)a->rows; g.K = (int)a->K; g.N = (int)a->N;
        g.x = x.p; g.x_row = x.pitch;
        for (int i = 0; i < 2; i++) { g.w[i] = w[i].p; g.w_row[i] = w[i].pitch; }
        g.e = e;
        const bool vec = a->K % 8 == 0 && tma_ready(x.p, x.pitch) && tma_ready(w[0].p, w[0].pitch) && tma_ready(w[1].p, w[1].pitch);
        const long long ctas = (a->N + (a->pair ? 7 : 15)) / (a->pair ? 8 : 16);
        const auto go = [&](auto pair, auto tokens) {
            constexpr bool PAIR = decltype(pair)::value;
            constexpr int TOKENS = decltype(tokens)::value;
            auto with = [&](auto kern, int warps) { return launch_chained(kern, dim3((unsigned)ctas), dim3(32 * warps), 0, s, g); };
            // (8 warps have more of the matrix on its way where CTAs are few: 8 rows of 4096 -> 4096 8.0 us, with 4 warps 10.3; 4 start and end
            // sooner where they are many: 1 row of 2560 -> a pair of 8960 17.1 us, with 8 warps 20.4.  The sums' order depends on it: not on alignment.)
            if (ctas <= 4 * device_sm_count()) return vec ? with(k_few_rows<F, TOKENS, PAIR, true, 8>, 8) : with(k_few_rows<F, TOKENS, PAIR, false, 8>, 8);
            return vec ? with(k_few_rows<F, TOKENS, PAIR, true, 4>, 4) : with(k_few_rows<F, TOKENS, PAIR, false, 4>, 4);
        };
        using N8 = std::integral_constant<int, 8>;
        using N16 = std::integral_constant<int, 16>;
        using N32 = std::integral_constant<int, 32>;
        if (a->rows <= 8) return a->pair ? go(std::true_type{}, N8{}) : go(std::false_type{}, N8{});
        if (a->rows > 16) return a->pair ? go(std::true_type{}, N32{}) : go(std::false_type{}, N32{});
        return a->pair ? go(std::true_type{}, N16{}) : go(std::false_type{}, N16{});
    }
    const int rc = a->pair ? ready<F>({&x, &w[0], &w[1]}, ws, s) : ready<F>({&x, &w[0]}, ws, s);
    if (rc != WKV_OK) return rc;
    const Cut cut = cut_for(a->rows, a->N, 1, (int)((a->K + KB - 1) / KB), a->pair);
    if (count) {
        *need = ws.used + align256(cut.part_bytes());
        return WKV_OK;
    }
    const Matrix xs[2] = {x, x};
    void *part = ws.take(cut.part_bytes());
    if (a->pair) return product<F, false, false, EPI_GATED>(xs, w, 1, 2, a->rows, a->N, a->K, cut, e, part, a->status, s);
    return product<F, false, false, EPI_LINEAR>(xs, w, 1, 1, a->rows, a->N, a->K, cut, e, part, a->status, s);
}

template <typename F>
int backward(const wkv_linear_args_t *a, Scratch ws, size_t *need, cudaStream_t s) {
    const bool count = need != nullptr;
    const int sources = 1 + a->pair, kb_n = (int)((a->N + KB - 1) / KB) * sources, kb_r = (int)((a->rows + KB - 1) / KB);
    const bool products = a->gx != nullptr || a->gw0 != nullptr || a->gw1 != nullptr;
    // gz: gy itself where nothing stands between them
    const bool act = keeps(a), own_gz = products && (act || !tma_ready(a->gy, a->N));
    const int rows_per = (int)std::max<long long>(16, ((a->rows * ((a->N + 255) / 256) + 148 * 8 - 1) / (148 * 8) + 7) / 8 * 8);
    const int row_blocks = (int)((a->rows + rows_per - 1) / rows_per);
    GradArgs ga = {};
    ga.rows = a->rows; ga.N = (int)a->N; ga.act = a->act; ga.rows_per = rows_per;
    ga.gy = a->gy; ga.mul = a->mul;
    if (act) {
        ga.z[0] = (const float *)a->saved;
        ga.z[1] = a->pair && a->saved != nullptr ? (const float *)((const char *)a->saved + saved_one(a)) : nullptr;
        ga.z_row = up8(a->N);
    }
    ga.gz_row = up8(a->N);
    if (own_gz) {
        for (int i = 0; i < sources; i++) ga.gz[i] = ws.take((size_t)a->rows * up8(a->N) * 2);
    }
    ga.gmul = a->gmul;
    if (a->gbias != nullptr) ga.part = (float *)ws.take((size_t)row_blocks * a->N * 4);
    int rc = WKV_OK;
    if (!count && (own_gz || a->gmul != nullptr || a->gbias != nullptr)) {
        const dim3 grid((unsigned)((a->N + 255) / 256), (unsigned)row_blocks);
        const bool vec = a->N % 8 == 0 && all_aligned({a->gy, a->mul, a->gmul});
        rc = a->pair ? launch_chained(vec ? k_grad_act<F, true, true> : k_grad_act<F, true, false>, grid, dim3(256), 0, s, ga)
                     : launch_chained(vec ? k_grad_act<F, false, true> : k_grad_act<F, false, false>, grid, dim3(256), 0, s, ga);
        if (rc == WKV_OK && a->gbias != nullptr) {
            FoldOut out = {};
            out.p[0] = a->gbias; out.dtype[0] = a->bias_dtype;
            for (int i = 1; i < 5; i++) out.start[i] = a->N;
            rc = fold_params(ga.part, row_blocks, a->N, out, s);
        }
        if (rc != WKV_OK) return rc;
    }
    Matrix gz[2];
    for (int i = 0; i < 2; i++) {
        const int j = a->pair ? i : 0;
        gz[i] = own_gz ? Matrix{ga.gz[j], a->rows, a->N, up8(a->N)} : Matrix{a->gy, a->rows, a->N, a->N};
    }
    size_t most = 0;
    if (a->gx != nullptr) {
        Matrix w[2] = {w_of(a, 0), w_of(a, a->pair)};
        rc = a->pair ? ready<F>({&w[0], &w[1]}, ws, s) : ready<F>({&w[0]}, ws, s);
        const Cut cut = cut_for(a->rows, a->K, 1, kb_n, false);
        most = std::max(most, align256(cut.part_bytes()));
        if (!count && rc == WKV_OK) {
            Epi e = {};
            e.vec = a->K % 8 == 0 && aligned16(a->gx);
            e.y[0] = a->gx; e.y_row = a->K;
            Scratch parts = ws;
            rc = product<F, false, true, EPI_PLAIN>(gz, w, sources, sources, a->rows, a->K, a->N, cut, e, parts.take(cut.part_bytes()), a->status, s);
        }
    }
    if (rc == WKV_OK && (a->gw0 != nullptr || a->gw1 != nullptr)) {
        Matrix x = x_of(a);
        rc = ready<F>({&x}, ws, s);
        const Matrix xs[2] = {x, x};
        const bool both = a->gw0 != nullptr && a->gw1 != nullptr;
        const Cut cut = cut_for(a->N, a->K, 1 + both, kb_r, false);
        most = std::max(most, align256(cut.part_bytes()));
        if (!count && rc == WKV_OK) {
            Epi e = {};
            e.vec = a->K % 8 == 0 && all_aligned({a->gw0, a->gw1});
            e.y[0] = a->gw0 != nullptr ? a->gw0 : a->gw1;
            e.y[1] = a->gw1;
            e.y_row = a->K;
            if (a->gw0 == nullptr) gz[0] = gz[1];
            Scratch parts = ws;
            rc = product<F, true, true, EPI_PLAIN>(gz, xs, 1 + both, 1, a->N, a->K, a->rows, cut, e, parts.take(cut.part_bytes()), a->status, s);
        }
    }
    if (count) *need = ws.used + most;
    return rc;
}

template <class Fn>
int by_16bit(int d, Fn f) { return d == WKV_BF16 ? f(__nv_bfloat16{}) : f(__half{}); }

}  // namespace
}  // namespace linear
}  // namespace wkv

using namespace wkv;
using namespace wkv::linear;

extern "C" size_t wkv_linear_saved_bytes(const wkv_linear_args_t *a) {
    return check_args(a) == WKV_OK && keeps(a) ? saved_one(a) * (1 + a->pair) : 0;
}

extern "C" size_t wkv_linear_forward_workspace(const wkv_linear_args_t *a) {
    size_t n = 0;
    if (check_args(a) == WKV_OK && a->rows > 0) by_16bit(a->dtype, [&](auto f) { return forward<decltype(f)>(a, Scratch{nullptr}, &n, nullptr); });
    return n;
}

extern "C" int wkv_linear_forward(const wkv_linear_args_t *a, void *stream) {
    const int e = check_args(a);
    if (e != WKV_OK || a->rows == 0) return e;
    if (a->x == nullptr || a->w0 == nullptr || (a->pair && a->w1 == nullptr) || a->y == nullptr) return WKV_ERR_NULL;
    if (a->saved != nullptr && a->saved_bytes < wkv_linear_saved_bytes(a)) return WKV_ERR_WORKSPACE;
    const size_t need = wkv_linear_forward_workspace(a);
    if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need)) return WKV_ERR_WORKSPACE;
    if (!all_aligned({a->workspace, a->saved})) return WKV_ERR_ALIGN;
    return by_16bit(a->dtype, [&](auto f) { return forward<decltype(f)>(a, Scratch{(char *)a->workspace}, nullptr, (cudaStream_t)stream); });
}

extern "C" size_t wkv_linear_backward_workspace(const wkv_linear_args_t *a) {
    size_t n = 0;
    if (check_args(a) == WKV_OK && a->rows > 0) by_16bit(a->dtype, [&](auto f) { return backward<decltype(f)>(a, Scratch{nullptr}, &n, nullptr); });
    return n;
}

extern "C" int wkv_linear_backward(const wkv_linear_args_t *a, void *stream) {
    const int e = check_args(a);
    if (e != WKV_OK) return e;
    const cudaStream_t s = (cudaStream_t)stream;
    if (a->rows == 0) {
        for (void *p : {a->gw0, a->gw1})
            if (p != nullptr && cudaMemsetAsync(p, 0, (size_t)a->N * a->K * 2, s) != cudaSuccess) return WKV_ERR_LAUNCH;
        if (a->gbias != nullptr && cudaMemsetAsync(a->gbias, 0, (size_t)a->N * elem_size(a->bias_dtype), s) != cudaSuccess) return WKV_ERR_LAUNCH;
        return WKV_OK;
    }
    if (a->gy == nullptr || (a->gx != nullptr && (a->w0 == nullptr || (a->pair && a->w1 == nullptr))) ||
        ((a->gw0 != nullptr || a->gw1 != nullptr) && a->x == nullptr) || (!a->pair && a->gw1 != nullptr))
        return WKV_ERR_NULL;
    if (a->gbias != nullptr && !known_dtype(a->bias_dtype)) return WKV_ERR_DTYPE;
    if (keeps(a) && (a->saved == nullptr || a->saved_bytes < wkv_linear_saved_bytes(a))) return WKV_ERR_WORKSPACE;
    const size_t need = wkv_linear_backward_workspace(a);
    if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need)) return WKV_ERR_WORKSPACE;
    if (!all_aligned({a->workspace, a->saved})) return WKV_ERR_ALIGN;
    return by_16bit(a->dtype, [&](auto f) { return backward<decltype(f)>(a, Scratch{(char *)a->workspace}, nullptr, s); });
}

extern "C" int wkv_linear_selftest_abort(const wkv_linear_args_t *a, int backward_call, int skip_block, unsigned limit, void *stream) {
    if (skip_block < 0 || limit < 1 || limit > 100000) return WKV_ERR_SHAPE;
    t_skip = skip_block;
    t_limit = limit;
    const int rc = backward_call ? wkv_linear_backward(a, stream) : wkv_linear_forward(a, stream);
    t_skip = -1;
    t_limit = WAIT_LIMIT;
    return rc;
}
