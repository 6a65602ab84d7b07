// Root-mean-square norm with the residual's addition, its gradient, and the same with an output in 8 bits.
//
//   h = x + residual        (stored in the residual's type; without a residual h = x and is not stored)
//   y = weight * h * r,     r = 1 / sqrt(mean(h^2) + eps)
//   8 bits: scale = max|y| / 448 over the row, or over each group of channels; q = e4m3(y / scale)
//
//   backward, with gh the gradient that reaches h from elsewhere:
//   xh = h r,  gx = gh + r (gy weight - xh mean(gy weight xh)),  gweight = sum over the rows of gy xh
//
// Both passes start from the sum before it is rounded: a backward pass from an h in bf16 was 2^-9 off in gweight, which is
// a sum in fp32.
//
// A row crosses HBM once per pass, a thread owns runs of 8 channels and keeps them in registers from
// the sum to the output.  A CTA takes every gridDim-th row, so that the weights (and the sums of their gradient) stay in
// registers.  Sums are fp32 and in a fixed order.  Bound by HBM forward, and backward for rows of a multiple of 8 channels, 8192 at most:
// 16384 rows of 4096 bf16 channels with a bf16 residual take 88 us (6.1 TB/s) and 117 (5.7 TB/s of its 10 bytes a channel).  Wider rows,
// and rows that start anywhere, spill registers backward (split_of): 4096 rows of 16384 channels 91 and 194 us.
#include <cuda_fp8.h>

#include "elem_io.cuh"
#include "wkv_internal.h"

namespace wkv {
namespace {

constexpr int RUN = 8;            // channels a thread takes at once

// sums (or maxima of non-negative values, given as bits) over the CTA; `red` has a place for each warp and is reused by
// alternating halves
__device__ __forceinline__ float cta_sum(float v, float *red, int nwarp) {
    v = warp_sum(v);
    if (nwarp == 1) return v;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < nwarp ? red[threadIdx.x & 31] : 0.f;
    return warp_sum(v);
}
__device__ __forceinline__ float2 cta_sum2(float2 v, float2 *red, int nwarp) {
    v.x = warp_sum(v.x); v.y = warp_sum(v.y);
    if (nwarp == 1) return v;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < nwarp ? red[threadIdx.x & 31] : make_float2(0.f, 0.f);
    v.x = warp_sum(v.x); v.y = warp_sum(v.y);
    return v;
}
__device__ __forceinline__ uint32_t warp_max_bits(uint32_t v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// How rows lie, and a thread's eight channels of a run.  RUNS: rows of a multiple of 8 channels, the channels are neighbours.
// PAIRS: of an even number, four pairs that are 64 channels apart.  ONES: of any number, single channels 32 apart.  In each a warp has
// 256 neighbouring channels and its accesses are whole pieces of a row.  (With neighbours in rows that are not aligned, 3635 rows
// of 6965 channels took 168 us forward and 288 backward; so 64 and 178.)
enum { RUNS, PAIRS, ONES };
template <int MODE>
struct Lie {
    static constexpr int UNIT = MODE == RUNS ? RUN : MODE == PAIRS ? 2 : 1, UNITS = RUN / UNIT, APART = MODE == RUNS ? RUN : 32 * UNIT;
    static __device__ __forceinline__ int first(int i) {
        const int tid = threadIdx.x, nt = blockDim.x;
        return MODE == RUNS ? (tid + i * nt) * RUN : ((tid >> 5) + i * (nt >> 5)) * (32 * RUN) + (tid & 31) * UNIT;
    }
    // how many of the channels from c on exist
    static __device__ __forceinline__ int left(int C, int c) { return c >= C ? 0 : MODE == RUNS ? RUN : min(RUN, (C - c + APART - 1) / APART * UNIT); }
    static __device__ __forceinline__ int channel(int c, int q) { return c + q / UNIT * APART + q % UNIT; }
    template <typename T>
    static __device__ __forceinline__ void load(Raw<T, RUN> &r, const T *p, int n) {
        if constexpr (MODE == RUNS) r.load(p, true, RUN);
        else if constexpr (MODE == ONES) r.template gather<32>(p, n);
        else {
#pragma unroll
            for (int i = 0; i < UNITS; i++) {
                Raw<T, 2> u;
                u.zero();
                if (2 * i < n) u.load(p + i * APART, true, 2);
#pragma unroll
                for (int k = 0; k < u.WORDS; k++) r.w[i * u.WORDS + k] = u.w[k];
            }
        }
    }
    template <typename T>
    static __device__ __forceinline__ void store(const Raw<T, RUN> &r, T *p, int n) {
        if constexpr (MODE == RUNS) r.store(p, true, RUN);
        else if constexpr (MODE == ONES) r.template scatter<32>(p, n);
        else {
#pragma unroll
            for (int i = 0; i < UNITS; i++) {
                Raw<T, 2> u;
#pragma unroll
                for (int k = 0; k < u.WORDS; k++) u.w[k] = r.w[i * u.WORDS + k];
                if (2 * i < n) u.store(p + i * APART, true, 2);
            }
        }
    }
    // into shared memory without passing through registers (not ONES)
    template <typename T>
    static __device__ __forceinline__ void load_async(Raw<T, RUN> *to, const T *p, int n) {
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
        constexpr int BYTES = UNIT * (int)sizeof(T), PIECE = BYTES < 16 ? BYTES : 16;
#pragma unroll
        for (int i = 0; i < UNITS; i++) {
            if (i * UNIT < n) {
#pragma unroll
                for (int k = 0; k < BYTES; k += PIECE) {
                    const char *from = (const char *)(p + i * APART) + k;
                    if constexpr (PIECE == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + i * BYTES + k), "l"(from) : "memory");
                    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst + i * BYTES + k), "l"(from), "n"(PIECE) : "memory");
                }
            }
        }
    }
};

struct NormArgs {
    const void *x, *res, *w;
    void *y, *h;
    float *scale;
    long long rows;
    int C, w_dtype, group, ngroup;
    float eps;
};

// scale and 1 / scale for a largest value given as bits: as an unsigned number a NaN is above every other value, so one in
// the row makes the scale, and with it every value of the row, NaN.  Below 2^-100 (a row of zeros) the scale is 1.
__device__ __forceinline__ float q8_scale(uint32_t top) {
    const float m = __uint_as_float(top);
    return m <= 7.8886e-31f ? 1.f : m * (1.f / 448.f);
}

// NV runs a thread, MAXT threads at most
template <typename X, typename R, int NV, int MAXT, bool Q8, int MODE>
__global__ void __launch_bounds__(MAXT, 1024 / MAXT) k_rms_norm_fwd(NormArgs a) {
    pdl_wait();
    pdl_trigger();
    __shared__ float red[2][32];
    __shared__ uint32_t redm[2][32];
    const int tid = threadIdx.x, nt = blockDim.x, nwarp = nt >> 5, C = a.C;
    const X *x = (const X *)a.x;
    const R *res = (const R *)a.res;
    using L = Lie<MODE>;
    float w[NV][RUN];
    int left[NV];                       // channels of the run that exist
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = L::first(i);
        left[i] = L::left(C, c);
#pragma unroll
        for (int q = 0; q < RUN; q++) w[i][q] = q < left[i] ? param_at(a.w, a.w_dtype, L::channel(c, q)) : 0.f;
    }
    Raw<X, RUN> rx[NV];
    Raw<R, RUN> rr[NV];
    auto fetch = [&](long long row) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const size_t at = (size_t)row * C + L::first(i);
            rx[i].zero(); rr[i].zero();
            if (left[i] > 0) {
                L::load(rx[i], x + at, left[i]);
                if (res) L::load(rr[i], res + at, left[i]);
            }
        }
    };
    int par = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, par ^= 1) {
        fetch(row);
        float h[NV][RUN], ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            float t[RUN];
            rx[i].get(h[i]);
            rr[i].get(t);
#pragma unroll
            for (int q = 0; q < RUN; q++) { h[i][q] += t[q]; ss += h[i][q] * h[i][q]; }
        }
        if (a.h) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                Raw<R, RUN> o;
                o.put(h[i]);
                if (left[i] > 0) L::store(o, (R *)a.h + (size_t)row * C + L::first(i), left[i]);
            }
        }
        const float r = rsqrtf(cta_sum(ss, red[par], nwarp) / (float)C + a.eps);
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int q = 0; q < RUN; q++) h[i][q] = h[i][q] * r * w[i][q];
        if constexpr (!Q8) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                Raw<X, RUN> o;
                o.put(h[i]);
                if (left[i] > 0) L::store(o, (X *)a.y + (size_t)row * C + L::first(i), left[i]);
            }
        } else {
            // the largest of each unit of a thread's channels
            uint32_t top[NV][L::UNITS];
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int u = 0; u < L::UNITS; u++) {
                    top[i][u] = 0u;
#pragma unroll
                    for (int q = u * L::UNIT; q < (u + 1) * L::UNIT; q++)
                        if (q < left[i]) top[i][u] = max(top[i][u], __float_as_uint(h[i][q]) & 0x7FFFFFFFu);
                }
            if (a.group) {
                // A group is some neighbouring lanes of one warp (RUNS: group / 8; PAIRS: half a unit's or all), and if these are all, one or
                // more of the units
                const int lanes = min(32, a.group / L::UNIT), units = MODE == RUNS ? 1 : max(1, a.group / L::APART);
#pragma unroll
                for (int i = 0; i < NV; i++) {
#pragma unroll
                    for (int u = 0; u < L::UNITS; u++) top[i][u] = warp_max_bits(top[i][u], lanes);
#pragma unroll
                    for (int m = 1; m < L::UNITS; m <<= 1)
                        if (m < units) {
                            uint32_t both[L::UNITS];
#pragma unroll
                            for (int u = 0; u < L::UNITS; u++) both[u] = max(top[i][u], top[i][u ^ m]);
#pragma unroll
                            for (int u = 0; u < L::UNITS; u++) top[i][u] = both[u];
                        }
#pragma unroll
                    for (int u = 0; u < L::UNITS; u++)
                        if (u * L::UNIT < left[i] && (tid & (lanes - 1)) == 0 && (u & (units - 1)) == 0)
                            a.scale[(size_t)row * a.ngroup + (L::first(i) + u * L::APART) / a.group] = q8_scale(top[i][u]);
                }
            } else {
                uint32_t m = 0u;
#pragma unroll
                for (int i = 0; i < NV; i++)
#pragma unroll
                    for (int u = 0; u < L::UNITS; u++) m = max(m, top[i][u]);
                m = warp_max_bits(m, 32);
                if (nwarp > 1) {
                    if ((tid & 31) == 0) redm[par][tid >> 5] = m;
                    __syncthreads();
                    m = warp_max_bits((tid & 31) < nwarp ? redm[par][tid & 31] : 0u, 32);
                }
#pragma unroll
                for (int i = 0; i < NV; i++)
#pragma unroll
                    for (int u = 0; u < L::UNITS; u++) top[i][u] = m;
                if (tid == 0) a.scale[row] = q8_scale(m);
            }
#pragma unroll
            for (int i = 0; i < NV; i++) {
                uint32_t o[2] = {0u, 0u};
#pragma unroll
                for (int q = 0; q < RUN; q += 2) {
                    // to nearest, at most 448; a NaN stays one
                    const float i0 = 1.f / q8_scale(top[i][q / L::UNIT]), i1 = L::UNIT > 1 ? i0 : 1.f / q8_scale(top[i][(q + 1) / L::UNIT]);
                    const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(h[i][q] * i0, h[i][q + 1] * i1), __NV_SATFINITE, __NV_E4M3);
                    o[q / 4] |= two << (8 * (q & 3));
                }
                if (left[i] > 0) {
                    unsigned char *p = (unsigned char *)a.y + (size_t)row * C + L::first(i);
                    if (MODE == RUNS) {
                        *reinterpret_cast<uint2 *>(p) = make_uint2(o[0], o[1]);
                    } else {
#pragma unroll
                        for (int u = 0; u < L::UNITS; u++) {
                            const uint32_t v = o[u * L::UNIT / 4] >> (8 * (u * L::UNIT & 3));
                            if (u * L::UNIT < left[i]) {
                                if (MODE == PAIRS) *reinterpret_cast<uint16_t *>(p + u * L::APART) = (uint16_t)v;
                                else p[u * L::APART] = (unsigned char)v;
                            }
                        }
                    }
                }
            }
        }
    }
}

template <int LEFT>
__device__ __forceinline__ void rows_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }
__device__ __forceinline__ void rows_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// rows on their way, for 1024 threads an SM with `bytes` of a row each: what fits in 200 KB, three at most
constexpr int rows_ahead(int bytes) { return 200 / bytes > 3 ? 3 : 200 / bytes < 1 ? 1 : 200 / bytes; }

struct NormBwdArgs {
    const void *h, *x, *res, *w, *gy, *gh;         // h, or x and the residual
    void *gx, *gres;
    float *part;                        // [gridDim.x, C], NULL when the weight needs no gradient
    long long rows;
    int C, w_dtype;
    float eps;
};

// SUM: h = x + residual (or x alone), else h is read
template <typename X, typename R, int NV, bool SUM>
struct BwdPlace {
    // (gy, x; h or the residual, gh -- the last passes through registers where threads have two runs: fp32 rows of 16384 channels
    // are 192 KB without it)
    static constexpr int TX = SUM ? 2 : 1, TR = NV == 1 ? 2 : 1;
    static constexpr int ROW = NV * RUN * (int)(TX * sizeof(X) + TR * sizeof(R)), AHEAD = rows_ahead(ROW);
};
template <typename X, typename R, int NV, int MAXT, bool SUM, int MODE>
__global__ void __launch_bounds__(MAXT, 1024 / MAXT) k_rms_norm_bwd(NormBwdArgs a) {
    pdl_wait();
    pdl_trigger();
    __shared__ float2 red[2][32];
    const int tid = threadIdx.x, nt = blockDim.x, nwarp = nt >> 5, C = a.C;
    const R *h = SUM ? (const R *)a.res : (const R *)a.h, *gh = (const R *)a.gh;
    const X *x = (const X *)a.x, *gy = (const X *)a.gy;
    using L = Lie<MODE>;
    float w[NV][RUN], gw[NV][RUN];
    int left[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = L::first(i);
        left[i] = L::left(C, c);
#pragma unroll
        for (int q = 0; q < RUN; q++) { w[i][q] = q < left[i] ? param_at(a.w, a.w_dtype, L::channel(c, q)) : 0.f; gw[i][q] = 0.f; }
    }
    using Place = BwdPlace<X, R, NV, SUM>;
    constexpr int AHEAD = Place::AHEAD, TX = Place::TX, TR = Place::TR;
    extern __shared__ __align__(16) char smem_raw[];
    Raw<X, RUN> *sx = reinterpret_cast<Raw<X, RUN> *>(smem_raw) + tid;                   // [AHEAD][NV][gy, x][threads]
    Raw<R, RUN> *sr = reinterpret_cast<Raw<R, RUN> *>(smem_raw + (size_t)AHEAD * NV * TX * nt * sizeof(Raw<X, RUN>)) + tid;     // [..][h, gh]
    auto fetch = [&](long long row, int slot) {
        if (row < a.rows) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const size_t at = (size_t)row * C + L::first(i);
                const int k = slot * NV + i;
                if (left[i] > 0) {
                    if constexpr (MODE != ONES) {
                        if (h) L::load_async(sr + (TR * k) * nt, h + at, left[i]);
                        if (TR == 2 && gh) L::load_async(sr + (TR * k + 1) * nt, gh + at, left[i]);
                        if (gy) L::load_async(sx + (TX * k) * nt, gy + at, left[i]);
                        if (SUM) L::load_async(sx + (TX * k + 1) * nt, x + at, left[i]);
                    } else {
                        // (there are no copies of 2 bytes: all loads, then all stores)
                        Raw<R, RUN> r0, r1;
                        Raw<X, RUN> x0, x1;
                        if (h) L::load(r0, h + at, left[i]);
                        if (TR == 2 && gh) L::load(r1, gh + at, left[i]);
                        if (gy) L::load(x0, gy + at, left[i]);
                        if (SUM) L::load(x1, x + at, left[i]);
                        if (h) sr[(TR * k) * nt] = r0;
                        if (TR == 2 && gh) sr[(TR * k + 1) * nt] = r1;
                        if (gy) sx[(TX * k) * nt] = x0;
                        if (SUM) sx[(TX * k + 1) * nt] = x1;
                    }
                }
            }
        }
        rows_commit();
    };
#pragma unroll
    for (int k = 0; k < AHEAD; k++) fetch(blockIdx.x + (long long)k * gridDim.x, k);
    int par = 0, slot = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, par ^= 1) {
        rows_wait<AHEAD - 1>();
        float hv[NV][RUN], g[NV][RUN];
        float2 s = make_float2(0.f, 0.f);       // sum h^2, sum gy w h
        Raw<R, RUN> keep[NV];
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int k = slot * NV + i;
#pragma unroll
            for (int q = 0; q < RUN; q++) { hv[i][q] = 0.f; g[i][q] = 0.f; }
            keep[i].zero();
            if (left[i] > 0) {
                if (h) sr[(TR * k) * nt].get(hv[i]);
                if (gh) {
                    if (TR == 2) keep[i] = sr[(TR * k + 1) * nt];
                    else L::load(keep[i], gh + (size_t)row * C + L::first(i), left[i]);
                }
                if (gy) sx[(TX * k) * nt].get(g[i]);
                if (SUM) {
                    float t[RUN];
                    sx[(TX * k + 1) * nt].get(t);
#pragma unroll
                    for (int q = 0; q < RUN; q++) hv[i][q] += t[q];
                }
                if (MODE == PAIRS) {           // (nothing was copied for channels that do not exist)
#pragma unroll
                    for (int q = 0; q < RUN; q++)
                        if (q >= left[i]) hv[i][q] = g[i][q] = 0.f;
                }
            }
#pragma unroll
            for (int q = 0; q < RUN; q++) { s.x += hv[i][q] * hv[i][q]; s.y += g[i][q] * w[i][q] * hv[i][q]; }
        }
        s = cta_sum2(s, red[par], nwarp);
        __syncwarp();                           // (the row has been read before anything is copied to its place)
        fetch(row + (long long)AHEAD * gridDim.x, slot);
        slot = slot + 1 == AHEAD ? 0 : slot + 1;
        const float r = rsqrtf(s.x / (float)C + a.eps), m = s.y * r / (float)C;      // m = mean(gy w xh)
#pragma unroll
        for (int i = 0; i < NV; i++) {
            float o[RUN];
            keep[i].get(o);
#pragma unroll
            for (int q = 0; q < RUN; q++) {
                const float xh = hv[i][q] * r;
                gw[i][q] += g[i][q] * xh;
                o[q] += r * (g[i][q] * w[i][q] - xh * m);
            }
            if (left[i] > 0) {
                const size_t at = (size_t)row * C + L::first(i);
                if (a.gx) { Raw<X, RUN> t; t.put(o); L::store(t, (X *)a.gx + at, left[i]); }
                if (a.gres) { Raw<R, RUN> t; t.put(o); L::store(t, (R *)a.gres + at, left[i]); }
            }
        }
    }
    if (a.part) {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int q = 0; q < RUN; q++)
                if (q < left[i]) a.part[(size_t)blockIdx.x * C + L::channel(L::first(i), q)] = gw[i][q];
    }
}

constexpr int MAX_C = 16384;
// How a row is divided: runs a thread, threads, CTAs for all SMs.  All kernels keep to 64 registers, 1024 threads an SM: with
// several CTAs there one loads while another sums or stores.  Forward nothing spills for that.  Backward a thread's weights, their gradient,
// h and gy do not always fit: with two runs (more than 8192 channels) every form spills 364 to 776 bytes a thread, with one run those for
// single channels (ONES) 152 to 336 and some of the others, with a 32-bit type, up to 36.  Us with a bf16 residual, forward and backward, and
// of their bytes: 4096 x 12288 76, 156 (62, 78); 4096 x 16384 91, 194 (83, 104); 3635 x 6965 64, 178 (31, 39); 3635 x 6966 38, 79 (31, 39).
// Another split of such rows has not been tried.  (Us: forward with twice the registers and the next row fetched ahead 98
// instead of 90, 8-bit output of 1999 x 5120 33 instead of 29; one run a thread 111.  Backward without rows on their way in shared
// memory 136 instead of 128, of 8192 x 8192 148 instead of 132; forward with them 97.)
struct Split {
    int nv, threads, ctas;
};
Split split_of(long long rows, int C, int nv) {
    Split s;
    const int runs = (C + RUN - 1) / RUN;
    s.nv = nv;
    s.threads = ((runs + nv - 1) / nv + 31) / 32 * 32;
    const long long n = (long long)device_sm_count() * (1024 / s.threads > 16 ? 16 : 1024 / s.threads);
    s.ctas = (int)(rows < n ? rows : n);
    return s;
}
Split forward_split(long long rows, int C) { return split_of(rows, C, 2); }
Split backward_split(long long rows, int C) { return split_of(rows, C, C <= 8192 ? 1 : 2); }

// how the rows of all the tensors lie
int lie_of(int C, std::initializer_list<std::pair<const void *, int>> tensors) {
    auto multiples = [&](int elements) {
        for (const auto &t : tensors) {
            const int bytes = elements * t.second;
            if (reinterpret_cast<uintptr_t>(t.first) & (uintptr_t)((bytes < 16 ? bytes : 16) - 1)) return false;
        }
        return C % elements == 0;
    };
    return multiples(RUN) ? RUNS : multiples(2) ? PAIRS : ONES;
}
template <class Fn>
int by_lie(int lie, Fn f) {
    switch (lie) {
        case RUNS: return f(std::integral_constant<int, RUNS>{});
        case PAIRS: return f(std::integral_constant<int, PAIRS>{});
        default: return f(std::integral_constant<int, ONES>{});
    }
}
template <auto KERN, class Args>
int run(const Args &k, const Split &sp, int smem, cudaStream_t s) {
    static unsigned char done[64];
    if (!set_max_smem_once(KERN, 227 * 1024 - 1024, done)) return WKV_ERR_LAUNCH;
    return launch_chained(KERN, dim3(sp.ctas), dim3(sp.threads), smem, s, k);
}

int check_norm(const wkv_rms_norm_args_t *a) {
    if (!a) return WKV_ERR_NULL;
    if (a->rows < 0 || a->C < 1 || a->C > MAX_C) return WKV_ERR_SHAPE;
    if (!known_dtype(a->dtype) || !known_dtype(a->w_dtype)) return WKV_ERR_DTYPE;
    if (a->res_dtype != a->dtype && a->res_dtype != WKV_F32) return WKV_ERR_DTYPE;
    if (!a->weight) return WKV_ERR_NULL;
    return WKV_OK;
}

// f is called with one value of x's type and one of the residual's
template <class Fn>
int by_types(int dtype, int res_dtype, Fn f) {
    return by_dtype(dtype, [&](auto x) {
        using X = decltype(x);
        return res_dtype == dtype ? f(X{}, X{}) : f(X{}, float{});
    });
}

}  // namespace
}  // namespace wkv

using namespace wkv;

extern "C" int wkv_rms_norm_forward(const wkv_rms_norm_args_t *a, void *stream) {
    int e = check_norm(a);
    if (e != WKV_OK) return e;
    if (a->scale) {
        if (a->group != 0 && a->group != 32 && a->group != 64 && a->group != 128 && a->group != 256) return WKV_ERR_SHAPE;
    }
    if (a->rows == 0) return WKV_OK;
    if (!a->x || !a->y || (a->residual && !a->h)) return WKV_ERR_NULL;
    if (!a->residual && a->res_dtype != a->dtype) return WKV_ERR_DTYPE;
    NormArgs k = {};
    k.x = a->x; k.res = a->residual; k.w = a->weight; k.y = a->y; k.h = a->residual ? a->h : nullptr;
    k.scale = a->scale;
    k.rows = a->rows; k.C = a->C; k.w_dtype = a->w_dtype; k.eps = a->eps;
    k.group = a->scale ? a->group : 0;
    k.ngroup = k.group ? (a->C + k.group - 1) / k.group : 1;
    const int xs = elem_size(a->dtype), rs = elem_size(a->res_dtype);
    const int lie = lie_of(a->C, {{a->x, xs}, {a->residual, rs}, {a->y, a->scale ? 1 : xs}, {k.h, rs}});
    const Split sp = forward_split(a->rows, a->C);
    cudaStream_t s = (cudaStream_t)stream;
    return by_types(a->dtype, a->res_dtype, [&](auto x, auto r) {
        using X = decltype(x);
        using R = decltype(r);
        const auto go = [&](auto kern) { return launch_chained(kern, dim3(sp.ctas), dim3(sp.threads), 0, s, k); };
        return by_lie(lie, [&](auto m) {
            constexpr int M = decltype(m)::value;
            if (sp.threads <= 512) return k.scale ? go(k_rms_norm_fwd<X, R, 2, 512, true, M>) : go(k_rms_norm_fwd<X, R, 2, 512, false, M>);
            return k.scale ? go(k_rms_norm_fwd<X, R, 2, 1024, true, M>) : go(k_rms_norm_fwd<X, R, 2, 1024, false, M>);
        });
    });
}

extern "C" size_t wkv_rms_norm_backward_workspace(const wkv_rms_norm_args_t *a) {
    if (check_norm(a) != WKV_OK) return 0;
    return align256((size_t)backward_split(a->rows, a->C).ctas * a->C * 4);
}

extern "C" int wkv_rms_norm_backward(const wkv_rms_norm_args_t *a, void *stream) {
    int e = check_norm(a);
    if (e != WKV_OK) return e;
    cudaStream_t s = (cudaStream_t)stream;
    const Split sp = backward_split(a->rows, a->C);
    if (a->rows > 0 && !a->h && !a->x) return WKV_ERR_NULL;
    if (!a->h && !a->residual && a->res_dtype != a->dtype) return WKV_ERR_DTYPE;
    if (a->gweight && a->rows > 0) {
        if (!a->workspace || a->workspace_bytes < wkv_rms_norm_backward_workspace(a)) return WKV_ERR_WORKSPACE;
        if (!aligned16(a->workspace)) return WKV_ERR_ALIGN;
    }
    NormBwdArgs k = {};
    k.h = a->h; k.x = a->x; k.res = a->residual; k.w = a->weight; k.gy = a->gy; k.gh = a->gh; k.gx = a->gx; k.gres = a->gresidual;
    k.part = a->gweight ? (float *)a->workspace : nullptr;
    k.rows = a->rows; k.C = a->C; k.w_dtype = a->w_dtype; k.eps = a->eps;
    const int xs = elem_size(a->dtype), rs = elem_size(a->res_dtype);
    const int lie = lie_of(a->C, {{a->h, rs}, {a->x, xs}, {a->residual, rs}, {a->gy, xs}, {a->gh, rs}, {a->gx, xs}, {a->gresidual, rs}});
    if (a->rows > 0) {
        e = by_types(a->dtype, a->res_dtype, [&](auto x, auto r) {
            using X = decltype(x);
            using R = decltype(r);
            const auto go = [&](auto sum) {
                constexpr bool SUM = decltype(sum)::value;
                using P1 = BwdPlace<X, R, 1, SUM>;
                return by_lie(lie, [&](auto m) {
                    constexpr int M = decltype(m)::value;
                    if (sp.nv == 2) {
                        using P2 = BwdPlace<X, R, 2, SUM>;
                        return run<k_rms_norm_bwd<X, R, 2, 1024, SUM, M>>(k, sp, sp.threads * P2::ROW * P2::AHEAD, s);
                    }
                    const int smem = sp.threads * P1::ROW * P1::AHEAD;
                    return sp.threads <= 512 ? run<k_rms_norm_bwd<X, R, 1, 512, SUM, M>>(k, sp, smem, s) : run<k_rms_norm_bwd<X, R, 1, 1024, SUM, M>>(k, sp, smem, s);
                });
            };
            return k.h ? go(std::false_type{}) : go(std::true_type{});
        });
        if (e != WKV_OK) return e;
    }
    if (!a->gweight) return WKV_OK;
    FoldOut f = {};
    f.p[0] = a->gweight; f.dtype[0] = a->w_dtype;
    f.start[0] = 0;
    for (int i = 1; i < 5; i++) f.start[i] = a->C;
    return fold_params((const float *)a->workspace, sp.ctas, a->C, f, s);
}
