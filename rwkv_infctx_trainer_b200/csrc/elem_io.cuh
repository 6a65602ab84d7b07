// Runs of consecutive elements of one type, read and written 16 bytes (or one run) at a time where the addresses
// allow it, and the fold of per-CTA parameter-gradient sums: shared by the norm, the short convolution and the
// selective scan.
#pragma once
#include <type_traits>

#include "wkv_common.cuh"

namespace wkv {

// N consecutive elements as they lie in memory, in whole 32-bit words (N * sizeof(F) is a multiple of 4)
template <typename F, int N>
struct alignas(N * sizeof(F) < 16 ? N * sizeof(F) : 16) Raw {
    static constexpr int WORDS = N * (int)sizeof(F) / 4;
    uint32_t w[WORDS];

    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < WORDS; i++) w[i] = 0u;
    }
    // vec: p is a multiple of the run's size (16 bytes at most) and all N elements exist; else element by element, the first
    // `n` of them
    __device__ __forceinline__ void load(const F *p, bool vec, int n) {
        if (vec) {
            if constexpr (WORDS % 4 == 0) {
#pragma unroll
                for (int i = 0; i < WORDS; i += 4) {
                    const uint4 q = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint32_t *>(p) + i);
                    w[i] = q.x; w[i + 1] = q.y; w[i + 2] = q.z; w[i + 3] = q.w;
                }
            } else if constexpr (WORDS == 2) {
                const uint2 q = *reinterpret_cast<const uint2 *>(p);
                w[0] = q.x; w[1] = q.y;
            } else {
#pragma unroll
                for (int i = 0; i < WORDS; i++) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
            }
        } else {
            zero();
#pragma unroll
            for (int i = 0; i < N; i++) {
                if (i < n) {
                    if constexpr (sizeof(F) == 4) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
                    else w[i / 2] |= (uint32_t) reinterpret_cast<const uint16_t *>(p)[i] << (16 * (i & 1));
                }
            }
        }
    }
    __device__ __forceinline__ void store(F *p, bool vec, int n) const {
        if (vec) {
            if constexpr (WORDS % 4 == 0) {
#pragma unroll
                for (int i = 0; i < WORDS; i += 4)
                    *reinterpret_cast<uint4 *>(reinterpret_cast<uint32_t *>(p) + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
            } else if constexpr (WORDS == 2) {
                *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
            } else {
#pragma unroll
                for (int i = 0; i < WORDS; i++) reinterpret_cast<uint32_t *>(p)[i] = w[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) {
                if (i < n) {
                    if constexpr (sizeof(F) == 4) reinterpret_cast<uint32_t *>(p)[i] = w[i];
                    else reinterpret_cast<uint16_t *>(p)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
                }
            }
        }
    }
    // the same one by one from elements S apart, the first `n` of them (the rest zeros): neighbouring lanes' S-apart elements are
    // one access for the warp where rows are not aligned
    template <int S>
    __device__ __forceinline__ void gather(const F *p, int n) {
        zero();
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (i < n) {
                if constexpr (sizeof(F) == 4) w[i] = reinterpret_cast<const uint32_t *>(p)[i * S];
                else w[i / 2] |= (uint32_t) reinterpret_cast<const uint16_t *>(p)[i * S] << (16 * (i & 1));
            }
        }
    }
    template <int S>
    __device__ __forceinline__ void scatter(F *p, int n) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (i < n) {
                if constexpr (sizeof(F) == 4) reinterpret_cast<uint32_t *>(p)[i * S] = w[i];
                else reinterpret_cast<uint16_t *>(p)[i * S] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
            }
        }
    }
    __device__ __forceinline__ void get(float *f) const {
        if constexpr (sizeof(F) == 4) {
#pragma unroll
            for (int i = 0; i < N; i++) f[i] = __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                float2 v;
                if constexpr (std::is_same<F, __nv_bfloat16>::value) v = unpack2(w[i / 2]);
                else v = __half22float2(*reinterpret_cast<const __half2 *>(&w[i / 2]));
                f[i] = v.x;
                f[i + 1] = v.y;
            }
        }
    }
    // (one rounding, to nearest)
    __device__ __forceinline__ void put(const float *f) {
        if constexpr (sizeof(F) == 4) {
#pragma unroll
            for (int i = 0; i < N; i++) w[i] = __float_as_uint(f[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                if constexpr (std::is_same<F, __nv_bfloat16>::value) w[i / 2] = pack2(f[i], f[i + 1]);
                else {
                    const __half2 h = __floats2half2_rn(f[i], f[i + 1]);
                    w[i / 2] = *reinterpret_cast<const uint32_t *>(&h);
                }
            }
        }
    }
};

// element i of a parameter of element type `dtype`
__device__ __forceinline__ float param_at(const void *p, int dtype, size_t i) {
    if (dtype == WKV_F32) return __ldg((const float *)p + i);
    if (dtype == WKV_BF16) return __bfloat162float(__ldg((const __nv_bfloat16 *)p + i));
    return __half2float(__ldg((const __half *)p + i));
}

inline bool known_dtype(int d) { return d == WKV_F32 || d == WKV_BF16 || d == WKV_F16; }
inline int elem_size(int d) { return d == WKV_F32 ? 4 : 2; }
inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Up to four parameter gradients side by side in one row of partial sums: columns [start[i], start[i+1]) go to p[i]
// (NULL: not wanted).
struct FoldOut {
    void *p[4];
    int dtype[4];
    long long start[5];
};
// sums the `rows` rows of part [rows, cols], always in the same order, into their outputs (timemix_fused.cu's
// k_fold_cols for outputs of unequal widths); rows = 0 gives zeros (param_fold.cu)
int fold_params(const float *part, int rows, long long cols, const FoldOut &out, cudaStream_t s);

// calls f with a value of the element type that the code stands for
template <class Fn>
inline int by_dtype(int d, Fn f) {
    switch (d) {
        case WKV_F32: return f(float{});
        case WKV_BF16: return f(__nv_bfloat16{});
        case WKV_F16: return f(__half{});
        default: return WKV_ERR_DTYPE;
    }
}

}  // namespace wkv
