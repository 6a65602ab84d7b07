// The fold of per-CTA parameter-gradient sums of the norm, the short convolution and the selective scan.
#include "elem_io.cuh"

namespace wkv {
namespace {

// 32 columns by 8 row groups per CTA, the groups meet in shared memory in a fixed order: the same bits every time.
// Bound by the latency of its loads (a few MB from L2): eight in flight per thread.  With few columns it has few CTAs: the 4096 rows of 320
// columns of a convolution of 8 x 8192 tokens of 64 channels are read by 10 (backward 91 us in all).
__global__ void __launch_bounds__(256) k_fold_params(const float *__restrict__ part, int rows, long long cols, FoldOut out) {
    pdl_wait();
    pdl_trigger();
    __shared__ float red[8][32];
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
    const long long col = (long long)blockIdx.x * 32 + lane;
    float a = 0.f;
    if (col < cols) {
#pragma unroll 8
        for (int r = g; r < rows; r += 8) a += part[(size_t)r * cols + col];
    }
    red[g][lane] = a;
    __syncthreads();
    if (g == 0 && col < cols) {
#pragma unroll
        for (int q = 1; q < 8; q++) a += red[q][lane];
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (out.p[i] != nullptr && col >= out.start[i] && col < out.start[i + 1]) store_as(out.p[i], out.dtype[i], (size_t)(col - out.start[i]), a);
    }
}

}  // namespace

int fold_params(const float *part, int rows, long long cols, const FoldOut &out, cudaStream_t s) {
    if (cols == 0) return WKV_OK;
    return launch_chained(k_fold_params, dim3((unsigned)((cols + 31) / 32)), dim3(256), 0, s, part, rows, cols, out);
}

}  // namespace wkv
