// column_sum.cu -- sums of partial gradients over the blocks that left them, in a fixed
// order, for GatedRecurrenceGradFn and LayerNormGradFn.
//
// A block takes 32 columns; its 32 warps take the rows in turn, four loads at a time,
// and their sums are added in order. The partials were written just before and come
// from L2; its blocks are on their SMs before the kernel that writes them ends.
#include "xm_common.cuh"
#include "xm_kernels.h"

namespace xm {
namespace {

constexpr int kWarps = 32;

__global__ void __launch_bounds__(32 * kWarps) column_sum_kernel(const float *part0, const float *part1, int rows, int dim,
                                                               float *out0, float *out1) {
    __shared__ float sums[kWarps][32];
    const float *const part = blockIdx.y == 0 ? part0 : part1;
    float *const out = blockIdx.y == 0 ? out0 : out1;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int d = blockIdx.x * 32 + lane;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    wait_for_before();
    if (d < dim) {
        const float *const p = part + d;
        int r = warp;
        for (; r + 3 * kWarps < rows; r += 4 * kWarps) {
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] += p[static_cast<size_t>(r + k * kWarps) * dim];
        }
        for (; r < rows; r += kWarps) s[0] += p[static_cast<size_t>(r) * dim];
    }
    sums[warp][lane] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (warp != 0 || d >= dim) return;
    float v = sums[0][lane];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) v += sums[w][lane];
    out[d] = v;
}

}  // namespace

cudaError_t launch_column_sums(const float *part0, const float *part1, int rows, int dim, float *out0, float *out1,
                               cudaStream_t stream) {
    const dim3 grid((dim + 31) / 32, part1 != nullptr ? 2 : 1);
    return launch_behind(column_sum_kernel, grid, dim3(32 * kWarps), 0, stream, part0, part1, rows, dim, out0, out1);
}

}  // namespace xm
