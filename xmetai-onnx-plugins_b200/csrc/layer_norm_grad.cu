// layer_norm_grad.cu -- LayerNormGradFn for sm_100a.
//
// Math, per row with xhat = (x - mean) rstd and g = dy weight:
//   dx = rstd (g - average(g) - xhat average(g xhat)) + d_residual,
// and over the rows d_weight = sum dy xhat, d_bias = sum dy.
#include <algorithm>

#include "xm_common.cuh"
#include "xm_kernels.h"

namespace xm {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float block_sum(float v, float *part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[threadIdx.x & (kThreads / 32 - 1)];
#pragma unroll
    for (int o = kThreads / 64; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
    return v;
}

// A block per row, two passes over it.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_grad_rows_kernel(const NormGradArgs p) {
    __shared__ float part[kThreads / 32];
    for (unsigned row = blockIdx.x; row < static_cast<unsigned>(p.rows); row += gridDim.x) {
        const size_t at = static_cast<size_t>(row) * p.dim;
        const float mean = p.rms ? 0.0f : p.stats[2 * static_cast<size_t>(row)];
        const float rstd = p.stats[2 * static_cast<size_t>(row) + 1];
        float sg = 0.0f, sx = 0.0f;
        for (int d = threadIdx.x; d < p.dim; d += kThreads) {
            const float g = to_f32<T>(static_cast<const T *>(p.dy)[at + d]) * (p.weight != nullptr ? p.weight[d] : 1.0f);
            sg += g;
            sx = fmaf(g, (to_f32<T>(static_cast<const T *>(p.x)[at + d]) - mean) * rstd, sx);
        }
        sg = p.rms ? 0.0f : block_sum(sg, part) / p.dim;
        sx = block_sum(sx, part) / p.dim;
        for (int d = threadIdx.x; d < p.dim; d += kThreads) {
            const float g = to_f32<T>(static_cast<const T *>(p.dy)[at + d]) * (p.weight != nullptr ? p.weight[d] : 1.0f);
            const float xhat = (to_f32<T>(static_cast<const T *>(p.x)[at + d]) - mean) * rstd;
            const float more = p.dres != nullptr ? to_f32<T>(static_cast<const T *>(p.dres)[at + d]) : 0.0f;
            static_cast<T *>(p.dx)[at + d] = from_f32<T>(fmaf(rstd, g - sg - xhat * sx, more));
        }
    }
}

// A thread per column walks the rows.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_grad_columns_kernel(const NormGradArgs p) {
    const int d = blockIdx.x * kThreads + threadIdx.x;
    if (d >= p.dim) return;
    float sw = 0.0f, sb = 0.0f;
    for (int row = 0; row < p.rows; ++row) {
        const float dy = to_f32<T>(static_cast<const T *>(p.dy)[static_cast<size_t>(row) * p.dim + d]);
        const float x = to_f32<T>(static_cast<const T *>(p.x)[static_cast<size_t>(row) * p.dim + d]);
        const float mean = p.rms ? 0.0f : p.stats[2 * static_cast<size_t>(row)];
        sw = fmaf(dy, (x - mean) * p.stats[2 * static_cast<size_t>(row) + 1], sw);
        sb += dy;
    }
    if (p.dweight != nullptr) p.dweight[d] = sw;
    if (p.dbias != nullptr) p.dbias[d] = sb;
}

template <typename T>
cudaError_t launch_type(const NormGradArgs &a, cudaStream_t stream) {
    if (a.rows > 0) norm_grad_rows_kernel<T><<<std::min(a.rows, 148 * 8), kThreads, 0, stream>>>(a);
    if (a.dweight != nullptr || a.dbias != nullptr)
        norm_grad_columns_kernel<T><<<(a.dim + kThreads - 1) / kThreads, kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

size_t layer_norm_grad_workspace(const NormGradArgs &) { return 0; }

cudaError_t launch_layer_norm_grad(const NormGradArgs &a, void *, cudaStream_t stream) {
    switch (a.io) {
        case IoType::kBF16: return launch_type<__nv_bfloat16>(a, stream);
        case IoType::kF16: return launch_type<__half>(a, stream);
        default: return launch_type<float>(a, stream);
    }
}

}  // namespace xm
