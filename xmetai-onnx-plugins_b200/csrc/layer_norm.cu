// layer_norm.cu -- LayerNormFn for sm_100a.
//
// Math, per row: s = x + residual (rounded to the I/O type), mean = average(s) or 0,
// rstd = 1 / sqrt(average((s - mean)^2) + eps), y = (s - mean) rstd weight + bias.
#include <algorithm>

#include "xm_common.cuh"
#include "xm_kernels.h"

namespace xm {
namespace {

constexpr int kThreads = 256;

// Sum over the block, the same in every thread.
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

// A block per row, three passes over it.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_kernel(const NormArgs p) {
    __shared__ float part[kThreads / 32];
    for (unsigned row = blockIdx.x; row < static_cast<unsigned>(p.rows); row += gridDim.x) {
        const size_t at = static_cast<size_t>(row) * p.dim;
        const T *s = static_cast<const T *>(p.x) + at;
        float sum = 0.0f;
        if (p.residual != nullptr) {
            T *const kept = static_cast<T *>(p.sum) + at;
            for (int d = threadIdx.x; d < p.dim; d += kThreads) {
                const T v = from_f32<T>(to_f32<T>(s[d]) + to_f32<T>(static_cast<const T *>(p.residual)[at + d]));
                kept[d] = v;
                sum += to_f32<T>(v);
            }
            s = kept;
        } else {
            for (int d = threadIdx.x; d < p.dim; d += kThreads) sum += to_f32<T>(s[d]);
        }
        const float mean = p.rms ? 0.0f : block_sum(sum, part) / p.dim;
        float sq = 0.0f;
        for (int d = threadIdx.x; d < p.dim; d += kThreads) {
            const float v = to_f32<T>(s[d]) - mean;
            sq = fmaf(v, v, sq);
        }
        const float rstd = 1.0f / sqrtf(block_sum(sq, part) / p.dim + p.eps);
        for (int d = threadIdx.x; d < p.dim; d += kThreads) {
            const float v = (to_f32<T>(s[d]) - mean) * rstd;
            static_cast<T *>(p.out)[at + d] = from_f32<T>(
                fmaf(v, p.weight != nullptr ? p.weight[d] : 1.0f, p.bias != nullptr ? p.bias[d] : 0.0f));
        }
        if (p.stats != nullptr && threadIdx.x == 0) {
            p.stats[2 * static_cast<size_t>(row)] = mean;
            p.stats[2 * static_cast<size_t>(row) + 1] = rstd;
        }
    }
}

template <typename T>
cudaError_t launch_type(const NormArgs &a, cudaStream_t stream) {
    norm_kernel<T><<<std::min(a.rows, 148 * 8), kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_layer_norm(const NormArgs &a, cudaStream_t stream) {
    switch (a.io) {
        case IoType::kBF16: return launch_type<__nv_bfloat16>(a, stream);
        case IoType::kF16: return launch_type<__half>(a, stream);
        default: return launch_type<float>(a, stream);
    }
}

}  // namespace xm
