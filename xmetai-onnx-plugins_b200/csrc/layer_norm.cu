// layer_norm.cu -- LayerNormFn for sm_100a.
//
// Math, per row: s = x + residual (rounded to the I/O type, as it is stored), mean =
// average(s) or 0, rstd = 1 / sqrt(average((s - mean)^2) + eps), y = (s - mean) rstd
// weight + bias.
//
// Bound by memory: x and the residual are read once and y and s written once. A row
// stays in the registers of its group of threads between the sum, the squares and the
// output, so it is not read again; rows that do not fit (above 16384 elements of
// the 16-bit types, 8192 of float32 or unaligned) are, from the caches.
#include <algorithm>

#include "xm_common.cuh"
#include "xm_kernels.h"
#include "xm_rows.cuh"

namespace xm {
namespace {

constexpr int threads_of(int group) { return group < 128 ? 128 : group; }

template <typename T, int VE, int kGroup>
__global__ void __launch_bounds__(threads_of(kGroup)) norm_kernel(const NormArgs p) {
    constexpr int kThreads = threads_of(kGroup), kRows = kThreads / kGroup;
    using Part = RowPart<T, VE, kGroup>;
    constexpr int kPairs = Part::kElems / 2;
    __shared__ float2 part[kGroup > 32 ? 2 * (kGroup / 32) : 1];
    const int g = threadIdx.x % kGroup, dim = p.dim;
    const float inv = 1.0f / static_cast<float>(dim);
    const unsigned rows = p.rows;
    const unsigned stride = gridDim.x * kRows;
    unsigned row = blockIdx.x * kRows + threadIdx.x / kGroup;
    const T *const X = static_cast<const T *>(p.x), *const R = static_cast<const T *>(p.residual);
    Part x, r;
    x.clear();
    r.clear();
    auto load = [&](unsigned i) {
        if (i >= rows) return;
        x.load(X + static_cast<size_t>(i) * dim, g, dim);
        if (R != nullptr) r.load(R + static_cast<size_t>(i) * dim, g, dim);
    };
    load(row);
    int turn = 0;
    // (all groups of a block make the same number of turns: their sums share barriers or shuffles)
    for (unsigned first = blockIdx.x * kRows; first < rows; first += stride, row += stride) {
        const bool there = row < rows;
        const size_t at = static_cast<size_t>(there ? row : 0) * dim;
        float2 v[kPairs];
        x.floats(v);
        if (R != nullptr) {
            float2 w[kPairs];
            r.floats(w);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) v[i] = __fadd2_rn(v[i], w[i]);
            Part s;
            s.from(v);
            if (there) s.store(static_cast<T *>(p.sum) + at, g, dim);
            s.floats(v);
        }
        load(row + stride);
        float mean = 0.0f;
        if (!p.rms) {
            float2 sum = twice(0.0f);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) sum = __fadd2_rn(sum, v[i]);
            mean = group_sum<kGroup>(make_float2(sum.x + sum.y, 0.0f), part, turn).x * inv;
            turn ^= 1;
        }
        float2 sq = twice(0.0f);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            v[i] = __fadd2_rn(v[i], twice(-mean));
            if (!Part::inside(2 * i, g, dim)) v[i].x = 0.0f;  // (behind the row's end)
            if (!Part::inside(2 * i + 1, g, dim)) v[i].y = 0.0f;
            sq = __ffma2_rn(v[i], v[i], sq);
        }
        const float rstd = 1.0f / sqrtf(group_sum<kGroup>(make_float2(sq.x + sq.y, 0.0f), part, turn).x * inv + p.eps);
        turn ^= 1;
        if (there) {
            float2 w[kPairs], b[kPairs];
            Part::vector(p.weight, g, dim, 1.0f, w);
            Part::vector(p.bias, g, dim, 0.0f, b);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) v[i] = __ffma2_rn(__fmul2_rn(v[i], twice(rstd)), w[i], b[i]);
            Part y;
            y.from(v);
            y.store(static_cast<T *>(p.out) + at, g, dim);
            if (p.stats != nullptr && g == 0) {
                p.stats[2 * static_cast<size_t>(row)] = mean;
                p.stats[2 * static_cast<size_t>(row) + 1] = rstd;
            }
        }
    }
}

constexpr int kWideThreads = 1024;

// Rows of any length: a block per row, three passes over it.
template <typename T>
__global__ void __launch_bounds__(kWideThreads) norm_wide_kernel(const NormArgs p) {
    __shared__ float2 part[2 * (kWideThreads / 32)];
    const float inv = 1.0f / static_cast<float>(p.dim);
    int turn = 0;
    for (unsigned row = blockIdx.x; row < static_cast<unsigned>(p.rows); row += gridDim.x) {
        const size_t at = static_cast<size_t>(row) * p.dim;
        const T *s = static_cast<const T *>(p.x) + at;
        float sum = 0.0f;
        if (p.residual != nullptr) {
            T *const kept = static_cast<T *>(p.sum) + at;
            for (int d = threadIdx.x; d < p.dim; d += kWideThreads) {
                const T v = from_f32<T>(to_f32<T>(s[d]) + to_f32<T>(static_cast<const T *>(p.residual)[at + d]));
                kept[d] = v;
                sum += to_f32<T>(v);
            }
            s = kept;  // (read again only by the thread that wrote it)
        } else {
            for (int d = threadIdx.x; d < p.dim; d += kWideThreads) sum += to_f32<T>(s[d]);
        }
        const float mean = p.rms ? 0.0f : group_sum<kWideThreads>(make_float2(sum, 0.0f), part, turn).x * inv;
        turn ^= 1;
        float sq = 0.0f;
        for (int d = threadIdx.x; d < p.dim; d += kWideThreads) {
            const float v = to_f32<T>(s[d]) - mean;
            sq = fmaf(v, v, sq);
        }
        const float rstd = 1.0f / sqrtf(group_sum<kWideThreads>(make_float2(sq, 0.0f), part, turn).x * inv + p.eps);
        for (int d = threadIdx.x; d < p.dim; d += kWideThreads) {
            const float v = (to_f32<T>(s[d]) - mean) * rstd;
            static_cast<T *>(p.out)[at + d] = from_f32<T>(
                fmaf(v, p.weight != nullptr ? p.weight[d] : 1.0f, p.bias != nullptr ? p.bias[d] : 0.0f));
        }
        if (!p.rms) turn ^= 1;  // (both sums took one)
        if (p.stats != nullptr && threadIdx.x == 0) {
            p.stats[2 * static_cast<size_t>(row)] = mean;
            p.stats[2 * static_cast<size_t>(row) + 1] = rstd;
        }
    }
}

template <typename T, int VE, int kGroup>
cudaError_t launch_group(const NormArgs &a, cudaStream_t stream) {
    constexpr int kThreads = threads_of(kGroup), kRows = kThreads / kGroup;
    const int64_t blocks = (static_cast<int64_t>(a.rows) + kRows - 1) / kRows;
    const int64_t most = static_cast<int64_t>(current_device_sm_count()) * (1024 / kThreads);
    norm_kernel<T, VE, kGroup><<<static_cast<unsigned>(std::min(blocks, most)), kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename T, int VE>
cudaError_t launch_rows(const NormArgs &a, cudaStream_t stream) {
    constexpr int kElems = kRowElems<T, VE>;
    if (a.dim <= 8 * kElems) return launch_group<T, VE, 8>(a, stream);
    if (a.dim <= 32 * kElems) return launch_group<T, VE, 32>(a, stream);
    if (a.dim <= 128 * kElems) return launch_group<T, VE, 128>(a, stream);
    if (a.dim <= 256 * kElems) return launch_group<T, VE, 256>(a, stream);
    if (a.dim <= 512 * kElems) return launch_group<T, VE, 512>(a, stream);
    if (a.dim <= 1024 * kElems) return launch_group<T, VE, 1024>(a, stream);
    norm_wide_kernel<T><<<std::min(a.rows, 2 * current_device_sm_count()), kWideThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_type(const NormArgs &a, cudaStream_t stream) {
    constexpr int kWord = 16 / static_cast<int>(sizeof(T));
    if (a.dim % kWord == 0 && aligned16(a.x) && aligned16(a.residual) && aligned16(a.out) && aligned16(a.sum) &&
        aligned16(a.weight) && aligned16(a.bias))
        return launch_rows<T, kWord>(a, stream);
    return launch_rows<T, 1>(a, stream);
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
