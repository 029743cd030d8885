// layer_norm.cu -- LayerNormFn for sm_100a.
//
// Math, per row: s = x + residual (rounded to the I/O type, as it is stored), mean =
// average(s) or 0, rstd = 1 / sqrt(average((s - mean)^2) + eps), y = (s - mean) rstd
// weight + bias.
//
// Bound by memory: x and the residual are read once and y and s written once. A row
// stays in the registers of its group of threads between the sum, the squares and the
// output, so it is not read again. Registers hold 16384 elements of the 16-bit types
// and 8192 of float32 in words, 8192 in pairs, 1024 singly (odd widths, and tensors or
// vectors off their alignment). Above that pairs and single elements are staged in
// shared memory, up to some 28000 of the 16-bit types and 14000 of float32. What fits
// neither is read again, from the caches.
#include <algorithm>

#include "xm_common.cuh"
#include "xm_kernels.h"
#include "xm_rows.cuh"

namespace xm {
namespace {

constexpr int threads_of(int group) { return group < 128 ? 128 : group; }

// Threads of an SM: pairs of 16-bit elements take more registers than 64 (16384 x 4098: 206 us with 1024).
template <typename T, int VE>
constexpr int kThreadsSm = VE == 2 && sizeof(T) == 2 ? 512 : 1024;

// A row in the registers of kGroup threads, the next one on its way. 16384 x 4096 in bf16 with a residual, 537 MB: 89 us,
// 92 % of copy bandwidth.
template <typename T, int VE, int kGroup>
__global__ void __launch_bounds__(threads_of(kGroup), kThreadsSm<T, VE> / threads_of(kGroup)) norm_kernel(const NormArgs p) {
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

// Rows in pairs or single elements that registers do not hold: staged some rows ahead, and read from shared memory for
// every pass: 16384 x 4097 in bf16 with a residual takes 163 us, 50 % of copy bandwidth (247 in registers, an element a load).
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 1536 / kThreads) norm_staged_kernel(const NormArgs p, int stages) {
    extern __shared__ float4 smem_f4[];
    __shared__ float2 part[2 * (kThreads / 32)];
    const int dim = p.dim;
    const size_t pitch = staged_pitch<T>(dim);
    const T *const X = static_cast<const T *>(p.x), *const R = static_cast<const T *>(p.residual);
    T *const ring = reinterpret_cast<T *>(smem_f4);  // [stages][x, residual where there is one][pitch]
    const size_t tensors = R != nullptr ? 2 : 1;
    const float inv = 1.0f / static_cast<float>(dim);
    auto copy = [&](long long row, int stage) {
        if (row < p.rows) {
            stage_row<kThreads>(ring + tensors * stage * pitch, X, static_cast<unsigned>(row), p.rows, dim);
            if (R != nullptr) stage_row<kThreads>(ring + (2 * stage + 1) * pitch, R, static_cast<unsigned>(row), p.rows, dim);
        }
        cp_async_commit();
    };
    for (int k = 0; k < stages - 1; ++k) copy(blockIdx.x + static_cast<long long>(k) * gridDim.x, k);
    int turn = 0, stage = 0;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        // (all but the last stages - 2 copies are here; two or three stages)
        if (stages == 2) cp_async_wait<0>();
        else cp_async_wait<1>();
        __syncthreads();
        copy(row + static_cast<long long>(stages - 1) * gridDim.x, stage == 0 ? stages - 1 : stage - 1);
        T *const s = ring + tensors * stage * pitch + staged_shift(X, static_cast<unsigned>(row), dim);
        const T *const r = ring + (2 * stage + 1) * pitch + (R != nullptr ? staged_shift(R, static_cast<unsigned>(row), dim) : 0);
        const size_t at = static_cast<size_t>(row) * dim;
        // (an element is read again only by the thread that wrote it)
        float sum = 0.0f;
        if (R != nullptr) {
            T *const kept = static_cast<T *>(p.sum) + at;
#pragma unroll 8
            for (int d = threadIdx.x; d < dim; d += kThreads) {
                const T v = from_f32<T>(to_f32<T>(s[d]) + to_f32<T>(r[d]));
                kept[d] = v;
                s[d] = v;
                sum += to_f32<T>(v);
            }
        } else if (!p.rms) {
#pragma unroll 8
            for (int d = threadIdx.x; d < dim; d += kThreads) sum += to_f32<T>(s[d]);
        }
        float mean = 0.0f;
        if (!p.rms) {
            mean = group_sum<kThreads>(make_float2(sum, 0.0f), part, turn).x * inv;
            turn ^= 1;
        }
        float sq = 0.0f;
#pragma unroll 8
        for (int d = threadIdx.x; d < dim; d += kThreads) {
            const float v = to_f32<T>(s[d]) - mean;
            sq = fmaf(v, v, sq);
        }
        const float rstd = 1.0f / sqrtf(group_sum<kThreads>(make_float2(sq, 0.0f), part, turn).x * inv + p.eps);
        turn ^= 1;
        T *const out = static_cast<T *>(p.out) + at;
#pragma unroll 8
        for (int d = threadIdx.x; d < dim; d += kThreads) {
            const float v = (to_f32<T>(s[d]) - mean) * rstd;
            out[d] = from_f32<T>(
                fmaf(v, p.weight != nullptr ? __ldg(p.weight + d) : 1.0f, p.bias != nullptr ? __ldg(p.bias + d) : 0.0f));
        }
        if (p.stats != nullptr && threadIdx.x == 0) {
            p.stats[2 * static_cast<size_t>(row)] = mean;
            p.stats[2 * static_cast<size_t>(row) + 1] = rstd;
        }
        stage = stage + 1 == stages ? 0 : stage + 1;
    }
}

constexpr int kWideThreads = 1024;

// Rows of any length: a block per row, three passes over it, of which the caches serve two. 4096 x 20480 in bf16 with a
// residual, 671 MB: 281 us, 37 % of copy bandwidth; element by element, instructions bound it.
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
    const int64_t most = static_cast<int64_t>(current_device_sm_count()) * (kThreadsSm<T, VE> / kThreads);
    norm_kernel<T, VE, kGroup><<<static_cast<unsigned>(std::min(blocks, most)), kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename T, int kThreads>
cudaError_t launch_staged(const NormArgs &a, cudaStream_t stream) {
    const size_t row = (a.residual != nullptr ? 2 : 1) * staged_pitch<T>(a.dim) * sizeof(T);
    const int stages = 3 * row <= kStagedBytes / 2 ? 3 : 2;
    const size_t smem = stages * row;
    const cudaError_t e = prepare_staged<norm_staged_kernel<T, kThreads>>();
    if (e != cudaSuccess) return e;
    const int64_t most = static_cast<int64_t>(current_device_sm_count()) *
                         std::min<int64_t>(kStagedBytes / smem, 1536 / kThreads);
    norm_staged_kernel<T, kThreads><<<static_cast<unsigned>(std::min<int64_t>(a.rows, most)), kThreads, smem, stream>>>(
        a, stages);
    return cudaGetLastError();
}

template <typename T, int VE>
cudaError_t launch_rows(const NormArgs &a, cudaStream_t stream) {
    if (a.dim <= 8 * kRowElems<T, VE, 8>) return launch_group<T, VE, 8>(a, stream);
    if (a.dim <= 16 * kRowElems<T, VE, 16>) return launch_group<T, VE, 16>(a, stream);
    if (a.dim <= 32 * kRowElems<T, VE, 32>) return launch_group<T, VE, 32>(a, stream);
    if (a.dim <= 128 * kRowElems<T, VE, 128>) return launch_group<T, VE, 128>(a, stream);
    if constexpr (VE > 1) {
        if (a.dim <= 256 * kRowElems<T, VE, 256>) return launch_group<T, VE, 256>(a, stream);
        if (a.dim <= 512 * kRowElems<T, VE, 512>) return launch_group<T, VE, 512>(a, stream);
    }
    if constexpr (kThreadsSm<T, VE> == 1024 && VE > 1) {
        if (a.dim <= 1024 * kRowElems<T, VE, 1024>) return launch_group<T, VE, 1024>(a, stream);
    }
    if constexpr (VE <= 2) {
        if (2 * 2 * staged_pitch<T>(a.dim) * sizeof(T) <= kStagedBytes) {
            if (staged_threads(a.dim) == 128) return launch_staged<T, 128>(a, stream);
            if (staged_threads(a.dim) == 256) return launch_staged<T, 256>(a, stream);
            return launch_staged<T, 512>(a, stream);
        }
    }
    norm_wide_kernel<T><<<std::min(a.rows, 2 * current_device_sm_count()), kWideThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_type(const NormArgs &a, cudaStream_t stream) {
    constexpr int kWord = 16 / static_cast<int>(sizeof(T));
    switch (row_unit(a.dim, sizeof(T), {a.x, a.residual, a.out, a.sum}, {a.weight, a.bias})) {
        case kWord: return launch_rows<T, kWord>(a, stream);
        case 2: return launch_rows<T, 2>(a, stream);
        default: return launch_rows<T, 1>(a, stream);
    }
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
