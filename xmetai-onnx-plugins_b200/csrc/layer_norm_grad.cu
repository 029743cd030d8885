// layer_norm_grad.cu -- LayerNormGradFn for sm_100a.
//
// Math, per row with xhat = (x - mean) rstd and g = dy weight:
//   dx = rstd (g - average(g) - xhat average(g xhat)) + d_residual,
// and over the rows d_weight = sum dy xhat, d_bias = sum dy.
//
// Bound by memory: dy, x and d_residual are read once and dx written once. A thread
// keeps the same columns for all rows that its block walks, so the sums over rows stay
// in registers next to the row itself; each block leaves one row of partial sums, which
// column_sum.cu adds in a fixed order. Registers hold 8192 elements of the 16-bit types
// and 4096 of float32 in words or pairs, 1024 singly (odd widths, and tensors or vectors
// off their alignment). Above that pairs and single elements are staged in shared
// memory, up to 8192. What fits neither takes a kernel for dx and one for the columns.
#include <algorithm>

#include "xm_common.cuh"
#include "xm_kernels.h"
#include "xm_rows.cuh"

namespace xm {
namespace {

constexpr int threads_of(int group) { return group < 128 ? 128 : group; }

// A row in the registers of kGroup threads, the next one on its way. 16384 x 4096 in bf16 with d_residual, 537 MB: 94 us,
// 88 % of copy bandwidth. part_w, part_b: [blocks][dim] partial sums of d_weight and d_bias, or null.
template <typename T, int VE, int kGroup>
__global__ void __launch_bounds__(threads_of(kGroup), 512 / threads_of(kGroup)) norm_grad_kernel(const NormGradArgs p, float *part_w,
                                                                                                 float *part_b) {
    constexpr int kThreads = threads_of(kGroup), kRows = kThreads / kGroup;
    using Part = RowPart<T, VE, kGroup>;
    constexpr int kElems = Part::kElems, kPairs = kElems / 2;
    dependents_may_launch();
    __shared__ float2 part[kGroup > 32 ? 2 * (kGroup / 32) : 1];
    __shared__ float2 sums[kRows > 1 ? kThreads * kPairs : 1];
    const int g = threadIdx.x % kGroup, dim = p.dim;
    const float inv = 1.0f / static_cast<float>(dim);
    const unsigned rows = p.rows;
    const unsigned stride = gridDim.x * kRows;
    unsigned row = blockIdx.x * kRows + threadIdx.x / kGroup;
    const T *const DY = static_cast<const T *>(p.dy), *const X = static_cast<const T *>(p.x),
                   *const DR = static_cast<const T *>(p.dres);
    float2 weight[kPairs], sw[kPairs], sb[kPairs];
    Part::vector(p.weight, g, dim, 1.0f, weight);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) sw[i] = sb[i] = twice(0.0f);
    Part next_dy, next_x, next_dr;
    float next_mean = 0.0f, next_rstd = 0.0f;
    next_dy.clear();
    next_x.clear();
    next_dr.clear();
    auto load = [&](unsigned i) {
        if (i >= rows) return;
        next_dy.load(DY + static_cast<size_t>(i) * dim, g, dim);
        next_x.load(X + static_cast<size_t>(i) * dim, g, dim);
        if (DR != nullptr) next_dr.load(DR + static_cast<size_t>(i) * dim, g, dim);
        if (!p.rms) next_mean = p.stats[2 * static_cast<size_t>(i)];
        next_rstd = p.stats[2 * static_cast<size_t>(i) + 1];
    };
    load(row);
    int turn = 0;
    // (all groups of a block make the same number of turns: their sums share barriers or shuffles)
    for (unsigned first = blockIdx.x * kRows; first < rows; first += stride, row += stride, turn ^= 1) {
        const bool there = row < rows;
        // as they are stored: a row's values are unpacked twice rather than held in twice the registers
        const Part dy = next_dy, x = next_x, dr = next_dr;
        const float rstd = next_rstd;
        const float2 mean2 = twice(-next_mean), rstd2 = twice(rstd);
        load(row + stride);
        float2 total = twice(0.0f);
        if (there) {
            float2 sg = twice(0.0f), sx = twice(0.0f), v[kPairs], h[kPairs];
            dy.floats(v);
            x.floats(h);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                h[i] = __fmul2_rn(__fadd2_rn(h[i], mean2), rstd2);
                sw[i] = __ffma2_rn(v[i], h[i], sw[i]);
                sb[i] = __fadd2_rn(sb[i], v[i]);
                v[i] = __fmul2_rn(v[i], weight[i]);
                sg = __fadd2_rn(sg, v[i]);
                sx = __ffma2_rn(v[i], h[i], sx);
            }
            total = make_float2(sg.x + sg.y, sx.x + sx.y);
        }
        total = group_sum<kGroup>(total, part, turn);
        if (there) {
            const float2 ag = twice(p.rms ? 0.0f : -total.x * inv), ax = twice(-total.y * inv);
            float2 v[kPairs], h[kPairs], more[kPairs];
            dy.floats(v);
            x.floats(h);
            dr.floats(more);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                h[i] = __fmul2_rn(__fadd2_rn(h[i], mean2), rstd2);
                v[i] = __ffma2_rn(h[i], ax, __ffma2_rn(v[i], weight[i], ag));
                v[i] = __ffma2_rn(v[i], rstd2, more[i]);
            }
            Part out;
            out.from(v);
            out.store(static_cast<T *>(p.dx) + static_cast<size_t>(row) * dim, g, dim);
        }
    }
    // the block's sums
    auto leave = [&](float *out, float2 (&s)[kPairs]) {
        if constexpr (kRows > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kPairs; ++i) sums[i * kThreads + threadIdx.x] = s[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                s[i] = twice(0.0f);
                for (int r = 0; r < kRows; ++r) s[i] = __fadd2_rn(s[i], sums[i * kThreads + r * kGroup + g]);
            }
        }
        if (threadIdx.x < kGroup) Part::store_vector(out + static_cast<size_t>(blockIdx.x) * dim, g, dim, s);
    };
    if (part_w != nullptr) leave(part_w, sw);
    if (part_b != nullptr) leave(part_b, sb);
}

// Rows in pairs or single elements that registers do not hold: staged some rows ahead, kPer columns to a thread: 16384 x
// 4097 in bf16 with d_residual takes 222 us, 37 % of copy bandwidth; element by element, instructions bound it.
template <typename T, int kThreads, int kPer>
__global__ void __launch_bounds__(kThreads, 512 / kThreads) norm_grad_staged_kernel(const NormGradArgs p, int stages, float *part_w,
                                                                         float *part_b) {
    extern __shared__ float4 smem_f4[];
    __shared__ float2 part[2 * (kThreads / 32)];
    dependents_may_launch();
    const int dim = p.dim;
    const size_t pitch = staged_pitch<T>(dim);
    T *const ring = reinterpret_cast<T *>(smem_f4);  // [stages][dy, x, d_residual][pitch]
    const T *const DY = static_cast<const T *>(p.dy), *const X = static_cast<const T *>(p.x),
                   *const DR = static_cast<const T *>(p.dres);
    const float inv = 1.0f / static_cast<float>(dim);
    float weight[kPer], sw[kPer], sb[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int d = threadIdx.x + k * kThreads;
        weight[k] = p.weight != nullptr && d < dim ? p.weight[d] : 1.0f;
        sw[k] = sb[k] = 0.0f;
    }
    auto copy = [&](long long row, int stage) {
        if (row < p.rows) {
            const unsigned i = static_cast<unsigned>(row);
            stage_row<kThreads>(ring + 3 * stage * pitch, DY, i, p.rows, dim);
            stage_row<kThreads>(ring + (3 * stage + 1) * pitch, X, i, p.rows, dim);
            if (DR != nullptr) stage_row<kThreads>(ring + (3 * stage + 2) * pitch, DR, i, p.rows, dim);
        }
        cp_async_commit();
    };
    for (int k = 0; k < stages - 1; ++k) copy(blockIdx.x + static_cast<long long>(k) * gridDim.x, k);
    int turn = 0, stage = 0;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        // (all but the last stages - 2 copies are here; two or three stages)
        if (stages == 2) cp_async_wait<0>();
        else cp_async_wait<1>();
        __syncthreads();
        copy(row + static_cast<long long>(stages - 1) * gridDim.x, stage == 0 ? stages - 1 : stage - 1);
        const unsigned i = static_cast<unsigned>(row);
        const T *const dy = ring + 3 * stage * pitch + staged_shift(DY, i, dim),
                       *const x = ring + (3 * stage + 1) * pitch + staged_shift(X, i, dim),
                       *const dr = ring + (3 * stage + 2) * pitch + (DR != nullptr ? staged_shift(DR, i, dim) : 0);
        const float mean = p.rms ? 0.0f : p.stats[2 * static_cast<size_t>(row)];
        const float rstd = p.stats[2 * static_cast<size_t>(row) + 1];
        float2 total = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int d = threadIdx.x + k * kThreads;
            if (d < dim) {
                const float v = to_f32<T>(dy[d]), h = (to_f32<T>(x[d]) - mean) * rstd;
                sw[k] = fmaf(v, h, sw[k]);
                sb[k] += v;
                const float gr = v * weight[k];
                total.x += gr;
                total.y = fmaf(gr, h, total.y);
            }
        }
        total = group_sum<kThreads>(total, part, turn);
        const float ag = p.rms ? 0.0f : total.x * inv, ax = total.y * inv;
        T *const out = static_cast<T *>(p.dx) + static_cast<size_t>(row) * dim;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int d = threadIdx.x + k * kThreads;
            if (d < dim) {
                const float h = (to_f32<T>(x[d]) - mean) * rstd;
                out[d] = from_f32<T>(
                    fmaf(rstd, to_f32<T>(dy[d]) * weight[k] - ag - h * ax, DR != nullptr ? to_f32<T>(dr[d]) : 0.0f));
            }
        }
        stage = stage + 1 == stages ? 0 : stage + 1;
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int d = threadIdx.x + k * kThreads;
        if (d < dim) {
            if (part_w != nullptr) part_w[static_cast<size_t>(blockIdx.x) * dim + d] = sw[k];
            if (part_b != nullptr) part_b[static_cast<size_t>(blockIdx.x) * dim + d] = sb[k];
        }
    }
}

constexpr int kWideThreads = 1024;

// Rows of any length: a block per row, two passes over it, an element a load; the columns' kernel reads dy and x once more.
// Together 8192 x 12288 in bf16 with d_residual, 805 MB: 898 us, 14 % of copy bandwidth.
template <typename T>
__global__ void __launch_bounds__(kWideThreads) norm_grad_wide_kernel(const NormGradArgs p) {
    __shared__ float2 part[2 * (kWideThreads / 32)];
    const float inv = 1.0f / static_cast<float>(p.dim);
    int turn = 0;
    for (unsigned row = blockIdx.x; row < static_cast<unsigned>(p.rows); row += gridDim.x, turn ^= 1) {
        const size_t at = static_cast<size_t>(row) * p.dim;
        const float mean = p.rms ? 0.0f : p.stats[2 * static_cast<size_t>(row)];
        const float rstd = p.stats[2 * static_cast<size_t>(row) + 1];
        float2 sum = make_float2(0.0f, 0.0f);
        for (int d = threadIdx.x; d < p.dim; d += kWideThreads) {
            const float g = to_f32<T>(static_cast<const T *>(p.dy)[at + d]) * (p.weight != nullptr ? p.weight[d] : 1.0f);
            sum.x += g;
            sum.y = fmaf(g, (to_f32<T>(static_cast<const T *>(p.x)[at + d]) - mean) * rstd, sum.y);
        }
        sum = group_sum<kWideThreads>(sum, part, turn);
        const float ag = p.rms ? 0.0f : sum.x * inv, ax = sum.y * inv;
        for (int d = threadIdx.x; d < p.dim; d += kWideThreads) {
            const float g = to_f32<T>(static_cast<const T *>(p.dy)[at + d]) * (p.weight != nullptr ? p.weight[d] : 1.0f);
            const float xhat = (to_f32<T>(static_cast<const T *>(p.x)[at + d]) - mean) * rstd;
            const float more = p.dres != nullptr ? to_f32<T>(static_cast<const T *>(p.dres)[at + d]) : 0.0f;
            static_cast<T *>(p.dx)[at + d] = from_f32<T>(fmaf(rstd, g - ag - xhat * ax, more));
        }
    }
}

constexpr int kColThreads = 256;

// Partial sums of a block of columns over a range of rows.
template <typename T>
__global__ void __launch_bounds__(kColThreads) norm_grad_columns_kernel(const NormGradArgs p, float *part_w, float *part_b) {
    const int d = blockIdx.x * kColThreads + threadIdx.x;
    if (d >= p.dim) return;
    float sw = 0.0f, sb = 0.0f;
    for (unsigned row = blockIdx.y; row < static_cast<unsigned>(p.rows); row += gridDim.y) {
        const size_t at = static_cast<size_t>(row) * p.dim + d;
        const float dy = to_f32<T>(static_cast<const T *>(p.dy)[at]);
        const float mean = p.rms ? 0.0f : p.stats[2 * static_cast<size_t>(row)];
        sw = fmaf(dy, (to_f32<T>(static_cast<const T *>(p.x)[at]) - mean) * p.stats[2 * static_cast<size_t>(row) + 1], sw);
        sb += dy;
    }
    if (part_w != nullptr) part_w[static_cast<size_t>(blockIdx.y) * p.dim + d] = sw;
    if (part_b != nullptr) part_b[static_cast<size_t>(blockIdx.y) * p.dim + d] = sb;
}

constexpr int kStagedMax = 16 * 512;  // longest staged row

// Threads per row held in registers; -1: staged, 0: neither fits.
template <typename T, int VE>
int group_of(int dim) {
    if (dim <= 8 * kRowElems<T, VE, 8>) return 8;
    if (dim <= 16 * kRowElems<T, VE, 16>) return 16;
    if (dim <= 32 * kRowElems<T, VE, 32>) return 32;
    if (dim <= 128 * kRowElems<T, VE, 128>) return 128;
    if (VE > 1 && dim <= 256 * kRowElems<T, VE, 256>) return 256;
    if (VE > 1 && dim <= 512 * kRowElems<T, VE, 512>) return 512;
    return VE <= 2 && dim <= kStagedMax && 2 * 3 * staged_pitch<T>(dim) * sizeof(T) <= kStagedBytes ? -1 : 0;
}

// Stages of a staged row, and blocks of an SM.
template <typename T>
int stages_of(int dim, int *blocks) {
    const size_t row = 3 * staged_pitch<T>(dim) * sizeof(T);
    const int stages = 3 * row <= kStagedBytes / 2 ? 3 : 2;
    *blocks = static_cast<int>(std::min<size_t>(kStagedBytes / (stages * row), 512 / staged_threads(dim)));
    return stages;
}

// Blocks that leave partial sums: as many as are resident, fewer for few rows.
template <typename T, int VE>
int parts_of(const NormGradArgs &a) {
    const int group = group_of<T, VE>(a.dim), sms = current_device_sm_count();
    if (group == 0) {
        const int tiles = (a.dim + kColThreads - 1) / kColThreads;
        return std::max(1, std::min(a.rows, (8 * sms + tiles - 1) / tiles));
    }
    if (group < 0) {
        int blocks = 1;
        stages_of<T>(a.dim, &blocks);
        return std::max(1, std::min(a.rows, sms * blocks));
    }
    const int threads = threads_of(group), rows = threads / group;
    return std::max(1, std::min((a.rows + rows - 1) / rows, sms * (512 / threads)));
}
int parts_of(const NormGradArgs &a, int unit) {
    if (a.io == IoType::kF32) return unit > 2 ? parts_of<float, 4>(a) : unit == 2 ? parts_of<float, 2>(a) : parts_of<float, 1>(a);
    return unit > 2 ? parts_of<__half, 8>(a) : unit == 2 ? parts_of<__half, 2>(a) : parts_of<__half, 1>(a);
}

template <typename T, int kThreads, int kPer>
void launch_staged(const NormGradArgs &a, int parts, float *part_w, float *part_b, cudaStream_t stream) {
    int blocks = 1;
    const int stages = stages_of<T>(a.dim, &blocks);
    if (prepare_staged<norm_grad_staged_kernel<T, kThreads, kPer>>() != cudaSuccess) return;  // (the last error says so)
    norm_grad_staged_kernel<T, kThreads, kPer>
        <<<parts, kThreads, stages * 3 * staged_pitch<T>(a.dim) * sizeof(T), stream>>>(a, stages, part_w, part_b);
}

template <typename T, int VE, int kGroup>
void launch_group(const NormGradArgs &a, int parts, float *part_w, float *part_b, cudaStream_t stream) {
    norm_grad_kernel<T, VE, kGroup><<<parts, threads_of(kGroup), 0, stream>>>(a, part_w, part_b);
}

template <typename T, int VE>
void launch_rows(const NormGradArgs &a, int parts, float *part_w, float *part_b, cudaStream_t stream) {
    switch (group_of<T, VE>(a.dim)) {
        case 8: return launch_group<T, VE, 8>(a, parts, part_w, part_b, stream);
        case 16: return launch_group<T, VE, 16>(a, parts, part_w, part_b, stream);
        case 32: return launch_group<T, VE, 32>(a, parts, part_w, part_b, stream);
        case 128: return launch_group<T, VE, 128>(a, parts, part_w, part_b, stream);
    }
    if constexpr (VE > 1) {
        if (group_of<T, VE>(a.dim) == 256) return launch_group<T, VE, 256>(a, parts, part_w, part_b, stream);
        if (group_of<T, VE>(a.dim) == 512) return launch_group<T, VE, 512>(a, parts, part_w, part_b, stream);
    }
    if constexpr (VE <= 2) {
        if (group_of<T, VE>(a.dim) < 0) {
            if (staged_threads(a.dim) == 128) return launch_staged<T, 128, 16>(a, parts, part_w, part_b, stream);
            if (staged_threads(a.dim) == 256) return launch_staged<T, 256, 20>(a, parts, part_w, part_b, stream);
            return launch_staged<T, 512, 16>(a, parts, part_w, part_b, stream);
        }
    }
    if (a.rows > 0)
        norm_grad_wide_kernel<T><<<std::min(a.rows, 2 * current_device_sm_count()), kWideThreads, 0, stream>>>(a);
    if (part_w != nullptr || part_b != nullptr)
        norm_grad_columns_kernel<T><<<dim3((a.dim + kColThreads - 1) / kColThreads, parts), kColThreads, 0, stream>>>(
            a, part_w, part_b);
}

template <typename T>
void launch_type(const NormGradArgs &a, int unit, int parts, float *part_w, float *part_b, cudaStream_t stream) {
    if (unit > 2) launch_rows<T, 16 / static_cast<int>(sizeof(T))>(a, parts, part_w, part_b, stream);
    else if (unit == 2) launch_rows<T, 2>(a, parts, part_w, part_b, stream);
    else launch_rows<T, 1>(a, parts, part_w, part_b, stream);
}

}  // namespace

// (The partial sums' number depends on alignment; the largest.)
size_t layer_norm_grad_workspace(const NormGradArgs &a) {
    const int sums = (a.weight != nullptr) + a.want_dbias, parts = std::max({parts_of(a, 1), parts_of(a, 2), parts_of(a, 16)});
    // rows of the two sums begin on 16-byte words
    return parts > 1 ? static_cast<size_t>(sums) * ((static_cast<size_t>(parts) * a.dim + 3) / 4 * 4) * sizeof(float) : 0;
}

cudaError_t launch_layer_norm_grad(const NormGradArgs &a, void *workspace, cudaStream_t stream) {
    const size_t size = a.io == IoType::kF32 ? 4 : 2;
    int unit = row_unit(a.dim, size, {a.dy, a.x, a.dres, a.dx}, {a.weight});
    if (parts_of(a, unit) == 1) unit = row_unit(a.dim, size, {a.dy, a.x, a.dres, a.dx}, {a.weight, a.dweight, a.dbias});
    const int parts = parts_of(a, unit);
    float *part_w = a.dweight, *part_b = a.dbias;
    if (parts > 1) {
        float *next = static_cast<float *>(workspace);
        if (part_w != nullptr) part_w = next, next += (static_cast<size_t>(parts) * a.dim + 3) / 4 * 4;
        if (part_b != nullptr) part_b = next;
    }
    switch (a.io) {
        case IoType::kBF16: launch_type<__nv_bfloat16>(a, unit, parts, part_w, part_b, stream); break;
        case IoType::kF16: launch_type<__half>(a, unit, parts, part_w, part_b, stream); break;
        default: launch_type<float>(a, unit, parts, part_w, part_b, stream);
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || parts == 1 || (part_w == nullptr && part_b == nullptr)) return e;
    if (part_w == nullptr) return launch_column_sums(part_b, nullptr, parts, a.dim, a.dbias, nullptr, stream);
    return launch_column_sums(part_w, part_b, parts, a.dim, a.dweight, a.dbias, stream);
}

}  // namespace xm
