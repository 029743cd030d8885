// xm_rows.cuh -- rows held in registers by a group of threads, for layer norm and its
// backward pass.
//
// A group of kGroup threads owns a row: thread g has the chunks g, g + kGroup, ... of
// VE consecutive elements. VE is a 16-byte word where rows and tensors are aligned to
// words, two elements where they are aligned to those, else one element (still
// consecutive over the threads).
#pragma once

#include <initializer_list>

#include "xm_common.cuh"

namespace xm {

// Elements of a row that a thread holds: two words of each tensor (one in groups of up to 16, whose rows are short), or
// eight single elements.
template <typename T, int VE, int kGroup>
constexpr int kRowElems = VE == 1 ? 8 : (kGroup <= 16 ? 16 : 32) / static_cast<int>(sizeof(T));

// VE of rows of dim elements of `size` bytes, and of vectors of floats beside them.
inline int row_unit(int dim, size_t size, std::initializer_list<const void *> tensors,
                    std::initializer_list<const void *> vectors) {
    uintptr_t rows = static_cast<uintptr_t>(dim) * size, floats = 0;
    for (const void *p : tensors) rows |= reinterpret_cast<uintptr_t>(p);
    for (const void *p : vectors) floats |= reinterpret_cast<uintptr_t>(p);
    if ((rows | floats) % 16 == 0) return 16 / static_cast<int>(size);
    return rows % (2 * size) == 0 && floats % 8 == 0 ? 2 : 1;
}

template <typename T, int VE>
struct Chunk;  // VE elements as they are stored
template <>
struct Chunk<float, 4> {
    float4 w;
};
template <typename T>
struct Chunk<T, 8> {
    uint4 w;
};
template <>
struct Chunk<float, 2> {
    float2 w;
};
template <typename T>
struct Chunk<T, 2> {
    uint32_t w;
};
template <typename T>
struct Chunk<T, 1> {
    T w;
};

template <typename T, int VE>
__device__ __forceinline__ void chunk_floats(const Chunk<T, VE> &c, float *v) {
    if constexpr (VE == 1) {
        v[0] = to_f32<T>(c.w);
    } else if constexpr (VE == 2) {
        float2 f;
        if constexpr (sizeof(T) == 4) f = c.w;
        else f = unpack2<T>(c.w);
        v[0] = f.x; v[1] = f.y;
    } else if constexpr (VE == 4) {
        v[0] = c.w.x; v[1] = c.w.y; v[2] = c.w.z; v[3] = c.w.w;
    } else {
        const uint32_t w[4] = {c.w.x, c.w.y, c.w.z, c.w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}
template <typename T, int VE>
__device__ __forceinline__ Chunk<T, VE> to_chunk(const float *v) {
    Chunk<T, VE> c;
    if constexpr (VE == 1) c.w = from_f32<T>(v[0]);
    else if constexpr (VE == 2 && sizeof(T) == 4) c.w = make_float2(v[0], v[1]);
    else if constexpr (VE == 2) c.w = pack2<T>(v[0], v[1]);
    else if constexpr (VE == 4) c.w = make_float4(v[0], v[1], v[2], v[3]);
    else c.w = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    return c;
}

// VE consecutive floats (aligned to words, or pairs, where VE > 1).
template <int VE>
__device__ __forceinline__ void load_row_floats(const float *p, float *v) {
    if constexpr (VE == 1) {
        v[0] = __ldg(p);
    } else if constexpr (VE == 2) {
        const float2 w = __ldg(reinterpret_cast<const float2 *>(p));
        v[0] = w.x; v[1] = w.y;
    } else {
#pragma unroll
        for (int i = 0; i < VE; i += 4) {
            const float4 w = __ldg(reinterpret_cast<const float4 *>(p + i));
            v[i] = w.x; v[i + 1] = w.y; v[i + 2] = w.z; v[i + 3] = w.w;
        }
    }
}
template <int VE>
__device__ __forceinline__ void store_row_floats(float *p, const float *v) {
    if constexpr (VE == 1) {
        p[0] = v[0];
    } else if constexpr (VE == 2) {
        *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
    } else {
#pragma unroll
        for (int i = 0; i < VE; i += 4) *reinterpret_cast<float4 *>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    }
}

// A row's chunks of one thread, as they are stored; zeros behind its end.
template <typename T, int VE, int kGroup>
struct RowPart {
    static constexpr int kElems = kRowElems<T, VE, kGroup>, kChunks = kElems / VE;
    Chunk<T, VE> c[kChunks];
    __device__ __forceinline__ static int at(int k, int g) { return (k * kGroup + g) * VE; }
    __device__ __forceinline__ void clear() {
        const float zero[VE] = {};
#pragma unroll
        for (int k = 0; k < kChunks; ++k) c[k] = to_chunk<T, VE>(zero);
    }
    __device__ __forceinline__ void load(const T *row, int g, int dim) {
#pragma unroll
        for (int k = 0; k < kChunks; ++k)
            if (at(k, g) < dim) c[k] = *reinterpret_cast<const Chunk<T, VE> *>(row + at(k, g));
    }
    // the elements in pairs
    __device__ __forceinline__ void floats(float2 (&v)[kElems / 2]) const {
        float w[kElems];
#pragma unroll
        for (int k = 0; k < kChunks; ++k) chunk_floats<T, VE>(c[k], w + k * VE);
#pragma unroll
        for (int i = 0; i < kElems / 2; ++i) v[i] = make_float2(w[2 * i], w[2 * i + 1]);
    }
    __device__ __forceinline__ void from(const float2 (&v)[kElems / 2]) {
        float w[kElems];
#pragma unroll
        for (int i = 0; i < kElems / 2; ++i) w[2 * i] = v[i].x, w[2 * i + 1] = v[i].y;
#pragma unroll
        for (int k = 0; k < kChunks; ++k) c[k] = to_chunk<T, VE>(w + k * VE);
    }
    __device__ __forceinline__ void store(T *row, int g, int dim) const {
#pragma unroll
        for (int k = 0; k < kChunks; ++k)
            if (at(k, g) < dim) *reinterpret_cast<Chunk<T, VE> *>(row + at(k, g)) = c[k];
    }
    // a thread's elements of a vector of floats; `absent` behind the row's end and where there is no vector
    __device__ __forceinline__ static void vector(const float *p, int g, int dim, float absent, float2 (&v)[kElems / 2]) {
        float w[kElems];
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
#pragma unroll
            for (int i = 0; i < VE; ++i) w[k * VE + i] = absent;
            if (p != nullptr && at(k, g) < dim) load_row_floats<VE>(p + at(k, g), w + k * VE);
        }
#pragma unroll
        for (int i = 0; i < kElems / 2; ++i) v[i] = make_float2(w[2 * i], w[2 * i + 1]);
    }
    __device__ __forceinline__ static void store_vector(float *p, int g, int dim, const float2 (&v)[kElems / 2]) {
        float w[kElems];
#pragma unroll
        for (int i = 0; i < kElems / 2; ++i) w[2 * i] = v[i].x, w[2 * i + 1] = v[i].y;
#pragma unroll
        for (int k = 0; k < kChunks; ++k)
            if (at(k, g) < dim) store_row_floats<VE>(p + at(k, g), w + k * VE);
    }
    // whether the i-th element is in the row
    __device__ __forceinline__ static bool inside(int i, int g, int dim) { return at(i / VE, g) < dim; }
};

__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }

// Rows that are too long for registers in pairs or single elements, staged in shared memory: asynchronous copies of 16-byte
// words, from the one that holds a row's first element, behind up to a word's others. Elements are read from there by
// consecutive threads, eight to twenty to each up to 8192: fewer leave most of a row's time to its barriers (32768 x 1027 in
// bf16: 95 us, and 230 with 512 threads; backward 147 and 406), more too few warps.
constexpr int staged_threads(int dim) { return dim <= 2048 ? 128 : dim <= 5120 ? 256 : 512; }

template <typename T>
constexpr int kStagedWord = 16 / static_cast<int>(sizeof(T));
template <typename T>
__host__ __device__ constexpr size_t staged_pitch(int dim) {  // elements of a staged row, in whole words
    constexpr size_t kWord = kStagedWord<T>;
    return (static_cast<size_t>(dim) + 2 * kWord - 2) / kWord * kWord;
}
constexpr size_t kStagedBytes = 220 * 1024;  // of shared memory on an SM
template <auto kKernel>
cudaError_t prepare_staged() { return allow_shared<kKernel>(kStagedBytes); }
// Where row `row` of a tensor begins in its stage.
template <typename T>
__device__ __forceinline__ int staged_shift(const T *src, unsigned row, int dim) {
    const unsigned first = static_cast<unsigned>(reinterpret_cast<uintptr_t>(src) / sizeof(T));
    return static_cast<int>((first + row * static_cast<unsigned>(dim)) % kStagedWord<T>);
}
// Copies a row of a tensor of `rows` rows, and reads nothing outside of it.
template <int kThreads, typename T>
__device__ __forceinline__ void stage_row(T *dst, const T *src, unsigned row, unsigned rows, int dim) {
    constexpr int kWord = kStagedWord<T>;
    const int shift = staged_shift(src, row, dim);
    const T *const first = src + static_cast<size_t>(row) * dim;
    for (int i = static_cast<int>(threadIdx.x) * kWord - shift; i < dim; i += kThreads * kWord) {
        const bool begin = row == 0 && i < 0, end = row + 1 == rows && dim - i < kWord;
        if (!begin && !end) {
            cp_async16(dst + shift + i, first + i, 16);
        } else {  // the words in which the tensor begins and ends
            for (int k = max(i, 0); k < min(i + kWord, dim); ++k) dst[shift + k] = first[k];
        }
    }
}

// Sums of two values over a group, the same in all its threads and whatever the number of rows. `part`: shared memory
// of 2 x (kGroup / 32) pairs, used in turn (`turn` alternates), so that one barrier is enough.
template <int kGroup>
__device__ __forceinline__ float2 group_sum(float2 v, float2 *part, int turn) {
#pragma unroll
    for (int o = (kGroup < 32 ? kGroup : 32) / 2; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(kFullMask, v.x, o);
        v.y += __shfl_xor_sync(kFullMask, v.y, o);
    }
    if constexpr (kGroup > 32) {
        constexpr int kWarps = kGroup / 32;
        float2 *const p = part + turn * kWarps;
        if ((threadIdx.x & 31) == 0) p[threadIdx.x >> 5] = v;
        __syncthreads();
        v = p[threadIdx.x & (kWarps - 1)];
#pragma unroll
        for (int o = kWarps / 2; o > 0; o >>= 1) {
            v.x += __shfl_xor_sync(kFullMask, v.x, o);
            v.y += __shfl_xor_sync(kFullMask, v.y, o);
        }
    }
    return v;
}

}  // namespace xm
