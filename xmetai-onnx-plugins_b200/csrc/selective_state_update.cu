// selective_state_update.cu -- SelectiveStateUpdateFn for sm_100a.
//
// Math, per sequence and channel d (state n = 0 .. N - 1):
//   dt = softplus?(delta + bias), h_n = exp(dt A_n) h_n + dt u B_n,
//   y = (D u + sum_n C_n h_n) silu(z).
//
// Bound by memory: the state is read and written once, 8 bytes per (sequence,
// channel, state). A channel belongs to kLanes adjacent lanes with four
// consecutive states each (eight for N > 128), so a warp's state accesses are
// whole 16-byte words of consecutive memory. Where there are sequences enough, a
// thread takes kRows of them for the same channel: their loads are issued
// together, A is read once for all, and what is done once per (sequence, channel)
// -- loading delta, u and z, softplus, skip, gate and store -- falls to one lane
// of the kRows that share the channel; dt and dt u reach the others by shuffles,
// and the sums over states are scattered to their owners as they are reduced.
// (With every lane doing that work for every sequence the kernel issued 224
// instructions per warp and sequence and took 62 us for 256 sequences x 4096
// channels x 16 states.)
#include <algorithm>

#include "xm_common.cuh"
#include "xm_kernels.h"
#include "xm_sequences.cuh"

namespace xm {
namespace {

constexpr int kUpdThreads = 128;

// A lane's four values of a group: one word of consecutive ones (vec), or every
// `step`-th, so that neighbouring lanes still read neighbouring memory. The first
// `left` of them are below N; the others read zero and are not stored. kStream: as
// data that leaves the caches first. Large batches use it: their states pass
// through once per step, and keeping them would only push out A, B and C and
// delay the stores (256 sequences x 4096 channels x 16 states: 27.0 us against
// 31.6, 512 x 2048 x 64: 98 us against 114). Small ones may find their states in
// L2 at the next step.
template <bool kStream>
__device__ __forceinline__ float4 load_states(const float *p, int left, bool vec, int step) {
    if (vec) {
        if (left <= 0) return make_float4(0, 0, 0, 0);
        return kStream ? __ldcs(reinterpret_cast<const float4 *>(p)) : *reinterpret_cast<const float4 *>(p);
    }
    return make_float4(left > 0 ? p[0] : 0.0f, left > 1 ? p[step] : 0.0f, left > 2 ? p[2 * step] : 0.0f,
                       left > 3 ? p[3 * step] : 0.0f);
}

template <bool kStream>
__device__ __forceinline__ void store_states(float *p, int left, bool vec, int step, const float4 &v) {
    if (vec) {
        if (left <= 0) return;
        if (kStream) __stcs(reinterpret_cast<float4 *>(p), v);
        else *reinterpret_cast<float4 *>(p) = v;
        return;
    }
    if (left > 0) p[0] = v.x;
    if (left > 1) p[step] = v.y;
    if (left > 2) p[2 * step] = v.z;
    if (left > 3) p[3 * step] = v.w;
}

// The same for values of the I/O type.
template <typename T>
__device__ __forceinline__ float4 load_io4(const T *p, int left, bool vec, int step) {
    if (vec) {
        if (left <= 0) return make_float4(0, 0, 0, 0);
        if constexpr (sizeof(T) == 4) {
            return __ldg(reinterpret_cast<const float4 *>(p));
        } else {
            const uint2 w = __ldg(reinterpret_cast<const uint2 *>(p));
            const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
            return make_float4(a.x, a.y, b.x, b.y);
        }
    }
    return make_float4(left > 0 ? to_f32<T>(p[0]) : 0.0f, left > 1 ? to_f32<T>(p[step]) : 0.0f,
                       left > 2 ? to_f32<T>(p[2 * step]) : 0.0f, left > 3 ? to_f32<T>(p[3 * step]) : 0.0f);
}

// kFull: N = 4 kLanes kQuads and every access in words.
template <typename T, int kLanes, int kQuads, int kRows, bool kFull>
__global__ void __launch_bounds__(kUpdThreads) state_token_kernel(const ScanArgs p, bool words) {
    static_assert(kRows == 1 || kRows == 2 || (kRows == 4 && kLanes >= 4), "one lane per sequence");
    constexpr int kChannels = kUpdThreads / kLanes;
    const bool vec = kFull || words;
    const int N = kFull ? 4 * kLanes * kQuads : p.dstate;
    const int lane = threadIdx.x & 31, part = threadIdx.x % kLanes;
    const int own = part & (kRows - 1);  // which of the thread's sequences it owns
    const int c = blockIdx.x * kChannels + threadIdx.x / kLanes;
    const bool active = c < p.dim;
    const int d = active ? c : p.dim - 1;
    const int g = p.groups == 1 ? 0 : d / (p.dim / p.groups);
    const size_t row_elems = static_cast<size_t>(p.dim) * N, bc_elems = static_cast<size_t>(p.groups) * N;
    const int n0_lane = vec ? 4 * part : part;                      // this lane's first state
    const size_t here = static_cast<size_t>(d) * N + n0_lane;       // and its place in a row
    const T *const Bp = static_cast<const T *>(p.B) + static_cast<size_t>(g) * N + n0_lane;
    const T *const Cp = static_cast<const T *>(p.C) + static_cast<size_t>(g) * N + n0_lane;
    auto left = [&](int k) {  // how many of the lane's k-th four states are below N
        if (kFull) return 4;
        const int n = N - n0_lane - 4 * kLanes * k;
        return vec ? n : (n + kLanes - 1) / kLanes;
    };
    // (sequences are counted in 31 bits, the steps past the last one need the 32nd)
    const unsigned units = p.seq.units;
    for (unsigned n0 = blockIdx.y * kRows; n0 < units; n0 += gridDim.y * kRows) {
        int row[kRows];  // rows of the state are numbered in 31 bits
#pragma unroll
        for (int r = 0; r < kRows; ++r) row[r] = n0 + r < units ? static_cast<int>(seq_row(p.seq, n0 + r)) : -1;
        const unsigned mine = min(n0 + own, units - 1);
        const size_t at = static_cast<size_t>(mine) * p.dim + d;
        const float delta = to_f32<T>(static_cast<const T *>(p.delta)[at]);
        const float u = to_f32<T>(static_cast<const T *>(p.u)[at]);
        const float z = p.z != nullptr ? to_f32<T>(static_cast<const T *>(p.z)[at]) : 0.0f;
        float4 h[kRows][kQuads], b[kRows][kQuads], cc[kRows][kQuads];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const float *s = p.init + static_cast<size_t>(max(row[r], 0)) * row_elems + here;
            const size_t bc = static_cast<size_t>(min(n0 + r, units - 1)) * bc_elems;
#pragma unroll
            for (int k = 0; k < kQuads; ++k) {
                h[r][k] = load_states<(kRows > 1)>(s + 4 * kLanes * k, row[r] >= 0 ? left(k) : 0, vec, kLanes);
                b[r][k] = load_io4<T>(Bp + bc + 4 * kLanes * k, left(k), vec, kLanes);
                cc[r][k] = load_io4<T>(Cp + bc + 4 * kLanes * k, left(k), vec, kLanes);
            }
        }
        float4 a2[kQuads];
#pragma unroll
        for (int k = 0; k < kQuads; ++k) {
            a2[k] = load_states<false>(p.A + here + 4 * kLanes * k, left(k), vec, kLanes);
            a2[k] = make_float4(a2[k].x * kLog2e, a2[k].y * kLog2e, a2[k].z * kLog2e, a2[k].w * kLog2e);
        }
        float dt_own = delta + (p.bias != nullptr ? p.bias[d] : 0.0f);
        if (p.softplus) dt_own = softplus_pair(make_float2(dt_own, dt_own)).x;
        const float du_own = dt_own * u;
        float y[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int owner = (lane & ~(kRows - 1)) | r;
            const float dt = kRows == 1 ? dt_own : __shfl_sync(kFullMask, dt_own, owner);
            const float du = kRows == 1 ? du_own : __shfl_sync(kFullMask, du_own, owner);
            y[r] = 0.0f;
#pragma unroll
            for (int k = 0; k < kQuads; ++k) {
                float4 &v = h[r][k];
                v.x = fmaf(ex2_approx(dt * a2[k].x), v.x, du * b[r][k].x);
                v.y = fmaf(ex2_approx(dt * a2[k].y), v.y, du * b[r][k].y);
                v.z = fmaf(ex2_approx(dt * a2[k].z), v.z, du * b[r][k].z);
                v.w = fmaf(ex2_approx(dt * a2[k].w), v.w, du * b[r][k].w);
                // states at and behind N take no part, whatever dt u is
                if (left(k) > 0) y[r] = fmaf(cc[r][k].x, v.x, y[r]);
                if (left(k) > 1) y[r] = fmaf(cc[r][k].y, v.y, y[r]);
                if (left(k) > 2) y[r] = fmaf(cc[r][k].z, v.z, y[r]);
                if (left(k) > 3) y[r] = fmaf(cc[r][k].w, v.w, y[r]);
            }
            if (active && row[r] >= 0) {
                float *s = p.final_state + static_cast<size_t>(row[r]) * row_elems + here;
#pragma unroll
                for (int k = 0; k < kQuads; ++k) store_states<(kRows > 1)>(s + 4 * kLanes * k, left(k), vec, kLanes, h[r][k]);
            }
        }
        // Sum over the channel's lanes; the first steps leave each lane the sequence it owns.
        float v = y[0];
        if constexpr (kRows == 2) {
            const bool hi = own & 1;
            v = (hi ? y[1] : y[0]) + __shfl_xor_sync(kFullMask, hi ? y[0] : y[1], 1);
        }
        if constexpr (kRows == 4) {
            const bool hi = own & 2, odd = own & 1;
            const float k0 = (hi ? y[2] : y[0]) + __shfl_xor_sync(kFullMask, hi ? y[0] : y[2], 2);
            const float k1 = (hi ? y[3] : y[1]) + __shfl_xor_sync(kFullMask, hi ? y[1] : y[3], 2);
            v = (odd ? k1 : k0) + __shfl_xor_sync(kFullMask, odd ? k0 : k1, 1);
        }
        // (one sequence per thread adds in the same order, so a row's result does not depend on the batch)
        if constexpr (kRows == 1 && kLanes >= 4) {
            v += __shfl_xor_sync(kFullMask, v, 2);
            v += __shfl_xor_sync(kFullMask, v, 1);
        }
#pragma unroll
        for (int o = kRows == 1 && kLanes >= 4 ? 4 : kRows; o < kLanes; o *= 2) v += __shfl_xor_sync(kFullMask, v, o);
        v = fmaf(p.D != nullptr ? p.D[d] : 0.0f, u, v);
        if (p.z != nullptr) v *= z * rcp_approx(1.0f + ex2_approx(-z * kLog2e));
        bool kept = row[0] >= 0;  // the owned sequence owns a state row
#pragma unroll
        for (int r = 1; r < kRows; ++r)
            if (own == r) kept = row[r] >= 0;
        if (active && part < kRows && kept) static_cast<T *>(p.out)[at] = from_f32<T>(v);
    }
}

// As many sequences per thread as there are lanes for (four at most) where that
// leaves each SM eight blocks; below, one.
template <typename T, int kLanes, int kQuads>
cudaError_t launch_lanes(const ScanArgs &a, cudaStream_t stream) {
    constexpr int kRows = kLanes < 4 ? kLanes : 4;
    const size_t word = 4 * (a.io == IoType::kF32 ? 4 : 2);
    auto on = [](const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
    const bool vec = a.dstate % 4 == 0 && aligned16(a.init) && aligned16(a.final_state) && aligned16(a.A) &&
                     on(a.B, word) && on(a.C, word);
    const int64_t blocks = (a.dim + kUpdThreads / kLanes - 1) / (kUpdThreads / kLanes);
    const int64_t many = (static_cast<int64_t>(a.seq.units) + kRows - 1) / kRows;
    const bool wide = kRows > 1 && blocks * many >= 8LL * current_device_sm_count();
    const dim3 grid(static_cast<unsigned>(blocks),
                    static_cast<unsigned>(std::min<int64_t>(wide ? many : a.seq.units, 65535)));
    if (vec && a.dstate == 4 * kLanes * kQuads) {
        if (wide) state_token_kernel<T, kLanes, kQuads, kRows, true><<<grid, kUpdThreads, 0, stream>>>(a, vec);
        else state_token_kernel<T, kLanes, kQuads, 1, true><<<grid, kUpdThreads, 0, stream>>>(a, vec);
    } else {
        if (wide) state_token_kernel<T, kLanes, kQuads, kRows, false><<<grid, kUpdThreads, 0, stream>>>(a, vec);
        else state_token_kernel<T, kLanes, kQuads, 1, false><<<grid, kUpdThreads, 0, stream>>>(a, vec);
    }
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_type(const ScanArgs &a, cudaStream_t stream) {
    if (a.dstate <= 4) return launch_lanes<T, 1, 1>(a, stream);
    if (a.dstate <= 8) return launch_lanes<T, 2, 1>(a, stream);
    if (a.dstate <= 16) return launch_lanes<T, 4, 1>(a, stream);
    if (a.dstate <= 32) return launch_lanes<T, 8, 1>(a, stream);
    if (a.dstate <= 64) return launch_lanes<T, 16, 1>(a, stream);
    if (a.dstate <= 128) return launch_lanes<T, 32, 1>(a, stream);
    return launch_lanes<T, 32, 2>(a, stream);
}

}  // namespace

cudaError_t launch_selective_state_update(const ScanArgs &a, cudaStream_t stream) {
    switch (a.io) {
        case IoType::kBF16: return launch_type<__nv_bfloat16>(a, stream);
        case IoType::kF16: return launch_type<__half>(a, stream);
        default: return launch_type<float>(a, stream);
    }
}

}  // namespace xm
