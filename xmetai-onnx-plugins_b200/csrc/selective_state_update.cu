// selective_state_update.cu -- SelectiveStateUpdateFn for sm_100a.
//
// Math, per sequence and channel d (state n = 0 .. N - 1):
//   dt = softplus?(delta + bias), h_n = exp(dt A_n) h_n + dt u B_n,
//   y = (D u + sum_n C_n h_n) silu(z).
//
// Bound by memory: the state is read and written once, 8 bytes per (sequence,
// channel, state), against about a dozen instructions per four states. A channel
// belongs to kLanes adjacent lanes with four consecutive states each (eight for
// N > 128), so a warp's state accesses are whole 16-byte words of consecutive
// memory, and y is summed with xor shuffles. Where there are sequences enough, a
// thread takes kRows of them for the same channel: their loads are issued
// together, and A, D and the bias are read once for all.
#include <algorithm>

#include "xm_common.cuh"
#include "xm_kernels.h"
#include "xm_sequences.cuh"

namespace xm {
namespace {

constexpr int kUpdThreads = 128;

// Four consecutive states from `p`, `left` of them below N (vec: all, one word).
__device__ __forceinline__ float4 load_states(const float *p, int left, bool vec) {
    if (vec) return left > 0 ? *reinterpret_cast<const float4 *>(p) : make_float4(0, 0, 0, 0);
    return make_float4(left > 0 ? p[0] : 0.0f, left > 1 ? p[1] : 0.0f, left > 2 ? p[2] : 0.0f, left > 3 ? p[3] : 0.0f);
}

__device__ __forceinline__ void store_states(float *p, int left, bool vec, const float4 &v) {
    if (vec) {
        if (left > 0) *reinterpret_cast<float4 *>(p) = v;
        return;
    }
    if (left > 0) p[0] = v.x;
    if (left > 1) p[1] = v.y;
    if (left > 2) p[2] = v.z;
    if (left > 3) p[3] = v.w;
}

// Four consecutive values of the I/O type as floats, zeros from `left` on.
template <typename T>
__device__ __forceinline__ float4 load_io4(const T *p, int left, bool vec) {
    if (vec && left > 0) {
        if constexpr (sizeof(T) == 4) {
            return __ldg(reinterpret_cast<const float4 *>(p));
        } else {
            const uint2 w = __ldg(reinterpret_cast<const uint2 *>(p));
            const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
            return make_float4(a.x, a.y, b.x, b.y);
        }
    }
    return make_float4(left > 0 ? to_f32<T>(p[0]) : 0.0f, left > 1 ? to_f32<T>(p[1]) : 0.0f,
                       left > 2 ? to_f32<T>(p[2]) : 0.0f, left > 3 ? to_f32<T>(p[3]) : 0.0f);
}

template <typename T, int kLanes, int kQuads, int kRows>
__global__ void __launch_bounds__(kUpdThreads) state_token_kernel(const ScanArgs p, bool vec) {
    constexpr int kChannels = kUpdThreads / kLanes;
    const int N = p.dstate, part = threadIdx.x % kLanes;
    const int c = blockIdx.x * kChannels + threadIdx.x / kLanes;
    const bool active = c < p.dim;
    const int d = active ? c : p.dim - 1;
    const int g = d / (p.dim / p.groups);
    for (int n0 = blockIdx.y * kRows; n0 < p.seq.units; n0 += gridDim.y * kRows) {
        long long row[kRows];
        float4 h[kRows][kQuads];
        float delta[kRows], u[kRows], z[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) row[r] = n0 + r < p.seq.units ? seq_row(p.seq, n0 + r) : -1;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const float *s = p.init + (static_cast<size_t>(max(row[r], 0LL)) * p.dim + d) * N;
#pragma unroll
            for (int k = 0; k < kQuads; ++k) {
                const int n = 4 * (k * kLanes + part);
                h[r][k] = load_states(s + n, row[r] >= 0 ? N - n : 0, vec);
            }
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const size_t at = static_cast<size_t>(min(n0 + r, p.seq.units - 1)) * p.dim + d;
            delta[r] = to_f32<T>(static_cast<const T *>(p.delta)[at]);
            u[r] = to_f32<T>(static_cast<const T *>(p.u)[at]);
            z[r] = p.z != nullptr ? to_f32<T>(static_cast<const T *>(p.z)[at]) : 0.0f;
        }
        float4 a2[kQuads];
#pragma unroll
        for (int k = 0; k < kQuads; ++k) {
            const int n = 4 * (k * kLanes + part);
            a2[k] = load_states(p.A + static_cast<size_t>(d) * N + n, N - n, vec);
            a2[k] = make_float4(a2[k].x * kLog2e, a2[k].y * kLog2e, a2[k].z * kLog2e, a2[k].w * kLog2e);
        }
        const float bias = p.bias != nullptr ? p.bias[d] : 0.0f, skip = p.D != nullptr ? p.D[d] : 0.0f;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const size_t bc = (static_cast<size_t>(min(n0 + r, p.seq.units - 1)) * p.groups + g) * N;
            float dt = delta[r] + bias;
            if (p.softplus) dt = softplus_pair(make_float2(dt, dt)).x;
            const float du = dt * u[r];
            float y = 0.0f;
#pragma unroll
            for (int k = 0; k < kQuads; ++k) {
                const int n = 4 * (k * kLanes + part), left = N - n;
                const float4 b = load_io4<T>(static_cast<const T *>(p.B) + bc + n, left, vec);
                const float4 cc = load_io4<T>(static_cast<const T *>(p.C) + bc + n, left, vec);
                float4 &v = h[r][k];
                v.x = fmaf(ex2_approx(dt * a2[k].x), v.x, du * b.x);
                v.y = fmaf(ex2_approx(dt * a2[k].y), v.y, du * b.y);
                v.z = fmaf(ex2_approx(dt * a2[k].z), v.z, du * b.z);
                v.w = fmaf(ex2_approx(dt * a2[k].w), v.w, du * b.w);
                // states at and behind N take no part, whatever dt u is
                if (left > 0) y = fmaf(cc.x, v.x, y);
                if (left > 1) y = fmaf(cc.y, v.y, y);
                if (left > 2) y = fmaf(cc.z, v.z, y);
                if (left > 3) y = fmaf(cc.w, v.w, y);
            }
            if (active && row[r] >= 0) {
                float *s = p.final_state + (static_cast<size_t>(row[r]) * p.dim + d) * N;
#pragma unroll
                for (int k = 0; k < kQuads; ++k) {
                    const int n = 4 * (k * kLanes + part);
                    store_states(s + n, N - n, vec, h[r][k]);
                }
            }
#pragma unroll
            for (int o = kLanes / 2; o > 0; o /= 2) y += __shfl_xor_sync(kFullMask, y, o);
            y = fmaf(skip, u[r], y);
            if (p.z != nullptr) y *= z[r] * rcp_approx(1.0f + ex2_approx(-z[r] * kLog2e));
            if (active && part == 0 && row[r] >= 0)
                static_cast<T *>(p.out)[static_cast<size_t>(n0 + r) * p.dim + d] = from_f32<T>(y);
        }
    }
}

// Four sequences per thread where that leaves each SM eight blocks (the loads of
// one thread then cover the latency); below, one.
template <typename T, int kLanes, int kQuads>
cudaError_t launch_lanes(const ScanArgs &a, cudaStream_t stream) {
    const size_t word = 4 * (a.io == IoType::kF32 ? 4 : 2);
    auto on = [](const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
    const bool vec = a.dstate % 4 == 0 && aligned16(a.init) && aligned16(a.final_state) && aligned16(a.A) &&
                     on(a.B, word) && on(a.C, word);
    const int64_t blocks = (a.dim + kUpdThreads / kLanes - 1) / (kUpdThreads / kLanes);
    const int64_t groups = (static_cast<int64_t>(a.seq.units) + 3) / 4;
    const unsigned gx = static_cast<unsigned>(blocks);
    if (blocks * groups >= 8LL * current_device_sm_count())
        state_token_kernel<T, kLanes, kQuads, 4>
            <<<dim3(gx, static_cast<unsigned>(std::min<int64_t>(groups, 65535))), kUpdThreads, 0, stream>>>(a, vec);
    else
        state_token_kernel<T, kLanes, kQuads, 1>
            <<<dim3(gx, static_cast<unsigned>(std::min(a.seq.units, 65535))), kUpdThreads, 0, stream>>>(a, vec);
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
