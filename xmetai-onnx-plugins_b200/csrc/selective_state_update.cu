// selective_state_update.cu -- SelectiveStateUpdateFn for sm_100a.
//
// Math, per sequence and channel d (state n = 0 .. N - 1):
//   dt = softplus?(delta + bias), h_n = exp(dt A_n) h_n + dt u B_n,
//   y = (D u + sum_n C_n h_n) silu(z).
#include <algorithm>

#include "xm_common.cuh"
#include "xm_kernels.h"
#include "xm_sequences.cuh"

namespace xm {
namespace {

constexpr int kUpdThreads = 128;
constexpr float kUpdLog2e = 1.4426950408889634f;

// One warp per (sequence, channel), a state per lane and step of 32.
template <typename T>
__global__ void __launch_bounds__(kUpdThreads) state_token_kernel(const ScanArgs p) {
    const int n = blockIdx.x;
    const long long row = seq_row(p.seq, n);
    if (row < 0) return;
    const int lane = threadIdx.x & 31, N = p.dstate;
    constexpr int kWarps = kUpdThreads / 32;
    for (int d = blockIdx.y * kWarps + threadIdx.x / 32; d < p.dim; d += gridDim.y * kWarps) {
        const int g = d / (p.dim / p.groups);
        const size_t srow = (static_cast<size_t>(row) * p.dim + d) * N;
        const size_t at = static_cast<size_t>(n) * p.dim + d;
        const size_t bc = (static_cast<size_t>(n) * p.groups + g) * N;
        float dt = to_f32<T>(static_cast<const T *>(p.delta)[at]) + (p.bias != nullptr ? p.bias[d] : 0.0f);
        if (p.softplus) dt = softplus_dt(dt);
        const float u = to_f32<T>(static_cast<const T *>(p.u)[at]);
        float y = 0.0f;
        for (int s = lane; s < N; s += 32) {
            const float a = ex2_approx(dt * (p.A[static_cast<size_t>(d) * N + s] * kUpdLog2e));
            const float h = fmaf(a, p.init[srow + s], dt * u * to_f32<T>(static_cast<const T *>(p.B)[bc + s]));
            y = fmaf(to_f32<T>(static_cast<const T *>(p.C)[bc + s]), h, y);
            p.final_state[srow + s] = h;
        }
        for (int o = 16; o > 0; o >>= 1) y += __shfl_xor_sync(kFullMask, y, o);
        y = fmaf(p.D != nullptr ? p.D[d] : 0.0f, u, y);
        if (p.z != nullptr) {
            const float z = to_f32<T>(static_cast<const T *>(p.z)[at]);
            y *= __fdividef(z, 1.0f + __expf(-z));
        }
        if (lane == 0) static_cast<T *>(p.out)[at] = from_f32<T>(y);
    }
}

}  // namespace

cudaError_t launch_selective_state_update(const ScanArgs &a, cudaStream_t stream) {
    const dim3 grid(a.seq.units, std::min((a.dim + 3) / 4, 65535));
    switch (a.io) {
        case IoType::kBF16: state_token_kernel<__nv_bfloat16><<<grid, kUpdThreads, 0, stream>>>(a); break;
        case IoType::kF16: state_token_kernel<__half><<<grid, kUpdThreads, 0, stream>>>(a); break;
        default: state_token_kernel<float><<<grid, kUpdThreads, 0, stream>>>(a); break;
    }
    return cudaGetLastError();
}

}  // namespace xm
