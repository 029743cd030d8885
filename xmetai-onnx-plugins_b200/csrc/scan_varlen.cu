// scan_varlen.cu -- SelectiveScanVarlenFn for sm_100a.
//
// Math, per token t and channel d (state n = 0 .. N - 1):
//   dt = softplus?(delta + bias), h_n = exp(dt A_n) h_n + dt u B_n,
//   y = (D u + sum_n C_n h_n) silu(z).
#include <algorithm>

#include "xm_common.cuh"
#include "xm_kernels.h"
#include "xm_sequences.cuh"

namespace xm {
namespace {

constexpr int kScanThreads = 128;
constexpr float kScanLog2e = 1.4426950408889634f;

// One warp per (sequence, channel), eight states per lane, walking the tokens.
template <typename T>
__global__ void __launch_bounds__(kScanThreads) scan_walk_kernel(const ScanArgs p) {
    const SeqArgs &q = p.seq;
    const int n = blockIdx.x;
    const int start = seq_start(q, n), end = seq_end(q, n, start);
    const long long row = seq_row(q, n);
    const bool live = p.init != nullptr && seq_live(q, n, row);
    const int lane = threadIdx.x & 31, N = p.dstate;
    constexpr int kWarps = kScanThreads / 32;
    for (int d = blockIdx.y * kWarps + threadIdx.x / 32; d < p.dim; d += gridDim.y * kWarps) {
        const int g = d / (p.dim / p.groups);
        const size_t srow = (static_cast<size_t>(row < 0 ? 0 : row) * p.dim + d) * N;
        float h[8], a2[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int s = lane + 32 * j;
            a2[j] = s < N ? p.A[static_cast<size_t>(d) * N + s] * kScanLog2e : 0.0f;
            h[j] = live && s < N ? p.init[srow + s] : 0.0f;
        }
        const float bias = p.bias != nullptr ? p.bias[d] : 0.0f, skip = p.D != nullptr ? p.D[d] : 0.0f;
        for (int t = start; t < end; ++t) {
            const size_t at = static_cast<size_t>(t) * p.dim + d;
            const size_t bc = (static_cast<size_t>(t) * p.groups + g) * N;
            float dt = to_f32<T>(static_cast<const T *>(p.delta)[at]) + bias;
            if (p.softplus) dt = softplus_dt(dt);
            const float u = to_f32<T>(static_cast<const T *>(p.u)[at]);
            float y = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int s = lane + 32 * j;
                if (s < N) {
                    const float b = to_f32<T>(static_cast<const T *>(p.B)[bc + s]);
                    const float c = to_f32<T>(static_cast<const T *>(p.C)[bc + s]);
                    h[j] = fmaf(ex2_approx(dt * a2[j]), h[j], dt * u * b);
                    y = fmaf(c, h[j], y);
                }
            }
            for (int o = 16; o > 0; o >>= 1) y += __shfl_xor_sync(kFullMask, y, o);
            y = fmaf(skip, u, y);
            if (p.z != nullptr) {
                const float z = to_f32<T>(static_cast<const T *>(p.z)[at]);
                y *= __fdividef(z, 1.0f + __expf(-z));
            }
            if (lane == 0) static_cast<T *>(p.out)[at] = from_f32<T>(y);
        }
        if (p.final_state != nullptr && row >= 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (lane + 32 * j < N) p.final_state[srow + lane + 32 * j] = h[j];
        }
    }
}

}  // namespace

size_t scan_varlen_workspace(const ScanArgs &) { return 0; }

cudaError_t launch_scan_varlen(const ScanArgs &a, void *, cudaStream_t stream) {
    const dim3 grid(a.seq.units, std::min((a.dim + 3) / 4, 65535));
    switch (a.io) {
        case IoType::kBF16: scan_walk_kernel<__nv_bfloat16><<<grid, kScanThreads, 0, stream>>>(a); break;
        case IoType::kF16: scan_walk_kernel<__half><<<grid, kScanThreads, 0, stream>>>(a); break;
        default: scan_walk_kernel<float><<<grid, kScanThreads, 0, stream>>>(a); break;
    }
    return cudaGetLastError();
}

}  // namespace xm
