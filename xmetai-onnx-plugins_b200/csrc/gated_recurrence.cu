// gated_recurrence.cu -- GatedRecurrenceFn and GatedRecurrenceUpdateFn for sm_100a.
//
// Math, per channel: a_t = b + (1 - b) sigmoid(f_t), h_t = a_t h_(t-1) + (1 - a_t) x_t.
#include <algorithm>

#include "xm_common.cuh"
#include "xm_gate.cuh"
#include "xm_kernels.h"
#include "xm_sequences.cuh"

namespace xm {
namespace {

constexpr int kThreads = 128;

// A thread per (sequence, channel) walks the tokens.
template <typename T>
__global__ void __launch_bounds__(kThreads) gate_kernel(const GateArgs p) {
    const int d = blockIdx.x * kThreads + threadIdx.x;
    if (d >= p.dim) return;
    const float low = p.bound != nullptr ? p.bound[d] : 0.0f, rest = 1.0f - low;
    for (unsigned i = blockIdx.y; i < static_cast<unsigned>(p.seq.units); i += gridDim.y) {
        const int t0 = seq_start(p.seq, i), t1 = seq_end(p.seq, i, t0);
        const long long row = seq_row(p.seq, i);
        float h = p.init != nullptr && seq_live(p.seq, i, row) ? p.init[row * p.dim + d] : 0.0f;
        for (int t = t0; t < t1; ++t) {
            const size_t at = static_cast<size_t>(t) * p.dim + d;
            const Gate g = gate_of(to_f32<T>(static_cast<const T *>(p.f)[at]));
            const float x = to_f32<T>(static_cast<const T *>(p.x)[at]);
            h = fmaf(fmaf(rest, g.keep, low), h, rest * g.take * x);
            static_cast<T *>(p.out)[at] = from_f32<T>(h);
        }
        if (p.final_state != nullptr && row >= 0) p.final_state[row * p.dim + d] = h;
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) gate_token_kernel(const GateArgs p) {
    const int d = blockIdx.x * kThreads + threadIdx.x;
    if (d >= p.dim) return;
    const float low = p.bound != nullptr ? p.bound[d] : 0.0f, rest = 1.0f - low;
    for (unsigned i = blockIdx.y; i < static_cast<unsigned>(p.seq.units); i += gridDim.y) {
        const long long row = seq_row(p.seq, i);
        if (row < 0) continue;
        const size_t at = static_cast<size_t>(i) * p.dim + d;
        const Gate g = gate_of(to_f32<T>(static_cast<const T *>(p.f)[at]));
        const float x = to_f32<T>(static_cast<const T *>(p.x)[at]);
        const float h = fmaf(fmaf(rest, g.keep, low), p.init[row * p.dim + d], rest * g.take * x);
        p.final_state[row * p.dim + d] = h;
        static_cast<T *>(p.out)[at] = from_f32<T>(h);
    }
}

dim3 grid_of(const GateArgs &a) { return dim3((a.dim + kThreads - 1) / kThreads, std::min(a.seq.units, 65535)); }

template <typename T>
cudaError_t launch_type(const GateArgs &a, cudaStream_t stream) {
    gate_kernel<T><<<grid_of(a), kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_token_type(const GateArgs &a, cudaStream_t stream) {
    gate_token_kernel<T><<<grid_of(a), kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_gated_recurrence(const GateArgs &a, cudaStream_t stream) {
    switch (a.io) {
        case IoType::kBF16: return launch_type<__nv_bfloat16>(a, stream);
        case IoType::kF16: return launch_type<__half>(a, stream);
        default: return launch_type<float>(a, stream);
    }
}

cudaError_t launch_gated_recurrence_update(const GateArgs &a, cudaStream_t stream) {
    switch (a.io) {
        case IoType::kBF16: return launch_token_type<__nv_bfloat16>(a, stream);
        case IoType::kF16: return launch_token_type<__half>(a, stream);
        default: return launch_token_type<float>(a, stream);
    }
}

}  // namespace xm
