// gated_recurrence_grad.cu -- GatedRecurrenceGradFn for sm_100a.
//
// Math, per channel, from a sequence's last token to its first, with c the
// gradient that reaches the state behind a token (d_final_state at first):
//   G_t = dy_t + c,  dx_t = (1 - a_t) G_t,  c <- a_t G_t,
//   df_t = G_t (h_(t-1) - x_t) (1 - a_t) sigmoid(f_t),
//   d_bound += G_t (h_(t-1) - x_t) sigmoid(-f_t).
#include <algorithm>

#include "xm_common.cuh"
#include "xm_gate.cuh"
#include "xm_kernels.h"
#include "xm_sequences.cuh"

namespace xm {
namespace {

constexpr int kThreads = 128;

// A thread per channel walks all sequences backwards.
template <typename T>
__global__ void __launch_bounds__(kThreads) gate_grad_kernel(const GateGradArgs p) {
    const int d = blockIdx.x * kThreads + threadIdx.x;
    if (d >= p.dim) return;
    const float low = p.bound != nullptr ? p.bound[d] : 0.0f, rest = 1.0f - low;
    float sum = 0.0f;
    for (int i = 0; i < p.seq.units; ++i) {
        const int t0 = seq_start(p.seq, i), t1 = seq_end(p.seq, i, t0);
        const size_t srow = static_cast<size_t>(i) * p.dim + d;
        float c = p.dfinal != nullptr ? p.dfinal[srow] : 0.0f;
        for (int t = t1 - 1; t >= t0; --t) {
            const size_t at = static_cast<size_t>(t) * p.dim + d;
            const Gate g = gate_of(to_f32<T>(static_cast<const T *>(p.f)[at]));
            const float x = to_f32<T>(static_cast<const T *>(p.x)[at]);
            const float before = t > t0 ? to_f32<T>(static_cast<const T *>(p.y)[at - p.dim])
                                        : (p.init != nullptr ? p.init[srow] : 0.0f);
            const float G = to_f32<T>(static_cast<const T *>(p.dy)[at]) + c;
            const float take = rest * g.take, da = G * (before - x);
            static_cast<T *>(p.dx)[at] = from_f32<T>(take * G);
            static_cast<T *>(p.df)[at] = from_f32<T>(da * take * g.keep);
            sum = fmaf(da, g.take, sum);
            c = fmaf(rest, g.keep, low) * G;
        }
        if (p.dinit != nullptr) p.dinit[srow] = c;
    }
    if (p.dbound != nullptr) p.dbound[d] = sum;
}

template <typename T>
cudaError_t launch_type(const GateGradArgs &a, cudaStream_t stream) {
    gate_grad_kernel<T><<<(a.dim + kThreads - 1) / kThreads, kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

size_t gated_recurrence_grad_workspace(const GateGradArgs &) { return 0; }

cudaError_t launch_gated_recurrence_grad(const GateGradArgs &a, void *, cudaStream_t stream) {
    switch (a.io) {
        case IoType::kBF16: return launch_type<__nv_bfloat16>(a, stream);
        case IoType::kF16: return launch_type<__half>(a, stream);
        default: return launch_type<float>(a, stream);
    }
}

}  // namespace xm
