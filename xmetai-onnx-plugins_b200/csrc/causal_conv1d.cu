// causal_conv1d.cu -- CausalConv1dFn and CausalConv1dUpdateFn for sm_100a.
//
// Math, per channel d: y_t = act(bias + sum_{k < W} w_k x_(t - (W - 1) + k)),
// act = identity or v sigmoid(v); x before the sequence's first token comes from
// its state, the last W - 1 inputs of the tokens that went before.
#include <algorithm>

#include "xm_common.cuh"
#include "xm_kernels.h"
#include "xm_sequences.cuh"

namespace xm {
namespace {

constexpr int kConvThreads = 128;

__device__ __forceinline__ float conv_act(float v, bool silu) {
    return silu ? __fdividef(v, 1.0f + __expf(-v)) : v;
}

// One thread per (sequence, channel), walking the tokens.
template <typename T>
__global__ void __launch_bounds__(kConvThreads) conv_walk_kernel(const ConvArgs p) {
    const int n = blockIdx.x;
    const SeqArgs &q = p.seq;
    const int start = seq_start(q, n), end = seq_end(q, n, start);
    const long long row = seq_row(q, n);
    const bool live = p.init != nullptr && seq_live(q, n, row);
    const int W = p.width;
    for (int d = blockIdx.y * kConvThreads + threadIdx.x; d < p.dim; d += gridDim.y * kConvThreads) {
        float w[4], v[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // taps, and the window's inputs, right-aligned
        T raw[4];
        for (int k = 0; k < 4; ++k) {
            w[k] = 0.0f;
            raw[k] = from_f32<T>(0.0f);
        }
        const size_t srow = (static_cast<size_t>(row < 0 ? 0 : row) * p.dim + d) * (W - 1);
        for (int k = 0; k < W; ++k) w[4 - W + k] = p.weight[static_cast<size_t>(d) * W + k];
        for (int k = 0; k < W - 1; ++k) {
            if (live) raw[4 - (W - 1) + k] = static_cast<const T *>(p.init)[srow + k];
            v[4 - (W - 1) + k] = to_f32<T>(raw[4 - (W - 1) + k]);
        }
        const float b = p.bias != nullptr ? p.bias[d] : 0.0f;
        for (int t = start; t < end; ++t) {
            const int r = t / max(1, q.seqlen), c = t - r * q.seqlen;
            const size_t at = p.channels_last ? static_cast<size_t>(t) * p.dim + d
                                              : (static_cast<size_t>(r) * p.dim + d) * q.seqlen + c;
            for (int k = 0; k < 3; ++k) {
                v[k] = v[k + 1];
                raw[k] = raw[k + 1];
            }
            raw[3] = static_cast<const T *>(p.x)[at];
            v[3] = to_f32<T>(raw[3]);
            float y = b;
            for (int k = 4 - W; k < 4; ++k) y = fmaf(w[k], v[k], y);
            static_cast<T *>(p.out)[at] = from_f32<T>(conv_act(y, p.silu));
        }
        if (p.final_state != nullptr && row >= 0)
            for (int k = 0; k < W - 1; ++k) static_cast<T *>(p.final_state)[srow + k] = raw[4 - (W - 1) + k];
    }
}

template <typename T>
__global__ void __launch_bounds__(kConvThreads) conv_token_kernel(const ConvArgs p) {
    const int n = blockIdx.x;
    const long long row = seq_row(p.seq, n);
    if (row < 0) return;
    const int W = p.width;
    for (int d = blockIdx.y * kConvThreads + threadIdx.x; d < p.dim; d += gridDim.y * kConvThreads) {
        const size_t srow = (static_cast<size_t>(row) * p.dim + d) * (W - 1);
        const T x = static_cast<const T *>(p.x)[static_cast<size_t>(n) * p.dim + d];
        float y = p.bias != nullptr ? p.bias[d] : 0.0f;
        const float *w = p.weight + static_cast<size_t>(d) * W;
        for (int k = 0; k < W - 1; ++k) {
            const T s = static_cast<const T *>(p.init)[srow + k];
            y = fmaf(w[k], to_f32<T>(s), y);
            if (k > 0) static_cast<T *>(p.final_state)[srow + k - 1] = s;
        }
        static_cast<T *>(p.final_state)[srow + W - 2] = x;
        y = fmaf(w[W - 1], to_f32<T>(x), y);
        static_cast<T *>(p.out)[static_cast<size_t>(n) * p.dim + d] = from_f32<T>(conv_act(y, p.silu));
    }
}

template <typename F>
cudaError_t by_type(IoType io, F &&f) {
    switch (io) {
        case IoType::kBF16: f(__nv_bfloat16{}); break;
        case IoType::kF16: f(__half{}); break;
        default: f(float{}); break;
    }
    return cudaGetLastError();
}

dim3 conv_grid(const ConvArgs &a) {
    return dim3(a.seq.units, static_cast<unsigned>(std::min((a.dim + kConvThreads - 1) / kConvThreads, 65535)));
}

}  // namespace

cudaError_t launch_causal_conv1d(const ConvArgs &a, cudaStream_t stream) {
    return by_type(a.io, [&](auto t) { conv_walk_kernel<decltype(t)><<<conv_grid(a), kConvThreads, 0, stream>>>(a); });
}

cudaError_t launch_causal_conv1d_update(const ConvArgs &a, cudaStream_t stream) {
    return by_type(a.io, [&](auto t) { conv_token_kernel<decltype(t)><<<conv_grid(a), kConvThreads, 0, stream>>>(a); });
}

}  // namespace xm
