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

constexpr int kStages = 2;

template <typename T, int V>
struct ScanSmem {
    GateJoin<V> join;
    // words of x and f, each read only by the thread that copied it
    uint32_t ring[V * sizeof(T) == 4 ? kStages : 0][2][kGateSteps][kGateThreads];
};

// V channels per lane: two of the 16-bit types in a word (rows of even length, aligned
// to words), else one. Words come by asynchronous copies a step ahead.
template <typename T, int V>
__global__ void __launch_bounds__(kGateThreads, 3) gate_kernel(const GateArgs p, const GateSpans g) {
    extern __shared__ float4 smem_f4[];
    constexpr bool kAsync = V * sizeof(T) == 4;
    auto &sm = *reinterpret_cast<ScanSmem<T, V> *>(smem_f4);
    const SeqArgs &q = p.seq;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned rank = g.cluster > 1 ? cluster_rank() : 0;
    const int id = blockIdx.x / g.cluster, tile = id % g.tiles, width = gridDim.x / g.cluster / g.tiles;
    const int c0 = (tile * 32 + lane) * V;
    const bool active = c0 < p.dim;  // (V divides dim)
    const int c = active ? c0 : 0;
    float low[V], rest[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        low[v] = p.bound != nullptr ? p.bound[c + v] : 0.0f;
        rest[v] = 1.0f - low[v];
    }
    const T *const X = static_cast<const T *>(p.x) + c, *const F = static_cast<const T *>(p.f) + c;
    T *const Y = static_cast<T *>(p.out) + c;
    auto init_of = [&](int seq, float (&h)[V]) {
        const long long row = seq_row(q, seq);
        const bool live = p.init != nullptr && seq_live(q, seq, row);
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = live ? p.init[row * p.dim + c + v] : 0.0f;
    };
    auto store_final = [&](int seq, const float (&h)[V]) {
        const long long row = seq_row(q, seq);
        if (p.final_state == nullptr || row < 0 || !active) return;
#pragma unroll
        for (int v = 0; v < V; ++v) p.final_state[row * p.dim + c + v] = h[v];
    };
    // sequences without tokens keep their starting states
    if (p.final_state != nullptr && (q.cu != nullptr || q.seqlen == 0)) {
        const int first = id / g.tiles * g.cluster + rank;
        for (long long s0 = (static_cast<long long>(first) * kGateWarps + warp) * 32; s0 < q.units;
             s0 += 32LL * kGateWarps * g.cluster * width) {
            const int s = static_cast<int>(s0) + lane;
            bool empty = false;
            if (s < q.units) {
                const int t = seq_start(q, s);
                empty = seq_end(q, s, t) == t;
            }
            for (unsigned left = __ballot_sync(kFullMask, empty); left != 0; left &= left - 1) {
                const int e = static_cast<int>(s0) + __ffs(left) - 1;
                float h[V];
                init_of(e, h);
                store_final(e, h);
            }
        }
    }
    if (g.cluster > 1) cluster_barrier();  // every block has begun before another writes into its shared memory
    const int stride = g.cluster * kGateTokens;  // tokens of a step
    int parity = 0;
    for (int i = id / g.tiles; i < g.rows; i += width) {
        const Span span = gate_span(q, g, i);
        const int mine = span.lo + rank * kGateTokens + warp * kGateSteps;
        auto copy = [&](int t0, int stage) {
            if constexpr (kAsync) {
                if (active) {
#pragma unroll
                    for (int k = 0; k < kGateSteps; ++k) {
                        if (t0 + k < span.hi) {
                            const size_t at = static_cast<size_t>(t0 + k) * p.dim;
                            cp_async4(&sm.ring[stage][0][k][tid], X + at, 4);
                            cp_async4(&sm.ring[stage][1][k][tid], F + at, 4);
                        }
                    }
                }
                cp_async_commit();
            }
        };
        for (int k = 0; k < kStages; ++k) copy(mine + k * stride, k);
        float carry[V];
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = 0.0f;
        SeqAt seq{0, 0, 0};
        int step = 0;
        for (int base = span.lo; base < span.hi; base += stride, ++step) {
            const int t0 = mine + step * stride, left = span.hi - t0;
            const int stage = step % kStages;
            cp_async_wait<kStages - 1>();
            float P[kGateSteps][V], h[kGateSteps][V];
            auto token = [&](int k, float (&x)[V], float (&f)[V]) {
                if constexpr (kAsync) {
                    unpack_word<T, V>(&sm.ring[stage][0][k][tid], x);
                    unpack_word<T, V>(&sm.ring[stage][1][k][tid], f);
                } else {
                    const size_t at = static_cast<size_t>(t0 + k) * p.dim;
                    unpack_word<T, V>(X + at, x);
                    unpack_word<T, V>(F + at, f);
                }
            };
            if (left > 0 && seq.end <= t0) seq = seq_at(q, t0);
            const bool inside = left >= kGateSteps && seq.start < t0 && seq.end > t0 + kGateSteps;
            float rp[V], rh[V];  // the running pair
#pragma unroll
            for (int v = 0; v < V; ++v) rp[v] = 1.0f, rh[v] = 0.0f;
            if (inside) {
#pragma unroll
                for (int k = 0; k < kGateSteps; ++k) {
                    float x[V], f[V];
                    token(k, x, f);
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const Gate gate = gate_of(f[v]);
                        const float a = fmaf(rest[v], gate.keep, low[v]);
                        rh[v] = fmaf(a, rh[v], rest[v] * gate.take * x[v]);
                        rp[v] *= a;
                        P[k][v] = rp[v];
                        h[k][v] = rh[v];
                    }
                }
            } else {
                SeqAt at = seq;
#pragma unroll
                for (int k = 0; k < kGateSteps; ++k) {
                    if (k < left) {
                        if (at.end <= t0 + k) at = seq_at(q, t0 + k);
                        if (at.start == t0 + k) {
                            init_of(at.seq, rh);
#pragma unroll
                            for (int v = 0; v < V; ++v) rp[v] = kCut;
                        }
                        float x[V], f[V];
                        token(k, x, f);
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            const Gate gate = gate_of(f[v]);
                            const float a = fmaf(rest[v], gate.keep, low[v]);
                            rh[v] = fmaf(a, rh[v], rest[v] * gate.take * x[v]);
                            rp[v] = rp[v] < 0.0f ? kCut : rp[v] * a;
                        }
                    }
#pragma unroll
                    for (int v = 0; v < V; ++v) P[k][v] = rp[v], h[k][v] = rh[v];
                }
            }
            copy(t0 + kStages * stride, stage);
            float start[V];
#pragma unroll
            for (int v = 0; v < V; ++v) rp[v] = rp[v] < 0.0f ? kCut : fmaxf(rp[v], kLeast);
            gate_join<V>(sm.join, parity, g.cluster, rank, rp, rh, carry, start);
            parity ^= 1;
            bool finite = true;
#pragma unroll
            for (int v = 0; v < V; ++v) finite = finite && fabsf(start[v]) <= 3.4028235e38f;
            finite = finite || !active;
            if (inside && __all_sync(kFullMask, finite)) {
                if (active) {
#pragma unroll
                    for (int k = 0; k < kGateSteps; ++k) {
                        float y[V];
#pragma unroll
                        for (int v = 0; v < V; ++v) y[v] = fmaf(P[k][v], start[v], h[k][v]);
                        store_word<T, V>(Y + static_cast<size_t>(t0 + k) * p.dim, y);
                    }
                }
            } else {
                SeqAt at = seq;
#pragma unroll
                for (int k = 0; k < kGateSteps; ++k) {
                    if (k >= left) break;
                    if (at.end <= t0 + k) at = seq_at(q, t0 + k);
                    float y[V];
#pragma unroll
                    for (int v = 0; v < V; ++v) y[v] = through(P[k][v], start[v]) + h[k][v];
                    if (active) store_word<T, V>(Y + static_cast<size_t>(t0 + k) * p.dim, y);
                    if (at.end == t0 + k + 1) store_final(at.seq, y);
                }
            }
        }
        cp_async_wait<0>();
    }
}

constexpr int kThreads = 128;

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

template <typename T, int V>
cudaError_t launch_words(const GateArgs &a, cudaStream_t stream) {
    const GateSpans g = gate_spans(a.seq, a.dim, 32 * V);
    return launch_gate_clusters(gate_kernel<T, V>, sizeof(ScanSmem<T, V>), g, stream, a, g);
}

template <typename T>
cudaError_t launch_type(const GateArgs &a, cudaStream_t stream) {
    if constexpr (sizeof(T) == 2) {
        auto words = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; };
        if (a.dim % 2 == 0 && words(a.x) && words(a.f) && words(a.out)) return launch_words<T, 2>(a, stream);
    }
    return launch_words<T, 1>(a, stream);
}

template <typename T>
cudaError_t launch_token_type(const GateArgs &a, cudaStream_t stream) {
    const dim3 grid((a.dim + kThreads - 1) / kThreads, std::min(a.seq.units, 65535));
    gate_token_kernel<T><<<grid, kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

GateSpans gate_spans(const SeqArgs &q, int dim, int channels) {
    GateSpans g{};
    g.tiles = (dim + channels - 1) / channels;
    const int64_t want = 4LL * current_device_sm_count();  // blocks that fill the device
    if (q.cu != nullptr) {
        g.rows = 1;
        g.length = q.tokens;
    } else {
        // rows shorter than a block's tokens share a span, as long as there are blocks enough
        const int64_t per = q.seqlen > 0 ? std::max<int64_t>(1, kGateTokens / q.seqlen) : q.units;
        g.length = static_cast<int>(std::min<int64_t>(per * q.seqlen, q.tokens));
        g.rows = g.length > 0 ? static_cast<int>((q.tokens + g.length - 1) / g.length) : 1;
    }
    g.cluster = 1;
    while (g.cluster < kGateMaxCluster && g.cluster * kGateTokens < g.length &&
           static_cast<int64_t>(g.rows) * g.tiles * g.cluster < want)
        g.cluster *= 2;
    return g;
}

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
