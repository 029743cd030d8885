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

constexpr int kWarps = 4, kThreads = 32 * kWarps;  // a block's warps follow one another along the tokens
constexpr int kSteps = 16;                         // tokens of a warp
constexpr int kTokens = kWarps * kSteps;           // tokens of a block
constexpr int kStages = 3;                         // tiles of x and f in use and under way

__device__ unsigned int g_gate_wait_failures, g_gate_failures_taken;
__global__ void gate_swap_failures() { g_gate_failures_taken = atomicExch(&g_gate_wait_failures, 0u); }

template <typename T, bool kWords>
struct ScanSmem {
    GateJoin<kWarps> join;
    GateTile<T, kTokens> ring[kWords ? kStages : 0][2];
};

template <typename T, bool kWords>
__global__ void __launch_bounds__(kThreads, 4) gate_kernel(const GateArgs p, const GateSpans g) {
    extern __shared__ float4 smem_f4[];
    auto &sm = *reinterpret_cast<ScanSmem<T, kWords> *>(smem_f4);
    const SeqArgs &q = p.seq;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned rank = g.cluster > 1 ? cluster_rank() : 0;
    const int id = blockIdx.x / g.cluster, tile = id % g.tiles, slot = id / g.tiles;
    const Lane<T, kWords> ch(tile, lane, p.dim);
    const float2 low = ch.floats(p.bound, 0.0f), rest = make_float2(1.0f - low.x, 1.0f - low.y);
    const T *const X = static_cast<const T *>(p.x), *const F = static_cast<const T *>(p.f);
    T *const Y = static_cast<T *>(p.out);
    auto init_of = [&](int seq) {
        const long long row = seq_row(q, seq);
        return ch.floats(p.init != nullptr && seq_live(q, seq, row) ? p.init + row * p.dim : nullptr, 0.0f);
    };
    auto store_final = [&](int seq, float2 h) {
        const long long row = seq_row(q, seq);
        if (p.final_state != nullptr && row >= 0) ch.store_floats(p.final_state + row * p.dim, h);
    };
    if (p.final_state != nullptr)  // sequences without tokens keep their starting states
        for_empty_sequences<kWarps>(q, slot * g.cluster + rank, g.width * g.cluster, [&](int s) { store_final(s, init_of(s)); });
    if (g.cluster > 1) gate_join_begin(sm.join);
    if constexpr (kWords) clear_ring(sm.ring, p.dim, tile);
    const int stride = g.cluster * kTokens;  // tokens of a step
    unsigned turn = 0;
    bool lost = false;
    for (int i = slot; i < g.rows; i += g.width) {
        const Span span = gate_span(q, g, i);
        const int first = span.lo + rank * kTokens;  // the block's first token
        auto copy = [&](int step, int stage) {
            if constexpr (kWords) {
                const int t = first + step * stride;
                if (t < span.hi) {
                    copy_tile<kThreads>(sm.ring[stage][0], X, t, 0, span.hi, p.dim, tile);
                    copy_tile<kThreads>(sm.ring[stage][1], F, t, 0, span.hi, p.dim, tile);
                }
                cp_async_commit();
            }
        };
        if constexpr (kWords) {
            for (int k = 0; k < kStages; ++k) copy(k, k);
            cp_async_wait<kStages - 1>();
            __syncthreads();
        }
        float2 carry = both(0.0f);
        SeqAt seq{0, 0, 0};
        int step = 0, stage = 0;
        for (int base = span.lo; base < span.hi; base += stride, ++step, ++turn, stage = stage + 1 == kStages ? 0 : stage + 1) {
            const int t0 = first + step * stride + warp * kSteps, left = span.hi - t0;
            float2 P[kSteps], h[kSteps];
            auto token = [&](int k, float2 &x, float2 &f) {
                if constexpr (kWords) {
                    const GateTile<T, kTokens>(&tiles)[2] = sm.ring[stage];
                    x = tiles[0].at(warp * kSteps + k, lane);
                    f = tiles[1].at(warp * kSteps + k, lane);
                } else {
                    const size_t at = static_cast<size_t>(t0 + k) * p.dim;
                    x = ch.load(X + at);
                    f = ch.load(F + at);
                }
            };
            if (left > 0 && seq.end <= t0) seq = seq_at(q, t0);
            // no sequence starts or ends in the warp's tokens
            const bool inside = left >= kSteps && seq.start < t0 && seq.end > t0 + kSteps;
            GatePair run{both(1.0f), both(0.0f)};
            bool cut = false;
            if (inside) {
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    float2 x, f;
                    token(k, x, f);
                    const Gate2 gate = gate_of(f, low, rest);
                    run.h = __ffma2_rn(gate.a, run.h, __fmul2_rn(gate.u, x));
                    run.P = __fmul2_rn(run.P, gate.a);
                    P[k] = run.P;
                    h[k] = run.h;
                }
            } else {
                SeqAt at = seq;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    if (k < left) {
                        if (at.end <= t0 + k) at = seq_at(q, t0 + k);
                        if (at.start == t0 + k) {
                            run.h = init_of(at.seq);
                            cut = true;
                        }
                        float2 x, f;
                        token(k, x, f);
                        const Gate2 gate = gate_of(f, low, rest);
                        run.h = __ffma2_rn(gate.a, run.h, __fmul2_rn(gate.u, x));
                        run.P = cut ? both(0.0f) : above_zero(__fmul2_rn(run.P, gate.a));
                    }
                    P[k] = run.P;
                    h[k] = run.h;
                }
            }
            if (inside) run.P = above_zero(run.P);
            if constexpr (kWords) cp_async_wait<kStages - 2>();  // the next tiles, which the join's barrier makes everyone's
            const float2 start = gate_join(sm.join, turn, g.cluster, rank, run, carry, lost);
            copy(step + kStages, stage);  // into this step's tiles: all have read them
            if (inside && __all_sync(kFullMask, finite2(start))) {
                if (ch.active[0]) {
                    T *y = Y + static_cast<size_t>(t0) * p.dim;
#pragma unroll
                    for (int k = 0; k < kSteps; ++k, y += p.dim) ch.store(y, __ffma2_rn(P[k], start, h[k]));
                }
            } else {
                SeqAt at = seq;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    if (k >= left) break;
                    if (at.end <= t0 + k) at = seq_at(q, t0 + k);
                    const float2 y = join_any(GatePair{inside ? above_zero(P[k]) : P[k], h[k]}, start);
                    if (ch.active[0]) ch.store(Y + static_cast<size_t>(t0 + k) * p.dim, y);
                    if (at.end == t0 + k + 1) store_final(at.seq, y);
                }
            }
        }
        cp_async_wait<0>();
        __syncthreads();  // (the ring is filled anew)
    }
    if (g.cluster > 1) {
        if (lost && threadIdx.x == 0) atomicAdd(&g_gate_wait_failures, 1u);
        cluster_barrier();
    }
}

constexpr int kTokenThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kTokenThreads) gate_token_kernel(const GateArgs p) {
    const int d = blockIdx.x * kTokenThreads + threadIdx.x;
    if (d >= p.dim) return;
    const float low = p.bound != nullptr ? p.bound[d] : 0.0f;
    for (unsigned i = blockIdx.y; i < static_cast<unsigned>(p.seq.units); i += gridDim.y) {
        const long long row = seq_row(p.seq, i);
        if (row < 0) continue;
        const size_t at = static_cast<size_t>(i) * p.dim + d;
        const Gate2 g = gate_of(both(to_f32<T>(static_cast<const T *>(p.f)[at])), both(low), both(1.0f - low));
        const float x = to_f32<T>(static_cast<const T *>(p.x)[at]);
        const float h = fmaf(g.a.x, p.init[row * p.dim + d], g.u.x * x);
        p.final_state[row * p.dim + d] = h;
        static_cast<T *>(p.out)[at] = from_f32<T>(h);
    }
}

template <typename T>
cudaError_t launch_type(const GateArgs &a, cudaStream_t stream) {
    const GateSpans g = gate_spans(a.seq, a.dim, kTokens);
    if (a.dim * sizeof(T) % 16 == 0 && aligned16(a.x) && aligned16(a.f) && aligned16(a.out))
        return launch_gate_clusters(gate_kernel<T, true>, kThreads, sizeof(ScanSmem<T, true>), g, stream, a, g);
    return launch_gate_clusters(gate_kernel<T, false>, kThreads, sizeof(ScanSmem<T, false>), g, stream, a, g);
}

template <typename T>
cudaError_t launch_token_type(const GateArgs &a, cudaStream_t stream) {
    const dim3 grid((a.dim + kTokenThreads - 1) / kTokenThreads, std::min(a.seq.units, 65535));
    gate_token_kernel<T><<<grid, kTokenThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

GateSpans gate_spans(const SeqArgs &q, int dim, int tokens) {
    GateSpans g{};
    g.tiles = (dim + kGateChannels - 1) / kGateChannels;
    const int64_t want = 4LL * current_device_sm_count();  // blocks that fill the device
    if (q.cu != nullptr) {
        g.rows = 1;
        g.length = q.tokens;
    } else {
        // rows shorter than a block's tokens share a span
        const int64_t per = q.seqlen > 0 ? std::max<int64_t>(1, tokens / q.seqlen) : q.units;
        g.length = static_cast<int>(std::min<int64_t>(per * q.seqlen, q.tokens));
        g.rows = g.length > 0 ? static_cast<int>((static_cast<int64_t>(q.tokens) + g.length - 1) / g.length) : 1;
    }
    g.cluster = 1;
    while (g.cluster < kGateMaxCluster && g.cluster * tokens < g.length &&
           static_cast<int64_t>(g.rows) * g.tiles * g.cluster < want)
        g.cluster *= 2;
    const int64_t most = std::max<int64_t>(1, (int64_t(1) << 30) / (static_cast<int64_t>(g.tiles) * g.cluster));
    g.width = static_cast<int>(std::min<int64_t>(g.rows, most));
    return g;
}

cudaError_t gate_take_wait_failures(unsigned int *count) {
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) {
        gate_swap_failures<<<1, 1>>>();
        e = cudaGetLastError();
    }
    return e == cudaSuccess ? cudaMemcpyFromSymbol(count, g_gate_failures_taken, sizeof(*count)) : e;
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
