// gated_recurrence_grad.cu -- GatedRecurrenceGradFn for sm_100a.
//
// Math, per channel, from a sequence's last token to its first, with c the
// gradient that reaches the state behind a token (d_final_state at first):
//   G_t = dy_t + c,  dx_t = (1 - a_t) G_t,  c <- a_t G_t,
//   df_t = G_t (h_(t-1) - x_t) (1 - a_t) sigmoid(f_t),
//   d_bound += G_t (h_(t-1) - x_t) sigmoid(-f_t).
// The recurrence of c is scanned as xm_gate.cuh says, from the last token to the
// first.
#include <algorithm>

#include "xm_common.cuh"
#include "xm_gate.cuh"
#include "xm_kernels.h"
#include "xm_sequences.cuh"

namespace xm {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;  // a block's warps follow one another along the tokens
constexpr int kSteps = 8;                          // tokens of a warp
constexpr int kTokens = kWarps * kSteps;           // tokens of a block
constexpr int kStages = 3;                         // tiles in use and under way

__device__ unsigned int g_gate_grad_wait_failures, g_gate_grad_failures_taken;
__global__ void gate_grad_swap_failures() { g_gate_grad_failures_taken = atomicExch(&g_gate_grad_wait_failures, 0u); }

template <typename T, bool kWords>
struct GradSmem {
    GateJoin<kWarps> join;
    GateTile<T, kTokens> ring[kWords ? kStages : 0][4];  // dy, x, f, and y of the token before
};

// part: [width x cluster][dim] sums of d_bound, or null.
template <typename T, bool kWords>
__global__ void __launch_bounds__(kThreads, 2) gate_grad_kernel(const GateGradArgs p, const GateSpans g, float *part) {
    extern __shared__ float4 smem_f4[];
    auto &sm = *reinterpret_cast<GradSmem<T, kWords> *>(smem_f4);
    const SeqArgs &q = p.seq;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned rank = g.cluster > 1 ? cluster_rank() : 0;
    const int id = blockIdx.x / g.cluster, tile = id % g.tiles, slot = id / g.tiles;
    const Lane<T, kWords> ch(tile, lane, p.dim);
    const float2 low = ch.floats(p.bound, 0.0f), rest = make_float2(1.0f - low.x, 1.0f - low.y);
    const T *const DY = static_cast<const T *>(p.dy), *const X = static_cast<const T *>(p.x),
                   *const F = static_cast<const T *>(p.f), *const H = static_cast<const T *>(p.y);
    T *const DX = static_cast<T *>(p.dx), *const DF = static_cast<T *>(p.df);
    auto state_row = [&](const float *base, int seq) {
        return ch.floats(base != nullptr ? base + static_cast<size_t>(seq) * p.dim : nullptr, 0.0f);
    };
    auto store_dinit = [&](int seq, float2 c) {
        if (p.dinit != nullptr) ch.store_floats(p.dinit + static_cast<size_t>(seq) * p.dim, c);
    };
    if (p.dinit != nullptr)  // sequences without tokens: the gradient passes through
        for_empty_sequences<kWarps>(q, slot * g.cluster + rank, g.width * g.cluster,
                            [&](int s) { store_dinit(s, state_row(p.dfinal, s)); });
    if (g.cluster > 1) gate_join_begin(sm.join);
    if constexpr (kWords) clear_ring(sm.ring, p.dim, tile);
    const int stride = g.cluster * kTokens;  // tokens of a step
    float2 dlow = both(0.0f);                    // sum of da (1 - a)
    unsigned turn = 0;
    bool lost = false;
    for (int i = slot; i < g.rows; i += g.width) {
        const Span span = gate_span(q, g, i);
        const int first = span.hi - (rank + 1) * kTokens;  // the block's lowest token of the first step
        auto copy = [&](int step, int stage) {
            if constexpr (kWords) {
                const int t = first - step * stride;
                if (t + kTokens > span.lo) {
                    copy_tile<kThreads>(sm.ring[stage][0], DY, t, span.lo, span.hi, p.dim, tile);
                    copy_tile<kThreads>(sm.ring[stage][1], X, t, span.lo, span.hi, p.dim, tile);
                    copy_tile<kThreads>(sm.ring[stage][2], F, t, span.lo, span.hi, p.dim, tile);
                    copy_tile<kThreads>(sm.ring[stage][3], H, t - 1, span.lo, span.hi, p.dim, tile);
                }
                cp_async_commit();
            }
        };
        if constexpr (kWords) {
            for (int k = 0; k < kStages - 1; ++k) copy(k, k);
            cp_async_wait<kStages - 2>();
            __syncthreads();
        }
        float2 carry = both(0.0f);
        SeqAt seq{0, span.hi, 0};
        int step = 0, stage = 0;
        for (int base = span.lo; base < span.hi; base += stride, ++step, ++turn, stage = stage + 1 == kStages ? 0 : stage + 1) {
            // the warp's tokens are t1, t1 - 1, ...; k counts them
            const int row1 = kTokens - 1 - warp * kSteps;
            const int t1 = first - step * stride + row1, left = t1 + 1 - span.lo;
            auto load = [&](int which, const T *base_ptr, int k, int back) {
                if constexpr (kWords) return sm.ring[stage][which].at(row1 - k, lane);
                else return ch.load(base_ptr + static_cast<size_t>(t1 - k - back) * p.dim);
            };
            if (left > 0 && seq.start > t1) seq = seq_at(q, t1);
            // no sequence starts or ends in the warp's tokens
            const bool inside = left >= kSteps && seq.end > t1 + 1 && seq.start < t1 + 1 - kSteps;
            float2 P[kSteps], G[kSteps], u[kSteps], r[kSteps];  // P and G before the start is known
            GatePair run{both(1.0f), both(0.0f)};
            bool cut = false;
            if (inside) {
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    const Gate2 gate = gate_of(load(2, F, k, 0), low, rest);
                    u[k] = gate.u;
                    r[k] = gate.r;
                    P[k] = run.P;
                    G[k] = __fadd2_rn(load(0, DY, k, 0), run.h);
                    run.h = __fmul2_rn(gate.a, G[k]);
                    run.P = __fmul2_rn(run.P, gate.a);
                }
            } else {
                SeqAt at = seq;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    u[k] = r[k] = P[k] = G[k] = both(0.0f);
                    if (k < left) {
                        if (at.start > t1 - k) at = seq_at(q, t1 - k);
                        if (at.end == t1 - k + 1) {
                            run.h = state_row(p.dfinal, at.seq);
                            cut = true;
                        }
                        const Gate2 gate = gate_of(load(2, F, k, 0), low, rest);
                        u[k] = gate.u;
                        r[k] = gate.r;
                        if (cut) run.P = both(0.0f);
                        P[k] = run.P;
                        G[k] = __fadd2_rn(load(0, DY, k, 0), run.h);
                        run.h = __fmul2_rn(gate.a, G[k]);
                        run.P = cut ? both(0.0f) : above_zero(__fmul2_rn(run.P, gate.a));
                    }
                }
            }
            if (inside) run.P = above_zero(run.P);
            if constexpr (kWords) cp_async_wait<kStages - 3>();  // the next tiles, which the join's barrier makes everyone's
            const float2 start = gate_join(sm.join, turn, g.cluster, rank, run, carry, lost);
            copy(step + kStages - 1, stage == 0 ? kStages - 1 : stage - 1);  // into the tiles of the step before: all are done with them
            auto finish = [&](int k, float2 Gk, float2 before) {
                const size_t at = static_cast<size_t>(t1 - k) * p.dim;
                const float2 x = load(1, X, k, 0);
                const float2 diff = make_float2(before.x - x.x, before.y - x.y);
                const float2 w = __fmul2_rn(__fmul2_rn(Gk, diff), u[k]);
                if (ch.active[0]) {
                    ch.store(DX + at, __fmul2_rn(u[k], Gk));
                    ch.store(DF + at, __fmul2_rn(w, r[k]));
                }
                dlow = __fadd2_rn(dlow, w);
            };
            if (inside && __all_sync(kFullMask, finite2(start))) {
#pragma unroll
                for (int k = 0; k < kSteps; ++k) finish(k, __ffma2_rn(P[k], start, G[k]), load(3, H, k, 1));
            } else {
                SeqAt at = seq;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    if (k >= left) break;
                    if (at.start > t1 - k) at = seq_at(q, t1 - k);
                    const float2 Gk = join_any(GatePair{inside ? above_zero(P[k]) : P[k], G[k]}, start);
                    const bool begins = at.start == t1 - k;
                    finish(k, Gk, begins ? state_row(p.init, at.seq) : load(3, H, k, 1));
                    if (begins) store_dinit(at.seq, __fmul2_rn(__ffma2_rn(rest, r[k], low), Gk));
                }
            }
        }
        cp_async_wait<0>();
        __syncthreads();  // (the ring is filled anew)
    }
    if (g.cluster > 1) {
        if (lost && threadIdx.x == 0) atomicAdd(&g_gate_grad_wait_failures, 1u);
        cluster_barrier();
    }
    if (part != nullptr) {  // the block's sum, the warps' added in order
        sm.join.warp[0][warp][lane].h = dlow;
        __syncthreads();
        if (warp == 0) {
            float2 sum = both(0.0f);
            for (int w = 0; w < kWarps; ++w) sum = __fadd2_rn(sum, sm.join.warp[0][w][lane].h);
            sum = make_float2(sum.x / rest.x, sum.y / rest.y);  // da (1 - a) = da (1 - bound) sigmoid(-f)
            ch.store_floats(part + static_cast<size_t>(slot * g.cluster + rank) * p.dim, sum);
        }
    }
}

template <typename T>
cudaError_t launch_type(const GateGradArgs &a, float *part, const GateSpans &g, cudaStream_t stream) {
    if (a.dim * sizeof(T) % 16 == 0 && aligned16(a.dy) && aligned16(a.x) && aligned16(a.f) && aligned16(a.y) &&
        aligned16(a.dx) && aligned16(a.df))
        return launch_gate_clusters(gate_grad_kernel<T, true>, kThreads, sizeof(GradSmem<T, true>), g, stream, a, g, part);
    return launch_gate_clusters(gate_grad_kernel<T, false>, kThreads, sizeof(GradSmem<T, false>), g, stream, a, g, part);
}

}  // namespace

cudaError_t gate_grad_take_wait_failures(unsigned int *count) {
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) {
        gate_grad_swap_failures<<<1, 1>>>();
        e = cudaGetLastError();
    }
    return e == cudaSuccess ? cudaMemcpyFromSymbol(count, g_gate_grad_failures_taken, sizeof(*count)) : e;
}

size_t gated_recurrence_grad_workspace(const GateGradArgs &a) {
    if (!a.want_dbound || a.dim == 0) return 0;
    const GateSpans g = gate_spans(a.seq, a.dim, kTokens);
    const size_t parts = static_cast<size_t>(g.width) * g.cluster;
    return parts > 1 ? parts * a.dim * sizeof(float) : 0;
}

cudaError_t launch_gated_recurrence_grad(const GateGradArgs &a, void *workspace, cudaStream_t stream) {
    const GateSpans g = gate_spans(a.seq, a.dim, kTokens);
    const int parts = g.width * g.cluster;
    float *part = a.dbound == nullptr ? nullptr : parts > 1 ? static_cast<float *>(workspace) : a.dbound;
    cudaError_t e;
    switch (a.io) {
        case IoType::kBF16: e = launch_type<__nv_bfloat16>(a, part, g, stream); break;
        case IoType::kF16: e = launch_type<__half>(a, part, g, stream); break;
        default: e = launch_type<float>(a, part, g, stream);
    }
    if (e != cudaSuccess || a.dbound == nullptr || parts == 1) return e;
    return launch_column_sums(part, nullptr, parts, a.dim, a.dbound, nullptr, stream);
}

}  // namespace xm
