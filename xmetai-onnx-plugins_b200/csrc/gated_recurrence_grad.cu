// gated_recurrence_grad.cu -- GatedRecurrenceGradFn for sm_100a.
//
// Math, per channel, from a sequence's last token to its first, with c the
// gradient that reaches the state behind a token (d_final_state at first):
//   G_t = dy_t + c,  dx_t = (1 - a_t) G_t,  c <- a_t G_t,
//   df_t = G_t (h_(t-1) - x_t) (1 - a_t) sigmoid(f_t),
//   d_bound += G_t (h_(t-1) - x_t) sigmoid(-f_t).
// The recurrence of c is walked as xm_gate.cuh says, from the last token to the
// first.
#include <algorithm>
#include <climits>

#include "xm_common.cuh"
#include "xm_gate.cuh"
#include "xm_kernels.h"
#include "xm_sequences.cuh"

namespace xm {
namespace {

constexpr int kMaxParts = 1024;  // partial sums of d_bound per channel

// Tokens of a group: in a ring, what is kept of more does not fit beside four blocks; in a segment 16 take as long, with
// twice the instructions to fetch in short calls.
constexpr int kGroup = 8;

template <typename T, int kRow>
using GradTile = GateTile<T, kGroup, kRow>;

// Segments of an SM: one wave, as many as it has room for (16384 x 4096 packed takes 188 us; with six stages, of which
// eight fit, 197).
template <typename T>
constexpr int kPerSm = sizeof(T) == 4 ? 7 : 12;

// Groups in use and under way, of the tensors f, dy; x, and y of the token before.
constexpr int kStages = 4;

template <typename T, int kRow>
__device__ __forceinline__ float2 state_row(const GateGradArgs &p, const Lane<T, kRow> &ch, const float *base, int seq) {
    return ch.floats(base != nullptr ? base + static_cast<size_t>(seq) * p.dim : nullptr, 0.0f);
}
template <typename T, int kRow>
__device__ __forceinline__ void store_dinit(const GateGradArgs &p, const Lane<T, kRow> &ch, int seq, float2 c) {
    if (p.dinit != nullptr) ch.store_floats(p.dinit + static_cast<size_t>(seq) * p.dim, c);
}
// Sequences without tokens: the gradient passes through; warp of warps with the same channels.
template <typename T, int kRow>
__device__ __forceinline__ void pass_empty(const GateGradArgs &p, const Lane<T, kRow> &ch, int warp, int warps) {
    if (p.dinit != nullptr)
        for_empty_sequences(p.seq, warp, warps, [&](int s) { store_dinit(p, ch, s, state_row(p, ch, p.dfinal, s)); });
}

// A warp walks segment j of a span. kEnds: the first pass. first_pass(): it is through; nothing of it is read before.
// dlow: sum of da sigmoid(-f).
template <typename T, int kRow, bool kEnds, int kStages, int kTensors, typename Wait>
__device__ __forceinline__ void walk_segment(const GateGradArgs &p, const GateCut &g, GradTile<T, kRow> (*ring)[kTensors],
                                             const Lane<T, kRow> &ch, int tile, float2 low, float2 rest, Span span,
                                             int length, int j, const GatePairs &pairs, float2 &dlow, Wait &&first_pass) {
    const SeqArgs &q = p.seq;
    const T *const DY = static_cast<const T *>(p.dy), *const X = static_cast<const T *>(p.x),
                   *const F = static_cast<const T *>(p.f), *const H = static_cast<const T *>(p.y);
    T *const DX = static_cast<T *>(p.dx), *const DF = static_cast<T *>(p.df);
    const int s0 = span.lo + min(static_cast<long long>(j) * length, static_cast<long long>(max(span.hi - span.lo, 0)));
    const int s1 = min(static_cast<long long>(s0) + length, static_cast<long long>(span.hi));
    if (s0 >= s1) return;
    int end = s1;
    SeqAt seq = seq_at(q, kEnds ? s0 : s1 - 1);
    if (kEnds) {
        if (seq.start >= s0) return;  // no sequence enters the segment
        end = min(s1, seq.end);
    }
    auto copy = [&](int hi, int stage) {
        const int t = hi - kGroup;
        if (hi > s0) {
            copy_tile(ring[stage][0], F, t, s0, s1, p.dim, tile);
            copy_tile(ring[stage][1], DY, t, s0, s1, p.dim, tile);
            if constexpr (!kEnds) {
                copy_tile(ring[stage][2], X, t, s0, s1, p.dim, tile);
                copy_tile(ring[stage][3], H, t - 1, span.lo, s1, p.dim, tile);
            }
        }
        cp_async_commit();
    };
    for (int k = 0; k < kStages - 1; ++k) copy(end - k * kGroup, k);
    first_pass();
    float2 c = both(0.0f), P = both(1.0f);
    if (seq.end <= end) {  // (== unless the offsets descend)
        c = state_row(p, ch, p.dfinal, seq.seq);
    } else if (!kEnds && j + 1 < g.segments) {  // what comes from the segments behind
        int k = min(max(seq.end - 1 - span.lo, 0) / length, g.segments - 1);
        c = pairs.h(k);
        for (--k; k > j; --k) c = __ffma2_rn(pairs.P(k), c, pairs.h(k));
    }
    SeqAt next{0, 0, 0};
    float2 next_c = both(0.0f), first_h = both(0.0f);
    auto look_ahead = [&] {  // this sequence's starting state, and the sequence before it
        if (kEnds || seq.start < s0) return;
        first_h = state_row(p, ch, p.init, seq.seq);
        if (seq.start == s0) return;
        next = seq_before(q, seq);
        next_c = state_row(p, ch, p.dfinal, next.seq);
    };
    look_ahead();
    int stage = 0;
    for (int hi = end; hi > s0; hi -= kGroup) {
        cp_async_wait<kStages - 2>();
        __syncwarp();
        copy(hi - (kStages - 1) * kGroup, stage == 0 ? kStages - 1 : stage - 1);  // read by all a group ago
        // token hi - 1 - k of a tensor
        auto load = [&](int which, const T *base, int k, int back) {
            return ring[stage][which].at(kGroup - 1 - k, shift_of<T, kRow>(base, hi - 1 - k - back, p.dim));
        };
        const int last = min(kGroup, hi - s0);
        if constexpr (kEnds) {
            float2 a[kGroup], b[kGroup];  // (of no meaning before the segment)
#pragma unroll
            for (int k = 0; k < kGroup; ++k) {
                a[k] = gate_of(load(0, F, k, 0), low, rest).a;
                b[k] = __fmul2_rn(a[k], load(1, DY, k, 0));
            }
#pragma unroll
            for (int k = 0; k < kGroup; ++k) {
                if (k >= last) continue;
                c = __ffma2_rn(a[k], c, b[k]);
                P = __fmul2_rn(P, a[k]);
            }
        } else {
            float2 G[kGroup], take[kGroup], keep[kGroup];  // (of no meaning before the segment)
#pragma unroll
            for (int k = 0; k < kGroup; ++k) {
                const Gate2 gate = gate_of(load(0, F, k, 0), low, rest);
                G[k] = gate.a;
                take[k] = gate.take;
                keep[k] = gate.keep;
            }
            T *dx = DX + static_cast<size_t>(hi - 1) * p.dim, *df = DF + static_cast<size_t>(hi - 1) * p.dim;
            auto token = [&](int k, float2 before) {
                const float2 x = load(2, X, k, 0);
                const float2 diff = __fadd2_rn(before, make_float2(-x.x, -x.y));
                dlow = __fadd2_rn(dlow, __fmul2_rn(__fmul2_rn(G[k], diff), take[k]));
                const float2 d = __fmul2_rn(__fmul2_rn(G[k], rest), take[k]);
                if (ch.active[0]) {
                    ch.store(dx, d);
                    ch.store(df, __fmul2_rn(__fmul2_rn(d, diff), keep[k]));
                }
            };
            if (last == kGroup && seq.start < hi - kGroup) {
#pragma unroll
                for (int k = 0; k < kGroup; ++k) {
                    const float2 v = __fadd2_rn(load(1, DY, k, 0), c);
                    c = __fmul2_rn(G[k], v);
                    G[k] = v;
                }
#pragma unroll
                for (int k = 0; k < kGroup; ++k, dx -= p.dim, df -= p.dim) token(k, load(3, H, k, 1));
            } else {
                for (int k0 = 0; k0 < last;) {  // the tokens of a sequence, k0 .. k1 - 1
                    const int end = hi - seq.start, k1 = end > k0 && end < last ? end : last;
#pragma unroll
                    for (int k = 0; k < kGroup; ++k) {
                        if (k < k0 || k >= k1) continue;
                        const float2 v = __fadd2_rn(load(1, DY, k, 0), c);
                        c = __fmul2_rn(G[k], v);
                        G[k] = v;
                        token(k, end == k1 && k == k1 - 1 ? first_h : load(3, H, k, 1));
                        dx -= p.dim;
                        df -= p.dim;
                    }
                    k0 = k1;
                    if (end != k1) continue;
                    store_dinit(p, ch, seq.seq, c);
                    seq = next;
                    c = next_c;
                    if (hi - k1 > s0) look_ahead();
                }
            }
        }
        stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    if constexpr (kEnds) {
        pairs.P(j) = above_zero(P);
        pairs.h(j) = c;
    }
    cp_async_wait<0>();
    __syncwarp();  // (the ring is filled anew)
}

// A segment to each warp. kEnds: the first pass over segments (all but a span's first).
// part: [width x segments][dim] sums of d_bound, or null. Both passes read f and dy: 16384 x 4096 packed in bf16, 1.07 GB,
// 188 us, 87 % of copy bandwidth.
template <typename T, int kRow, bool kEnds>
__global__ void __launch_bounds__(32, 8) gate_grad_kernel(const GateGradArgs p, const GateCut g, float *part) {
    extern __shared__ float4 smem_f4[];
    dependents_may_launch();
    const int tile = blockIdx.x % g.tiles, segs = kEnds ? g.segments - 1 : g.segments;
    const int j = blockIdx.x / g.tiles % segs + (kEnds ? 1 : 0), slot = blockIdx.x / g.tiles / segs;
    const Lane<T, kRow> ch(tile, threadIdx.x & 31, p.dim);
    const float2 low = ch.floats(p.bound, 0.0f), rest = make_float2(1.0f - low.x, 1.0f - low.y);
    bool waited = kEnds;
    auto first_pass = [&] {
        if (!waited) wait_for_before();
        waited = true;
    };
    if (!kEnds) pass_empty(p, ch, slot * segs + j, g.width * segs);
    float2 dlow = both(0.0f);
    for (int i = slot; i < g.spans; i += g.width) {
        const Span span = gate_span(p.seq, g, i);
        constexpr int kTensors = kEnds ? 2 : 4;
        walk_segment<T, kRow, kEnds, kStages, kTensors>(
            p, g, reinterpret_cast<GradTile<T, kRow>(*)[kTensors]>(smem_f4), ch, tile, low, rest, span,
            segment_length(g, span), j, global_pairs(g, i, tile), dlow, first_pass);
    }
    first_pass();  // (also warps without tokens: what follows waits for this kernel only)
    if (!kEnds && part != nullptr) ch.store_floats(part + static_cast<size_t>(slot * segs + j) * p.dim, dlow);
}

// Both passes in one block, a segment to each of its warps: as many as have room for their copies.
template <typename T>
struct GradBlock {
    static constexpr int kWarps = sizeof(T) == 4 ? 6 : 8, kStages = sizeof(T) == 4 ? 4 : 6;
};
constexpr int kShortest = 24;  // tokens of a row that a block shares (50 x 386 in float32: 9.7 us, by a warp alone 13.9)
template <typename T, int kRow>
struct GradBlockSmem {
    GradTile<T, kRow> ring[GradBlock<T>::kWarps][GradBlock<T>::kStages][4];
    BlockPairs<GradBlock<T>::kWarps> pairs;
};

// part: [width][dim] sums of d_bound, or null.
template <typename T, int kRow>
__global__ void __launch_bounds__(32 * GradBlock<T>::kWarps, 1) gate_grad_block_kernel(const GateGradArgs p, const GateCut g,
                                                                                  float *part) {
    extern __shared__ float4 smem_f4[];
    constexpr int kWarps = GradBlock<T>::kWarps, kStages = GradBlock<T>::kStages;
    auto &sm = *reinterpret_cast<GradBlockSmem<T, kRow> *>(smem_f4);
    dependents_may_launch();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tile = blockIdx.x % g.tiles, slot = blockIdx.x / g.tiles;
    const Lane<T, kRow> ch(tile, lane, p.dim);
    const float2 low = ch.floats(p.bound, 0.0f), rest = make_float2(1.0f - low.x, 1.0f - low.y);
    pass_empty(p, ch, slot * kWarps + warp, g.width * kWarps);
    float2 dlow = both(0.0f);
    for (int i = slot; i < g.spans; i += g.width) {
        const Span span = gate_span(p.seq, g, i);
        const int length = segment_length(g, span);
        const GatePairs pairs = sm.pairs.view();
        if (warp > 0)
            walk_segment<T, kRow, true, kStages, 4>(p, g, sm.ring[warp], ch, tile, low, rest, span, length, warp, pairs,
                                                      dlow, [] {});
        __syncthreads();
        walk_segment<T, kRow, false, kStages, 4>(p, g, sm.ring[warp], ch, tile, low, rest, span, length, warp, pairs, dlow,
                                                   [] {});
        __syncthreads();
    }
    if (part != nullptr) {  // the block's sum, the warps' added in order
        sm.pairs.h[warp][lane] = dlow;
        __syncthreads();
        if (warp == 0) {
            float2 sum = sm.pairs.h[0][lane];
            for (int w = 1; w < kWarps; ++w) sum = __fadd2_rn(sum, sm.pairs.h[w][lane]);
            ch.store_floats(part + static_cast<size_t>(slot) * p.dim, sum);
        }
    }
}

template <typename T, int kRow, int kWarps>
struct GradRingSmem {
    static constexpr int kStages = kWarps == 8 && sizeof(T) == 2 ? 3 : 2;
    Ring<kWarps> hand;
    GateTile<T, kGroup, kRow> ring[kWarps][kStages][4];  // f, dy, x, and y of the token before
};

// A row to a block, its warps' groups in turn; everything moves once. 8 x 2048 x 4096 in bf16, 805 MB: 131 us, 94 % of copy
// bandwidth. part: [width][dim] sums of d_bound, or null.
template <typename T, int kRow, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, 16 / kWarps) gate_grad_ring_kernel(const GateGradArgs p, const GateCut g,
                                                                           float *part) {
    extern __shared__ float4 smem_f4[];
    auto &sm = *reinterpret_cast<GradRingSmem<T, kRow, kWarps> *>(smem_f4);
    constexpr int kStages = GradRingSmem<T, kRow, kWarps>::kStages;
    dependents_may_launch();
    const SeqArgs &q = p.seq;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tile = blockIdx.x % g.tiles, slot = blockIdx.x / g.tiles;
    const Lane<T, kRow> ch(tile, lane, p.dim);
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
        for_empty_sequences(q, slot * kWarps + warp, g.width * kWarps,
                            [&](int s) { store_dinit(s, state_row(p.dfinal, s)); });
    float2 dlow = both(0.0f);  // sum of da sigmoid(-f)
    for (int i = slot; i < g.spans; i += g.width) {
        const Span span = gate_span(q, g, i);
        constexpr int kTurn = kWarps * kGroup;  // tokens of a round
        const int first = span.hi - warp * kGroup;
        auto copy = [&](int hi, int stage) {
            const int t = hi - kGroup;
            if (hi > span.lo) {
                copy_tile(sm.ring[warp][stage][0], F, t, span.lo, span.hi, p.dim, tile);
                copy_tile(sm.ring[warp][stage][1], DY, t, span.lo, span.hi, p.dim, tile);
                copy_tile(sm.ring[warp][stage][2], X, t, span.lo, span.hi, p.dim, tile);
                copy_tile(sm.ring[warp][stage][3], H, t - 1, span.lo, span.hi, p.dim, tile);
            }
            cp_async_commit();
        };
        for (int k = 0; k < kStages - 1; ++k) copy(first - k * kTurn, k);
        SeqAt seq{0, span.hi, 0};
        int stage = 0;
        for (int hi = first; hi > span.lo; hi -= kTurn) {
            cp_async_wait<kStages - 2>();
            __syncwarp();
            copy(hi - (kStages - 1) * kTurn, stage == 0 ? kStages - 1 : stage - 1);  // read by all a round ago
            // token hi - 1 - k of a tensor
            auto load = [&](int which, const T *base, int k, int back) {
                return sm.ring[warp][stage][which].at(kGroup - 1 - k, shift_of<T, kRow>(base, hi - 1 - k - back, p.dim));
            };
            if (seq.start >= hi) seq = seq_at(q, hi - 1);
            const bool more = hi - kGroup > span.lo;  // a group before
            const int next = warp + 1 == kWarps ? 0 : warp + 1;
            float2 P[kGroup], G[kGroup], take[kGroup], keep[kGroup];  // (of no meaning before the span)
#pragma unroll
            for (int k = 0; k < kGroup; ++k) {
                const Gate2 gate = gate_of(load(0, F, k, 0), low, rest);
                P[k] = gate.a;
                take[k] = gate.take;
                keep[k] = gate.keep;
            }
            T *dx = DX + static_cast<size_t>(hi - 1) * p.dim, *df = DF + static_cast<size_t>(hi - 1) * p.dim;
            auto token = [&](int k, float2 Gk, float2 before) {
                const float2 x = load(2, X, k, 0);
                const float2 diff = __fadd2_rn(before, make_float2(-x.x, -x.y));
                dlow = __fadd2_rn(dlow, __fmul2_rn(__fmul2_rn(Gk, diff), take[k]));
                const float2 d = __fmul2_rn(__fmul2_rn(Gk, rest), take[k]);
                if (ch.active[0]) {
                    ch.store(dx, d);
                    ch.store(df, __fmul2_rn(__fmul2_rn(d, diff), keep[k]));
                }
            };
            // (whether a group takes and gives depends on hi alone, so that offsets that descend leave nobody waiting)
            if (hi < span.hi && hi - kGroup >= span.lo && seq.end > hi && seq.start < hi - kGroup) {
                // P[k] becomes the product up to and with token k, G[k] is run from zero
                float2 c = both(0.0f);
#pragma unroll
                for (int k = 0; k < kGroup; ++k) {
                    G[k] = __fadd2_rn(load(1, DY, k, 0), c);
                    c = __fmul2_rn(P[k], G[k]);
                    if (k > 0) P[k] = __fmul2_rn(P[k], P[k - 1]);
                }
                const float2 start = sm.hand.take(warp);
                if (!__all_sync(kFullMask, finite2(start))) {  // (also for what lanes without channels find)
#pragma unroll
                    for (int k = 0; k < kGroup; ++k) P[k] = above_zero(P[k], start);
                }
                if (more) sm.hand.give(next, __ffma2_rn(P[kGroup - 1], start, c));
#pragma unroll
                for (int k = 0; k < kGroup; ++k, dx -= p.dim, df -= p.dim)
                    token(k, k == 0 ? __fadd2_rn(G[0], start) : __ffma2_rn(P[k - 1], start, G[k]), load(3, H, k, 1));
            } else {
                const int last = min(kGroup, hi - span.lo);
                float2 c = hi < span.hi ? sm.hand.take(warp) : both(0.0f);
                for (int k0 = 0; k0 < last;) {  // the tokens of a sequence, k0 .. k1 - 1
                    if (seq.start > hi - 1 - k0) seq = seq_at(q, hi - 1 - k0);
                    if (seq.end == hi - k0) c = state_row(p.dfinal, seq.seq);
                    const int end = hi - seq.start, k1 = end > k0 && end < last ? end : last;
                    float2 before = both(0.0f);
                    if (end == k1) before = state_row(p.init, seq.seq);
#pragma unroll
                    for (int k = 0; k < kGroup; ++k) {
                        if (k < k0 || k >= k1) continue;
                        const float2 Gk = __fadd2_rn(load(1, DY, k, 0), c);
                        c = __fmul2_rn(P[k], Gk);
                        token(k, Gk, end == k1 && k == k1 - 1 ? before : load(3, H, k, 1));
                        dx -= p.dim;
                        df -= p.dim;
                    }
                    if (end == k1) store_dinit(seq.seq, c);
                    k0 = k1;
                }
                if (more) sm.hand.give(next, c);
            }
            stage = stage + 1 == kStages ? 0 : stage + 1;
        }
        cp_async_wait<0>();
        __syncthreads();  // the rings are filled anew, the hands start anew
    }
    if (part != nullptr) {  // the block's sum, the warps' added in order
        sm.hand.slot[warp][lane] = dlow;
        __syncthreads();
        if (warp == 0) {
            float2 sum = sm.hand.slot[0][lane];
            for (int w = 1; w < kWarps; ++w) sum = __fadd2_rn(sum, sm.hand.slot[w][lane]);
            ch.store_floats(part + static_cast<size_t>(slot) * p.dim, sum);
        }
    }
}

template <typename T, int kRow>
cudaError_t launch_row(const GateGradArgs &a, const GateCut &g, float *part, cudaStream_t stream) {
    if (g.ring == 4)
        return launch_gate<gate_grad_ring_kernel<T, kRow, 4>>(4, sizeof(GradRingSmem<T, kRow, 4>), g, 1, false, stream,
                           a, g, part);
    if (g.ring == 8)
        return launch_gate<gate_grad_ring_kernel<T, kRow, 8>>(8, sizeof(GradRingSmem<T, kRow, 8>), g, 1, false, stream,
                           a, g, part);
    if (g.block != 0)
        return launch_gate<gate_grad_block_kernel<T, kRow>>(g.block, sizeof(GradBlockSmem<T, kRow>), g, 1, false, stream,
                                                              a, g, part);
    constexpr size_t kSmem = kStages * sizeof(GradTile<T, kRow>);  // of one tensor
    if (g.segments > 1) {
        const cudaError_t e = launch_gate<gate_grad_kernel<T, kRow, true>>(1, 2 * kSmem, g,
                                          g.segments - 1, false, stream, a, g, part);
        if (e != cudaSuccess) return e;
    }
    return launch_gate<gate_grad_kernel<T, kRow, false>>(1, 4 * kSmem, g, g.segments,
                       gate_behind(g), stream, a, g, part);
}

template <typename T>
cudaError_t launch_type(const GateGradArgs &a, const GateCut &g, float *part, cudaStream_t stream) {
    switch (row_of(a.dim, sizeof(T), {a.dy, a.x, a.f, a.y, a.dx, a.df})) {
        case kRowWords: return launch_row<T, kRowWords>(a, g, part, stream);
        case kRowPairs: return launch_row<T, kRowPairs>(a, g, part, stream);
        default: return launch_row<T, kRowAny>(a, g, part, stream);
    }
}

template <typename T>
GateCut cut_of_type(const GateGradArgs &a) {
    return gate_cut(a.seq, a.dim, GradBlock<T>::kWarps, kShortest, kPerSm<T>, a.want_dbound ? kMaxParts : INT_MAX);
}
GateCut cut_of(const GateGradArgs &a) {
    return a.io == IoType::kF32 ? cut_of_type<float>(a) : cut_of_type<__nv_bfloat16>(a);
}

// Partial sums of d_bound.
int parts_of(const GateCut &g) { return g.width * (g.block != 0 ? 1 : g.segments); }

}  // namespace

size_t gated_recurrence_grad_workspace(const GateGradArgs &a) {
    if (a.dim == 0) return 0;
    const GateCut g = cut_of(a);
    const size_t parts = parts_of(g);
    return 2 * gate_pairs(g) * sizeof(float2) + (a.want_dbound && parts > 1 ? parts * a.dim * sizeof(float) : 0);
}

cudaError_t launch_gated_recurrence_grad(const GateGradArgs &a, void *workspace, cudaStream_t stream) {
    GateCut g = cut_of(a);
    g.P = static_cast<float2 *>(workspace);
    g.h = g.P + gate_pairs(g);
    const int parts = parts_of(g);
    float *part = a.dbound == nullptr ? nullptr : parts > 1 ? reinterpret_cast<float *>(g.h + gate_pairs(g)) : a.dbound;
    cudaError_t e;
    switch (a.io) {
        case IoType::kBF16: e = launch_type<__nv_bfloat16>(a, g, part, stream); break;
        case IoType::kF16: e = launch_type<__half>(a, g, part, stream); break;
        default: e = launch_type<float>(a, g, part, stream);
    }
    if (e != cudaSuccess || a.dbound == nullptr || parts == 1) return e;
    return launch_column_sums(part, nullptr, parts, a.dim, a.dbound, nullptr, stream);
}

}  // namespace xm
