// gated_recurrence.cu -- GatedRecurrenceFn and GatedRecurrenceUpdateFn for sm_100a.
//
// Math, per channel: a_t = b + (1 - b) sigmoid(f_t), h_t = a_t h_(t-1) + (1 - a_t) x_t.
#include <algorithm>
#include <climits>

#include "xm_common.cuh"
#include "xm_gate.cuh"
#include "xm_kernels.h"
#include "xm_rows.cuh"
#include "xm_sequences.cuh"

namespace xm {
namespace {

constexpr int kStages = 3;  // groups of x and f in use and under way, of a warp with a row or segment
// And of a warp in a ring. Of four: what leaves an SM as many blocks as its registers do (16-bit types: five; 8 x 2048 x
// 4096 takes 72 us, and 83 with three stages and four blocks), or its copies (float32: two; 8 x 1024 x 4096 takes 70 us,
// and 78 with two stages and four blocks). Of eight, an SM has two at most.
template <typename T, int kWarps>
constexpr int kRingStages = kWarps == 8 || sizeof(T) == 4 ? 3 : 2;

// Segments of an SM: one wave that fills it, and leaves room for the next pass (16384 x 4096 packed takes 110 us; with six
// stages, of which nine fit an SM, 119 at best).
constexpr int kPerSm = 12;

template <typename T, int kRow>
using ScanTile = GateTile<T, kGateGroup, kRow>;

template <typename T, int kRow>
__device__ __forceinline__ float2 init_of(const GateArgs &p, const Lane<T, kRow> &ch, long long row) {
    return ch.floats(p.init != nullptr && row >= 0 ? p.init + row * p.dim : nullptr, 0.0f);
}
template <typename T, int kRow>
__device__ __forceinline__ void store_final(const GateArgs &p, const Lane<T, kRow> &ch, long long row, float2 h) {
    if (p.final_state != nullptr && row >= 0) ch.store_floats(p.final_state + row * p.dim, h);
}
// Sequences without tokens keep their starting states; warp of warps with the same channels.
template <typename T, int kRow>
__device__ __forceinline__ void keep_empty(const GateArgs &p, const Lane<T, kRow> &ch, int warp, int warps) {
    if (p.final_state == nullptr) return;
    for_empty_sequences(p.seq, warp, warps, [&](int s) {
        long long from;
        const long long row = seq_rows(p.seq, s, &from);
        store_final(p, ch, row, init_of(p, ch, from));
    });
}

// A warp walks segment j of a span. kEnds: the first pass. first_pass(): it is through; nothing is stored, and nothing
// of it read, before.
template <typename T, int kRow, bool kEnds, int kStages, typename Wait>
__device__ __forceinline__ void walk_segment(const GateArgs &p, const GateCut &g, ScanTile<T, kRow> (*ring)[2],
                                             const Lane<T, kRow> &ch, int tile, float2 low, float2 rest, Span span,
                                             int length, int j, const GatePairs &pairs, Wait &&first_pass) {
    const SeqArgs &q = p.seq;
    const T *const X = static_cast<const T *>(p.x), *const F = static_cast<const T *>(p.f);
    T *const Y = static_cast<T *>(p.out);
    const int s0 = span.lo + min(static_cast<long long>(j) * length, static_cast<long long>(max(span.hi - span.lo, 0)));
    const int s1 = min(static_cast<long long>(s0) + length, static_cast<long long>(span.hi));
    if (s0 >= s1) return;
    int begin = s0;
    SeqAt seq = seq_at(q, kEnds ? s1 - 1 : s0);
    if (kEnds) {
        if (seq.end <= s1 || s1 >= span.hi) return;  // no sequence leaves the segment
        begin = max(s0, seq.start);
    }
    auto copy = [&](int t, int stage) {
        if (t < s1) {
            copy_tile(ring[stage][0], X, t, 0, s1, p.dim, tile);
            copy_tile(ring[stage][1], F, t, 0, s1, p.dim, tile);
        }
        cp_async_commit();
    };
    for (int k = 0; k < kStages - 1; ++k) copy(begin + k * kGateGroup, k);
    first_pass();
    float2 h = both(0.0f), P = both(1.0f);
    long long from, row = seq_rows(q, seq.seq, &from);
    // where the warp's first token does not begin a sequence, the state comes from the segments before
    SeqAt next{0, 0, 0};
    long long next_row = -1;
    float2 next_h = both(0.0f);
    if (seq.start >= begin) {  // (== unless the offsets descend)
        h = init_of(p, ch, from);
        if (kEnds) pairs.start(j) = h;
        else if (seq.end > s1 && g.segments > 1) h = pairs.start(j);
    } else if (!kEnds && j > 0) {
        int k = max(seq.start - span.lo, 0) / length;
        h = pairs.h(k);
        for (++k; k < j; ++k) h = __ffma2_rn(pairs.P(k), h, pairs.h(k));
    }
    auto look_ahead = [&] {  // the sequence behind this one, and its starting state
        if (kEnds || seq.end >= s1) return;
        next = seq_behind(q, seq);
        next_row = seq_rows(q, next.seq, &from);
        // one that leaves the segment: its last warp may have stored its final state in the same place
        next_h = next.end > s1 && g.segments > 1 ? pairs.start(j) : init_of(p, ch, from);
    };
    look_ahead();
    int stage = 0;
    for (int t = begin; t < s1; t += kGateGroup) {
        cp_async_wait<kStages - 2>();
        __syncwarp();
        copy(t + (kStages - 1) * kGateGroup, stage == 0 ? kStages - 1 : stage - 1);  // read by all a group ago
        auto token = [&](int k, float2 &x, float2 &f) {
            x = ring[stage][0].at(k, shift_of<T, kRow>(X, t + k, p.dim));
            f = ring[stage][1].at(k, shift_of<T, kRow>(F, t + k, p.dim));
        };
        float2 a[kGateGroup], b[kGateGroup];  // (of no meaning behind the segment's end)
#pragma unroll
        for (int k = 0; k < kGateGroup; ++k) {
            float2 x, f;
            token(k, x, f);
            const Gate2 gate = gate_of(f, low, rest);
            a[k] = gate.a;
            b[k] = __fmul2_rn(gate.u, x);
        }
        T *y = Y + static_cast<size_t>(t) * p.dim;
        if (t + kGateGroup <= s1 && (kEnds || seq.end > t + kGateGroup)) {
#pragma unroll
            for (int k = 0; k < kGateGroup; ++k) {
                h = __ffma2_rn(a[k], h, b[k]);
                if (kEnds) P = __fmul2_rn(P, a[k]);
                b[k] = h;
            }
            if (!kEnds && ch.active[0]) {
#pragma unroll
                for (int k = 0; k < kGateGroup; ++k, y += p.dim) ch.store(y, b[k]);
            }
        } else {
            const int last = min(kGateGroup, s1 - t);
            for (int k0 = 0; k0 < last;) {  // the tokens of a sequence, k0 .. k1 - 1
                const int end = kEnds ? last : seq.end - t, k1 = end > k0 && end < last ? end : last;
#pragma unroll
                for (int k = 0; k < kGateGroup; ++k) {
                    if (k < k0 || k >= k1) continue;
                    h = __ffma2_rn(a[k], h, b[k]);
                    if (kEnds) P = __fmul2_rn(P, a[k]);
                    b[k] = h;
                }
                k0 = k1;
                if (kEnds || end != k1) continue;
                store_final(p, ch, row, h);
                seq = next;
                row = next_row;
                h = next_h;
                look_ahead();
            }
            if (!kEnds && ch.active[0]) {
#pragma unroll
                for (int k = 0; k < kGateGroup; ++k, y += p.dim)
                    if (k < last) ch.store(y, b[k]);
            }
        }
        stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    if (kEnds) {
        pairs.P(j) = above_zero(P);
        pairs.h(j) = h;
    }
    cp_async_wait<0>();
    __syncwarp();  // (the ring is filled anew)
}

// A segment to each warp. kEnds: the first pass over segments (all but a span's last). Both read x and f: 16384 x 4096
// packed in bf16, 671 MB, 110 us, 93 % of copy bandwidth.
template <typename T, int kRow, bool kEnds>
__global__ void __launch_bounds__(32, 8) gate_kernel(const GateArgs p, const GateCut g) {
    extern __shared__ float4 smem_f4[];
    if (kEnds) dependents_may_launch();
    const int tile = blockIdx.x % g.tiles, segs = kEnds ? g.segments - 1 : g.segments;
    const int j = blockIdx.x / g.tiles % segs, slot = blockIdx.x / g.tiles / segs;
    const Lane<T, kRow> ch(tile, threadIdx.x & 31, p.dim);
    const float2 low = ch.floats(p.bound, 0.0f), rest = make_float2(1.0f - low.x, 1.0f - low.y);
    bool waited = kEnds;
    auto first_pass = [&] {
        if (!waited) wait_for_before();
        waited = true;
    };
    if (!kEnds && p.final_state != nullptr && (p.seq.cu != nullptr || p.seq.seqlen == 0)) first_pass();
    if (!kEnds) keep_empty(p, ch, slot * segs + j, g.width * segs);
    for (int i = slot; i < g.spans; i += g.width) {
        const Span span = gate_span(p.seq, g, i);
        walk_segment<T, kRow, kEnds, kStages>(p, g, reinterpret_cast<ScanTile<T, kRow>(*)[2]>(smem_f4), ch, tile, low,
                                                rest, span, segment_length(g, span), j, global_pairs(g, i, tile), first_pass);
    }
    first_pass();  // (also warps without tokens: what follows waits for this kernel only)
}

// Both passes in one block, a segment to each of its warps: as many as have room for their copies.
template <typename T>
struct ScanBlock {
    static constexpr int kWarps = sizeof(T) == 4 ? 8 : 16, kStages = sizeof(T) == 4 ? 3 : 2;
};
constexpr int kShortest = 64;  // tokens of a row that a block shares (48 x 512: 4.8 us by a warp alone, 5.3)
template <typename T, int kRow>
struct BlockSmem {
    ScanTile<T, kRow> ring[ScanBlock<T>::kWarps][ScanBlock<T>::kStages][2];
    BlockPairs<ScanBlock<T>::kWarps> pairs;
};

template <typename T, int kRow>
__global__ void __launch_bounds__(32 * ScanBlock<T>::kWarps, 1) gate_block_kernel(const GateArgs p, const GateCut g) {
    extern __shared__ float4 smem_f4[];
    constexpr int kWarps = ScanBlock<T>::kWarps, kStages = ScanBlock<T>::kStages;
    auto &sm = *reinterpret_cast<BlockSmem<T, kRow> *>(smem_f4);
    const int warp = threadIdx.x >> 5, tile = blockIdx.x % g.tiles, slot = blockIdx.x / g.tiles;
    const Lane<T, kRow> ch(tile, threadIdx.x & 31, p.dim);
    const float2 low = ch.floats(p.bound, 0.0f), rest = make_float2(1.0f - low.x, 1.0f - low.y);
    keep_empty(p, ch, slot * kWarps + warp, g.width * kWarps);
    for (int i = slot; i < g.spans; i += g.width) {
        const Span span = gate_span(p.seq, g, i);
        const int length = segment_length(g, span);
        const GatePairs pairs = sm.pairs.view();
        walk_segment<T, kRow, true, kStages>(p, g, sm.ring[warp], ch, tile, low, rest, span, length, warp, pairs, [] {});
        __syncthreads();
        walk_segment<T, kRow, false, kStages>(p, g, sm.ring[warp], ch, tile, low, rest, span, length, warp, pairs, [] {});
        __syncthreads();
    }
}

// A row to a block, its warps' groups in turn: x, f and y move once. 8 x 2048 x 4096 in bf16, 403 MB: 72 us, 85 % of copy
// bandwidth, with an instruction issued every second cycle.
template <typename T, int kRow, int kWarps>
struct RingSmem {
    Ring<kWarps> hand;
    GateTile<T, kGateGroup, kRow> ring[kWarps][kRingStages<T, kWarps>][2];
};

template <typename T, int kRow, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, kWarps == 4 ? 5 : 2) gate_ring_kernel(const GateArgs p, const GateCut g) {
    extern __shared__ float4 smem_f4[];
    constexpr int kStages = kRingStages<T, kWarps>;
    auto &sm = *reinterpret_cast<RingSmem<T, kRow, kWarps> *>(smem_f4);
    const SeqArgs &q = p.seq;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tile = blockIdx.x % g.tiles, slot = blockIdx.x / g.tiles;
    const Lane<T, kRow> ch(tile, lane, p.dim);
    const float2 low = ch.floats(p.bound, 0.0f), rest = make_float2(1.0f - low.x, 1.0f - low.y);
    const T *const X = static_cast<const T *>(p.x), *const F = static_cast<const T *>(p.f);
    T *const Y = static_cast<T *>(p.out);
    keep_empty(p, ch, slot * kWarps + warp, g.width * kWarps);
    for (int i = slot; i < g.spans; i += g.width) {
        const Span span = gate_span(q, g, i);
        constexpr int kTurn = kWarps * kGateGroup;  // tokens of a round
        const int first = span.lo + warp * kGateGroup;
        auto copy = [&](int t, int stage) {
            if (t < span.hi) {
                copy_tile(sm.ring[warp][stage][0], X, t, 0, span.hi, p.dim, tile);
                copy_tile(sm.ring[warp][stage][1], F, t, 0, span.hi, p.dim, tile);
            }
            cp_async_commit();
        };
        for (int k = 0; k < kStages - 1; ++k) copy(first + k * kTurn, k);
        SeqAt seq{0, 0, 0};
        int stage = 0;
        for (int t = first; t < span.hi; t += kTurn) {
            cp_async_wait<kStages - 2>();
            __syncwarp();
            copy(t + (kStages - 1) * kTurn, stage == 0 ? kStages - 1 : stage - 1);  // read by all a round ago
            auto token = [&](int k, float2 &x, float2 &f) {
                x = sm.ring[warp][stage][0].at(k, shift_of<T, kRow>(X, t + k, p.dim));
                f = sm.ring[warp][stage][1].at(k, shift_of<T, kRow>(F, t + k, p.dim));
            };
            if (seq.end <= t) seq = seq_at(q, t);
            const bool more = t + kGateGroup < span.hi;  // a group behind
            const int next = warp + 1 == kWarps ? 0 : warp + 1;
            // (whether a group takes and gives depends on t alone, so that offsets that descend leave nobody waiting)
            if (t > span.lo && t + kGateGroup <= span.hi && seq.start < t && seq.end > t + kGateGroup) {
                float2 P[kGateGroup], h[kGateGroup];
#pragma unroll
                for (int k = 0; k < kGateGroup; ++k) {
                    float2 x, f;
                    token(k, x, f);
                    const Gate2 gate = gate_of(f, low, rest);
                    P[k] = gate.a;
                    h[k] = __fmul2_rn(gate.u, x);
                }
#pragma unroll
                for (int k = 1; k < kGateGroup; ++k) {
                    h[k] = __ffma2_rn(P[k], h[k - 1], h[k]);
                    P[k] = __fmul2_rn(P[k], P[k - 1]);
                }
                const float2 start = sm.hand.take(warp);
                if (!__all_sync(kFullMask, finite2(start))) {  // (also for what lanes without channels find)
#pragma unroll
                    for (int k = 0; k < kGateGroup; ++k) P[k] = above_zero(P[k], start);
                }
                if (more) sm.hand.give(next, __ffma2_rn(P[kGateGroup - 1], start, h[kGateGroup - 1]));
                if (ch.active[0]) {
                    T *y = Y + static_cast<size_t>(t) * p.dim;
#pragma unroll
                    for (int k = 0; k < kGateGroup; ++k, y += p.dim) ch.store(y, __ffma2_rn(P[k], start, h[k]));
                }
            } else {
                SeqAt at = seq;
                float2 h = t > span.lo ? sm.hand.take(warp) : both(0.0f);
#pragma unroll 1
                for (int k = 0; k < kGateGroup && t + k < span.hi; ++k) {
                    if (at.end <= t + k) at = seq_at(q, t + k);
                    if (at.start == t + k) {
                        long long from;
                        seq_rows(q, at.seq, &from);
                        h = init_of(p, ch, from);
                    }
                    float2 x, f;
                    token(k, x, f);
                    const Gate2 gate = gate_of(f, low, rest);
                    h = __ffma2_rn(gate.a, h, __fmul2_rn(gate.u, x));
                    if (ch.active[0]) ch.store(Y + static_cast<size_t>(t + k) * p.dim, h);
                    if (at.end == t + k + 1) store_final(p, ch, seq_row(q, at.seq), h);
                }
                if (more) sm.hand.give(next, h);
            }
            stage = stage + 1 == kStages ? 0 : stage + 1;
        }
        cp_async_wait<0>();
        __syncthreads();  // the rings are filled anew, the hands start anew
    }
}

// One token per sequence: bound by memory, 8 bytes of state and three elements per channel. A thread takes kVec
// neighbouring channels (a word of the I/O type, or one where rows are not whole words) of kRows sequences, whose loads
// are issued together. 256 x 4096 in fp16, 15 MB: 3.5 us in a graph, 64 % of copy bandwidth.
constexpr int kTokenThreads = 128;

template <int kVec>
__device__ __forceinline__ void load_state(const float *p, float (&v)[kVec]) {
    if constexpr (kVec == 1) {
        v[0] = *p;
    } else {
#pragma unroll
        for (int i = 0; i < kVec; i += 4) {
            const float4 w = *reinterpret_cast<const float4 *>(p + i);
            v[i] = w.x; v[i + 1] = w.y; v[i + 2] = w.z; v[i + 3] = w.w;
        }
    }
}

template <typename T, int kVec, int kRows>
__global__ void __launch_bounds__(kTokenThreads) gate_token_kernel(const GateArgs p) {
    using Word = Chunk<T, kVec>;
    const int d = (blockIdx.x * kTokenThreads + threadIdx.x) * kVec;
    if (d >= p.dim) return;
    // (sequences are counted in 31 bits, the steps past the last one need the 32nd)
    const unsigned units = p.seq.units;
    for (unsigned i0 = blockIdx.y * kRows; i0 < units; i0 += gridDim.y * kRows) {
        long long row[kRows];
        Word x[kRows], f[kRows];
        float h[kRows][kVec];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const unsigned i = min(i0 + r, units - 1);
            const size_t at = static_cast<size_t>(i) * p.dim + d;
            row[r] = i0 + r < units ? seq_row(p.seq, i) : -1;
            x[r] = *reinterpret_cast<const Word *>(static_cast<const T *>(p.x) + at);
            f[r] = *reinterpret_cast<const Word *>(static_cast<const T *>(p.f) + at);
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r)
            if (row[r] >= 0) load_state<kVec>(p.init + row[r] * p.dim + d, h[r]);
        float low[kVec];
#pragma unroll
        for (int k = 0; k < kVec; ++k) low[k] = 0.0f;
        if (p.bound != nullptr) load_state<kVec>(p.bound + d, low);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            if (row[r] < 0) continue;
            float xs[kVec], fs[kVec];
            chunk_floats<T, kVec>(x[r], xs);
            chunk_floats<T, kVec>(f[r], fs);
#pragma unroll
            for (int k = 0; k < kVec; k += 2) {
                constexpr int kNext = kVec > 1 ? 1 : 0;
                const float2 b = make_float2(low[k], low[k + kNext]);
                const Gate2 g = gate_of(make_float2(fs[k], fs[k + kNext]), b, make_float2(1.0f - b.x, 1.0f - b.y));
                const float2 v = __ffma2_rn(g.a, make_float2(h[r][k], h[r][k + kNext]),
                                            __fmul2_rn(g.u, make_float2(xs[k], xs[k + kNext])));
                h[r][k] = v.x;
                if (kVec > 1) h[r][k + kNext] = v.y;
            }
            store_row_floats<kVec>(p.final_state + row[r] * p.dim + d, h[r]);
            *reinterpret_cast<Word *>(static_cast<T *>(p.out) + static_cast<size_t>(i0 + r) * p.dim + d) =
                to_chunk<T, kVec>(h[r]);
        }
    }
}

template <typename T, int kRow>
cudaError_t launch_row(const GateArgs &a, const GateCut &g, cudaStream_t stream) {
    constexpr size_t kSmem = kStages * 2 * sizeof(ScanTile<T, kRow>);
    if (g.block != 0)
        return launch_gate<gate_block_kernel<T, kRow>>(g.block, sizeof(BlockSmem<T, kRow>), g, 1, false, stream, a, g);
    if (g.ring == 4)
        return launch_gate<gate_ring_kernel<T, kRow, 4>>(4, sizeof(RingSmem<T, kRow, 4>), g, 1, false, stream, a, g);
    if (g.ring == 8)
        return launch_gate<gate_ring_kernel<T, kRow, 8>>(8, sizeof(RingSmem<T, kRow, 8>), g, 1, false, stream, a, g);
    if (g.segments > 1) {
        const cudaError_t e = launch_gate<gate_kernel<T, kRow, true>>(1, kSmem, g, g.segments - 1, false, stream, a, g);
        if (e != cudaSuccess) return e;
    }
    return launch_gate<gate_kernel<T, kRow, false>>(1, kSmem, g, g.segments, gate_behind(g), stream, a, g);
}

template <typename T>
cudaError_t launch_type(const GateArgs &a, const GateCut &g, cudaStream_t stream) {
    switch (row_of(a.dim, sizeof(T), {a.x, a.f, a.out})) {
        case kRowWords: return launch_row<T, kRowWords>(a, g, stream);
        case kRowPairs: return launch_row<T, kRowPairs>(a, g, stream);
        default: return launch_row<T, kRowAny>(a, g, stream);
    }
}

// Several sequences per thread where that leaves each SM eight blocks; below, one.
template <typename T, int kVec, int kRows>
cudaError_t launch_token_rows(const GateArgs &a, cudaStream_t stream) {
    const int64_t blocks = (a.dim + static_cast<int64_t>(kTokenThreads) * kVec - 1) / (kTokenThreads * kVec);
    const int64_t rows = (static_cast<int64_t>(a.seq.units) + kRows - 1) / kRows;
    if (kRows > 1 && blocks * rows < 8LL * current_device_sm_count()) return launch_token_rows<T, kVec, 1>(a, stream);
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(std::min<int64_t>(rows, 65535)));
    gate_token_kernel<T, kVec, kRows><<<grid, kTokenThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

int block_of(const GateArgs &a) {
    return a.io == IoType::kF32 ? ScanBlock<float>::kWarps : ScanBlock<__nv_bfloat16>::kWarps;
}

template <typename T>
cudaError_t launch_token_type(const GateArgs &a, cudaStream_t stream) {
    constexpr int kWord = 16 / static_cast<int>(sizeof(T));
    if (a.dim % kWord == 0 && aligned16(a.x) && aligned16(a.f) && aligned16(a.out) && aligned16(a.init) &&
        aligned16(a.final_state) && aligned16(a.bound))
        return launch_token_rows<T, kWord, 2>(a, stream);
    return launch_token_rows<T, 1, 4>(a, stream);
}

}  // namespace

GateCut gate_cut(const SeqArgs &q, int dim, int block, int shortest, int per_sm, int parts) {
    GateCut g{};
    g.tiles = (dim + kGateChannels - 1) / kGateChannels;
    // Rows shorter than this share a span, where that leaves an SM eight warps (5 x 6 x 547: 4.5 us apart, 10 together).
    constexpr int kShort = 64;
    const int64_t sms = current_device_sm_count();
    if (q.cu != nullptr) {
        g.spans = 1;
        g.length = q.tokens;
    } else {
        const int64_t share = std::min<int64_t>(kShort / std::max<int64_t>(q.seqlen, 1),
                                                static_cast<int64_t>(q.units) * g.tiles / (8 * sms));
        const int64_t per = q.seqlen > 0 ? std::max<int64_t>(1, share) : q.units;
        g.length = static_cast<int>(std::min<int64_t>(per * q.seqlen, q.tokens));
        g.spans = g.length > 0 ? static_cast<int>((static_cast<int64_t>(q.tokens) + g.length - 1) / g.length) : 1;
    }
    const int64_t warps = static_cast<int64_t>(g.spans) * g.tiles;
    // A row per block needs four fifths of the device's blocks to be the faster (8 x 2048 x 1024, 128 blocks: 34 us, and
    // 38 in eight segments; 4 x 2048 x 4096, 256 blocks: 42 and 64), of eight warps up to two blocks an SM (those 256: 50
    // with four; 6 x 2048 x 4096, 384 blocks: 75 with eight and 58 with four). With fewer, one wave of per_sm
    // segments an SM, of 32 tokens at least (512 x 4096: 8.8 us in 16, 14 in 32), and no more than one join can go through
    // in good time (32768 x 64: 31 us in 160, 34 in 128, 90 in 1024). Many rows of fewer than 256 tokens: a warp each
    // (8 x 128 x 4096: 8.9 us, 10.9 in rings).
    g.segments = 1;
    if (g.length >= 128) {
        if (warps * 5 >= sms * 4) g.ring = g.length < 256 ? 0 : warps > 2 * sms ? 4 : 8;
        else g.segments = static_cast<int>(std::min<int64_t>({std::max<int64_t>(sms * per_sm / warps, 1),
                                                              (int64_t(g.length) + 31) / 32, 192}));
    }
    // Short rows in one block and launch: as long as a warp has a group or two (192 x 512: 6.7 us, 7.1 in two kernels;
    // 384: 9.0 and 8.2, with three microseconds less on the host; 1024: 16 and 9.8), and in the place of rings of an SM
    // each up to four (4 x 256 x 2048: 7.9 us, 10.5 in rings; 1024: 19 and 21).
    if (g.length >= shortest && warps <= sms && g.length <= (g.ring != 0 ? 64 : 24) * block) {
        g.ring = 0;
        g.block = g.segments = block;
    }
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(parts, (int64_t(1) << 30) / g.tiles) / g.segments);
    g.width = static_cast<int>(std::min<int64_t>(g.spans, most));
    return g;
}

size_t gated_recurrence_workspace(const GateArgs &a) {
    return a.dim == 0 ? 0 : 3 * gate_pairs(gate_cut(a.seq, a.dim, block_of(a), kShortest, kPerSm, INT_MAX)) * sizeof(float2);
}

cudaError_t launch_gated_recurrence(const GateArgs &a, void *workspace, cudaStream_t stream) {
    GateCut g = gate_cut(a.seq, a.dim, block_of(a), kShortest, kPerSm, INT_MAX);
    g.P = static_cast<float2 *>(workspace);
    g.h = g.P + gate_pairs(g);
    g.start = g.h + gate_pairs(g);
    switch (a.io) {
        case IoType::kBF16: return launch_type<__nv_bfloat16>(a, g, stream);
        case IoType::kF16: return launch_type<__half>(a, g, stream);
        default: return launch_type<float>(a, g, stream);
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
