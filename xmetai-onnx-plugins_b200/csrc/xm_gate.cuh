// xm_gate.cuh -- what the gated linear recurrence and its backward pass share: the
// gate, the walk over sequences, and how a call is cut.
//
// Both are first-order recurrences per channel, h <- a h + b, forwards over the
// tokens or backwards. A warp holds 64 channels, two per lane, and takes groups of
// tokens, whose tiles come by asynchronous copies some groups ahead. A group is run
// from zero, with the product P of the a up to each token beside it: the value with
// the true start h0 is h + P h0, so everything but one multiply-add per group can be
// done before h0 is known.
//
// With rows enough for the device, a block's warps take a row's groups in turn (ring):
// each waits for its start, which the warp before leaves in shared memory, hands the
// value at its group's end on at once and then stores its outputs. Every operand is
// read once.
//
// With fewer rows, a row is cut into segments of a warp each. A first pass walks the
// segments that a sequence leaves, from zero, and keeps h and P at the segment's end;
// the second joins these pairs from the sequence's start up to its own segment and
// walks with the true start. Short rows do both in one block, behind one launch, long
// ones in two kernels.
#pragma once

#include <algorithm>
#include <initializer_list>

#include "xm_common.cuh"
#include "xm_sequences.cuh"

namespace xm {

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// keep = sigmoid(f), take = sigmoid(-f) = 1 - keep, each with its own relative
// precision: with t = exp(-f), r = 1 / (1 + t) and t r, no difference of nearby values
// is formed. The exponent stops at 2^126, where r is float32's smallest normal value
// and t r one: nothing overflows, and NaN stays NaN.
// For two channels: a = low + rest keep (the share kept), u = rest take (taken up), as (rest t) r. rest meets t first:
// where f is far below zero, r is next to the smallest normal value, and rest r would lose its bits below it before t
// brought them back (bound 0.99999, f = -87: u off by 3e-3). Far above zero r is 1, and rest t loses no more than u itself
// has to.
struct Gate2 {
    float2 keep, take, a, u;
};
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ Gate2 gate_of(float2 f, float2 low, float2 rest) {
    const float2 e = __fmul2_rn(f, both(-kLog2e));
    const float2 t = make_float2(ex2_approx(min_nan(e.x, 126.0f)), ex2_approx(min_nan(e.y, 126.0f)));
    const float2 s = __fadd2_rn(t, both(1.0f));
    Gate2 g;
    g.keep = make_float2(rcp_approx(s.x), rcp_approx(s.y));
    g.a = __ffma2_rn(g.keep, rest, low);
    g.u = __fmul2_rn(__fmul2_rn(t, rest), g.keep);
    g.take = __fmul2_rn(t, g.keep);
    return g;
}

constexpr int kGateChannels = 64;  // channels of a warp
constexpr int kGateGroup = 16;     // tokens that segments are whole multiples of

// How a call is cut. A span is a batch row, several short ones, or the packed row.
struct GateCut {
    int spans, length;  // length: tokens of a span; with cu it is [cu[0], cu[units])
    int width;          // spans walked at the same time
    int segments;       // of a span
    int ring;           // warps of a block that take a span's groups in turn (segments is 1), or 0
    int block;          // warps of a block that shares a span in segments, or 0; without both a segment to each warp
    int tiles;          // groups of channels
    float2 *P, *h, *start;  // [spans][segments][tiles][32]: the pairs, and the state that a leaving sequence started from
};

// Tokens [lo, hi) of segment j of span i.
struct Span {
    int lo, hi;
};
__device__ __forceinline__ Span gate_span(const SeqArgs &q, const GateCut &g, int i) {
    if (q.cu != nullptr) return Span{seq_start(q, 0), seq_start(q, q.units)};
    const int lo = i * g.length;
    return Span{lo, lo + min(g.length, q.tokens - lo)};
}
__device__ __forceinline__ int segment_length(const GateCut &g, Span s) {
    if (g.segments == 1) return max(s.hi - s.lo, 1);
    const int n = (max(s.hi - s.lo, 0) + g.segments - 1) / g.segments;
    return max((n + kGateGroup - 1) / kGateGroup * kGateGroup, kGateGroup);
}

// First packed sequence that starts behind t (units: none). A warp looks at 32 offsets at a time: a round of loads for up
// to 32 sequences, two for a thousand, where halving takes one for every doubling.
__device__ __forceinline__ int seq_first_behind(const SeqArgs &q, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = q.units;  // it is one of [lo, hi]
    while (hi - lo > 32) {
        const int step = (hi - lo - 1) / 32 + 1;  // the last of every `step` offsets
        const long long at = lo + (lane + 1LL) * step - 1;
        const unsigned behind = __ballot_sync(kFullMask, at < hi && seq_start(q, static_cast<int>(min(at, hi - 1LL))) > t);
        if (behind != 0) {
            const int k = __ffs(behind) - 1;
            hi = lo + (k + 1) * step - 1;
            lo += k * step;
        } else {
            lo += (hi - lo) / step * step;
        }
    }
    const unsigned behind = __ballot_sync(kFullMask, lo + lane < hi && seq_start(q, min(lo + lane, q.units)) > t);
    return behind != 0 ? lo + __ffs(behind) - 1 : hi;
}

// The sequence that holds a token: [start, end) of sequence seq. Called by whole warps.
struct SeqAt {
    int seq, start, end;
};
__device__ __forceinline__ SeqAt seq_at(const SeqArgs &q, int t) {
    if (q.cu == nullptr) {
        const int i = t / q.seqlen;
        return SeqAt{i, i * q.seqlen, (i + 1) * q.seqlen};
    }
    const int next = max(seq_first_behind(q, t), 1);
    return SeqAt{next - 1, seq_start(q, next - 1), seq_start(q, next)};
}
// The same for the token behind, or before, a sequence that is known.
__device__ __forceinline__ SeqAt seq_behind(const SeqArgs &q, const SeqAt &s) {
    if (q.cu != nullptr && s.seq + 2 <= q.units) {
        const int end = seq_start(q, s.seq + 2);
        if (end > s.end) return SeqAt{s.seq + 1, s.end, end};
    }
    return seq_at(q, s.end);
}
__device__ __forceinline__ SeqAt seq_before(const SeqArgs &q, const SeqAt &s) {
    if (q.cu != nullptr && s.seq >= 1) {
        const int start = seq_start(q, s.seq - 1);
        if (start < s.start) return SeqAt{s.seq - 1, start, s.start};
    }
    return seq_at(q, s.start - 1);
}

// State row of sequence i, and in *start the one that it starts from (-1: none). Both of its entries are asked for at once.
__device__ __forceinline__ long long seq_rows(const SeqArgs &q, int i, long long *start) {
    const bool live = q.live == nullptr || index_at(q.live, q.live64, i) != 0;
    const long long row = seq_row(q, i);
    *start = live ? row : -1;
    return row;
}

// Calls f(sequence) for the sequences without tokens, shared out over `warps` warps with the same channels.
template <typename F>
__device__ __forceinline__ void for_empty_sequences(const SeqArgs &q, int warp, int warps, F &&f) {
    if (q.cu == nullptr && q.seqlen > 0) return;
    for (long long s0 = static_cast<long long>(warp) * 32; s0 < q.units; s0 += 32LL * warps) {
        const int s = static_cast<int>(s0) + static_cast<int>(threadIdx.x & 31);
        bool empty = false;
        if (s < q.units) {
            const int t = seq_start(q, s);
            empty = seq_end(q, s, t) == t;
        }
        for (unsigned left = __ballot_sync(kFullMask, empty); left != 0; left &= left - 1)
            f(static_cast<int>(s0) + __ffs(left) - 1);
    }
}

// Products of gates are kept above zero, so that an infinite start outlasts their underflow as it does step by step. (To a
// finite start this adds 2^-149 of it, no more than the last bits of products next to underflow do.)
__device__ __forceinline__ float2 above_zero(float2 P) { return make_float2(fmaxf(P.x, 1.4e-45f), fmaxf(P.y, 1.4e-45f)); }
__device__ __forceinline__ bool finite1(float v) { return fabsf(v) <= 3.4028235e38f; }
__device__ __forceinline__ bool finite2(float2 v) { return finite1(v.x) && finite1(v.y); }
// The same in the channel whose start is not finite alone: a neighbour's zeros are its own.
__device__ __forceinline__ float2 above_zero(float2 P, float2 start) {
    const float2 Q = above_zero(P);
    return make_float2(finite1(start.x) ? P.x : Q.x, finite1(start.y) ? P.y : Q.y);
}

// How rows lie: of whole 16-byte words and aligned to them, of pairs of elements, or anyhow.
constexpr int kRowWords = 2, kRowPairs = 1, kRowAny = 0;
inline int row_of(int dim, size_t size, std::initializer_list<const void *> tensors) {
    uintptr_t all = static_cast<uintptr_t>(dim) * size;
    for (const void *p : tensors) all |= reinterpret_cast<uintptr_t>(p);
    return all % 16 == 0 ? kRowWords : all % (2 * size) == 0 ? kRowPairs : kRowAny;
}

// A lane's two neighbouring channels.
template <typename T, int kRow>
struct Lane {
    int c[2];  // (0 where there is none)
    bool active[2];
    __device__ __forceinline__ Lane(int tile, int lane, int dim) {
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const int at = tile * kGateChannels + 2 * lane + v;
            active[v] = at < dim;
            c[v] = active[v] ? at : 0;
        }
    }
    __device__ __forceinline__ float2 floats(const float *p, float absent) const {
        return p != nullptr ? make_float2(p[c[0]], p[c[1]]) : both(absent);
    }
    __device__ __forceinline__ void store_floats(float *p, float2 v) const {
        if (active[0]) p[c[0]] = v.x;
        if (active[1]) p[c[1]] = v.y;
    }
    // `row`: a token's first channel; only by lanes whose first channel is active
    __device__ __forceinline__ void store(T *row, float2 v) const {
        if constexpr (kRow != kRowAny) {
            if constexpr (sizeof(T) == 2) *reinterpret_cast<uint32_t *>(row + c[0]) = pack2<T>(v.x, v.y);
            else *reinterpret_cast<float2 *>(row + c[0]) = v;
        } else {
            row[c[0]] = from_f32<T>(v.x);
            if (active[1]) row[c[1]] = from_f32<T>(v.y);
        }
    }
};

// A group's tokens of one tensor in shared memory, and the warp's copy that fills it, in 16-byte words. Rows of 16-bit types
// that are not whole words are copied from the one that holds their first element, and lie behind `shift` others; those of
// float32 are copied in 4-byte words.
template <typename T, int kRows, int kRow>
struct GateTile {
    static constexpr bool kShifts = kRow != kRowWords && sizeof(T) == 2;
    alignas(16) T v[kRows][kGateChannels + (kShifts ? 8 : 0)];
    __device__ __forceinline__ float2 at(int row, int shift) const {
        const int c = 2 * (threadIdx.x & 31);
        if constexpr (kShifts && kRow == kRowAny)
            return make_float2(to_f32<T>(v[row][c + shift]), to_f32<T>(v[row][c + 1 + shift]));
        else if constexpr (sizeof(T) == 2) return unpack2<T>(*reinterpret_cast<const uint32_t *>(&v[row][c + shift]));
        else return *reinterpret_cast<const float2 *>(&v[row][c]);
    }
};
// The shift of a token's row.
template <typename T, int kRow>
__device__ __forceinline__ int shift_of(const T *src, int t, int dim) {
    if (kRow == kRowWords || sizeof(T) != 2) return 0;
    const unsigned first = static_cast<unsigned>(reinterpret_cast<uintptr_t>(src) >> 1);
    return (first + static_cast<unsigned>(t) * static_cast<unsigned>(dim)) & 7;  // (a tile's first channel is a multiple of 8)
}
// Rows first .. first + kRows - 1 of a tensor's channels; those outside [lo, hi) are left out. Reads nothing outside the
// tensor's rows 0 .. hi - 1.
template <typename T, int kRows, int kRow>
__device__ __forceinline__ void copy_tile(GateTile<T, kRows, kRow> &dst, const T *src, int first, int lo, int hi, int dim,
                                          int tile) {
    const int lane = threadIdx.x & 31;
    if constexpr (kRow == kRowWords) {
        constexpr int kPer = 16 / static_cast<int>(sizeof(T)), kWordsRow = kGateChannels / kPer;
        constexpr int kStep = 32 / kWordsRow;  // rows per pass
        const int col = lane % kWordsRow * kPer, row = lane / kWordsRow;
        if (tile * kGateChannels + col >= dim) return;
        const T *p = src + static_cast<int64_t>(first + row) * dim + tile * kGateChannels + col;
        if (first >= lo && first + kRows <= hi) {
#pragma unroll
            for (int k = 0; k < kRows; k += kStep, p += static_cast<int64_t>(kStep) * dim)
                cp_async16(&dst.v[row + k][col], p, 16);
            return;
        }
#pragma unroll
        for (int k = 0; k < kRows; k += kStep, p += static_cast<int64_t>(kStep) * dim) {
            const int t = first + row + k;
            if (t >= lo && t < hi) cp_async16(&dst.v[row + k][col], p, 16);
        }
    } else if constexpr (sizeof(T) == 2) {
        constexpr int kWordsRow = kGateChannels / 8 + 1;
        const int n = min(kGateChannels, dim - tile * kGateChannels);
        const T *const end = src + static_cast<int64_t>(hi) * dim;
#pragma unroll
        for (int i0 = 0; i0 < kRows * kWordsRow; i0 += 32) {
            const int i = i0 + lane, row = i / kWordsRow, word = i - row * kWordsRow, t = first + row;
            if (i >= kRows * kWordsRow || t < lo || t >= hi) continue;
            const T *const p = src + static_cast<int64_t>(t) * dim + tile * kGateChannels;
            const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(p) >> 1) & 7;
            const T *const from = p + (8 * word - shift);
            if (8 * word >= n + shift) continue;
            if (from >= src) {
                cp_async16(&dst.v[row][8 * word], from, static_cast<int>(min(end - from, int64_t(8))) * 2);
            } else {  // the word in which the tensor begins
                for (int k = shift; k < min(8, shift + n); ++k) dst.v[row][k] = p[k - shift];
            }
        }
    } else {
        const int n = min(kGateChannels, dim - tile * kGateChannels);
        const T *row = src + static_cast<int64_t>(first) * dim + tile * kGateChannels;
#pragma unroll 4
        for (int k = 0; k < kRows; ++k, row += dim) {
            if (first + k < lo || first + k >= hi) continue;
            if (lane < n) cp_async4(&dst.v[k][lane], row + lane, 4);
            if (lane + 32 < n) cp_async4(&dst.v[k][lane + 32], row + lane + 32, 4);
        }
    }
}

// What the first pass leaves of a span's segments, for one lane: in global memory, or in a block's shared memory.
struct GatePairs {
    float2 *P_, *h_, *start_;
    size_t base, step;
    __device__ __forceinline__ float2 &P(int k) const { return P_[base + k * step]; }
    __device__ __forceinline__ float2 &h(int k) const { return h_[base + k * step]; }
    __device__ __forceinline__ float2 &start(int k) const { return start_[base + k * step]; }
};
__device__ __forceinline__ GatePairs global_pairs(const GateCut &g, int span, int tile) {
    const size_t base = (static_cast<size_t>(span) * g.segments * g.tiles + tile) * 32 + (threadIdx.x & 31);
    return GatePairs{g.P, g.h, g.start, base, static_cast<size_t>(g.tiles) * 32};
}
template <int kWarps>
struct BlockPairs {
    float2 P[kWarps][32], h[kWarps][32], start[kWarps][32];
    __device__ __forceinline__ GatePairs view() {
        return GatePairs{&P[0][0], &h[0][0], &start[0][0], static_cast<size_t>(threadIdx.x & 31), 32};
    }
};

// The cut of a call (without pointers). block: warps of the operator's block that shares a row, of `shortest` tokens at
// least; per_sm: segments of a wave on an SM; parts: at most as many partial sums per tile.
GateCut gate_cut(const SeqArgs &q, int dim, int block, int shortest, int per_sm, int parts);
inline size_t gate_pairs(const GateCut &g) {  // elements of each of P, h and start
    return g.segments > 1 && g.block == 0 ? static_cast<size_t>(g.spans) * g.segments * g.tiles * 32 : 0;
}

// Whether the second pass's blocks may begin while the first ends: worth a microsecond or two where segments are short (512 x
// 4096 in 16: 8.8 us against 9.6; 2 x 257 x 63: 7.2 against 9.2). Long ones want their blocks spread evenly, which slots
// that fall free one by one do not give (16384 x 4096 packed in 27: 116 us against 110, backward 204 against 188).
inline bool gate_behind(const GateCut &g) { return g.segments > 1 && g.length / g.segments <= 64; }

// Hands a value on from the warp of group n to that of group n + 1 of a ring: slot and barrier are the receiver's. The
// giver only arrives; it writes the slot again a round later, when the receiver is long past its wait. (Barriers by
// number known to the compiler: a block that may use any holds all sixteen, and four blocks an SM's.)
template <int kWarps>
struct Ring {
    float2 slot[kWarps][32];
    template <int kAt>
    __device__ __forceinline__ static void arrive(int warp) {
        if constexpr (kAt + 1 < kWarps) {
            if (warp != kAt) return arrive<kAt + 1>(warp);
        }
        asm volatile("bar.arrive %0, 64;" ::"n"(kAt + 1) : "memory");
    }
    template <int kAt>
    __device__ __forceinline__ static void sync(int warp) {
        if constexpr (kAt + 1 < kWarps) {
            if (warp != kAt) return sync<kAt + 1>(warp);
        }
        asm volatile("bar.sync %0, 64;" ::"n"(kAt + 1) : "memory");
    }
    __device__ __forceinline__ void give(int warp, float2 v) {
        slot[warp][threadIdx.x & 31] = v;
        arrive<0>(warp);
    }
    __device__ __forceinline__ float2 take(int warp) const {
        sync<0>(warp);
        return slot[warp][threadIdx.x & 31];
    }
};

// Launches kKernel with `warps` to a block. behind: it waits by itself for the kernel before.
template <auto kKernel, typename... Args>
cudaError_t launch_gate(int warps, size_t smem, const GateCut &g, int segments, bool behind, cudaStream_t stream,
                        const Args &...args) {
    const cudaError_t e = allow_shared<kKernel>(smem);
    if (e != cudaSuccess) return e;
    const dim3 grid(static_cast<unsigned>(g.width) * segments * g.tiles), block(32 * warps);
    if (behind) return launch_behind(kKernel, grid, block, smem, stream, args...);
    kKernel<<<grid, block, smem, stream>>>(args...);
    return cudaGetLastError();
}

}  // namespace xm
