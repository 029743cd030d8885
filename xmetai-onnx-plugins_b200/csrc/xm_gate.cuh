// xm_gate.cuh -- what the gated linear recurrence and its backward pass share: the
// gate, the walk over sequences, and the scan over the token axis.
//
// Both are first-order recurrences per channel, h <- a h + b, forwards over the
// tokens or backwards. A lane holds two channels, a warp kGateSteps consecutive
// tokens of 64 channels; the block's warps follow one another along the axis, and so
// do the blocks of a cluster. Each warp runs its tokens from zero and keeps, per
// token, h and the product P of the a up to it, so that the value with the true start
// h0 is h + P h0: the start needs to be known only after the loads and exponentials
// are done. The starts come by joining (P, h) pairs, first over the block's warps in
// shared memory, then over the cluster's blocks in each other's shared memory, and
// the cluster walks on with the last value as carry. So the axis is read once, every
// wait is a hardware barrier, and the order of all operations is fixed.
#pragma once

#include <algorithm>

#include "xm_common.cuh"
#include "xm_sequences.cuh"

namespace xm {

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// keep = sigmoid(f), take = sigmoid(-f) = 1 - keep, each with its own relative
// precision: with t = exp(-f), r = 1 / (1 + t) and t r, no difference of nearby values
// is formed. The exponent stops at 2^126, where r is float32's smallest normal value
// and t r one: nothing overflows, and NaN stays NaN.
// For two channels: r' = rest r, a = low + r' (the share kept), u = t r' (taken up).
struct Gate2 {
    float2 r, a, u;
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
    g.r = make_float2(rcp_approx(s.x), rcp_approx(s.y));
    const float2 k = __fmul2_rn(g.r, rest);
    g.a = __fadd2_rn(k, low);
    g.u = __fmul2_rn(k, t);
    return g;
}

constexpr int kGateWarps = 8;  // warps of a block along the tokens
constexpr int kGateThreads = 32 * kGateWarps;
constexpr int kGateSteps = 8;                         // tokens of a warp
constexpr int kGateTokens = kGateWarps * kGateSteps;  // tokens of a block
constexpr int kGateChannels = 64;                     // channels of a block
constexpr int kGateMaxCluster = 8;

// The tokens that a cluster walks: a batch row, several short ones, or the packed row.
struct GateSpans {
    int rows;     // spans
    int length;   // tokens of a span; with cu the span is [cu[0], cu[units])
    int tiles;    // blocks of channels
    int cluster;  // blocks of a cluster
    int width;    // spans walked at the same time
};

struct Span {
    int lo, hi;
};
__device__ __forceinline__ Span gate_span(const SeqArgs &q, const GateSpans &s, int i) {
    if (q.cu != nullptr) return Span{seq_start(q, 0), seq_start(q, q.units)};
    const int lo = i * s.length;
    return Span{lo, lo + min(s.length, q.tokens - lo)};
}

// The sequence that holds a token: [start, end) of sequence seq.
struct SeqAt {
    int seq, start, end;
};
__device__ __forceinline__ SeqAt seq_at(const SeqArgs &q, int t) {
    if (q.cu == nullptr) {
        const int i = t / q.seqlen;
        return SeqAt{i, i * q.seqlen, (i + 1) * q.seqlen};
    }
    const int next = max(seq_first_from(q, t + 1), 1);  // first that starts behind t
    return SeqAt{next - 1, seq_start(q, next - 1), seq_start(q, next)};
}

// Calls f(sequence) for the sequences without tokens, shared out over the warps of all
// blocks with the same channels (block `block` of `blocks`).
template <typename F>
__device__ __forceinline__ void for_empty_sequences(const SeqArgs &q, int block, int blocks, F &&f) {
    if (q.cu == nullptr && q.seqlen > 0) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (long long s0 = (static_cast<long long>(block) * kGateWarps + warp) * 32; s0 < q.units;
         s0 += 32LL * kGateWarps * blocks) {
        const int s = static_cast<int>(s0) + lane;
        bool empty = false;
        if (s < q.units) {
            const int t = seq_start(q, s);
            empty = seq_end(q, s, t) == t;
        }
        for (unsigned left = __ballot_sync(kFullMask, empty); left != 0; left &= left - 1)
            f(static_cast<int>(s0) + __ffs(left) - 1);
    }
}

// A (P, h) pair stands for h0 -> P h0 + h. Where a sequence starts inside, nothing of
// h0 gets through, whatever it is (infinities and NaN too): a token's P is then kCut,
// and a warp's pair is flagged. Products of gates are kept above zero, so that an
// infinite h0 outlasts their underflow as it does step by step.
constexpr float kCut = -1.0f;
constexpr float kLeast = 1.4e-45f;
__device__ __forceinline__ float2 above_zero(float2 P) { return make_float2(fmaxf(P.x, kLeast), fmaxf(P.y, kLeast)); }

struct GatePair {
    float2 P, h;
};

// Shared memory of the join; parity alternates from step to step.
struct GateJoin {
    GatePair warp[2][kGateWarps][32];
    GatePair block[2][kGateMaxCluster][32];
    unsigned char warp_cut[2][kGateWarps];
    int block_cut[2][kGateMaxCluster];
};

__device__ __forceinline__ GatePair load_pair(const GatePair &p) {
    const float4 w = *reinterpret_cast<const float4 *>(&p);
    return GatePair{make_float2(w.x, w.y), make_float2(w.z, w.w)};
}
__device__ __forceinline__ float2 apply(const GatePair &p, bool cut, float2 h0) {
    return cut ? p.h : __ffma2_rn(p.P, h0, p.h);
}

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// All threads of the cluster: what each wrote before, into any block's shared memory, is visible behind it.
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t address_in_block(const void *smem, unsigned rank) {
    uint32_t there;
    asm("mapa.shared::cluster.u32 %0, %1, %2;"
        : "=r"(there)
        : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(smem))), "r"(rank));
    return there;
}

// Joins the warps' pairs of one step. Returns the value that this warp's tokens start
// from and moves `carry` from the step's start to its end. Called by all threads of
// the cluster; also a __syncthreads() of the block.
__device__ __forceinline__ float2 gate_join(GateJoin &s, int parity, int cluster, unsigned rank, const GatePair &mine,
                                            bool cut, float2 &carry) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    *reinterpret_cast<float4 *>(&s.warp[parity][warp][lane]) = make_float4(mine.P.x, mine.P.y, mine.h.x, mine.h.y);
    if (lane == 0) s.warp_cut[parity][warp] = cut;
    __syncthreads();
    const uint2 cuts = *reinterpret_cast<const uint2 *>(&s.warp_cut[parity][0]);
    auto cut_of = [&](int w) { return ((w < 4 ? cuts.x : cuts.y) >> (8 * (w & 3)) & 1) != 0; };
    float2 start = carry;
    if (cluster > 1) {
        if (warp == kGateWarps - 1) {  // the block's pair, to every block
            GatePair b = load_pair(s.warp[parity][0][lane]);
#pragma unroll
            for (int w = 1; w < kGateWarps; ++w) {
                const GatePair p = load_pair(s.warp[parity][w][lane]);
                b.h = apply(p, cut_of(w), b.h);
                b.P = above_zero(__fmul2_rn(b.P, p.P));
            }
            for (int r = 0; r < cluster; ++r) {
                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(
                                 address_in_block(&s.block[parity][rank][lane], r)),
                             "f"(b.P.x), "f"(b.P.y), "f"(b.h.x), "f"(b.h.y)
                             : "memory");
                if (lane == 0)
                    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(
                                     address_in_block(&s.block_cut[parity][rank], r)),
                                 "r"((cuts.x | cuts.y) != 0 ? 1 : 0)
                                 : "memory");
            }
        }
        cluster_barrier();
        for (int r = 0; r < cluster; ++r) {
            if (r == static_cast<int>(rank)) start = carry;
            carry = apply(load_pair(s.block[parity][r][lane]), s.block_cut[parity][r] != 0, carry);
        }
#pragma unroll
        for (int w = 0; w < kGateWarps - 1; ++w) {
            if (w < warp) start = apply(load_pair(s.warp[parity][w][lane]), cut_of(w), start);
        }
    } else {
#pragma unroll
        for (int w = 0; w < kGateWarps; ++w) {
            if (w == warp) start = carry;
            carry = apply(load_pair(s.warp[parity][w][lane]), cut_of(w), carry);
        }
    }
    return start;
}

// A token's part of its warp's start: h0 -> P h0, with the care of kCut and kLeast.
__device__ __forceinline__ float through(float P, float h0) {
    if (P < 0.0f) return 0.0f;
    return P == 0.0f && !(fabsf(h0) <= 3.4028235e38f) ? h0 : P * h0;
}
__device__ __forceinline__ bool finite2(float2 v) { return fabsf(v.x) <= 3.4028235e38f && fabsf(v.y) <= 3.4028235e38f; }

// A lane's two channels: neighbours, moved as one word (kWords: rows of whole 16-byte
// words, aligned to them), else 32 apart and moved one by one.
template <typename T, bool kWords>
struct Lane {
    int c[2];        // channels (0 where there is none)
    bool active[2];
    __device__ __forceinline__ Lane(int tile, int lane, int dim) {
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const int at = tile * kGateChannels + (kWords ? 2 * lane + v : lane + 32 * v);
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
    // `row`: a token's first channel
    __device__ __forceinline__ float2 load(const T *row) const { return make_float2(to_f32<T>(row[c[0]]), to_f32<T>(row[c[1]])); }
    __device__ __forceinline__ void store(T *row, float2 v) const {
        if constexpr (kWords) {
            if (!active[0]) return;
            if constexpr (sizeof(T) == 2) *reinterpret_cast<uint32_t *>(row + c[0]) = pack2<T>(v.x, v.y);
            else *reinterpret_cast<float2 *>(row + c[0]) = v;
        } else {
            if (active[0]) row[c[0]] = from_f32<T>(v.x);
            if (active[1]) row[c[1]] = from_f32<T>(v.y);
        }
    }
};

// A block's tokens of one tensor in shared memory, and the copy that fills it: 16-byte
// words of consecutive threads.
template <typename T>
struct GateTile {
    T v[kGateTokens][kGateChannels];
    __device__ __forceinline__ float2 at(int row, int lane) const {
        if constexpr (sizeof(T) == 2) return unpack2<T>(*reinterpret_cast<const uint32_t *>(&v[row][2 * lane]));
        else return *reinterpret_cast<const float2 *>(&v[row][2 * lane]);
    }
};
// Rows first + 0 .. kGateTokens - 1 of a tensor's channels; those outside [lo, hi) are left out.
template <typename T>
__device__ __forceinline__ void copy_tile(GateTile<T> &dst, const T *src, int first, int lo, int hi, int dim, int tile) {
    constexpr int kPer = 16 / static_cast<int>(sizeof(T)), kWordsRow = kGateChannels / kPer;
    constexpr int kRows = kGateThreads / kWordsRow;  // rows per pass
    const int col = threadIdx.x % kWordsRow * kPer, row = threadIdx.x / kWordsRow;
    if (tile * kGateChannels + col >= dim) return;
    const T *p = src + static_cast<int64_t>(first + row) * dim + tile * kGateChannels + col;
#pragma unroll
    for (int k = 0; k < kGateTokens; k += kRows) {
        const int t = first + row + k;
        if (t >= lo && t < hi) cp_async16(&dst.v[row + k][col], p, 16);
        p += static_cast<int64_t>(kRows) * dim;
    }
}

// How a call is cut: blocks of channels, spans, and the cluster along the tokens.
GateSpans gate_spans(const SeqArgs &q, int dim);

template <typename... Params, typename... Args>
cudaError_t launch_gate_clusters(void (*kernel)(Params...), size_t smem, const GateSpans &g, cudaStream_t stream,
                                 const Args &...args) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(g.width) * g.tiles * g.cluster);
    cfg.blockDim = dim3(kGateThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = g.cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = g.cluster > 1 ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kernel, args...);
    return e == cudaSuccess ? cudaGetLastError() : e;
}

}  // namespace xm
