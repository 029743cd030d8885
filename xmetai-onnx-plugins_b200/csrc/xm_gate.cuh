// xm_gate.cuh -- what the gated linear recurrence and its backward pass share: the
// gate, the walk over sequences, and the scan over the token axis.
//
// Both are first-order recurrences per channel, h <- a h + b, forwards over the
// tokens or backwards. A warp owns kSteps consecutive tokens of 32 V channels; the
// block's warps follow one another along the axis, and so do the blocks of a
// cluster. Each warp runs its tokens from zero and keeps, per token, h and the
// product P of the a up to it, so that the value with the true start h0 is
// h + P h0: the start needs to be known only after the loads and exponentials are
// done. The starts come by joining (P, h) pairs, first over the block's warps in
// shared memory, then over the cluster's blocks in each other's shared memory, and
// the cluster walks on with the last value as carry. So the axis is read once, every
// wait is a hardware barrier, and the order of all operations is fixed.
#pragma once

#include <algorithm>

#include "xm_common.cuh"
#include "xm_sequences.cuh"

namespace xm {

// keep = sigmoid(f), take = sigmoid(-f) = 1 - keep, each with its own relative
// precision: with t = exp(-|f|) <= 1 the larger is r = 1 / (1 + t) and the smaller
// t r, so no difference of nearby values is formed and nothing overflows.
struct Gate {
    float keep, take;
};
__device__ __forceinline__ Gate gate_of(float f) {
    const float t = ex2_approx(-fabsf(f) * kLog2e);
    const float r = rcp_approx(1.0f + t), s = t * r;
    return f >= 0.0f ? Gate{r, s} : Gate{s, r};
}

constexpr int kGateWarps = 8;                     // warps of a block along the tokens
constexpr int kGateThreads = 32 * kGateWarps;
constexpr int kGateSteps = 8;                     // tokens of a warp
constexpr int kGateTokens = kGateWarps * kGateSteps;  // tokens of a block
constexpr int kGateMaxCluster = 8;

// The tokens that a cluster walks: a batch row, several short ones, or the packed row.
struct GateSpans {
    int rows;     // spans
    int length;   // tokens of a span; with cu the span is [cu[0], cu[units])
    int tiles;    // blocks of channels
    int cluster;  // blocks of a cluster
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

// A (P, h) pair stands for h0 -> P h0 + h. Where a sequence starts inside, nothing of
// h0 gets through, whatever it is (infinities and NaN too): P = kCut says so. Products
// of gates are kept above zero, so that an infinite h0 outlasts their underflow as it
// does step by step.
constexpr float kCut = -1.0f;
constexpr float kLeast = 1.4e-45f;
__device__ __forceinline__ float apply(float P, float h, float h0) { return P < 0.0f ? h : fmaf(P, h0, h); }
__device__ __forceinline__ float product(float P, float before) {
    return P < 0.0f || before < 0.0f ? kCut : fmaxf(P * before, kLeast);
}

// Shared memory of the join; parity alternates from step to step.
template <int V>
struct GateJoin {
    float2 warp[2][kGateWarps][32 * V];
    float2 block[2][kGateMaxCluster][32 * V];
};

template <int V>
__device__ __forceinline__ void load_pairs(const float2 *p, float (&P)[V], float (&h)[V]) {
    if constexpr (V == 2) {
        const float4 w = *reinterpret_cast<const float4 *>(p);
        P[0] = w.x; h[0] = w.y; P[1] = w.z; h[1] = w.w;
    } else {
        P[0] = p->x; h[0] = p->y;
    }
}
template <int V>
__device__ __forceinline__ void store_pairs(float2 *p, const float (&P)[V], const float (&h)[V]) {
    if constexpr (V == 2) *reinterpret_cast<float4 *>(p) = make_float4(P[0], h[0], P[1], h[1]);
    else *p = make_float2(P[0], h[0]);
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
__device__ __forceinline__ void store_to_block(const void *smem, unsigned rank, float2 v) {
    const uint32_t here = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
    uint32_t there;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(rank));
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(v.x), "f"(v.y) : "memory");
}

// Joins the warps' pairs (P, h) of one step. Returns the value that this warp's
// tokens start from and moves `carry` from the step's start to its end. Called by
// all threads of the cluster.
template <int V>
__device__ __forceinline__ void gate_join(GateJoin<V> &s, int parity, int cluster, unsigned rank, const float (&P)[V],
                                          const float (&h)[V], float (&carry)[V], float (&start)[V]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    store_pairs<V>(&s.warp[parity][warp][V * lane], P, h);
    __syncthreads();
    if (cluster > 1) {
        if (warp == kGateWarps - 1) {  // the block's pair, to every block
            float bp[V], bh[V];
            load_pairs<V>(&s.warp[parity][0][V * lane], bp, bh);
#pragma unroll
            for (int w = 1; w < kGateWarps; ++w) {
                float wp[V], wh[V];
                load_pairs<V>(&s.warp[parity][w][V * lane], wp, wh);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    bh[v] = apply(wp[v], wh[v], bh[v]);
                    bp[v] = product(wp[v], bp[v]);
                }
            }
            for (int r = 0; r < cluster; ++r)
#pragma unroll
                for (int v = 0; v < V; ++v) store_to_block(&s.block[parity][rank][V * lane + v], r, make_float2(bp[v], bh[v]));
        }
        cluster_barrier();
        for (int r = 0; r < cluster; ++r) {
            if (r == static_cast<int>(rank)) {
#pragma unroll
                for (int v = 0; v < V; ++v) start[v] = carry[v];
            }
            float bp[V], bh[V];
            load_pairs<V>(&s.block[parity][r][V * lane], bp, bh);
#pragma unroll
            for (int v = 0; v < V; ++v) carry[v] = apply(bp[v], bh[v], carry[v]);
        }
#pragma unroll
        for (int w = 0; w < kGateWarps - 1; ++w) {
            if (w >= warp) break;
            float wp[V], wh[V];
            load_pairs<V>(&s.warp[parity][w][V * lane], wp, wh);
#pragma unroll
            for (int v = 0; v < V; ++v) start[v] = apply(wp[v], wh[v], start[v]);
        }
    } else {
#pragma unroll
        for (int w = 0; w < kGateWarps; ++w) {
            if (w == warp) {
#pragma unroll
                for (int v = 0; v < V; ++v) start[v] = carry[v];
            }
            float wp[V], wh[V];
            load_pairs<V>(&s.warp[parity][w][V * lane], wp, wh);
#pragma unroll
            for (int v = 0; v < V; ++v) carry[v] = apply(wp[v], wh[v], carry[v]);
        }
    }
}

// A token's part of its warp's start: h0 -> P h0, with the care of kCut and kLeast.
__device__ __forceinline__ float through(float P, float h0) {
    if (P < 0.0f) return 0.0f;
    return P == 0.0f && !(fabsf(h0) <= 3.4028235e38f) ? h0 : P * h0;
}

template <typename T, int V>
__device__ __forceinline__ void unpack_word(const void *p, float (&v)[V]) {
    if constexpr (V == 2) {
        const float2 f = unpack2<T>(*static_cast<const uint32_t *>(p));
        v[0] = f.x;
        v[1] = f.y;
    } else {
        v[0] = to_f32<T>(*static_cast<const T *>(p));
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_word(T *p, const float (&v)[V]) {
    if constexpr (V == 2) *reinterpret_cast<uint32_t *>(p) = pack2<T>(v[0], v[1]);
    else *p = from_f32<T>(v[0]);
}

// How a call is cut: blocks of channels, spans, and the cluster along the tokens.
GateSpans gate_spans(const SeqArgs &q, int dim, int channels);

// One cluster per tile and span, or fewer that take several spans in turn.
template <typename... Params, typename... Args>
cudaError_t launch_gate_clusters(void (*kernel)(Params...), size_t smem, const GateSpans &g, cudaStream_t stream,
                                 const Args &...args) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    const int64_t most = std::max<int64_t>(1, (int64_t(1) << 30) / (static_cast<int64_t>(g.tiles) * g.cluster));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(g.rows, most) * g.tiles * g.cluster));
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
