// xm_gate.cuh -- what the gated linear recurrence and its backward pass share: the
// gate, the walk over sequences, and the scan over the token axis.
//
// Both are first-order recurrences per channel, h <- a h + b, forwards over the
// tokens or backwards. A lane holds two channels, a warp some consecutive
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
#include "xm_umma.cuh"

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

constexpr int kGateChannels = 64;  // channels of a block
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
template <int kWarps, typename F>
__device__ __forceinline__ void for_empty_sequences(const SeqArgs &q, int block, int blocks, F &&f) {
    if (q.cu == nullptr && q.seqlen > 0) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (long long s0 = (static_cast<long long>(block) * kWarps + warp) * 32; s0 < q.units;
         s0 += 32LL * kWarps * blocks) {
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

// A (P, h) pair stands for h0 -> P h0 + h. Where a sequence starts inside, P is zero
// and nothing of h0 may get through; elsewhere products of gates are kept above zero,
// so that an infinite h0 outlasts their underflow as it does step by step. As long as
// h0 is finite a multiply-add does both, and it only gives a finite value if h0 was
// one; values that come out infinite or NaN are joined once more with `join_any`.
struct GatePair {
    float2 P, h;
};
constexpr float kLeast = 1.4e-45f;
__device__ __forceinline__ float2 above_zero(float2 P) { return make_float2(fmaxf(P.x, kLeast), fmaxf(P.y, kLeast)); }
__device__ __forceinline__ bool finite2(float2 v) { return fabsf(v.x) <= 3.4028235e38f && fabsf(v.y) <= 3.4028235e38f; }
__device__ __forceinline__ float2 join(const GatePair &p, float2 h0) { return __ffma2_rn(p.P, h0, p.h); }
__device__ __forceinline__ float2 join_any(const GatePair &p, float2 h0) {
    return make_float2(p.P.x == 0.0f ? p.h.x : fmaf(p.P.x, h0.x, p.h.x), p.P.y == 0.0f ? p.h.y : fmaf(p.P.y, h0.y, p.h.y));
}
__device__ __forceinline__ float2 product(float2 P, float2 before) {
    const float2 v = __fmul2_rn(P, before);
    return make_float2(P.x == 0.0f || before.x == 0.0f ? 0.0f : fmaxf(v.x, kLeast),
                       P.y == 0.0f || before.y == 0.0f ? 0.0f : fmaxf(v.y, kLeast));
}

// Shared memory of the join; parity alternates from step to step.
template <int kWarps>
struct GateJoin {
    GatePair warp[2][kWarps][32];
    GatePair block[2][kGateMaxCluster][32];
    uint64_t arrived[2];  // the cluster's pairs of a step are here
};

__device__ __forceinline__ GatePair load_pair(const GatePair &p) {
    const float4 w = *reinterpret_cast<const float4 *>(&p);
    return GatePair{make_float2(w.x, w.y), make_float2(w.z, w.w)};
}

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
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
// A pair into another block's shared memory; its bytes count on that block's `arrived`. (A cluster barrier per step,
// whose release waits for the block's own stores to global memory, took two to five microseconds under load.)
__device__ __forceinline__ void send_pair(uint32_t there, uint32_t arrived, const GatePair &p) {
    asm volatile(
        "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(there),
        "f"(p.P.x), "f"(p.P.y), "f"(p.h.x), "f"(p.h.y), "r"(arrived)
        : "memory");
}
// Waits for a phase of `arrived`, a bounded number of times.
__device__ __forceinline__ bool wait_arrived(uint64_t *arrived, uint32_t phase) {
    const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(arrived));
    for (uint32_t i = 0; i < (1u << 22); ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t"
            "}\n"
            : "=r"(done)
            : "r"(a), "r"(phase)
            : "memory");
        if (done) return true;
    }
    return false;
}

// Before the first join and behind the last, by all threads of a cluster of several blocks: every block has begun, and
// none has left, while others write into its shared memory.
template <int kWarps>
__device__ __forceinline__ void gate_join_begin(GateJoin<kWarps> &s) {
    if (threadIdx.x == 0) {
        umma::mbar_init(&s.arrived[0], 1);
        umma::mbar_init(&s.arrived[1], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    cluster_barrier();
}

// The values before and behind this block's part of the step.
template <int K, int kWarps>
__device__ __forceinline__ void join_blocks(const GateJoin<kWarps> &s, int parity, unsigned rank, float2 &start,
                                            float2 &carry) {
    const int lane = threadIdx.x & 31;
    GatePair p[K];
#pragma unroll
    for (int r = 0; r < K; ++r) p[r] = load_pair(s.block[parity][r][lane]);
#pragma unroll
    for (int r = 0; r < K; ++r) {
        if (r == static_cast<int>(rank)) start = carry;
        carry = join(p[r], carry);
    }
}

// Joins the warps' pairs of step `turn`, counted from 0 over the kernel. Returns the
// value that this warp's tokens start from and moves `carry` from the step's start to
// its end. Called by all threads of the cluster; also a __syncthreads() of the block.
// `lost`: a wait gave up, here or before.
template <int kWarps>
__device__ __forceinline__ float2 gate_join(GateJoin<kWarps> &s, unsigned turn, int cluster, unsigned rank,
                                            const GatePair &mine, float2 &carry, bool &lost) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, parity = turn & 1;
    *reinterpret_cast<float4 *>(&s.warp[parity][warp][lane]) = make_float4(mine.P.x, mine.P.y, mine.h.x, mine.h.y);
    __syncthreads();
    float2 start = carry, behind = carry;
    if (cluster > 1) {
        if (warp == kWarps - 1) {  // the block's pair, to every block
            GatePair p[kWarps];
#pragma unroll
            for (int w = 0; w < kWarps; ++w) p[w] = load_pair(s.warp[parity][w][lane]);
            GatePair b = p[0];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) b.h = join(p[w], b.h), b.P = product(p[w].P, b.P);
            if (!finite2(b.h)) {
                b.h = p[0].h;
#pragma unroll
                for (int w = 1; w < kWarps; ++w) b.h = join_any(p[w], b.h);
            }
            for (int r = 0; r < cluster; ++r)
                send_pair(address_in_block(&s.block[parity][rank][lane], r), address_in_block(&s.arrived[parity], r), b);
            if (lane == 0) umma::mbar_arrive_expect_tx(&s.arrived[parity], cluster * 32 * sizeof(GatePair));
        }
        if (!lost) lost = !wait_arrived(&s.arrived[parity], turn >> 1 & 1);
        if (cluster == 2) join_blocks<2>(s, parity, rank, start, behind);
        else if (cluster == 4) join_blocks<4>(s, parity, rank, start, behind);
        else join_blocks<8>(s, parity, rank, start, behind);
#pragma unroll
        for (int w = 0; w < kWarps - 1; ++w)
            if (w < warp) start = join(load_pair(s.warp[parity][w][lane]), start);
    } else {
        GatePair p[kWarps];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) p[w] = load_pair(s.warp[parity][w][lane]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w == warp) start = behind;
            behind = join(p[w], behind);
        }
    }
    if (!__all_sync(kFullMask, finite2(start) && finite2(behind))) {
        behind = start = carry;
        for (int r = 0; r < (cluster > 1 ? cluster : 0); ++r) {
            if (r == static_cast<int>(rank)) start = behind;
            behind = join_any(load_pair(s.block[parity][r][lane]), behind);
        }
        for (int w = 0; w < kWarps; ++w) {
            if (cluster == 1) behind = join_any(load_pair(s.warp[parity][w][lane]), behind);
            if (w < warp) start = join_any(load_pair(s.warp[parity][w][lane]), start);
        }
    }
    carry = behind;
    return start;
}

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
    // (words: only by active lanes)
    __device__ __forceinline__ void store(T *row, float2 v) const {
        if constexpr (kWords) {
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
template <typename T, int kTokens>
struct GateTile {
    T v[kTokens][kGateChannels];
    __device__ __forceinline__ float2 at(int row, int lane) const {
        if constexpr (sizeof(T) == 2) return unpack2<T>(*reinterpret_cast<const uint32_t *>(&v[row][2 * lane]));
        else return *reinterpret_cast<const float2 *>(&v[row][2 * lane]);
    }
};
// Rows first + 0 .. kTokens - 1 of a tensor's channels; those outside [lo, hi) are left out.
template <int kThreads, typename T, int kTokens>
__device__ __forceinline__ void copy_tile(GateTile<T, kTokens> &dst, const T *src, int first, int lo, int hi, int dim,
                                          int tile) {
    constexpr int kPer = 16 / static_cast<int>(sizeof(T)), kWordsRow = kGateChannels / kPer;
    constexpr int kRows = kThreads / kWordsRow;  // rows per pass
    const int col = threadIdx.x % kWordsRow * kPer, row = threadIdx.x / kWordsRow;
    if (tile * kGateChannels + col >= dim) return;
    const T *p = src + static_cast<int64_t>(first + row) * dim + tile * kGateChannels + col;
    if (first >= lo && first + kTokens <= hi) {
#pragma unroll
        for (int k = 0; k < kTokens; k += kRows, p += static_cast<int64_t>(kRows) * dim) cp_async16(&dst.v[row + k][col], p, 16);
        return;
    }
#pragma unroll
    for (int k = 0; k < kTokens; k += kRows, p += static_cast<int64_t>(kRows) * dim) {
        const int t = first + row + k;
        if (t >= lo && t < hi) cp_async16(&dst.v[row + k][col], p, 16);
    }
}

// Zeros where copy_tile leaves channels behind the last one out: what is computed of them stays finite.
template <typename R>
__device__ __forceinline__ void clear_ring(R &ring, int dim, int tile) {
    if ((tile + 1) * kGateChannels <= dim) return;
    for (unsigned i = threadIdx.x; i < sizeof(R) / 16; i += blockDim.x)
        reinterpret_cast<float4 *>(&ring)[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    __syncthreads();
}

// How a call is cut: blocks of channels, spans, and the cluster along the tokens, of which a block takes `tokens` at a
// time.
GateSpans gate_spans(const SeqArgs &q, int dim, int tokens);

template <typename... Params, typename... Args>
cudaError_t launch_gate_clusters(void (*kernel)(Params...), int threads, size_t smem, const GateSpans &g, cudaStream_t stream,
                                 const Args &...args) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(g.width) * g.tiles * g.cluster);
    cfg.blockDim = dim3(threads);
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
