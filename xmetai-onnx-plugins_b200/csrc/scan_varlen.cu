// scan_varlen.cu -- SelectiveScanVarlenFn for sm_100a.
//
// Math, per token t and channel d (state n = 0 .. N - 1):
//   dt = softplus?(delta + bias), h_n = exp(dt A_n) h_n + dt u B_n,
//   y = (D u + sum_n C_n h_n) silu(z).
// The recurrence is diagonal in n with no contraction, so it has no tensor-core
// form: the cost is one exponential and two and a half packed FP32 instructions
// per (token, channel, state).
//
// Design. A channel's states live in registers: one lane per channel for up to
// 16 states, a power of two of lanes with 16 states each above. Adjacent lanes
// are adjacent channels, so the token-major tensors are read and written in
// whole sectors; the B / C rows of a tile of tokens are staged in shared memory
// as float32 and read by broadcast.
//
// The token axis of a batch row is cut into blocks of equal length whatever the
// sequences are, so the work is balanced without the host knowing their
// lengths. A block walks the sequences that it meets: at a sequence's start it
// takes up that sequence's state, at its end it stores the final one. Where
// blocks cut sequences, a first pass (kEnds) runs the tokens between the last
// sequence start in a block and the block's end, from the sequence's state or
// from zero, and leaves the state H and, with a zero start, the sum S of dt; the
// second pass (outputs) forms its start h <- exp(A S) h + H over the blocks
// since the sequence's start. A sequence's state row is read in the first pass
// where a later block stores the final state into it, so in-place states are
// never read after another block's store.
#include <algorithm>

#include "xm_common.cuh"
#include "xm_kernels.h"
#include "xm_sequences.cuh"

namespace xm {
namespace {

constexpr int kScanThreads = 128;
constexpr int kScanStage = 512;  // states x tokens of a staged B / C tile

struct ScanGeom {
    int lpc;         // lanes per channel
    int row_tokens;  // tokens of a batch row
    int bl, nbr;     // tokens per block, blocks per row
    int chan_blocks; // channel blocks of a group
    int tile;        // tokens per staged tile: a multiple of 8
    bool vec_bc;     // B / C rows as 16-byte words (one lane per channel, N = NS)
    bool vec_state;  // state rows as 16-byte words
    float *H, *I;    // [blocks][dim][dstate]: state at a block's end; start of the sequence that leaves it
    float *S;        // [blocks][dim]: sum of dt over a block that a sequence crosses
};

// One token's state update; returns sum_n C_n h_n over this lane's states when
// kOut. `row` is this lane's first state of the token's B row, `coff` the
// distance to the C row, `qs` the distance between its groups of four states.
template <int NS, bool PAD, bool kOut>
__device__ __forceinline__ float scan_token(float2 (&h)[NS / 2], const float2 (&a2)[NS / 2], float dt, float du,
                                            const float *row, int coff, int qs, unsigned real) {
    const float2 dt2 = make_float2(dt, dt), du2 = make_float2(du, du);
    float2 y2 = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int q = 0; q < NS / 4; ++q) {
        const float4 b = *reinterpret_cast<const float4 *>(row + q * qs);
        float4 c = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if constexpr (kOut) c = *reinterpret_cast<const float4 *>(row + coff + q * qs);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = 2 * q + k;
            const float2 x = __fmul2_rn(dt2, a2[i]);
            const float2 a = make_float2(ex2_approx(x.x), ex2_approx(x.y));
            const float2 b2 = k == 0 ? make_float2(b.x, b.y) : make_float2(b.z, b.w);
            h[i] = __ffma2_rn(a, h[i], __fmul2_rn(b2, du2));
            if constexpr (PAD) {  // states past N stay zero whatever u holds
                if (!(real >> (2 * i) & 1)) h[i].x = 0.0f;
                if (!(real >> (2 * i + 1) & 1)) h[i].y = 0.0f;
            }
            if constexpr (kOut) y2 = __ffma2_rn(h[i], k == 0 ? make_float2(c.x, c.y) : make_float2(c.z, c.w), y2);
        }
    }
    return y2.x + y2.y;
}

__device__ __forceinline__ float scan_silu(float z) { return z * rcp_approx(1.0f + ex2_approx(-z * kLog2e)); }

// dt of one token
__device__ __forceinline__ float scan_dt(float delta, float bias, bool softplus) {
    const float x = delta + bias;
    return softplus ? softplus_pair(make_float2(x, x)).x : x;
}

// Stages the B (and C) rows of tokens [t, t + tile) below `stop` as float32 into
// dst: [tile][NP] B, then [tile][NP] C, zeros elsewhere. kFixed: rows of exactly
// NS states as 16-byte words, loaded ahead into registers.
template <typename T, int NS, bool kOut>
struct BcStage {
    static constexpr int kTile = kScanStage / NS;
    static constexpr int kPer = 16 / static_cast<int>(sizeof(T));   // states per word
    static constexpr int kWords = kScanStage / kPer;                // words of one tensor's tile
    static constexpr int kRegs = (kOut ? 2 : 1) * kWords / kScanThreads < 1 ? 1 : (kOut ? 2 : 1) * kWords / kScanThreads;
    uint4 r[kRegs];

    __device__ __forceinline__ void load(const T *B, const T *C, size_t stride, int t, int stop) {
#pragma unroll
        for (int i = 0; i < kRegs; ++i) {
            int w = threadIdx.x + i * kScanThreads;
            const bool c = kOut && w >= kWords;
            w -= c ? kWords : 0;
            const int tok = t + w / (NS / kPer);
            r[i] = make_uint4(0, 0, 0, 0);
            if (w < kWords && tok < stop)
                r[i] = __ldg(reinterpret_cast<const uint4 *>((c ? C : B) + tok * stride + (w % (NS / kPer)) * kPer));
        }
    }
    __device__ __forceinline__ void store(float *dst) const {
#pragma unroll
        for (int i = 0; i < kRegs; ++i) {
            int w = threadIdx.x + i * kScanThreads;
            if (w >= (kOut ? 2 : 1) * kWords) break;
            float4 *o = reinterpret_cast<float4 *>(dst + w * kPer);  // C's tile follows B's
            if constexpr (sizeof(T) == 4) {
                o[0] = *reinterpret_cast<const float4 *>(&r[i]);
            } else {
                const float2 a = unpack2<T>(r[i].x), b = unpack2<T>(r[i].y), c = unpack2<T>(r[i].z),
                             d = unpack2<T>(r[i].w);
                o[0] = make_float4(a.x, a.y, b.x, b.y);
                o[1] = make_float4(c.x, c.y, d.x, d.y);
            }
        }
    }
};

template <typename T>
__device__ __forceinline__ void stage_any(const T *B, const T *C, size_t stride, int N, int NP, int tile, int t,
                                          int stop, float *dst) {
    for (int e = threadIdx.x; e < tile * NP; e += kScanThreads) {
        const int i = e / NP, n = e - i * NP;
        const bool ok = n < N && t + i < stop;
        const size_t at = (t + i) * stride + n;
        dst[e] = ok ? to_f32<T>(B[at]) : 0.0f;
        if (C != nullptr) dst[tile * NP + e] = ok ? to_f32<T>(C[at]) : 0.0f;
    }
}

// First sequence whose start is at or behind t (units: none); dense rows directly.
__device__ __forceinline__ int first_from(const SeqArgs &q, int t, int row, bool at_row_start) {
    if (q.cu == nullptr) return at_row_start ? row : row + 1;
    int lo = 0, hi = q.units;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (seq_start(q, mid) >= t) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// NS states per lane. kMulti: several lanes per channel. PAD: N < NS * lanes.
// kEnds: the first pass.
template <typename T, int NS, bool kMulti, bool PAD, bool kEnds>
__global__ void __launch_bounds__(kScanThreads) scan_block_kernel(const ScanArgs p, const ScanGeom g) {
    extern __shared__ float4 smem_f4[];
    float *const stage = reinterpret_cast<float *>(smem_f4);
    constexpr bool kOut = !kEnds;
    const SeqArgs &q = p.seq;
    const int tid = threadIdx.x, N = p.dstate;
    const int lpc = kMulti ? g.lpc : 1;
    const int part = kMulti ? tid & (lpc - 1) : 0;
    const int NP = NS * lpc, qs = 4 * lpc;
    const int cblocks = g.chan_blocks * p.groups;
    const int cblk = blockIdx.x % cblocks;
    const int blk = blockIdx.x / cblocks;
    const int grp = cblk / g.chan_blocks;
    const int dpg = p.dim / p.groups;
    const int ci = (cblk - grp * g.chan_blocks) * (kScanThreads / lpc) + tid / lpc;
    const bool active = ci < dpg;
    const int d = grp * dpg + (active ? ci : dpg - 1);
    const int per_row = kEnds ? g.nbr - 1 : g.nbr;
    const int row = blk / per_row, j = blk - row * per_row;
    const int row0 = row * g.row_tokens, row1 = row0 + g.row_tokens;
    const int t0 = row0 + j * g.bl, t1 = t0 + min(g.bl, row1 - t0);
    const int b0 = row * g.nbr;  // the row's first block in H, I, S

    float2 h[NS / 2], a2[NS / 2];
    unsigned real = 0;
    auto state_of = [&](int i) { return 4 * ((i >> 2) * lpc + part) + (i & 3); };  // i-th state of this lane
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int n = state_of(i);
        const float a = n < N ? p.A[static_cast<size_t>(d) * N + n] * kLog2e : 0.0f;
        (i & 1 ? a2[i / 2].y : a2[i / 2].x) = a;
        real |= n < N ? 1u << i : 0u;
    }
    auto zero = [&] {
#pragma unroll
        for (int i = 0; i < NS / 2; ++i) h[i] = make_float2(0.0f, 0.0f);
    };
    // v <- or -> the lane's states of row `r` of a [rows][dim][dstate] tensor
    auto load_row = [&](const float *base, long long r, float2 (&v)[NS / 2]) {
        const float *s = base + (static_cast<size_t>(r) * p.dim + d) * N;
#pragma unroll
        for (int i = 0; i < NS; i += 4) {
            const int n = state_of(i);
            if (g.vec_state) {
                const float4 w = n < N ? *reinterpret_cast<const float4 *>(s + n) : make_float4(0, 0, 0, 0);
                v[i / 2] = make_float2(w.x, w.y);
                v[i / 2 + 1] = make_float2(w.z, w.w);
            } else {
                v[i / 2] = make_float2(n < N ? s[n] : 0.0f, n + 1 < N ? s[n + 1] : 0.0f);
                v[i / 2 + 1] = make_float2(n + 2 < N ? s[n + 2] : 0.0f, n + 3 < N ? s[n + 3] : 0.0f);
            }
        }
    };
    auto store_row = [&](float *base, long long r, const float2 (&v)[NS / 2]) {
        if (!active) return;
        float *s = base + (static_cast<size_t>(r) * p.dim + d) * N;
#pragma unroll
        for (int i = 0; i < NS; i += 4) {
            const int n = state_of(i);
            if (g.vec_state) {
                if (n < N)
                    *reinterpret_cast<float4 *>(s + n) =
                        make_float4(v[i / 2].x, v[i / 2].y, v[i / 2 + 1].x, v[i / 2 + 1].y);
            } else {
                if (n < N) s[n] = v[i / 2].x;
                if (n + 1 < N) s[n + 1] = v[i / 2].y;
                if (n + 2 < N) s[n + 2] = v[i / 2 + 1].x;
                if (n + 3 < N) s[n + 3] = v[i / 2 + 1].y;
            }
        }
    };
    auto load_start = [&](int n) {  // the state that sequence n starts from
        const long long r = seq_row(q, n);
        if (p.init != nullptr && seq_live(q, n, r)) load_row(p.init, r, h);
        else zero();
    };
    auto store_final = [&](int n) {
        if (p.final_state == nullptr) return;
        const long long r = seq_row(q, n);
        if (r >= 0) store_row(p.final_state, r, h);
    };

    // The tokens to walk, [t, stop), the sequence n that holds t and its end e.
    const int units = q.cu != nullptr ? q.units : row + 1;
    int n, e, t, stop;
    float ssum = 0.0f;
    bool crossing = false;  // kEnds: the sequence began before this block
    zero();
    if constexpr (kEnds) {
        n = first_from(q, t1, row, false) - 1;
        if (n < 0) return;
        const int s = seq_start(q, n);
        e = seq_end(q, n, s);
        if (e <= t1) return;  // nothing continues behind this block
        crossing = s < t0;
        t = max(s, t0);
        stop = t1;
        if (!crossing) {
            load_start(n);
            store_row(g.I, b0 + j, h);
        }
    } else {
        n = first_from(q, t0, row, j == 0) - 1;
        int s = n >= 0 ? seq_start(q, n) : 0;
        e = n >= 0 ? seq_end(q, n, s) : 0;
        stop = q.cu != nullptr ? min(t1, seq_start(q, units)) : t1;
        t = t0;
        if (e > t0) {
            const int bs = min(max(0, (s - row0) / g.bl), j - 1);
            load_row(g.H, b0 + bs, h);
            for (int b = bs + 1; b < j; ++b) {
                float2 v[NS / 2];
                load_row(g.H, b0 + b, v);
                const float sd = g.S[static_cast<size_t>(b0 + b) * p.dim + d];
#pragma unroll
                for (int i = 0; i < NS / 2; ++i) {
                    const float2 x = __fmul2_rn(make_float2(sd, sd), a2[i]);
                    h[i] = __ffma2_rn(make_float2(ex2_approx(x.x), ex2_approx(x.y)), h[i], v[i]);
                }
            }
        } else {
            t = n + 1 < units ? max(t0, seq_start(q, n + 1)) : t0;
            e = t;  // the event at t takes up sequence n + 1
        }
    }
    const bool last_block = j == g.nbr - 1;
    // At t = e: sequence n is done; take up the next one with tokens.
    bool holding = !kEnds && e > t;  // h belongs to sequence n
    auto event = [&](int at) {
        if (holding) store_final(n);
        holding = false;
        e = INT_MAX;
        for (++n; n < units; ++n) {
            const int s = seq_start(q, n);
            if (at >= stop && s >= t1 && !last_block) return;  // starts in a later block
            const int end = seq_end(q, n, s);
            if (end <= at) {  // no tokens: its final state is the one it starts from
                load_start(n);
                store_final(n);
                continue;
            }
            if (at >= stop) return;
            e = end;
            if (end > t1) load_row(g.I, b0 + j, h);
            else load_start(n);
            holding = true;
            return;
        }
    };

    const float bias = p.bias != nullptr ? p.bias[d] : 0.0f;
    const float skip = p.D != nullptr ? p.D[d] : 0.0f;
    const T *const up = static_cast<const T *>(p.u) + d;
    const T *const dp = static_cast<const T *>(p.delta) + d;
    const T *const zp = kOut && p.z != nullptr ? static_cast<const T *>(p.z) + d : nullptr;
    T *const op = static_cast<T *>(p.out) + d;
    const size_t bstride = static_cast<size_t>(p.groups) * N;
    const T *const Bp = static_cast<const T *>(p.B) + static_cast<size_t>(grp) * N;
    const T *const Cp = kOut ? static_cast<const T *>(p.C) + static_cast<size_t>(grp) * N : nullptr;
    const int tile = g.tile, coff = tile * NP, buf = (kOut ? 2 : 1) * tile * NP;
    const size_t D = p.dim;

    auto finish = [&](float y, float u, float z) {
        if constexpr (kMulti)
            for (int o = lpc >> 1; o > 0; o >>= 1) y += __shfl_xor_sync(kFullMask, y, o);
        y = fmaf(skip, u, y);
        return zp != nullptr ? y * scan_silu(z) : y;
    };

    BcStage<T, NS, kOut> ahead;
    const int first = t;
    int side = 0;
    if (!kMulti && g.vec_bc && t < stop) ahead.load(Bp, Cp, bstride, t, stop);
    T ru[8], rd[8], rz[8];
    auto prefetch = [&](int at) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const size_t o = static_cast<size_t>(min(at + i, stop - 1)) * D;
            ru[i] = up[o];
            rd[i] = dp[o];
            if (zp != nullptr) rz[i] = zp[o];
        }
    };
    if (t < stop) prefetch(t);
    for (; t < stop; t += 8) {
        const int in_tile = (t - first) % tile;
        if (in_tile == 0) {
            if (!kMulti && g.vec_bc) {
                // two buffers: a warp may still read the last tile while others store this one
                side ^= 1;
                ahead.store(stage + side * buf);
                __syncthreads();
                ahead.load(Bp, Cp, bstride, t + tile, stop);
            } else {
                __syncthreads();
                stage_any<T>(Bp, Cp, bstride, N, NP, tile, t, stop, stage);
                __syncthreads();
            }
        }
        const float *rows = stage + side * buf + in_tile * NP + 4 * part;
        if constexpr (!kEnds)
            if (t == e) event(t);
        if (t + 8 <= stop && (kEnds || e >= t + 8)) {
            float uu[8], dt[8], zz[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uu[i] = to_f32<T>(ru[i]);
                dt[i] = to_f32<T>(rd[i]) + bias;
                if (zp != nullptr) zz[i] = to_f32<T>(rz[i]);
                else zz[i] = 0.0f;
            }
            prefetch(t + 8);
            if (p.softplus) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float2 v = softplus_pair(make_float2(dt[i], dt[i + 1]));
                    dt[i] = v.x;
                    dt[i + 1] = v.y;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = scan_token<NS, PAD, kOut>(h, a2, dt[i], dt[i] * uu[i], rows + i * NP, coff, qs, real);
                if constexpr (kOut) {
                    const float v = finish(y, uu[i], zz[i]);
                    if (active && part == 0) op[(static_cast<size_t>(t) + i) * D] = from_f32<T>(v);
                } else {
                    ssum += dt[i];
                }
            }
        } else {
            // a sequence ends inside the group, or the walk does: token by token
            for (int i = 0; i < 8 && t + i < stop; ++i) {
                if constexpr (!kEnds)
                    if (i > 0 && t + i == e) event(t + i);
                const size_t o = (static_cast<size_t>(t) + i) * D;
                const float u = to_f32<T>(up[o]), dt = scan_dt(to_f32<T>(dp[o]), bias, p.softplus);
                const float y = scan_token<NS, PAD, kOut>(h, a2, dt, dt * u, rows + i * NP, coff, qs, real);
                if constexpr (kOut) {
                    const float v = finish(y, u, zp != nullptr ? to_f32<T>(zp[o]) : 0.0f);
                    if (active && part == 0) op[o] = from_f32<T>(v);
                } else {
                    ssum += dt;
                }
            }
            if (t + 8 < stop) prefetch(t + 8);
        }
    }
    if constexpr (kEnds) {
        store_row(g.H, b0 + j, h);
        if (crossing && active && part == 0) g.S[static_cast<size_t>(b0 + j) * p.dim + d] = ssum;
    } else if (e <= stop || !holding) {
        event(stop);
    }
}

struct ScanPlan {
    ScanGeom g;
    int ns;
    bool multi, pad, ends;
    size_t state_bytes, sum_bytes, total;
};

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

ScanPlan plan_scan(const ScanArgs &a) {
    ScanPlan pl{};
    ScanGeom &g = pl.g;
    const int N = a.dstate;
    pl.ns = N <= 8 ? 8 : 16;
    g.lpc = 1;
    while (g.lpc * pl.ns < N) g.lpc *= 2;
    pl.multi = g.lpc > 1;
    pl.pad = N != pl.ns * g.lpc;
    g.tile = std::max(8, kScanStage / (pl.ns * g.lpc));
    const int cpb = kScanThreads / g.lpc, dpg = a.dim / a.groups;
    g.chan_blocks = std::max(1, (dpg + cpb - 1) / cpb);
    const int rows = a.seq.cu != nullptr ? 1 : a.seq.units;
    g.row_tokens = a.seq.cu != nullptr ? a.seq.tokens : a.seq.seqlen;
    // Blocks until every SM has about four CTAs (four warps per scheduler), of 64 tokens at least.
    const int64_t want = static_cast<int64_t>(4) * current_device_sm_count();
    const int64_t ctas = std::max<int64_t>(1, static_cast<int64_t>(g.chan_blocks) * a.groups * rows);
    const int64_t nbr = std::min<int64_t>({(want + ctas - 1) / ctas, std::max(1, g.row_tokens / 64), 128});
    g.bl = static_cast<int>((g.row_tokens + nbr - 1) / nbr);
    g.bl = std::max(8, (g.bl + 7) / 8 * 8);
    g.nbr = std::max(1, (g.row_tokens + g.bl - 1) / g.bl);
    pl.ends = g.nbr > 1;
    if (pl.ends) {
        const size_t blocks = static_cast<size_t>(rows) * g.nbr;
        pl.state_bytes = round256(blocks * a.dim * N * sizeof(float));
        pl.sum_bytes = round256(blocks * a.dim * sizeof(float));
        pl.total = 2 * pl.state_bytes + pl.sum_bytes;
    }
    return pl;
}

template <typename T, int NS, bool kMulti, bool PAD, bool kEnds>
cudaError_t launch_pass(const ScanArgs &a, const ScanPlan &pl, cudaStream_t stream) {
    const ScanGeom &g = pl.g;
    const int64_t rows = a.seq.cu != nullptr ? 1 : a.seq.units;
    const int64_t ctas = rows * (kEnds ? g.nbr - 1 : g.nbr) * g.chan_blocks * a.groups;
    if (ctas > INT32_MAX) return cudaErrorInvalidConfiguration;
    const size_t smem = static_cast<size_t>(kEnds ? 1 : 2) * (g.vec_bc ? 2 : 1) * g.tile * NS * g.lpc * sizeof(float);
    scan_block_kernel<T, NS, kMulti, PAD, kEnds>
        <<<static_cast<unsigned>(ctas), kScanThreads, smem, stream>>>(a, g);
    return cudaGetLastError();
}

template <typename T, int NS, bool kMulti, bool PAD>
cudaError_t launch_passes(const ScanArgs &a, const ScanPlan &pl, cudaStream_t stream) {
    if (pl.ends) {
        const cudaError_t e = launch_pass<T, NS, kMulti, PAD, true>(a, pl, stream);
        if (e != cudaSuccess) return e;
    }
    return launch_pass<T, NS, kMulti, PAD, false>(a, pl, stream);
}

template <typename T>
cudaError_t launch_type(const ScanArgs &a, const ScanPlan &pl, cudaStream_t stream) {
    if (pl.multi)
        return pl.pad ? launch_passes<T, 16, true, true>(a, pl, stream) : launch_passes<T, 16, true, false>(a, pl, stream);
    if (pl.ns == 16)
        return pl.pad ? launch_passes<T, 16, false, true>(a, pl, stream)
                      : launch_passes<T, 16, false, false>(a, pl, stream);
    return pl.pad ? launch_passes<T, 8, false, true>(a, pl, stream) : launch_passes<T, 8, false, false>(a, pl, stream);
}

}  // namespace

size_t scan_varlen_workspace(const ScanArgs &a) { return plan_scan(a).total; }

cudaError_t launch_scan_varlen(const ScanArgs &a, void *workspace, cudaStream_t stream) {
    ScanPlan pl = plan_scan(a);
    ScanGeom &g = pl.g;
    const size_t elem = a.io == IoType::kF32 ? 4 : 2;
    g.vec_bc = !pl.multi && !pl.pad && aligned16(a.B) && aligned16(a.C) && (a.dstate * elem) % 16 == 0;
    g.vec_state = a.dstate % 4 == 0 && aligned16(a.init) && aligned16(a.final_state);
    if (pl.ends) {
        char *ws = static_cast<char *>(workspace);
        g.H = reinterpret_cast<float *>(ws);
        g.I = reinterpret_cast<float *>(ws + pl.state_bytes);
        g.S = reinterpret_cast<float *>(ws + 2 * pl.state_bytes);
    }
    switch (a.io) {
        case IoType::kBF16: return launch_type<__nv_bfloat16>(a, pl, stream);
        case IoType::kF16: return launch_type<__half>(a, pl, stream);
        default: return launch_type<float>(a, pl, stream);
    }
}

}  // namespace xm
