// scan_varlen.cu -- SelectiveScanVarlenFn for sm_100a.
//
// Math, per token t and channel d (state n = 0 .. N - 1):
//   dt = softplus?(delta + bias), h_n = exp(dt A_n) h_n + dt u B_n,
//   y = (D u + sum_n C_n h_n) silu(z).
// The recurrence is diagonal in n with no contraction, so it has no tensor-core
// form: the cost is one exponential and two and a half packed FP32 instructions
// per (token, channel, state).
//
// Design. States live in registers: kLanes lanes share two adjacent channels, each
// with NS states of both, so a B or C value read from shared memory serves two
// channels (what shared memory returns to registers, 128 bytes a clock, is the
// second bound). A warp owns 64 / kLanes adjacent channels and walks the tokens
// in groups of eight:
//   prep      a lane takes the delta and u of one token and a quarter of the
//             channels, computes dt and dt u and puts them into shared memory;
//             the group's B / C rows follow as float32;
//   states    token by token, each lane reads its channels' (dt, dt u) and the B
//             and C of its states (broadcasts), updates the states and leaves
//             sum_n C_n h_n in shared memory;
//   epilogue  the lane that prepped a token adds the skip, gates and stores
//             with one wide store.
// u, delta, z, B and C arrive in shared memory by asynchronous copies two groups
// ahead. (Loads into registers a group ahead were waited for long before their
// use: a lone warp took 495 clocks a token with them and 357 without.) So
// addresses, conversions, softplus and gate cost a few instructions per
// token beside the states' work, and the tensors move in 16-byte words. With up
// to 16 states a warp needs no other warp (B and C come from the caches), and a
// block is one warp: the finest grain for balancing. With more states, four
// warps share the staged B / C rows.
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
#include <cfloat>
#include <climits>

#include "xm_common.cuh"
#include "xm_kernels.h"
#include "xm_sequences.cuh"

namespace xm {
namespace {

constexpr int kGroup = 8;   // tokens per group
constexpr int kStages = 3;  // groups in flight or in use

struct ScanGeom {
    int row_tokens;   // tokens of a batch row
    int bl, nbr;      // tokens per block, blocks per row
    int chan_blocks;  // channel blocks of a group
    bool vec_io;      // u, delta, z, out rows in words of a warp's channels (16 bytes at most)
    bool vec_bc;      // B / C rows in 16-byte words
    bool vec_state;   // rows of the states and of A in 16-byte words
    float *H, *I;     // [blocks][dim][dstate]: state at a block's end; start of the sequence that leaves it
    float *S;         // [blocks][dim]: sum of dt over a block that a sequence crosses
};

template <int kBytes>
__device__ __forceinline__ void copy_async(void *smem, const void *gmem) {
    const uint32_t s = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
    if constexpr (kBytes == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(s), "l"(gmem) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(s), "l"(gmem), "n"(kBytes) : "memory");
}

__device__ __forceinline__ float scan_silu(float z) { return z * rcp_approx(1.0f + ex2_approx(-z * kLog2e)); }

// V consecutive floats of shared memory (aligned to V, at most 16 bytes).
template <int V>
__device__ __forceinline__ void load_floats(const float *p, float (&v)[V]) {
    if constexpr (V == 1) v[0] = *p;
    if constexpr (V == 2) {
        const float2 w = *reinterpret_cast<const float2 *>(p);
        v[0] = w.x; v[1] = w.y;
    }
    if constexpr (V >= 4) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const float4 w = *reinterpret_cast<const float4 *>(p + i);
            v[i] = w.x; v[i + 1] = w.y; v[i + 2] = w.z; v[i + 3] = w.w;
        }
    }
}

// V consecutive elements of shared memory as floats (aligned to V elements, at
// most 16 bytes).
template <typename T, int V>
__device__ __forceinline__ void load_elems(const T *p, float (&v)[V]) {
    if constexpr (V * sizeof(T) == 2) {
        v[0] = to_f32<T>(*p);
    } else if constexpr (sizeof(T) == 4) {
        load_floats<V>(p, v);
    } else {
        uint32_t w[V / 2];
        if constexpr (V == 2) w[0] = *reinterpret_cast<const uint32_t *>(p);
        if constexpr (V == 4) {
            const uint2 r = *reinterpret_cast<const uint2 *>(p);
            w[0] = r.x; w[1] = r.y;
        }
        if constexpr (V == 8) {
            const uint4 r = *reinterpret_cast<const uint4 *>(p);
            w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
        }
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 f = unpack2<T>(w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T *p, const float (&v)[V]) {
    if constexpr (V * sizeof(T) <= 4) {
        if constexpr (V == 1) *p = from_f32<T>(v[0]);
        else *reinterpret_cast<uint32_t *>(p) = pack2<T>(v[0], v[1]);
    } else if constexpr (sizeof(T) == 4) {
        if constexpr (V == 2) *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
#pragma unroll
        for (int i = 0; i + 4 <= V; i += 4)
            *reinterpret_cast<float4 *>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else if constexpr (V == 4) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    } else {
        *reinterpret_cast<uint4 *>(p) =
            make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
}

// Shapes of a kernel instance: NS states of each of two channels per lane, kLanes
// lanes per channel pair.
template <typename T, int NS, int kLanes>
struct Shape {
    static constexpr int NP = NS * kLanes;            // states held per channel
    static constexpr int kWarps = NP > 16 ? 4 : 1;    // warps that share the B / C rows
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int CPW = 64 / kLanes;           // channels per warp
    static constexpr int V = CPW >= 4 ? CPW / 4 : 1;  // channels that a lane preps
    static constexpr int kLpt = CPW / V;              // lanes per prepped token
    static constexpr int kPer = 16 / static_cast<int>(sizeof(T));  // elements of a 16-byte word
    // one stage of the ring, in elements: delta, u, z [kGroup][CPW], and for the block B, C [kGroup][NP]
    static constexpr int kIo = kGroup * CPW, kBc = kGroup * NP;
    static constexpr int kCopy = CPW * static_cast<int>(sizeof(T)) < 16 ? CPW : kPer;  // elements of an io copy
    static constexpr int kIoStage = 3 * kIo, kBcStage = 2 * kBc;
    // floats per warp: (dt, dt u) pairs, outputs, bias, D; and per block: B, C
    static constexpr int kWarpFloats = 3 * kGroup * CPW + 2 * CPW;
    static constexpr int kBcFloats = 2 * kBc;
    static constexpr size_t kSmem = (kWarps * kWarpFloats + kBcFloats) * sizeof(float) +
                                    kStages * (kWarps * kIoStage + kBcStage) * sizeof(T);
};

// Place (in floats) of a channel pair's (dt, dt u, dt, dt u) in its token's row:
// the row's 16-byte words are permuted so that the prep's stores (8 lanes: two
// tokens, four neighbouring runs of channels) and the states' loads meet no bank
// twice. y_at: the same for a channel's output.
template <int CPW>
__device__ __forceinline__ int pair_at(int tok, int pair) {
    int w = pair;
    if constexpr (CPW == 32) w ^= ((w >> 3) & 1) ^ ((tok & 1) << 1);
    if constexpr (CPW == 16) w ^= tok & 1;
    return (tok * (CPW / 2) + w) * 4;
}
template <int CPW>
__device__ __forceinline__ int y_at(int tok, int c) {
    return tok * CPW + (CPW == 32 ? c ^ ((tok & 1) << 2) : c);
}

// One token's state update of both channels; returns their sums of C_n h_n over
// this lane's states when kOut. dd: (dt, dt u) of both; `row`: this lane's first
// group of four states in the token's B row, C at row + coff. kSafe: states past
// N (clear bits of `real`) are held at zero whatever dt u is; otherwise they stay
// there only while it is finite.
// (Moving 4 of the 16 exponentials to a polynomial on the FMA pipe left the time
// of a full machine as it was, 213 -> 218 clocks per token and warp, and 8 of them
// cost 20 %: instruction issue is as near its bound as the exponential unit.)
template <int NS, int kLanes, bool kOut, bool kSafe>
__device__ __forceinline__ float2 scan_token(float2 (&h)[NS], const float2 (&a2)[NS], float4 dd, const float *row,
                                             int coff, unsigned real) {
    const float2 dt[2] = {make_float2(dd.x, dd.x), make_float2(dd.z, dd.z)};
    const float2 du[2] = {make_float2(dd.y, dd.y), make_float2(dd.w, dd.w)};
    float2 a[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const float2 x = __fmul2_rn(dt[i / (NS / 2)], a2[i]);
        a[i] = make_float2(ex2_approx(x.x), ex2_approx(x.y));
    }
    float2 y[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
    for (int q = 0; q < NS / 4; ++q) {
        const float4 b4 = *reinterpret_cast<const float4 *>(row + 4 * kLanes * q);
        float4 c4 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if constexpr (kOut) c4 = *reinterpret_cast<const float4 *>(row + coff + 4 * kLanes * q);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float2 b = k == 0 ? make_float2(b4.x, b4.y) : make_float2(b4.z, b4.w);
            const float2 c = k == 0 ? make_float2(c4.x, c4.y) : make_float2(c4.z, c4.w);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const int i = m * (NS / 2) + 2 * q + k;
                h[i] = __ffma2_rn(a[i], h[i], __fmul2_rn(b, du[m]));
                if constexpr (kSafe) {
                    if (!(real >> (4 * q + 2 * k) & 1)) h[i].x = 0.0f;
                    if (!(real >> (4 * q + 2 * k + 1) & 1)) h[i].y = 0.0f;
                }
                if constexpr (kOut) y[m] = __ffma2_rn(h[i], c, y[m]);
            }
        }
    }
    return make_float2(y[0].x + y[0].y, y[1].x + y[1].y);
}

// First sequence whose start is at or behind t (units: none); dense rows directly.
__device__ __forceinline__ int first_from(const SeqArgs &q, int t, int row, bool at_row_start) {
    if (q.cu == nullptr) return at_row_start ? row : row + 1;
    return seq_first_from(q, t);
}

// kEnds: the first pass.
template <typename T, int NS, int kLanes, bool kEnds>
__global__ void __launch_bounds__(Shape<T, NS, kLanes>::kThreads) scan_block_kernel(const ScanArgs p,
                                                                                      const ScanGeom g) {
    using S = Shape<T, NS, kLanes>;
    constexpr bool kOut = !kEnds;
    constexpr int NP = S::NP, CPW = S::CPW, V = S::V;
    extern __shared__ float4 smem_f4[];
    const SeqArgs &q = p.seq;
    const int tid = threadIdx.x, lane = tid & 31, N = p.dstate;
    float *const bc = reinterpret_cast<float *>(smem_f4);  // [kGroup][NP] B, then C
    float *const dd = bc + S::kBcFloats + (tid >> 5) * S::kWarpFloats;  // [kGroup][CPW / 2] (dt, dt u) x 2
    float *const ys = dd + 2 * kGroup * CPW;                           // [kGroup][CPW]
    float *const par = ys + kGroup * CPW;                              // bias [CPW], D [CPW]
    T *const ring = reinterpret_cast<T *>(bc + S::kBcFloats + S::kWarps * S::kWarpFloats);
    T *const io_ring = ring + (tid >> 5) * (kStages * S::kIoStage);
    T *const bc_ring = ring + S::kWarps * (kStages * S::kIoStage);
    const int part = lane % kLanes, pair = lane / kLanes;
    const int cblocks = g.chan_blocks * p.groups;
    const int cblk = blockIdx.x % cblocks;
    const int blk = blockIdx.x / cblocks;
    const int grp = cblk / g.chan_blocks;
    const int dpg = p.dim / p.groups;
    const int c0 = ((cblk - grp * g.chan_blocks) * S::kWarps + (tid >> 5)) * CPW;  // the warp's first channel in the group
    // this lane's two channels; past the group's last one they repeat it and nothing of them is stored
    const int own = c0 + 2 * pair;
    const bool active[2] = {own < dpg, own + 1 < dpg};
    const int d[2] = {grp * dpg + min(own, dpg - 1), grp * dpg + min(own + 1, dpg - 1)};
    const int per_row = kEnds ? g.nbr - 1 : g.nbr;
    const int row = blk / per_row, j = blk - row * per_row;
    const int row0 = row * g.row_tokens, row1 = row0 + g.row_tokens;
    const int t0 = row0 + j * g.bl, t1 = t0 + min(g.bl, row1 - t0);
    const int b0 = row * g.nbr;  // the row's first block in H, I, S
    auto barrier = [&] {
        if constexpr (S::kWarps == 1) __syncwarp();
        else __syncthreads();
    };

    float2 h[NS], a2[NS];  // [channel][state pair]
    auto state_of = [&](int i) { return 4 * ((i >> 2) * kLanes + part) + (i & 3); };  // i-th state of this lane
    auto zero = [&] {
#pragma unroll
        for (int i = 0; i < NS; ++i) h[i] = make_float2(0.0f, 0.0f);
    };
    // v <- or -> the lane's states of row `r` of a [rows][dim][dstate] tensor
    auto load_row = [&](const float *base, long long r, float2 (&v)[NS]) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const float *s = base + (static_cast<size_t>(r) * p.dim + d[m]) * N;
#pragma unroll
            for (int i = 0; i < NS; i += 4) {
                const int n = state_of(i), k = m * (NS / 2) + i / 2;
                if (g.vec_state) {
                    const float4 w = n < N ? *reinterpret_cast<const float4 *>(s + n) : make_float4(0, 0, 0, 0);
                    v[k] = make_float2(w.x, w.y);
                    v[k + 1] = make_float2(w.z, w.w);
                } else {
                    v[k] = make_float2(n < N ? s[n] : 0.0f, n + 1 < N ? s[n + 1] : 0.0f);
                    v[k + 1] = make_float2(n + 2 < N ? s[n + 2] : 0.0f, n + 3 < N ? s[n + 3] : 0.0f);
                }
            }
        }
    };
    auto store_row = [&](float *base, long long r, const float2 (&v)[NS]) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            if (!active[m]) continue;
            float *s = base + (static_cast<size_t>(r) * p.dim + d[m]) * N;
#pragma unroll
            for (int i = 0; i < NS; i += 4) {
                const int n = state_of(i), k = m * (NS / 2) + i / 2;
                if (g.vec_state) {
                    if (n < N) *reinterpret_cast<float4 *>(s + n) = make_float4(v[k].x, v[k].y, v[k + 1].x, v[k + 1].y);
                } else {
                    if (n < N) s[n] = v[k].x;
                    if (n + 1 < N) s[n + 1] = v[k].y;
                    if (n + 2 < N) s[n + 2] = v[k + 1].x;
                    if (n + 3 < N) s[n + 3] = v[k + 1].y;
                }
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
    float ssum[2] = {0.0f, 0.0f};
    bool crossing = false;  // kEnds: the sequence began before this block
    int from_block = -1;    // outputs: the block in which the sequence that reaches into this one begins
    if constexpr (kEnds) {
        n = first_from(q, t1, row, false) - 1;
        if (n < 0) return;
        const int s = seq_start(q, n);
        e = seq_end(q, n, s);
        if (e <= t1) return;  // nothing continues behind this block
        crossing = s < t0;
        t = max(s, t0);
        stop = t1;
    } else {
        n = first_from(q, t0, row, j == 0) - 1;
        int s = n >= 0 ? seq_start(q, n) : 0;
        e = n >= 0 ? seq_end(q, n, s) : 0;
        stop = q.cu != nullptr ? min(t1, seq_start(q, units)) : t1;
        t = t0;
        if (e > t0) {
            from_block = min(max(0, (s - row0) / g.bl), j - 1);
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

    if (part == 0) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            par[2 * pair + m] = p.bias != nullptr ? p.bias[d[m]] : 0.0f;
            par[CPW + 2 * pair + m] = p.D != nullptr ? p.D[d[m]] : 0.0f;
        }
    }
    // The prep's view: token `tok` of the group, channels [ch, ch + V) of the warp, `valid` of them in the group.
    const int tok = lane / S::kLpt, ch = lane % S::kLpt * V;
    const int valid = tok < kGroup ? min(V, max(0, dpg - c0 - ch)) : 0;
    const size_t D = p.dim;
    const size_t io0 = static_cast<size_t>(grp) * dpg + c0;  // the warp's first channel
    const bool gate = kOut && p.z != nullptr;
    const T *const io_src[3] = {static_cast<const T *>(p.delta) + io0, static_cast<const T *>(p.u) + io0,
                                gate ? static_cast<const T *>(p.z) + io0 : nullptr};
    T *const op = static_cast<T *>(p.out) + io0 + ch;
    const size_t bstride = static_cast<size_t>(p.groups) * N;
    const T *const Bp = static_cast<const T *>(p.B) + static_cast<size_t>(grp) * N;
    const T *const Cp = static_cast<const T *>(p.C) + static_cast<size_t>(grp) * N;
    // Brings the group at token `at` into stage `st`; nothing behind the walk is read.
    auto fetch = [&](int at, int st) {
        T *const io = io_ring + st * S::kIoStage;
        T *const rows = bc_ring + st * S::kBcStage;
        if (g.vec_io) {
            constexpr int kPerRow = CPW / S::kCopy, kCopies = kGroup * kPerRow;
#pragma unroll
            for (int k = 0; k < (kCopies + 31) / 32; ++k) {
                const int w = lane + 32 * k;
                const int i = w / kPerRow, c = w % kPerRow * S::kCopy;
                if (w < kCopies && at + i < stop && c0 + c < dpg) {
                    const size_t o = static_cast<size_t>(at + i) * D + c;
#pragma unroll
                    for (int m = 0; m < 3; ++m)
                        if (m < 2 || gate) copy_async<S::kCopy * sizeof(T)>(io + m * S::kIo + i * CPW + c, io_src[m] + o);
                }
            }
        } else {
            for (int w = lane; w < S::kIo; w += 32) {
                const int i = w / CPW, c = w % CPW;
                if (at + i < stop && c0 + c < dpg) {
                    const size_t o = static_cast<size_t>(at + i) * D + c;
#pragma unroll
                    for (int m = 0; m < 3; ++m)
                        if (m < 2 || gate) io[m * S::kIo + w] = io_src[m][o];
                }
            }
        }
        if (g.vec_bc) {
            constexpr int kPerRow = NP / S::kPer, kCopies = (kOut ? 2 : 1) * kGroup * kPerRow;
#pragma unroll
            for (int k = 0; k < (kCopies + S::kThreads - 1) / S::kThreads; ++k) {
                const int w = tid + S::kThreads * k;
                const int m = w / (kGroup * kPerRow), i = w / kPerRow % kGroup, c = w % kPerRow * S::kPer;
                if (w < kCopies && at + i < stop && c < N)
                    copy_async<16>(rows + w * S::kPer, (m == 0 ? Bp : Cp) + static_cast<size_t>(at + i) * bstride + c);
            }
        } else {
            for (int w = tid; w < (kOut ? 2 : 1) * S::kBc; w += S::kThreads) {
                const int m = w / S::kBc, i = w / NP % kGroup, n = w % NP;
                if (at + i < stop && n < N) rows[w] = (m == 0 ? Bp : Cp)[static_cast<size_t>(at + i) * bstride + n];
            }
        }
        cp_async_commit();
    };
    if (N != NP) {  // padding states read B = C = 0
        for (int w = tid; w < kStages * S::kBcStage; w += S::kThreads) bc_ring[w] = from_f32<T>(0.0f);
        barrier();
    }

    // The first groups are on their way before the states and A are waited for.
    if (t < stop) {
        fetch(t, 0);
        fetch(t + kGroup, 1);
    }
    unsigned real = 0;  // which of a channel's NS states here are below N
#pragma unroll
    for (int i = 0; i < NS; ++i) real |= state_of(i) < N ? 1u << i : 0u;
    load_row(p.A, 0, a2);
#pragma unroll
    for (int i = 0; i < NS; ++i) a2[i] = __fmul2_rn(a2[i], make_float2(kLog2e, kLog2e));
    zero();
    if constexpr (kEnds) {
        if (!crossing) {
            load_start(n);
            store_row(g.I, b0 + j, h);
        }
    } else if (from_block >= 0) {
        load_row(g.H, b0 + from_block, h);
        // four blocks' loads at a time: one by one, each would wait for the caches
        constexpr int kJoin = 4;
        for (int b = from_block + 1; b < j; b += kJoin) {
            float2 v[kJoin][NS];
            float sd[kJoin][2];
#pragma unroll
            for (int k = 0; k < kJoin; ++k) {
                const int at = b0 + min(b + k, j - 1);
                load_row(g.H, at, v[k]);
                sd[k][0] = g.S[static_cast<size_t>(at) * p.dim + d[0]];
                sd[k][1] = g.S[static_cast<size_t>(at) * p.dim + d[1]];
            }
#pragma unroll
            for (int k = 0; k < kJoin; ++k) {
                if (b + k >= j) break;
                // In two factors of half the exponent: a block's growth may pass float32's range where zero has to
                // stay zero and a small state grow to what token by token gives (2^254 takes every state there is
                // to infinity).
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    const float m = 0.5f * sd[k][i / (NS / 2)];
                    const float2 x = __fmul2_rn(make_float2(m, m), a2[i]);
                    const float2 e = make_float2(ex2_approx(fminf(x.x, 127.0f)), ex2_approx(fminf(x.y, 127.0f)));
                    h[i] = __ffma2_rn(e, __fmul2_rn(e, h[i]), v[k][i]);
                }
            }
        }
    }
    int st = 0;  // stage of the group at t
    for (; t < stop; t += kGroup) {
        cp_async_wait<kStages - 2>();
        barrier();
        // prep
        const T *const io = io_ring + st * S::kIoStage;
        bool odd = false;  // with padding states: some dt u of the warp is not finite
        if (valid > 0 && t + tok < stop) {
            float dt[V], du[V], u[V], bias[V];
            load_floats<V>(par + ch, bias);
            load_elems<T, V>(io + tok * CPW + ch, dt);
            load_elems<T, V>(io + S::kIo + tok * CPW + ch, u);
#pragma unroll
            for (int i = 0; i < V; ++i) dt[i] += bias[i];
            if (p.softplus) {
#pragma unroll
                for (int i = 0; i < V; i += 2) {
                    const float2 v = softplus_pair(make_float2(dt[i], dt[V > 1 ? i + 1 : i]));
                    dt[i] = v.x;
                    if (V > 1) dt[i + 1] = v.y;
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) du[i] = dt[i] * u[i];
            if (N != NP) {
#pragma unroll
                for (int i = 0; i < V; ++i) odd |= !(fabsf(du[i]) <= 3.402823466e38f);
            }
            if constexpr (V >= 2) {
#pragma unroll
                for (int i = 0; i < V; i += 2)
                    *reinterpret_cast<float4 *>(dd + pair_at<CPW>(tok, (ch + i) / 2)) =
                        make_float4(dt[i], du[i], dt[i + 1], du[i + 1]);
            } else {
                *reinterpret_cast<float2 *>(dd + pair_at<CPW>(tok, ch / 2) + 2 * (ch & 1)) = make_float2(dt[0], du[0]);
            }
        }
        {
            const T *const src = bc_ring + st * S::kBcStage;
#pragma unroll
            for (int w = tid * S::kPer; w < (kOut ? 2 : 1) * S::kBc; w += S::kThreads * S::kPer) {
                float v[S::kPer];
                load_elems<T, S::kPer>(src + w, v);
#pragma unroll
                for (int i = 0; i < S::kPer; i += 4)
                    *reinterpret_cast<float4 *>(bc + w + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            }
        }
        // the stage of the group before this one is free: its last readers passed the barrier above
        fetch(t + 2 * kGroup, st == 0 ? kStages - 1 : st - 1);
        barrier();
        // states
        if constexpr (!kEnds)
            if (t == e) event(t);
        odd = N != NP && __any_sync(kFullMask, odd);
        const float *rows = bc + 4 * part;
        // Sums over the channel pair's lanes: the first exchange leaves a lane one of the two channels.
        auto joined = [&](float2 y) {
            const bool hi = part & 1;
            float v = hi ? y.y : y.x;
            v += __shfl_xor_sync(kFullMask, hi ? y.x : y.y, 1);
#pragma unroll
            for (int o = 2; o < kLanes; o *= 2) v += __shfl_xor_sync(kFullMask, v, o);
            return v;
        };
        if (t + kGroup <= stop && (kEnds || e >= t + kGroup) && !odd) {
            // The outputs are stored behind the loop: a store between two tokens would keep
            // the next one's loads, and with them its exponentials, behind this one's sums.
            float v8[kGroup];
#pragma unroll
            for (int i = 0; i < kGroup; ++i) {
                const float4 v = *reinterpret_cast<const float4 *>(dd + pair_at<CPW>(i, pair));
                const float2 y = scan_token<NS, kLanes, kOut, false>(h, a2, v, rows + i * NP, kGroup * NP, real);
                if constexpr (kOut) {
                    v8[i] = joined(y);
                } else {
                    ssum[0] += v.x;
                    ssum[1] += v.z;
                }
            }
            if constexpr (kOut) {
                if (part < 2) {
#pragma unroll
                    for (int i = 0; i < kGroup; ++i) ys[y_at<CPW>(i, 2 * pair + part)] = v8[i];
                }
            }
        } else {
            // a sequence or the walk ends inside the group, or padding states need care
#pragma unroll 1
            for (int i = 0; i < kGroup && t + i < stop; ++i) {
                if constexpr (!kEnds)
                    if (i > 0 && t + i == e) event(t + i);
                const float4 v = *reinterpret_cast<const float4 *>(dd + pair_at<CPW>(i, pair));
                const float2 y = scan_token<NS, kLanes, kOut, true>(h, a2, v, rows + i * NP, kGroup * NP, real);
                if constexpr (kOut) {
                    const float o = joined(y);
                    if (part < 2) ys[y_at<CPW>(i, 2 * pair + part)] = o;
                } else {
                    ssum[0] += v.x;
                    ssum[1] += v.z;
                }
            }
        }
        barrier();
        // epilogue
        if constexpr (kOut) {
            if (valid > 0 && t + tok < stop) {
                float y[V], u[V], z[V], skip[V];
                load_floats<V>(par + CPW + ch, skip);
                load_elems<T, V>(io + S::kIo + tok * CPW + ch, u);
                if (gate) load_elems<T, V>(io + 2 * S::kIo + tok * CPW + ch, z);
                if constexpr (V >= 4) {
#pragma unroll
                    for (int i = 0; i < V; i += 4) {
                        const float4 w = *reinterpret_cast<const float4 *>(ys + y_at<CPW>(tok, ch + i));
                        y[i] = w.x; y[i + 1] = w.y; y[i + 2] = w.z; y[i + 3] = w.w;
                    }
                } else {
                    load_floats<V>(ys + y_at<CPW>(tok, ch), y);
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    y[i] = fmaf(skip[i], u[i], y[i]);
                    if (gate) y[i] *= scan_silu(z[i]);
                }
                T *o = op + static_cast<size_t>(t + tok) * D;
                if (g.vec_io) {
                    store_pack<T, V>(o, y);
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (i < valid) o[i] = from_f32<T>(y[i]);
                }
            }
        }
        st = st == kStages - 1 ? 0 : st + 1;
    }
    cp_async_wait<0>();
    if constexpr (kEnds) {
        store_row(g.H, b0 + j, h);
        if (crossing && part == 0) {
#pragma unroll
            for (int m = 0; m < 2; ++m)  // a sum past float32's range stays finite: times A = 0 it has to be 0
                if (active[m])
                    g.S[static_cast<size_t>(b0 + j) * p.dim + d[m]] = fminf(fmaxf(ssum[m], -FLT_MAX), FLT_MAX);
        }
    } else if (e <= stop || !holding) {
        event(stop);
    }
}

struct ScanPlan {
    ScanGeom g;
    int ns, lanes;
    bool ends;
    size_t state_bytes, sum_bytes, total;
};

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// Lanes per channel pair, states per lane and the channel blocks of a group.
void plan_channels(const ScanArgs &a, ScanPlan &pl) {
    const int N = a.dstate;
    pl.ns = N <= 8 ? 4 : 8;
    pl.lanes = 2;
    while (pl.lanes * pl.ns < N) pl.lanes *= 2;
    const int cpb = 64 / pl.lanes * (N > 16 ? 4 : 1), dpg = a.dim / a.groups;
    pl.g.chan_blocks = std::max(1, (dpg + cpb - 1) / cpb);
}

ScanPlan plan_scan(const ScanArgs &a) {
    ScanPlan pl{};
    ScanGeom &g = pl.g;
    const int N = a.dstate;
    plan_channels(a, pl);
    const int rows = a.seq.cu != nullptr ? 1 : a.seq.units;
    g.row_tokens = a.seq.cu != nullptr ? a.seq.tokens : a.seq.seqlen;
    const int64_t ctas = std::max<int64_t>(1, static_cast<int64_t>(g.chan_blocks) * a.groups * rows);
    const int64_t warps = ctas * (N > 16 ? 4 : 1), slots = 4LL * current_device_sm_count();
    // Cut rows into the number of blocks with the least estimated time, in clocks (measured at d_state 16):
    // a scheduler with w warps takes walk[w] for a token of each; it holds 3 of the second pass and 4 of
    // the first, whose tokens cost 0.76 as much; a CTA spends 7000 before and behind its tokens, a second
    // launch 5000, and the last block's join 450 per block.
    // Microseconds by number of blocks: a row of 512 tokens x 4096 channels 89 uncut, 37 in 8, 34 by the rule
    // (13), 52 in 32; 4096 x 256: 682, 173 in 8, 45 (74), 56 in 128; 8192 x 2048: 1376, 342 in 8, 196 (27),
    // 304 in 128; four rows of 1024 x 1024: 175, 65 in 8, 58 (13), 78 in 32; eight rows of 2048 x 4096: 480
    // uncut (the rule's), 660 to 685 in 2 to 6.
    constexpr double kWalk[5] = {0.0, 335.0, 470.0, 640.0, 848.0};
    auto pass = [&](int64_t count, int64_t bl, int cap, double factor) {
        const int64_t full = count / (cap * slots), rest = count % (cap * slots);
        const double start = 7000.0;
        double t = full * (factor * bl * kWalk[cap] + start);
        if (rest > 0) t += factor * bl * kWalk[(rest + slots - 1) / slots] + start;
        return t;
    };
    double best = 0.0;
    const int most = std::min(128, 1 + g.row_tokens / kGroup);
    for (int nbr = 1; nbr <= most; ++nbr) {
        const int64_t each = (static_cast<int64_t>(g.row_tokens) + nbr - 1) / nbr;
        const int64_t bl = std::max<int64_t>(kGroup, (each + kGroup - 1) / kGroup * kGroup);
        if (nbr > 1 && (g.row_tokens + bl - 1) / bl != nbr) continue;
        double cost = pass(warps * nbr, bl, 3, 1.0);
        if (nbr > 1) cost += pass(warps * (nbr - 1), bl, 4, 0.76) + 5000.0 + 450.0 * nbr;
        if (nbr == 1 || cost < best) {
            best = cost;
            g.bl = static_cast<int>(std::min<int64_t>(bl, INT32_MAX));
            g.nbr = nbr;
        }
    }
    pl.ends = g.nbr > 1;
    if (pl.ends) {
        const size_t blocks = static_cast<size_t>(rows) * g.nbr;
        pl.state_bytes = round256(blocks * a.dim * N * sizeof(float));
        pl.sum_bytes = round256(blocks * a.dim * sizeof(float));
        pl.total = 2 * pl.state_bytes + pl.sum_bytes;
    }
    return pl;
}

template <typename T, int NS, int kLanes, bool kEnds>
cudaError_t launch_pass(const ScanArgs &a, const ScanGeom &g, cudaStream_t stream) {
    using S = Shape<T, NS, kLanes>;
    const int64_t rows = a.seq.cu != nullptr ? 1 : a.seq.units;
    const int64_t ctas = rows * (kEnds ? g.nbr - 1 : g.nbr) * g.chan_blocks * a.groups;
    if constexpr (S::kSmem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(scan_block_kernel<T, NS, kLanes, kEnds>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(S::kSmem));
        if (e != cudaSuccess) return e;
    }
    scan_block_kernel<T, NS, kLanes, kEnds><<<static_cast<unsigned>(ctas), S::kThreads, S::kSmem, stream>>>(a, g);
    return cudaGetLastError();
}

template <typename T, int NS, int kLanes>
cudaError_t launch_passes(const ScanArgs &a, const ScanPlan &pl, cudaStream_t stream) {
    using S = Shape<T, NS, kLanes>;
    ScanGeom g = pl.g;
    auto on = [&](const void *p) { return reinterpret_cast<uintptr_t>(p) % (S::kCopy * sizeof(T)) == 0; };
    g.vec_io = a.dim / a.groups % std::max(S::kCopy, S::V) == 0 && on(a.u) && on(a.delta) && on(a.z) && on(a.out);
    g.vec_bc = a.dstate % S::kPer == 0 && aligned16(a.B) && aligned16(a.C);
    g.vec_state = a.dstate % 4 == 0 && aligned16(a.A) && aligned16(a.init) && aligned16(a.final_state);
    if (pl.ends) {
        const cudaError_t e = launch_pass<T, NS, kLanes, true>(a, g, stream);
        if (e != cudaSuccess) return e;
    }
    return launch_pass<T, NS, kLanes, false>(a, g, stream);
}

template <typename T>
cudaError_t launch_type(const ScanArgs &a, const ScanPlan &pl, cudaStream_t stream) {
    if (pl.ns == 4) return launch_passes<T, 4, 2>(a, pl, stream);
    switch (pl.lanes) {
        case 2: return launch_passes<T, 8, 2>(a, pl, stream);
        case 4: return launch_passes<T, 8, 4>(a, pl, stream);
        case 8: return launch_passes<T, 8, 8>(a, pl, stream);
        case 16: return launch_passes<T, 8, 16>(a, pl, stream);
        default: return launch_passes<T, 8, 32>(a, pl, stream);
    }
}

}  // namespace

int64_t scan_varlen_blocks(const ScanArgs &a) {
    ScanPlan pl{};
    plan_channels(a, pl);
    return static_cast<int64_t>(pl.g.chan_blocks) * a.groups * (a.seq.cu != nullptr ? 1 : a.seq.units);
}

size_t scan_varlen_workspace(const ScanArgs &a) { return plan_scan(a).total; }

cudaError_t launch_scan_varlen(const ScanArgs &a, void *workspace, cudaStream_t stream) {
    ScanPlan pl = plan_scan(a);
    if (pl.ends) {
        char *ws = static_cast<char *>(workspace);
        pl.g.H = reinterpret_cast<float *>(ws);
        pl.g.I = reinterpret_cast<float *>(ws + pl.state_bytes);
        pl.g.S = reinterpret_cast<float *>(ws + 2 * pl.state_bytes);
    }
    switch (a.io) {
        case IoType::kBF16: return launch_type<__nv_bfloat16>(a, pl, stream);
        case IoType::kF16: return launch_type<__half>(a, pl, stream);
        default: return launch_type<float>(a, pl, stream);
    }
}

}  // namespace xm
