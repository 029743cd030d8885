// causal_conv1d.cu -- CausalConv1dFn and CausalConv1dUpdateFn for sm_100a.
//
// Math, per channel d: y_t = act(bias + sum_{k < W} w_k x_(t - (W - 1) + k)),
// act = identity or v sigmoid(v); x before the sequence's first token comes from
// its state, the last W - 1 inputs of the tokens that went before.
//
// Bound by memory: x is read and y written once, against 2 W + 4 operations per
// element, so each layout's kernel moves words or half words of 16 bytes and keeps
// enough of them in flight:
//   conv_tokens_kernel    [tokens, dim]: a thread owns the channels of half a word
//                         and walks a block of tokens, the window in registers;
//   conv_channels_kernel  [dim, tokens]: a thread owns a word of consecutive
//                         tokens and takes the W - 1 before it from its
//                         neighbour lane;
//   conv_token_kernel     one token per sequence: a thread owns the channels of
//                         a word or half of one, their state and their weights.
//
// The states may be updated in place. With tokens first, one thread does all that
// touches a sequence's state of a channel: the one whose block holds the
// sequence's first token. It computes the first W - 1 tokens, which alone see the
// starting state, even where they reach into the next block, and then stores the
// final state. With channels first a small second launch stores it.
#include <algorithm>
#include <climits>

#include "xm_common.cuh"
#include "xm_kernels.h"
#include "xm_sequences.cuh"

namespace xm {
namespace {

constexpr int kConvThreads = 128;

__device__ __forceinline__ void cp_async8(void *smem, const void *gmem) {
    const uint32_t s = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(s), "l"(gmem) : "memory");
}

__device__ __forceinline__ float conv_act(float v, bool silu) {
    return silu ? v * rcp_approx(1.0f + ex2_approx(-v * kLog2e)) : v;
}

// y[i] = act(b[i] + sum_k w[k][i] x_k[i]) over V values, in pairs (FFMA2) where V is even.
template <int V, int W>
__device__ __forceinline__ void conv_values(float (&y)[V], const float (&b)[V], const float (&w)[W][V],
                                            const float (&x)[W][V], bool silu) {
    if constexpr (V == 1) {
        y[0] = b[0];
#pragma unroll
        for (int k = 0; k < W; ++k) y[0] = fmaf(w[k][0], x[k][0], y[0]);
        y[0] = conv_act(y[0], silu);
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            float2 v = make_float2(b[i], b[i + 1]);
#pragma unroll
            for (int k = 0; k < W; ++k)
                v = __ffma2_rn(make_float2(w[k][i], w[k][i + 1]), make_float2(x[k][i], x[k][i + 1]), v);
            if (silu) {
                const float2 t = __fmul2_rn(v, make_float2(-kLog2e, -kLog2e));
                const float2 e = __fadd2_rn(make_float2(ex2_approx(t.x), ex2_approx(t.y)), make_float2(1.0f, 1.0f));
                v = __fmul2_rn(v, make_float2(rcp_approx(e.x), rcp_approx(e.y)));
            }
            y[i] = v.x;
            y[i + 1] = v.y;
        }
    }
}

// Weights and bias of channels [d, d + V), weights by tap. `words`: both 16-byte aligned.
template <int V, int W>
__device__ __forceinline__ void conv_load_weights(const ConvArgs &p, int d, bool words, float (&w)[W][V], float (&b)[V]) {
    const float *src = p.weight + static_cast<size_t>(d) * W;
    float flat[V * W];
    if (V % 4 == 0 && words) {
#pragma unroll
        for (int i = 0; i + 4 <= V * W; i += 4) {
            const float4 v = __ldg(reinterpret_cast<const float4 *>(src + i));
            flat[i] = v.x; flat[i + 1] = v.y; flat[i + 2] = v.z; flat[i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V * W; ++i) flat[i] = __ldg(src + i);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int k = 0; k < W; ++k) w[k][i] = flat[i * W + k];
        b[i] = 0.0f;
    }
    if (p.bias != nullptr) {
        if (V % 4 == 0 && words) {
#pragma unroll
            for (int i = 0; i + 4 <= V; i += 4) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(p.bias + d + i));
                b[i] = v.x; b[i + 1] = v.y; b[i + 2] = v.z; b[i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) b[i] = __ldg(p.bias + d + i);
        }
    }
}

// Channels or tokens of one 16-byte word.
template <typename T>
constexpr int kWord = 16 / static_cast<int>(sizeof(T));

// One word's elements as floats.
template <typename T>
__device__ __forceinline__ void word_floats(const uint4 &r, float (&v)[kWord<T>]) {
    if constexpr (sizeof(T) == 4) {
        v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y);
        v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
    } else {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

template <typename T>
__device__ __forceinline__ uint4 floats_word(const float (&v)[kWord<T>]) {
    if constexpr (sizeof(T) == 4)
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    else
        return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}

// V elements from p: a 16-byte word, half of one, or a single element.
template <typename T, int V>
struct Elems {
    uint4 r;
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (V == 1) {
            if constexpr (sizeof(T) == 4) r.x = __float_as_uint(*p);
            else r.x = *reinterpret_cast<const unsigned short *>(p);
        } else if constexpr (V * sizeof(T) == 8) {
            const uint2 w = *reinterpret_cast<const uint2 *>(p);
            r.x = w.x;
            r.y = w.y;
        } else {
            r = *reinterpret_cast<const uint4 *>(p);
        }
    }
    __device__ __forceinline__ void floats(float (&v)[V]) const {
        if constexpr (V == 1) {
            if constexpr (sizeof(T) == 4) v[0] = __uint_as_float(r.x);
            else v[0] = unpack2<T>(r.x).x;
        } else if constexpr (V * sizeof(T) == 8) {
            if constexpr (sizeof(T) == 4) {
                v[0] = __uint_as_float(r.x);
                v[1] = __uint_as_float(r.y);
            } else {
                const float2 a = unpack2<T>(r.x), b = unpack2<T>(r.y);
                v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
            }
        } else {
            word_floats<T>(r, v);
        }
    }
};

template <typename T, int V>
__device__ __forceinline__ void store_elems(T *p, const float (&v)[V]) {
    if constexpr (V == 1) *p = from_f32<T>(v[0]);
    else if constexpr (V * sizeof(T) == 8 && sizeof(T) == 2)
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    else if constexpr (V * sizeof(T) == 8) *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
    else *reinterpret_cast<uint4 *>(p) = floats_word<T>(v);
}

// First sequence that starts at or behind t (units: none).
__device__ __forceinline__ int conv_first_from(const SeqArgs &q, int t) {
    if (q.cu == nullptr) return q.seqlen > 0 ? static_cast<int>((static_cast<long long>(t) + q.seqlen - 1) / q.seqlen) : 0;
    return seq_first_from(q, t);
}

// ------------------------------------------------------------------ tokens first

constexpr int kBatch = 4;    // tokens copied and used together
constexpr int kFlights = 4;  // batches in flight or in use

// Thread: V channels from channel V * (blockIdx.x * threads + thread); blockIdx.y:
// the block of `block` tokens. Each thread walks the sequences that meet it. Its
// words arrive by asynchronous copies in slots of shared memory that no other
// thread touches, three batches of four tokens ahead, so nothing is waited for
// but the batch in use and no barrier is needed. (Loads into registers, four or
// eight tokens ahead, left 16384 tokens x 4096 channels at 69 to 79 us.) Half words
// leave room for six CTAs per SM, whole words for four: 53 us against 57.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads) conv_tokens_kernel(const ConvArgs p, int block, int nblocks, bool words) {
    __shared__ uint2 conv_slots[V > 1 ? kFlights * kBatch * kConvThreads : 1];
    static_assert(V == 1 || V * sizeof(T) == 8, "a thread's channels are half a word");
    const SeqArgs &q = p.seq;
    const int d = (blockIdx.x * kConvThreads + threadIdx.x) * V;
    if (d >= p.dim) return;
    const size_t D = p.dim;
    const T *const x = static_cast<const T *>(p.x) + d;
    T *const out = static_cast<T *>(p.out) + d;
    float w[W][V], b[V];
    conv_load_weights<V, W>(p, d, words, w, b);
    for (int blk = blockIdx.y; blk < nblocks; blk += gridDim.y) {
        const int t0 = blk * block, t1 = t0 + min(block, q.tokens - t0);
        const bool last = blk == nblocks - 1;
        int n = conv_first_from(q, t0) - 1;  // the sequence that may reach into the block
        for (; n < q.units; ++n) {
            if (n < 0) continue;
            const int s = seq_start(q, n);
            if (s >= t1 && !last) break;
            const int e = seq_end(q, n, s);
            const bool own = s >= t0;  // this block holds the sequence's first token
            // its tokens here: an owned sequence's first W - 1 always, another's never
            const int from = own ? s : max(t0, min(e, s + W - 1));
            const int to = own ? max(min(e, t1), min(e, s + W - 1)) : min(e, t1);
            const long long row = own ? seq_row(q, n) : -1;
            const bool live = own && p.init != nullptr && seq_live(q, n, row);
            const size_t srow = (static_cast<size_t>(max(row, 0LL)) * D + d) * (W - 1);
            float win[W][V];  // the window's inputs; the last row is the token's own
#pragma unroll
            for (int k = 0; k < W - 1; ++k) {
                const int at = from - (W - 1) + k;
                if (own) {  // from = s: all before it is state
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        win[k + 1][i] =
                            live ? to_f32<T>(static_cast<const T *>(p.init)[srow + i * (W - 1) + k]) : 0.0f;
                } else if (from < to) {
                    Elems<T, V> r;
                    r.load(x + static_cast<size_t>(at) * D);
                    r.floats(win[k + 1]);
                }
            }
            auto step = [&](int t, const Elems<T, V> &r) {
                float y[V];
#pragma unroll
                for (int k = 0; k + 1 < W; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) win[k][i] = win[k + 1][i];
                r.floats(win[W - 1]);
                conv_values<V, W>(y, b, w, win, p.silu);
                store_elems<T, V>(out + static_cast<size_t>(t) * D, y);
            };
            int t = from;
            if constexpr (V > 1) {
                const int batches = (to - from) / kBatch;
                uint2 *const slot = conv_slots + threadIdx.x;
                auto bring = [&](int i) {
                    if (i < batches) {
#pragma unroll
                        for (int k = 0; k < kBatch; ++k)
                            cp_async8(slot + ((i % kFlights) * kBatch + k) * kConvThreads,
                                      x + (static_cast<size_t>(from) + i * kBatch + k) * D);
                    }
                    cp_async_commit();
                };
                if (batches > 0) {
#pragma unroll
                    for (int i = 0; i < kFlights - 1; ++i) bring(i);
                }
                for (int i = 0; i < batches; ++i, t += kBatch) {
                    cp_async_wait<kFlights - 2>();
                    Elems<T, V> cur[kBatch];
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        const uint2 v = slot[((i % kFlights) * kBatch + k) * kConvThreads];
                        cur[k].r.x = v.x;
                        cur[k].r.y = v.y;
                    }
                    bring(i + kFlights - 1);
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) step(t + k, cur[k]);
                }
            }
            for (; t < to; ++t) {
                Elems<T, V> r;
                r.load(x + static_cast<size_t>(t) * D);
                step(t, r);
            }
            if (own && p.final_state != nullptr && row >= 0) {
                T keep[V][W - 1];
#pragma unroll
                for (int k = 0; k < W - 1; ++k) {
                    const int at = e - (W - 1) + k;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        if (at >= s) keep[i][k] = x[static_cast<size_t>(at) * D + i];
                        else
                            keep[i][k] = live ? static_cast<const T *>(p.init)[srow + i * (W - 1) + (W - 1) + at - s]
                                              : from_f32<T>(0.0f);
                    }
                }
#pragma unroll
                for (int i = 0; i < V; ++i)
#pragma unroll
                    for (int k = 0; k < W - 1; ++k) static_cast<T *>(p.final_state)[srow + i * (W - 1) + k] = keep[i][k];
            }
        }
    }
}

// ------------------------------------------------------------------ channels first

// The state that sequence n of channel ch starts from (zeros where it starts anew).
template <typename T, int W>
__device__ __noinline__ float4 conv_start(const ConvArgs &p, int n, int ch) {
    float f[3] = {0.0f, 0.0f, 0.0f};
    const long long row = seq_row(p.seq, n);
    if (seq_live(p.seq, n, row)) {
        const T *s = static_cast<const T *>(p.init) + (static_cast<size_t>(row) * p.dim + ch) * (W - 1);
#pragma unroll
        for (int k = 0; k < W - 1; ++k) f[k] = to_f32<T>(s[k]);
    }
    return make_float4(f[0], f[1], f[2], 0.0f);
}

// One row of a [rows, seqlen] x: its channel, its sequences and their states.
template <typename T, int W>
struct ConvRow {
    const ConvArgs &p;
    const T *x;
    T *out;
    int ch;  // channel
    int n0;  // dense: the batch row's sequence
    float w[W], b;

    __device__ __forceinline__ ConvRow(const ConvArgs &args, long long row, long long batch, unsigned channel) : p(args) {
        take(row, batch, channel);
    }
    __device__ __forceinline__ void take(long long row, long long batch, unsigned channel) {
        x = static_cast<const T *>(p.x) + row * p.seq.seqlen;
        out = static_cast<T *>(p.out) + row * p.seq.seqlen;
        ch = static_cast<int>(channel);
        n0 = p.seq.cu != nullptr ? 0 : static_cast<int>(batch);
#pragma unroll
        for (int k = 0; k < W; ++k) w[k] = __ldg(p.weight + static_cast<size_t>(ch) * W + k);
        b = p.bias != nullptr ? __ldg(p.bias + ch) : 0.0f;
    }
    // The W - 1 inputs before sequence n's first token: its state, or zeros.
    __device__ __forceinline__ void start_of(int n, float (&h)[W - 1]) const {
        const float4 v = p.init != nullptr ? conv_start<T, W>(p, n, ch) : make_float4(0, 0, 0, 0);
        const float f[3] = {v.x, v.y, v.z};
#pragma unroll
        for (int k = 0; k < W - 1; ++k) h[k] = f[k];
    }
};

// The sequence [s, e) of a row that holds a token; n outside [0, units): none.
struct ConvSpan {
    int n, s, e;
    __device__ __forceinline__ void find(const SeqArgs &q, int t, int dense) {
        if (q.cu == nullptr) {
            n = dense, s = 0, e = q.seqlen;
            return;
        }
        n = conv_first_from(q, t + 1) - 1;  // the last one that starts at or before t
        s = n >= 0 ? seq_start(q, n) : 0;
        e = n >= 0 ? seq_end(q, n, s) : 0;
    }
    __device__ __forceinline__ bool holds(int t) const { return n >= 0 && t >= s && t < e; }
};

// The W - 1 inputs before token t of sequence q, from the state where they lie before it.
template <typename T, int W>
__device__ __forceinline__ void conv_history(const ConvRow<T, W> &r, const ConvSpan &q, int t, float (&h)[W - 1]) {
    if (!q.holds(t)) return;
    float st[W - 1];
    if (t - q.s < W - 1) r.start_of(q.n, st);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
        const int at = t - (W - 1) + k;
        if (at >= q.s) {
            h[k] = to_f32<T>(r.x[at]);
        } else {
#pragma unroll
            for (int i = 0; i < W - 1; ++i)
                if (W - 1 + at - q.s == i) h[k] = st[i];
        }
    }
}

// Elements [f, end) of the flat x, token by token from (row, batch, ch, c).
template <typename T, int W>
__device__ __noinline__ void conv_any(const ConvArgs &p, long long f, long long end, long long row, long long batch,
                                      unsigned ch, unsigned c) {
    const unsigned L = p.seq.seqlen;
    while (f < end) {
        const int count = static_cast<int>(min(end - f, static_cast<long long>(L - c)));
        const ConvRow<T, W> r(p, row, batch, ch);
        ConvSpan q;
        q.find(p.seq, static_cast<int>(c), r.n0);
        float h[W - 1];
        conv_history<T, W>(r, q, static_cast<int>(c), h);
        for (int t = static_cast<int>(c); t < static_cast<int>(c) + count; ++t) {
            if (t >= q.e) {
                q.find(p.seq, t, r.n0);
                conv_history<T, W>(r, q, t, h);
            }
            if (!q.holds(t)) continue;
            const float in = to_f32<T>(r.x[t]);
            float y = r.b;
#pragma unroll
            for (int k = 0; k < W - 1; ++k) y = fmaf(r.w[k], h[k], y);
            r.out[t] = from_f32<T>(conv_act(fmaf(r.w[W - 1], in, y), p.silu));
#pragma unroll
            for (int k = 0; k + 2 < W; ++k) h[k] = h[k + 1];
            h[W - 2] = in;
        }
        f += count;
        ++row;
        c = 0;
        if (++ch == static_cast<unsigned>(p.dim) && p.seq.cu == nullptr) {
            ch = 0;
            ++batch;
        }
    }
}

// x as a flat [rows * seqlen] array, row = batch * dim + channel (or the channel,
// packed). A warp takes an item of kRuns runs of 32 words, loaded together; a lane
// takes the W - 1 inputs before its word from its neighbour lane. Items inside one
// sequence do nothing else; in the others every lane looks up its word's row and
// sequences, and a word that crosses into another row or sequence masks its taps.
// Words that are not whole, the word behind a cut first one, and rows shorter than
// a word, go token by token.
// `skew`: elements between x's address and the 16-byte boundary below; words are
// counted from there. States are only read here; conv_final_kernel stores them.
template <typename T, int W, int kRuns>
__global__ void __launch_bounds__(kConvThreads) conv_channels_kernel(const ConvArgs p, long long total, int skew,
                                                                       bool vec, long long items) {
    constexpr int V = kWord<T>;
    constexpr int kRun = 32 * V;
    const SeqArgs &q = p.seq;
    const int lane = threadIdx.x & 31;
    const unsigned L = q.seqlen;
    const bool packed = q.cu != nullptr;
    const T *const x = static_cast<const T *>(p.x);
    for (long long item = static_cast<long long>(blockIdx.x) * (kConvThreads / 32) + (threadIdx.x >> 5); item < items;
         item += static_cast<long long>(gridDim.x) * (kConvThreads / 32)) {
        const long long f_item = item * (kRun * kRuns) - skew;  // the item's first element
        uint4 raw[kRuns], before = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < kRuns; ++m) {
            const long long f0 = f_item + m * kRun + lane * V;
            raw[m] = make_uint4(0, 0, 0, 0);
            if (vec && f0 >= 0 && f0 + V <= total) raw[m] = __ldg(reinterpret_cast<const uint4 *>(x + f0));
        }
        if (vec && lane == 0 && f_item >= V && f_item <= total)
            before = __ldg(reinterpret_cast<const uint4 *>(x + f_item - V));
        // Row, channel and token of the item's first element; its words add a 32-bit offset to them.
        const long long base0 = max(f_item, 0LL);
        const bool small = total <= 0xffffffffLL;
        const long long row_0 = small ? static_cast<unsigned>(base0) / L : base0 / L;
        const long long batch_0 =
            packed ? 0 : small ? static_cast<unsigned>(row_0) / static_cast<unsigned>(p.dim) : row_0 / p.dim;
        const unsigned c_0 = static_cast<unsigned>(base0 - row_0 * L);
        const unsigned ch_0 = static_cast<unsigned>(row_0 - batch_0 * p.dim);
        float tail[W - 1];  // lane 0: the inputs before the run's first word
        {
            float v[V];
            word_floats<T>(before, v);
#pragma unroll
            for (int k = 0; k < W - 1; ++k) tail[k] = v[V - (W - 1) + k];
        }
        // A run's inputs: the lane's own and the W - 1 before them.
        auto run_inputs = [&](const uint4 &word, float (&v)[V + W - 1]) {
            float own[V];
            word_floats<T>(word, own);
#pragma unroll
            for (int i = 0; i < V; ++i) v[W - 1 + i] = own[i];
#pragma unroll
            for (int k = 0; k < W - 1; ++k) {
                const float r = __shfl_sync(kFullMask, own[V - (W - 1) + k], (lane + 31) & 31);
                v[k] = lane == 0 ? tail[k] : r;
                tail[k] = r;  // lane 0: lane 31's, which the next run's first word follows
            }
        };
        auto word_values = [&](const ConvRow<T, W> &r, const float (&v)[V + W - 1], float (&y)[V]) {
            float in[W][V], ww[W][V], bb[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                bb[i] = r.b;
#pragma unroll
                for (int k = 0; k < W; ++k) {
                    in[k][i] = v[i + k];
                    ww[k][i] = r.w[k];
                }
            }
            conv_values<V, W>(y, bb, ww, in, p.silu);
        };
        if (vec && f_item >= 0 && f_item + kRuns * kRun <= total && static_cast<uint64_t>(c_0) + kRuns * kRun <= L) {
            const ConvRow<T, W> r(p, row_0, batch_0, ch_0);
            const int t0 = static_cast<int>(c_0);
            ConvSpan span;
            span.find(q, t0, r.n0);
            if (span.holds(t0) && t0 + kRuns * kRun <= span.e && (t0 == span.s || t0 - span.s >= W - 1)) {
#pragma unroll
                for (int m = 0; m < kRuns; ++m) {
                    float v[V + W - 1], y[V];
                    run_inputs(raw[m], v);
                    if (m == 0 && t0 == span.s && lane == 0) {
                        float h[W - 1];
                        r.start_of(span.n, h);
#pragma unroll
                        for (int k = 0; k < W - 1; ++k) v[k] = h[k];
                    }
                    word_values(r, v, y);
                    *reinterpret_cast<uint4 *>(r.out + t0 + m * kRun + lane * V) = floats_word<T>(y);
                }
                continue;
            }
        }
        // word by word (not unrolled: this code would crowd the instruction cache)
        ConvRow<T, W> r(p, row_0, batch_0, ch_0);
        ConvSpan span{-1, 0, 0};
        long long row_held = row_0;
#pragma unroll 1
        for (int m = 0; m < kRuns; ++m) {
            uint4 word = raw[0];
#pragma unroll
            for (int i = 1; i < kRuns; ++i)
                if (m == i) word = raw[i];
            float v[V + W - 1], y[V];
            run_inputs(word, v);
            const long long f0 = f_item + m * kRun + lane * V;
            const long long lo = max(f0, 0LL), hi = min(f0 + V, total);
            if (lo < hi) {
                unsigned c = c_0 + static_cast<unsigned>(lo - base0), ch = ch_0;
                long long row = row_0, batch = batch_0;
                if (c >= L) {
                    const unsigned rows = c / L;
                    c -= rows * L;
                    row += rows;
                    ch += rows;
                    if (!packed && ch >= static_cast<unsigned>(p.dim)) {
                        const unsigned more = ch / static_cast<unsigned>(p.dim);
                        batch += more;
                        ch -= more * static_cast<unsigned>(p.dim);
                    }
                }
                // (0 < f0 < V: the word before is cut by x's begin, so the neighbour lane holds no inputs for this one)
                if (!vec || lo != f0 || hi != f0 + V || L < V || (f0 > 0 && f0 < V)) {
                    conv_any<T, W>(p, lo, hi, row, batch, ch, c);
                } else {
                    if (row != row_held) {
                        r.take(row, batch, ch);
                        row_held = row;
                        span.e = 0;
                    }
                    const int t0 = static_cast<int>(c);
                    if (!span.holds(t0)) span.find(q, t0, r.n0);
                    if (span.holds(t0) && t0 + V <= span.e && t0 - span.s >= W - 1) {
                        word_values(r, v, y);
                        *reinterpret_cast<uint4 *>(r.out + t0) = floats_word<T>(y);
                    } else {
                        // At most two rows: token by token in registers, the window taken from the state at
                        // each sequence's start.
                        const int here = static_cast<int>(min(static_cast<unsigned>(V), L - c));
                        T *const to = static_cast<T *>(p.out) + f0;
                        unsigned held = 0;
                        float h[W - 1];
#pragma unroll
                        for (int k = 0; k < W - 1; ++k) h[k] = v[k];
                        const int into = t0 - span.s;  // tokens of the sequence before the word
                        if (span.holds(t0) && into > 0 && into < W - 1) {
                            float st[W - 1];
                            r.start_of(span.n, st);
#pragma unroll
                            for (int k = 0; k < W - 1; ++k)
#pragma unroll
                                for (int i = 0; i < W - 1; ++i)
                                    if (k + into < W - 1 && k + into == i) h[k] = st[i];
                        }
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            if (i == here) {
                                const bool wraps = !packed && ch + 1 == static_cast<unsigned>(p.dim);
                                r.take(row + 1, wraps ? batch + 1 : batch, wraps ? 0 : ch + 1);
                                row_held = row + 1;
                                span.e = 0;
                            }
                            const int t = i >= here ? i - here : t0 + i;
                            if (t >= span.e) span.find(q, t, r.n0);
                            if (t == span.s && span.n >= 0) r.start_of(span.n, h);
                            float a = r.b;
#pragma unroll
                            for (int k = 0; k < W - 1; ++k) a = fmaf(r.w[k], h[k], a);
                            a = fmaf(r.w[W - 1], v[W - 1 + i], a);
#pragma unroll
                            for (int k = 0; k + 2 < W; ++k) h[k] = h[k + 1];
                            h[W - 2] = v[W - 1 + i];
                            y[i] = conv_act(a, p.silu);
                            held |= span.holds(t) ? 1u << i : 0u;
                        }
                        if (held == (1u << V) - 1) {
                            *reinterpret_cast<uint4 *>(to) = floats_word<T>(y);
                        } else {
#pragma unroll
                            for (int i = 0; i < V; ++i)
                                if (held >> i & 1) to[i] = from_f32<T>(y[i]);
                        }
                    }
                }
            }
            __syncwarp();
        }
    }
}

// The final states behind conv_channels_kernel: a thread per (sequence, channel).
// (A launch of its own: the state rows may be the ones that other words' first
// tokens still read.)
template <typename T, int W>
__global__ void __launch_bounds__(kConvThreads) conv_final_kernel(const ConvArgs p) {
    const SeqArgs &q = p.seq;
    const long long count = static_cast<long long>(q.units) * p.dim;
    for (long long i = static_cast<long long>(blockIdx.x) * kConvThreads + threadIdx.x; i < count;
         i += static_cast<long long>(gridDim.x) * kConvThreads) {
        const int n = static_cast<int>(i / p.dim), d = static_cast<int>(i - static_cast<long long>(n) * p.dim);
        const long long row = seq_row(q, n);
        if (row < 0) continue;
        const bool live = p.init != nullptr && seq_live(q, n, row);
        const int first = q.cu != nullptr ? 0 : n * q.seqlen;
        const int s = seq_start(q, n) - first, e = seq_end(q, n, s + first) - first;
        const T *const x =
            static_cast<const T *>(p.x) + (static_cast<long long>(q.cu != nullptr ? 0 : n) * p.dim + d) * q.seqlen;
        const size_t at0 = (static_cast<size_t>(row) * p.dim + d) * (W - 1);
        T keep[W - 1];
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
            const int at = e - (W - 1) + k;
            if (at >= s) keep[k] = x[at];
            else keep[k] = live ? static_cast<const T *>(p.init)[at0 + (W - 1) + at - s] : from_f32<T>(0.0f);
        }
#pragma unroll
        for (int k = 0; k < W - 1; ++k) static_cast<T *>(p.final_state)[at0 + k] = keep[k];
    }
}

// ------------------------------------------------------------------ one token

// Thread: V channels, kRows sequences (loads issued together; the weights are
// read once for all).
template <typename T, int V, int W, int kRows>
__global__ void __launch_bounds__(kConvThreads) conv_token_kernel(const ConvArgs p, bool words) {
    constexpr int S = V * (W - 1);  // state elements of the thread's channels in a row
    const int d = (blockIdx.x * kConvThreads + threadIdx.x) * V;
    if (d >= p.dim) return;
    const size_t D = p.dim;
    // (sequences are counted in 31 bits, the steps past the last one need the 32nd)
    const unsigned units = p.seq.units;
    for (unsigned n0 = blockIdx.y * kRows; n0 < units; n0 += gridDim.y * kRows) {
        long long row[kRows];
        Elems<T, V> x[kRows], s[kRows][W - 1];
#pragma unroll
        for (int r = 0; r < kRows; ++r) row[r] = n0 + r < units ? seq_row(p.seq, n0 + r) : -1;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            if (row[r] < 0) continue;
            x[r].load(static_cast<const T *>(p.x) + (static_cast<size_t>(n0) + r) * D + d);
            const T *from = static_cast<const T *>(p.init) + (static_cast<size_t>(row[r]) * D + d) * (W - 1);
#pragma unroll
            for (int k = 0; k < W - 1; ++k) s[r][k].load(from + k * V);
        }
        float w[W][V], b[V];
        conv_load_weights<V, W>(p, d, words, w, b);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            if (row[r] < 0) continue;
            float xv[V], old[S], y[V];
            x[r].floats(xv);
#pragma unroll
            for (int k = 0; k < W - 1; ++k) {
                float part[V];
                s[r][k].floats(part);
#pragma unroll
                for (int i = 0; i < V; ++i) old[k * V + i] = part[i];
            }
            float now[S];  // the state, x shifted in (exact: the values round back to what they were)
            float win[W][V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
#pragma unroll
                for (int k = 0; k < W - 1; ++k) {
                    win[k][i] = old[i * (W - 1) + k];
                    now[i * (W - 1) + k] = k + 1 < W - 1 ? old[i * (W - 1) + k + 1] : xv[i];
                }
                win[W - 1][i] = xv[i];
            }
            conv_values<V, W>(y, b, w, win, p.silu);
            T *to = static_cast<T *>(p.final_state) + (static_cast<size_t>(row[r]) * D + d) * (W - 1);
#pragma unroll
            for (int k = 0; k < W - 1; ++k) {
                float part[V];
#pragma unroll
                for (int i = 0; i < V; ++i) part[i] = now[k * V + i];
                store_elems<T, V>(to + k * V, part);
            }
            store_elems<T, V>(static_cast<T *>(p.out) + (static_cast<size_t>(n0) + r) * D + d, y);
        }
    }
}

// ------------------------------------------------------------------ launches

template <typename F>
cudaError_t by_type(IoType io, F &&f) {
    switch (io) {
        case IoType::kBF16: return f(__nv_bfloat16{});
        case IoType::kF16: return f(__half{});
        default: return f(float{});
    }
}

template <typename T, int V, int W>
cudaError_t launch_tokens(const ConvArgs &a, cudaStream_t stream) {
    const int64_t groups = (static_cast<int64_t>(a.dim) + V * kConvThreads - 1) / (V * kConvThreads);
    // Six CTAs are resident per SM. Blocks of about 128 tokens, sized so that the grid is whole waves of
    // them (with four resident, 16384 tokens x 4096 channels took 62 us in blocks of 64, 1.7 waves, and 57 us
    // so); 4 tokens at least.
    const int64_t resident = 6LL * current_device_sm_count(), tokens = a.seq.tokens;
    const int64_t waves = std::max<int64_t>(1, (tokens * groups + 64 * resident) / (128 * resident));
    const int64_t want = std::max<int64_t>(1, resident * waves / groups);
    const int block = static_cast<int>(std::max<int64_t>(4, ((tokens + want - 1) / want + 3) / 4 * 4));
    const int nblocks = static_cast<int>(std::max<int64_t>(1, (tokens + block - 1) / block));
    const dim3 grid(static_cast<unsigned>(groups), static_cast<unsigned>(std::min(nblocks, 65535)));
    conv_tokens_kernel<T, V, W><<<grid, kConvThreads, 0, stream>>>(a, block, nblocks, aligned16(a.weight) && aligned16(a.bias));
    return cudaGetLastError();
}

template <typename T, int W>
cudaError_t launch_channels(const ConvArgs &a, cudaStream_t stream) {
    constexpr int V = kWord<T>;
    const long long total =
        (a.seq.cu != nullptr ? 1LL : static_cast<long long>(a.seq.units)) * a.dim * static_cast<long long>(a.seq.seqlen);
    const auto at = [](const void *p) { return static_cast<int>(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T)); };
    const int skew = at(a.x);
    auto launch = [&](auto kernel, int runs) {
        const long long words = (total + skew + V - 1) / V, items = (words + 32 * runs - 1) / (32 * runs);
        const long long blocks = (items + kConvThreads / 32 - 1) / (kConvThreads / 32);
        kernel<<<static_cast<unsigned>(std::min(blocks, 1LL << 30)), kConvThreads, 0, stream>>>(a, total, skew,
                                                                                              at(a.out) == skew, items);
        return cudaGetLastError();
    };
    // Runs per item share its arithmetic and cover latency, but an item that straddles rows or sequences goes word
    // by word. Eight runs where none does (rows of whole items) or few do (rows, or sequences on average, of eight
    // items or more), else four. Microseconds per 2^26 elements in bfloat16 (items of 2048), four and eight: rows of
    // 2048 tokens 76 and 58, of 4096 76 and 58, of 2000 129 and 134, 2500 129 and 142, 5000 110 and 125, 8200 96 and
    // 106, 16400 88 and 85, 24000 83 and 77; rows of 2048 off a 16-byte boundary 129 and 135; packed sequences of
    // 800 on average 253 and 275, 8192 114 and 116, 16384 101 and 95, 32768 92 and 78. float32 (items of 1024) turns
    // between 4100 (158 and 168) and 8196 (146 and 134).
    const int64_t item = 8 * 32 * V;
    const int64_t length = a.seq.cu != nullptr ? a.seq.tokens / a.seq.units : a.seq.seqlen;
    const bool whole = a.seq.cu == nullptr && skew == 0 && length % item == 0;
    const cudaError_t e = whole || length >= 8 * item ? launch(conv_channels_kernel<T, W, 8>, 8)
                                                      : launch(conv_channels_kernel<T, W, 4>, 4);
    if (e != cudaSuccess || a.final_state == nullptr) return e;
    const long long blocks = (static_cast<long long>(a.seq.units) * a.dim + kConvThreads - 1) / kConvThreads;
    conv_final_kernel<T, W><<<static_cast<unsigned>(std::min(blocks, 1LL << 20)), kConvThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

// The states of sequences without tokens, and of empty rows, in any layout: tokens
// [0, 0) with the tokens-first kernel touch nothing but states.
template <typename T, int W>
cudaError_t launch_width(const ConvArgs &a, cudaStream_t stream) {
    constexpr int V = kWord<T> / 2;
    auto on8 = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 8 == 0; };
    const bool vec = a.dim % V == 0 && on8(a.x) && on8(a.out);
    if (a.channels_last || a.seq.tokens == 0)
        return vec ? launch_tokens<T, V, W>(a, stream) : launch_tokens<T, 1, W>(a, stream);
    return launch_channels<T, W>(a, stream);
}

template <typename T, int V, int W>
cudaError_t launch_token(const ConvArgs &a, cudaStream_t stream) {
    const int64_t blocks = (static_cast<int64_t>(a.dim) + V * kConvThreads - 1) / (V * kConvThreads);
    const int64_t groups = (static_cast<int64_t>(a.seq.units) + 3) / 4;
    const unsigned gx = static_cast<unsigned>(blocks);
    const bool words = aligned16(a.weight) && aligned16(a.bias);
    // Four sequences per thread where that leaves each SM four blocks; below, one, and half words, which
    // need half the registers and give twice the threads (256 sequences x 4096 channels: 5.6 us against 9.6).
    if (blocks * groups >= 4LL * current_device_sm_count()) {
        conv_token_kernel<T, V, W, 4>
            <<<dim3(gx, static_cast<unsigned>(std::min<int64_t>(groups, 65535))), kConvThreads, 0, stream>>>(a, words);
    } else {
        constexpr int H = V > 1 ? V / 2 : 1;
        const unsigned hx = static_cast<unsigned>((static_cast<int64_t>(a.dim) + H * kConvThreads - 1) / (H * kConvThreads));
        conv_token_kernel<T, H, W, 1>
            <<<dim3(hx, static_cast<unsigned>(std::min(a.seq.units, 65535))), kConvThreads, 0, stream>>>(a, words);
    }
    return cudaGetLastError();
}

template <typename T, int W>
cudaError_t launch_token_width(const ConvArgs &a, cudaStream_t stream) {
    constexpr int V = kWord<T>;
    const bool vec = a.dim % V == 0 && aligned16(a.x) && aligned16(a.out) && aligned16(a.init) &&
                     aligned16(a.final_state);
    return vec ? launch_token<T, V, W>(a, stream) : launch_token<T, 1, W>(a, stream);
}

}  // namespace

cudaError_t launch_causal_conv1d(const ConvArgs &a, cudaStream_t stream) {
    return by_type(a.io, [&](auto t) {
        using T = decltype(t);
        if (a.width == 2) return launch_width<T, 2>(a, stream);
        return a.width == 3 ? launch_width<T, 3>(a, stream) : launch_width<T, 4>(a, stream);
    });
}

cudaError_t launch_causal_conv1d_update(const ConvArgs &a, cudaStream_t stream) {
    return by_type(a.io, [&](auto t) {
        using T = decltype(t);
        if (a.width == 2) return launch_token_width<T, 2>(a, stream);
        return a.width == 3 ? launch_token_width<T, 3>(a, stream) : launch_token_width<T, 4>(a, stream);
    });
}

}  // namespace xm
