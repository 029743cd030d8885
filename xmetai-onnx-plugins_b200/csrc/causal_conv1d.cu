// causal_conv1d.cu -- CausalConv1dFn and CausalConv1dUpdateFn for sm_100a.
//
// Math, per channel d: y_t = act(bias + sum_{k < W} w_k x_(t - (W - 1) + k)),
// act = identity or v sigmoid(v); x before the sequence's first token comes from
// its state, the last W - 1 inputs of the tokens that went before.
//
// Bound by memory: x is read and y written once, against 2 W + 4 operations per
// element, so each layout's kernel moves 16-byte words and keeps enough of them
// in flight:
//   conv_tokens_kernel    [tokens, dim]: a thread owns the channels of one word
//                         and walks a block of tokens, the window in registers;
//   conv_channels_kernel  [dim, tokens]: a thread owns a word of consecutive
//                         tokens and takes the W - 1 before it from its
//                         neighbour lane;
//   conv_token_kernel     one token per sequence: a thread owns the channels of
//                         one word, their state and their weights.
//
// Where sequences are cut, over blocks of tokens or words, one thread does all
// that touches a sequence's state of a channel: the one at the sequence's first
// token. It computes the first W - 1 tokens, which alone see the starting state,
// even where they reach into the next block or word, and then stores the final
// state. So in-place states are safe and need no second launch.
#include <algorithm>
#include <climits>

#include "xm_common.cuh"
#include "xm_kernels.h"
#include "xm_sequences.cuh"

namespace xm {
namespace {

constexpr int kConvThreads = 128;

__device__ __forceinline__ float conv_act(float v, bool silu) {
    return silu ? v * rcp_approx(1.0f + ex2_approx(-v * kLog2e)) : v;
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

// V elements from p: one word when V is the word's, else a single element.
template <typename T, int V>
struct Elems {
    uint4 r;
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (V == 1) {
            if constexpr (sizeof(T) == 4) r.x = __float_as_uint(*p);
            else r.x = *reinterpret_cast<const unsigned short *>(p);
        } else {
            r = *reinterpret_cast<const uint4 *>(p);
        }
    }
    __device__ __forceinline__ void floats(float (&v)[V]) const {
        if constexpr (V == 1) {
            if constexpr (sizeof(T) == 4) v[0] = __uint_as_float(r.x);
            else v[0] = unpack2<T>(r.x).x;
        } else {
            word_floats<T>(r, v);
        }
    }
};

template <typename T, int V>
__device__ __forceinline__ void store_elems(T *p, const float (&v)[V]) {
    if constexpr (V == 1) *p = from_f32<T>(v[0]);
    else *reinterpret_cast<uint4 *>(p) = floats_word<T>(v);
}

// First sequence that starts at or behind t (units: none).
__device__ __forceinline__ int conv_first_from(const SeqArgs &q, int t) {
    if (q.cu == nullptr) return q.seqlen > 0 ? static_cast<int>((static_cast<long long>(t) + q.seqlen - 1) / q.seqlen) : 0;
    int lo = 0, hi = q.units;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (seq_start(q, mid) >= t) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// ------------------------------------------------------------------ tokens first

constexpr int kAheadTokens = 4;  // tokens whose loads are issued together

// Thread: V channels from channel V * (blockIdx.x * threads + thread); blockIdx.y:
// the block of `block` tokens. Each thread walks the sequences that meet it.
template <typename T, int V, int W>
__global__ void __launch_bounds__(kConvThreads) conv_tokens_kernel(const ConvArgs p, int block, int nblocks) {
    const SeqArgs &q = p.seq;
    const int d = (blockIdx.x * kConvThreads + threadIdx.x) * V;
    if (d >= p.dim) return;
    const size_t D = p.dim;
    const T *const x = static_cast<const T *>(p.x) + d;
    T *const out = static_cast<T *>(p.out) + d;
    float w[W][V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int k = 0; k < W; ++k) w[k][i] = p.weight[static_cast<size_t>(d + i) * W + k];
        b[i] = p.bias != nullptr ? p.bias[d + i] : 0.0f;
    }
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
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    y[i] = b[i];
#pragma unroll
                    for (int k = 0; k < W; ++k) y[i] = fmaf(w[k][i], win[k][i], y[i]);
                    y[i] = conv_act(y[i], p.silu);
                }
                store_elems<T, V>(out + static_cast<size_t>(t) * D, y);
            };
            int t = from;
            if (t + kAheadTokens <= to) {
                Elems<T, V> cur[kAheadTokens], nxt[kAheadTokens];
#pragma unroll
                for (int i = 0; i < kAheadTokens; ++i) cur[i].load(x + static_cast<size_t>(t + i) * D);
                for (; t + kAheadTokens <= to; t += kAheadTokens) {
                    const bool more = t + 2 * kAheadTokens <= to;
#pragma unroll
                    for (int i = 0; i < kAheadTokens; ++i)
                        if (more) nxt[i].load(x + static_cast<size_t>(t + kAheadTokens + i) * D);
#pragma unroll
                    for (int i = 0; i < kAheadTokens; ++i) step(t + i, cur[i]);
#pragma unroll
                    for (int i = 0; i < kAheadTokens; ++i) cur[i] = nxt[i];
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

constexpr int kWordsPerThread = 4;  // words whose loads are issued together

// x as a flat [rows * seqlen] array, row = batch * dim + channel (or the channel,
// packed). A warp takes kWordsPerThread runs of 32 words. `skew`: elements between
// x's address and the 16-byte boundary below; words are counted from there.
template <typename T, int W>
__global__ void __launch_bounds__(kConvThreads) conv_channels_kernel(const ConvArgs p, long long total, int skew,
                                                                       bool vec, long long items) {
    constexpr int V = kWord<T>;
    const SeqArgs &q = p.seq;
    const int lane = threadIdx.x & 31, L = q.seqlen;
    const T *const x = static_cast<const T *>(p.x);
    T *const out = static_cast<T *>(p.out);
    for (long long item = static_cast<long long>(blockIdx.x) * (kConvThreads / 32) + (threadIdx.x >> 5); item < items;
         item += static_cast<long long>(gridDim.x) * (kConvThreads / 32)) {
        const long long base = item * (32 * kWordsPerThread);  // the run's first word
        // Row, channel and token of the run's first element; its words add a 32-bit offset to them.
        const long long base0 = max(base * V - skew, 0LL);
        const long long row_0 = base0 / L, batch_0 = q.cu != nullptr ? 0 : row_0 / p.dim;
        const unsigned c_0 = static_cast<unsigned>(base0 - row_0 * L);
        const unsigned ch_0 = static_cast<unsigned>(row_0 - batch_0 * p.dim);
        uint4 raw[kWordsPerThread];
#pragma unroll
        for (int m = 0; m < kWordsPerThread; ++m) {
            const long long f0 = (base + 32 * m + lane) * V - skew;
            raw[m] = make_uint4(0, 0, 0, 0);
            if (vec && f0 >= 0 && f0 + V <= total) {
                raw[m] = __ldg(reinterpret_cast<const uint4 *>(x + f0));
            } else if (f0 < total && f0 + V > 0) {
                uint32_t e[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    e[i] = 0u;
                    if (f0 + i >= 0 && f0 + i < total) {
                        if constexpr (sizeof(T) == 4) e[i] = __float_as_uint(x[f0 + i]);
                        else e[i] = reinterpret_cast<const unsigned short *>(x)[f0 + i];
                    }
                }
                if constexpr (sizeof(T) == 4) raw[m] = make_uint4(e[0], e[1], e[2], e[3]);
                else raw[m] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
            }
        }
#pragma unroll
        for (int m = 0; m < kWordsPerThread; ++m) {
            const long long f0 = (base + 32 * m + lane) * V - skew;
            float v[V + W - 1];  // the W - 1 inputs before the word, then its own
            float own_v[V];
            word_floats<T>(raw[m], own_v);
#pragma unroll
            for (int i = 0; i < V; ++i) v[W - 1 + i] = own_v[i];
#pragma unroll
            for (int k = 0; k < W - 1; ++k) {
                v[k] = __shfl_up_sync(kFullMask, own_v[V - (W - 1) + k], 1);
                if (lane == 0) {
                    const long long at = f0 - (W - 1) + k;
                    v[k] = at >= 0 && at < total ? to_f32<T>(x[at]) : 0.0f;
                }
            }
            if (f0 >= total || f0 + V <= 0) continue;
            const long long lo = max(f0, 0LL), hi = min(f0 + V, total);
            unsigned c = c_0 + static_cast<unsigned>(lo - base0), ch = ch_0;
            long long r = row_0, batch = batch_0;
            if (c >= static_cast<unsigned>(L)) {
                const unsigned rows = c / static_cast<unsigned>(L);
                c -= rows * static_cast<unsigned>(L);
                r += rows;
                ch += rows;
                if (q.cu == nullptr && ch >= static_cast<unsigned>(p.dim)) {
                    const unsigned more = ch / static_cast<unsigned>(p.dim);
                    batch += more;
                    ch -= more * static_cast<unsigned>(p.dim);
                }
            }
            // Row by row (one, unless rows are shorter than a word).
            for (long long f = lo; f < hi;) {
                const int count = static_cast<int>(min(hi - f, static_cast<long long>(L) - c));  // its tokens here
                const int tb = static_cast<int>(batch) * L;  // number of the row's first token (0 where packed)
                const T *const xr = x + r * L;
                T *const yr = out + r * L;
                float w[W];
#pragma unroll
                for (int k = 0; k < W; ++k) w[k] = __ldg(p.weight + static_cast<size_t>(ch) * W + k);
                const float b = p.bias != nullptr ? __ldg(p.bias + ch) : 0.0f;
                const int t0 = static_cast<int>(c), t1 = t0 + count;
                // sequences of the row: dense rows have one, the batch's
                int n = q.cu != nullptr ? conv_first_from(q, t0) : static_cast<int>(batch);
                const int n_end = q.cu != nullptr ? q.units : n + 1;
                if (q.cu != nullptr && n > 0) --n;
                auto begin = [&](int i) { return seq_start(q, i) - tb; };
                auto state_of = [&](int i, bool &live) {
                    const long long row = seq_row(q, i);
                    live = p.init != nullptr && seq_live(q, i, row);
                    return row;
                };
                auto state_at = [&](long long row, int k) {
                    return static_cast<const T *>(p.init)[(static_cast<size_t>(row) * p.dim + ch) * (W - 1) + k];
                };
                auto finish = [&](int i, int s, int e, long long row, bool live) {
                    if (p.final_state == nullptr || row < 0) return;
                    T keep[W - 1];
#pragma unroll
                    for (int k = 0; k < W - 1; ++k) {
                        const int at = e - (W - 1) + k;
                        if (at >= s) keep[k] = xr[at];
                        else keep[k] = live ? state_at(row, W - 1 + at - s) : from_f32<T>(0.0f);
                    }
#pragma unroll
                    for (int k = 0; k < W - 1; ++k)
                        static_cast<T *>(p.final_state)[(static_cast<size_t>(row) * p.dim + ch) * (W - 1) + k] = keep[k];
                };
                const int s0 = n < n_end ? begin(n) : INT_MAX;
                const int e0 = n < n_end ? max(s0, begin(n + 1)) : INT_MAX;
                if (vec && count == V && e0 >= t1 && s0 <= t0 && (s0 == t0 || t0 - s0 >= W - 1) &&
                    (q.cu == nullptr || (s0 < t0 && e0 > t1))) {
                    // the whole word in one sequence, all its inputs here (or its state at the row's start)
                    bool live = false;
                    long long row = -1;
                    if (s0 == t0) {
                        row = state_of(n, live);
#pragma unroll
                        for (int k = 0; k < W - 1; ++k) v[k] = live ? to_f32<T>(state_at(row, k)) : 0.0f;
                    }
                    float y[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        y[i] = b;
#pragma unroll
                        for (int k = 0; k < W; ++k) y[i] = fmaf(w[k], v[i + k], y[i]);
                        y[i] = conv_act(y[i], p.silu);
                    }
                    *reinterpret_cast<uint4 *>(yr + t0) = floats_word<T>(y);
                    if (s0 == t0) finish(n, s0, e0, row, live);
                } else {
                    // sequence by sequence and token by token
                    for (; n < n_end; ++n) {
                        const int s = begin(n);
                        if (s >= t1 && t1 < L) break;
                        const int e = max(s, begin(n + 1));
                        const bool own = s >= t0;  // this word holds the sequence's first token
                        if (own && s >= t1 && s < L) break;
                        if (s < 0) continue;
                        const int from = own ? s : max(t0, min(e, s + W - 1));
                        const int to = own ? max(min(e, t1), min(e, s + W - 1)) : min(e, t1);
                        bool live = false;
                        const long long row = own ? state_of(n, live) : -1;
                        for (int t = from; t < to; ++t) {
                            float y = b;
#pragma unroll
                            for (int k = 0; k < W; ++k) {
                                const int at = t - (W - 1) + k;
                                const float in = at >= s ? to_f32<T>(xr[at])
                                                         : live ? to_f32<T>(state_at(row, W - 1 + at - s)) : 0.0f;
                                y = fmaf(w[k], in, y);
                            }
                            yr[t] = from_f32<T>(conv_act(y, p.silu));
                        }
                        if (own) finish(n, s, e, row, live);
                    }
                }
                f += count;
                ++r;
                c = 0;
                if (++ch == static_cast<unsigned>(p.dim) && q.cu == nullptr) {
                    ch = 0;
                    ++batch;
                }
            }
        }
    }
}

// ------------------------------------------------------------------ one token

// Thread: V channels, kRows sequences (loads issued together; the weights are
// read once for all).
template <typename T, int V, int W, int kRows>
__global__ void __launch_bounds__(kConvThreads) conv_token_kernel(const ConvArgs p) {
    constexpr int S = V * (W - 1);  // state elements of the thread's channels in a row
    const int d = (blockIdx.x * kConvThreads + threadIdx.x) * V;
    if (d >= p.dim) return;
    const size_t D = p.dim;
    for (int n0 = blockIdx.y * kRows; n0 < p.seq.units; n0 += gridDim.y * kRows) {
        long long row[kRows];
        Elems<T, V> x[kRows], s[kRows][W - 1];
#pragma unroll
        for (int r = 0; r < kRows; ++r) row[r] = n0 + r < p.seq.units ? seq_row(p.seq, n0 + r) : -1;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            if (row[r] < 0) continue;
            x[r].load(static_cast<const T *>(p.x) + (static_cast<size_t>(n0) + r) * D + d);
            const T *from = static_cast<const T *>(p.init) + (static_cast<size_t>(row[r]) * D + d) * (W - 1);
#pragma unroll
            for (int k = 0; k < W - 1; ++k) s[r][k].load(from + k * V);
        }
        float w[V][W], b[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
            for (int k = 0; k < W; ++k) w[i][k] = __ldg(p.weight + static_cast<size_t>(d + i) * W + k);
            b[i] = p.bias != nullptr ? __ldg(p.bias + d + i) : 0.0f;
        }
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
#pragma unroll
            for (int i = 0; i < V; ++i) {
                y[i] = b[i];
#pragma unroll
                for (int k = 0; k < W - 1; ++k) {
                    y[i] = fmaf(w[i][k], old[i * (W - 1) + k], y[i]);
                    now[i * (W - 1) + k] = k + 1 < W - 1 ? old[i * (W - 1) + k + 1] : xv[i];
                }
                y[i] = conv_act(fmaf(w[i][W - 1], xv[i], y[i]), p.silu);
            }
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
    // Blocks of 32 tokens, shorter while that leaves SMs without blocks.
    const int64_t sms = current_device_sm_count();
    int block = 32;
    while (block > 4 && groups * ((a.seq.tokens + block - 1) / block) < 4 * sms) block /= 2;
    const int nblocks = std::max(1, static_cast<int>((static_cast<int64_t>(a.seq.tokens) + block - 1) / block));
    const dim3 grid(static_cast<unsigned>(groups), static_cast<unsigned>(std::min(nblocks, 65535)));
    conv_tokens_kernel<T, V, W><<<grid, kConvThreads, 0, stream>>>(a, block, nblocks);
    return cudaGetLastError();
}

template <typename T, int W>
cudaError_t launch_channels(const ConvArgs &a, cudaStream_t stream) {
    constexpr int V = kWord<T>;
    const long long total =
        (a.seq.cu != nullptr ? 1LL : static_cast<long long>(a.seq.units)) * a.dim * static_cast<long long>(a.seq.seqlen);
    const auto at = [](const void *p) { return static_cast<int>(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T)); };
    const int skew = at(a.x);
    const long long words = (total + skew + V - 1) / V, items = (words + 32 * kWordsPerThread - 1) / (32 * kWordsPerThread);
    const long long blocks = (items + kConvThreads / 32 - 1) / (kConvThreads / 32);
    conv_channels_kernel<T, W><<<static_cast<unsigned>(std::min(blocks, 1LL << 30)), kConvThreads, 0, stream>>>(
        a, total, skew, at(a.out) == skew, items);
    return cudaGetLastError();
}

// The states of sequences without tokens, and of empty rows, in any layout: tokens
// [0, 0) with the tokens-first kernel touch nothing but states.
template <typename T, int W>
cudaError_t launch_width(const ConvArgs &a, cudaStream_t stream) {
    constexpr int V = kWord<T>;
    const bool vec = a.dim % V == 0 && aligned16(a.x) && aligned16(a.out);
    if (a.channels_last || a.seq.tokens == 0)
        return vec ? launch_tokens<T, V, W>(a, stream) : launch_tokens<T, 1, W>(a, stream);
    return launch_channels<T, W>(a, stream);
}

template <typename T, int V, int W>
cudaError_t launch_token(const ConvArgs &a, cudaStream_t stream) {
    const int64_t blocks = (static_cast<int64_t>(a.dim) + V * kConvThreads - 1) / (V * kConvThreads);
    const int64_t groups = (static_cast<int64_t>(a.seq.units) + 3) / 4;
    const unsigned gx = static_cast<unsigned>(blocks);
    // Four sequences per thread where that leaves each SM four blocks.
    if (blocks * groups >= 4LL * current_device_sm_count())
        conv_token_kernel<T, V, W, 4>
            <<<dim3(gx, static_cast<unsigned>(std::min<int64_t>(groups, 65535))), kConvThreads, 0, stream>>>(a);
    else
        conv_token_kernel<T, V, W, 1>
            <<<dim3(gx, static_cast<unsigned>(std::min(a.seq.units, 65535))), kConvThreads, 0, stream>>>(a);
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
