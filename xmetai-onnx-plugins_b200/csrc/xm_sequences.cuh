// xm_sequences.cuh -- device view of a call's sequences and the state rows they
// own (SeqArgs), shared by the causal convolution and the selective scan.
#pragma once

#include "xm_common.cuh"
#include "xm_kernels.h"

namespace xm {

__device__ __forceinline__ long long index_at(const void *p, bool is64, int i) {
    return is64 ? __ldg(static_cast<const long long *>(p) + i) : __ldg(static_cast<const int *>(p) + i);
}

// First token of sequence i (i = units: the end of the last one). Packed offsets
// are clamped into [0, tokens].
__device__ __forceinline__ int seq_start(const SeqArgs &q, int i) {
    if (q.cu == nullptr) return i * q.seqlen;
    return static_cast<int>(min(max(index_at(q.cu, q.cu64, i), 0LL), static_cast<long long>(q.tokens)));
}

// End of sequence i that starts at `start`; offsets that descend give an empty sequence.
__device__ __forceinline__ int seq_end(const SeqArgs &q, int i, int start) { return max(start, seq_start(q, i + 1)); }

// First packed sequence that starts at or behind t (units: none).
__device__ __forceinline__ int seq_first_from(const SeqArgs &q, int t) {
    int lo = 0, hi = q.units;
    while (lo < hi) {
        const int mid = lo + ((hi - lo) >> 1);  // lo + hi would pass 31 bits
        if (seq_start(q, mid) >= t) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// State row of sequence i, or -1 where it owns none.
__device__ __forceinline__ long long seq_row(const SeqArgs &q, int i) {
    if (q.slots == nullptr) return i;
    const long long s = index_at(q.slots, q.slots64, i);
    return s >= 0 && s < q.n_rows ? s : -1;
}

// Whether sequence i, which owns `row`, starts from that row's state.
__device__ __forceinline__ bool seq_live(const SeqArgs &q, int i, long long row) {
    return row >= 0 && (q.live == nullptr || index_at(q.live, q.live64, i) != 0);
}

}  // namespace xm
