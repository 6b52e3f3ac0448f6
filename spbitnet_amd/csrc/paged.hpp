// paged.hpp -- what the operators of a batch of new tokens over a paged key /
// value cache share: host checks of the descriptors, and the device search of a
// token's sequence.
#pragma once

#include "common.hpp"
#include "spbitnet_amd.h"

namespace spb {

inline bool aligned_to(const void* p, size_t n) {
    return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0;
}

// Host checks of a cache and of a batch; 0 or the status of invalid().
int check_paged_cache(const char* fn, const spb_paged_cache* c);
int check_paged_batch(const char* fn, const spb_paged_batch* b);

// Unsigned division of 0 <= x < 2^31 by a fixed d >= 1: floor(x / d) =
// umulhi(x, m) >> s with m = ceil(2^(32 + s) / d), 2^s < d <= 2^(s + 1).  m < 2^32
// and m d - 2^(32 + s) < d <= 2^(s + 1), so x times that excess stays below
// 2^(32 + s) for x < 2^31: exact.  d = 1 has no such m below 2^32 and is m = 0.
struct FastDiv {
    uint32_t d = 1, m = 0, s = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div) {
        if (d <= 1) return;
        while ((2u << s) < d) ++s;
        m = static_cast<uint32_t>(((uint64_t{1} << (32 + s)) + d - 1) / d);
    }
    __device__ __forceinline__ uint32_t div(uint32_t x) const {
        return m == 0 ? x : __umulhi(x, m) >> s;
    }
};

// A batch as the kernels take it.
struct BatchArgs {
    const int* starts;  // [seqs + 1]
    const int* lens;    // [seqs]
    const int* table;   // [seqs][width]
    int seqs, width, tokens, pages;
    int capacity;  // positions that a row of the table holds
    FastDiv page;
};

BatchArgs batch_args(const spb_paged_cache& c, const spb_paged_batch& b);

// A sequence's tokens [first, first + count) of the batch and its cached
// positions, whatever the arrays hold: never past the batch or the table.
struct SeqSpan {
    int first, count, len;
};

__device__ __forceinline__ SeqSpan seq_span(const BatchArgs& b, int s) {
    SeqSpan r;
    const int a = b.starts[s], e = b.starts[s + 1], n = b.lens[s];
    r.first = min(max(a, 0), b.tokens);
    r.count = max(min(max(e, 0), b.tokens) - r.first, 0);
    r.len = min(max(n, 0), b.capacity);
    return r;
}

}  // namespace spb
