// ah_seqs.h -- which sequence a token, or a workgroup's tile of tokens, belongs to.
#pragma once

#include "ah_internal.h"

// The last of n things, in the order of their starts, that starts at or before `at` (the first one if none does): the
// wave's lanes look at 64 of them at a time.
template <class F> AH_DEV uint32_t last_starting(uint32_t n, uint32_t at, F start) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = 0;
    while (n > 1) {
        const uint32_t step = (n + 63) / 64, i = lane * step;
        const uint32_t count = (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(i < n && start(lo + (i < n ? i : 0)) <= at));
        const uint32_t skip = (count ? count - 1 : 0) * step;
        lo += skip;
        n = n - skip < step ? n - skip : step;
    }
    return lo;
}

// The sequence for which holds(i) is true (any, if there is none).  Where the entries of q_start in range ascend, sequence i
// holds what lies between start(i) and start(i + 1).  One out of range leads the search astray: a find that the entries
// beside it don't confirm is looked up among all sequences.
template <class S, class H>
AH_DEV uint32_t sequence_among(const int32_t *q_start, uint32_t n_seq, uint32_t n_tok, uint32_t at, S start, H holds) {
    uint32_t s = last_starting(n_seq, at, start);
    auto in_range = [&](uint32_t i) { return (uint32_t)q_start[i] <= n_tok; };
    if (in_range(s) && in_range(s + 1) && (start(s) <= at ? s + 1 == n_seq || start(s + 1) > at : s == 0)) return s;
    for (uint32_t base = 0; base < n_seq; base += 64) {
        const uint32_t i = base + (threadIdx.x & 63);
        const uint64_t b = __builtin_amdgcn_ballot_w64(i < n_seq && holds(i < n_seq ? i : 0));
        if (b) s = base + 63 - (uint32_t)__builtin_clzll(b);
    }
    return s;
}
