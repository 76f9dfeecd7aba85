// ah_attn.h -- what the kernels of attention over the 4-bit cache share (ah_attn.hip, ah_blocks.hip): a sequence's tokens
// and keys.
#pragma once

#include "ah_kv4.h"
#include "ah_seqs.h"

// What a workgroup of a sequence works on.
struct Span {
    uint32_t q0, nq;      // its tokens
    int32_t ctx;          // keys
    bool bad;
};
AH_DEV Span span_of(const AttnArgs &a, uint32_t s) {
    Span p;
    const int32_t b = a.q_start[s], e = a.q_start[s + 1], c = a.ctx[s];
    const uint64_t room = (uint64_t)a.table_stride << a.c.page_shift;
    p.bad = b < 0 || e < b || (uint32_t)e > a.n_tok || (uint32_t)(e - b) > a.max_q || c < 0 || (uint64_t)c > room;
    p.q0 = p.bad ? 0 : (uint32_t)b;
    p.nq = p.bad ? 0 : (uint32_t)(e - b);
    p.ctx = p.bad ? 0 : c;
    return p;
}

template <class S, class H> AH_DEV uint32_t sequence_of(const AttnArgs &a, uint32_t at, S start, H holds) {
    return sequence_among(a.q_start, a.n_seq, a.n_tok, at, start, holds);
}
