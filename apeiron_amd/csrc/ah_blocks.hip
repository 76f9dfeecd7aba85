// ah_blocks.hip -- the choice of blocks for attention over parts of a long context in the paged 4-bit cache (layout:
// ah_kv4.h): the means of the blocks' keys, and for every (token, KV head) the blocks that its queries score highest.
#include "ah_attn.h"

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr unsigned long long kKeyCache = AH_ERR_CACHE_RANGE;

// ---- means -----------------------------------------------------------------------------------------
//
// A block whose last position is among the tokens: the mean of its keys, a wave a KV head.  Lane (p, g) sums the eight
// channels of group g over every (64 / (D / 8))-th position from p on, in f64: the cache's values have eleven
// significant bits between 2^-24 and 2^16, so the sums are exact in any order, and a block's mean is the same however
// its positions came.  It is rounded to f32 and then to f16.
template <int D> __global__ void __launch_bounds__(256) block_means_kernel(MeansArgs a) {
    constexpr uint32_t G = D / 8, P = 64 / G;
    const uint32_t tok = blockIdx.x, lane = threadIdx.x & 63, g = lane % G, ph = lane / G;
    const int32_t seq = a.t.seq[tok], pos = a.t.pos[tok];
    if (seq < 0) return;
    const uint32_t len = 1u << a.shift;
    bool ok = (uint32_t)seq < a.t.n_seq && pos >= 0 && (uint32_t)pos >> a.c.page_shift < a.t.table_stride;
    const uint32_t page = ok ? (uint32_t)a.t.table[(size_t)seq * a.t.table_stride + ((uint32_t)pos >> a.c.page_shift)] : 0;
    ok = ok && page < a.c.n_pages;
    if (!ok) {
        if (threadIdx.x == 0) ah_record(a.status, ((unsigned long long)tok << 8) + kKeyCache);
        return;
    }
    if ((~(uint32_t)pos & (len - 1)) != 0) return;
    const uint32_t in = (uint32_t)pos & ((1u << a.c.page_shift) - 1), first = in + 1 - len;  // of the page's positions
    for (uint32_t h = threadIdx.x >> 6; h < a.c.n_kv; h += blockDim.x >> 6) {
        double sum[8] = {};
        for (uint32_t i = ph; i < len; i += P) {
            const uint32_t at = first + i, t = at & 31;
            const uint8_t *tile = a.c.base + kv4_tile(a.c, page, h, at >> 5);
            uint32_t w;
            _Float16 d;
            __builtin_memcpy(&w, tile + kv4_k_code(D, t, g), 4);
            __builtin_memcpy(&d, tile + kv4_k_scale(D, t, g / 4), 2);
#pragma unroll
            for (int n = 0; n < 8; ++n) sum[n] += (double)((float)((int)(w >> (4 * ((n >> 1) + 4 * (n & 1))) & 15u) - 8) * (float)d);
        }
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (uint32_t o = G; o < 64; o <<= 1) sum[n] += __shfl_xor(sum[n], (int)o, 64);
        if (ph == 0) {
            f16x8 m;
#pragma unroll
            for (int n = 0; n < 8; ++n) m[n] = (_Float16)(float)(sum[n] / (double)len);
            const size_t block = ((size_t)page << (a.c.page_shift - a.shift)) + (in >> a.shift);
            __builtin_memcpy(a.means + (block * a.c.n_kv + h) * D + 8 * g, &m, 16);
        }
    }
}

// ---- the choice --------------------------------------------------------------------------------------
//
// A workgroup for a (token, KV head).  The query at position p of block b reads the blocks 0 .. first - 1, b - last .. b
// and, of those between, the `top` of the highest score scale sum_h q_h . mean (h over the KV head's queries; of equal ones
// the first).  Scores are f64: the order of two blocks is the formula's, not the rounding's.  They are ranked as whole
// numbers of the same order; the top-th is found bit by bit from the highest one in which any two differ.

AH_DEV uint64_t rank_of(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);  // (-0 is 0)
    return v != v ? 0 : b >> 63 ? ~b : b | 1ull << 63;
}

template <int D> __global__ void __launch_bounds__(256) block_choice_kernel(BlockArgs b) {
    constexpr uint32_t L = D / 8, kPer = 64 / L, kAhead = 4;  // lanes of a block's mean, blocks of a wave
    extern __shared__ uint64_t lds_keys[];  // [b.lds_keys]
    __shared__ uint64_t red[2][4];
    __shared__ uint32_t cnt[2][4], cnt2[2][4];
    const AttnArgs &a = b.a;
    const uint32_t unit = blockIdx.x, tok = unit / a.c.n_kv, kvh = unit - tok * a.c.n_kv, tid = threadIdx.x, lane = tid & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    for (uint32_t i = unit * 256 + tid; i < a.n_seq; i += gridDim.x * 256)
        if (span_of(a, i).bad) ah_record(a.status, ((unsigned long long)i << 8) + kKeyCache);
    auto start = [&](uint32_t i) { return (uint32_t)a.q_start[i]; };
    auto holds = [&](uint32_t i) {
        const Span p = span_of(a, i);
        return tok >= p.q0 && tok - p.q0 < p.nq;
    };
    const uint32_t s = sequence_of(a, tok, start, holds);
    const Span p = span_of(a, s);
    uint32_t *list = b.list + (size_t)unit * a.list_stride;
    int32_t *chosen = b.chosen ? b.chosen + (size_t)unit * b.top : nullptr;
    if (tok < p.q0 || tok - p.q0 >= p.nq) {
        if (tid == 0) list[0] = kNoList;
        return;
    }
    const int32_t pos = p.ctx - (int32_t)p.nq + (int32_t)(tok - p.q0);
    const uint32_t own = pos < 0 ? 0 : (uint32_t)pos >> b.shift;
    const uint32_t n = own > b.first + (uint64_t)b.last ? own - b.last - b.first : 0;  // blocks to choose among, from b.first on
    const uint32_t per = a.c.page_shift - b.shift;                                     // (log2) blocks of a page
    const int32_t *table = a.table + (size_t)s * a.table_stride;
    auto page_of = [&](uint32_t block) { return (uint32_t)table[block >> per]; };
    auto entry = [&](uint32_t block) {
        const uint32_t page = page_of(block);
        if (page >= a.c.n_pages) {
            ah_record(a.status, ((unsigned long long)s << 8) + kKeyCache);
            return kNoList;
        }
        return ((page * a.c.n_kv + kvh) << (a.c.page_shift - 5)) + ((block & ((1u << per) - 1)) << (b.shift - 5));
    };
    if (n <= b.top) {  // all of them
        const uint32_t all = pos < 0 ? 0 : own + 1;
        for (uint32_t i = tid; i < all; i += 256) list[1 + i] = entry(i);
        if (tid == 0) list[0] = pos < 0 ? 0 : (uint32_t)pos + 1;
        if (chosen)
            for (uint32_t i = tid; i < b.top; i += 256) chosen[i] = i < n ? (int32_t)(b.first + i) : -1;
        return;
    }
    const bool in_lds = n <= b.lds_keys;
    uint64_t *far = b.keys + (size_t)unit * b.most;
    auto key_at = [&](uint32_t i) { return in_lds ? lds_keys[i] : far[i]; };

    // scores: L lanes a block, eight channels each
    const uint32_t g = lane % L, first = wave * kPer + lane / L;
    double q[8] = {};
    {
        const float *x = a.q + (size_t)tok * a.q_stride + (size_t)kvh * a.group * D + 8 * g;
        for (uint32_t h = 0; h < a.group; ++h) {
            float v[8];
            __builtin_memcpy(v, x + (size_t)h * D, 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] += (double)v[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] *= (double)a.scale;
    }
    uint64_t any = 0, every = ~0ull;
    for (uint32_t base = 0; base < n; base += 4 * kPer * kAhead) {
        f16x8 m[kAhead];
        bool ok[kAhead];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            const uint32_t i = base + j * 4 * kPer + first, block = b.first + (i < n ? i : n - 1);
            const uint32_t page = page_of(block);
            ok[j] = page < a.c.n_pages;
            const size_t at = ((size_t)(ok[j] ? page : 0) << per) + (block & ((1u << per) - 1));
            __builtin_memcpy(&m[j], b.means + (at * a.c.n_kv + kvh) * D + 8 * g, 16);
        }
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            const uint32_t i = base + j * 4 * kPer + first;
            double v = 0.0;
#pragma unroll
            for (int c = 0; c < 8; ++c) v = __builtin_fma(q[c], (double)(float)m[j][c], v);
#pragma unroll
            for (uint32_t o = 1; o < L; o <<= 1) v += __shfl_xor(v, (int)o, 64);
            const uint64_t key = ok[j] ? rank_of(v) : 0;
            if (i < n) {
                if (g == 0) {
                    if (in_lds) lds_keys[i] = key;
                    else far[i] = key;
                }
                any |= key;
                every &= key;
            }
        }
    }
#pragma unroll
    for (uint32_t o = L; o < 64; o <<= 1) {
        any |= __shfl_xor(any, (int)o, 64);
        every &= __shfl_xor(every, (int)o, 64);
    }
    if (lane == 0) {
        red[0][wave] = any;
        red[1][wave] = every;
    }
    __syncthreads();
    any = red[0][0] | red[0][1] | red[0][2] | red[0][3];
    every = red[1][0] & red[1][1] & red[1][2] & red[1][3];
    uint32_t turn = 0;
    auto count = [&](uint64_t at_least) {  // keys >= at_least
        uint32_t c = 0;
        for (uint32_t i = tid; i < n; i += 256) c += key_at(i) >= at_least;
#pragma unroll
        for (uint32_t o = 1; o < 64; o <<= 1) c += (uint32_t)__shfl_xor((int)c, (int)o, 64);
        if (lane == 0) cnt[turn][wave] = c;
        __syncthreads();
        c = cnt[turn][0] + cnt[turn][1] + cnt[turn][2] + cnt[turn][3];
        turn ^= 1;
        return c;
    };
    // the largest T with at least `top` keys >= T
    uint64_t T = every;
    uint32_t found = n;
    if (any != every) {
        int bit = 63 - __builtin_clzll(any ^ every);
        T = every & ~((2ull << bit) - 1);
        for (; bit >= 0 && found != b.top; --bit) {
            const uint64_t to = T | 1ull << bit;
            const uint32_t c = count(to);
            if (c >= b.top) {
                T = to;
                found = c;
            }
        }
    }
    const uint32_t above = found == b.top ? 0 : T == ~0ull ? 0 : count(T + 1), ties = found == b.top ? b.top : b.top - above;
    // keys above T, and the first `ties` that equal it (all from T on, where there are just as many)
    uint32_t gt0 = 0, eq0 = 0;
    for (uint32_t base = 0; base < n; base += 256) {
        const uint32_t i = base + tid;
        const uint64_t key = i < n ? key_at(i) : 0;
        const bool gt = i < n && found != b.top && key > T, eq = i < n && (found == b.top ? key >= T : key == T);
        const uint64_t bg = __builtin_amdgcn_ballot_w64(gt), be = __builtin_amdgcn_ballot_w64(eq), below = (1ull << lane) - 1;
        if (lane == 0) {
            cnt[turn][wave] = (uint32_t)__builtin_popcountll(bg);
            cnt2[turn][wave] = (uint32_t)__builtin_popcountll(be);
        }
        __syncthreads();
        uint32_t g_at = gt0 + (uint32_t)__builtin_popcountll(bg & below), e_at = eq0 + (uint32_t)__builtin_popcountll(be & below);
#pragma unroll
        for (uint32_t w = 0; w < 4; ++w) {
            g_at += w < wave ? cnt[turn][w] : 0;
            e_at += w < wave ? cnt2[turn][w] : 0;
            gt0 += cnt[turn][w];
            eq0 += cnt2[turn][w];
        }
        turn ^= 1;
        if (gt || (eq && e_at < ties)) {
            const uint32_t at = g_at + (e_at < ties ? e_at : ties);
            list[1 + b.first + at] = entry(b.first + i);
            if (chosen) chosen[at] = (int32_t)(b.first + i);
        }
    }
    for (uint32_t i = tid; i < b.first; i += 256) list[1 + i] = entry(i);
    for (uint32_t i = tid; i <= b.last; i += 256) list[1 + b.first + b.top + i] = entry(own - b.last + i);
    if (tid == 0) list[0] = ((b.first + b.top + b.last) << b.shift) + ((uint32_t)pos & ((1u << b.shift) - 1)) + 1;
}

} // namespace

hipError_t ah_launch_block_means(const MeansArgs &a, hipStream_t stream) {
    const dim3 grid(a.t.n_tok), block(64 * (a.c.n_kv < 4 ? a.c.n_kv : 4));
    if (a.c.dim == 64) hipLaunchKernelGGL(block_means_kernel<64>, grid, block, 0, stream, a);
    else if (a.c.dim == 128) hipLaunchKernelGGL(block_means_kernel<128>, grid, block, 0, stream, a);
    else hipLaunchKernelGGL(block_means_kernel<256>, grid, block, 0, stream, a);
    return hipGetLastError();
}

hipError_t ah_launch_block_choice(const BlockArgs &a, hipStream_t stream) {
    const dim3 grid(a.a.n_tok * a.a.c.n_kv), block(256);
    const size_t lds = a.lds_keys * sizeof(uint64_t);
    if (a.a.c.dim == 64) hipLaunchKernelGGL(block_choice_kernel<64>, grid, block, lds, stream, a);
    else if (a.a.c.dim == 128) hipLaunchKernelGGL(block_choice_kernel<128>, grid, block, lds, stream, a);
    else hipLaunchKernelGGL(block_choice_kernel<256>, grid, block, lds, stream, a);
    return hipGetLastError();
}

hipError_t ah_blocks_init_attrs() {
    const int most = (int)(kLdsKeys * sizeof(uint64_t));
    hipError_t e = hipSuccess;
    for (const void *k : {(const void *)block_choice_kernel<64>, (const void *)block_choice_kernel<128>, (const void *)block_choice_kernel<256>})
        if (e == hipSuccess) e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, most);
    return e;
}
