// ah_blocks.hip -- the choice of blocks for attention over parts of a long context in the paged 4-bit cache (layout:
// ah_kv4.h): the means of the blocks' keys, for every (token, KV head) the blocks that its queries score highest, and
// attention over many such lists (over few it is attn_rows_kernel's).
#include "ah_attn.h"

namespace {

constexpr unsigned long long kKeyCache = AH_ERR_CACHE_RANGE;

// ---- means -----------------------------------------------------------------------------------------
//
// A block whose last position is among the tokens: the mean of its keys, a wave a KV head.  Lane (p, g) sums the eight
// channels of group g over every (64 / (D / 8))-th position from p on, in f64: the cache's values have eleven
// significant bits between 2^-24 and 2^16, so the sums are exact in any order, and a block's mean is the same however
// its positions came.  It is rounded to f32 and then to f16: half a step of f16 in a mean moves a score by 2^-11 of |q| |k|, and a
// mean is 16-bit in memory because the choice reads all of them (16.8 MB for 64 contexts of 32768 keys of 2 heads of 128).
//   What bounds it: a workgroup a token, nearly all of which end no block: the launch and one round trip to learn that, another for
// the page, one for the block (64 single tokens 4.2 to 5.2 us); 2039 tokens of a prompt 7.4.
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
#pragma unroll 8
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
// The query at position p of block b reads the blocks 0 .. first - 1, b - last .. b and, of those between, the `top` of the
// highest score scale sum_h q_h . mean (h over the KV head's queries; of equal ones the first).  Scores are f64: the order of two
// blocks is the formula's, not the rounding's.  They are ranked as whole numbers of the same order.
//   What bounds it: for a token by itself round trips and barriers (512 means a KV head of 32768 keys: 11 us for one token, of which
// means and scores 4, the choice by one wave 4; 64 such tokens 13), for many f64 products and one wave's choice a token (2039
// tokens of up to 250 blocks 16.5 us).  Bits counted over a workgroup with a barrier each: 41 us for 25 of a token's
// whole call.  In one launch with the attention, which then has a CU for a token, it took as long as in two.
AH_DEV uint64_t rank_of(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);  // (-0 is 0)
    return v != v ? 0 : b >> 63 ? ~b : b | 1ull << 63;
}
template <int CTRL> AH_DEV double dpp64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xF, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
AH_DEV uint32_t count(bool x) { return (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(x)); }
AH_DEV uint32_t before(bool x) {  // lanes below this one where x is true
    const uint64_t m = __builtin_amdgcn_ballot_w64(x);
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}
// The largest T with at least `top` keys >= T, bit by bit: many(x) counts the keys >= x; found: how many are >= T.  As soon as
// those are just `top`, the rest of the bits does not matter.
template <class F> AH_DEV uint64_t threshold(uint32_t top, uint32_t n, F many, uint32_t &found) {
    uint64_t T = 0;
    found = n;
    for (int bit = 63; bit >= 0 && found != top; --bit) {
        const uint32_t c = many(T | 1ull << bit);
        if (c >= top) {
            T |= 1ull << bit;
            found = c;
        }
    }
    return T;
}

AH_DEV void record_bad(const BlockArgs &b, uint32_t at, uint32_t of) {  // sequences out of range: every of-th from at on
    for (uint32_t i = at; i < b.a.n_seq; i += of)
        if (span_of(b.a, i).bad) ah_record(b.a.status, ((unsigned long long)i << 8) + kKeyCache);
}

// What a (token, KV head) reads and where it stands in the cache.
struct Query {
    uint32_t s, own, n;  // its sequence and block; blocks to choose among, from b.first on
    int32_t pos;
};
AH_DEV Query query_of(const BlockArgs &b, const Span &p, uint32_t s, uint32_t tok) {
    Query x;
    x.s = s;
    x.pos = p.ctx - (int32_t)p.nq + (int32_t)(tok - p.q0);
    x.own = x.pos < 0 ? 0 : (uint32_t)x.pos >> b.shift;
    x.n = x.own > b.first + (uint64_t)b.last ? x.own - b.last - b.first : 0;
    return x;
}
AH_DEV uint32_t page_of(const BlockArgs &b, uint32_t s, uint32_t block) {
    return (uint32_t)b.a.table[(size_t)s * b.a.table_stride + (block >> (b.a.c.page_shift - b.shift))];
}
AH_DEV size_t mean_at(const BlockArgs &b, uint32_t page, uint32_t kvh, uint32_t block) {  // the place of a block's mean, in heads
    const uint32_t per = b.a.c.page_shift - b.shift;
    return (((size_t)page << per) + (block & ((1u << per) - 1))) * b.a.c.n_kv + kvh;
}
// A block's first tile, as attention's list has it.
AH_DEV uint32_t entry_of(const BlockArgs &b, uint32_t s, uint32_t kvh, uint32_t block) {
    const Kv4Ref &c = b.a.c;
    const uint32_t page = page_of(b, s, block), per = c.page_shift - b.shift;
    if (page >= c.n_pages) {
        ah_record(b.a.status, ((unsigned long long)s << 8) + kKeyCache);
        return kNoList;
    }
    return ((page * c.n_kv + kvh) << (c.page_shift - 5)) + ((block & ((1u << per) - 1)) << (b.shift - 5));
}
// What a query reads without a choice, by `lanes` lanes; true where that is all.
AH_DEV bool list_fixed(const BlockArgs &b, const Query &x, uint32_t kvh, uint32_t *list, int32_t *chosen, uint32_t lane, uint32_t lanes) {
    if (x.n <= b.top) {
        const uint32_t all = x.pos < 0 ? 0 : x.own + 1;
        for (uint32_t i = lane; i < all; i += lanes) list[1 + i] = entry_of(b, x.s, kvh, i);
        if (lane == 0) list[0] = x.pos < 0 ? 0 : (uint32_t)x.pos + 1;
        if (chosen)
            for (uint32_t i = lane; i < b.top; i += lanes) chosen[i] = i < x.n ? (int32_t)(b.first + i) : -1;
        return true;
    }
    for (uint32_t i = lane; i < b.first; i += lanes) list[1 + i] = entry_of(b, x.s, kvh, i);
    for (uint32_t i = lane; i <= b.last; i += lanes) list[1 + b.first + b.top + i] = entry_of(b, x.s, kvh, x.own - b.last + i);
    if (lane == 0) list[0] = ((b.first + b.top + b.last) << b.shift) + ((uint32_t)x.pos & ((1u << b.shift) - 1)) + 1;
    return false;
}

// The `top` largest of the keys of lanes in `valid` (of equal ones the first), by the bits from the highest on: `alive` are the
// lanes still equal to the top-th as far as the bits go.  least: nothing chosen is smaller.
AH_DEV bool largest(uint64_t key, uint64_t valid, uint32_t top, uint64_t &least) {
    uint64_t alive = valid, taken = 0, prefix = 0;
    uint32_t need = top;
#pragma unroll
    for (int word = 1; word >= 0; --word) {
        const uint32_t v = (uint32_t)(key >> (32 * word));
        for (int bit = 31; bit >= 0 && (uint32_t)__builtin_popcountll(alive) != need; --bit) {
            const uint64_t ones = __builtin_amdgcn_ballot_w64((v >> bit & 1u) != 0) & alive;
            const uint32_t c = (uint32_t)__builtin_popcountll(ones);
            if (c >= need) {
                alive = ones;
                prefix |= 1ull << (32 * word + bit);
            } else {
                taken |= ones;
                need -= c;
                alive &= ~ones;
            }
        }
    }
    least = prefix;
    const uint64_t me = 1ull << (threadIdx.x & 63);
    return (taken & me) || ((alive & me) && __builtin_amdgcn_mbcnt_hi((uint32_t)(alive >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)alive, 0)) < need);
}
// The choice among n > top keys by one wave: emit(place, block) for the chosen ones, ascending.  With top at most 64, the top-th of
// the lanes' largest keys bounds the top-th of all from below, and few keys pass it; where no more than 64 do, a lane each,
// those are chosen among.  false: it is left to many_keys.
template <class K, class E> AH_DEV bool few_keys(uint32_t n, uint32_t top, uint64_t *room, K key_at, E emit) {
    constexpr uint32_t kBatch = 8;  // keys of a lane on their way
    if (top > 64) return false;
    const uint32_t lane = threadIdx.x & 63;
    uint64_t most = 0, k[kBatch];
    auto batch = [&](uint32_t base) {
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j) {
            const uint32_t i = base + 64 * j + lane;
            k[j] = key_at(i < n ? i : n - 1);
            k[j] = i < n ? k[j] : 0;
        }
    };
    for (uint32_t base = 0; base < n; base += 64 * kBatch) {
        batch(base);
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j) most = k[j] > most ? k[j] : most;
    }
    uint64_t bound, least;
    (void)largest(most, ~0ull, top, bound);
    uint32_t c = 0;
    for (uint32_t base = 0; base < n; base += 64 * kBatch) {
        if (n > 64 * kBatch) batch(base);
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j) {
            const uint32_t i = base + 64 * j + lane;
            const bool in = i < n && k[j] >= bound;
            const uint32_t at = c + before(in);
            if (in && at < 64) {
                room[at] = k[j];
                room[64 + at] = i;
            }
            c += count(in);
        }
    }
    if (c > 64) return false;
    __builtin_amdgcn_wave_barrier();
    const bool in = largest(lane < c ? room[lane] : 0, c == 64 ? ~0ull : (1ull << c) - 1, top, least);
    if (in) emit(before(in), (uint32_t)room[64 + lane]);
    return true;
}
// Any n and top, `waves` waves together (one: no barriers): many(x) counts the keys >= x over all of them.
template <class K, class E, class M> AH_DEV void many_keys(uint32_t n, uint32_t top, K key_at, E emit, M many) {
    uint32_t found;
    const uint64_t T = threshold(top, n, many, found);
    const uint32_t above = found == top || T == ~0ull ? 0 : many(T + 1);
    const uint32_t lane = threadIdx.x & 63, ties = top - above;
    uint32_t gt = 0, eq = 0;
    for (uint32_t base = 0; base < n; base += 64) {
        const uint64_t k = base + lane < n ? key_at(base + lane) : 0;
        const bool x = base + lane < n && found != top && k > T, y = base + lane < n && (found == top ? k >= T : k == T);
        const uint32_t g = gt + before(x), e = eq + before(y);
        if (x || (y && e < ties)) emit(g + (e < ties ? e : ties), base + lane);
        gt += count(x);
        eq += count(y);
    }
}

// The choice for a (token, KV head) by a workgroup of W waves, into `list` (as attention's, kNoList where the token is no
// sequence's).  Scores: D / 8 lanes a block, eight channels each, the means of several blocks a lane on their way (a load touches
// few lines; with a lane for a whole mean it touches 64).  16 waves: all blocks of 32768 keys are on their way at once.
//   Where a context has more blocks than LDS has room for scores (it is longer than planned, or the longest of all), they go by
// passes: after one, the `top` largest stand in front, in the order of their blocks, with their numbers, and the next pass's behind
// them; of equal scores the first is still the first.
struct Passes {
    uint64_t *keys;    // [what LDS holds]
    uint32_t *number;  // [top]: of what is kept
    uint32_t top;
    // (blocks are counted from the first that is chosen among)
    AH_DEV uint32_t block_of(uint32_t i, uint32_t kept, uint32_t done) const { return i < kept ? number[i] : done + (i - kept); }
    AH_DEV void keep(uint32_t at, uint32_t i, uint32_t block) const {  // (at <= i: nothing is overwritten that is still to be read)
        const uint64_t key = keys[i];
        keys[at] = key;
        number[at] = block;
    }
};
template <int D, int W> struct ChoiceLds {
    double q[D];
    uint64_t room[128];
    uint32_t cnt[2][W], done;
};
template <int D, int W> AH_DEV void choose(const BlockArgs &b, uint32_t unit, uint32_t *list, uint64_t *lds_keys, ChoiceLds<D, W> &L) {
    constexpr uint32_t kLanes = D / 8, kPer = 64 / kLanes, kAhead = W >= 16 ? D == 256 ? 3 : 4 : 8;  // lanes of a block's mean, blocks of a wave
    const AttnArgs &a = b.a;
    const uint32_t tok = unit / a.c.n_kv, kvh = unit - tok * a.c.n_kv, tid = threadIdx.x, lane = tid & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane % kLanes;
    // q's sum over the heads, before the sequence is known
    double q[8] = {};
    {
        const float *x = a.q + (size_t)tok * a.q_stride + (size_t)kvh * a.group * D + 8 * g;
#pragma unroll 8
        for (uint32_t h = 0; h < a.group; ++h) {
            float v[8];
            __builtin_memcpy(v, x + (size_t)h * D, 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] += (double)v[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] *= (double)a.scale;
    }
    auto start = [&](uint32_t i) { return (uint32_t)a.q_start[i]; };
    auto holds = [&](uint32_t i) {
        const Span p = span_of(a, i);
        return tok >= p.q0 && tok - p.q0 < p.nq;
    };
    const uint32_t s = __builtin_amdgcn_readfirstlane(sequence_of(a, tok, start, holds));
    const Span p = span_of(a, s);
    int32_t *chosen = b.chosen ? b.chosen + (size_t)unit * b.top : nullptr;
    if (tok < p.q0 || tok - p.q0 >= p.nq) {
        if (tid == 0) list[0] = kNoList;
        if (tid == 0) record_bad(b, unit, gridDim.x);
        return;
    }
    const Query x = query_of(b, p, s, tok);
    const uint32_t n = x.n;
    auto score = [&](uint32_t from, uint32_t num, uint64_t *keys) {  // of the blocks from .. from + num - 1
        const uint32_t first = wave * kPer + lane / kLanes, step = W * kPer;
        for (uint32_t base = 0; base < num; base += step * kAhead) {
            f16x8 m[kAhead];
            uint32_t page[kAhead];
            auto block_at = [&](uint32_t i) { return b.first + from + (i < num ? i : num - 1); };
#pragma unroll
            for (uint32_t j = 0; j < kAhead; ++j) page[j] = page_of(b, s, block_at(base + j * step + first));
#pragma unroll
            for (uint32_t j = 0; j < kAhead; ++j)
                __builtin_memcpy(&m[j], b.means + mean_at(b, page[j] < a.c.n_pages ? page[j] : 0, kvh, block_at(base + j * step + first)) * D + 8 * g, 16);
#pragma unroll
            for (uint32_t j = 0; j < kAhead; ++j) {
                const uint32_t i = base + j * step + first;
                double v = 0.0;
#pragma unroll
                for (int c = 0; c < 8; ++c) v = __builtin_fma(q[c], (double)(float)m[j][c], v);
                v += dpp64<0xB1>(v);   // lanes 1 0 3 2
                v += dpp64<0x4E>(v);   // lanes 2 3 0 1
                v += dpp64<0x141>(v);  // the other half of eight, mirrored
                if (kLanes >= 16) v += dpp64<0x140>(v);  // of sixteen
                if (kLanes == 32) v += __shfl_xor(v, 16, 64);
                const uint64_t key = page[j] < a.c.n_pages ? rank_of(v) : 0;
                if (i < num && g == 0) keys[i] = key;
            }
        }
    };
    auto fixed = [&] {
        (void)list_fixed(b, x, kvh, list, chosen, lane, 64);
        if (lane == 0) record_bad(b, unit, gridDim.x);
    };
    auto key_at = [&](uint32_t i) { return lds_keys[i]; };
    auto choice = [&](uint32_t num, auto emit, bool begin) {  // among the keys in LDS
        __syncthreads();
        if (wave == 0) {
            const bool all = few_keys(num, b.top, L.room, key_at, emit);
            if (lane == 0) L.done = all;
        }
        if (begin && wave == 1) fixed();
        __syncthreads();
        if (L.done) return;
        uint32_t turn = 0;
        auto many = [&](uint64_t at_least) {
            uint32_t c = 0;
            for (uint32_t base = 64 * wave; base < num; base += 64 * W) c += count(base + lane < num && key_at(base + lane) >= at_least);
            if (lane == 0) L.cnt[turn][wave] = c;
            __syncthreads();
            c = 0;
#pragma unroll
            for (uint32_t w = 0; w < W; ++w) c += L.cnt[turn][w];
            turn ^= 1;
            return c;
        };
        many_keys(num, b.top, key_at, [&](uint32_t at, uint32_t i) {
            if (wave == 0) emit(at, i);
        }, many);
    };
    auto put = [&](uint32_t at, uint32_t block) {
        list[1 + b.first + at] = entry_of(b, s, kvh, b.first + block);
        if (chosen) chosen[at] = (int32_t)(b.first + block);
    };
    if (n <= b.top) {
        if (wave == 1) fixed();
        return;
    }
    if (__builtin_expect(n <= b.lds_keys, true)) {
        score(0, n, lds_keys);
        choice(n, put, true);
        return;
    }
    // Blocks done .. done + now - 1, behind the `kept` largest of those before them.
    if (wave == 0 && lane < kLanes) {  // (for every pass, rather than in registers through the choice)
#pragma unroll
        for (int i = 0; i < 8; ++i) L.q[8 * g + i] = q[i];
    }
    const Passes P = {lds_keys, reinterpret_cast<uint32_t *>(lds_keys + b.lds_keys), b.top};
    uint32_t done = 0, kept = 0;
    for (;;) {
        const uint32_t now = n - done < b.lds_keys - kept ? n - done : b.lds_keys - kept;
        const bool last = done + now == n;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = L.q[8 * g + i];
        score(done, now, lds_keys + kept);
        choice(kept + now, [&](uint32_t at, uint32_t i) {
            const uint32_t block = P.block_of(i, kept, done);
            if (last) put(at, block);
            else P.keep(at, i, block);
        }, done == 0);
        if (last) return;
        done += now;
        kept = b.top;
    }
}
template <int D> __global__ void __launch_bounds__(1024, 8) block_choice_kernel(BlockArgs b) {
    extern __shared__ uint64_t lds_keys[];  // [b.lds_keys]
    __shared__ ChoiceLds<D, 16> L;
    choose<D, 16>(b, blockIdx.x, b.list + (size_t)blockIdx.x * b.a.list_stride, lds_keys, L);
}

// A workgroup for 16 tokens of a sequence and a KV head: scores of 16 blocks and the 16 tokens by f64 matrix products (lane
// (r, h): token r, blocks h + 4 i of the result), then a token's choice by one wave: the means are read once for 16 tokens, and no
// barrier stands inside a choice.  16 waves rather than 4: 2039 tokens of 16001 keys 16.5 us for 20.
template <int D> constexpr uint32_t kSomeWaves = D == 256 ? 8 : 16;  // (as many as the registers allow)
template <int D> __global__ void __launch_bounds__(64 * kSomeWaves<D>) block_choices_kernel(BlockArgs b) {
    typedef double f64x4 __attribute__((ext_vector_type(4)));
    constexpr int Q = D / 4;  // channels of a lane's quarter
    extern __shared__ uint64_t lds[];
    __shared__ uint64_t room[kSomeWaves<D>][128];
    const AttnArgs &a = b.a;
    const uint32_t at = blockIdx.x / a.c.n_kv, kvh = blockIdx.x - at * a.c.n_kv, lane = threadIdx.x & 63, r = lane & 15, h = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    double *qs = reinterpret_cast<double *>(lds);  // [16][D + 2]
    uint64_t *keys = lds + 16 * (D + 2);           // [16][stride]
    const uint32_t stride = b.lds_keys + 1;
    if (kvh == 0 && threadIdx.x == 0) record_bad(b, at, b.tiles);
    auto start = [&](uint32_t i) { return (uint32_t)a.q_start[i] / 16 + i; };
    auto holds = [&](uint32_t i) {
        const Span p = span_of(a, i);
        return at >= start(i) && at - start(i) < (p.nq + 15) / 16;
    };
    const uint32_t s = sequence_of(a, at, start, holds);
    const Span p = span_of(a, s);
    const uint32_t tile = at - start(s);
    if (tile >= (p.nq + 15) / 16) return;
    const uint32_t tok0 = p.q0 + 16 * tile, live = p.nq - 16 * tile < 16 ? p.nq - 16 * tile : 16;
    const uint32_t most = query_of(b, p, s, tok0 + live - 1).n;  // (the last token's: the most; no other has two fewer)
    uint32_t *numbers = reinterpret_cast<uint32_t *>(keys + 16 * stride);  // [16][top]
    if (most > b.top) {
        for (uint32_t i = threadIdx.x; i < 16 * D; i += 64 * kSomeWaves<D>) {
            const uint32_t t = i / D, c = i % D;
            const float *x = a.q + (size_t)(tok0 + (t < live ? t : 0)) * a.q_stride + (size_t)kvh * a.group * D + c;
            double v = 0.0;
#pragma unroll 8
            for (uint32_t g = 0; g < a.group; ++g) v += (double)x[(size_t)g * D];
            qs[t * (D + 2) + c] = v * (double)a.scale;
        }
        __syncthreads();
    }
    // Blocks done .. done + now - 1, behind the `kept` largest of those before them (Passes).
    uint32_t done = 0, kept = 0;
    for (;;) {
        const uint32_t now = most <= b.top ? most : most - done < b.lds_keys - kept ? most - done : b.lds_keys - kept;
        const bool last = done + now == most;
        if (most > b.top) {
            double q[Q];
#pragma unroll
            for (int i = 0; i < Q; ++i) q[i] = qs[r * (D + 2) + h * Q + i];
            for (uint32_t base = 16 * wave; base < now; base += 16 * kSomeWaves<D>) {
                const uint32_t i = base + r, block = b.first + done + (i < now ? i : now - 1), page = page_of(b, s, block);
                const bool ok = page < a.c.n_pages;
                _Float16 m[Q];
                __builtin_memcpy(m, b.means + mean_at(b, ok ? page : 0, kvh, block) * D + h * Q, 2 * Q);
                f64x4 v = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
                for (int c = 0; c < Q; ++c) v = __builtin_amdgcn_mfma_f64_16x16x4f64((double)(float)m[c], q[c], v, 0, 0, 0);
                const uint32_t good = (uint32_t)__builtin_amdgcn_ballot_w64(ok);  // of the blocks: lanes 0 to 15
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const uint32_t j = h + 4 * n;
                    if (base + j < now) keys[r * stride + kept + base + j] = good >> j & 1 ? rank_of(v[n]) : 0;
                }
            }
            __syncthreads();
        }
        for (uint32_t t = wave; t < live; t += kSomeWaves<D>) {
            const uint32_t tok = tok0 + t, unit = tok * a.c.n_kv + kvh;
            const Query x = query_of(b, p, s, tok);
            uint32_t *list = b.list + (size_t)unit * a.list_stride;
            int32_t *chosen = b.chosen ? b.chosen + (size_t)unit * b.top : nullptr;
            if (done ? x.n <= b.top : list_fixed(b, x, kvh, list, chosen, lane, 64)) continue;
            const Passes P = {keys + t * stride, numbers + t * b.top, b.top};
            const uint32_t n = kept + (x.n - done < now ? x.n - done : now);
            auto key_at = [&](uint32_t i) { return P.keys[i]; };
            auto emit = [&](uint32_t to, uint32_t i) {
                const uint32_t block = P.block_of(i, kept, done);
                if (last) {
                    list[1 + b.first + to] = entry_of(b, s, kvh, b.first + block);
                    if (chosen) chosen[to] = (int32_t)(b.first + block);
                } else {
                    P.keep(to, i, block);
                }
            };
            if (few_keys(n, b.top, room[wave], key_at, emit)) continue;
            many_keys(n, b.top, key_at, emit, [&](uint64_t at_least) {
                uint32_t c = 0;
                for (uint32_t i = lane; i < (n + 63) / 64 * 64; i += 64) c += count(i < n && key_at(i) >= at_least);
                return c;
            });
        }
        if (last) return;
        done += now;
        kept = b.top;
        __syncthreads();
    }
}

// ---- attention over a list of blocks ---------------------------------------------------------------------
//
// attn_rows_kernel's eight packed rows (ah_attn.hip), all of one token: the KV head's queries see the same keys, 0 .. keys - 1 of
// the listed blocks one after the other, so only the last tile needs a mask.  A wave takes a whole list: with enough of them
// nobody needs to be met.
//   What bounds it: vector work, 88% of a SIMD's cycles while a CU works (210 instructions a tile of 32 keys of 64 channels: a
// list is one token's, so its queries alone share what converting the codes costs).  2039 tokens, 7 heads over 2, lists of up to
// 1184 keys, 8.8 GFLOP: 72 us.
template <int D, class T> AH_DEV void attend_rows(const AttnArgs &a, uint32_t tok, uint32_t kvh, uint32_t keys, T tile_at) {
    constexpr int NJ = D / 32;
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, h = lane >> 4, row = r & 7;
    const uint32_t tiles = (keys + 31) / 32;
    const bool live = row < a.group, low = r >= 8;
    KTile<D> k;
    VTile<D> v;
    bool ok = true;
    if (tiles) {
        const uint8_t *t = tile_at(0, ok);
        k.load(t, r, h);
        v.load(t, r, h);
    }
    f16x8 qh[NJ];
    float f;
    {
        const float *q = a.q + (size_t)tok * a.q_stride + (size_t)(kvh * a.group + (live ? row : 0)) * D + h * (D / 4);
        float x[NJ][8], top = 0.0f, up;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            __builtin_memcpy(x[j], q + 8 * j, 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[j][i] = live ? x[j][i] : 0.0f;
                top = __builtin_fmaxf(top, __builtin_fabsf(x[j][i]));
            }
        }
        top = __builtin_fmaxf(top, xor_lanes(top, 16));
        top = __builtin_fmaxf(top, xor_lanes(top, 32));
        q_scale(a.scale, top, up, f);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = x[j][i] * up;
                const _Float16 hv = (_Float16)y;
                qh[j][i] = low ? (_Float16)(y - (float)hv) : hv;
            }
    }
    f32x4 acc[NJ][2];
#pragma unroll
    for (int g = 0; g < NJ; ++g) acc[g][0] = acc[g][1] = (f32x4)0.0f;
    float m = kNoMax, l = 0.0f;
    const Masks mk;
    const float minus_low = low ? -1.0f : 0.0f;
    for (uint32_t ti = 0; ti < tiles; ++ti) {
        bool ok_next;
        const uint8_t *tn = tile_at(ti + 1 < tiles ? ti + 1 : ti, ok_next);
        f32x4 c[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            f32x4 rest = (f32x4)0.0f;  // (as in attn_rows)
            c[half] = (f32x4)0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                f32x4 &to = D > 64 && j >= NJ / 2 ? rest : c[half];
                to = mfma16(k_frag(k.code(half, j), k.scale(half, j), mk), qh[j], to);
            }
            if (D > 64) c[half] += rest;
        }
        k.load(tn, r, h);
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float y = c[i >> 2][i & 3];
            x[i] = y + ror8(y);
        }
        if (!ok || 32 * ti + 32 > keys) {
            const uint32_t end = ok ? keys : 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 32 * ti + 16 * (i >> 2) + 4 * h + (i & 3) < end ? x[i] : -__builtin_inff();
        }
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = __builtin_fmaxf(top, x[i]);
        top *= f;
        if (__builtin_amdgcn_ballot_w64(top > m + kSlack) != 0ull) {
            top = __builtin_fmaxf(top, xor_lanes(top, 16));
            top = __builtin_fmaxf(top, xor_lanes(top, 32));
            const float up = __builtin_fmaxf(m, top), alpha = __builtin_amdgcn_exp2f(m - up);
            m = up;
            l *= alpha;
#pragma unroll
            for (int g = 0; g < NJ; ++g) {
                acc[g][0] *= alpha;
                acc[g][1] *= alpha;
            }
        }
        const float base = kUp - m;
        float ls = 0.0f;
        f16x2 pl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * i], f, base)), e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * i + 1], f, base));
            ls = i ? ls + e0 : e0;
            ls += e1;
            const f16x2 ph = pack16(e0, e1);
            pl[i] = pack16(__builtin_fmaf((float)ph[0], minus_low, e0), __builtin_fmaf((float)ph[1], minus_low, e1));
        }
        l += ls;
        const f16x8 pf = join8(pl[0], pl[1], pl[2], pl[3]);
#pragma unroll
        for (int g = 0; g < NJ; ++g) {
            f16x8 even, odd;
            v_frags(v.w[g >> 1][2 * (g & 1)], v.w[g >> 1][2 * (g & 1) + 1], v.d[g], mk, even, odd);
            acc[g][0] = mfma16(even, pf, acc[g][0]);
            acc[g][1] = mfma16(odd, pf, acc[g][1]);
        }
        v.load(tn, r, h);
        ok = ok_next;
    }
    l += xor_lanes(l, 16);
    l += xor_lanes(l, 32);
    float *out = a.out + (size_t)tok * a.out_stride + (size_t)kvh * a.group * D;
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
#pragma unroll
    for (int g = 0; g < NJ; ++g) {
        float o[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float e = acc[g][0][i], d = acc[g][1][i];
            o[2 * i] = (e + ror8(e)) * inv;
            o[2 * i + 1] = (d + ror8(d)) * inv;
        }
        if (!low && live) __builtin_memcpy(out + (size_t)row * D + 32 * g + 8 * h, o, 32);
    }
}

// A wave a (token, KV head), four of them a workgroup.
template <int D> __global__ void __launch_bounds__(256, D == 256 ? 2 : D == 128 ? 3 : 4) attend_lists_kernel(AttnArgs a) {
    const uint32_t unit = 4 * blockIdx.x + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tok = unit / a.c.n_kv, kvh = unit - tok * a.c.n_kv;
    if (tok >= a.n_tok) return;
    bool none = true;
    for (uint32_t base = 0; none && base < a.seqs; base += 64) {
        const uint32_t i = base + (threadIdx.x & 63);
        const Span p = span_of(a, i < a.seqs ? i : 0);
        none = !__builtin_amdgcn_ballot_w64(i < a.seqs && tok >= p.q0 && tok - p.q0 < p.nq);
    }
    if (none) return;
    typedef const uint32_t __attribute__((address_space(4))) *cptr;
    const cptr list = (cptr)(uintptr_t)(a.list + (size_t)unit * a.list_stride);
    auto tile_at = [&](uint32_t tile, bool &ok) {
        const uint32_t at = list[1 + (tile >> a.block_shift)];
        ok = at != kNoList;
        return (const uint8_t *)a.c.base + (uint64_t)((ok ? at : 0) + (tile & ((1u << a.block_shift) - 1))) * (36u * D);
    };
    attend_rows<D>(a, tok, kvh, list[0], tile_at);
}

} // namespace

hipError_t ah_launch_block_means(const MeansArgs &a, hipStream_t stream) {
    const dim3 grid(a.t.n_tok), block(64 * (a.c.n_kv < 4 ? a.c.n_kv : 4));
    if (a.c.dim == 64) hipLaunchKernelGGL(block_means_kernel<64>, grid, block, 0, stream, a);
    else if (a.c.dim == 128) hipLaunchKernelGGL(block_means_kernel<128>, grid, block, 0, stream, a);
    else hipLaunchKernelGGL(block_means_kernel<256>, grid, block, 0, stream, a);
    return hipGetLastError();
}

template <int D> void launch_choice(const BlockArgs &a, hipStream_t stream) {
    if (!a.tiles) {
        hipLaunchKernelGGL(block_choice_kernel<D>, dim3(a.a.n_tok * a.a.c.n_kv), dim3(1024), a.lds_bytes, stream, a);
        return;
    }
    hipLaunchKernelGGL(block_choices_kernel<D>, dim3(a.tiles * a.a.c.n_kv), dim3(64 * kSomeWaves<D>), a.lds_bytes, stream, a);
}

hipError_t ah_launch_block_choice(const BlockArgs &a, hipStream_t stream) {
    if (a.a.c.dim == 64) launch_choice<64>(a, stream);
    else if (a.a.c.dim == 128) launch_choice<128>(a, stream);
    else launch_choice<256>(a, stream);
    return hipGetLastError();
}

hipError_t ah_launch_attend_lists(const AttnArgs &a, hipStream_t stream) {
    const dim3 grid((a.n_tok * a.c.n_kv + 3) / 4), block(256);
    if (a.c.dim == 64) hipLaunchKernelGGL(attend_lists_kernel<64>, grid, block, 0, stream, a);
    else if (a.c.dim == 128) hipLaunchKernelGGL(attend_lists_kernel<128>, grid, block, 0, stream, a);
    else hipLaunchKernelGGL(attend_lists_kernel<256>, grid, block, 0, stream, a);
    return hipGetLastError();
}

hipError_t ah_blocks_init_attrs() {
    const int most = (int)kChoiceLds;
    hipError_t e = hipSuccess;
    for (const void *k : {(const void *)block_choice_kernel<64>, (const void *)block_choice_kernel<128>, (const void *)block_choice_kernel<256>,
                          (const void *)block_choices_kernel<64>, (const void *)block_choices_kernel<128>, (const void *)block_choices_kernel<256>})
        if (e == hipSuccess) e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, most);
    return e;
}
