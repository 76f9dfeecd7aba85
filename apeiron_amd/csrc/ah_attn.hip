// ah_attn.hip -- attention over the paged 4-bit cache (layout: ah_kv4.h).
//
// o = sum_t softmax_t(scale q . k_t) v_t over the keys t a query at position p sees: t <= p and, with a
// window, t > p - window or t < sinks.  One pass over the cache with the running maximum and sum of the
// softmax in f32, K q and P V on the f16 matrix cores.  The cache's values are exact in f16; q and p are
// carried as f16 pairs hi + lo, both rounded to nearest (23 bits: a lost half would cost 12 of them), each pair's
// two products summed in the f32 accumulator.  What is left are f32's roundings of scores, exponentials and
// running sums: 4e-7 to 9e-7 of the outputs (root mean square against 64 bits, 4001 to 30000 keys), 7e-7 to
// 2.1e-6 with plain f32 operations.
#include "ah_attn.h"

namespace {

// The tiles that rows at positions lo .. hi see: [0, head) and [tail, end).
struct Tiles {
    uint32_t head, tail, end, count;
};
AH_DEV Tiles tiles_of(const AttnArgs &a, int32_t lo, int32_t hi) {
    Tiles t;
    t.end = hi < 0 ? 0 : ((uint32_t)hi >> 5) + 1;
    t.tail = t.head = 0;
    if (a.window && (int64_t)lo + 1 > (int64_t)a.window) {
        t.tail = ((uint32_t)lo + 1 - a.window) >> 5;
        const uint32_t h = (uint32_t)(((uint64_t)a.sinks + 31) >> 5);
        t.head = h < t.tail ? h : t.tail;
        if (t.tail > t.end) t.tail = t.end;
    }
    if (t.head > t.tail) t.head = t.tail;
    t.count = t.head + (t.end - t.tail);
    return t;
}

// What a launch reads of the contexts:
//   kAll: the positions that a query sees, in its sequence's pages;
//   kPrefix: every row the first first_key positions, in the pages of one table: the whole batch as one sequence;
//   kAfter: as kAll, from position first_key on;
//   kTwo: as kAll, the positions below first_key in the pages of a table of their own, for each sequence anew;
//   kBlocks: every (token, KV head) the blocks that it has a list of, as if they stood one after the other.
// kPrefix and kAfter leave their pieces for attn_meet_kernel, pieces of kAfter without a key with no weight.
enum { kAll, kPrefix, kAfter, kBlocks, kTwo };
template <int MODE> AH_DEV Span span_in(const AttnArgs &a, uint32_t s, uint32_t kvh) {
    if (MODE == kPrefix) return {0, a.n_tok, (int32_t)a.first_key, false};
    if (MODE == kBlocks) {  // [0] of a list: its keys, kNoList where the token is no sequence's
        const uint32_t keys = a.list[((size_t)s * a.c.n_kv + kvh) * a.list_stride];
        bool none = a.seqs == 0 && keys == kNoList;
        if (a.seqs) {
            none = true;
            for (uint32_t base = 0; none && base < a.seqs; base += 64) {
                const uint32_t i = base + (threadIdx.x & 63);
                const Span p = span_of(a, i < a.seqs ? i : 0);
                none = !__builtin_amdgcn_ballot_w64(i < a.seqs && s >= p.q0 && s - p.q0 < p.nq);
            }
        }
        return {s, none ? 0u : 1u, none ? 0 : (int32_t)keys, none};
    }
    Span p = span_of(a, s);
    if ((MODE == kAfter || MODE == kTwo) && p.nq && p.ctx - (int32_t)p.nq < (int32_t)a.first_key) p = {0, 0, 0, true};
    return p;
}
template <int MODE> AH_DEV int32_t position_of(const Span &p, uint32_t tok) {  // of a span's token
    return MODE == kPrefix ? p.ctx - 1 : p.ctx - (int32_t)p.nq + (int32_t)tok;
}
template <int MODE> AH_DEV Tiles tiles_in(const AttnArgs &a, int32_t lo, int32_t hi) {
    if (MODE != kAfter && MODE != kTwo) return tiles_of(a, lo, hi);
    Tiles t;
    t.end = hi < 0 ? 0 : ((uint32_t)hi >> 5) + 1;
    t.head = MODE == kTwo ? (a.first_key >> 5) + ((a.first_key & 31) != 0) : 0;  // (a tile may be in both)
    t.tail = a.first_key >> 5;
    t.count = t.head + (t.end > t.tail ? t.end - t.tail : 0);
    return t;
}

// Tiles of a piece: the planned chunk, or more where a context is longer than the caller's bound.
AH_DEV uint32_t piece_of(const AttnArgs &a, const Tiles &t) {
    const uint32_t need = (t.count + a.splits - 1) / a.splits;
    return need > a.chunk ? need : a.chunk;
}

// Tile `tile` for head kvh in the cache, through a sequence's row of the page table; `ok` false where
// the page is outside.  The index is read through the scalar cache: it is the same for the whole wave.
AH_DEV const uint8_t *tile_at(const AttnArgs &a, const int32_t *table, uint32_t kvh, uint32_t tile, bool &ok) {
    typedef const int32_t __attribute__((address_space(4))) *cptr;
    const uint32_t in = a.c.page_shift - 5, pi = tile >> in;
    const uint32_t page = (uint32_t)((cptr)(uintptr_t)table)[pi];
    ok = page < a.c.n_pages;
    return a.c.base + kv4_tile(a.c, ok ? page : 0, kvh, tile & ((1u << in) - 1));
}

// (prefix: of kTwo, a tile of the first table)
template <int MODE> AH_DEV const uint8_t *tile_in(const AttnArgs &a, uint32_t s, uint32_t kvh, uint32_t tile, bool &ok, bool prefix = false) {
    if (MODE != kBlocks) return tile_at(a, MODE == kTwo && prefix ? a.first_table : a.table + (size_t)s * a.table_stride, kvh, tile, ok);
    typedef const uint32_t __attribute__((address_space(4))) *cptr;
    const uint32_t at = ((cptr)(uintptr_t)a.list)[((size_t)s * a.c.n_kv + kvh) * a.list_stride + 1 + (tile >> a.block_shift)];
    ok = at != kNoList;
    return a.c.base + (uint64_t)((ok ? at : 0) + (tile & ((1u << a.block_shift) - 1))) * (36u * a.c.dim);
}

// Rows (token, head of the group) as the 16 columns of the products: every wave takes tiles of 32 tokens of
// the workgroup's piece of the context, each with its own running maximum, and the four meet in LDS.  A
// lane (r, h) holds the scores of column r, tokens 4 h + i of both half-tiles.
//   PACK: 8 rows, column r the hi half of row r & 7 for r < 8 and the lo half for r >= 8: one product gives
//   both (they meet by a rotation of the columns), half the matrix work where a call has few rows.
//   Otherwise 16 rows, or C times 16, whose columns share a tile's converted codes, and a product for each half.
// A tile's K is used first and its V last, so the next tile's K loads go out as soon as the scores are
// formed and its V loads as soon as the output is: a wave always has half a tile on its way.
//   What bounds it: for many keys in all the cache's bytes (64 sequences of 1 to 16384 keys, 12 heads of 128 over
// 2: 151 MB in 48 us, 3.2 TB/s; 128 of 4000 with 8 KV heads 590 MB in 131, 4.5 TB/s), for few the chain of a launch, a
// page's index, a tile, the partial results' way to the last workgroup and back (4001 keys: 9.8 us).  A unit
// over all keys in one workgroup, joined by nobody, costs 0.7 us a tile and wave; a second launch for the join
// 5 us more; equal shares of all units' tiles for every workgroup (two units in one) up to 10.
template <int D, bool PACK, int MODE, int C = 1> AH_DEV void attn_rows(const AttnArgs &a, uint32_t block, uint32_t grid) {
    constexpr int NJ = D / 32;  // contraction steps of K q, and blocks of channels
    constexpr uint32_t R = PACK ? 8 : 16 * C, kRed = 16 * C;
    static_assert(C == 1 || (!PACK && MODE == kPrefix), "more columns are for rows that all see the same keys");
    extern __shared__ float lds[];
    float *red_o = lds;                   // [4][16 C][D + 4]
    float *red_m = lds + 4 * kRed * (D + 4);  // [4][16 C], then the sums
    float *red_l = red_m + 4 * kRed;
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, h = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // pieces run slowest: the workgroups without work (pieces past a short context) are the last ones, and
    // every XCD (workgroups go to them in turn) gets its share of those with work; a context's pieces go
    // round the XCDs
    const uint32_t units = grid / a.splits, split = block / units, unit = (block - split * units + split) % units;
    const uint32_t per = units / a.n_seq, s = unit / per, rest = unit - s * per, rt = rest / a.c.n_kv, kvh = rest - rt * a.c.n_kv;
    const Span p = span_in<MODE>(a, s, kvh);
    if (MODE != kBlocks && p.bad && split == 0 && rest == 0 && threadIdx.x == 0) ah_record(a.status, ((unsigned long long)s << 8) + AH_ERR_CACHE_RANGE);
    const uint32_t rows = p.nq * a.group, row0 = rt * R;
    if (row0 >= rows || (MODE == kAll && rows > a.most_rows)) return;
    const uint32_t row = row0 + r % R, tok = row / a.group;
    const bool live = row < rows, low = PACK && r >= 8;
    const uint32_t last = row0 + R - 1 < rows ? row0 + R - 1 : rows - 1;
    const int32_t lo = position_of<MODE>(p, row0 / a.group), hi = position_of<MODE>(p, last / a.group);
    const int32_t pos = live ? position_of<MODE>(p, tok) : -1;
    // the keys below which the window hides one (for this row, and for the last of the rows), and the sinks
    const int32_t low_key = MODE == kAfter || MODE == kTwo ? (int32_t)a.first_key : a.window ? pos - (int32_t)a.window + 1 : 0;
    const int32_t low_all = MODE == kAfter || MODE == kTwo ? (int32_t)a.first_key : a.window ? hi - (int32_t)a.window + 1 : 0;
    const int32_t sink_key = (int32_t)a.sinks;
    const Tiles T = tiles_in<MODE>(a, lo, hi);
    const uint32_t chunk = piece_of(a, T), t0 = split * chunk, t1 = t0 + chunk < T.count ? t0 + chunk : T.count;
    if (MODE != kAfter && split > 0 && t0 >= T.count) return;

    // the first tile's loads go out before q is prepared
    KTile<D> k;
    VTile<D> v;
    bool ok = true;
    uint32_t ti = t0 + wave;
    auto tile_of = [&](uint32_t i) { return i < T.head ? i : T.tail + (i - T.head); };
    if (ti < t1) {
        const uint8_t *t = tile_in<MODE>(a, s, kvh, tile_of(ti), ok, ti < T.head);
        k.load(t, r, h);
        v.load(t, r, h);
    }

    // q, scaled by a power of two so that its largest magnitude is in [2^13, 2^14), as hi + lo
    f16x8 qh[C][NJ], ql[C][PACK ? 1 : NJ];
    float f[C];
#pragma unroll
    for (int n = 0; n < C; ++n) {
        const uint32_t rw = row + 16 * n, tk = rw / a.group, hq = kvh * a.group + rw % a.group;
        const bool there = rw < rows;
        const float *q = a.q + (size_t)(p.q0 + tk) * a.q_stride + (size_t)hq * D + h * (D / 4);
        float x[NJ][8], top = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if (there) __builtin_memcpy(x[j], q + 8 * j, 32);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i) x[j][i] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = __builtin_fmaxf(top, __builtin_fabsf(x[j][i]));
        }
        top = __builtin_fmaxf(top, xor_lanes(top, 16));
        top = __builtin_fmaxf(top, xor_lanes(top, 32));
        float sign;
        q_scale(a.scale, top, sign, f[n]);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = x[j][i] * sign;
                const _Float16 hv = (_Float16)y, lv = (_Float16)(y - (float)hv);
                qh[n][j][i] = low ? lv : hv;
                if (!PACK) ql[n][j][i] = lv;
            }
    }

    f32x4 acc[C][NJ][2];
    float m[C], l[C];
#pragma unroll
    for (int n = 0; n < C; ++n) {
#pragma unroll
        for (int g = 0; g < NJ; ++g) acc[n][g][0] = acc[n][g][1] = (f32x4)0.0f;
        m[n] = kNoMax;
        l[n] = 0.0f;
    }
    const Masks mk;
    const float minus_low = low ? -1.0f : 0.0f;
    for (; ti < t1; ti += 4) {
        const uint32_t tile = tile_of(ti), next = ti + 4 < t1 ? ti + 4 : ti;
        bool ok_next;
        const uint8_t *tn = tile_in<MODE>(a, s, kvh, tile_of(next), ok_next, next < T.head);
        f32x4 c[C][2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            // The lo halves' products, or packed the second half of the channels', apart: a score is rounded half as often at its
            // own size.  Of 1000 calls behind a prefix 0 and 8 were over 1e-6 off with and without (plain f32 operations 268), for
            // 2% of the time.  (kAll stays as it was.)
            constexpr bool kApart = MODE != kAll && (!PACK || D > 64);
            f32x4 rest[C];
#pragma unroll
            for (int n = 0; n < C; ++n) c[n][half] = rest[n] = (f32x4)0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const f16x8 kf = k_frag(k.code(half, j), k.scale(half, j), mk);
#pragma unroll
                for (int n = 0; n < C; ++n) {
                    if (PACK && kApart && j >= NJ / 2) rest[n] = mfma16(kf, qh[n][j], rest[n]);
                    else c[n][half] = mfma16(kf, qh[n][j], c[n][half]);
                    if (!PACK && !kApart) c[n][half] = mfma16(kf, ql[n][j], c[n][half]);
                    if (!PACK && kApart) rest[n] = mfma16(kf, ql[n][j], rest[n]);
                }
            }
            if (kApart)
#pragma unroll
                for (int n = 0; n < C; ++n) c[n][half] += rest[n];
        }
        k.load(tn, r, h);
        f16x8 pf[C], pg[C];
        const int32_t first = (int32_t)(tile * 32);
        // a tile that every row sees whole needs no mask
        const bool prefix = MODE == kTwo && ti < T.head;
        const bool whole = ok && (prefix ? first + 31 < (int32_t)a.first_key : first + 31 <= lo && (first >= low_all || first + 32 <= sink_key));
        if (!whole && !ok && lane == 0) ah_record(a.status, ((unsigned long long)s << 8) + AH_ERR_CACHE_RANGE);
#pragma unroll
        for (int n = 0; n < C; ++n) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = c[n][i >> 2][i & 3];
                x[i] = PACK ? y + ror8(y) : y;
            }
            if (!whole) {
                const int32_t top_key = ok ? C == 1 ? pos : row + 16 * n < rows ? position_of<MODE>(p, 0) : -1 : -1;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int32_t key = first + 16 * (i >> 2) + 4 * (int32_t)h + (i & 3);
                    const bool see = key <= top_key && (prefix ? key < (int32_t)a.first_key : key >= low_key || key < sink_key);
                    x[i] = see ? x[i] : -__builtin_inff();
                }
            }
            float top = x[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) top = __builtin_fmaxf(top, x[i]);
            top *= f[n];
            if (__builtin_amdgcn_ballot_w64(top > m[n] + kSlack) != 0ull) {
                top = __builtin_fmaxf(top, xor_lanes(top, 16));
                top = __builtin_fmaxf(top, xor_lanes(top, 32));
                const float up = __builtin_fmaxf(m[n], top), alpha = __builtin_amdgcn_exp2f(m[n] - up);
                m[n] = up;
                l[n] *= alpha;
#pragma unroll
                for (int g = 0; g < NJ; ++g) {
                    acc[n][g][0] *= alpha;
                    acc[n][g][1] *= alpha;
                }
            }
            const float base = kUp - m[n];
            float ls = 0.0f;  // the tile's weights, as in attn_tile_kernel
            f16x2 ph[4], pl[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * i], f[n], base)), e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[2 * i + 1], f[n], base));
                ls = i ? ls + e0 : e0;
                ls += e1;
                ph[i] = pack16(e0, e1);
                // what is left of p past its hi half; a packed column takes that or p itself
                const float k = PACK ? minus_low : -1.0f;
                pl[i] = pack16(__builtin_fmaf((float)ph[i][0], k, e0), __builtin_fmaf((float)ph[i][1], k, e1));
            }
            l[n] += ls;
            pg[n] = join8(pl[0], pl[1], pl[2], pl[3]);
            pf[n] = PACK ? pg[n] : join8(ph[0], ph[1], ph[2], ph[3]);
        }
#pragma unroll
        for (int g = 0; g < NJ; ++g) {
            f16x8 even, odd;
            v_frags(v.w[g >> 1][2 * (g & 1)], v.w[g >> 1][2 * (g & 1) + 1], v.d[g], mk, even, odd);
#pragma unroll
            for (int n = 0; n < C; ++n) {
                acc[n][g][0] = mfma16(even, pf[n], acc[n][g][0]);
                acc[n][g][1] = mfma16(odd, pf[n], acc[n][g][1]);
                if (!PACK) {
                    acc[n][g][0] = mfma16(even, pg[n], acc[n][g][0]);
                    acc[n][g][1] = mfma16(odd, pg[n], acc[n][g][1]);
                }
            }
        }
        v.load(tn, r, h);
        ok = ok_next;
    }

    // the lanes' sums of a column, then the four waves
#pragma unroll
    for (int n = 0; n < C; ++n) {
        l[n] += xor_lanes(l[n], 16);
        l[n] += xor_lanes(l[n], 32);
        if (h == 0 && !low) {
            red_m[wave * kRed + 16 * n + r] = m[n];
            red_l[wave * kRed + 16 * n + r] = l[n];
        }
#pragma unroll
        for (int g = 0; g < NJ; ++g) {
            float o[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = acc[n][g][0][i], d = acc[n][g][1][i];
                o[2 * i] = PACK ? e + ror8(e) : e;
                o[2 * i + 1] = PACK ? d + ror8(d) : d;
            }
            if (!low) __builtin_memcpy(red_o + (wave * kRed + 16 * n + r) * (D + 4) + 32 * g + 8 * h, o, 32);
        }
    }
    __syncthreads();
    const uint32_t pieces = MODE == kPrefix || MODE == kAfter ? 2 : T.count ? (T.count + chunk - 1) / chunk : 1;  // (2: a part of what a launch after this joins)
    const size_t all = (size_t)a.n_tok * a.n_heads;
    auto flat_of = [&](uint32_t rw) { return (size_t)(p.q0 + rw / a.group) * a.n_heads + kvh * a.group + rw % a.group; };
    auto out_of = [&](uint32_t rw) { return a.out + (size_t)(p.q0 + rw / a.group) * a.out_stride + (size_t)(kvh * a.group + rw % a.group) * D; };
    const uint32_t n_rows = last - row0 + 1;
    const __amdgpu_buffer_rsrc_t po = ah_rsrc(a.part_o, (uint32_t)(a.splits * all * D * 4)), pm = ah_rsrc(a.part_ml, (uint32_t)(a.splits * all * 8));
#pragma unroll
    for (int n = 0; n < C; ++n) {
        const uint32_t rr = 16 * n + (threadIdx.x >> 4);
        if (rr < n_rows) {
            float M = kNoMax, L = 0.0f, w4[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) M = __builtin_fmaxf(M, red_m[w * kRed + rr]);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                w4[w] = __builtin_amdgcn_exp2f(red_m[w * kRed + rr] - M);
                L += red_l[w * kRed + rr] * w4[w];
            }
            const float inv = pieces > 1 ? 1.0f : L > 0.0f || L != L ? 1.0f / L : 0.0f;
            const size_t at = split * all + flat_of(row0 + rr);
            for (uint32_t c = 4 * (threadIdx.x & 15); c < (uint32_t)D; c += 64) {
                f32x4 o = (f32x4)0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    f32x4 y;
                    __builtin_memcpy(&y, red_o + (w * kRed + rr) * (D + 4) + c, 16);
                    o += y * w4[w];
                }
                o *= inv;
                if (pieces > 1) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), po, (int)(4 * (at * D + c)), 0, kDevice);
                else __builtin_memcpy(out_of(row0 + rr) + c, &o, 16);
            }
            if (pieces > 1 && (threadIdx.x & 15) == 0)
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, (f32x2){M, L}), pm, (int)(8 * at), 0, kDevice);
        }
    }
    if (MODE == kPrefix || MODE == kAfter || pieces == 1) return;
    // The pieces are joined in groups of a.join and the groups then into one, each by the workgroup that arrives
    // last: it finds the others' partial results complete (device-scope stores, waited for before the count) and
    // reads them with device-scope loads.  One workgroup reads a piece's rows in about 0.1 us, so two levels of
    // sqrt(pieces) keep a long context's join near the time of a tile.  Counters are left at zero for the next call.
    constexpr uint32_t kLanes = D / 4;  // of a row, 16 bytes each
    auto arrive = [&](uint32_t *counter, uint32_t of) {  // whether this workgroup is the last of them
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) {
            const uint32_t n = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (n == of - 1) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            red_m[0] = __builtin_bit_cast(float, n);
        }
        __syncthreads();
        return __builtin_bit_cast(uint32_t, red_m[0]) == of - 1;
    };
    // pieces first, first + step, ..: to the output, or as one piece in the first one's place
    auto join = [&](uint32_t first, uint32_t step, uint32_t n, bool out) {
        for (uint32_t rr = threadIdx.x / kLanes; rr < n_rows; rr += 256 / kLanes) {
            const uint32_t gl = threadIdx.x % kLanes;
            const size_t flat = flat_of(row0 + rr);
            float M = kNoMax;
            for (uint32_t k = gl; k < n; k += kLanes)
                M = __builtin_fmaxf(M, __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(pm, (int)(8 * ((first + k * step) * all + flat)), 0, kDevice)));
#pragma unroll
            for (uint32_t o = 1; o < kLanes; o <<= 1) M = __builtin_fmaxf(M, xor_lanes(M, (int)o));
            float L = 0.0f;
            f32x4 sum = (f32x4)0.0f;
#pragma unroll 8
            for (uint32_t k = 0; k < n; ++k) {
                const size_t at = (first + k * step) * all + flat;
                const f32x2 ml = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(pm, (int)(8 * at), 0, kDevice));
                const f32x4 o = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(po, (int)(4 * (at * D + 4 * gl)), 0, kDevice));
                const float w = __builtin_amdgcn_exp2f(ml[0] - M);
                L += ml[1] * w;
                sum += o * w;
            }
            if (out) {
                sum *= L > 0.0f || L != L ? 1.0f / L : 0.0f;
                __builtin_memcpy(out_of(row0 + rr) + 4 * gl, &sum, 16);
            } else {
                const size_t at = first * all + flat;
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sum), po, (int)(4 * (at * D + 4 * gl)), 0, kDevice);
                if (gl == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, (f32x2){M, L}), pm, (int)(8 * at), 0, kDevice);
            }
        }
    };
    const uint32_t group = split / a.join, first = group * a.join, groups = (pieces + a.join - 1) / a.join;
    const uint32_t members = first + a.join <= pieces ? a.join : pieces - first;
    if (members > 1) {
        if (!arrive(a.count + units + unit * ((a.splits + a.join - 1) / a.join) + group, members)) return;
        join(first, 1, members, groups == 1);
    }
    if (groups > 1 && arrive(a.count + unit, groups)) join(0, a.join, groups, true);
}
template <int D, bool PACK, int MODE>
__global__ void __launch_bounds__(256, D == 256 ? 2 : D == 128 ? 3 : 4) attn_rows_kernel(AttnArgs a) {
    attn_rows<D, PACK, MODE>(a, blockIdx.x, gridDim.x);
}

// Chunks of tokens: 128 rows (token, head of the group) a workgroup, 32 a wave as the columns of 32x32 products,
// over 64 keys at a time.  The four waves turn a tile's codes into f16 in LDS together (once for 128 rows), in
// one of two buffers while they compute on the other: one barrier a tile.  A lane (c, h) = (lane & 31,
// lane >> 5) holds column c's scores of the tokens 8 b + 4 h + i; V's rows lie in LDS with the tokens in the
// order of those scores, so p stays in its lane here too.
//   LDS: K [64 tokens][D], V [D channels][64 tokens], rows 16 bytes longer than their values: 16 lanes' rows
//   start 4 banks apart, so a 16-byte read of the wave meets no conflict.
//   What bounds it: the matrix cores, which the two halves of q and of p use twice (8192 tokens, 12 heads of 128:
// 206 GFLOP of keys and values, 412 with the halves, in 393 us: 1050 TFLOP/s; a large f16 library product reaches
// 1068 on this card); half of their peak, the rest the vector work of the exponentials and the codes' conversion that the
// products do not cover (about 7 instructions hide behind one).  Heads of 64 have 11.7 vector instructions a product:
// while a CU works these take 56% of a SIMD's cycles and the products 35%.  Heads of 256 have 8.1, but one wave a SIMD to
// cover either: 43% and 40%.  For chunks of a few hundred tokens the unit's start and the join (1205 tokens of 5
// sequences over up to 6007 keys, heads of 64: 67 and 8 us under a tracer).  With the four waves
// each converting its own fragments (no LDS) 8192 tokens took 670 us.
template <int D> struct TileLds {
    static constexpr int kK = 2 * D + 16, kV = 144, kBytes = 64 * kK + D * kV;
};
template <int D, int MODE> AH_DEV void attn_tiles(const AttnArgs &a, uint32_t block, uint32_t grid) {
    constexpr int NK = D / 16, NN = D / 32, NU = D / 64;  // contraction steps of K q; channel blocks; 16-byte units
    constexpr int kAhead = D == 256 ? 3 : 1;  // more, where the registers do not cost a wave per SIMD
    typedef TileLds<D> Lds;
    extern __shared__ uint8_t tile_lds[];
    const uint32_t lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Pieces slowest; then the last rows first: with a causal mask they have the most keys.  Even sequences have `per`
    // units of 128 rows each.  Of uneven ones, sequence s has its units from start(s) on: floor of its first row / 128,
    // and one more for each sequence before it, so that few numbers have no rows.
    const uint32_t units = grid / a.splits, split = block / units;
    uint32_t unit = block - split * units;
    if (a.per && a.n_seq > 1) {  // workgroups go to the eight XCDs in turn: neighbouring units to one, whose L2 they share
        const uint32_t x = unit & 7, more = units & 7;
        unit = x * (units / 8) + (x < more ? x : more) + unit / 8;
    }
    const uint32_t at = units / a.c.n_kv - 1 - unit / a.c.n_kv, kvh = unit % a.c.n_kv;
    auto start = [&](uint32_t i) { return (uint32_t)((uint64_t)(uint32_t)a.q_start[i] * a.group >> 7) + i; };
    auto holds = [&](uint32_t i) {
        const Span p = span_of(a, i);
        return at >= start(i) && at - start(i) < (p.nq * a.group + 127) / 128;
    };
    const uint32_t s = a.per ? at / a.per : sequence_of(a, at, start, holds), rt = at - (a.per ? s * a.per : start(s));
    if (MODE != kPrefix && split == 0 && kvh == 0 && at < a.n_seq && threadIdx.x == 0 && span_in<MODE>(a, at, 0).bad)
        ah_record(a.status, ((unsigned long long)at << 8) + AH_ERR_CACHE_RANGE);
    const Span p = span_in<MODE>(a, s, kvh);
    const uint32_t rows = p.nq * a.group, row0 = rt * 128;
    if (rt >= (rows + 127) / 128 || (MODE == kAll && rows < a.least_rows)) return;
    const uint32_t last = row0 + 127 < rows ? row0 + 127 : rows - 1;
    const Tiles T = tiles_in<MODE>(a, position_of<MODE>(p, row0 / a.group), position_of<MODE>(p, last / a.group));
    const uint32_t chunk = piece_of(a, T), t0 = split * chunk, t1 = t0 + chunk < T.count ? t0 + chunk : T.count;
    if (MODE != kAfter && split > 0 && t0 >= T.count) return;
    // this wave's rows and the positions they span
    const uint32_t wrow = row0 + 32 * wave, row = wrow + c, tok = row / a.group, hq = kvh * a.group + row % a.group;
    const bool live = row < rows, any = wrow < rows;
    const uint32_t wlast = wrow + 31 < rows ? wrow + 31 : rows - 1;
    const int32_t lo = position_of<MODE>(p, wrow / a.group), hi = any ? position_of<MODE>(p, wlast / a.group) : -1;
    const int32_t pos = live ? position_of<MODE>(p, tok) : -1;
    // the keys below which the window hides one (for this row, and for the last of the rows), and the sinks
    const int32_t low_key = MODE == kAfter ? (int32_t)a.first_key : a.window ? pos - (int32_t)a.window + 1 : 0;
    const int32_t low_all = MODE == kAfter ? (int32_t)a.first_key : a.window ? hi - (int32_t)a.window + 1 : 0;
    const int32_t sink_key = (int32_t)a.sinks;
    auto tile_of = [&](uint32_t i) { return i < T.head ? i : T.tail + (i - T.head); };

    // A wave's share of a tile of 64 tokens: of its K and V units (1 KB of codes of 32 tokens), every fourth.
    constexpr int NS = D == 64 ? 1 : D / 128;  // of each kind
    const uint32_t kr = lane & 15, kq = lane >> 4;
    u32x4 kw[NS], vw[NS];
    uint32_t kd[NS];
    f16x8 vd[NS][2];
    auto unit_at = [&](int i) { return D == 64 ? wave & 1 : wave + 4 * i; };  // of 2 NU: tile * NU + chunk
    const bool do_k = D != 64 || wave < 2, do_v = D != 64 || wave >= 2;
    uint32_t bad = 0;  // of the tiles whose codes are on their way: bit 0 and 1
    auto fetch = [&](uint32_t ti) {
        bad = 0;
        const uint8_t *base[2];
#pragma unroll
        for (uint32_t j = 0; j < 2; ++j) {
            bool ok;
            base[j] = tile_at(a, a.table + (size_t)s * a.table_stride, kvh, tile_of(ti + j < t1 ? ti + j : t1 - 1), ok);
            if (!ok || ti + j >= t1) bad |= 1u << j;
            if (!ok && ti + j < t1 && lane == 0) ah_record(a.status, ((unsigned long long)s << 8) + AH_ERR_CACHE_RANGE);
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const uint32_t u = unit_at(i), ch = u % NU;
            const uint8_t *t = u < (uint32_t)NU ? base[0] : base[1];
            if (do_k) {
                const uint32_t blk = D == 64 ? kq >> 1 : D == 128 ? kq : 2 * kq + (ch & 1);
                __builtin_memcpy(&kw[i], t + ch * 1024 + (kr * 4 + kq) * 16, 16);
                __builtin_memcpy(&kd[i], t + 32 * D + (kr * (D / 32) + blk) * 4, 4);
            }
            if (do_v) {
                __builtin_memcpy(&vw[i], t + 16 * D + (ch * 16 + kr) * 64 + kq * 16, 16);
#pragma unroll
                for (int b = 0; b < 2; ++b) __builtin_memcpy(&vd[i][b], t + 34 * D + ((2 * ch + b) * 4 + kq) * 16, 16);
            }
        }
    };
    const Masks mk;
    // the share's conversions, in steps small enough to stand between two products
    constexpr int kSpreads = D == 64 ? 4 : 6 * NS;
    auto spread_k = [&](uint8_t *buf, int i, int w) {
        const uint32_t u = unit_at(i), ch = u % NU, t32 = 32 * (u / NU);
        const uint32_t half = D == 64 ? w >> 1 : D == 128 ? ch : ch >> 1;
        const uint32_t chan = D == 64 ? kq * 16 + 8 * (w & 1) : D == 128 ? kq * 32 + 8 * w : kq * 64 + (ch & 1) * 32 + 8 * w;
        const f16x8 v = k_frag(kw[i][w], pair_of(half ? kd[i] >> 16 : kd[i]), mk);
        __builtin_memcpy(buf + (t32 + 16 * half + kr) * Lds::kK + 2 * chan, &v, 16);
    };
    auto spread_v = [&](uint8_t *buf, int i, int b) {
        const uint32_t u = unit_at(i), ch = u % NU, t32 = 32 * (u / NU);
        f16x8 even, odd;
        v_frags(vw[i][2 * b], vw[i][2 * b + 1], vd[i][b], mk, even, odd);
        uint8_t *to = buf + 64 * Lds::kK + 2 * (16 * (2 * ch + b) + kr) * Lds::kV + 2 * (t32 + (kq & 1) * 8 + (kq >> 1) * 4);
        __builtin_memcpy(to, &even, 8);  // half-tile 0's four tokens, then half-tile 1's
        __builtin_memcpy(to + 32, reinterpret_cast<const char *>(&even) + 8, 8);
        __builtin_memcpy(to + Lds::kV, &odd, 8);
        __builtin_memcpy(to + Lds::kV + 32, reinterpret_cast<const char *>(&odd) + 8, 8);
    };
    auto spread_step = [&](uint8_t *buf, int n) {
        if (D == 64) {
            if (do_k) spread_k(buf, 0, n);
            else if (n < 2) spread_v(buf, 0, n);
        } else {
            const int i = n / 6, k = n % 6;
            if (k < 4) spread_k(buf, i, k);
            else spread_v(buf, i, k - 4);
        }
    };
    auto spread = [&](uint8_t *buf) {
#pragma unroll
        for (int n = 0; n < kSpreads; ++n) spread_step(buf, n);
    };

    f32x16 acc[NN];
#pragma unroll
    for (int n = 0; n < NN; ++n) acc[n] = (f32x16)0.0f;
    float m = kNoMax, l = 0.0f;
    if (t0 < t1) {
        fetch(t0);
        f16x8 qh[NK], ql[NK];
        float f;
        {
            const float *q = a.q + (size_t)(p.q0 + (live ? tok : 0)) * a.q_stride + (size_t)(live ? hq : 0) * D + 8 * h;
            float x[NK][8], top = 0.0f, up;
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                __builtin_memcpy(x[k], q + 16 * k, 32);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[k][i] = live ? x[k][i] : 0.0f;
                    top = __builtin_fmaxf(top, __builtin_fabsf(x[k][i]));
                }
            }
            q_scale(a.scale, __builtin_fmaxf(top, xor_lanes(top, 32)), up, f);
#pragma unroll
            for (int k = 0; k < NK; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float y = x[k][i] * up;
                    const _Float16 hv = (_Float16)y;
                    qh[k][i] = hv;
                    ql[k][i] = (_Float16)(y - (float)hv);
                }
        }
        uint32_t bad_now = bad;
        spread(tile_lds);
        if (t0 + 2 < t1) fetch(t0 + 2);
        __syncthreads();
        for (uint32_t ti = t0, at = 0; ti < t1; ti += 2, at ^= 1) {
            const uint8_t *buf = tile_lds + at * Lds::kBytes;
            const int32_t first0 = (int32_t)(32 * tile_of(ti)), first1 = (int32_t)(32 * tile_of(ti + 1 < t1 ? ti + 1 : ti));
            // a wave whose rows all stand before the tile (a causal mask) only helps to load
            const bool work = any && (first0 <= hi || first1 <= hi);
            uint8_t *other = tile_lds + (at ^ 1) * Lds::kBytes;
            if (work) {
                // Two halves of 32 keys, their matrix and vector work side by side: the exponentials of one half
                // stand between the products K q of the other, those of the other between the products P V of the
                // first, and the next tile's conversion between the last products.  (Past the last tile that
                // converts what is left in the registers into a buffer that nobody reads.)
                f32x16 sc[2];
                // A half's weights are summed alone and added to l once.  Added one by one, those below the last place of a sum that
                // one key rules are each lost or rounded up: 40037 keys of 2^-20 to 2^-24 of the first, 7e-5 of the outputs.
                float ls;
                uint32_t ph[8], pl[8], pn[8], pm[8];  // f16 pairs
                auto k_read = [&](int j, int k) {
                    f16x8 v;
                    __builtin_memcpy(&v, buf + (32 * j + c) * Lds::kK + 2 * (16 * k + 8 * h), 16);
                    return v;
                };
                auto v_read = [&](int g, int n) {
                    f16x8 v;
                    __builtin_memcpy(&v, buf + 64 * Lds::kK + (32 * n + c) * Lds::kV + 2 * (16 * g + 8 * h), 16);
                    return v;
                };
                auto mask = [&](int j) {
                    const int32_t first = j ? first1 : first0;
                    const bool ok = !(bad_now >> j & 1u);
                    if (ok && first + 31 <= lo && (first >= low_all || first + 32 <= sink_key)) return;
                    const int32_t top_key = ok ? pos : -1;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int32_t key = first + 8 * (i >> 2) + 4 * (int32_t)h + (i & 3);
                        const bool see = key <= top_key && (key >= low_key || key < sink_key);
                        sc[j][i] = see ? sc[j][i] : -__builtin_inff();
                    }
                };
                auto follow = [&](int j) {  // the running maximum
                    float top = sc[j][0];
#pragma unroll
                    for (int i = 1; i < 16; ++i) top = __builtin_fmaxf(top, sc[j][i]);
                    top *= f;
                    if (__builtin_amdgcn_ballot_w64(top > m + kSlack) == 0ull) return;
                    const float up = __builtin_fmaxf(m, __builtin_fmaxf(top, xor_lanes(top, 32))), alpha = __builtin_amdgcn_exp2f(m - up);
                    m = up;
                    l *= alpha;
#pragma unroll
                    for (int n = 0; n < NN; ++n) acc[n] *= alpha;
                };
                // (the empty asm keeps a pair between the products it is written between: the compiler would gather
                // all of them where they are used)
                auto exp_pair = [&](int j, int i, float base, uint32_t &hi2, uint32_t &lo2) {
                    const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j][2 * i], f, base));
                    const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j][2 * i + 1], f, base));
                    ls = i ? ls + e0 : e0;
                    ls += e1;
                    const f16x2 t = pack16(e0, e1);
                    hi2 = __builtin_bit_cast(uint32_t, t);
                    lo2 = __builtin_bit_cast(uint32_t, pack16(__builtin_fmaf((float)t[0], -1.0f, e0), __builtin_fmaf((float)t[1], -1.0f, e1)));
                    __asm__ volatile("" : "+v"(hi2), "+v"(lo2), "+v"(ls));
                };
                auto frag = [](const uint32_t *v) { return __builtin_bit_cast(f16x8, (u32x4){v[0], v[1], v[2], v[3]}); };
                // One stream of fragments from LDS, read kAhead steps before its two products: the halves' K rows, then
                // the channels of V for 16 tokens after 16.
                constexpr int kK = 2 * NK, kAll = kK + 4 * NN, kRing = kAhead + 1;
                f16x8 ring[kRing];
                auto read = [&](int i) {
                    if (i < kK) ring[i % kRing] = k_read(i / NK, i % NK);
                    else if (i < kAll) ring[i % kRing] = v_read((i - kK) / NN, (i - kK) % NN);
                };
#pragma unroll
                for (int i = 0; i < kAhead; ++i) read(i);
                sc[0] = sc[1] = (f32x16)0.0f;
#pragma unroll
                for (int k = 0; k < NK; ++k) {
                    read(k + kAhead);
                    sc[0] = mfma32(ring[k % kRing], qh[k], sc[0]);
                    sc[0] = mfma32(ring[k % kRing], ql[k], sc[0]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                mask(0);
                follow(0);
                const float base0 = kUp - m;
#pragma unroll
                for (int k = 0; k < NK; ++k) {
                    read(NK + k + kAhead);
                    sc[1] = mfma32(ring[(NK + k) % kRing], qh[k], sc[1]);
                    sc[1] = mfma32(ring[(NK + k) % kRing], ql[k], sc[1]);
#pragma unroll
                    for (int i = 8 * k / NK; i < 8 * (k + 1) / NK; ++i) exp_pair(0, i, base0, ph[i], pl[i]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                l += ls;
                mask(1);
                // p of the first half was taken at the maximum so far: a new one scales its product with the rest
                f16x8 pf[2], pg[2];
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    pf[g] = frag(ph + 4 * g);
                    pg[g] = frag(pl + 4 * g);
                }
                float top1 = sc[1][0];
#pragma unroll
                for (int i = 1; i < 16; ++i) top1 = __builtin_fmaxf(top1, sc[1][i]);
                top1 *= f;
                const bool moves = __builtin_amdgcn_ballot_w64(top1 > m + kSlack) != 0ull;
                float alpha = 1.0f;
                if (moves) {
                    const float up = __builtin_fmaxf(m, __builtin_fmaxf(top1, xor_lanes(top1, 32)));
                    alpha = __builtin_amdgcn_exp2f(m - up);
                    m = up;
                    l *= alpha;
                }
                const float base1 = kUp - m;
#pragma unroll
                for (int q = 0; q < 2 * NN; ++q) {
                    const int g = q / NN, n = q % NN;
                    read(kK + q + kAhead);
                    acc[n] = mfma32(ring[(kK + q) % kRing], pf[g], acc[n]);
                    acc[n] = mfma32(ring[(kK + q) % kRing], pg[g], acc[n]);
#pragma unroll
                    for (int i = 8 * q / (2 * NN); i < 8 * (q + 1) / (2 * NN); ++i) exp_pair(1, i, base1, pn[i], pm[i]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                l += ls;
                if (moves) {
#pragma unroll
                    for (int n = 0; n < NN; ++n) acc[n] *= alpha;
                }
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    pf[g] = frag(pn + 4 * g);
                    pg[g] = frag(pm + 4 * g);
                }
#pragma unroll
                for (int q = 0; q < 2 * NN; ++q) {
                    const int g = q / NN, n = q % NN;
                    read(kK + 2 * NN + q + kAhead);
                    acc[n] = mfma32(ring[(kK + 2 * NN + q) % kRing], pf[g], acc[n]);
                    acc[n] = mfma32(ring[(kK + 2 * NN + q) % kRing], pg[g], acc[n]);
#pragma unroll
                    for (int i = kSpreads * q / (2 * NN); i < kSpreads * (q + 1) / (2 * NN); ++i) spread_step(other, i);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                spread(other);
            }
            const uint32_t bad_next = bad;
            if (ti + 4 < t1) fetch(ti + 4);
            bad_now = bad_next;
            __syncthreads();
        }
    }
    l += xor_lanes(l, 32);
    const uint32_t pieces = MODE == kAll && D == 64 && a.join && T.count ? (T.count + chunk - 1) / chunk : 1;
    if (D == 64 && pieces > 1) {
        // Few pieces are joined by the unit's workgroup that arrives last (as in attn_rows_kernel), each lane its own place
        // of all of them, in their order whichever is last: a launch less, but a memory round trip for each piece.
        // 2048 tokens in 2 pieces 57 -> 46 us, 512 over 4096 keys in 6 41 -> 46.  Larger heads have no registers for it:
        // of 128, 3 to 5 us slower in every call, of 256 in 2 pieces 84 -> 89.
        const size_t flat = (size_t)(p.q0 + tok) * a.n_heads + hq, all = (size_t)a.n_tok * a.n_heads;
        const __amdgpu_buffer_rsrc_t po = ah_rsrc(a.part_o, (uint32_t)(a.splits * all * D * 4)), pm = ah_rsrc(a.part_ml, (uint32_t)(a.splits * all * 8));
        if (live) {
            const size_t at = split * all + flat;
#pragma unroll
            for (int n = 0; n < NN; ++n)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const f32x4 o = {acc[n][4 * b], acc[n][4 * b + 1], acc[n][4 * b + 2], acc[n][4 * b + 3]};
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), po, (int)(4 * (at * D + 32 * n + 8 * b + 4 * h)), 0, kDevice);
                }
            if (h == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, (f32x2){m, l}), pm, (int)(8 * at), 0, kDevice);
        }
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        uint32_t *turn = reinterpret_cast<uint32_t *>(tile_lds);
        if (threadIdx.x == 0) {
            uint32_t *counter = a.count + (block - split * units);
            const uint32_t n = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (n == pieces - 1) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            *turn = n;
        }
        __syncthreads();
        if (*turn != pieces - 1 || !live) return;
        m = kNoMax;
        for (uint32_t k = 0; k < pieces; ++k)
            m = __builtin_fmaxf(m, __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(pm, (int)(8 * (k * all + flat)), 0, kDevice)));
        l = 0.0f;
#pragma unroll
        for (int n = 0; n < NN; ++n) acc[n] = (f32x16)0.0f;
#pragma unroll 1
        for (uint32_t k = 0; k < pieces; ++k) {
            const size_t at = k * all + flat;
            const f32x2 ml = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(pm, (int)(8 * at), 0, kDevice));
            const float w = __builtin_amdgcn_exp2f(ml[0] - m);
            l += ml[1] * w;
#pragma unroll
            for (int n = 0; n < NN; ++n)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const f32x4 o = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(po, (int)(4 * (at * D + 32 * n + 8 * b + 4 * h)), 0, kDevice));
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[n][4 * b + i] += o[i] * w;
                }
        }
    }
    if (!live) return;
    const size_t flat = (size_t)(p.q0 + tok) * a.n_heads + hq, all = (size_t)a.n_tok * a.n_heads;
    const bool part = MODE != kAll || (a.splits > 1 && !(D == 64 && a.join));
    const float inv = part ? 1.0f : l > 0.0f || l != l ? 1.0f / l : 0.0f;
    float *dst = part ? a.part_o + (split * all + flat) * D : a.out + (size_t)(p.q0 + tok) * a.out_stride + (size_t)hq * D;
#pragma unroll
    for (int n = 0; n < NN; ++n)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const f32x4 o = (f32x4){acc[n][4 * b], acc[n][4 * b + 1], acc[n][4 * b + 2], acc[n][4 * b + 3]} * inv;
            __builtin_memcpy(dst + 32 * n + 8 * b + 4 * h, &o, 16);
        }
    if (part && h == 0) {
        float *ml = a.part_ml + 2 * (split * all + flat);
        ml[0] = m;
        ml[1] = l;
    }
}

template <int D, int MODE> __global__ void __launch_bounds__(256, D == 64 ? 3 : D == 128 ? 2 : 1) attn_tile_kernel(AttnArgs a) {
    attn_tiles<D, MODE>(a, blockIdx.x, gridDim.x);
}
// A common prefix, by 16, 32 or 128 rows of the whole batch, and beside it in the same launch what each sequence has after it, by 8
// or 16: the one alone leaves CUs without work at its end, and a launch more costs 5 us.  What bounds the units of 16 and 32 is
// the vector work of converting codes and of the exponentials: of 12 heads of 128 over 2 of 64 sequences behind 16384 keys, 6.4
// MB and 6.6 GFLOP, 13 with the halves, in 28 us (by 16 rows 31, by 128 35): vector work takes 57% of a SIMD's cycles while a
// CU works, products 24%.  By 128 rows (16 sequences of 25 to 49 tokens behind 8003 keys, 30 GFLOP, 60 with the halves, 82 us)
// 42% and 39%.
template <int D, int ROWS, bool PACK>
__global__ void __launch_bounds__(256, ROWS == 16 ? (D == 256 ? 2 : D == 128 ? 3 : 4) : D == 64 ? 3 : D == 128 ? 2 : 1) attn_shared_kernel(AttnArgs prefix, AttnArgs after) {
    if (blockIdx.x >= prefix.grid) attn_rows<D, PACK, kAfter>(after, blockIdx.x - prefix.grid, after.grid);
    else if (ROWS == 128) attn_tiles<D, kPrefix>(prefix, blockIdx.x, prefix.grid);
    else attn_rows<D, false, kPrefix, ROWS == 32 ? 2 : 1>(prefix, blockIdx.x, prefix.grid);
}

// Joins the pieces of attn_tile_kernel's contexts: a wave takes 256 / D heads of a token, four channels a lane.  A piece
// past a row's keys was never written; which those are follows from the same tiles_of.  Bound by the partial results'
// bytes.
template <int D>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a) {
    constexpr uint32_t kLanes = D / 4, kHeads = 64 / kLanes;
    const uint32_t lane = threadIdx.x & 63, it = 4 * blockIdx.x + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t per = (a.n_heads + kHeads - 1) / kHeads, tok = it / per, head = (it - tok * per) * kHeads + lane / kLanes, g = a.group;
    if (tok >= a.n_tok) return;
    auto start = [&](uint32_t i) { return (uint32_t)a.q_start[i]; };
    auto holds = [&](uint32_t i) {
        const Span p = span_of(a, i);
        return tok >= p.q0 && tok - p.q0 < p.nq;
    };
    const uint32_t s = sequence_of(a, tok, start, holds);
    const Span p = span_of(a, s);
    if (tok < p.q0 || tok - p.q0 >= p.nq || p.nq * g < a.least_rows || head >= a.n_heads) return;
    const uint32_t i = tok - p.q0;
    const uint32_t row = i * g + head % g, row0 = row - row % a.rows;
    const uint32_t last = row0 + a.rows - 1 < p.nq * g ? row0 + a.rows - 1 : p.nq * g - 1;
    const int32_t pos0 = p.ctx - (int32_t)p.nq;
    const Tiles T = tiles_of(a, pos0 + (int32_t)(row0 / g), pos0 + (int32_t)(last / g));
    const uint32_t chunk = piece_of(a, T), pieces = T.count ? (T.count + chunk - 1) / chunk : 1, c = 4 * (lane % kLanes);
    const size_t all = (size_t)a.n_tok * a.n_heads, flat = (size_t)tok * a.n_heads + head;
    float M = kNoMax, L = 0.0f;
#pragma unroll 4
    for (uint32_t k = 0; k < pieces; ++k) M = __builtin_fmaxf(M, a.part_ml[2 * (k * all + flat)]);
    f32x4 sum = (f32x4)0.0f;
#pragma unroll 4
    for (uint32_t k = 0; k < pieces; ++k) {
        f32x2 ml;
        f32x4 o;
        __builtin_memcpy(&ml, a.part_ml + 2 * (k * all + flat), 8);
        __builtin_memcpy(&o, a.part_o + (k * all + flat) * D + c, 16);
        const float w = __builtin_amdgcn_exp2f(ml[0] - M);
        L += ml[1] * w;
        sum += o * w;
    }
    sum *= L > 0.0f || L != L ? 1.0f / L : 0.0f;
    __builtin_memcpy(a.out + (size_t)tok * a.out_stride + (size_t)head * D + c, &sum, 16);
}

// Joins what kPrefix and kAfter leave, a.splits pieces of every token of a sequence: a workgroup takes 256 / D heads of a token,
// each of its waves every fourth piece, eight of them on their way, and they meet in LDS.  Bound by the launch and the partial
// results' bytes: 64 tokens of 12 heads of 128 4.7 us, 608 tokens, 37 MB, 11 us.
template <int D>
__global__ void __launch_bounds__(256) attn_meet_kernel(AttnArgs a) {
    constexpr uint32_t kLanes = D / 4, kHeads = 64 / kLanes, kAhead = 8;
    __shared__ f32x4 red[4][64];
    __shared__ f32x2 red_ml[4][64];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t per = (a.n_heads + kHeads - 1) / kHeads, tok = blockIdx.x / per, head = (blockIdx.x - tok * per) * kHeads + lane / kLanes;
    auto start = [&](uint32_t i) { return (uint32_t)a.q_start[i]; };
    auto holds = [&](uint32_t i) {
        const Span p = span_in<kAfter>(a, i, 0);
        return tok >= p.q0 && tok - p.q0 < p.nq;
    };
    const size_t all = (size_t)a.n_tok * a.n_heads, flat = (size_t)tok * a.n_heads + (head < a.n_heads ? head : 0);
    const uint32_t c = 4 * (lane % kLanes);
    float M = kNoMax, L = 0.0f;
    f32x4 sum = (f32x4)0.0f;
    for (uint32_t k0 = wave; k0 < a.splits; k0 += 4 * kAhead) {
        f32x2 ml[kAhead];
        f32x4 o[kAhead];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            const uint32_t k = k0 + 4 * j < a.splits ? k0 + 4 * j : k0;
            __builtin_memcpy(&ml[j], a.part_ml + 2 * (k * all + flat), 8);
            __builtin_memcpy(&o[j], a.part_o + (k * all + flat) * D + c, 16);
        }
        float top = M;
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) top = __builtin_fmaxf(top, ml[j][0]);
        const float keep = __builtin_amdgcn_exp2f(M - top);
        L *= keep;
        sum *= keep;
        M = top;
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            const float w = k0 + 4 * j < a.splits ? __builtin_amdgcn_exp2f(ml[j][0] - M) : 0.0f;
            if (k0 + 4 * j < a.splits) {
                L += ml[j][1] * w;
                sum += o[j] * w;
            }
        }
    }
    red[wave][lane] = sum;
    red_ml[wave][lane] = (f32x2){M, L};
    const Span p = span_in<kAfter>(a, sequence_of(a, tok, start, holds), 0);
    __syncthreads();
    if (wave != 0 || tok < p.q0 || tok - p.q0 >= p.nq || head >= a.n_heads) return;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = __builtin_fmaxf(M, red_ml[w][lane][0]);
    L = 0.0f;
    sum = (f32x4)0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float x = __builtin_amdgcn_exp2f(red_ml[w][lane][0] - M);
        L += red_ml[w][lane][1] * x;
        sum += red[w][lane] * x;
    }
    sum *= L > 0.0f || L != L ? 1.0f / L : 0.0f;
    __builtin_memcpy(a.out + (size_t)tok * a.out_stride + (size_t)head * D + c, &sum, 16);
}

template <int D, int C = 1> constexpr size_t attn_lds() { return C * (4 * 16 * (D + 4) + 128) * sizeof(float); }

template <int D, int MODE> void launch_rows(const AttnArgs &a, hipStream_t stream) {
    if (a.rows == 16) hipLaunchKernelGGL((attn_rows_kernel<D, false, MODE>), dim3(a.grid), dim3(256), attn_lds<D>(), stream, a);
    else hipLaunchKernelGGL((attn_rows_kernel<D, true, MODE>), dim3(a.grid), dim3(256), attn_lds<D>(), stream, a);
}
template <int D, int MODE> void launch_tiles(const AttnArgs &a, hipStream_t stream) {
    hipLaunchKernelGGL((attn_tile_kernel<D, MODE>), dim3(a.grid), dim3(256), 2 * TileLds<D>::kBytes, stream, a);
}
template <int D> uint32_t join_grid(const AttnArgs &a) { return (a.n_tok * ((a.n_heads + 256 / D - 1) / (256 / D)) + 3) / 4; }

template <int D> hipError_t launch(const AttnArgs &a, hipStream_t stream) {
    if (a.rows != 128) {
        launch_rows<D, kAll>(a, stream);
        return hipGetLastError();
    }
    launch_tiles<D, kAll>(a, stream);
    if (a.splits > 1 && !a.join) hipLaunchKernelGGL(attn_join_kernel<D>, dim3(join_grid<D>(a)), dim3(256), 0, stream, a);
    return hipGetLastError();
}
template <int D, int ROWS> constexpr size_t shared_lds() {
    return ROWS == 128 ? (2 * TileLds<D>::kBytes > attn_lds<D>() ? 2 * TileLds<D>::kBytes : attn_lds<D>()) : attn_lds<D, ROWS / 16>();
}
template <int D, int ROWS> void launch_both(const AttnArgs &prefix, const AttnArgs &after, hipStream_t stream) {
    const dim3 grid(prefix.grid + after.grid);
    if (after.rows == 16) hipLaunchKernelGGL((attn_shared_kernel<D, ROWS, false>), grid, dim3(256), (shared_lds<D, ROWS>()), stream, prefix, after);
    else hipLaunchKernelGGL((attn_shared_kernel<D, ROWS, true>), grid, dim3(256), (shared_lds<D, ROWS>()), stream, prefix, after);
}
template <int D> hipError_t launch_shared(const AttnArgs &prefix, const AttnArgs &after, const AttnArgs &both, hipStream_t stream) {
    if (after.rows == 128) {
        launch_tiles<D, kPrefix>(prefix, stream);
        launch_tiles<D, kAfter>(after, stream);
    } else if (prefix.rows == 128) {
        launch_both<D, 128>(prefix, after, stream);
    } else if (D == 128 && prefix.rows == 32) {
        launch_both<D, D == 128 ? 32 : 16>(prefix, after, stream);
    } else {
        launch_both<D, 16>(prefix, after, stream);
    }
    hipLaunchKernelGGL(attn_meet_kernel<D>, dim3(both.n_tok * ((both.n_heads + 256 / D - 1) / (256 / D))), dim3(256), 0, stream, both);
    return hipGetLastError();
}
template <int D> hipError_t launch_some(const AttnArgs &a, hipStream_t stream) {
    if (D < 256 && a.first_table) launch_rows<D, D < 256 ? kTwo : kBlocks>(a, stream);
    else launch_rows<D, kBlocks>(a, stream);
    return hipGetLastError();
}

template <class K> hipError_t allow_lds(K *k, size_t bytes) {
    return hipFuncSetAttribute(reinterpret_cast<const void *>(k), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}
template <int MODE> hipError_t allow_rows() {
    const hipError_t e = allow_lds(attn_rows_kernel<256, false, MODE>, attn_lds<256>());
    return e != hipSuccess ? e : allow_lds(attn_rows_kernel<256, true, MODE>, attn_lds<256>());
}
template <int MODE> hipError_t allow_tiles() {
    const hipError_t e = allow_lds(attn_tile_kernel<128, MODE>, 2 * TileLds<128>::kBytes);
    return e != hipSuccess ? e : allow_lds(attn_tile_kernel<256, MODE>, 2 * TileLds<256>::kBytes);
}

} // namespace

hipError_t ah_launch_attn(const AttnArgs &a, hipStream_t stream) {
    return a.c.dim == 64 ? launch<64>(a, stream) : a.c.dim == 128 ? launch<128>(a, stream) : launch<256>(a, stream);
}
hipError_t ah_launch_attn_shared(const AttnArgs &p, const AttnArgs &s, const AttnArgs &both, hipStream_t stream) {
    return p.c.dim == 64 ? launch_shared<64>(p, s, both, stream) : p.c.dim == 128 ? launch_shared<128>(p, s, both, stream) : launch_shared<256>(p, s, both, stream);
}
hipError_t ah_launch_attn_some(const AttnArgs &a, hipStream_t stream) {
    return a.c.dim == 64 ? launch_some<64>(a, stream) : a.c.dim == 128 ? launch_some<128>(a, stream) : launch_some<256>(a, stream);
}

template <int D, int ROWS> hipError_t allow_both() {
    const hipError_t e = allow_lds(attn_shared_kernel<D, ROWS, false>, shared_lds<D, ROWS>());
    return e != hipSuccess ? e : allow_lds(attn_shared_kernel<D, ROWS, true>, shared_lds<D, ROWS>());
}
template <int D> hipError_t allow_shared() {
    hipError_t e = allow_both<D, 16>();
    if (e == hipSuccess && D == 128) e = allow_both<D, D == 128 ? 32 : 16>();
    return e != hipSuccess ? e : allow_both<D, 128>();
}

hipError_t ah_attn_init_attrs() {
    hipError_t e = allow_rows<kAll>();
    if (e == hipSuccess) e = allow_rows<kBlocks>();
    if (e == hipSuccess) e = allow_tiles<kAll>();
    if (e == hipSuccess) e = allow_tiles<kPrefix>();
    if (e == hipSuccess) e = allow_tiles<kAfter>();
    if (e == hipSuccess) e = allow_shared<64>();
    if (e == hipSuccess) e = allow_shared<128>();
    return e != hipSuccess ? e : allow_shared<256>();
}
