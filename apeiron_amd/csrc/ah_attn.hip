// ah_attn.hip -- attention over the paged 4-bit cache (layout: ah_kv4.h).
//
// o = sum_t softmax_t(scale q . k_t) v_t over the keys t a query at position p sees: t <= p and, with a
// window, t > p - window or t < sinks.  One pass over the cache with the running maximum and sum of the
// softmax in f32, K q and P V on the f16 matrix cores.  The cache's values are exact in f16; q and p are
// carried as f16 pairs hi + lo (22 bits), each pair's two products summed in the f32 accumulator, so the
// result is that of f32 arithmetic.
#include "ah_kv4.h"

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNoMax = -3.402823466e38f;  // below every finite score
// The running maximum follows the scores only when one passes it by more than this (in powers of two):
// then p <= 2^kSlack, and a rescale of the accumulators is rare after the first tiles.
constexpr float kSlack = 4.0f;
// p is kept times 2^kUp: a weight of 2^-13 of the largest still has its 22 bits in two f16 halves (f16's
// subnormals end at 2^-24), and the largest, 2^(kUp + kSlack), is a finite f16.
constexpr float kUp = 9.0f;

AH_DEV f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// 8 codes of a dword as f16 values: low nibbles of its half-words, then the next ones.  1024 + c has c in
// its lowest mantissa bits; (1024 + c) - 1032 and the product by d are exact.
AH_DEV f16x2 nibbles(uint32_t w, uint32_t at) {
    return __builtin_bit_cast(f16x2, ((w >> at) & 0x000F000Fu) | 0x64006400u) - (f16x2)((_Float16)1032.0f);
}
AH_DEV f16x2 pair_of(uint16_t h) { return (f16x2)(__builtin_bit_cast(_Float16, h)); }
AH_DEV f16x8 k_frag(uint32_t w, f16x2 d) {
    f16x8 f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const f16x2 v = nibbles(w, 4 * k) * d;
        f[2 * k] = v[0];
        f[2 * k + 1] = v[1];
    }
    return f;
}
// The tokens' values of the even (at = 0) or odd (at = 4) channel of a pair: two dwords, four tokens each.
AH_DEV f16x8 v_frag(uint32_t w0, uint32_t w1, uint32_t at, f16x8 d) {
    f16x8 f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const f16x2 v = nibbles(k < 2 ? w0 : w1, 8 * (k & 1) + at) * (f16x2){d[2 * k], d[2 * k + 1]};
        f[2 * k] = v[0];
        f[2 * k + 1] = v[1];
    }
    return f;
}

AH_DEV float xor_lanes(float v, int mask) { return __shfl_xor(v, mask, 64); }

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

// Tiles of a piece: the planned chunk, or more where a context is longer than the caller's bound.
AH_DEV uint32_t piece_of(const AttnArgs &a, const Tiles &t) {
    const uint32_t need = (t.count + a.splits - 1) / a.splits;
    return need > a.chunk ? need : a.chunk;
}

// Sixteen rows (token, head of the group) a workgroup, as the columns of the products: every wave takes
// tiles of 32 tokens of the workgroup's piece of the context, each with its own running maximum, and the
// four meet in LDS.  A lane (r, h) holds the scores of column r, tokens 4 h + i of both half-tiles.
template <int D>
__global__ void __launch_bounds__(256) attn_rows_kernel(AttnArgs a) {
    constexpr int NJ = D / 32;  // contraction steps of K q, and blocks of channels
    extern __shared__ float lds[];
    float *red_o = lds;                   // [4][16][D + 4]
    float *red_m = lds + 4 * 16 * (D + 4);  // [4][16], then the sums
    float *red_l = red_m + 64;
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, h = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t split = blockIdx.x % a.splits, rest = blockIdx.x / a.splits, kvh = rest % a.c.n_kv, rt = rest / a.c.n_kv;
    const uint32_t s = blockIdx.y;
    const Span p = span_of(a, s);
    if (p.bad && blockIdx.x == 0 && threadIdx.x == 0) ah_record(a.status, ((unsigned long long)s << 8) + AH_ERR_CACHE_RANGE);
    const uint32_t rows = p.nq * a.group, row0 = rt * 16;
    if (row0 >= rows) return;
    const uint32_t row = row0 + r, tok = row / a.group, hq = kvh * a.group + row % a.group;
    const bool live = row < rows;
    const int32_t pos0 = p.ctx - (int32_t)p.nq;
    const uint32_t last = row0 + 15 < rows ? row0 + 15 : rows - 1;
    const int32_t lo = pos0 + (int32_t)(row0 / a.group), hi = pos0 + (int32_t)(last / a.group);
    const int32_t pos = live ? pos0 + (int32_t)tok : -1;
    const Tiles T = tiles_of(a, lo, hi);
    const uint32_t chunk = piece_of(a, T), t0 = split * chunk, t1 = t0 + chunk < T.count ? t0 + chunk : T.count;
    if (split > 0 && t0 >= T.count) return;

    // q, scaled by a power of two so that its largest magnitude is in [2^13, 2^14), as hi + lo
    f16x8 qh[NJ], ql[NJ];
    float f;
    {
        const float *q = a.q + (size_t)(p.q0 + tok) * a.q_stride + (size_t)hq * D + h * (D / 4);
        float x[NJ][8], top = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if (live) __builtin_memcpy(x[j], q + 8 * j, 32);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i) x[j][i] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = __builtin_fmaxf(top, __builtin_fabsf(x[j][i]));
        }
        top = __builtin_fmaxf(top, xor_lanes(top, 16));
        top = __builtin_fmaxf(top, xor_lanes(top, 32));
        int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;  // top in [2^e, 2^(e+1))
        e = e < -100 ? -100 : e > 127 ? 127 : e;
        const float up = __builtin_ldexpf(1.0f, 13 - e);
        f = a.scale * kLog2e * __builtin_ldexpf(1.0f, e - 13);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = x[j][i] * up;
                const _Float16 hv = (_Float16)v;
                qh[j][i] = hv;
                ql[j][i] = (_Float16)(v - (float)hv);
            }
    }

    f32x4 acc[NJ][2];
#pragma unroll
    for (int g = 0; g < NJ; ++g) acc[g][0] = acc[g][1] = (f32x4)0.0f;
    float m = kNoMax, l = 0.0f;
    for (uint32_t ti = t0 + wave; ti < t1; ti += 4) {
        const uint32_t tile = ti < T.head ? ti : T.tail + (ti - T.head);
        const uint32_t pi = tile >> (a.c.page_shift - 5);
        const uint32_t page = (uint32_t)a.table[(size_t)s * a.table_stride + pi];
        if (page >= a.c.n_pages) {
            if (lane == 0) ah_record(a.status, ((unsigned long long)s << 8) + AH_ERR_CACHE_RANGE);
            continue;
        }
        const uint8_t *t = a.c.base + kv4_tile(a.c, page, kvh, tile & ((1u << (a.c.page_shift - 5)) - 1));
        // K: per half-tile NJ dwords of codes, and the scales of this lane's channels
        uint32_t kc[2][NJ];
        uint16_t kd[2][D == 256 ? 2 : 1];
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
            u32x4 w;
            __builtin_memcpy(&w, t + c * 1024 + (r * 4 + h) * 16, 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (D == 64) kc[i >> 1][i & 1] = w[i];
                else kc[c / (D / 128)][4 * (c % (D / 128)) + i] = w[i];
            }
        }
        {
            const uint8_t *sc = t + 32 * D + r * (D / 32) * 4;
#pragma unroll
            for (int b = 0; b < (D == 256 ? 2 : 1); ++b) {
                uint32_t w;
                __builtin_memcpy(&w, sc + 4 * (D == 64 ? h >> 1 : D == 128 ? h : 2 * h + b), 4);
                kd[0][b] = (uint16_t)w;
                kd[1][b] = (uint16_t)(w >> 16);
            }
        }
        float x[8];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            f32x4 c = (f32x4)0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const f16x8 k = k_frag(kc[half][j], pair_of(kd[half][D == 256 ? j / 4 : 0]));
                c = mfma16(k, qh[j], c);
                c = mfma16(k, ql[j], c);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) x[4 * half + i] = c[i] * f;
        }
        const int32_t first = (int32_t)(tile * 32);
        // a tile that every row sees whole needs no mask
        const bool whole = first + 31 <= lo && (!a.window || (int64_t)first > (int64_t)hi - (int64_t)a.window || first + 32 <= (int64_t)a.sinks);
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int32_t k = first + 16 * (i >> 2) + 4 * (int32_t)h + (i & 3);
                const bool see = k <= pos && (!a.window || (int64_t)k > (int64_t)pos - (int64_t)a.window || (uint32_t)k < a.sinks);
                x[i] = see ? x[i] : -__builtin_inff();
            }
        }
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = __builtin_fmaxf(top, x[i]);
        if (__builtin_amdgcn_ballot_w64(top > m + kSlack) != 0ull) {
            top = __builtin_fmaxf(top, xor_lanes(top, 16));
            top = __builtin_fmaxf(top, xor_lanes(top, 32));
            const float next = __builtin_fmaxf(m, top);
            const float alpha = __builtin_amdgcn_exp2f(m - next);
            m = next;
            l *= alpha;
#pragma unroll
            for (int g = 0; g < NJ; ++g) {
                acc[g][0] *= alpha;
                acc[g][1] *= alpha;
            }
        }
        const float base = m - kUp;
        f16x8 ph, pl;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float e = __builtin_amdgcn_exp2f(x[i] - base);
            l += e;
            const _Float16 hv = (_Float16)e;
            ph[i] = hv;
            pl[i] = (_Float16)(e - (float)hv);
        }
        // V: per pair of channel blocks 16 bytes (two blocks' eight tokens), and the tokens' scales
#pragma unroll
        for (int g2 = 0; g2 < D / 64; ++g2) {
            u32x4 w;
            __builtin_memcpy(&w, t + 16 * D + (g2 * 16 + r) * 64 + h * 16, 16);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int g = 2 * g2 + b;
                f16x8 d;
                __builtin_memcpy(&d, t + 34 * D + (g * 4 + h) * 16, 16);
#pragma unroll
                for (int odd = 0; odd < 2; ++odd) {
                    const f16x8 v = v_frag(w[2 * b], w[2 * b + 1], 4 * odd, d);
                    acc[g][odd] = mfma16(v, ph, acc[g][odd]);
                    acc[g][odd] = mfma16(v, pl, acc[g][odd]);
                }
            }
        }
    }

    // the lanes' sums of a column, then the four waves
    l += xor_lanes(l, 16);
    l += xor_lanes(l, 32);
    if (h == 0) {
        red_m[wave * 16 + r] = m;
        red_l[wave * 16 + r] = l;
    }
#pragma unroll
    for (int g = 0; g < NJ; ++g) {
        float o[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[2 * i] = acc[g][0][i];
            o[2 * i + 1] = acc[g][1][i];
        }
        __builtin_memcpy(red_o + (wave * 16 + r) * (D + 4) + 32 * g + 8 * h, o, 32);
    }
    __syncthreads();
    const uint32_t rr = threadIdx.x >> 4, row_out = row0 + rr;
    if (row_out >= rows) return;
    float M = kNoMax, L = 0.0f, w4[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) M = __builtin_fmaxf(M, red_m[w * 16 + rr]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        w4[w] = __builtin_amdgcn_exp2f(red_m[w * 16 + rr] - M);
        L += red_l[w * 16 + rr] * w4[w];
    }
    const uint32_t tok_out = p.q0 + row_out / a.group, head_out = kvh * a.group + row_out % a.group;
    const size_t flat = (size_t)tok_out * a.n_heads + head_out;
    const float inv = a.splits > 1 ? 1.0f : L > 0.0f || L != L ? 1.0f / L : 0.0f;
    float *dst = a.splits > 1 ? a.part_o + ((size_t)split * a.n_tok * a.n_heads + flat) * D
                              : a.out + (size_t)tok_out * a.out_stride + (size_t)head_out * D;
    for (uint32_t c = 4 * (threadIdx.x & 15); c < (uint32_t)D; c += 64) {
        f32x4 o = (f32x4)0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            f32x4 v;
            __builtin_memcpy(&v, red_o + (w * 16 + rr) * (D + 4) + c, 16);
            o += v * w4[w];
        }
        o *= inv;
        __builtin_memcpy(dst + c, &o, 16);
    }
    if (a.splits > 1 && (threadIdx.x & 15) == 0) {
        float *ml = a.part_ml + 2 * ((size_t)split * a.n_tok * a.n_heads + flat);
        ml[0] = M;
        ml[1] = L;
    }
}

// Joins the pieces of a context: one wave per row (token, head).  A piece past the row's keys was never
// written; which those are follows from the same tiles_of.
template <int D>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a, uint32_t tile_rows) {
    const uint32_t lane = threadIdx.x & 63, s = blockIdx.y;
    const Span p = span_of(a, s);
    const uint32_t n = p.nq * a.n_heads, it = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (it >= n) return;
    const uint32_t i = it / a.n_heads, head = it % a.n_heads, g = a.group;
    const uint32_t row = i * g + head % g, row0 = row - row % tile_rows;
    const uint32_t last = row0 + tile_rows - 1 < p.nq * g ? row0 + tile_rows - 1 : p.nq * g - 1;
    const int32_t pos0 = p.ctx - (int32_t)p.nq;
    const Tiles T = tiles_of(a, pos0 + (int32_t)(row0 / g), pos0 + (int32_t)(last / g));
    const uint32_t chunk = piece_of(a, T), pieces = T.count ? (T.count + chunk - 1) / chunk : 1;
    const size_t all = (size_t)a.n_tok * a.n_heads, flat = (size_t)(p.q0 + i) * a.n_heads + head;
    float M = kNoMax;
    for (uint32_t k = lane; k < pieces; k += 64) M = __builtin_fmaxf(M, a.part_ml[2 * (k * all + flat)]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) M = __builtin_fmaxf(M, xor_lanes(M, o));
    float L = 0.0f, acc[D / 64];
#pragma unroll
    for (int c = 0; c < D / 64; ++c) acc[c] = 0.0f;
    for (uint32_t k = 0; k < pieces; ++k) {
        const float *ml = a.part_ml + 2 * (k * all + flat), w = __builtin_amdgcn_exp2f(ml[0] - M);
        L += ml[1] * w;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) acc[c] += a.part_o[(k * all + flat) * D + 64 * c + lane] * w;
    }
    const float inv = L > 0.0f || L != L ? 1.0f / L : 0.0f;
    float *dst = a.out + (size_t)(p.q0 + i) * a.out_stride + (size_t)head * D;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) dst[64 * c + lane] = acc[c] * inv;
}

template <int D> constexpr size_t attn_lds() { return (4 * 16 * (D + 4) + 128) * sizeof(float); }

template <int D>
hipError_t launch(const AttnArgs &a, hipStream_t stream) {
    const uint32_t tiles = (a.max_q * a.group + 15) / 16;
    const size_t lds = attn_lds<D>();
    hipLaunchKernelGGL(attn_rows_kernel<D>, dim3(a.splits * tiles * a.c.n_kv, a.n_seq), dim3(256), lds, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    hipLaunchKernelGGL(attn_join_kernel<D>, dim3((a.max_q * a.n_heads + 3) / 4, a.n_seq), dim3(256), 0, stream, a, 16u);
    return hipGetLastError();
}

} // namespace

hipError_t ah_launch_attn(const AttnArgs &a, hipStream_t stream) {
    return a.c.dim == 64 ? launch<64>(a, stream) : a.c.dim == 128 ? launch<128>(a, stream) : launch<256>(a, stream);
}

hipError_t ah_attn_init_attrs() {
    return hipFuncSetAttribute(reinterpret_cast<const void *>(attn_rows_kernel<256>), hipFuncAttributeMaxDynamicSharedMemorySize,
                               (int)attn_lds<256>());
}
