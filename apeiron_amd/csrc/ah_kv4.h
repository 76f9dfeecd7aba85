// ah_kv4.h -- the paged 4-bit key/value cache: its layout in memory, and the launch arguments of the
// operators between a token's projections (ah_token.hip, ah_attn.hip, ah_sample.hip), planned by
// ah_abi_token.cpp.
//
// A block is 32 channels of one token and KV head.  With m its element of largest magnitude (the
// positive one of two), d is the f16 number of 8 significant bits nearest to -m / 8, the code of x
// is clamp(rint(x / d), -8, 7) + 8 (x / d the f32 quotient) and stands for (code - 8) d.  Eight
// significant bits of scale and at most three of the code fit f16's eleven, so every value of the
// cache is exact in f16, subnormals included: the matrix cores take the values themselves.
//
// A tile is 32 tokens (positions) of one KV head, 36 D bytes: K codes (16 D), V codes (16 D), K
// scales (2 D), V scales (2 D).  A page is page_len / 32 tiles of every head, [head][tile].  Inside a
// tile the codes lie as the operands of v_mfma_f32_16x16x32_f16 want them, so that a lane's 16-byte
// load is one or more whole fragments.  Lane (r, h) = (lane & 15, lane >> 4) holds row r and the
// contraction's quarter h:
//   K: row r is token 16 s + r of half-tile s, and quarter h the channels h D/4 .. (h+1) D/4 - 1 (the
//      order of a contraction is free, as long as q's fragments keep it), so all of a lane's channels
//      share one scale (D <= 128) or two (D = 256);
//   V: row r is channel pair (2 cp, 2 cp + 1), cp = 16 g + r of block g, and quarter h the tokens
//      4 h .. 4 h + 3 of both half-tiles: those whose scores the same lane holds after K q, since
//      the product's rows come out as 4 h + i.  P never changes lanes.
// A token's append therefore writes single bytes of the V codes (no two tokens share a byte).
#pragma once

#include "ah_internal.h"

constexpr uint32_t kKvTile = 32;  // tokens of a tile

struct Kv4Ref {
    uint8_t *base;
    uint32_t n_pages, page_shift, n_kv, dim;  // page_len = 1 << page_shift
};

// Byte offset of tile `t` of page `page`, head `h`.
__host__ __device__ inline uint64_t kv4_tile(const Kv4Ref &c, uint32_t page, uint32_t h, uint32_t t) {
    return ((((uint64_t)page * c.n_kv + h) << (c.page_shift - 5)) + t) * (36u * c.dim);
}
// Offsets inside a tile.  tok: position in the tile; li: group of 8 channels; cp: channel pair.
__host__ __device__ inline uint32_t kv4_k_code(uint32_t dim, uint32_t tok, uint32_t li) {
    const uint32_t n = dim / 32, h = li / n, j = li % n, r = tok & 15, s = tok >> 4;  // j: 8-channel groups of the quarter
    return dim == 64 ? (r * 4 + h) * 16 + s * 8 + j * 4 : (s * (dim / 128) + j / 4) * 1024 + (r * 4 + h) * 16 + (j & 3) * 4;
}
__host__ __device__ inline uint32_t kv4_k_scale(uint32_t dim, uint32_t tok, uint32_t blk) {
    return 32 * dim + ((tok & 15) * (dim / 32) + blk) * 4 + (tok >> 4) * 2;
}
__host__ __device__ inline uint32_t kv4_v_code(uint32_t dim, uint32_t tok, uint32_t cp) {
    const uint32_t i = tok & 3, h = (tok >> 2) & 3, s = tok >> 4, g = cp >> 4, r = cp & 15;
    // tokens 0, 2, 1, 3 of a dword's bytes: a mask of its low nibbles is the f16 pair (0, 1), and
    // shifted by a byte (2, 3)
    return 16 * dim + ((g >> 1) * 16 + r) * 64 + h * 16 + (g & 1) * 8 + s * 4 + ((i & 1) << 1 | i >> 1);
}
__host__ __device__ inline uint32_t kv4_v_scale(uint32_t dim, uint32_t tok, uint32_t blk) {
    return 34 * dim + (blk * 4 + ((tok >> 2) & 3)) * 16 + ((tok >> 4) * 4 + (tok & 3)) * 2;
}

struct ah_kv4 {
    Kv4Ref ref = {};
    size_t bytes = 0;
};

constexpr uint32_t kRopeMaxDim = 512;
struct RopeRef {
    const double *theta;  // radians a position, [rot / 2]
    double amplitude;
    uint32_t dim, rot, interleaved;
};
struct ah_rope {
    RopeRef ref = {};
    double *host = nullptr;  // the same frequencies
};

struct NormArgs {
    const float *x, *r, *gain;
    float *sum, *y;
    int8_t *codes;
    int64_t *scales;
    uint16_t *values;
    double eps;
    uint32_t n_tok, n;
    unsigned long long *status;
};

struct KvTokens {
    const int32_t *seq, *pos, *table;
    uint32_t n_tok, n_seq, table_stride;
};
struct AppendArgs {
    Kv4Ref c;
    RopeRef rope;  // theta null: no rotation
    KvTokens t;
    const float *q, *k, *v;
    float *q_out;
    uint64_t q_stride, qo_stride, k_stride, v_stride;  // elements from token to token
    uint32_t n_heads;                                  // of q; 0: no q
    unsigned long long *status;
};
struct KvReadArgs {
    Kv4Ref c;
    KvTokens t;
    uint16_t *k, *v;  // f16 [n_tok][n_kv][dim]
    unsigned long long *status;
};
struct RopeArgs {
    RopeRef rope;
    const float *x;
    float *y;
    uint64_t x_stride, y_stride;
    const int32_t *pos;
    uint32_t n_tok, n_heads;
};

struct AttnArgs {
    Kv4Ref c;
    const int32_t *q_start, *ctx, *table;
    const float *q;
    float *out;
    uint64_t q_stride, out_stride;
    uint32_t n_seq, n_tok, n_heads, group, max_q, table_stride;
    uint32_t window, sinks;  // window 0: none
    float scale;
    // the split of the contexts: `splits` pieces of `chunk` tiles each; with several, partial results
    // go to part_o [splits][n_tok * n_heads][dim] and part_ml [splits][n_tok * n_heads][2]
    uint32_t splits, chunk;
    uint32_t rows;  // rows (token, head of a KV head's group) of a workgroup: 8, 16 or 128
    uint32_t grid;
    // sequences that the launch takes: for 8 and 16 rows those with at most most_rows, for 128 with at least least_rows
    uint32_t most_rows, least_rows;
    uint32_t per;  // units of 128 rows of every sequence; 0: they differ
    float *part_o, *part_ml;
    // The join in the launch: of attn_rows_kernel, pieces of a group, and the arrivals (zero between calls) of every
    // unit's groups, [unit], then of every group's pieces, [unit][group]; of attn_tile_kernel, whether it is there, and
    // the arrivals of every unit's pieces
    uint32_t join;
    uint32_t *count;
    unsigned long long *status;
};

// What a row's scan and count leave for the launches after them (ah_sample.hip).
struct SampleLimits {
    uint32_t g0, g1, bk, before_k;
    double mass_k, mass_0, all;
    uint32_t top, last, done;  // the largest key, the last bin to look at, whether the token is drawn
};
struct SampleArgs {
    const float *logits;
    uint64_t stride;
    uint32_t n_rows, n_vocab;
    const float *temperature, *top_p, *min_p, *u;
    const int32_t *top_k;
    int32_t *tokens;
    float *probs;
    unsigned long long *status;
    uint32_t *arrived;  // [n_counts], zero between calls
    uint32_t n_counts;
    // planned by ah_sample_plan: groups and chunks of a row, chunks of a workgroup and workgroups of a row (in the scan,
    // and after it), and the scratch
    uint32_t groups, chunks, scan_per, scan_parts, per, parts;
    bool draw;  // in the gather's launch
    SampleLimits *limits;                          // [row]
    double *bin_mass, *chunk_mass;                 // [row][bin], [row][chunk]
    float *group_max;                              // [row][group]
    uint32_t *bin_count, *bits;                    // [row][bin]; a bit for each token listed, [row][chunk]
};
constexpr uint32_t kSampleList = 4096, kSampleMaxChunks = 512;

// Threads of a token's workgroup: of the norm a lane per 8 values up to 1024 lanes, then more passes; of the others
// whole waves for `items` lanes' work, up to four.
inline uint32_t norm_lanes(size_t n) {
    const size_t need = (n + 7) / 8;
    return need <= 64 ? 64 : need <= 128 ? 128 : need <= 256 ? 256 : need <= 512 ? 512 : 1024;
}
inline uint32_t lanes_for(size_t items) { return items >= 256 ? 256 : (uint32_t)(items + 63) / 64 * 64; }
inline uint32_t rope_lanes(size_t dim, size_t n_heads) { return lanes_for((dim + 7) / 8 * n_heads); }  // (a head takes up to 64)
inline uint32_t append_lanes(const Kv4Ref &c, size_t n_heads) { return lanes_for(c.dim / 8 * (n_heads + 2 * (size_t)c.n_kv)); }  // the read's: no heads

hipError_t ah_launch_norm(const NormArgs &a, hipStream_t stream);
hipError_t ah_launch_rope(const RopeArgs &a, hipStream_t stream);
hipError_t ah_launch_kv4_append(const AppendArgs &a, hipStream_t stream);
hipError_t ah_launch_kv4_read(const KvReadArgs &a, hipStream_t stream);
hipError_t ah_launch_attn(const AttnArgs &a, hipStream_t stream);
size_t ah_sample_plan(SampleArgs &a, uint32_t cus, uint8_t *base);
hipError_t ah_launch_sample(const SampleArgs &a, hipStream_t stream);
