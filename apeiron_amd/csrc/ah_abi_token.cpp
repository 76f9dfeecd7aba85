// ah_abi_token.cpp -- host side of the operators between a token's projections: argument checks, the
// rope and cache handles, and the plan of the attention's splits.
#include "ah_host.h"
#include "ah_kv4.h"

#include <cmath>
#include <new>

namespace {

constexpr size_t kMaxU32 = 0x7fffffff;
// Workgroups that a split attention over few rows aims at.  ah_ctx::d_count has an entry for every unit and for every
// group of its pieces: at most kAttnGroups / 2 of each (two pieces, one group), and fewer of both with more pieces.
constexpr size_t kAttnGroups = 2048;
static_assert(kAttnGroups <= kCounts, "an entry for each unit and each group of pieces");

constexpr size_t max_grid(size_t threads) { return 0xffffffffu / threads; }  // workgroups of a launch: under 2^32 threads

bool tokens_ok(const ah_kv4_tokens *t) {
    return t->d_seq && t->d_pos && t->d_table && t->n_seq && t->table_stride && t->n_tok <= kMaxU32 && t->n_seq <= kMaxU32 &&
           t->table_stride <= kMaxU32;
}
KvTokens tokens_of(const ah_kv4_tokens *t) {
    return {t->d_seq, t->d_pos, t->d_table, (uint32_t)t->n_tok, (uint32_t)t->n_seq, (uint32_t)t->table_stride};
}

// The tiles that a sequence's rows see at most.
size_t most_tiles(const AttnArgs &a, size_t max_ctx, size_t max_q) {
    const size_t room = (size_t)a.table_stride << a.c.page_shift, tiles = ((max_ctx < room ? max_ctx : room) + 31) / 32;
    if (!a.window) return tiles;
    const size_t seen = (a.window + max_q + 31) / 32 + 1 + ((size_t)a.sinks + 31) / 32;
    return tiles < seen ? tiles : seen;
}

// Room for the partial results of `rows` rows in each of a.splits pieces, behind `kept` bytes of the scratch.
int32_t attn_scratch(ah_ctx *ctx, AttnArgs &a, size_t rows, size_t kept, void *stream) {
    if (a.splits == 1 && kept == 0) return AH_OK;
    const size_t o = align256(a.splits * rows * a.c.dim * sizeof(float));
    const int32_t st = ensure_scratch(ctx, kept + (a.splits > 1 ? o + a.splits * rows * 2 * sizeof(float) : 0), stream);
    if (st) return st;
    a.part_o = reinterpret_cast<float *>(static_cast<uint8_t *>(ctx->scratch.p) + kept);
    a.part_ml = reinterpret_cast<float *>(static_cast<uint8_t *>(ctx->scratch.p) + kept + o);
    a.count = ctx->d_count;
    return AH_OK;
}
// At most these pieces: 256 MiB of partial results.
size_t most_pieces(const AttnArgs &a, size_t rows) {
    const size_t n = ((size_t)256 << 20) / (rows * (a.c.dim + 2) * sizeof(float));
    return n < 1 ? 1 : n;
}
// Pieces of `chunk` tiles each, and the scratch that they take behind `kept` bytes.
int32_t attn_pieces(ah_ctx *ctx, AttnArgs &a, size_t units, size_t tiles, size_t chunk, size_t kept, void *stream) {
    chunk = chunk < 1 ? 1 : chunk;
    a.chunk = (uint32_t)chunk;
    a.splits = (uint32_t)((tiles + chunk - 1) / chunk);
    a.splits = a.splits < 1 ? 1 : a.splits;
    if (a.rows != 128) a.join = a.splits <= 40 ? a.splits : (uint32_t)std::ceil(std::sqrt((double)a.splits));
    else a.join = a.splits <= 3 && a.c.dim == 64 && units <= kCounts;
    if (units > max_grid(256) / a.splits) return AH_ERR_INVALID_ARG;
    a.grid = (uint32_t)(units * a.splits);
    AH_HIP(ctx, hipSetDevice(ctx->device));
    return attn_scratch(ctx, a, (size_t)a.n_tok * a.n_heads, kept, stream);
}
int32_t attn_launch(ah_ctx *ctx, AttnArgs &a, size_t units, size_t tiles, size_t chunk, void *stream) {
    const int32_t st = attn_pieces(ctx, a, units, tiles, chunk, 0, stream);
    if (st) return st;
    AH_HIP(ctx, ah_launch_attn(a, pick(ctx, stream)));
    return AH_OK;
}

// Sequences of at most `most` rows over at most `tiles` tiles, by workgroups of 8 or 16: their pieces.
int32_t attn_rows_plan(ah_ctx *ctx, AttnArgs &a, size_t tiles, size_t most, size_t kept, void *stream) {
    a.rows = most <= 8 ? 8 : 16;
    a.most_rows = (uint32_t)most;
    const size_t per = (most + a.rows - 1) / a.rows, base = per * a.c.n_kv * a.n_seq, rows = (size_t)a.n_tok * a.n_heads;
    // With few units a piece's tiles (0.7 us for each of a wave) stand against the join (0.1 us a piece):
    // sqrt(1.75 tiles) pieces, past 40 of them two joins and 16 tiles a piece.  One sequence of 4001 keys in pieces
    // of 4, 8, 16 and 24 tiles: 10.6, 10.0, 10.7 and 13.3 us.  Once that passes a workgroup a CU (two, where two
    // joins pay for themselves: 120000 keys in 256 workgroups 24.5 us, in 469 21.8), pieces of 32 tiles, since a
    // workgroup costs its start and end.  With 2 KV heads of 128, in pieces of 16, 32 and 64 tiles: 128 sequences
    // of 1000 keys 16.6, 13.4 and 13.4 us, of 4000 41.9, 35.8 and 35.6; 64 of 1 to 16384 52, 46 and 52.
    const double wish = std::sqrt(1.75 * (double)tiles), groups = wish <= 40.0 ? 256.0 : 512.0;
    double pieces = wish <= 40.0 ? wish : (double)tiles / 16.0;
    if (pieces * (double)base > groups) {
        const double most_pieces = (double)(kAttnGroups / base), by_tiles = (double)tiles / 32.0;
        pieces = by_tiles < most_pieces ? by_tiles : most_pieces;
        pieces = pieces * (double)base > groups ? pieces : groups / (double)base;
    }
    size_t chunk = pieces < 1.0 ? tiles : 4 * (size_t)((double)tiles / (4.0 * pieces) + 0.5);  // whole rounds of the four waves
    size_t fit = base <= kAttnGroups / 2 ? kAttnGroups / base : 1;
    fit = fit < most_pieces(a, rows) ? fit : most_pieces(a, rows);
    chunk = chunk < (tiles + fit - 1) / fit ? (tiles + fit - 1) / fit : chunk;
    return attn_pieces(ctx, a, base, tiles, chunk, kept, stream);
}
int32_t attn_rows(ah_ctx *ctx, AttnArgs a, size_t max_ctx, size_t most, void *stream) {
    const int32_t st = attn_rows_plan(ctx, a, most_tiles(a, max_ctx, most / a.group), most, 0, stream);
    if (st) return st;
    AH_HIP(ctx, ah_launch_attn(a, pick(ctx, stream)));
    return AH_OK;
}

// Sequences of at least a.least_rows rows, by workgroups of 128.
int32_t attn_tiles(ah_ctx *ctx, AttnArgs a, size_t max_ctx, void *stream) {
    a.rows = 128;
    const size_t rows = (size_t)a.n_tok * a.n_heads, per = ((size_t)a.max_q * a.group + 127) / 128;
    const size_t tiles = most_tiles(a, max_ctx, a.max_q);
    // the numbers that units of 128 rows have (of uneven sequences at most one more for each)
    const bool even = (size_t)a.n_tok == (size_t)a.n_seq * a.max_q;
    a.per = even || a.n_seq == 1 ? (uint32_t)per : 0;
    const size_t units = a.per ? per * a.n_seq : ((size_t)a.n_tok * a.group >> 7) + a.n_seq;
    // Pieces by the time that they take, in us: workgroups in rounds of as many as the CUs hold (their registers and
    // LDS: three of heads of 64, two of 128, one of 256), the matrix work of a CU's shared among them (tile: that of 128
    // rows and 32 keys), a workgroup's start and end, and a piece's results written and read again in a launch more.
    // One sequence, 2 KV heads, in 1100 / units pieces and in these: 512 tokens over 4096 keys, heads of 64, 128 and
    // 256, 44 -> 41, 57 -> 50 and 85 -> 63 us; 2048 tokens of a prompt 54 -> 44, 69 -> 56 and 112 -> 71.
    // (with least_rows, most of the other sequences are single tokens)
    const size_t chunks = a.n_tok - (a.n_seq - 1), tokens = !a.least_rows ? a.n_tok : a.n_tok > a.n_seq && chunks > a.max_q ? chunks : a.max_q;
    size_t base = even ? per * a.n_seq * a.c.n_kv : (tokens * a.group + 127) / 128 * a.c.n_kv;
    // Uneven sequences: the longest ones' workgroups are alone in the end, as if there were fewer.  With this and
    // without, us: heads of 64, 2 chunks of 600 over up to 8000 keys 73 and 87 (six other calls the same); of 256, 5 of
    // 301 over 6007 162 and 203.  Elsewhere it asks for too many pieces of the larger heads: of 128, 5 of 301 over 6007 110
    // and 89, 16 of 100 over 2000 55 and 48; of 256, 85 and 68 there, 8 of 256 over 4096 115 and 109.
    if (!even && !a.least_rows) base = (base * 3 + 4) / 5;
    const double tile = a.c.dim * 0.0077, alone = 1.4 * tile, start = 5.0, join = (double)rows * a.c.dim * 8.0 / 4e6;
    const size_t held = a.c.dim == 64 ? 3 : a.c.dim == 128 ? 2 : 1, cus = (size_t)ctx->cu_count, places = held * cus;
    auto round = [&](size_t n, size_t per_piece) {  // n workgroups at once
        const double t = (double)((n + cus - 1) / cus) * tile;
        return (double)per_piece * (t > alone ? t : alone) + start;
    };
    // Pieces of a length end together.  Under a causal mask (whole prompts) half of the workgroups and half of the keys
    // are there, longest first, and the shorter ones share the CUs or fill in, with a part of a piece at the end; uneven
    // sequences fill in too.  With the causal form and without, us: heads of 64, prompts of 2048 and 4096 tokens 42 and 45,
    // 93 and 113; of 128, 2048 55 and 59; of 256 72 and 88, 196 and 246 (and 4 prompts of 700 72 and 57: the other way).
    const bool causal = even && max_ctx < 2 * (size_t)a.max_q;
    size_t splits = 1, most = (tiles + 7) / 8;
    most = most < most_pieces(a, rows) ? most : most_pieces(a, rows);
    double best = 0.0;
    for (size_t n = 1; n <= most && n <= 64; ++n) {
        const size_t all = causal ? base * (n + 1) / 2 : base * n, full = all / places, rest = all % places, per_piece = (tiles + n - 1) / n;
        double t;
        if (causal && all > places) {
            t = ((double)base * (double)tiles * 0.5 / (double)places + (n > 1 ? 0.3 : 0.0) * (double)per_piece) * (held * tile > alone ? held * tile : alone) +
                start * (double)all / (double)places;
        } else if (causal) {
            const double shared = (double)((all + cus - 1) / cus), t0 = (shared - (shared - 1.0) * 0.5 / (double)n) * tile;
            t = (double)per_piece * (t0 > alone ? t0 : alone) + start;
        } else if (!even && full) {
            t = (double)all / (double)places * round(places, per_piece);
        } else {
            t = (double)full * round(places, per_piece) + (rest ? round(rest, per_piece) : 0.0);
        }
        if (n > 1) t += 3.0 + (double)n * (a.c.dim == 64 && n <= 3 ? 0.5 : 1.0) * join;
        if (n == 1 || t < best) {
            best = t;
            splits = n;
        }
    }
    return attn_launch(ctx, a, units * a.c.n_kv, tiles, (tiles + splits - 1) / splits, stream);
}

// The checks that every form of attention makes, and its arguments.
int32_t attn_args(ah_ctx *ctx, const ah_kv4 *cache, const ah_kv4_attn *p, const float *d_q, size_t q_stride, float *d_out,
                  size_t out_stride, AttnArgs &a) {
    const size_t dim = cache->ref.dim, kv = cache->ref.n_kv;
    if (!p->d_q_start || !p->d_ctx || !p->d_table || !d_q || !d_out || p->n_seq > 65535 || p->n_tok > kMaxU32 ||
        p->n_heads > 65536 || p->n_heads % kv || p->table_stride == 0 || p->table_stride > kMaxU32 || q_stride < p->n_heads * dim ||
        out_stride < p->n_heads * dim || p->window > kMaxU32 || p->sinks > kMaxU32)
        return AH_ERR_INVALID_ARG;
    a = {};
    a.c = cache->ref;
    a.q_start = p->d_q_start;
    a.ctx = p->d_ctx;
    a.table = p->d_table;
    a.q = d_q;
    a.out = d_out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.n_seq = (uint32_t)p->n_seq;
    a.n_tok = (uint32_t)p->n_tok;
    a.n_heads = (uint32_t)p->n_heads;
    a.group = (uint32_t)(p->n_heads / kv);
    a.max_q = (uint32_t)(p->max_q < p->n_tok ? p->max_q : p->n_tok);
    a.table_stride = (uint32_t)p->table_stride;
    a.window = (uint32_t)p->window;
    a.sinks = (uint32_t)p->sinks;
    a.scale = p->scale;
    a.status = ctx->d_status;
    return (size_t)a.max_q * a.group > kMaxU32 / 256 ? AH_ERR_INVALID_ARG : AH_OK;
}
bool empty(const ah_kv4_attn *p) { return p->n_seq == 0 || p->n_tok == 0 || p->n_heads == 0 || p->max_q == 0; }

} // namespace

extern "C" {

int32_t ah_norm_quant_dev(ah_ctx *ctx, const float *d_x, const float *d_residual, const float *d_gain, float eps, size_t n_tok,
                          size_t n, float *d_sum, float *d_y, int8_t *d_codes, int64_t *d_scales, uint16_t *d_values,
                          void *stream) {
    if (!ctx || (d_codes == nullptr) != (d_scales == nullptr)) return AH_ERR_INVALID_ARG;
    if (!(eps >= 0.0f) || n > AH_MAX_N_IN || n_tok > kMaxU32) return AH_ERR_INVALID_ARG;
    if (n_tok == 0 || n == 0) return AH_OK;
    if (!d_x || !d_gain || (reinterpret_cast<uintptr_t>(d_scales) & 7) || n_tok > max_grid(norm_lanes(n))) return AH_ERR_INVALID_ARG;
    NormArgs a = {d_x, d_residual, d_gain, d_sum, d_y, d_codes, d_scales, d_values, (double)eps, (uint32_t)n_tok, (uint32_t)n,
                  ctx->d_status};
    AH_HIP(ctx, hipSetDevice(ctx->device));
    AH_HIP(ctx, ah_launch_norm(a, pick(ctx, stream)));
    return AH_OK;
}

int32_t ah_rope_create(ah_ctx *ctx, const ah_rope_spec *spec, ah_rope **out) {
    if (!ctx || !spec || !out) return AH_ERR_INVALID_ARG;
    *out = nullptr;
    const size_t dim = spec->head_dim, rot = spec->rot_dim;
    if (dim > kRopeMaxDim || rot < 2 || rot > dim || (rot & 1) || (dim & 1) || spec->layout > AH_ROPE_INTERLEAVED ||
        spec->scaling > AH_ROPE_BANDS || !(spec->base > 0.0) || !std::isfinite(spec->base) || !std::isfinite(spec->amplitude))
        return AH_ERR_INVALID_ARG;
    const bool scaled = spec->scaling != AH_ROPE_NONE, bands = spec->scaling == AH_ROPE_BANDS;
    if (scaled && (!(spec->factor > 0.0) || !std::isfinite(spec->factor))) return AH_ERR_INVALID_ARG;
    if (spec->scaling == AH_ROPE_NTK && rot == 2) return AH_ERR_INVALID_ARG;
    if (bands && (!(spec->high > spec->low) || !std::isfinite(spec->high) || !std::isfinite(spec->low) ||
                  !(spec->original_ctx > 0.0) || !std::isfinite(spec->original_ctx)))
        return AH_ERR_INVALID_ARG;
    ah_rope *r = new (std::nothrow) ah_rope();
    double *host = r ? new (std::nothrow) double[rot / 2] : nullptr;
    if (!host) {
        delete r;
        return AH_ERR_OUT_OF_MEMORY;
    }
    const double base =
        spec->scaling == AH_ROPE_NTK ? spec->base * std::pow(spec->factor, (double)rot / (double)(rot - 2)) : spec->base;
    for (size_t j = 0; j < rot / 2; ++j) {
        double t = std::pow(base, -2.0 * (double)j / (double)rot);
        if (spec->scaling == AH_ROPE_LINEAR) t /= spec->factor;
        if (bands) {
            double g = (spec->original_ctx * t / 6.283185307179586476925 - spec->low) / (spec->high - spec->low);
            g = g < 0.0 ? 0.0 : g > 1.0 ? 1.0 : g;
            t = t * ((1.0 - g) / spec->factor + g);
        }
        host[j] = t;
    }
    r->host = host;
    r->ref.dim = (uint32_t)dim;
    r->ref.rot = (uint32_t)rot;
    r->ref.interleaved = spec->layout == AH_ROPE_INTERLEAVED;
    r->ref.amplitude = spec->amplitude != 0.0 ? spec->amplitude : bands ? 0.1 * std::log(spec->factor) + 1.0 : 1.0;
    void *d = nullptr;
    hipError_t e = hipSetDevice(ctx->device);
    if (e == hipSuccess) e = hipMalloc(&d, rot / 2 * sizeof(double));
    if (e == hipSuccess) e = hipMemcpy(d, host, rot / 2 * sizeof(double), hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        ctx->last_hip = (int)e;
        if (d) (void)hipFree(d);
        delete[] host;
        delete r;
        return e == hipErrorOutOfMemory ? AH_ERR_OUT_OF_MEMORY : AH_ERR_HIP;
    }
    r->ref.theta = static_cast<const double *>(d);
    *out = r;
    return AH_OK;
}

int32_t ah_rope_free(ah_ctx *ctx, ah_rope *rope) {
    if (!ctx || !rope) return AH_ERR_INVALID_ARG;
    AH_HIP(ctx, hipSetDevice(ctx->device));
    AH_HIP(ctx, hipStreamSynchronize(ctx->stream));
    AH_HIP(ctx, hipFree(const_cast<double *>(rope->ref.theta)));
    delete[] rope->host;
    delete rope;
    return AH_OK;
}

int32_t ah_rope_info(const ah_rope *rope, double *theta, double *amplitude) {
    if (!rope) return AH_ERR_INVALID_ARG;
    if (theta)
        for (uint32_t j = 0; j < rope->ref.rot / 2; ++j) theta[j] = rope->host[j];
    if (amplitude) *amplitude = rope->ref.amplitude;
    return AH_OK;
}

int32_t ah_rope_dev(ah_ctx *ctx, const ah_rope *rope, const float *d_x, size_t x_stride, size_t n_heads, const int32_t *d_pos,
                    size_t n_tok, float *d_y, size_t y_stride, void *stream) {
    if (!ctx || !rope || n_tok > kMaxU32 || n_heads > 65536) return AH_ERR_INVALID_ARG;
    if (n_tok == 0 || n_heads == 0) return AH_OK;
    const size_t row = n_heads * rope->ref.dim;
    if (!d_x || !d_y || !d_pos || x_stride < row || y_stride < row || (d_x == d_y && x_stride != y_stride) ||
        n_tok > max_grid(rope_lanes(rope->ref.dim, n_heads)))
        return AH_ERR_INVALID_ARG;
    RopeArgs a = {rope->ref, d_x, d_y, x_stride, y_stride, d_pos, (uint32_t)n_tok, (uint32_t)n_heads};
    AH_HIP(ctx, hipSetDevice(ctx->device));
    AH_HIP(ctx, ah_launch_rope(a, pick(ctx, stream)));
    return AH_OK;
}

int32_t ah_kv4_create(ah_ctx *ctx, size_t n_pages, size_t page_len, size_t n_kv_heads, size_t head_dim, ah_kv4 **out) {
    if (!ctx || !out) return AH_ERR_INVALID_ARG;
    *out = nullptr;
    if (n_pages == 0 || n_pages > kMaxU32 || page_len < 32 || page_len > 1024 || (page_len & (page_len - 1)) || n_kv_heads == 0 ||
        n_kv_heads > 4096 || (head_dim != 64 && head_dim != 128 && head_dim != 256))
        return AH_ERR_INVALID_ARG;
    size_t bytes;
    if (__builtin_mul_overflow(n_pages, n_kv_heads * (page_len / 32) * 36 * head_dim, &bytes)) return AH_ERR_INVALID_ARG;
    ah_kv4 *c = new (std::nothrow) ah_kv4();
    if (!c) return AH_ERR_OUT_OF_MEMORY;
    void *d = nullptr;
    hipError_t e = hipSetDevice(ctx->device);
    if (e == hipSuccess) e = hipMalloc(&d, bytes);
    if (e == hipSuccess) e = hipMemset(d, 0, bytes);
    if (e == hipSuccess) e = hipStreamSynchronize(nullptr);
    if (e != hipSuccess) {
        ctx->last_hip = (int)e;
        if (d) (void)hipFree(d);
        delete c;
        return e == hipErrorOutOfMemory ? AH_ERR_OUT_OF_MEMORY : AH_ERR_HIP;
    }
    c->bytes = bytes;
    c->ref.base = static_cast<uint8_t *>(d);
    c->ref.n_pages = (uint32_t)n_pages;
    c->ref.page_shift = (uint32_t)__builtin_ctzll(page_len);
    c->ref.n_kv = (uint32_t)n_kv_heads;
    c->ref.dim = (uint32_t)head_dim;
    *out = c;
    return AH_OK;
}

int32_t ah_kv4_free(ah_ctx *ctx, ah_kv4 *cache) {
    if (!ctx || !cache) return AH_ERR_INVALID_ARG;
    AH_HIP(ctx, hipSetDevice(ctx->device));
    AH_HIP(ctx, hipStreamSynchronize(ctx->stream));
    AH_HIP(ctx, hipFree(cache->ref.base));
    delete cache;
    return AH_OK;
}

int32_t ah_kv4_info(const ah_kv4 *cache, size_t *bytes, size_t *n_pages, size_t *page_len, size_t *n_kv_heads, size_t *head_dim) {
    if (!cache) return AH_ERR_INVALID_ARG;
    if (bytes) *bytes = cache->bytes;
    if (n_pages) *n_pages = cache->ref.n_pages;
    if (page_len) *page_len = (size_t)1 << cache->ref.page_shift;
    if (n_kv_heads) *n_kv_heads = cache->ref.n_kv;
    if (head_dim) *head_dim = cache->ref.dim;
    return AH_OK;
}

int32_t ah_kv4_append_dev(ah_ctx *ctx, ah_kv4 *cache, const ah_rope *rope, const ah_kv4_tokens *tokens, const float *d_q,
                          size_t q_stride, size_t n_heads, float *d_q_out, size_t q_out_stride, const float *d_k, size_t k_stride,
                          const float *d_v, size_t v_stride, void *stream) {
    if (!ctx || !cache || !tokens) return AH_ERR_INVALID_ARG;
    if (tokens->n_tok == 0) return AH_OK;
    if (!tokens_ok(tokens) || !d_k || !d_v || n_heads > 65536) return AH_ERR_INVALID_ARG;
    const size_t dim = cache->ref.dim, kv = cache->ref.n_kv * dim;
    if (k_stride < kv || v_stride < kv || (rope && rope->ref.dim != dim) || tokens->n_tok > max_grid(append_lanes(cache->ref, n_heads)))
        return AH_ERR_INVALID_ARG;
    if (n_heads && (!d_q || !d_q_out || q_stride < n_heads * dim || q_out_stride < n_heads * dim ||
                    (d_q == d_q_out && q_stride != q_out_stride)))
        return AH_ERR_INVALID_ARG;
    AppendArgs a = {};
    a.c = cache->ref;
    if (rope) a.rope = rope->ref;
    a.t = tokens_of(tokens);
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.q_out = d_q_out;
    a.q_stride = q_stride;
    a.qo_stride = q_out_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.n_heads = (uint32_t)n_heads;
    a.status = ctx->d_status;
    AH_HIP(ctx, hipSetDevice(ctx->device));
    AH_HIP(ctx, ah_launch_kv4_append(a, pick(ctx, stream)));
    return AH_OK;
}

int32_t ah_kv4_read_dev(ah_ctx *ctx, const ah_kv4 *cache, const ah_kv4_tokens *tokens, uint16_t *d_k, uint16_t *d_v, void *stream) {
    if (!ctx || !cache || !tokens) return AH_ERR_INVALID_ARG;
    if (tokens->n_tok == 0 || (!d_k && !d_v)) return AH_OK;
    if (!tokens_ok(tokens) || tokens->n_tok > max_grid(append_lanes(cache->ref, 0))) return AH_ERR_INVALID_ARG;
    KvReadArgs a = {cache->ref, tokens_of(tokens), d_k, d_v, ctx->d_status};
    AH_HIP(ctx, hipSetDevice(ctx->device));
    AH_HIP(ctx, ah_launch_kv4_read(a, pick(ctx, stream)));
    return AH_OK;
}

int32_t ah_kv4_attn_dev(ah_ctx *ctx, const ah_kv4 *cache, const ah_kv4_attn *p, const float *d_q, size_t q_stride, float *d_out,
                        size_t out_stride, void *stream) {
    if (!ctx || !cache || !p) return AH_ERR_INVALID_ARG;
    if (empty(p)) return AH_OK;
    AttnArgs a;
    const int32_t bad = attn_args(ctx, cache, p, d_q, q_stride, d_out, out_stride, a);
    if (bad) return bad;
    const size_t kv = a.c.n_kv;
    // The kernel: 8 packed rows or 16 rows a workgroup, or 128 over tiles in LDS.  Those start later and need many rows
    // of a sequence (they convert the cache's codes once for all of them, the others once for 16).  2 KV heads, rows a
    // sequence and sequences: 56 and 64 of 1000 keys, heads of 64, 128 and 256, 15, 22 and 37 us by 16 rows against 24,
    // 34 and 53; 120 and 16 of 2000 16, 25 and 41 against 22, 31 and 51; 8 KV heads of 128: 80 and 16 of 2000 keys (640
    // units of 16 rows) 47 against 50, 120 and 16 (1024) 72 against 59; one of 512 rows of 2 KV heads (64 units) 24
    // against 23.
    const size_t unit_rows = (size_t)a.max_q * a.group, units = (unit_rows + 15) / 16 * kv * p->n_seq;
    if (unit_rows <= 64 || (unit_rows <= 128 && units <= 640) || units <= 64) return attn_rows(ctx, a, p->max_ctx, unit_rows, stream);
    // A few long chunks among single tokens (the others' mean is a part of 128 rows): the two kinds by a launch each.
    const size_t few = a.group <= 8 ? 8 : 32, others = a.n_tok > a.max_q ? a.n_tok - a.max_q : 0;
    if (a.n_seq > 1 && a.group <= few && others * a.group < (size_t)128 * (a.n_seq - 1)) {
        const int32_t st = attn_rows(ctx, a, p->max_ctx, few, stream);
        if (st) return st;
        a.least_rows = (uint32_t)few + 1;
    }
    return attn_tiles(ctx, a, p->max_ctx, stream);
}

int32_t ah_kv4_attn_shared_dev(ah_ctx *ctx, const ah_kv4 *cache, const ah_kv4_attn *p, size_t prefix_len, const int32_t *d_prefix_table,
                               const float *d_q, size_t q_stride, float *d_out, size_t out_stride, void *stream) {
    if (!ctx || !cache || !p || p->window || p->sinks || prefix_len > kMaxU32) return AH_ERR_INVALID_ARG;
    if (prefix_len == 0) return ah_kv4_attn_dev(ctx, cache, p, d_q, q_stride, d_out, out_stride, stream);
    if (empty(p)) return AH_OK;
    AttnArgs a;
    const int32_t bad = attn_args(ctx, cache, p, d_q, q_stride, d_out, out_stride, a);
    if (bad) return bad;
    const size_t rows = (size_t)a.n_tok * a.n_heads, batch = (size_t)a.n_tok * a.group;
    if (!d_prefix_table || batch > kMaxU32 / 256 || rows * a.c.dim > ((size_t)1 << 30) - 1 ||
        overlap(d_q, q_stride, a.n_heads * a.c.dim, d_out, out_stride, a.n_heads * a.c.dim, a.n_tok))
        return AH_ERR_INVALID_ARG;
    a.first_key = (uint32_t)prefix_len;
    const size_t kv = a.c.n_kv, per_seq = (size_t)a.max_q * a.group, room = (size_t)a.table_stride << a.c.page_shift;
    const size_t end = p->max_ctx < room ? p->max_ctx : room, tiles = end > prefix_len ? (end + 31) / 32 - prefix_len / 32 : 0;
    // A short prefix of few sequences, each reads for itself: it costs less than a second launch and the join.  (Single tokens of 14
    // heads of 64 over 2, us a call for itself and together: 8 behind 2048 keys 12.9 and 15.9, 16 behind 4096 13.6 and 15.6, 64
    // behind 512 12.3 and 14.6, 32 behind 2048 and 512 more 15.1 and 14.8, 4 behind 16384 16.9 and 15.1; 12 of 128 over 2: 8 behind
    // 2048 14.2 and 16.2, 16 behind 4096 17.5 and 17.1, 8 behind 8192 19.5 and 15.9; 32 over 8: 16 behind 2048 19.7 and 16.0.
    // Heads of 256 gain nothing.)
    if (a.c.dim < 256 && prefix_len <= 4096 && a.n_seq * ((per_seq + 15) / 16) * kv * a.c.dim * prefix_len <= (size_t)1 << 23) {
        a.first_table = d_prefix_table;
        const int32_t st = attn_rows_plan(ctx, a, (prefix_len + 31) / 32 + tiles, per_seq, 0, stream);
        if (st) return st;
        AH_HIP(ctx, ah_launch_attn_some(a, pick(ctx, stream)));
        return AH_OK;
    }
    AttnArgs pre = a, own = a;
    const size_t cus = (size_t)ctx->cu_count, most = most_pieces(a, rows);
    auto cut = [&](AttnArgs &x, size_t units, size_t tiles, size_t n) {  // into n pieces
        n = n < most / 2 ? n : most / 2;
        n = n < 1 ? 1 : n;
        const size_t chunk = tiles ? (tiles + n - 1) / n : 1;
        x.chunk = (uint32_t)chunk;
        x.splits = (uint32_t)(tiles ? (tiles + chunk - 1) / chunk : 1);
        x.grid = (uint32_t)(units * x.splits);
        return units <= max_grid(256) / 2 / x.splits;
    };
    // What follows the prefix: each sequence for itself, by units of 8 or 16 rows, or of 128 where its rows are many and the units
    // of 16 twelve a CU and more (2 KV heads of 128, sequences x tokens and their keys, units, us by 16 and by 128: 16 x 128 of
    // 128 1536 100 and 112; 64 x 49 of 2048 2432 181 and 186; 32 x 128 of 128 12 a CU 109 and 103; 32 x 256 of 256 6144 213
    // and 189; 16 x 512 of 512 6144 242 and 198).
    own.rows = per_seq <= 8 ? 8 : 16;
    size_t own_units = (per_seq + own.rows - 1) / own.rows * kv * a.n_seq;
    if (per_seq > 128 && own_units >= 12 * cus) {
        own.rows = 128;
        own.per = (size_t)a.n_tok == (size_t)a.n_seq * a.max_q || a.n_seq == 1 ? (uint32_t)((per_seq + 127) / 128) : 0;
        own_units = (own.per ? (size_t)own.per * a.n_seq : ((size_t)a.n_tok * a.group >> 7) + a.n_seq) * kv;
    }
    // The prefix: the whole batch as one sequence.  Units of 16 rows; of 32, for heads of 128, from 2^23 rows x keys on (a
    // tile's codes are converted for twice the rows, by half as many waves); of 128, with the tiles in LDS, where the rows are many
    // more.  2 KV heads behind 8192 keys, rows of a KV head, us by 16, 32, 128: heads of 128, 48 rows 16, 19, 22; 384 26, 27, 36; 768
    // 38, 36, 44; 1764 71, 58, 60; 2352 81, 67, 68; 4704 133, 115, 113; 384 rows behind 16384 keys 39, 34, 47, behind 2048 17,
    // 20, 23; of 64 (16 and 128) 1400 36 and 38, 1715 48 and 41; of 256 1024 66 and 80, 1568 94 and 95, 1960 113 and 108.
    pre.n_seq = 1;
    pre.table = d_prefix_table;
    pre.table_stride = (uint32_t)((prefix_len - 1) >> a.c.page_shift) + 1;
    pre.rows = own.rows == 128 || batch > (a.c.dim == 128 ? 2560 : 1536) ? 128 : a.c.dim == 128 && batch * kv * prefix_len >= (size_t)1 << 23 ? 32 : 16;
    const size_t units = (batch + pre.rows - 1) / pre.rows, all = (prefix_len + 31) / 32;
    pre.per = (uint32_t)units;
    // Pieces by the time that they take, as attn_tiles has it: workgroups in rounds, and a piece's results written and read.
    const size_t held = pre.rows == 16 ? 4 : a.c.dim == 64 ? 3 : a.c.dim == 128 ? 2 : 1;
    const double tile = pre.rows == 128 ? a.c.dim * 0.0077 : pre.rows == 32 ? 0.22 : 0.18, alone = pre.rows == 128 ? 1.4 * tile : tile, start = 5.0, join = (double)rows * a.c.dim * 8.0 / 4e6 + 0.05;
    size_t pieces = 1;
    double best = 0.0;
    for (size_t n = 1; n <= (all + 3) / 4 && n <= 256; ++n) {
        const size_t wgs = units * kv * n, full = wgs / (held * cus), rest = wgs % (held * cus), per_piece = (all + n - 1) / n;
        auto round = [&](size_t m) {
            const double t = (double)((m + cus - 1) / cus) * tile;
            return (double)per_piece * (t > alone ? t : alone) + start;
        };
        const double t = (double)full * round(held * cus) + (rest ? round(rest) : 0.0) + (double)n * join;
        if (n == 1 || t < best) {
            best = t;
            pieces = n;
        }
    }
    if (!cut(pre, units * kv, all, pieces)) return AH_ERR_INVALID_ARG;
    // (four tiles a piece or more: a wave each)
    size_t fill = 2 * cus / own_units;
    fill = fill < (tiles + 3) / 4 ? fill : (tiles + 3) / 4;
    if (!cut(own, own_units, tiles, fill)) return AH_ERR_INVALID_ARG;
    a.splits = pre.splits + own.splits;
    AH_HIP(ctx, hipSetDevice(ctx->device));
    const int32_t st = attn_scratch(ctx, a, rows, 0, stream);
    if (st) return st;
    pre.part_o = a.part_o;
    pre.part_ml = a.part_ml;
    own.part_o = a.part_o + (size_t)pre.splits * rows * a.c.dim;
    own.part_ml = a.part_ml + (size_t)pre.splits * rows * 2;
    AH_HIP(ctx, ah_launch_attn_shared(pre, own, a, pick(ctx, stream)));
    return AH_OK;
}

// Block sizes that the pages are cut into.
static bool block_ok(const ah_kv4 *cache, size_t len) {
    return len >= 32 && !(len & (len - 1)) && len <= (size_t)1 << cache->ref.page_shift;
}

int32_t ah_kv4_block_means_dev(ah_ctx *ctx, const ah_kv4 *cache, const ah_kv4_tokens *tokens, size_t block_len, uint16_t *d_means, void *stream) {
    if (!ctx || !cache || !tokens || !block_ok(cache, block_len)) return AH_ERR_INVALID_ARG;
    if (tokens->n_tok == 0) return AH_OK;
    if (!tokens_ok(tokens) || !d_means || (reinterpret_cast<uintptr_t>(d_means) & 15) || tokens->n_tok > max_grid(256)) return AH_ERR_INVALID_ARG;
    MeansArgs a = {cache->ref, tokens_of(tokens), (uint32_t)__builtin_ctzll(block_len), d_means, ctx->d_status};
    AH_HIP(ctx, hipSetDevice(ctx->device));
    AH_HIP(ctx, ah_launch_block_means(a, pick(ctx, stream)));
    return AH_OK;
}

int32_t ah_kv4_attn_blocks_dev(ah_ctx *ctx, const ah_kv4 *cache, const ah_kv4_attn *p, const ah_kv4_blocks *blocks, const float *d_q,
                               size_t q_stride, float *d_out, size_t out_stride, int32_t *d_chosen, void *stream) {
    if (!ctx || !cache || !p || !blocks || p->window || p->sinks || !block_ok(cache, blocks->block_len) || blocks->n_top == 0 ||
        blocks->n_top > 4096 || blocks->n_first > 4096 || blocks->n_last > 4096)
        return AH_ERR_INVALID_ARG;
    if (empty(p)) return AH_OK;
    BlockArgs b = {};
    const int32_t bad = attn_args(ctx, cache, p, d_q, q_stride, d_out, out_stride, b.a);
    if (bad) return bad;
    AttnArgs &a = b.a;
    const size_t units = (size_t)a.n_tok * a.c.n_kv, per_page = ((size_t)1 << a.c.page_shift) / blocks->block_len;
    if (!blocks->d_means || (reinterpret_cast<uintptr_t>(blocks->d_means) & 15) || units > max_grid(256) || a.group > 4096 ||
        overlap(d_q, q_stride, a.n_heads * a.c.dim, d_out, out_stride, a.n_heads * a.c.dim, a.n_tok))
        return AH_ERR_INVALID_ARG;
    b.means = blocks->d_means;
    b.shift = (uint32_t)__builtin_ctzll(blocks->block_len);
    b.top = (uint32_t)blocks->n_top;
    b.first = (uint32_t)blocks->n_first;
    b.last = (uint32_t)blocks->n_last;
    b.chosen = d_chosen;
    // Lists, then the attention's partial results.  `room`: blocks that a table has pages for; `planned`: of the largest context
    // expected, which the choice's LDS and the attention's pieces go by (a table is as wide as the longest context allowed).
    const size_t places = a.table_stride * per_page, room = places < kMaxU32 / 32 ? places : kMaxU32 / 32;
    const size_t expected = p->max_ctx / blocks->block_len + (p->max_ctx % blocks->block_len != 0), planned = expected < room ? expected : room;
    const size_t read = b.top + (size_t)b.first + b.last + 1, entries = read < room ? read : room;
    a.list_stride = (uint32_t)entries + 1;
    a.block_shift = b.shift - 5;
    // Scores of a query's blocks in LDS (8 bytes), all of a context of the planned length; those of a longer one, or past what LDS
    // holds, go by passes behind the largest so far with their numbers (4 bytes).  `rows` queries; `more`: 8 bytes beside each.
    struct Fit {
        size_t keys, bytes;
    };
    auto fit = [&](size_t rows, size_t more) {
        const size_t least = b.top + (size_t)256 < room ? b.top + (size_t)256 : room;  // (a pass is 256 blocks and more)
        const size_t held = kChoiceLds / (8 * rows) - more, passes = held > b.top / 2 + 1 ? held - (b.top / 2 + 1) : 0;
        const size_t want = planned > least ? planned : least, keys = want <= held && want == room ? want : want < passes ? want : passes;
        return Fit{keys, rows * (keys + more) * 8 + (keys < room ? rows * b.top * 4 : 0)};
    };
    // 16 tokens of a sequence are chosen for together once every CU has two (token, KV head)s (four with heads of 256, whose
    // workgroups are smaller).  2 KV heads, 8192 keys, us a token for itself and together: heads of 128, 128 tokens of a sequence
    // 35 and 42, 256 51 and 51, 512 88 and 62, 64 x 4 55 and 50; of 256, 256 tokens 71 and 81, 512 124 and 97.  (Tiles of one or two
    // tokens: 512 x 1 104 and 112, 128 x 2 56 and 62.)  By passes too, where 16 tokens' scores outgrow LDS and one's don't: blocks
    // of 64, heads of 128, 2048 tokens over 70000, 100000 and 200000 keys 280 and 147, 321 and 158, 477 and 205, 512 over 100000 108 and
    // 93; of 256, 2048 over 100000 552 and 274; 400 blocks of 100000 2242 and 2107, 550 the same; past that a pass is too short.
    const Fit one = fit(1, 0), many = fit(16, a.c.dim + 3);
    const size_t tiles = (size_t)a.n_tok / 16 + a.n_seq;
    const bool together = a.max_q >= 4 && units >= (a.c.dim == 256 ? 4 : 2) * (size_t)ctx->cu_count && (many.keys == room || many.keys >= b.top + (size_t)128) &&
                          tiles * a.c.n_kv <= max_grid(1024);
    b.lds_keys = (uint32_t)(together ? many : one).keys;
    b.lds_bytes = (uint32_t)(together ? many : one).bytes;
    b.tiles = together ? (uint32_t)tiles : 0;
    if (!together && units > max_grid(1024)) return AH_ERR_INVALID_ARG;
    const size_t kept = align256(units * a.list_stride * sizeof(uint32_t));
    // Up to eight queries a KV head, and lists enough for four waves a CU and more: a wave each.  (us with a wave each and in
    // pieces, 2 KV heads, lists of 1152 keys: heads of 64, 512 lists 46 and 39, 1024 49 and 52; of 128 61 and 53, 63 and 74; of
    // 256 94 and 83, 98 and 119.)
    const bool alone = a.group <= 8 && together && units >= 4 * (size_t)ctx->cu_count;
    a.seqs = together ? a.n_seq : 0;
    AttnArgs rows = a;
    int32_t st;
    if (alone) {
        AH_HIP(ctx, hipSetDevice(ctx->device));
        st = ensure_scratch(ctx, kept, stream);
    } else {
        rows.n_seq = a.n_tok;  // every token for itself
        st = attn_rows_plan(ctx, rows, (planned < entries ? planned : entries) << a.block_shift, a.group, kept, stream);
    }
    if (st) return st;
    b.list = static_cast<uint32_t *>(ctx->scratch.p);
    rows.list = b.list;
    AH_HIP(ctx, ah_launch_block_choice(b, pick(ctx, stream)));
    if (alone) AH_HIP(ctx, ah_launch_attend_lists(rows, pick(ctx, stream)));
    else AH_HIP(ctx, ah_launch_attn_some(rows, pick(ctx, stream)));
    return AH_OK;
}

int32_t ah_sample_dev(ah_ctx *ctx, const float *d_logits, size_t row_stride, size_t n_rows, size_t n_vocab,
                      const ah_sample_params *params, const float *d_u, int32_t *d_tokens, float *d_probs, void *stream) {
    if (!ctx || n_rows > 65536 || n_vocab > (1u << 20)) return AH_ERR_INVALID_ARG;
    if (n_rows == 0) return AH_OK;
    if (n_vocab == 0 || row_stride < n_vocab || !d_logits || !d_u || !d_tokens) return AH_ERR_INVALID_ARG;
    SampleArgs a = {};
    a.logits = d_logits;
    a.stride = row_stride;
    a.n_rows = (uint32_t)n_rows;
    a.n_vocab = (uint32_t)n_vocab;
    if (params) {
        a.temperature = params->d_temperature;
        a.top_k = params->d_top_k;
        a.top_p = params->d_top_p;
        a.min_p = params->d_min_p;
    }
    a.u = d_u;
    a.tokens = d_tokens;
    a.probs = d_probs;
    a.status = ctx->d_status;
    a.arrived = ctx->d_count;
    a.n_counts = (uint32_t)kCounts;
    AH_HIP(ctx, hipSetDevice(ctx->device));
    const uint32_t cus = (uint32_t)ctx->cu_count;
    const int32_t st = ensure_scratch(ctx, ah_sample_plan(a, cus, nullptr), stream);
    if (st) return st;
    (void)ah_sample_plan(a, cus, static_cast<uint8_t *>(ctx->scratch.p));
    AH_HIP(ctx, ah_launch_sample(a, pick(ctx, stream)));
    return AH_OK;
}

} // extern "C"
