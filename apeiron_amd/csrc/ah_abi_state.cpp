// ah_abi_state.cpp -- host side of a recurrent layer's operators: argument checks and the launches' shapes.
#include "ah_host.h"
#include "ah_state.h"

namespace {

constexpr size_t kMaxU32 = 0x7fffffff, kMaxGrid = 0xffffffffu / 256;  // (workgroups of 256 threads: under 2^32 threads)
constexpr size_t kMaxStride = (size_t)1 << 23;  // floats: 64 rows and more within a range-checked resource's 32 bits

// The sequences of a call; false where they are refused.
bool seqs_of(const ah_state_seqs *p, StateSeqs &s) {
    if (!p->d_q_start || !p->d_from || !p->d_to || p->n_seq > 65535 || p->n_tok > kMaxU32 || p->n_slots > kMaxU32) return false;
    s = {p->d_q_start, p->d_from, p->d_to, (uint32_t)p->n_seq, (uint32_t)p->n_tok, (uint32_t)(p->max_q < p->n_tok ? p->max_q : p->n_tok), (uint32_t)p->n_slots};
    return true;
}

} // namespace

extern "C" {

int32_t ah_conv_dev(ah_ctx *ctx, const ah_state_seqs *seqs, const ah_conv *p, const float *d_x, size_t x_stride, float *d_y, size_t y_stride,
                    void *stream) {
    if (!ctx || !seqs || !p || p->width < 2 || p->width > kConvMaxWidth || p->n_channels > ((size_t)1 << 20)) return AH_ERR_INVALID_ARG;
    if (seqs->n_seq == 0 || p->n_channels == 0) return AH_OK;
    ConvArgs a = {};
    if (!seqs_of(seqs, a.s) || !p->d_weight || !p->d_state) return AH_ERR_INVALID_ARG;
    const size_t C = p->n_channels, n_tok = a.s.n_tok;
    if (n_tok && (!d_x || !d_y || x_stride < C || y_stride < C || x_stride > kMaxStride || y_stride > kMaxStride || overlap(d_x, x_stride, C, d_y, y_stride, C, n_tok))) return AH_ERR_INVALID_ARG;
    a.x = d_x;
    a.y = d_y;
    a.x_stride = x_stride;
    a.y_stride = y_stride;
    a.weight = p->d_weight;
    a.bias = p->d_bias;
    a.state = p->d_state;
    a.n_ch = (uint32_t)C;
    a.width = (uint32_t)p->width;
    a.silu = p->silu != 0;
    a.status = ctx->d_status;
    const size_t blocks = (C + 1023) / 1024, max_q = a.s.max_q ? a.s.max_q : 1;
    const bool even = n_tok == (size_t)a.s.n_seq * a.s.max_q || a.s.n_seq == 1;
    a.per = even ? (uint32_t)((max_q + kConvTile - 1) / kConvTile) : 0;
    const size_t tiles = even ? (size_t)a.per * a.s.n_seq : n_tok / kConvTile + a.s.n_seq;
    if (tiles > kMaxGrid / blocks) return AH_ERR_INVALID_ARG;
    a.tiles = (uint32_t)tiles;
    AH_HIP(ctx, hipSetDevice(ctx->device));
    AH_HIP(ctx, ah_launch_conv(a, pick(ctx, stream)));
    return AH_OK;
}

int32_t ah_delta_rule_dev(ah_ctx *ctx, const ah_state_seqs *seqs, const ah_delta_rule *p, const float *d_q, size_t q_stride, const float *d_k,
                          size_t k_stride, const float *d_v, size_t v_stride, const float *d_a, size_t a_stride, const float *d_b, size_t b_stride,
                          float *d_out, size_t out_stride, void *stream) {
    if (!ctx || !seqs || !p) return AH_ERR_INVALID_ARG;
    const size_t H = p->n_heads, K = p->n_k_heads, dk = p->k_dim, dv = p->v_dim;
    if ((dk != 64 && dk != 128) || (dv != 64 && dv != 128 && dv != 256) || H > 4096 || K == 0 || H % K || (p->d_a_log == nullptr) != (p->d_dt_bias == nullptr))
        return AH_ERR_INVALID_ARG;
    if (seqs->n_seq == 0 || H == 0) return AH_OK;
    DeltaArgs a = {};
    if (!seqs_of(seqs, a.s) || !p->d_state) return AH_ERR_INVALID_ARG;
    const size_t n = a.s.n_tok;
    if (n && (!d_q || !d_k || !d_v || !d_a || !d_b || !d_out || q_stride < K * dk || k_stride < K * dk || v_stride < H * dv || a_stride < H || b_stride < H ||
              out_stride < H * dv || overlap(d_q, q_stride, K * dk, d_out, out_stride, H * dv, n) || overlap(d_k, k_stride, K * dk, d_out, out_stride, H * dv, n) ||
              overlap(d_v, v_stride, H * dv, d_out, out_stride, H * dv, n) || overlap(d_a, a_stride, H, d_out, out_stride, H * dv, n) ||
              overlap(d_b, b_stride, H, d_out, out_stride, H * dv, n)))
        return AH_ERR_INVALID_ARG;
    if ((size_t)a.s.n_seq * H * (dv / 32) > kMaxU32 || out_stride > kMaxStride) return AH_ERR_INVALID_ARG;
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.a = d_a;
    a.b = d_b;
    a.a_log = p->d_a_log;
    a.dt_bias = p->d_dt_bias;
    a.out = d_out;
    a.state = p->d_state;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.a_stride = a_stride;
    a.b_stride = b_stride;
    a.out_stride = out_stride;
    a.n_heads = (uint32_t)H;
    a.group = (uint32_t)(H / K);
    a.k_dim = (uint32_t)dk;
    a.v_dim = (uint32_t)dv;
    a.scale = p->scale;
    a.norm_eps = p->norm_eps;
    a.status = ctx->d_status;
    AH_HIP(ctx, hipSetDevice(ctx->device));
    // A sequence of up to 8 tokens goes token by token, a longer one by chunks; the bound is 16 tokens where the batch gives
    // every CU a head and 24 where it gives two.  (Heads of 128 x 128, us by tokens and by chunks: 16 heads, 8 tokens 24.6 and
    // 23.9, 16 tokens 42 and 24; 256 heads, 16 tokens 51 and 57, 24 tokens 70 and 58; 512 heads, 24 tokens 76 and 90; 1024
    // heads, 16 tokens 110 and 165, 32 tokens 193 and 171.)  Sequences of one length all go the same way.
    const size_t cus = (size_t)ctx->cu_count, units = (size_t)a.s.n_seq * H, most_steps = units < cus ? 8 : units < 2 * cus ? 16 : 24;
    const bool chunks = a.s.max_q > most_steps, even = a.s.n_seq == 1 || n == (size_t)a.s.n_seq * a.s.max_q;
    a.chunk_from = !chunks ? 0xffffffffu : even ? 0 : (uint32_t)most_steps + 1;
    if (!chunks && units * (dv / 32) > 4 * kMaxGrid) return AH_ERR_INVALID_ARG;
    if (chunks) {
        // (uneven: at most `longs` sequences go by chunks, and as many of the longest would have the batch's tokens)
        const size_t longest = n / (most_steps + 1), longs = even || longest > a.s.n_seq ? a.s.n_seq : longest, as_long = (n + a.s.max_q - 1) / a.s.max_q;
        const size_t columns = (even ? a.s.n_seq : as_long) * H * (dv / 16), bytes = delta_block((uint32_t)dk, (uint32_t)dv).bytes, per = (a.s.max_q + kDeltaChunk - 1) / kDeltaChunk;
        // A workgroup of the chain takes 16 columns of S; 32 or 64 where there are more of them than CUs and then than fill six
        // rounds: a chunk's block is read by fewer workgroups.  (16 heads of 128 x 128, us with 16, 32, 64: 1 x 64 tokens 25,
        // 25, 30; 2 x 301 35, 39, 52; 5 x 301 66, 62, 63; 4 x 2048 274, 205, 336; 8 x 1024 326, 241, 246; 16 x 512 410, 284,
        // 269; columns of 64: 64 x 512 1189, 801, 692.)  In an uneven batch, where `as_long` counts the single tokens in and their
        // workgroups stand beside the chain's, 32 from 7/8 of the CUs on.  (One of 512 among 16 single tokens, us with 16, 32: 12, 14,
        // 15, 16, 17 and 24 heads (192 to 384 columns) 43 and 45, 48 and 49, 53 and 49, 45 and 45, 55 and 51, 55 and 49; among 64 54 and
        // 53, 66 and 57, 64 and 60, 62 and 55, 69 and 63, 83 and 72; heads of 64 x 64, 24, 30 and 32 among 16: 35 and 36, 40 and 41, 37
        // and 38; among 256, 16 of 128 166 and 146; 16 of up to 301 220 and 157, with 64 143.)
        a.longs = (uint32_t)longs;
        a.tiles = columns >= 6 * cus ? 4 : columns > cus || (!even && 8 * columns >= 7 * cus) ? 2 : 1;
        // All chunks are prepared at once, or, where the chain leaves half of the CUs without work and the blocks would not
        // stay in the 256 MB of the last cache, by groups of as many as give every CU one, the next group's preparation beside a
        // group's chain.  (us at once and by groups: 16 heads, 4096 tokens (148 MB) 151 and 160, 6144 249 and 232, 8192 348 and
        // 304, 32768 1275 and 1169; 8 heads, 8192 tokens 239 and 234, 12000 374 and 332, 16384 554 and 444.)
        const size_t half = (cus + units - 1) / units;
        size_t need;
        if (even && columns <= cus / 2 && per * units * bytes > ((size_t)192 << 20)) {
            a.ring = 2 * (uint32_t)half;
            need = align256(a.s.n_seq * (size_t)a.ring * H * bytes) + units * dk * dv * sizeof(float);
        } else {
            // Slots for the chunks: one for every 64 tokens and one more for every sequence, or one for every 8 tokens, which is
            // fewer where most sequences have a few tokens (1023 of one token and one of 512, 8 heads: 0.2 GB rather than
            // 1.2, 268 us and 285).
            const size_t by_seq = n / kDeltaChunk + a.s.n_seq, by_tokens = n / 8 + 1;
            a.slot_seq = even || by_seq <= by_tokens;
            a.slot_shift = a.slot_seq ? 6 : 3;
            const size_t slots = a.slot_seq ? by_seq : by_tokens;
            const size_t alone = even ? 0 : (units * (dv / 32) + 7) / 8;  // workgroups of the sequences that go token by token
            if (slots * H > kMaxGrid / 2 || longs * H * (dv / 16) / a.tiles + alone > kMaxGrid / 2) return AH_ERR_INVALID_ARG;
            a.slots = (uint32_t)slots;
            need = slots * H * bytes;
        }
        const int32_t st = ensure_scratch(ctx, need, stream);
        if (st) return st;
        a.blocks = static_cast<uint8_t *>(ctx->scratch.p);
        if (a.ring) a.carry = reinterpret_cast<float *>(a.blocks + align256(a.s.n_seq * (size_t)a.ring * H * bytes));
    }
    AH_HIP(ctx, ah_launch_delta(a, !chunks || !even, chunks, pick(ctx, stream)));
    return AH_OK;
}

} // extern "C"
