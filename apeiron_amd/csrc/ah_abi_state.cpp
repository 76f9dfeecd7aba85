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
    // Tiles of 32 tokens; of 16 or 8 where those leave the CUs without four workgroups each.
    const bool even = n_tok == (size_t)a.s.n_seq * a.s.max_q || a.s.n_seq == 1;
    size_t tiles = 0;
    for (a.tile = 32;; a.tile /= 2) {
        a.per = even ? (uint32_t)((max_q + a.tile - 1) / a.tile) : 0;
        tiles = even ? (size_t)a.per * a.s.n_seq : n_tok / a.tile + a.s.n_seq;
        if (a.tile == 8 || tiles * blocks >= 4 * (size_t)ctx->cu_count) break;
    }
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
    // A sequence of up to 8 tokens goes token by token, a longer one by chunks.  Sequences of one length all go the same way.
    const size_t most_steps = 8;
    const bool chunks = a.s.max_q > most_steps, even = a.s.n_seq == 1 || n == (size_t)a.s.n_seq * a.s.max_q;
    a.chunk_from = !chunks ? 0xffffffffu : even ? 0 : (uint32_t)most_steps + 1;
    if (chunks) {
        // slots for the chunks: one for every 64 tokens and one more for every sequence, or one for every 8 tokens
        const size_t by_seq = n / kDeltaChunk + a.s.n_seq, by_tokens = n / most_steps + 1;
        a.slot_seq = even || by_seq <= by_tokens;
        a.slot_shift = a.slot_seq ? 6 : 3;
        const size_t slots = a.slot_seq ? by_seq : by_tokens;
        if (slots * H > kMaxGrid || (size_t)a.s.n_seq * H * (dv / 16) > kMaxGrid / 2) return AH_ERR_INVALID_ARG;
        a.slots = (uint32_t)slots;
        const size_t most = (size_t)a.s.n_seq * H * (dv / 16);
        a.tiles = most >= 4 * (size_t)ctx->cu_count ? 4 : most > (size_t)ctx->cu_count ? 2 : 1;
        const int32_t st = ensure_scratch(ctx, slots * H * delta_block((uint32_t)dk, (uint32_t)dv).bytes, stream);
        if (st) return st;
        a.blocks = static_cast<uint8_t *>(ctx->scratch.p);
    }
    AH_HIP(ctx, ah_launch_delta(a, !chunks || !even, chunks, pick(ctx, stream)));
    return AH_OK;
}

} // extern "C"
