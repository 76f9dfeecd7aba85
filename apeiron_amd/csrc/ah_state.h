// ah_state.h -- launch arguments of a recurrent layer's operators (ah_state.hip): the short causal convolution and
// the gated delta rule, whose sequences carry a state of fixed size from call to call in a slot of the caller's memory.
#pragma once

#include "ah_internal.h"

struct StateSeqs {
    const int32_t *q_start, *from, *to;  // [n_seq + 1], [n_seq], [n_seq]
    uint32_t n_seq, n_tok, max_q, n_slots;
};

constexpr uint32_t kConvMaxWidth = 8, kConvTile = 8;  // tokens of a workgroup: W - 1 at least
struct ConvArgs {
    StateSeqs s;
    const float *x, *weight, *bias;
    float *y, *state;
    uint64_t x_stride, y_stride;
    uint32_t n_ch, width, silu;
    uint32_t tiles, per;  // numbers that tiles of tokens have, those of every sequence (0: they differ)
    unsigned long long *status;
};

struct DeltaArgs {
    StateSeqs s;
    const float *q, *k, *v, *a, *b, *a_log, *dt_bias;
    float *out, *state;
    uint64_t q_stride, k_stride, v_stride, a_stride, b_stride, out_stride;
    uint32_t n_heads, group, k_dim, v_dim;  // group: heads that share a head of q and k
    float scale, norm_eps;                  // norm_eps < 0: q and k are taken as they are
    // Sequences of chunk_from tokens or more go by chunks of 64, the others token by token.  What the chunks' preparation leaves
    // is a block of delta_block_bytes for every (slot, head); sequence s has its chunks' slots from
    // (q_start[s] >> slot_shift) + s * slot_seq on.
    uint32_t chunk_from, longs, slots, slot_shift, slot_seq;  // longs: at most so many go by chunks
    uint32_t tiles;  // of 16 columns of S for a workgroup of the chain: 1, 2 or 4
    uint8_t *blocks;
    uint32_t chain_grid;  // workgroups of the chain; a launch may have others after them
    // By groups of ring / 2 chunks (0: all at once): what a launch's chain begins with, the first chunk that it prepares, and S
    // of every (sequence, head) between two launches.
    uint32_t ring, begin, prepared;
    float *carry;
    unsigned long long *status;
};

constexpr uint32_t kDeltaChunk = 64;
// A chunk's block: fragments (1 KB: 16 bytes of each lane, f16 operands of v_mfma_f32_16x16x32_f16) of W, of the decayed keys,
// of q and of P, each as a half that is the f16 value and one that is the rest; U0 as f32; factors.
struct DeltaBlock {
    uint32_t w, k, q, p, u, f, bytes;  // offsets
};
__host__ __device__ inline constexpr DeltaBlock delta_block(uint32_t dk, uint32_t dv) {
    const uint32_t rows = 4 * (dk / 32) * 2048, w = 0, k = w + rows, q = k + rows, p = q + rows, u = p + 6 * 2048, f = u + (dv / 16) * 4096;
    return {w, k, q, p, u, f, f + 1024};
}
// Factors, in floats: of o's rows from S (the inverse scales of q's rows in them); then W's largest magnitude and inverse scale,
// each [tile of tokens][slice of 32 channels]; the inverse scales of the keys by slice; U0's largest magnitude by columns; e^(the
// chunk's decay); of o's rows from P (the inverse scales of q's and P's rows in them).
constexpr uint32_t kFRow = 0, kFWMax = 64, kFW = 80, kFK = 96, kFU = 108, kFDecay = 124, kFP = 128;

hipError_t ah_launch_conv(const ConvArgs &a, hipStream_t stream);
hipError_t ah_launch_delta(const DeltaArgs &a, bool steps, bool chunks, hipStream_t stream);
hipError_t ah_state_init_attrs();
