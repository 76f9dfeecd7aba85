// ah_state.h -- launch arguments of a recurrent layer's operators (ah_state.hip): the short causal convolution and
// the gated delta rule, whose sequences carry a state of fixed size from call to call in a slot of the caller's memory.
#pragma once

#include "ah_internal.h"

struct StateSeqs {
    const int32_t *q_start, *from, *to;  // [n_seq + 1], [n_seq], [n_seq]
    uint32_t n_seq, n_tok, max_q, n_slots;
};

constexpr uint32_t kConvMaxWidth = 8;
struct ConvArgs {
    StateSeqs s;
    const float *x, *weight, *bias;
    float *y, *state;
    uint64_t x_stride, y_stride;
    uint32_t n_ch, width, silu;
    uint32_t tile, tiles, per;  // tokens of a workgroup, numbers that workgroups of tokens have, those of every sequence (0: they differ)
    unsigned long long *status;
};

struct DeltaArgs {
    StateSeqs s;
    const float *q, *k, *v, *a, *b, *a_log, *dt_bias;
    float *out, *state;
    uint64_t q_stride, k_stride, v_stride, a_stride, b_stride, out_stride;
    uint32_t n_heads, group, k_dim, v_dim;  // group: heads that share a head of q and k
    float scale, norm_eps;                  // norm_eps < 0: q and k are taken as they are
    unsigned long long *status;
};

hipError_t ah_launch_conv(const ConvArgs &a, hipStream_t stream);
hipError_t ah_launch_delta(const DeltaArgs &a, hipStream_t stream);
