// ah_host.h -- the device context and the host helpers that every entry point shares.
#pragma once

#include <hip/hip_runtime.h>

#include "apeiron_hip.h"

// Counters by which workgroups of a launch find the last of them: a unit's of a split attention, a row's of sampling.
constexpr size_t kCounts = 65536;

struct ah_ctx {
    int device = -1;
    uint8_t *noalloc = nullptr;  // this device's copy of the no-alloc scratch (ah_abi.cpp)
    hipStream_t stream = nullptr;
    // Two status words: [0] every call's refusals; [1] the refusals of a fused FFN's down
    // projection, reported only when [0] holds none (the reference refuses the FFN at its first
    // failing step, so a refused hidden activation is never projected).
    unsigned long long *d_status = nullptr;
    uint32_t *d_count = nullptr;  // [kCounts], zero between calls
    int last_hip = 0;
    uint32_t last_bad_bits = 0;  // f16 bits behind the last AH_ERR_NONFINITE_SCALE
    int cu_count = 256;
    uint32_t design[32] = {};  // GEMM design per GGUF type (ah_set_gemm_design; 0 = AUTO)
    void *scratch = nullptr;  // device scratch for GEMM operands / host-form staging
    // the unfused prefill FFN's gate / up outputs when the caller keeps none (grown on demand)
    void *ffn_buf = nullptr;
    size_t ffn_buf_bytes = 0;
    uint32_t ffn_form = AH_FFN_PREFILL_AUTO;  // ah_set_ffn_prefill_form
    size_t scratch_bytes = 0;
    // streaming-GEMV occupancy by (type, LDS bytes): a runtime query per launch costs more host
    // time than a small GEMV takes on the device
    static constexpr int kOccSlots = 16;
    uint32_t occ_key[kOccSlots] = {};
    int occ_val[kOccSlots] = {};
    int occ_n = 0;
};

#define AH_HIP(ctx, call)                                                                       \
    do {                                                                                        \
        hipError_t e_ = (call);                                                                 \
        if (e_ != hipSuccess) {                                                                 \
            if (ctx) (ctx)->last_hip = (int)e_;                                                 \
            return AH_ERR_HIP;                                                                  \
        }                                                                                       \
    } while (0)

inline hipStream_t pick(ah_ctx *ctx, void *stream) {
    return stream ? static_cast<hipStream_t>(stream) : ctx->stream;
}

inline int32_t ensure_scratch(ah_ctx *ctx, size_t bytes) {
    if (bytes <= ctx->scratch_bytes) return AH_OK;
    if (ctx->scratch) {
        // the old scratch may still be read by queued kernels
        AH_HIP(ctx, hipDeviceSynchronize());
        AH_HIP(ctx, hipFree(ctx->scratch));
        ctx->scratch = nullptr;
        ctx->scratch_bytes = 0;
    }
    size_t want = bytes + (bytes >> 2) + 4096;
    if (hipMalloc(&ctx->scratch, want) != hipSuccess) {
        ctx->scratch = nullptr;
        return AH_ERR_OUT_OF_MEMORY;
    }
    ctx->scratch_bytes = want;
    return AH_OK;
}

inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }
