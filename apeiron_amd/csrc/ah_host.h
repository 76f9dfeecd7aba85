// ah_host.h -- the device context and the host helpers that every entry point shares.
#pragma once

#include <hip/hip_runtime.h>

#include <new>

#include "apeiron_hip.h"

// Counters by which workgroups of a launch find the last of them: a unit's of a split attention, a row's of sampling.
constexpr size_t kCounts = 65536;

// Device memory that a context's calls share and that grows with what they need.  A graph keeps the addresses of the
// calls captured into it, so memory that a captured call has used is not freed when it is outgrown: it is kept for the
// graph's replays until ah_destroy.
struct Grown {
    struct Old {
        void *p;
        Old *next;
    };
    void *p = nullptr;
    size_t bytes = 0, old_bytes = 0;
    Old *old = nullptr;
    bool captured = false;
};

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
    Grown scratch;  // GEMM operands, split partials, sampling's tables, host-form staging
    Grown ffn_buf;  // the unfused prefill FFN's gate / up outputs when the caller keeps none
    uint32_t ffn_form = AH_FFN_PREFILL_AUTO;  // ah_set_ffn_prefill_form
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

// `want` (at least `bytes`) bytes of g, if it has not `bytes` yet, for a call on `stream`.
inline int32_t grow(ah_ctx *ctx, Grown &g, size_t bytes, size_t want, void *stream) {
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(pick(ctx, stream), &capture) != hipSuccess) {
        (void)hipGetLastError();
        capture = hipStreamCaptureStatusActive;  // (kept for nothing rather than freed under a graph)
    }
    if (bytes > g.bytes) {
        AH_HIP(ctx, hipSetDevice(ctx->device));
        if (g.captured) {
            Grown::Old *o = new (std::nothrow) Grown::Old{g.p, g.old};
            if (!o) return AH_ERR_OUT_OF_MEMORY;
            g.old = o;
            g.old_bytes += g.bytes;
            const size_t more = g.bytes + (g.bytes >> 2);  // all that is kept stays under four times what is in use
            want = want < more ? more : want;
        } else if (g.p) {
            // the old memory may still be read by queued kernels
            AH_HIP(ctx, hipDeviceSynchronize());
            AH_HIP(ctx, hipFree(g.p));
        }
        g.p = nullptr;
        g.bytes = 0;
        g.captured = false;
        if (hipMalloc(&g.p, want) != hipSuccess) {
            g.p = nullptr;
            return AH_ERR_OUT_OF_MEMORY;
        }
        g.bytes = want;
    }
    g.captured = g.captured || (capture == hipStreamCaptureStatusActive && g.p);
    return AH_OK;
}
inline void release(Grown &g) {
    if (g.p) (void)hipFree(g.p);
    while (g.old) {
        Grown::Old *o = g.old;
        g.old = o->next;
        (void)hipFree(o->p);
        delete o;
    }
}

inline int32_t ensure_scratch(ah_ctx *ctx, size_t bytes, void *stream) {
    return grow(ctx, ctx->scratch, bytes, bytes + (bytes >> 2) + 4096, stream);
}

inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }
