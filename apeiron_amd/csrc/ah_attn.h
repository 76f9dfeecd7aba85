// ah_attn.h -- what the kernels of attention over the 4-bit cache share (ah_attn.hip, ah_blocks.hip): a tile's codes as
// operands, q's two halves, a sequence's tokens and keys.
#pragma once

#include "ah_kv4.h"
#include "ah_seqs.h"

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Cache policy of the partial results that one workgroup writes and another reads in the same launch: device
// scope (sc1), past the XCDs' own L2s.
constexpr int kDevice = 16;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNoMax = -3.402823466e38f;  // below every finite score
// The running maximum follows the scores only when one passes it by more than this (in powers of two):
// then p <= 2^kSlack, and a rescale of the accumulators is rare after the first tiles.
constexpr float kSlack = 4.0f;
// p is kept times 2^kUp: two f16 halves hold it within 2^-23 of itself or 2^-36 of the largest weight, whichever is
// more (f16's subnormals are 2^-24 apart), and the largest, 2^(kUp + kSlack), is a finite f16.
constexpr float kUp = 11.0f;

AH_DEV f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

AH_DEV f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// Codes as f16 values.  1024 + c has c in its lowest mantissa bits, 1024 + 16 c in the next four:
// (1024 + c) - 1032, (1024 + 16 c) / 16 - 72 and the products by d are exact.  The masks stay in registers
// (an instruction takes one constant from outside them), so a pair is one v_and_or and two packed steps.
struct Masks {
    uint32_t low, high;
    AH_DEV Masks() : low(0x000F000Fu), high(0x00F000F0u) { __asm__("" : "+v"(low), "+v"(high)); }
};
AH_DEV f16x2 low_nibbles(uint32_t w, const Masks &k) {
    return __builtin_bit_cast(f16x2, (w & k.low) | 0x64006400u) - (f16x2)((_Float16)1032.0f);
}
AH_DEV f16x2 high_nibbles(uint32_t w, const Masks &k) {
    return __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (w & k.high) | 0x64006400u), (f16x2)((_Float16)0.0625f), (f16x2)((_Float16)-72.0f));
}
AH_DEV f16x8 join8(f16x2 a, f16x2 b, f16x2 c, f16x2 d) {
    return (f16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
AH_DEV f16x2 pair_of(uint32_t h) { return __builtin_bit_cast(f16x2, (h & 0xffffu) | h << 16); }
// Eight channels of a K row: a dword's nibbles 0 and 4, 1 and 5, 2 and 6, 3 and 7.
AH_DEV f16x8 k_frag(uint32_t w, f16x2 d, const Masks &k) {
    const uint32_t v = w >> 8;
    return join8(low_nibbles(w, k) * d, high_nibbles(w, k) * d, low_nibbles(v, k) * d, high_nibbles(v, k) * d);
}
// The eight tokens' values of both channels of a pair: two dwords, four tokens each.
AH_DEV void v_frags(uint32_t w0, uint32_t w1, f16x8 d, const Masks &k, f16x8 &even, f16x8 &odd) {
    const f16x2 d0 = {d[0], d[1]}, d1 = {d[2], d[3]}, d2 = {d[4], d[5]}, d3 = {d[6], d[7]};
    const uint32_t u0 = w0 >> 8, u1 = w1 >> 8;
    even = join8(low_nibbles(w0, k) * d0, low_nibbles(u0, k) * d1, low_nibbles(w1, k) * d2, low_nibbles(u1, k) * d3);
    odd = join8(high_nibbles(w0, k) * d0, high_nibbles(u0, k) * d1, high_nibbles(w1, k) * d2, high_nibbles(u1, k) * d3);
}

AH_DEV float xor_lanes(float v, int mask) { return __shfl_xor(v, mask, 64); }

// One lane's part of a tile.
template <int D> struct KTile {
    u32x4 w[D / 64];                       // codes (ah_kv4.h)
    uint32_t d[D == 256 ? 2 : 1];          // both half-tiles' scales of the lane's channels
    AH_DEV void load(const uint8_t *t, uint32_t r, uint32_t h) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c) __builtin_memcpy(&w[c], t + c * 1024 + (r * 4 + h) * 16, 16);
        __builtin_memcpy(d, t + 32 * D + (r * (D / 32) + (D == 64 ? h >> 1 : D == 128 ? h : 2 * h)) * 4, D == 256 ? 8 : 4);
    }
    AH_DEV uint32_t code(int half, int j) const {
        return D == 64 ? w[0][2 * half + j] : w[half * (D / 128) + j / 4][j & 3];
    }
    AH_DEV f16x2 scale(int half, int j) const {
        const uint32_t v = d[D == 256 ? j / 4 : 0];
        return pair_of(half ? v >> 16 : v);
    }
};
template <int D> struct VTile {
    u32x4 w[D / 64];
    f16x8 d[D / 32];
    AH_DEV void load(const uint8_t *t, uint32_t r, uint32_t h) {
#pragma unroll
        for (int c = 0; c < D / 64; ++c) __builtin_memcpy(&w[c], t + 16 * D + (c * 16 + r) * 64 + h * 16, 16);
#pragma unroll
        for (int g = 0; g < D / 32; ++g) __builtin_memcpy(&d[g], t + 34 * D + (g * 4 + h) * 16, 16);
    }
};

AH_DEV float ror8(float v) {  // lane r ^ 8 of each 16 (a rotation by 8)
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128, 0xF, 0xF, true));
}
AH_DEV f16x2 pack16(float a, float b) { return __builtin_convertvector((f32x2){a, b}, f16x2); }  // to nearest: what is cut off has no bias

// q's power-of-two scale: `up` makes the row's largest magnitude (of `top` over its lanes) lie in [2^13, 2^14) and
// carries the scale's sign; scores times f are in powers of two.  f > 0, so that the largest product is also
// the largest score and a masked -inf stays that.
AH_DEV void q_scale(float scale, float top, float &up, float &f) {
    int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;  // top in [2^e, 2^(e+1))
    e = e < -100 ? -100 : e > 127 ? 127 : e;
    up = __builtin_ldexpf(1.0f, 13 - e);
    f = __builtin_fmaxf(__builtin_fabsf(scale) * kLog2e * __builtin_ldexpf(1.0f, e - 13), 0x1p-126f);
    up = scale == 0.0f ? 0.0f : scale < 0.0f ? -up : scale > 0.0f ? up : scale;
}

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

template <class S, class H> AH_DEV uint32_t sequence_of(const AttnArgs &a, uint32_t at, S start, H holds) {
    return sequence_among(a.q_start, a.n_seq, a.n_tok, at, start, holds);
}

} // namespace
