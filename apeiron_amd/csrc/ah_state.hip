// ah_state.hip -- a recurrent layer's operators: the short causal convolution over its channels and the gated delta
// rule.  What a sequence carries from call to call is of fixed size and lies in a slot of the caller's memory: read
// from one slot (none: zeros), written to one (none: dropped), which may be the same.
#include "ah_seqs.h"
#include "ah_state.h"

namespace {

constexpr unsigned long long kKeyNonFinite = AH_ERR_NONFINITE_INPUT, kKeyRange = AH_ERR_CACHE_RANGE;

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Seq {
    uint32_t q0, nq;
    int32_t from, to;
    bool bad;
};
AH_DEV Seq seq_of(const StateSeqs &a, uint32_t s) {
    Seq p;
    const int32_t b = a.q_start[s], e = a.q_start[s + 1];
    p.from = a.from[s];
    p.to = a.to[s];
    p.bad = b < 0 || e < b || (uint32_t)e > a.n_tok || (uint32_t)(e - b) > a.max_q || p.from >= (int32_t)a.n_slots || p.to >= (int32_t)a.n_slots;
    p.q0 = p.bad ? 0 : (uint32_t)b;
    p.nq = p.bad ? 0 : (uint32_t)(e - b);
    return p;
}

// v / (1 + e^-v).  e^-v = 2^t (1 + r ln 2), t the f32 product v log2(e) and r what that rounding and log2(e)'s left out, a few
// last places of t; the quotient by v_rcp_f32 with a Newton step.  Past t = 100 the power is formed 2^-64 times as large (1 + it is
// it) and the quotient multiplied by as much, so that neither it nor v_rcp_f32's result leaves f32's normal numbers; below -130
// the result is -0 as it is there.  Within 6 2^-24 of the result, or half of f32's smallest number.  (5 x 1021 tokens of 4099
// channels with a library exponential and division: 41 us for 39.)
AH_DEV float silu(float v) {
    constexpr float kHi = -1.44269502162933349609f, kLo = -1.92596299112661746887e-8f, kLn2 = 0.69314718f;
    const float m = v < -130.0f ? -130.0f : v, w = __builtin_fminf(m, 130.0f);  // (past 130 the power is 0, and 1 + it 1)
    float t = w * kHi;
    __asm__("" : "+v"(t));  // (t - 64 of the rounded product, which r belongs to: no fused w kHi - 64)
    const float r = __builtin_fmaf(w, kHi, -t) + w * kLo;
    const bool far = t > 100.0f;
    float e = __builtin_amdgcn_exp2f(far ? t - 64.0f : t);
    e = __builtin_fmaf(e, r * kLn2, e);
    const float d = 1.0f + e, q = __builtin_amdgcn_rcpf(d);
    float y = m * q;
    y = __builtin_fmaf(__builtin_fmaf(-d, y, m), q, y);
    return far ? y * 0x1p-64f : y;
}
AH_DEV bool finite(float v) { return __builtin_fabsf(v) < __builtin_inff(); }
// 1 / sqrt(sum + eps): NaN, not 0, for a sum of squares that left f32, so that the row is refused rather than taken as zeros.
AH_DEV float inverse_norm(float sum, float eps) { return 1.0f / __builtin_sqrtf(sum + eps) + (sum - sum); }

// ---- the short causal convolution --------------------------------------------------------------------
//
// y_t = act(bias + sum_i w_i x_(t - W + 1 + i)).  A lane has four channels of a tile of eight tokens: it asks for the tile's
// rows and the W - 1 before them at once, so that no load waits for another.  Bytes bound it: x once, y once; the rows
// before a tile come from L2 a second time.  (64 to 8192 tokens of 1024 to 6144 channels: tiles of 8 86 us, of 16 91, of 32 93 at
// 8192 x 6144, 13.9, 15.9 and 21.9 at 512 x 6144, the smallest never behind by more than the noise.)  8192 x 6144 takes 86 us,
// 4.7 TB/s of the 5.0 that a copy reaches, 3831 tokens of 4099 channels 33.5 us, 4.0 TB/s (rows off the 16-byte grid); a token of
// 64 sequences, 12.7 MB, 8.4 us: a launch, the sequence's numbers, its rows and the writes, one after the other.  The tile that holds a sequence's first token
// alone reads the state and also writes the new one, so that both may lie in the same slot.  Rows come and go through
// range-checked resources: no branch stands between the loads.
static_assert(kConvTile >= kConvMaxWidth - 1, "the rows before a tile lie in the one before it");
AH_DEV f32x4 ld4(__amdgpu_buffer_rsrc_t r, uint32_t at) { return __builtin_bit_cast(f32x4, ah_ld128(r, 4 * at)); }
AH_DEV void st4(__amdgpu_buffer_rsrc_t r, uint32_t at, f32x4 v, uint32_t take) {
    if (take == 4) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, (int)(4 * at), 0, 0);
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 3; ++i) {
        const float x = v[i];
        if (i < take) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, x), r, (int)(4 * (at + i)), 0, 0);
    }
}

template <int W> __global__ void __launch_bounds__(256) conv_kernel(ConvArgs a) {
    const uint32_t at = blockIdx.x % a.tiles, block = blockIdx.x / a.tiles, c0 = 4 * (block * 256 + threadIdx.x);
    const uint32_t take = c0 >= a.n_ch ? 0 : a.n_ch - c0 < 4 ? a.n_ch - c0 : 4;
    const __amdgpu_buffer_rsrc_t wr = ah_rsrc(a.weight, 4 * a.n_ch * W);
    float w[4 * W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
        const f32x4 v = ld4(wr, c0 * W + 4 * j);
        __builtin_memcpy(w + 4 * j, &v, 16);
    }
    f32x4 bias = (f32x4)0.0f;
    if (a.bias) bias = ld4(ah_rsrc(a.bias, 4 * a.n_ch), c0);
    auto start = [&](uint32_t i) { return (uint32_t)a.s.q_start[i] / kConvTile + i; };
    auto holds = [&](uint32_t i) {
        const Seq p = seq_of(a.s, i);
        return !p.bad && at >= start(i) && at - start(i) < (p.nq ? (p.nq + kConvTile - 1) / kConvTile : 1);
    };
    const uint32_t s = a.per ? at / a.per : sequence_among(a.s.q_start, a.s.n_seq, a.s.n_tok, at, start, holds), n = at - (a.per ? s * a.per : start(s));
    const Seq p = seq_of(a.s, s);
    const uint32_t t0 = n * kConvTile;
    if (!p.bad && (n == 0 || t0 < p.nq)) {
        const uint32_t rows = t0 >= p.nq ? 0 : p.nq - t0 < kConvTile ? p.nq - t0 : kConvTile, x_stride = (uint32_t)a.x_stride, y_stride = (uint32_t)a.y_stride;
        const uint32_t back = n ? W - 1 : 0;  // rows of the tile before this one (a tile has at least as many)
        const __amdgpu_buffer_rsrc_t xr = ah_rsrc(a.x + (size_t)(p.q0 + t0 - back) * a.x_stride, rows + back ? 4 * ((rows + back - 1) * x_stride + a.n_ch) : 0);
        const __amdgpu_buffer_rsrc_t yr = ah_rsrc(a.y + (size_t)(p.q0 + t0) * a.y_stride, rows ? 4 * ((rows - 1) * y_stride + a.n_ch) : 0);
        const uint32_t slot = 4 * (W - 1) * a.n_ch;
        const __amdgpu_buffer_rsrc_t old = ah_rsrc(a.state + (size_t)(p.from < 0 ? 0 : p.from) * (W - 1) * a.n_ch, p.from < 0 ? 0 : slot);
        f32x4 row[W - 1], now[kConvTile];
#pragma unroll
        for (uint32_t j = 0; j < W - 1; ++j) row[j] = n ? ld4(xr, j * x_stride + c0) : ld4(old, j * a.n_ch + c0);
#pragma unroll
        for (uint32_t j = 0; j < kConvTile; ++j) now[j] = ld4(xr, (back + j) * x_stride + c0);
        if (n == 0 && p.to >= 0) {  // the last W - 1 of the state's rows and the sequence's
            const __amdgpu_buffer_rsrc_t to = ah_rsrc(a.state + (size_t)p.to * (W - 1) * a.n_ch, slot);
            const uint32_t first = p.nq < W - 1 ? 0 : p.nq - (W - 1);
            const __amdgpu_buffer_rsrc_t end = ah_rsrc(a.x + (size_t)(p.q0 + first) * a.x_stride, p.nq ? 4 * ((p.nq - first - 1) * x_stride + a.n_ch) : 0);
            f32x4 kept[W - 1];
#pragma unroll
            for (uint32_t j = 0; j < W - 1; ++j)  // row nq + j of both, one after the other
                kept[j] = p.nq + j < W - 1 ? ld4(old, (p.nq + j) * a.n_ch + c0) : ld4(end, (p.nq + j - (W - 1) - first) * x_stride + c0);
#pragma unroll
            for (uint32_t j = 0; j < W - 1; ++j) st4(to, j * a.n_ch + c0, kept[j], take);
        }
        bool odd = false;
#pragma unroll
        for (uint32_t j = 0; j < kConvTile; ++j) {
            f32x4 out;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v = bias[i];
#pragma unroll
                for (int k = 0; k < W - 1; ++k) v = __builtin_fmaf(w[i * W + k], row[k][i], v);
                v = __builtin_fmaf(w[i * W + W - 1], now[j][i], v);
                odd = odd || ((uint32_t)i < take && j < rows && !finite(v));
                out[i] = a.silu ? silu(v) : v;
            }
            if (j < rows) st4(yr, j * y_stride + c0, out, take);
#pragma unroll
            for (int k = 0; k + 1 < W - 1; ++k) row[k] = row[k + 1];
            row[W - 2] = now[j];
        }
        if (odd) ah_record(a.status, ((unsigned long long)s << 8) + kKeyNonFinite);
    }
    if (block == 0 && threadIdx.x == 0) {
        if (a.per) {
            if (p.bad && n == 0) ah_record(a.status, ((unsigned long long)s << 8) + kKeyRange);
        } else {  // (a sequence out of range has no tile)
            for (uint32_t i = at; i < a.s.n_seq; i += a.tiles)
                if (seq_of(a.s, i).bad) ah_record(a.status, ((unsigned long long)i << 8) + kKeyRange);
        }
    }
}

// ---- the gated delta rule ----------------------------------------------------------------------------
//
// Token by token, with a head's S [k_dim][v_dim] in registers: S = e^g S, u = beta (v - S^T k), S += k u^T,
// o = scale S^T q.  A wave takes 32 columns of S: lane (r, c) = (lane >> 3, lane & 7) rows R r .. R r + R - 1 of columns
// 4 c .. 4 c + 3, so that a row's 32 columns are a line and the sums over rows cross eight lanes; columns do not depend on each
// other, and every one of them forms the token's norms, decay and rate anew rather than wait for one that does.
//   What bounds it: S's bytes, read once and written once (a token of 64 sequences, 16 heads of 128 x 128, 136 MB: 24 us, 5.6 TB/s,
// some of it from the last cache); a few tokens of few heads their chain, 2.2 us a token (rows, three sums, S's update).
AH_DEV float sum_rows(float v) {  // over the eight lanes of a column
    v += __shfl_xor(v, 8, 64);
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
// log(1 + e^x)
AH_DEV float softplus(float x) { return __builtin_fmaxf(x, 0.0f) + log1pf(expf(-__builtin_fabsf(x))); }
AH_DEV float decay_of(const DeltaArgs &a, float x, uint32_t h) { return a.a_log ? -expf(a.a_log[h]) * softplus(x + a.dt_bias[h]) : x; }
AH_DEV float rate_of(const DeltaArgs &a, float x) { return a.a_log ? 1.0f / (1.0f + expf(-x)) : x; }

template <int DK> AH_DEV void steps(const DeltaArgs &a, uint32_t unit) {  // a wave's (sequence, head, 32 columns)
    constexpr int R = DK / 8;
    const uint32_t lane = threadIdx.x & 63, r = lane >> 3, c = lane & 7, nvb = a.v_dim / 32;
    const uint32_t vb = unit % nvb, h = unit / nvb % a.n_heads, s = unit / nvb / a.n_heads;
    if (s >= a.s.n_seq) return;
    const Seq p = seq_of(a.s, s);
    if (p.bad && vb == 0 && h == 0 && lane == 0) ah_record(a.status, ((unsigned long long)s << 8) + kKeyRange);
    if (p.bad || p.nq >= a.chunk_from) return;
    const size_t tile = ((size_t)h * DK + R * r) * a.v_dim + 32 * vb + 4 * c, slot = (size_t)a.n_heads * DK * a.v_dim;
    f32x4 S[R];
    if (p.from >= 0) {
        const float *from = a.state + (size_t)p.from * slot + tile;
#pragma unroll
        for (int i = 0; i < R; ++i) __builtin_memcpy(&S[i], from + (size_t)i * a.v_dim, 16);
    } else {
#pragma unroll
        for (int i = 0; i < R; ++i) S[i] = (f32x4)0.0f;
    }
    bool odd = false;
    for (uint32_t t = 0; t < p.nq; ++t) {
        const size_t tok = p.q0 + t;
        float k[R], q[R];
        f32x4 v;
        __builtin_memcpy(k, a.k + tok * a.k_stride + (size_t)(h / a.group) * DK + R * r, 4 * R);
        __builtin_memcpy(q, a.q + tok * a.q_stride + (size_t)(h / a.group) * DK + R * r, 4 * R);
        __builtin_memcpy(&v, a.v + tok * a.v_stride + (size_t)h * a.v_dim + 32 * vb + 4 * c, 16);
        const float keep = expf(decay_of(a, a.a[tok * a.a_stride + h], h)), rate = rate_of(a, a.b[tok * a.b_stride + h]);
        float fk = 1.0f, fq = a.scale;
        if (a.norm_eps >= 0.0f) {
            float kk = 0.0f, qq = 0.0f;
#pragma unroll
            for (int i = 0; i < R; ++i) {
                kk = __builtin_fmaf(k[i], k[i], kk);
                qq = __builtin_fmaf(q[i], q[i], qq);
            }
            fk = inverse_norm(sum_rows(kk), a.norm_eps);
            fq *= inverse_norm(sum_rows(qq), a.norm_eps);
        }
        f32x4 m = (f32x4)0.0f, o = (f32x4)0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            S[i] *= keep;
            m += S[i] * k[i];
        }
        f32x4 u;
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = rate * (v[i] - fk * sum_rows(m[i]));
#pragma unroll
        for (int i = 0; i < R; ++i) {
            S[i] += (fk * k[i]) * u;
            o += S[i] * q[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[i] = fq * sum_rows(o[i]);
            odd = odd || !finite(o[i]) || !finite(u[i]);
        }
        if (r == 0) __builtin_memcpy(a.out + tok * a.out_stride + (size_t)h * a.v_dim + 32 * vb + 4 * c, &o, 16);
    }
    if (p.to >= 0) {
        float *to = a.state + (size_t)p.to * slot + tile;
#pragma unroll
        for (int i = 0; i < R; ++i) __builtin_memcpy(to + (size_t)i * a.v_dim, &S[i], 16);
    }
    if (odd) ah_record(a.status, ((unsigned long long)s << 8) + kKeyNonFinite);
}

template <int DK> __global__ void __launch_bounds__(256) delta_step_kernel(DeltaArgs a) {
    steps<DK>(a, 4 * blockIdx.x + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
}

// ---- the gated delta rule, by chunks -----------------------------------------------------------------
//
// With gamma_i the sum of g over a chunk's tokens up to i and D_ij = e^(gamma_i - gamma_j), the rule over 64 tokens is
//   A_ij = beta_i D_ij k_i . k_j (j < i),  T = (1 + A)^-1,  W = T (beta e^gamma k),  U0 = T (beta v),
//   U = U0 - W S,  o = scale (e^gamma q S + P U),  P_ij = D_ij q_i . k_j (j <= i),  S' = e^gamma_63 S + (e^(gamma_63 - gamma) k)^T U.
// delta_prepare_kernel makes W, U0, P and the decayed keys of all chunks at once; delta_chain_kernel then walks a sequence's
// chunks with S in registers, two products deep a chunk.  No exponent above a sum of g's is ever formed, and sums of g are f64.
//   Token by token a head's S passes registers once a token (8192 tokens of 16 heads: 20.7 ms); by chunks of 64 it takes 6 dk dv
// products of 64 tokens on the matrix cores and a chain 64 times shorter (306 us).  Shorter chunks have a longer chain, longer
// ones more of the triangle (T by recursion: 64 is four tiles of 16).
//   f32 by f16: every factor of a product is carried as hi + lo, two f16 of a value scaled by a power of two so that the largest
// of its group (a row of q, k or P, a tile, a slice, a chunk) lies in [2^13, 2^14): 22 bits, or 2^-38 of the group's largest.  Three products
// (hi hi, hi lo, lo hi) are summed in the f32 accumulator, at 5 times the rate of the f32 matrix instructions.
//   Tokens that are summed over share a scale (beta v: 64 of them, 16 columns; U: the same, by a bound of up to 32 dk / 32 times the
// largest |S| above it), so that U is held to 2^-31 of the largest |S| and 2^-37 of the largest |beta v|, and not to 22 bits of
// itself where a decay clears a far larger state within the chunk.
//   Layouts: a lane (r, h) = (lane & 15, lane >> 4) of a 16x16 product holds column r and rows 4 h + i of the result, and of an
// operand row (or column) r and a quarter of the 32 values that are summed over.  Which those are is free as long as both
// operands agree: rows 4 h + i of two neighbouring tiles.  So a result is the next product's operand where it lies.  Row m of the
// two tiles of a slice of 32 channels of S is channel 2 m of the slice in the one and 2 m + 1 in the other.
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

AH_DEV f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Two halves of an operand.
struct Frag {
    u32x4 hi, lo;
};
AH_DEV f16x2 pack16(float a, float b) { return __builtin_convertvector((f32x2){a, b}, f16x2); }
AH_DEV void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const f16x2 t = pack16(a, b);
    hi = __builtin_bit_cast(uint32_t, t);
    lo = __builtin_bit_cast(uint32_t, pack16(a - (float)t[0], b - (float)t[1]));
}
AH_DEV Frag split8(const float *x, float scale) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t hi, lo;
        split2(x[2 * i] * scale, x[2 * i + 1] * scale, hi, lo);
        f.hi[i] = hi;
        f.lo[i] = lo;
    }
    return f;
}
AH_DEV f32x4 mm3(const Frag &a, const Frag &b, f32x4 c) {
    c = mfma16(__builtin_bit_cast(f16x8, a.hi), __builtin_bit_cast(f16x8, b.hi), c);
    c = mfma16(__builtin_bit_cast(f16x8, a.hi), __builtin_bit_cast(f16x8, b.lo), c);
    return mfma16(__builtin_bit_cast(f16x8, a.lo), __builtin_bit_cast(f16x8, b.hi), c);
}
// The power of two that brings `top` into [2^13, 2^14), and its inverse.
struct Scale {
    float up, down;
};
AH_DEV Scale scale_of(float top) {
    int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
    e = e < -100 ? -100 : e > 127 ? 127 : e;
    return {__builtin_ldexpf(1.0f, 13 - e), __builtin_ldexpf(1.0f, e - 13)};
}
template <int CTRL> AH_DEV float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
AH_DEV float max16(float v) {  // over each 16 lanes
    v = __builtin_fmaxf(v, dpp<0x121>(v));  // rotations by 1, 2, 4 and 8
    v = __builtin_fmaxf(v, dpp<0x122>(v));
    v = __builtin_fmaxf(v, dpp<0x124>(v));
    return __builtin_fmaxf(v, dpp<0x128>(v));
}
AH_DEV float lane_of(float v, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); }
AH_DEV float wave_max(float v) {
    v = max16(v);
    return __builtin_fmaxf(__builtin_fmaxf(lane_of(v, 0), lane_of(v, 16)), __builtin_fmaxf(lane_of(v, 32), lane_of(v, 48)));
}
AH_DEV float top4(float top, f32x4 v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) top = __builtin_fmaxf(top, __builtin_fabsf(v[i]));
    return top;
}
// Of a tile of tokens and a step of 32 of them, the fragment's place among the six that a lower triangle has.
AH_DEV constexpr uint32_t tri(uint32_t tile, uint32_t step) { return tile < 2 ? tile : 2 * tile - 2 + step; }

// The chunk of a slot, and of which sequence: its first token, and how many there are (0: none).
struct Chunk {
    uint32_t s, tok0, live;
};
AH_DEV Chunk chunk_of(const DeltaArgs &a, uint32_t at) {
    auto within = [&](const Seq &p, uint32_t i) {
        const uint32_t first = ((uint32_t)p.q0 >> a.slot_shift) + i * a.slot_seq;
        return !p.bad && p.nq >= a.chunk_from && at >= first && at - first < (p.nq + kDeltaChunk - 1) / kDeltaChunk;
    };
    uint32_t s, q0, nq;
    if (a.s.n_seq <= 64) {  // a lane a sequence: one round trip to memory
        const uint32_t lane = threadIdx.x & 63, i = lane < a.s.n_seq ? lane : a.s.n_seq - 1;
        const Seq p = seq_of(a.s, i);
        const uint64_t found = __builtin_amdgcn_ballot_w64(within(p, i));
        if (!found) return {0, 0, 0};
        s = (uint32_t)__builtin_ctzll(found);
        q0 = (uint32_t)__builtin_amdgcn_readlane((int)p.q0, (int)s);
        nq = (uint32_t)__builtin_amdgcn_readlane((int)p.nq, (int)s);
    } else {
        auto first = [&](uint32_t i) { return ((uint32_t)a.s.q_start[i] >> a.slot_shift) + i * a.slot_seq; };
        auto holds = [&](uint32_t i) { return within(seq_of(a.s, i), i); };
        s = sequence_among(a.s.q_start, a.s.n_seq, a.s.n_tok, at, first, holds);
        const Seq p = seq_of(a.s, s);
        if (!within(p, s)) return {s, 0, 0};
        q0 = p.q0;
        nq = p.nq;
    }
    const uint32_t done = kDeltaChunk * (at - ((q0 >> a.slot_shift) + s * a.slot_seq)), rest = nq - done;
    return {s, q0 + done, rest < kDeltaChunk ? rest : kDeltaChunk};
}

// A product of 16x16 f32 blocks: x [16][ld] in LDS, y in registers as a result lies (lane (r, h): y[4 h + i][r]).
AH_DEV f32x4 block_product(const float *x, uint32_t ld, f32x4 y, f32x4 c, uint32_t r, uint32_t h) {
    f32x4 row;
    __builtin_memcpy(&row, x + r * ld + 4 * h, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(row[i], y[i], c, 0, 0, 0);
    return c;
}

constexpr uint32_t kLd = 68;  // floats of a row of the chunk's triangle in LDS
// A wave's rows of q or k from memory: lanes side by side on a row, 16 bytes each.  (A lane for a row and its quarter, as operands
// lie, takes 64 lines at once and four times as long.)
template <int DK> struct Rows {
    static constexpr uint32_t kLanes = DK / 4, kAtOnce = 64 / kLanes, kLoads = 16 / kAtOnce;  // of a row; rows of a load; loads of 16 rows
    f32x4 x[kLoads];
    static AH_DEV uint32_t row(uint32_t i, uint32_t lane) { return kAtOnce * i + lane / kLanes; }
    static AH_DEV uint32_t col(uint32_t lane) { return 4 * (lane % kLanes); }
};
AH_DEV float sum16(float v) {  // over each 16 lanes
    v += dpp<0x121>(v);
    v += dpp<0x122>(v);
    v += dpp<0x124>(v);
    return v + dpp<0x128>(v);
}

template <int DK> struct PrepareLds {
    _Float16 kh[64][DK + 8], kl[64][DK + 8];
    union {
        float A[64 * kLd];
        u32x4 t[6][2][64];
    };
    double gamma[64];
    float beta[64], fk[64], fq[64], fw[64], fd[64], tinv[4];  // (fk, fq: the rows' scales undone)
};
// Eight waves a chunk and head.  Waves 0 to 3 have the keys and beta_i k_i . k_j of 16 tokens i each, and make T of them; waves 4 to
// 7 have q of the same tokens, P and q's fragments.  W and U0 are shared by all.  Barriers wait for LDS alone: loads and stores stay
// on their way.  What bounds it is vector work beside the waits at barriers (62% of a SIMD's cycles while a CU works, products 9%):
// halves of every factor, T's recursion, the scales.  A chunk and head of 128 x 128 takes 26 us where two share a CU (5 x 301
// tokens, 16 heads), 2048 of them 110.
template <int DK> AH_DEV void prepare(const DeltaArgs &a, const Chunk &c, uint32_t hd, uint8_t *block, PrepareLds<DK> &L) {
    constexpr int NT = DK / 32;
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, h = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
    const bool keys = wave < 4;
    const uint32_t kh = hd / a.group, dv = a.v_dim;
    const DeltaBlock B = delta_block(DK, dv);
    float *fac = reinterpret_cast<float *>(block + B.f);
    typedef Rows<DK> R;
    R x;
    {
        const float *from = keys ? a.k : a.q;
        const size_t stride = keys ? a.k_stride : a.q_stride;
#pragma unroll
        for (uint32_t i = 0; i < R::kLoads; ++i) {
            const uint32_t t = 16 * w + R::row(i, lane);
            __builtin_memcpy(&x.x[i], from + (size_t)(c.tok0 + (t < c.live ? t : 0)) * stride + (size_t)kh * DK + R::col(lane), 16);
        }
    }
    if (wave == 7) {  // gates, a lane a token: gamma by a scan
        float beta = 0.0f, g = 0.0f;
        if (lane < c.live) {
            g = decay_of(a, a.a[(size_t)(c.tok0 + lane) * a.a_stride + hd], hd);
            g = g < -1000.0f ? -1000.0f : g;  // (e^g is 0 as well, and sums stay finite)
            beta = rate_of(a, a.b[(size_t)(c.tok0 + lane) * a.b_stride + hd]);
        }
        double gamma = g;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double v = __shfl_up(gamma, o, 64);
            gamma += (int)lane >= o ? v : 0.0;
        }
        L.gamma[lane] = gamma;
        L.beta[lane] = beta;
    }
    // Every row by a scale of its own: its length is no part of what it is to the rule, where it is divided by it (with one scale
    // for a chunk's 64 keys a key of 2^-20 of the longest kept 18 bits).
    float up[R::kLoads];
#pragma unroll
    for (uint32_t i = 0; i < R::kLoads; ++i) {
        const uint32_t t = 16 * w + R::row(i, lane);
        __asm__("" : "+v"(x.x[i]));  // (the loads themselves stay outside the choice)
        x.x[i] = t < c.live ? x.x[i] : (f32x4)0.0f;
        float sum = 0.0f, top = max16(top4(0.0f, x.x[i]));
#pragma unroll
        for (int n = 0; n < 4; ++n) sum = __builtin_fmaf(x.x[i][n], x.x[i][n], sum);
        sum = sum16(sum);
        if (DK == 128) {
            sum += __shfl_xor(sum, 16, 64);
            top = __builtin_fmaxf(top, __shfl_xor(top, 16, 64));
        }
        const Scale z = scale_of(top);
        up[i] = z.up;
        if (R::col(lane) == 0) {
            const float f = keys ? 1.0f : a.scale, v = a.norm_eps >= 0.0f ? f * inverse_norm(sum, a.norm_eps) : f;
            (keys ? L.fk : L.fq)[t] = t < c.live ? v * z.down : 0.0f;
        }
    }
    auto put_rows = [&] {
#pragma unroll
        for (uint32_t i = 0; i < R::kLoads; ++i) {
            const uint32_t t = 16 * w + R::row(i, lane), col = R::col(lane);
            uint32_t hi[2], lo[2];
            split2(x.x[i][0] * up[i], x.x[i][1] * up[i], hi[0], lo[0]);
            split2(x.x[i][2] * up[i], x.x[i][3] * up[i], hi[1], lo[1]);
            __builtin_memcpy(&L.kh[t][col], hi, 8);
            __builtin_memcpy(&L.kl[t][col], lo, 8);
        }
    };
    auto row_frag = [&](uint32_t t, int n) {  // eight channels a lane
        Frag f;
        __builtin_memcpy(&f.hi, &L.kh[t][32 * n + 8 * h], 16);
        __builtin_memcpy(&f.lo, &L.kl[t][32 * n + 8 * h], 16);
        return f;
    };
    auto store_frag = [&](uint32_t to, const Frag &f) {
        __builtin_memcpy(block + to + lane * 16, &f.hi, 16);
        __builtin_memcpy(block + to + 1024 + lane * 16, &f.lo, 16);
    };
    const uint32_t row = 16 * w + r;
    Frag f[NT];  // of the wave's rows
    if (!keys) {  // through the keys' place, before they are there
        put_rows();
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            f[t] = row_frag(row, t);
            // for the chain in the order of S: even channels, then odd ones
            auto halves = [](u32x4 v) {
                return (u32x4){__builtin_amdgcn_perm(v[1], v[0], 0x05040100), __builtin_amdgcn_perm(v[3], v[2], 0x05040100),
                               __builtin_amdgcn_perm(v[1], v[0], 0x07060302), __builtin_amdgcn_perm(v[3], v[2], 0x07060302)};
            };
            store_frag(B.q + (w * NT + t) * 2048, {halves(f[t].hi), halves(f[t].lo)});
        }
    }
    ah_lds_barrier();
    const double gr = L.gamma[row], all = L.gamma[63];
    if (keys) put_rows();
    else if (h == 0) fac[kFRow + row] = L.fq[row] * expf((float)gr);
    if (wave == 4) {  // e^gamma of each token to W's keys, what is left of the chunk's decay to the state's
        const double gamma = L.gamma[lane];
        L.fw[lane] = L.beta[lane] * expf((float)gamma) * L.fk[lane];
        L.fd[lane] = expf((float)(all - gamma)) * L.fk[lane];
        if (lane == 0) fac[kFDecay] = expf((float)all);
    }
    ah_lds_barrier();

    // k_j . k_i or k_j . q_i of the wave's tokens i and the tiles of j up to them: a lane has i = r, j = 16 t + 4 h + n
    if (keys) {
#pragma unroll
        for (int t = 0; t < NT; ++t) f[t] = row_frag(row, t);
    }
    const uint32_t end = keys ? row : row + 1;
    const float fr = keys ? L.beta[row] * L.fk[row] : 1.0f;  // (q's own length follows with o's rows)
    f32x4 p[4];
#pragma unroll
    for (uint32_t jt = 0; jt < 4; ++jt) {
        p[jt] = (f32x4)0.0f;
        if (jt > w) continue;
        float d[4];  // (formed for every lane: a branch for each would wait for each one's factors in turn)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const uint32_t j = 16 * jt + 4 * h + n;
            d[n] = fr * expf((float)(gr - L.gamma[j])) * L.fk[j];
            __asm__("" : "+v"(d[n]));
        }
        f32x4 v = (f32x4)0.0f, v1 = (f32x4)0.0f, v2 = (f32x4)0.0f;  // mm3's three sums, side by side
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const Frag g = row_frag(16 * jt + r, t);
            v = mfma16(__builtin_bit_cast(f16x8, g.hi), __builtin_bit_cast(f16x8, f[t].hi), v);
            v1 = mfma16(__builtin_bit_cast(f16x8, g.hi), __builtin_bit_cast(f16x8, f[t].lo), v1);
            v2 = mfma16(__builtin_bit_cast(f16x8, g.lo), __builtin_bit_cast(f16x8, f[t].hi), v2);
        }
        v += v1 + v2;
#pragma unroll
        for (int n = 0; n < 4; ++n) p[jt][n] = 16 * jt + 4 * h + n < end ? d[n] * v[n] : 0.0f;
        if (keys) __builtin_memcpy(&L.A[row * kLd + 16 * jt + 4 * h], &p[jt], 16);
    }
    // v's columns of this wave (every eighth 16), as operands that sum over the tokens: on their way while T is made
    f32x4 vx[4];
    auto load_v = [&](uint32_t cb) {
#pragma unroll
        for (uint32_t t = 0; t < 4; ++t)
#pragma unroll
            for (uint32_t n = 0; n < 4; ++n) {
                const uint32_t j = 16 * t + 4 * h + n;
                vx[t][n] = a.v[(size_t)(c.tok0 + (j < c.live ? j : 0)) * a.v_stride + (size_t)hd * dv + 16 * cb + r];
            }
    };
    const uint32_t cb_first = dv == 64 ? w : wave;  // (of four columns of tiles, the waves 4 to 7 take one each)
    const bool has_v = dv > 64 || !keys;
    if (has_v) load_v(cb_first);
    ah_lds_barrier();

    // T = (1 + A)^-1 in place: the diagonal blocks by substitution, a lane a column; then blocks of 32, then the whole
    const f32x4 zero = (f32x4)0.0f;
    auto at_block = [&](uint32_t i, uint32_t j) { return &L.A[16 * i * kLd + 16 * j]; };
    auto as_result = [&](const float *y) {  // a block as a result lies
        f32x4 v;
#pragma unroll
        for (int n = 0; n < 4; ++n) v[n] = y[(4 * h + n) * kLd + r];
        return v;
    };
    auto put = [&](float *y, f32x4 v) {
#pragma unroll
        for (int n = 0; n < 4; ++n) y[(4 * h + n) * kLd + r] = v[n];
    };
    if (keys) {
        float *D = &L.A[16 * w * kLd + 16 * w], y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float v = i == (int)r ? 1.0f : 0.0f;
#pragma unroll
            for (int m = 0; m < i; ++m) v = __builtin_fmaf(-D[i * kLd + m], y[m], v);
            y[i] = v;
        }
        if (h == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) D[i * kLd + r] = y[i];
        }
    } else {  // P of the wave's tokens
        float most = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t) most = top4(most, p[t]);
        most = __builtin_fmaxf(most, __shfl_xor(most, 16, 64));
        const Scale s = scale_of(__builtin_fmaxf(most, __shfl_xor(most, 32, 64)));  // of the row
        if (h == 0) fac[kFP + row] = L.fq[row] * s.down;
#pragma unroll
        for (uint32_t t = 0; t < 2; ++t) {
            if (t == 1 && w < 2) continue;
            float y[8];
            __builtin_memcpy(y, &p[2 * t], 32);
            store_frag(B.p + tri(w, t) * 2048, split8(y, s.up));
        }
    }
    ah_lds_barrier();
    if (wave < 2) {
        const uint32_t b = 2 * w;
        const f32x4 y = block_product(at_block(b + 1, b), kLd, as_result(at_block(b, b)), zero, r, h);
        put(at_block(b + 1, b), -block_product(at_block(b + 1, b + 1), kLd, y, zero, r, h));
    }
    ah_lds_barrier();
    f32x4 z = zero;
    const uint32_t col = w & 1, low = w >> 1;  // block (2 + low, col)
    if (keys) {
        for (uint32_t m = 0; m <= low; ++m) {
            f32x4 y = zero;
            for (uint32_t n = col; n < 2; ++n) y = block_product(at_block(2 + m, n), kLd, as_result(at_block(n, col)), y, r, h);
            z = block_product(at_block(2 + low, 2 + m), kLd, y, z, r, h);
        }
    }
    ah_lds_barrier();
    if (keys) put(at_block(2 + low, col), -z);
    ah_lds_barrier();
    {  // the wave's rows of T as operands, in T's place
        float y[2][8], most = 0.0f;
#pragma unroll
        for (uint32_t t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const uint32_t tile = 2 * t + n / 4;
                y[t][n] = keys && tile <= w ? L.A[row * kLd + 16 * tile + 4 * h + (n & 3)] : 0.0f;
                most = __builtin_fmaxf(most, __builtin_fabsf(y[t][n]));
            }
        const Scale s = scale_of(wave_max(most));
        ah_lds_barrier();
        if (keys) {
            if (lane == 0) L.tinv[w] = s.down;
#pragma unroll
            for (uint32_t t = 0; t < 2; ++t) {
                if (t == 1 && w < 2) continue;
                const Frag g = split8(y[t], s.up);
                L.t[tri(w, t)][0][lane] = g.hi;
                L.t[tri(w, t)][1][lane] = g.lo;
            }
        }
    }
    ah_lds_barrier();
    auto t_frag = [&](uint32_t tile, uint32_t t) { return Frag{L.t[tri(tile, t)][0][lane], L.t[tri(tile, t)][1][lane]}; };
    // A slice of 32 channels of the keys, by two waves (w and w + 4), with the tokens as what is summed over: W's transpose (a lane
    // has token r and channels 4 h + n) of two tiles of tokens each, and the decayed keys of every other channel each.
    if (w < (uint32_t)NT) {
        const uint32_t half = wave >> 2;
        float y[2][2][8], fw[2][8], fd[2][8], wt = 0.0f, dt = 0.0f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const uint32_t j = 32 * t + 16 * (n / 4) + 4 * h + (n & 3);
                fw[t][n] = L.fw[j];
                fd[t][n] = L.fd[j];
                f16x2 hi, lo;
                __builtin_memcpy(&hi, &L.kh[j][32 * w + 2 * r], 4);
                __builtin_memcpy(&lo, &L.kl[j][32 * w + 2 * r], 4);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float v = (float)hi[k] + (float)lo[k];
                    y[k][t][n] = v;
                    wt = __builtin_fmaxf(wt, __builtin_fabsf(v * fw[t][n]));
                    dt = __builtin_fmaxf(dt, __builtin_fabsf(v * fd[t][n]));
                }
            }
        const Scale ws = scale_of(wave_max(wt)), ds = scale_of(wave_max(dt));
        if (lane == 0 && half == 0) fac[kFK + w] = ds.down;
        Frag kw[2][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float u[8];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
#pragma unroll
                for (int n = 0; n < 8; ++n) u[n] = y[k][t][n] * fw[t][n];
                kw[k][t] = split8(u, ws.up);
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) u[n] = (half ? y[1][t][n] : y[0][t][n]) * fd[t][n];
            store_frag(B.k + ((2 * w + half) * 2 + t) * 2048, split8(u, ds.up));
        }
#pragma unroll
        for (uint32_t n = 0; n < 2; ++n) {
            const uint32_t it = n ? 3 - half : half;  // (0 and 3, 1 and 2: three steps each)
            f32x4 v[2] = {zero, zero};
#pragma unroll
            for (uint32_t t = 0; t <= n; ++t) {
                const Frag g = t_frag(it, t);
                v[0] = mm3(kw[0][t], g, v[0]);
                v[1] = mm3(kw[1][t], g, v[1]);
            }
            const float down = ws.down * L.tinv[it];
            v[0] *= down;
            v[1] *= down;
            const float most = wave_max(top4(top4(0.0f, v[0]), v[1]));
            const Scale s = scale_of(most);
            if (lane == 0) {
                fac[kFW + 4 * it + w] = s.down;
                fac[kFWMax + 4 * it + w] = most;
            }
            float u[8];
            __builtin_memcpy(u, v, 32);
            store_frag(B.w + (it * NT + w) * 2048, split8(u, s.up));
        }
    }
    // U0
    for (uint32_t cb = cb_first; has_v && cb < dv / 16; cb += 8) {
        if (cb != cb_first) load_v(cb);
        float y[2][8], most = 0.0f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const uint32_t j = 32 * t + 16 * (n / 4) + 4 * h + (n & 3);
                float v = vx[2 * t + n / 4][n & 3];
                __asm__("" : "+v"(v));  // (the load itself stays outside the choice)
                y[t][n] = j < c.live ? v * L.beta[j] : 0.0f;
                most = __builtin_fmaxf(most, __builtin_fabsf(y[t][n]));
            }
        const Scale s = scale_of(wave_max(most));
        const Frag vf[2] = {split8(y[0], s.up), split8(y[1], s.up)};
        most = 0.0f;
#pragma unroll
        for (uint32_t it = 0; it < 4; ++it) {
            f32x4 u = zero;
#pragma unroll
            for (uint32_t t = 0; t <= it / 2; ++t) u = mm3(t_frag(it, t), vf[t], u);
            u *= s.down * L.tinv[it];
            most = top4(most, u);
            __builtin_memcpy(block + B.u + (cb * 4 + it) * 1024 + lane * 16, &u, 16);
        }
        most = wave_max(most);
        if (lane == 0) fac[kFU + cb] = most;
    }
}
template <int DK> __global__ void __launch_bounds__(512, 4) delta_prepare_kernel(DeltaArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_bytes[];
    const uint32_t at = blockIdx.x / a.n_heads, hd = blockIdx.x - at * a.n_heads;
    const Chunk c = chunk_of(a, at);
    if (c.live) prepare<DK>(a, c, hd, a.blocks + ((size_t)at * a.n_heads + hd) * delta_block(DK, a.v_dim).bytes, *reinterpret_cast<PrepareLds<DK> *>(lds_bytes));
}

// The nth sequence that goes by chunks, from the lanes that look for it; n_seq if there is none.  (Workgroups for every sequence
// of a batch of mostly single tokens ended at once, but took as long to start as the others: one of 512 tokens among 256 158 us
// for 146, among 16 67 for 46.)
AH_DEV uint32_t nth_long(const DeltaArgs &a, uint32_t nth, Seq &found) {
    for (uint32_t base = 0; base < a.s.n_seq; base += 64) {
        const uint32_t i = base + (threadIdx.x & 63);
        const Seq p = seq_of(a.s, i < a.s.n_seq ? i : a.s.n_seq - 1);
        const uint64_t all = __builtin_amdgcn_ballot_w64(i < a.s.n_seq && !p.bad && p.nq >= a.chunk_from);
        const uint32_t n = (uint32_t)__builtin_popcountll(all);
        if (nth < n) {
            const bool me = (all >> (threadIdx.x & 63) & 1) && __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0)) == nth;
            const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(me));
            found = {(uint32_t)__builtin_amdgcn_readlane((int)p.q0, at), (uint32_t)__builtin_amdgcn_readlane((int)p.nq, at), __builtin_amdgcn_readlane(p.from, at),
                     __builtin_amdgcn_readlane(p.to, at), false};
            return base + (uint32_t)at;
        }
        nth -= n;
    }
    return a.s.n_seq;
}
// A sequence's chunks in turn, for NC times 16 columns of a head's S.  Waves 0 to 3 are the chain: wave w makes U of the tokens
// 16 w .. 16 w + 15 (the first half of a chunk's time) and the rows of slice w of S (the second); what the others need goes
// through LDS as operands.  Waves 4 to 7 make o of the same tokens: q S beside U, P U beside S.  Two barriers a chunk.
//   What comes from memory is asked for two chunks ahead, and touched a few chunks before that, each of a head's workgroups a
// part, so that it waits in the XCD's L2.
//   What bounds it is that chain of two products, their scales and halves, and two barriers: 1.9 us a chunk of 128 x 128 where the
// blocks lie in the last cache (8192 tokens of 16 heads: 128 workgroups of 256 CUs, 238 us), whatever the columns; more columns
// a workgroup take longer a chunk and read a block fewer times.  In 5 x 301 tokens (NC 2, 29 us) products take 16% of a SIMD's
// cycles while a CU works, vector work 27%, and the waves wait 37% of theirs.
template <int DK, int NC> struct ChainLds {
    u32x4 sf[NC][DK / 32][2][64], uf[NC][2][2][64];
    float sinv[NC][4], stop[NC][4], uinv[NC];
};
template <int DK, int NC> AH_DEV void chain(const DeltaArgs &a, ChainLds<DK, NC> &L) {
    constexpr int NT = DK / 32;
    constexpr uint32_t kTouch = 4;  // chunks
    auto &sf = L.sf;
    auto &uf = L.uf;
    auto &sinv = L.sinv;
    auto &stop = L.stop;
    auto &uinv = L.uinv;
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, h = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
    // columns slowest: a head's workgroups go to one XCD (they go to the eight in turn) wherever eight divides the heads
    const uint32_t units = a.longs * a.n_heads, part = blockIdx.x / units, unit = blockIdx.x - part * units, nth = unit / a.n_heads, hd = unit - nth * a.n_heads;
    Seq p;
    uint32_t s = nth;
    if (a.chunk_from) s = nth_long(a, nth, p);
    else p = seq_of(a.s, s);
    if (s >= a.s.n_seq) return;
    if (p.bad && part == 0 && hd == 0 && threadIdx.x == 0) ah_record(a.status, ((unsigned long long)s << 8) + kKeyRange);
    if (p.bad) return;
    // this launch's chunks: begin .. chunks - 1 of `whole`
    const uint32_t whole = (p.nq + kDeltaChunk - 1) / kDeltaChunk, begin = a.ring ? a.begin : 0, end = a.ring ? a.begin + a.ring / 2 : whole;
    const uint32_t chunks = whole < end ? whole : end, dv = a.v_dim, cb = part * NC;
    if (begin && begin >= whole) return;
    const DeltaBlock B = delta_block(DK, dv);
    const size_t step = (size_t)a.n_heads * B.bytes, first = (a.ring ? s * a.ring : (p.q0 >> a.slot_shift) + s * a.slot_seq) * step + (size_t)hd * B.bytes;
    auto block_of = [&](uint32_t n) {
        const uint32_t m = n < chunks ? n : chunks - 1;
        return a.blocks + first + (a.ring ? m % a.ring : m) * step;
    };
    auto frag = [&](const uint8_t *b) {
        Frag f;
        __builtin_memcpy(&f.hi, b + lane * 16, 16);
        __builtin_memcpy(&f.lo, b + 1024 + lane * 16, 16);
        return f;
    };
    // S between a sequence's launches
    float *carry = a.carry + (size_t)unit * DK * dv;
    const float *old = begin ? carry : p.from >= 0 ? a.state + ((size_t)p.from * a.n_heads + hd) * DK * dv : nullptr;
    float *now = chunks < whole ? carry : p.to >= 0 ? a.state + ((size_t)p.to * a.n_heads + hd) * DK * dv : nullptr;
    bool odd = false;
    if (wave < 4) {
        const bool own = w < (uint32_t)NT;
        const size_t tile = (size_t)(32 * w + 8 * h) * dv + 16 * cb + r;
        f32x4 S[NC][2];
#pragma unroll
        for (int c = 0; c < NC; ++c) S[c][0] = S[c][1] = (f32x4)0.0f;
        if (own && old) {
            const float *from = old + tile;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) S[c][k][i] = from[(size_t)(2 * i + k) * dv + 16 * c];
        }
        // of a chunk: W, U0 and the factors (a lane each) for the first half of its time, the keys for the second
        struct Ahead {
            Frag W[NT], K[2][2];
            f32x4 u0[NC];
            float f, wmax;
        } ahead[2];
        auto load_first = [&](uint32_t n, Ahead &x) {
            const uint8_t *b = block_of(n);
#pragma unroll
            for (int t = 0; t < NT; ++t) x.W[t] = frag(b + B.w + (w * NT + t) * 2048);
#pragma unroll
            for (int c = 0; c < NC; ++c) __builtin_memcpy(&x.u0[c], b + B.u + ((cb + c) * 4 + w) * 1024 + lane * 16, 16);
        };
        auto load_second = [&](uint32_t n, Ahead &x) {
            const uint8_t *b = block_of(n);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int t = 0; t < 2; ++t) x.K[k][t] = frag(b + B.k + ((2 * (own ? w : 0) + k) * 2 + t) * 2048);
            x.f = reinterpret_cast<const float *>(b + B.f)[64 + lane];
        };
        auto publish = [&] {  // this wave's rows of S
            if (!own) return;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float top = wave_max(top4(top4(0.0f, S[c][0]), S[c][1]));
                const Scale z = scale_of(top);
                float x[8];
                __builtin_memcpy(x, S[c], 32);
                const Frag f = split8(x, z.up);
                sf[c][w][0][lane] = f.hi;
                sf[c][w][1][lane] = f.lo;
                if (lane == 0) {
                    sinv[c][w] = z.down;
                    stop[c][w] = top;
                }
            }
        };
        auto chunk = [&](uint32_t n, Ahead &x) {
            float udown[NC];
            // the largest of W of each slice: of the four tiles' factors, four lanes each
            x.wmax = __builtin_fmaxf(x.f, dpp<0x124>(x.f));
            x.wmax = __builtin_fmaxf(x.wmax, dpp<0x128>(x.wmax));
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                f32x4 u = x.u0[c];
                float top = lane_of(x.f, kFU - 64 + cb + c);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const Frag f = {sf[c][t][0][lane], sf[c][t][1][lane]};
                    const f32x4 v = mm3(x.W[t], f, (f32x4)0.0f);
                    u -= v * (lane_of(x.f, kFW - 64 + 4 * w + t) * sinv[c][t]);
                    top = __builtin_fmaf(32.0f * lane_of(x.wmax, t), stop[c][t], top);
                }
                // one scale for all of U: |U| is at most |U0| and 32 times the largest of W and S of each slice
                const Scale z = scale_of(top);
                uint32_t hi[2], lo[2];
                split2(u[0] * z.up, u[1] * z.up, hi[0], lo[0]);
                split2(u[2] * z.up, u[3] * z.up, hi[1], lo[1]);
                __builtin_memcpy(reinterpret_cast<char *>(&uf[c][w >> 1][0][lane]) + 8 * (w & 1), hi, 8);
                __builtin_memcpy(reinterpret_cast<char *>(&uf[c][w >> 1][1][lane]) + 8 * (w & 1), lo, 8);
                if (threadIdx.x == 0) uinv[c] = z.down;
                udown[c] = z.down;
#pragma unroll
                for (int i = 0; i < 4; ++i) odd = odd || !finite(u[i]);
            }
            load_first(n + 2, x);
            ah_lds_barrier();
            if (own) {
                const float decay = lane_of(x.f, kFDecay - 64), kdown = lane_of(x.f, kFK - 64 + w);
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const Frag f[2] = {{uf[c][0][0][lane], uf[c][0][1][lane]}, {uf[c][1][0][lane], uf[c][1][1][lane]}};
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const f32x4 v = mm3(x.K[k][1], f[1], mm3(x.K[k][0], f[0], (f32x4)0.0f));
                        S[c][k] = S[c][k] * decay + v * (kdown * udown[c]);
                    }
                }
            }
            load_second(n + 2, x);
            publish();
            ah_lds_barrier();
        };
        if (chunks > begin) {
#pragma unroll
            for (uint32_t n = 0; n < 2; ++n) {
                load_first(begin + n, ahead[n]);
                __builtin_amdgcn_sched_barrier(0);
                load_second(begin + n, ahead[n]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        publish();
        ah_lds_barrier();
        for (uint32_t n = begin; n + 1 < chunks; n += 2) {
            chunk(n, ahead[0]);
            chunk(n + 1, ahead[1]);
        }
        if ((chunks - begin) & 1) chunk(chunks - 1, ahead[0]);
        if (own && now) {
            float *to = now + tile;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        to[(size_t)(2 * i + k) * dv + 16 * c] = S[c][k][i];
                        odd = odd || (p.nq && !finite(S[c][k][i]));  // (the last chunk's U may be finite and what it adds not)
                    }
        }
    } else {
        struct Ahead {
            Frag Q[NT], P[2];
            f32x4 qf, pf;
            uint32_t touched;
        } ahead[2];
        auto load_first = [&](uint32_t n, Ahead &x) {
            const uint8_t *b = block_of(n);
#pragma unroll
            for (int t = 0; t < NT; ++t) x.Q[t] = frag(b + B.q + (w * NT + t) * 2048);
        };
        auto load_second = [&](uint32_t n, Ahead &x) {
            const uint8_t *b = block_of(n);
            __builtin_memcpy(&x.qf, reinterpret_cast<const float *>(b + B.f) + kFRow + 16 * w + 4 * h, 16);
            __builtin_memcpy(&x.pf, reinterpret_cast<const float *>(b + B.f) + kFP + 16 * w + 4 * h, 16);
#pragma unroll
            for (uint32_t t = 0; t < 2; ++t) x.P[t] = frag(b + B.p + tri(w, w < 2 ? 0 : t) * 2048);
        };
        // A line of 128 bytes for each lane, of what all of a head's workgroups read: each takes a part, each wave of it a fourth.
        const uint32_t parts = dv / (16 * NC), lines = B.u / 128, each = (lines + 4 * parts - 1) / (4 * parts);
        auto touch = [&](uint32_t n) {
            uint32_t v;
            const uint32_t at = (4 * part + w) * each + (lane < each ? lane : 0);
            __builtin_memcpy(&v, block_of(n) + 128 * (at < lines ? at : lines - 1), 4);
            return v;
        };
        auto chunk = [&](uint32_t n, Ahead &x) {
            f32x4 o[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) o[c] = (f32x4)0.0f;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const Frag f = {sf[c][t][0][lane], sf[c][t][1][lane]};
                    o[c] += mm3(x.Q[t], f, (f32x4)0.0f) * sinv[c][t];
                }
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) o[c] *= x.qf;
            load_first(n + 2, x);
            ah_lds_barrier();
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                f32x4 v = mm3(x.P[0], {uf[c][0][0][lane], uf[c][0][1][lane]}, (f32x4)0.0f);
                if (w >= 2) v = mm3(x.P[1], {uf[c][1][0][lane], uf[c][1][1][lane]}, v);
                o[c] += v * (x.pf * uinv[c]);
            }
            load_second(n + 2, x);
            // (range-checked stores: a branch around them would have every later wait for loads wait for them too)
            const uint32_t live = p.nq - kDeltaChunk * n < kDeltaChunk ? p.nq - kDeltaChunk * n : kDeltaChunk, stride = (uint32_t)a.out_stride;
            const __amdgpu_buffer_rsrc_t to = ah_rsrc(a.out + (size_t)(p.q0 + kDeltaChunk * n) * a.out_stride + (size_t)hd * dv + 16 * cb, 4 * ((live - 1) * stride + 16 * NC));
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const uint32_t t = 16 * w + 4 * h + i;
                    const float y = o[c][i];
                    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, y), to, (int)(4 * (t * stride + 16 * c + r)), 0, 0);
                    odd = odd || (t < live && !finite(y));
                }
            __asm__ volatile("" ::"v"(x.touched));
            x.touched = touch(n + kTouch);
            ah_lds_barrier();
        };
        if (chunks > begin) {
#pragma unroll
            for (uint32_t n = 0; n < 2; ++n) {
                load_first(begin + n, ahead[n]);
                __builtin_amdgcn_sched_barrier(0);
                load_second(begin + n, ahead[n]);
                ahead[n].touched = touch(begin + n + 2);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        ah_lds_barrier();
        for (uint32_t n = begin; n + 1 < chunks; n += 2) {
            chunk(n, ahead[0]);
            chunk(n + 1, ahead[1]);
        }
        if ((chunks - begin) & 1) chunk(chunks - 1, ahead[0]);
    }
    if (odd) ah_record(a.status, ((unsigned long long)s << 8) + kKeyNonFinite);
}
template <int DK, int NC> __global__ void __launch_bounds__(512) delta_chain_kernel(DeltaArgs a) {
    __shared__ ChainLds<DK, NC> L;
    if (blockIdx.x < a.chain_grid) chain<DK, NC>(a, L);
    else steps<DK>(a, 8 * (blockIdx.x - a.chain_grid) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
}
// The chain of one group of chunks beside the preparation of the next, where the chain leaves CUs to it: every sequence's chunks
// begin .. begin + ring / 2 - 1 and, by the workgroups after the chain's, the ring / 2 after those.  The blocks of two groups
// are there at once, [sequence][ring][head].  A launch of 16 chunks of 16 heads takes 40 us: 30 of chain, and 256 preparations
// in the 128 CUs that it leaves, one a CU (the chain's registers leave a CU no room for two).
template <int DK> __global__ void __launch_bounds__(512) delta_both_kernel(DeltaArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_bytes[];
    __shared__ ChainLds<DK, 1> L;
    if (blockIdx.x < a.chain_grid) {
        chain<DK, 1>(a, L);
        return;
    }
    const uint32_t half = a.ring / 2, at = blockIdx.x - a.chain_grid, hd = at % a.n_heads, i = at / a.n_heads, s = i / half, n = a.prepared + i % half;
    const Seq p = seq_of(a.s, s);
    if (p.bad || kDeltaChunk * n >= p.nq) return;
    const uint32_t rest = p.nq - kDeltaChunk * n;
    const Chunk c = {s, p.q0 + kDeltaChunk * n, rest < kDeltaChunk ? rest : kDeltaChunk};
    prepare<DK>(a, c, hd, a.blocks + (((size_t)s * a.ring + n % a.ring) * a.n_heads + hd) * delta_block(DK, a.v_dim).bytes,
                *reinterpret_cast<PrepareLds<DK> *>(lds_bytes));
}

// The chain, and in the workgroups after it, where the lengths differ, the sequences that go token by token.
template <int DK, int NC> void launch_chain(DeltaArgs a, bool mixed, hipStream_t stream) {
    a.chain_grid = a.longs * a.n_heads * (a.v_dim / (16 * NC));
    hipLaunchKernelGGL((delta_chain_kernel<DK, NC>), dim3(a.chain_grid + (mixed ? (a.s.n_seq * a.n_heads * (a.v_dim / 32) + 7) / 8 : 0)), dim3(512), 0, stream, a);
}
// Groups of chunks: each launch has the chain of one and the preparation of the next.
template <int DK> void launch_groups(DeltaArgs a, hipStream_t stream) {
    const uint32_t half = a.ring / 2, all = (a.s.max_q + kDeltaChunk - 1) / kDeltaChunk, groups = (all + half - 1) / half;
    const uint32_t chain_grid = a.s.n_seq * a.n_heads * (a.v_dim / 16), prepare_grid = a.s.n_seq * half * a.n_heads;
    for (uint32_t g = 0; g <= groups; ++g) {
        a.begin = g ? (g - 1) * half : 0;
        a.chain_grid = g ? chain_grid : 0;
        a.prepared = g * half;
        hipLaunchKernelGGL(delta_both_kernel<DK>, dim3(a.chain_grid + (g < groups ? prepare_grid : 0)), dim3(512), sizeof(PrepareLds<DK>), stream, a);
    }
}
template <int DK> void launch_chunks(const DeltaArgs &a, bool mixed, hipStream_t stream) {
    if (a.ring) {
        launch_groups<DK>(a, stream);
        return;
    }
    hipLaunchKernelGGL(delta_prepare_kernel<DK>, dim3(a.slots * a.n_heads), dim3(512), sizeof(PrepareLds<DK>), stream, a);
    if (a.tiles == 1) launch_chain<DK, 1>(a, mixed, stream);
    else if (a.tiles == 2) launch_chain<DK, 2>(a, mixed, stream);
    else launch_chain<DK, 4>(a, mixed, stream);
}

template <int W> hipError_t launch_conv(const ConvArgs &a, hipStream_t stream) {
    hipLaunchKernelGGL(conv_kernel<W>, dim3(a.tiles * ((a.n_ch + 1023) / 1024)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

} // namespace

hipError_t ah_launch_conv(const ConvArgs &a, hipStream_t stream) {
    switch (a.width) {
    case 2: return launch_conv<2>(a, stream);
    case 3: return launch_conv<3>(a, stream);
    case 4: return launch_conv<4>(a, stream);
    case 5: return launch_conv<5>(a, stream);
    case 6: return launch_conv<6>(a, stream);
    case 7: return launch_conv<7>(a, stream);
    default: return launch_conv<8>(a, stream);
    }
}

hipError_t ah_launch_delta(const DeltaArgs &a, bool steps, bool chunks, hipStream_t stream) {
    if (chunks) {
        if (a.k_dim == 64) launch_chunks<64>(a, steps, stream);
        else launch_chunks<128>(a, steps, stream);
        return hipGetLastError();
    }
    const uint32_t units = a.s.n_seq * a.n_heads * (a.v_dim / 32);
    if (a.k_dim == 64) hipLaunchKernelGGL(delta_step_kernel<64>, dim3((units + 3) / 4), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(delta_step_kernel<128>, dim3((units + 3) / 4), dim3(256), 0, stream, a);
    return hipGetLastError();
}

hipError_t ah_state_init_attrs() {
    hipError_t e = hipSuccess;
    for (const void *k : {(const void *)delta_prepare_kernel<64>, (const void *)delta_both_kernel<64>})
        if (e == hipSuccess) e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(PrepareLds<64>));
    for (const void *k : {(const void *)delta_prepare_kernel<128>, (const void *)delta_both_kernel<128>})
        if (e == hipSuccess) e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(PrepareLds<128>));
    return e;
}
