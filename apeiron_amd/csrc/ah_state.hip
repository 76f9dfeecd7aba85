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

AH_DEV bool finite(float v) { return __builtin_fabsf(v) < __builtin_inff(); }

// ---- the short causal convolution --------------------------------------------------------------------
//
// y_t = act(bias + sum_i w_i x_(t - W + 1 + i)), a lane four channels of a tile of consecutive tokens: it keeps the
// W - 1 rows before the next one in registers, so a row is read once a tile and the rows before a tile once more.  The
// tile that holds a sequence's first token alone reads the state and also writes the new one, so that both may lie in
// the same slot.
AH_DEV void load4(float *v, const float *p, uint32_t take) {
    if (take == 4) {
        __builtin_memcpy(v, p, 16);
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) v[i] = i < take ? p[i] : 0.0f;
}
AH_DEV void store4(float *p, const float *v, uint32_t take) {
    if (take == 4) {
        __builtin_memcpy(p, v, 16);
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
        if (i < take) p[i] = v[i];
}

template <int W> __global__ void __launch_bounds__(256) conv_kernel(ConvArgs a) {
    const uint32_t at = blockIdx.x % a.tiles, block = blockIdx.x / a.tiles, c0 = 4 * (block * 256 + threadIdx.x);
    auto start = [&](uint32_t i) { return (uint32_t)a.s.q_start[i] / a.tile + i; };
    auto holds = [&](uint32_t i) {
        const Seq p = seq_of(a.s, i);
        return !p.bad && at >= start(i) && at - start(i) < (p.nq ? (p.nq + a.tile - 1) / a.tile : 1);
    };
    const uint32_t s = a.per ? at / a.per : sequence_among(a.s.q_start, a.s.n_seq, a.s.n_tok, at, start, holds), n = at - (a.per ? s * a.per : start(s));
    if (block == 0 && threadIdx.x == 0)
        for (uint32_t i = at; i < a.s.n_seq; i += a.tiles)
            if (seq_of(a.s, i).bad) ah_record(a.status, ((unsigned long long)i << 8) + kKeyRange);
    const Seq p = seq_of(a.s, s);
    const uint32_t t0 = n * a.tile, take = c0 >= a.n_ch ? 0 : a.n_ch - c0 < 4 ? a.n_ch - c0 : 4;
    if (p.bad || take == 0 || (n && t0 >= p.nq)) return;
    const uint32_t t1 = t0 + a.tile < p.nq ? t0 + a.tile : p.nq;
    const float *x = a.x + (size_t)p.q0 * a.x_stride + c0;
    float w[4][W], bias[4] = {0.0f, 0.0f, 0.0f, 0.0f}, row[W][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) w[i][j] = i < (int)take ? a.weight[(size_t)(c0 + i) * W + j] : 0.0f;
    if (a.bias) load4(bias, a.bias + c0, take);
    // rows before the tile: of the sequence, or of the state (row W - 1 - j of it stands j places before the first token)
    const float *old = a.state + (size_t)(p.from < 0 ? 0 : p.from) * (W - 1) * a.n_ch + c0;
    auto before = [&](float *v, int64_t t) {  // row t of the sequence, t >= 1 - W
        if (t >= 0) load4(v, x + (size_t)t * a.x_stride, take);
        else if (p.from >= 0) load4(v, old + (size_t)(W - 1 + t) * a.n_ch, take);
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = 0.0f;
    };
#pragma unroll
    for (int j = 0; j < W - 1; ++j) before(row[j], (int64_t)t0 - (W - 1) + j);
    float kept[W - 1][4];
    const bool keep = n == 0 && p.to >= 0;
    if (keep) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) before(kept[j], (int64_t)p.nq - (W - 1) + j);
    }
    float *y = a.y + (size_t)p.q0 * a.y_stride + c0;
    bool odd = false;
    for (uint32_t t = t0; t < t1; ++t) {
        load4(row[W - 1], x + (size_t)t * a.x_stride, take);
        float out[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v = bias[i];
#pragma unroll
            for (int j = 0; j < W; ++j) v = __builtin_fmaf(w[i][j], row[j][i], v);
            odd = odd || !finite(v);
            out[i] = a.silu ? v / (1.0f + expf(-v)) : v;
        }
        store4(y + (size_t)t * a.y_stride, out, take);
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) row[j][i] = row[j + 1][i];
    }
    if (keep) {
        float *to = a.state + (size_t)p.to * (W - 1) * a.n_ch + c0;
#pragma unroll
        for (int j = 0; j < W - 1; ++j) store4(to + (size_t)j * a.n_ch, kept[j], take);
    }
    if (odd) ah_record(a.status, ((unsigned long long)s << 8) + kKeyNonFinite);
}

// ---- the gated delta rule ----------------------------------------------------------------------------
//
// Token by token, with a head's S [k_dim][v_dim] in registers: S = e^g S, u = beta (v - S^T k), S += k u^T,
// o = scale S^T q.  A wave takes 32 columns of S: lane (r, c) = (lane >> 3, lane & 7) rows R r .. R r + R - 1 of columns
// 4 c .. 4 c + 3.
AH_DEV float sum_rows(float v) {  // over the eight lanes of a column
    v += __shfl_xor(v, 8, 64);
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
// log(1 + e^x)
AH_DEV float softplus(float x) { return __builtin_fmaxf(x, 0.0f) + log1pf(expf(-__builtin_fabsf(x))); }
AH_DEV float decay_of(const DeltaArgs &a, float x, uint32_t h) { return a.a_log ? -expf(a.a_log[h]) * softplus(x + a.dt_bias[h]) : x; }
AH_DEV float rate_of(const DeltaArgs &a, float x) { return a.a_log ? 1.0f / (1.0f + expf(-x)) : x; }

template <int DK> __global__ void __launch_bounds__(256) delta_step_kernel(DeltaArgs a) {
    constexpr int R = DK / 8;
    const uint32_t lane = threadIdx.x & 63, r = lane >> 3, c = lane & 7;
    const uint32_t unit = 4 * blockIdx.x + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nvb = a.v_dim / 32;
    const uint32_t vb = unit % nvb, h = unit / nvb % a.n_heads, s = unit / nvb / a.n_heads;
    if (s >= a.s.n_seq) return;
    const Seq p = seq_of(a.s, s);
    if (p.bad && vb == 0 && h == 0 && lane == 0) ah_record(a.status, ((unsigned long long)s << 8) + kKeyRange);
    if (p.bad) return;
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
            fk = 1.0f / __builtin_sqrtf(sum_rows(kk) + a.norm_eps);
            fq *= 1.0f / __builtin_sqrtf(sum_rows(qq) + a.norm_eps);
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

hipError_t ah_launch_delta(const DeltaArgs &a, hipStream_t stream) {
    const uint32_t units = a.s.n_seq * a.n_heads * (a.v_dim / 32);
    if (a.k_dim == 64) hipLaunchKernelGGL(delta_step_kernel<64>, dim3((units + 3) / 4), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(delta_step_kernel<128>, dim3((units + 3) / 4), dim3(256), 0, stream, a);
    return hipGetLastError();
}
