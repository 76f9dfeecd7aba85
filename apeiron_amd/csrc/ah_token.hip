// ah_token.hip -- the operators between a token's projections that touch each value once: the
// residual's addition with the RMS norm and the activation quantizer, rotary positions, and the
// append to the paged 4-bit cache (layout: ah_kv4.h) with its read-back.
#include "ah_kv4.h"
#include "ah_units.h"

namespace {

constexpr unsigned long long kKeyNonFinite = AH_ERR_NONFINITE_INPUT, kKeyCache = AH_ERR_CACHE_RANGE;

AH_DEV double wave_sum(double v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// ---- residual + RMS norm + quant_act ---------------------------------------------------------------
//
// s = x + r, R = 1 / sqrt(mean(s^2) + eps), y = (s R) gain, and quant_act of y's 32-blocks.  One
// workgroup per token: a lane keeps 8 consecutive values of each of its U passes in registers, so the
// row is read once and the quantizer's quads (four lanes a block, ah_units.h) hold whole blocks.  The
// sum of squares is kept in f64, which the f32 row's magnitude cannot overflow, and R as two f32: y is
// rounded to f32 once, to the nearest (but for values within about 2^-44 of themselves of the middle of two), and
// once more to seven bits by the quantizer, as the projections take it.  Codes that differ from the exact y's,
// which f32 rounds to a half: 58 of 42 million, with R and both products rounded 68.
//   What bounds it: memory (2039 tokens of 8957 with every output, 279 MB in 62.6 us: 4.45 TB/s, of 4.74
// that a copy reaches); under a few hundred tokens the launch (512 of 1536 4.9 us, one of 896 2.6).  Rows
// come through range-checked resources: with a branch for a row's last values the arrays of a lane left
// the registers (171 us), and several passes of eight values a lane cost less than a second read of the row.
// Eight consecutive values at any element boundary, `take` of them (constant indices only: the arrays stay
// in registers).
template <class T> AH_DEV void load8(T *v, const T *p, uint32_t take) {
    if (take == 8) {
        __builtin_memcpy(v, p, 8 * sizeof(T));
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) v[i] = i < take ? p[i] : (T)0;
}
template <class T> AH_DEV void store8(T *p, const T *v, uint32_t take) {
    if (take == 8) {
        __builtin_memcpy(p, v, 8 * sizeof(T));
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
        if (i < take) p[i] = v[i];
}

// The same of a row read through a range-checked resource: what lies past its end reads as zero, and no
// branch stands between the loads of a lane's passes.
AH_DEV void ld8(float *v, __amdgpu_buffer_rsrc_t r, uint32_t k0) {
    const u32x4 a = ah_ld128(r, 4 * k0), b = ah_ld128(r, 4 * k0 + 16);
    __builtin_memcpy(v, &a, 16);
    __builtin_memcpy(v + 4, &b, 16);
}
AH_DEV void st8(__amdgpu_buffer_rsrc_t r, uint32_t k0, const float *v) {
    u32x4 a, b;
    __builtin_memcpy(&a, v, 16);
    __builtin_memcpy(&b, v + 4, 16);
    __builtin_amdgcn_raw_buffer_store_b128(a, r, (int)(4 * k0), 0, 0);
    __builtin_amdgcn_raw_buffer_store_b128(b, r, (int)(4 * k0 + 16), 0, 0);
}

// (s (rh + rl)) g: the product by R with its own rounding's rest, then one rounding of both times g.
AH_DEV float rounded_once(float s, float rh, float rl, float g) {
#pragma clang fp contract(off)
    const float t = s * rh, rest = __builtin_fmaf(s, rl, __builtin_fmaf(s, rh, -t));
    return __builtin_fmaf(t, g, rest * g);
}

template <uint32_t U, bool RES>
__global__ void __launch_bounds__(1024) norm_quant_kernel(NormArgs a) {
    __shared__ double red[16];
    const uint32_t tid = threadIdx.x, T = blockDim.x, n = a.n, tok = blockIdx.x;
    const size_t row = (size_t)tok * n;
    float s[U][8], r[U][8], g[U][8];
    const __amdgpu_buffer_rsrc_t xr = ah_rsrc(a.x + row, 4 * n), rr = ah_rsrc(RES ? a.r + row : a.x, 4 * n), gr = ah_rsrc(a.gain, 4 * n);
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        const uint32_t k0 = 8 * (u * T + tid);
        ld8(s[u], xr, k0);
        if (RES) ld8(r[u], rr, k0);
        ld8(g[u], gr, k0);
    }
    double ss = 0.0;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            if (RES) s[u][i] += r[u][i];
            ss = __builtin_fma((double)s[u][i], (double)s[u][i], ss);
        }
    ss = wave_sum(ss);
    if (T > 64) {
        if ((tid & 63) == 0) red[tid >> 6] = ss;
        __syncthreads();
        ss = 0.0;
        for (uint32_t w = 0; w < T / 64; ++w) ss += red[w];
    }
    // v_rsq_f64 is good to about 2^-28; a Newton step squares that
    const double mean = ss / (double)n + a.eps, r0 = __builtin_amdgcn_rsq(mean);
    const double R = r0 * __builtin_fma(-0.5 * mean, r0 * r0, 1.5);
    const float rh = (float)R, rl = (float)(R - (double)rh);
    const uint32_t nb = (n + 31) / 32;
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        const uint32_t k0 = 8 * (u * T + tid), take = n > k0 ? (n - k0 < 8 ? n - k0 : 8) : 0;
        float y[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) y[i] = rounded_once(s[u][i], rh, rl, g[u][i]);
        if (a.sum) st8(ah_rsrc(a.sum + row, 4 * n), k0, s[u]);
        if (a.y) st8(ah_rsrc(a.y + row, 4 * n), k0, y);
        if (!a.codes && !a.values) continue;
        QuadIn in;
#pragma unroll
        for (int i = 0; i < 8; ++i) in.w[i] = __builtin_bit_cast(uint32_t, y[i]);
#pragma unroll
        for (int i = 8; i < 16; ++i) in.w[i] = 0;
        in.s0 = in.s1 = 0;
        in.take = take;
        const uint32_t b = k0 / 32;
        const QuadOut o = quad_quant(in, AH_SRC_F32, b, a.status, (unsigned long long)row);
        if (a.codes) {
            int8_t c[8];
            const u32x2 w = {o.c0, o.c1};
            __builtin_memcpy(c, &w, 8);
            store8(a.codes + row + k0, c, take);
            if ((tid & 3) == 0 && b < nb) a.scales[(size_t)tok * nb + b] = o.e < 0 ? 0 : (int64_t)(1ull << o.e);
        }
        if (a.values) {  // code * 2^(e - 32): seven bits, exact in bf16
            uint16_t v[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
                v[i] = (uint16_t)(__builtin_bit_cast(uint32_t, (float)(int8_t)(((i < 4 ? o.c0 : o.c1) >> (8 * (i & 3))) & 0xffu) * o.fsc) >> 16);
            store8(a.values + row + k0, v, take);
        }
    }
}

// ---- rotary positions ------------------------------------------------------------------------------
//
// The angle pos * theta and its cosine and sine are formed in f64 (a position of 10^5 leaves an f32
// angle no fraction) and rounded to f32 once; the rotation's products are rounded one by one, so that a
// rotated value does not depend on which of them the compiler would fuse.  A token's sines are formed once
// for all of its heads: a workgroup takes a token.  What bounds rope_kernel: memory (32768 tokens of 32 heads of 128,
// 1.07 GB in 242 us, 4.45 TB/s; 4093 of 14 heads 15.2 us against 12.4), the host's call for few (7.8 us).

AH_DEV void rope_table(const RopeRef &r, int32_t pos, float *cs, float *sn) {
    for (uint32_t i = threadIdx.x; i < r.rot / 2; i += blockDim.x) {
        double s, c;
        sincos((double)pos * r.theta[i], &s, &c);
        cs[i] = (float)(r.amplitude * c);
        sn[i] = (float)(r.amplitude * s);
    }
}

AH_DEV float turn(float a, float ca, float b, float sb) {
#pragma clang fp contract(off)
    const float p = a * ca, q = b * sb;
    return p + q;
}

// Elements e0 .. e0 + 7 of head row x (take of them) into v, rotated.
AH_DEV void load_rotated(const RopeRef &r, const float *x, uint32_t e0, uint32_t take, const float *cs, const float *sn, float *v) {
    load8(v, x + e0, take);
    if (!r.theta || e0 >= r.rot) return;
    if (r.interleaved) {
#pragma unroll
        for (uint32_t i = 0; i < 8; i += 2) {
            if (e0 + i >= r.rot) continue;
            const float c = cs[(e0 + i) / 2], s = sn[(e0 + i) / 2], a = v[i], b = v[i + 1];
            v[i] = turn(a, c, b, -s);
            v[i + 1] = turn(b, c, a, s);
        }
        return;
    }
    const uint32_t half = r.rot / 2;
    if ((half & 7) == 0) {  // the lane's elements lie on one side, and so do their partners
        float w[8];
        const bool first = e0 < half;
        const uint32_t j = first ? e0 : e0 - half;
        __builtin_memcpy(w, x + (first ? e0 + half : j), 32);
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) v[i] = turn(v[i], cs[j + i], w[i], first ? -sn[j + i] : sn[j + i]);
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t e = e0 + i;
        if (i >= take || e >= r.rot) continue;
        const bool first = e < half;
        const uint32_t j = first ? e : e - half;
        v[i] = turn(v[i], cs[j], x[first ? e + half : j], first ? -sn[j] : sn[j]);
    }
}

// One workgroup per token; a lane takes 8 elements of a head.  A head in place: every element of it is
// read before the first is written, which the barrier between the two orders.
__global__ void __launch_bounds__(256) rope_kernel(RopeArgs a) {
    __shared__ float cs[kRopeMaxDim / 2], sn[kRopeMaxDim / 2];
    const uint32_t tok = blockIdx.x, per = (a.rope.dim + 7) / 8, total = per * a.n_heads;
    rope_table(a.rope, a.pos[tok], cs, sn);
    __syncthreads();
    const float *x = a.x + tok * a.x_stride;
    float *y = a.y + tok * a.y_stride;
    const uint32_t hp = blockDim.x / per, step = hp * per;  // whole heads a pass (per <= 64)
    for (uint32_t p = 0; p < total; p += step) {
        const uint32_t it = p + threadIdx.x, head = it / per, e0 = 8 * (it % per);
        const bool live = threadIdx.x < step && it < total;
        const uint32_t take = live ? (a.rope.dim - e0 < 8 ? a.rope.dim - e0 : 8) : 0;
        float v[8];
        if (live) load_rotated(a.rope, x + (size_t)head * a.rope.dim, e0, take, cs, sn, v);
        __syncthreads();
        store8(y + (size_t)head * a.rope.dim + e0, v, take);
    }
}

// ---- append and read -------------------------------------------------------------------------------

// The tile and the place in it of a token's position.  -1: a padding token (seq < 0); 0: outside.
AH_DEV int kv4_place(const Kv4Ref &c, const KvTokens &t, uint32_t tok, uint32_t &page, uint32_t &in_page) {
    const int32_t s = t.seq[tok], p = t.pos[tok];
    if (s < 0) return -1;
    const uint32_t pi = (uint32_t)p >> c.page_shift;
    if ((uint32_t)s >= t.n_seq || p < 0 || pi >= t.table_stride) return 0;
    page = (uint32_t)t.table[(size_t)s * t.table_stride + pi];
    in_page = (uint32_t)p & ((1u << c.page_shift) - 1);
    return page < c.n_pages ? 1 : 0;
}

// The f16 number of 8 significant bits nearest to d (ties to even; subnormals by f16's step).
AH_DEV float eight_bits(float d) {
    int e = (int)((__builtin_bit_cast(uint32_t, d) >> 23) & 0xffu) - 127 - 7;
    e = e < -24 ? -24 : e;
    const float q = __builtin_rintf(__builtin_ldexpf(d, -e));
    return __builtin_fminf(__builtin_fmaxf(__builtin_ldexpf(q, e), -8160.0f), 8160.0f);
}

AH_DEV uint32_t quad_max(uint32_t v) {
    v = __builtin_elementwise_max(v, quad_xor1(v));
    return __builtin_elementwise_max(v, quad_xor2(v));
}
AH_DEV float quad_fmax(float v) {
    v = __builtin_fmaxf(v, __builtin_bit_cast(float, quad_xor1(__builtin_bit_cast(uint32_t, v))));
    return __builtin_fmaxf(v, __builtin_bit_cast(float, quad_xor2(__builtin_bit_cast(uint32_t, v))));
}

// A quad's 32-channel block: this lane's 8 codes (0..15), the scale, and whether the block holds a
// non-finite value (it is then all zeros).
AH_DEV bool block_codes(const float *v, uint32_t *c, float &d) {
    float hi = v[0], lo = v[0];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        hi = __builtin_fmaxf(hi, v[i]);
        lo = __builtin_fminf(lo, v[i]);
        top = __builtin_elementwise_max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
    }
    hi = quad_fmax(hi);
    lo = -quad_fmax(-lo);
    const bool bad = quad_max(top) >= 0x7f800000u;
    d = bad ? 0.0f : eight_bits((hi >= -lo ? hi : lo) * -0.125f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = d != 0.0f ? __builtin_rintf(v[i] / d) : 0.0f;
        c[i] = (uint32_t)((int)__builtin_fminf(__builtin_fmaxf(t, -8.0f), 7.0f) + 8);
    }
    return bad;
}

// One workgroup per token: cosines and sines once, then 8 channels a lane over q's heads, k's and v's; one
// launch for the three.  k and v are rounded to the cache's four bits here, once.  What bounds it: memory
// (4093 tokens, 12 heads of 128 and 2 KV heads, 60 MB in 15.1 us, 4.0 TB/s, the sines beside it), the launch
// for few (8 tokens 4.3 us).  Without q the stores: V's codes go out byte by byte, and of 8192 tokens of 2 KV heads
// of 128 10.7 MB are written for 2.4 (12 us; 524288 tokens 496 us, 1.9 times a copy's time, and of heads of
// 64, half a wave's lanes idle, 381 and 3 times).  A token's codes are bytes of its own in a tile that 32 tokens
// share, so tokens need no order.
__global__ void __launch_bounds__(256) kv4_append_kernel(AppendArgs a) {
    __shared__ float cs[128], sn[128];
    const uint32_t tok = blockIdx.x, dim = a.c.dim, per = dim / 8, kv = a.c.n_kv;
    const uint32_t total = per * (a.n_heads + 2 * kv);
    if (a.rope.theta) rope_table(a.rope, a.t.pos[tok], cs, sn);
    uint32_t page = 0, in_page = 0;
    const int placed = kv4_place(a.c, a.t, tok, page, in_page);
    if (placed == 0 && threadIdx.x == 0) ah_record(a.status, (((unsigned long long)tok * (2 * kv)) << 8) + kKeyCache);
    __syncthreads();
    // per divides the wave, so a head's lanes (and a block's quad) are in one wave and pass together
    for (uint32_t it = threadIdx.x; it < total; it += blockDim.x) {
        const uint32_t head = it / per, li = it % per;
        float v[8];
        if (head < a.n_heads) {
            const float *x = a.q + tok * a.q_stride + (size_t)head * dim;
            load_rotated(a.rope, x, 8 * li, 8, cs, sn, v);
            // the wave's loads of the head come before its stores: q may be rotated in place
            __builtin_amdgcn_wave_barrier();
            __builtin_memcpy(a.q_out + tok * a.qo_stride + (size_t)head * dim + 8 * li, v, 32);
            continue;
        }
        const bool is_v = head >= a.n_heads + kv;
        const uint32_t h = head - a.n_heads - (is_v ? kv : 0);
        if (is_v) __builtin_memcpy(v, a.v + tok * a.v_stride + (size_t)h * dim + 8 * li, 32);
        else load_rotated(a.rope, a.k + tok * a.k_stride + (size_t)h * dim, 8 * li, 8, cs, sn, v);
        uint32_t c[8];
        float d;
        const bool bad = block_codes(v, c, d);
        if (placed <= 0) continue;
        if (bad && (li & 3) == 0)
            ah_record(a.status, (((unsigned long long)tok * (2 * kv) + (head - a.n_heads)) << 8) + kKeyNonFinite);
        uint8_t *t = a.c.base + kv4_tile(a.c, page, h, in_page >> 5);
        const uint32_t tp = in_page & 31;
        const uint16_t ds = __builtin_bit_cast(uint16_t, (_Float16)d);
        if (!is_v) {
            uint32_t w = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) w |= c[i] << (4 * ((i >> 1) + 4 * (i & 1)));
            __builtin_memcpy(t + kv4_k_code(dim, tp, li), &w, 4);
            if ((li & 3) == 0) __builtin_memcpy(t + kv4_k_scale(dim, tp, li / 4), &ds, 2);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) t[kv4_v_code(dim, tp, 4 * li + i)] = (uint8_t)(c[2 * i] | c[2 * i + 1] << 4);
            if ((li & 3) == 0) __builtin_memcpy(t + kv4_v_scale(dim, tp, li / 4), &ds, 2);
        }
    }
}

// The values of tokens, for whoever wants them outside the attention: 4093 tokens 5.0 us, 524288 of 2 heads of 128 349 us,
// 2.4 times a copy's time (V's codes are read byte by byte); generation does not call it.
__global__ void __launch_bounds__(256) kv4_read_kernel(KvReadArgs a) {
    const uint32_t tok = blockIdx.x, dim = a.c.dim, per = dim / 8, kv = a.c.n_kv;
    uint32_t page = 0, in_page = 0;
    const int placed = kv4_place(a.c, a.t, tok, page, in_page);
    if (placed == 0 && threadIdx.x == 0) ah_record(a.status, ((unsigned long long)tok << 8) + kKeyCache);
    for (uint32_t it = threadIdx.x; it < 2 * kv * per; it += blockDim.x) {
        const uint32_t head = it / per, li = it % per;
        const bool is_v = head >= kv;
        const uint32_t h = is_v ? head - kv : head;
        uint16_t *out = is_v ? a.v : a.k;
        if (!out) continue;
        _Float16 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (_Float16)0.0f;
        if (placed > 0) {
            const uint8_t *t = a.c.base + kv4_tile(a.c, page, h, in_page >> 5);
            const uint32_t tp = in_page & 31;
            uint16_t ds;
            __builtin_memcpy(&ds, t + (is_v ? kv4_v_scale(dim, tp, li / 4) : kv4_k_scale(dim, tp, li / 4)), 2);
            const _Float16 d = __builtin_bit_cast(_Float16, ds);
            if (!is_v) {
                uint32_t w;
                __builtin_memcpy(&w, t + kv4_k_code(dim, tp, li), 4);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = (_Float16)(float)((int)((w >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15u) - 8) * d;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t b = t[kv4_v_code(dim, tp, 4 * li + i)];
                    v[2 * i] = (_Float16)(float)((int)(b & 15u) - 8) * d;
                    v[2 * i + 1] = (_Float16)(float)((int)(b >> 4) - 8) * d;
                }
            }
        }
        __builtin_memcpy(out + ((size_t)tok * kv + h) * dim + 8 * li, v, 16);
    }
}

} // namespace

hipError_t ah_launch_norm(const NormArgs &a, hipStream_t stream) {
    const uint32_t need = (a.n + 7) / 8, T = norm_lanes(a.n);
    auto *k = need <= 1024   ? (a.r ? norm_quant_kernel<1, true> : norm_quant_kernel<1, false>)
              : need <= 2048 ? (a.r ? norm_quant_kernel<2, true> : norm_quant_kernel<2, false>)
                             : (a.r ? norm_quant_kernel<4, true> : norm_quant_kernel<4, false>);
    hipLaunchKernelGGL(k, dim3(a.n_tok), dim3(T), 0, stream, a);
    return hipGetLastError();
}

hipError_t ah_launch_rope(const RopeArgs &a, hipStream_t stream) {
    hipLaunchKernelGGL(rope_kernel, dim3(a.n_tok), dim3(rope_lanes(a.rope.dim, a.n_heads)), 0, stream, a);
    return hipGetLastError();
}

hipError_t ah_launch_kv4_append(const AppendArgs &a, hipStream_t stream) {
    hipLaunchKernelGGL(kv4_append_kernel, dim3(a.t.n_tok), dim3(append_lanes(a.c, a.n_heads)), 0, stream, a);
    return hipGetLastError();
}

hipError_t ah_launch_kv4_read(const KvReadArgs &a, hipStream_t stream) {
    hipLaunchKernelGGL(kv4_read_kernel, dim3(a.t.n_tok), dim3(append_lanes(a.c, 0)), 0, stream, a);
    return hipGetLastError();
}
