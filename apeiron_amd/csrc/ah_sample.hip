// ah_sample.hip -- a token from the head's logits and a given random number.
//
// Order the row by (logit descending, index ascending).  With M the largest logit, a token's weight is
// the whole number w = rint(2^32 exp((l - M) / T)); sums of weights are exact in f64 (2^32 times at most
// 2^20 tokens), so no result depends on the order in which they are added.  Kept are the first k tokens
// (top-k), of those the ones whose preceding weight is below p times the weight of all k (top-p), and of
// those the ones with w >= min_p 2^32 (min-p); the first token always.  The draw is the smallest index
// at which the kept weight up to and with it, in index order, passes floor(u W).
//
// No sort: the kept set is a key and, within equal logits, an index; both come from selections by digits
// of the keys (the f32 bits as an unsigned number of the same order).
#include "ah_kv4.h"

namespace {

constexpr uint32_t kThreads = 1024, kMaxChunks = 256, kChunk = 4096;

AH_DEV uint32_t key_of(float l) {
    l = l != l ? -__builtin_inff() : l + 0.0f;  // NaN is never drawn; -0 and 0 are equal
    const uint32_t b = __builtin_bit_cast(uint32_t, l);
    return (int32_t)b < 0 ? ~b : b | 0x80000000u;
}
AH_DEV float logit_of(uint32_t k) { return __builtin_bit_cast(float, (int32_t)k < 0 ? k & 0x7fffffffu : ~k); }

// The weight of key k: a whole number of 2^-32, as f32 (exact: exp's 24 bits, rounded below 1).
AH_DEV float weight_of(uint32_t k, uint32_t top, float M, float inv_t) {
#pragma clang fp contract(off)
    if (k == top) return 0x1p32f;
    const float z = (logit_of(k) - M) * inv_t;
    return __builtin_rintf(expf(z) * 0x1p32f);
}

struct Shared {
    double mass[256];
    uint32_t count[256];
    double chunk[kMaxChunks];
    double wave_d[16];
    uint32_t wave_u[16];
    double d0;
    uint32_t u0, u1;
};

AH_DEV double block_sum(double v, Shared &S) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) S.wave_d[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0.0;
    for (uint32_t w = 0; w < kThreads / 64; ++w) t += S.wave_d[w];
    return t;
}
AH_DEV uint32_t block_min(uint32_t v, Shared &S) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = __builtin_elementwise_min(v, (uint32_t)__shfl_xor((int)v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) S.wave_u[threadIdx.x >> 6] = v;
    __syncthreads();
    uint32_t t = 0xffffffffu;
    for (uint32_t w = 0; w < kThreads / 64; ++w) t = __builtin_elementwise_min(t, S.wave_u[w]);
    return t;
}

// One workgroup per row.
__global__ void __launch_bounds__(kThreads) sample_row_kernel(SampleArgs a) {
    __shared__ Shared S;
    const uint32_t row = blockIdx.x, tid = threadIdx.x, V = a.n_vocab;
    const float *x = a.logits + (size_t)row * a.stride;
    float T = a.temperature ? a.temperature[row] : 1.0f;
    const int32_t k_in = a.top_k ? a.top_k[row] : 0;
    const float p_in = a.top_p ? a.top_p[row] : 1.0f, m_in = a.min_p ? a.min_p[row] : 0.0f, u_in = a.u[row];
    const unsigned long long key0 = (unsigned long long)row << 8;
    const bool bad_t = !(T >= 0.0f && T < __builtin_inff());
    if (tid == 0 && bad_t) ah_record(a.status, key0 + AH_ERR_INPUT_RANGE);

    uint32_t top = 0;
    bool nan = false;
    for (uint32_t i = tid; i < V; i += kThreads) {
        nan |= x[i] != x[i];
        top = __builtin_elementwise_max(top, key_of(x[i]));
    }
    if (nan) ah_record(a.status, key0 + AH_ERR_NONFINITE_INPUT);
    top = ~block_min(~top, S);
    const float M = logit_of(top);
    if (M == -__builtin_inff()) {  // nothing to draw
        if (tid == 0) {
            ah_record(a.status, key0 + AH_ERR_NONFINITE_INPUT);
            a.tokens[row] = -1;
            if (a.probs) a.probs[row] = 0.0f;
        }
        return;
    }
    if (bad_t || T == 0.0f || k_in == 1) {
        uint32_t at = 0xffffffffu;
        for (uint32_t i = tid; i < V; i += kThreads)
            if (key_of(x[i]) == top) at = __builtin_elementwise_min(at, i);
        at = block_min(at, S);
        if (tid == 0) {
            a.tokens[row] = (int32_t)at;
            if (a.probs) a.probs[row] = 1.0f;
        }
        return;
    }
    const float inv_t = 1.0f / T;

    // the cut: keys above `cut`, and of those equal to it the first `equal`, `have` being all of them
    uint32_t cut = 0, equal = 0xffffffffu;
    bool partial = false;  // not every token of the cut's logit is kept
    if (k_in > 1 && (uint32_t)k_in < V) {
        uint32_t need = (uint32_t)k_in, prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) S.count[tid] = 0;
            __syncthreads();
            for (uint32_t i = tid; i < V; i += kThreads) {
                const uint32_t k = key_of(x[i]);
                if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&S.count[(k >> shift) & 255u], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                uint32_t n = 0;
                int b = 255;
                for (; b > 0; --b) {
                    if (n + S.count[b] >= need) break;
                    n += S.count[b];
                }
                S.u0 = (uint32_t)b;
                S.u1 = n;
            }
            __syncthreads();
            prefix |= S.u0 << shift;
            need -= S.u1;
        }
        cut = prefix;
        equal = need;
        partial = S.count[S.u0] > need;
    }
    // the weight of the kept, and the cut by mass
    if (p_in < 1.0f) {
        const float w_cut = equal == 0xffffffffu ? 0.0f : weight_of(cut, top, M, inv_t);
        double W = 0.0;
        for (uint32_t i = tid; i < V; i += kThreads) {
            const uint32_t k = key_of(x[i]);
            if (equal == 0xffffffffu || k > cut) W += (double)weight_of(k, top, M, inv_t);
        }
        W = block_sum(W, S) + (equal == 0xffffffffu ? 0.0 : (double)equal * (double)w_cut);
        const double goal = (double)(p_in > 0.0f ? p_in : 0.0f) * W;
        double before = 0.0;
        uint32_t prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) {
                S.mass[tid] = 0.0;
                S.count[tid] = 0;
            }
            __syncthreads();
            for (uint32_t i = tid; i < V; i += kThreads) {
                const uint32_t k = key_of(x[i]);
                if ((equal == 0xffffffffu || k > cut) && (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))) {
                    atomicAdd(&S.mass[(k >> shift) & 255u], (double)weight_of(k, top, M, inv_t));
                    atomicAdd(&S.count[(k >> shift) & 255u], 1u);
                }
            }
            __syncthreads();
            if (tid == 0) {
                if (equal != 0xffffffffu && (shift == 24 || (cut >> (shift + 8)) == (prefix >> (shift + 8)))) {
                    S.mass[(cut >> shift) & 255u] += (double)equal * (double)w_cut;
                    S.count[(cut >> shift) & 255u] += equal;
                }
                double n = before;
                int b = 255, at = -1;
                for (; b >= 0; --b) {
                    if (!S.count[b]) continue;
                    at = b;  // the last digit in use, if no mass reaches the goal
                    if (n + S.mass[b] >= goal) break;
                    n += S.mass[b];
                }
                S.u0 = (uint32_t)at;
                S.u1 = b >= 0 ? 1u : 0u;
                S.d0 = b >= 0 ? n : n - S.mass[at];
            }
            __syncthreads();
            prefix |= S.u0 << shift;
            before = S.d0;
        }
        const uint32_t all = S.count[S.u0];
        const double w = (double)weight_of(prefix, top, M, inv_t);
        uint32_t n = all;
        if (w > 0.0) {
            double q = (goal - before) / w;
            n = q >= (double)all ? all : q <= 1.0 ? 1u : (uint32_t)q;
            while (n < all && before + (double)n * w < goal) ++n;
            while (n > 1 && before + (double)(n - 1) * w >= goal) --n;
        }
        partial = n < all || (equal != 0xffffffffu && prefix == cut && partial);
        cut = prefix;
        equal = n;
    }
    // the index of the last token kept of the cut's logit
    uint32_t last = 0xffffffffu;
    if (partial) {
        uint32_t seen = 0;
        for (uint32_t base = 0; base < V; base += kThreads) {
            const uint32_t i = base + tid;
            const bool eq = i < V && key_of(x[i]) == cut;
            const uint64_t b = __builtin_amdgcn_ballot_w64(eq);
            __syncthreads();
            if ((tid & 63) == 0) S.wave_u[tid >> 6] = (uint32_t)__builtin_popcountll(b);
            __syncthreads();
            uint32_t mine = seen, total = 0;
            for (uint32_t w = 0; w < kThreads / 64; ++w) {
                if (w < (tid >> 6)) mine += S.wave_u[w];
                total += S.wave_u[w];
            }
            mine += (uint32_t)__builtin_popcountll(b & ((1ull << (tid & 63)) - 1));
            if (eq && mine + 1 == equal) S.u0 = i;
            seen += total;
            if (seen >= equal) break;
        }
        __syncthreads();
        last = S.u0;
        __syncthreads();
    }
    const double floor_w = (double)(m_in > 0.0f ? (m_in < 1.0f ? m_in : 1.0f) : 0.0f) * 0x1p32;
    auto kept = [&](uint32_t i) -> double {
        const uint32_t k = key_of(x[i]);
        if (k < cut || (k == cut && i > last)) return 0.0;
        const float w = weight_of(k, top, M, inv_t);
        return (double)w < floor_w ? 0.0 : (double)w;
    };
    const uint32_t chunks = (V + kChunk - 1) / kChunk;
    double W = 0.0;
    for (uint32_t c = 0; c < chunks; ++c) {
        double s = 0.0;
        for (uint32_t j = 0; j < kChunk / kThreads; ++j) {
            const uint32_t i = c * kChunk + j * kThreads + tid;
            if (i < V) s += kept(i);
        }
        s = block_sum(s, S);
        if (tid == 0) S.chunk[c] = s;
        W += s;
    }
    __syncthreads();
    double goal = __builtin_floor((double)(u_in > 0.0f ? u_in : 0.0f) * W);
    goal = goal < W ? goal : W - 1.0;
    uint32_t c = 0;
    double before = 0.0;
    while (c + 1 < chunks && before + S.chunk[c] <= goal) before += S.chunk[c++];
    // inside the chunk: 1024 tokens at a time, a prefix sum over them
    for (uint32_t j = 0; j < kChunk / kThreads; ++j) {
        const uint32_t i = c * kChunk + j * kThreads + tid;
        const double w = i < V ? kept(i) : 0.0;
        double pre = w;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double t = __shfl_up(pre, o, 64);
            if ((int)(tid & 63) >= o) pre += t;
        }
        __syncthreads();
        if ((tid & 63) == 63) S.wave_d[tid >> 6] = pre;
        __syncthreads();
        double off = before, all = 0.0;
        for (uint32_t v = 0; v < kThreads / 64; ++v) {
            if (v < (tid >> 6)) off += S.wave_d[v];
            all += S.wave_d[v];
        }
        if (w > 0.0 && off + pre > goal && off + pre - w <= goal) {
            a.tokens[row] = (int32_t)i;
            if (a.probs) a.probs[row] = (float)(w / W);
        }
        before += all;
        if (before > goal) break;
    }
}

} // namespace

hipError_t ah_launch_sample(const SampleArgs &a, hipStream_t stream) {
    hipLaunchKernelGGL(sample_row_kernel, dim3(a.n_rows), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}
