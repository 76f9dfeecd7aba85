// ah_sample.hip -- a token from the head's logits and a given random number.
//
// Order the row by (logit descending, index ascending).  With M the largest logit, a token's weight is
// the whole number w = rint(2^32 exp((l - M) / T)); sums of weights are exact in f64 (2^32 times at most
// 2^20 tokens), so no result depends on the order in which they are added.  Kept are the first k tokens
// (top-k), of those the ones whose preceding weight is below p times the weight of all k (top-p), and of
// those the ones with w >= min_p 2^32 (min-p); the first token always.  The draw is the smallest index
// at which the kept weight up to and with it, in index order, passes floor(u W).
//
// No sort.  Four launches over segments of 512 tokens (a wave's eight tokens a lane), each reading the row
// at most once:
//   scan    the largest key of every group of 64 tokens and of every segment (a key is the f32 bits as an
//           unsigned number of the same order), and so M;
//   count   the tokens and their weight in 1024 bins of (M - l) / T.  With top-k, the k-th largest segment
//           or group maximum bounds the k-th largest logit from below, and only what reaches it is counted;
//   gather  from the bins: those kept for certain, those dropped, and the few that a limit falls into,
//           whose tokens are listed; and each segment's certain weight;
//   draw    one workgroup a row orders the listed tokens, cuts them, draws a segment and a token in it.
// A row whose listed tokens pass the lists' room (thousands of equal logits) is cut by selections over
// the whole row instead.  What bounds it: the row's bytes for many rows (one read from HBM, two more from
// the cache that holds it), four dependent launches for one.
#include "ah_kv4.h"

namespace {

constexpr uint32_t kT = 256;            // threads of every workgroup here
constexpr uint32_t kSeg = 512;          // tokens of a segment: eight a lane of one wave
constexpr uint32_t kGroup = 64;         // tokens of a group: eight lanes
constexpr uint32_t kGroups = kSeg / kGroup;
constexpr uint32_t kBins = 1024;
constexpr float kBinScale = kBins / 23.0f;  // w is 0 past (M - l) / T = 22.9
constexpr uint32_t kNone = 0xffffffffu;

AH_DEV uint32_t key_of(float l) {
    l = l != l ? -__builtin_inff() : l + 0.0f;  // NaN is never drawn; -0 and 0 are equal
    const uint32_t b = __builtin_bit_cast(uint32_t, l);
    return (int32_t)b < 0 ? ~b : b | 0x80000000u;
}
AH_DEV float logit_of(uint32_t k) { return __builtin_bit_cast(float, (int32_t)k < 0 ? k & 0x7fffffffu : ~k); }

// A row's parameters and what follows from its largest key.
struct Row {
    const float *x;
    float T, p, m, u;
    int32_t k;
    uint32_t V, top;
    float M, inv_t;
    double floor_w;
    float floor_f;  // the least f32 not below it
    bool bad_t, greedy, need_k, need_p;
    bool few;  // so few tokens asked for that the segments' maxima bound them: the bins are not needed
};
AH_DEV Row row_of(const SampleArgs &a, uint32_t row) {
    Row r;
    r.x = a.logits + (size_t)row * a.stride;
    r.V = a.n_vocab;
    r.T = a.temperature ? a.temperature[row] : 1.0f;
    r.k = a.top_k ? a.top_k[row] : 0;
    r.p = a.top_p ? a.top_p[row] : 1.0f;
    r.m = a.min_p ? a.min_p[row] : 0.0f;
    r.u = a.u[row];
    r.bad_t = !(r.T >= 0.0f && r.T < __builtin_inff());
    r.greedy = r.bad_t || r.T == 0.0f || r.k == 1;
    r.need_k = r.k > 1 && (uint32_t)r.k < r.V;
    r.need_p = r.p < 1.0f;
    r.few = !r.greedy && r.need_k && (uint64_t)r.k * 2 <= a.segs;
    r.floor_w = (double)(r.m > 0.0f ? (r.m < 1.0f ? r.m : 1.0f) : 0.0f) * 0x1p32;
    r.floor_f = (float)r.floor_w;
    if ((double)r.floor_f < r.floor_w) r.floor_f = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, r.floor_f) + 1);
    return r;
}
AH_DEV void set_top(Row &r, uint32_t top) {
    r.top = top;
    r.M = logit_of(top);
    r.inv_t = 1.0f / r.T;
}
// A logit's z = (l - M) / T, from the logit itself (NaN as -inf) or its key (0 past the row's end).
AH_DEV float z_at(const Row &r, float l) {
#pragma clang fp contract(off)
    l = __builtin_fmaxf(l, -__builtin_inff());
    return l == r.M ? 0.0f : (l - r.M) * r.inv_t;
}
AH_DEV float z_of(const Row &r, uint32_t k) { return k ? z_at(r, logit_of(k)) : -__builtin_inff(); }
// The weight: a whole number, as f32 (exact: exp's 24 bits, rounded below 1).  exp(z) = 2^(z log2 e), the
// product's own rounding carried as a factor next to 1: about 1.5 units of f32's last place.
AH_DEV float weight_at(float z) {
#pragma clang fp contract(off)
    const float l2e = 0x1.715476p+0f, rest = 0x1.4ae0cp-26f, ln2 = 0x1.62e43p-1f;  // log2 e = l2e + rest
    z = __builtin_fmaxf(z, -28.0f);  // (the weight is 0 there; z may be -inf)
    const float t = z * l2e, d = __builtin_fmaf(z, rest, __builtin_fmaf(z, l2e, -t)), e = __builtin_amdgcn_exp2f(t);
    return __builtin_rintf(__builtin_fmaf(e, d * ln2, e) * 0x1p32f);
}
// The bin of z, kBins where the weight is 0.
AH_DEV uint32_t bin_at(float z) { return (uint32_t)__builtin_fminf(z * -kBinScale, (float)kBins); }

// ---- workgroup scans (kT threads) -------------------------------------------------------------------

// v of another lane through DPP (no LDS); lanes without a source, and rows outside ROWS, get 0.
template <int CTRL, int ROWS> AH_DEV uint32_t dpp0(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS> AH_DEV double dpp0(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)dpp0<CTRL, ROWS>((uint32_t)(b >> 32)) << 32 | dpp0<CTRL, ROWS>((uint32_t)b));
}
struct Add {
    template <class T> AH_DEV T operator()(T a, T b) const { return a + b; }
};
struct Max {
    AH_DEV uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
};
// Inclusive prefix over the wave (0 the operation's identity): inside rows of 16 by shifts of 1, 2, 4 and 8,
// then the rows' ends passed on.
template <class Op, class T> AH_DEV T wave_prefix(T v) {
    const Op op;
    v = op(v, dpp0<0x111, 0xF>(v));
    v = op(v, dpp0<0x112, 0xF>(v));
    v = op(v, dpp0<0x114, 0xF>(v));
    v = op(v, dpp0<0x118, 0xF>(v));
    v = op(v, dpp0<0x142, 0xA>(v));
    return op(v, dpp0<0x143, 0xC>(v));
}
AH_DEV uint32_t last_lane(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, 63); }
AH_DEV double last_lane(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)last_lane((uint32_t)(b >> 32)) << 32 | last_lane((uint32_t)b));
}

struct Scan {
    double d[kT / 64];
    uint32_t u[kT / 64];
    AH_DEV double *of(double) { return d; }
    AH_DEV uint32_t *of(uint32_t) { return u; }
};
// Inclusive prefix of v over the workgroup's threads, and the total.
template <class Op, class T> AH_DEV T scan(T v, Scan &S, T &total) {
    const Op op;
    const uint32_t wave = threadIdx.x >> 6;
    T *at = S.of(v);
    v = wave_prefix<Op>(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) at[wave] = v;
    __syncthreads();
    total = (T)0;
#pragma unroll
    for (uint32_t w = 0; w < kT / 64; ++w) {
        if (w < wave) v = op(v, at[w]);
        total = op(total, at[w]);
    }
    return v;
}
AH_DEV double scan_d(double v, Scan &S, double &total) { return scan<Add>(v, S, total); }
AH_DEV uint32_t scan_u(uint32_t v, Scan &S, uint32_t &total) { return scan<Add>(v, S, total); }
AH_DEV double sum_d(double v, Scan &S) {
    double total;
    scan<Add>(v, S, total);
    return total;
}
AH_DEV uint32_t max_u(uint32_t v, Scan &S) {
    uint32_t total;
    scan<Max>(v, S, total);
    return total;
}
AH_DEV uint32_t min_u(uint32_t v, Scan &S) { return ~max_u(~v, S); }

// A lane's eight logits of a segment (-inf past the row's end), and their keys (0, below every key, there).
AH_DEV void load_logits(const Row &r, uint32_t seg, float *x) {
    const uint32_t i0 = seg * kSeg + 8 * (threadIdx.x & 63);
    if (i0 + 8 <= r.V) __builtin_memcpy(x, r.x + i0, 32);
    else
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) x[i] = i0 + i < r.V ? r.x[i0 + i] : -__builtin_inff();
}
AH_DEV void keys_of(const Row &r, uint32_t seg, const float *x, uint32_t *k) {
    const uint32_t i0 = seg * kSeg + 8 * (threadIdx.x & 63);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) k[i] = i0 + i < r.V ? key_of(x[i]) : 0u;
}
AH_DEV void load_keys(const Row &r, uint32_t seg, uint32_t *k) {
    float x[8];
    load_logits(r, seg, x);
    keys_of(r, seg, x, k);
}

AH_DEV uint32_t top_of(const SampleArgs &a, uint32_t row, Scan &S) {
    const uint32_t *g = a.seg_max + (size_t)row * a.segs;
    uint32_t top = 0;
    for (uint32_t i = threadIdx.x; i < a.segs; i += kT) top = __builtin_elementwise_max(top, g[i]);
    return max_u(top, S);
}

// The workgroup's row, and the segments of this wave: s0, s0 + 4, .. below s1.
AH_DEV void share(const SampleArgs &a, uint32_t &row, uint32_t &s0, uint32_t &s1) {
    row = blockIdx.x / a.parts;
    const uint32_t b = (blockIdx.x - row * a.parts) * a.per;
    s0 = b + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    s1 = b + a.per < a.segs ? b + a.per : a.segs;
}

// Calls f(segment, logits) for those of this wave's segments whose largest token's bin is at most `last`, the next
// one's logits on their way meanwhile; skipped(segment) with a lane for each of the others.
template <class F, class G> AH_DEV void each_segment(const SampleArgs &a, const Row &r, uint32_t row, uint32_t s0, uint32_t s1, uint32_t last, F f, G skipped) {
    constexpr uint32_t W = kT / 64;
    for (uint32_t base = s0; base < s1; base += 64 * W) {
        const uint32_t mine = base + W * (threadIdx.x & 63);
        const bool in = mine < s1, use = in && bin_at(z_of(r, a.seg_max[(size_t)row * a.segs + (in ? mine : base)])) <= last;
        if (in && !use) skipped(mine);
        uint64_t todo = __builtin_amdgcn_ballot_w64(use);
        float x[8], next[8];
        if (todo) load_logits(r, base + W * (uint32_t)__builtin_ctzll(todo), next);
        while (todo) {
            const uint32_t s = base + W * (uint32_t)__builtin_ctzll(todo);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = next[i];
            todo &= todo - 1;
            if (todo) load_logits(r, base + W * (uint32_t)__builtin_ctzll(todo), next);
            f(s, x);
        }
    }
}

__global__ void __launch_bounds__(kT) sample_scan_kernel(SampleArgs a) {
    uint32_t row, s0, s1;
    share(a, row, s0, s1);
    Row r;
    r.x = a.logits + (size_t)row * a.stride;
    r.V = a.n_vocab;
    if (blockIdx.x % a.parts == 0) {  // the row's bins, for the next launch
        for (uint32_t i = threadIdx.x; i < kBins; i += kT) {
            a.bin_mass[(size_t)row * kBins + i] = 0.0;
            a.bin_count[(size_t)row * kBins + i] = 0;
        }
    }
    bool nan = false;
    for (uint32_t s = s0; s < s1; s += kT / 64) {
        float x[8];
        uint32_t k[8], top = 0;
        load_logits(r, s, x);
        keys_of(r, s, x, k);
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            nan |= x[i] != x[i];
            top = __builtin_elementwise_max(top, k[i]);
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = __builtin_elementwise_max(top, (uint32_t)__shfl_xor((int)top, o, 64));
        const uint32_t lane = threadIdx.x & 63;
        const size_t seg = (size_t)row * a.segs + s;
        if ((lane & 7) == 0) a.group_max[seg * kGroups + lane / 8] = top;
#pragma unroll
        for (int o = 8; o < 64; o <<= 1) top = __builtin_elementwise_max(top, (uint32_t)__shfl_xor((int)top, o, 64));
        if (lane == 0) a.seg_max[seg] = top;
    }
    if (nan) ah_record(a.status, ((unsigned long long)row << 8) + AH_ERR_NONFINITE_INPUT);
}

// The last bin that can hold one of the first k: every segment's (or group's) largest is a token of its own, so the
// k-th largest of them bounds the k-th largest logit from below.  Segments do where there are twice k of them.
AH_DEV uint32_t bound_of(const SampleArgs &a, const Row &r, uint32_t row, Scan &S, uint32_t *count, uint32_t &found) {
    for (uint32_t i = threadIdx.x; i < kBins; i += kT) count[i] = 0;
    if (threadIdx.x == 0) found = kBins - 1;
    __syncthreads();
    const uint32_t *g = r.few ? a.seg_max + (size_t)row * a.segs : a.group_max + (size_t)row * a.segs * kGroups;
    const uint32_t n = r.few ? a.segs : a.segs * kGroups;
    for (uint32_t i = threadIdx.x; i < n; i += kT) {
        const uint32_t b = bin_at(z_of(r, g[i]));
        if (b < kBins) atomicAdd(&count[b], 1u);
    }
    __syncthreads();
    uint32_t c[4], total;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = count[4 * threadIdx.x + i];
    const uint32_t mine = (c[0] + c[1]) + (c[2] + c[3]);
    uint32_t cum = scan_u(mine, S, total) - mine;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (cum < (uint32_t)r.k && cum + c[i] >= (uint32_t)r.k) found = 4 * threadIdx.x + i;
        cum += c[i];
    }
    __syncthreads();
    return found;
}

__global__ void __launch_bounds__(kT) sample_count_kernel(SampleArgs a) {
    __shared__ double mass[kBins];
    __shared__ uint32_t count[kBins];
    __shared__ Scan S;
    __shared__ uint32_t found;
    uint32_t row, s0, s1;
    share(a, row, s0, s1);
    Row r = row_of(a, row);
    if (r.greedy || r.few || (!r.need_k && !r.need_p)) return;
    set_top(r, top_of(a, row, S));
    if (r.M == -__builtin_inff()) return;
    const uint32_t last = r.need_k ? bound_of(a, r, row, S, count, found) : kBins - 1;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kBins; i += kT) {
        count[i] = 0;
        mass[i] = 0.0;
    }
    __syncthreads();
    each_segment(
        a, r, row, s0, s1, last,
        [&](uint32_t, const float *x) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float z = z_at(r, x[i]);
                const uint32_t b = bin_at(z);
                if (b > last) continue;
                if (r.need_k) atomicAdd(&count[b], 1u);
                if (r.need_p) unsafeAtomicAdd(&mass[b], (double)weight_at(z));
            }
        },
        [](uint32_t) {});
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kBins; i += kT) {
        if (count[i]) atomicAdd(&a.bin_count[(size_t)row * kBins + i], count[i]);
        if (mass[i] > 0.0) unsafeAtomicAdd(&a.bin_mass[(size_t)row * kBins + i], mass[i]);
    }
}

// What the bins say.  Tokens of bins below g0 are kept and those of bins past g1 dropped (min-p apart); the
// k-th token is in bin bk (kNone: fewer than k tokens have weight), `before_k` tokens weighing `mass_k` ahead of
// that bin; `mass_0` is the weight ahead of bin g0 and `all` that of every bin.
struct Limits {
    uint32_t g0, g1, bk, before_k;
    double mass_k, mass_0, all;
};
struct LimitsLds {
    uint32_t bk, before_k, g0, g1;
    double mass_k, mass_0, w_low, w_high;
};
// A thread's four bins, loaded ahead of what else a kernel waits for.
struct Bins {
    uint32_t c[4];
    double m[4];
    AH_DEV Bins(const SampleArgs &a, uint32_t row) {
        __builtin_memcpy(c, a.bin_count + (size_t)row * kBins + 4 * threadIdx.x, 16);
        __builtin_memcpy(m, a.bin_mass + (size_t)row * kBins + 4 * threadIdx.x, 32);
    }
};
AH_DEV Limits limits_of(const SampleArgs &a, const Row &r, const Bins &B, Scan &S, LimitsLds &L) {
    Limits o = {kBins, kBins, kNone, 0, 0.0, 0.0, 0.0};
    if (!r.need_k && !r.need_p) return o;
    const uint32_t t = threadIdx.x;
    const uint32_t *c = B.c;
    const double *m = B.m;
    if (t == 0) {
        L.bk = kNone;
        L.g0 = L.g1 = kBins - 1;
    }
    uint32_t total;
    const uint32_t csum = (c[0] + c[1]) + (c[2] + c[3]);
    const double msum = (m[0] + m[1]) + (m[2] + m[3]);
    uint32_t cum = scan_u(csum, S, total) - csum;
    double all;
    const double m0 = scan_d(msum, S, all) - msum;
    double cm = m0;
    if (r.need_k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (cum < (uint32_t)r.k && cum + c[i] >= (uint32_t)r.k) {
                L.bk = 4 * t + i;
                L.before_k = cum;
                L.mass_k = cm;
                L.w_high = cm + m[i];
            }
            cum += c[i];
            cm += m[i];
        }
        __syncthreads();
        o.bk = L.bk;
    }
    if (o.bk != kNone) {
        o.before_k = L.before_k;
        o.mass_k = L.mass_k;
    }
    if (!r.need_p) {
        o.g0 = o.g1 = o.bk != kNone ? o.bk : kBins;
        return o;
    }
    // the weight of the first k is between these, and so is the limit between p times them
    const double p = (double)(r.p > 0.0f ? r.p : 0.0f);
    const double low = p * (o.bk != kNone ? o.mass_k : all), high = p * (o.bk != kNone ? L.w_high : all);
    cm = m0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double next = cm + m[i];
        const uint32_t b = 4 * t + i;
        if (next >= low && (b == 0 || cm < low)) {
            L.g0 = b;
            L.mass_0 = cm;
        }
        if (next >= high && (b == 0 || cm < high)) L.g1 = b;
        cm = next;
    }
    __syncthreads();
    o.g0 = L.g0;
    o.g1 = o.bk < L.g1 ? o.bk : L.g1;
    o.mass_0 = L.mass_0;
    o.all = all;
    return o;
}
// Whether a bin's tokens are listed: bins g0 to g1, and the top-k one where top-p needs its weight.  (No branches.)
struct Listed {
    uint32_t from, span, also;
    AH_DEV Listed(const Limits &o, const Row &r) {
        const uint32_t to = o.g1 < kBins ? o.g1 : kBins - 1;
        from = o.g0 <= to ? o.g0 : 0xfffff000u;  // (no bin is that far below it)
        span = o.g0 <= to ? to - o.g0 : 0u;
        also = r.need_p ? o.bk : kNone;
    }
    AH_DEV bool operator()(uint32_t b) const { return (b - from <= span) | (b == also); }
};

__global__ void __launch_bounds__(kT) sample_gather_kernel(SampleArgs a) {
    __shared__ Scan S;
    __shared__ LimitsLds L;
    __shared__ uint32_t count[kBins], found;
    uint32_t row, s0, s1;
    share(a, row, s0, s1);
    const Bins B(a, row);
    Row r = row_of(a, row);
    if (r.greedy) return;
    set_top(r, top_of(a, row, S));
    if (r.M == -__builtin_inff()) return;
    Limits o = {0, 0, kNone, 0, 0.0, 0.0, 0.0};
    if (r.few) o.g1 = bound_of(a, r, row, S, count, found);  // all that reaches the bound is listed
    else o = limits_of(a, r, B, S, L);
    const uint32_t lane = threadIdx.x & 63, g0 = o.g0 < kBins ? o.g0 : kBins;
    const Listed listed(o, r);
    // the last bin with a token to keep or to list (no bin: tokens without weight, as a whole)
    const uint32_t end_k = o.bk != kNone ? o.bk : o.g1;
    const uint32_t last = o.g0 == kBins ? kBins - 1 : end_k > o.g1 ? end_k : o.g1;
    each_segment(
        a, r, row, s0, s1, last,
        [&](uint32_t s, const float *x) {
            const size_t seg = (size_t)row * a.segs + s;
            uint32_t n = 0, mask = 0;
            double sure = 0.0;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const float z = z_at(r, x[i]);
                const uint32_t b = bin_at(z);
                // (no branches: the row's lanes take both sides nearly always)
                const float w = weight_at(z);
                sure += (double)(((b < g0) & (w >= r.floor_f)) ? w : 0.0f);
                mask |= (uint32_t)listed(b) << i;
            }
            n = (uint32_t)__builtin_popcount(mask);
            uint32_t total = 0;
            if (__builtin_amdgcn_ballot_w64(n != 0) != 0ull) {
                const uint32_t end = wave_prefix<Add>(n);
                total = last_lane(end);
                uint32_t at = end - n;
                if (total <= kSampleSegList) {
                    uint16_t *list = a.list + seg * kSampleSegList;
                    for (; mask; mask &= mask - 1) list[at++] = (uint16_t)(8 * lane + (uint32_t)__builtin_ctz(mask));
                }
            }
            if (__builtin_amdgcn_ballot_w64(sure > 0.0) != 0ull) sure = last_lane(wave_prefix<Add>(sure));
            if (lane == 0) {
                a.seg_mass[seg] = sure;
                a.seg_count[seg] = total;
            }
        },
        [&](uint32_t s) {
            a.seg_mass[(size_t)row * a.segs + s] = 0.0;
            a.seg_count[(size_t)row * a.segs + s] = 0;
        });
}

// ---- the cut ----------------------------------------------------------------------------------------

struct DrawLds {
    alignas(16) double mass[256];
    alignas(16) uint32_t count[256];
    Scan S;
    LimitsLds L;
    double seg[kSampleMaxSegs];
    uint32_t start[kSampleMaxSegs];
    uint32_t key[kSampleList], idx[kSampleList];
    uint32_t u0, u1;
    double d0;
};

// The kept set's last token in the order: keys above `key` are kept, and of those equal to it the ones up
// to index `last`.
struct Cut {
    uint32_t key, last;
};

// The index of the nth (1 ..) of n tokens in index order that have key `cut`.
template <class Key, class Index> AH_DEV uint32_t nth_equal(uint32_t n, Key key, Index index, uint32_t cut, uint32_t nth, DrawLds &D) {
    uint32_t seen = 0;
    for (uint32_t base = 0; base < n && seen < nth; base += kT) {
        const uint32_t i = base + threadIdx.x;
        const bool eq = i < n && key(i) == cut;
        uint32_t total;
        const uint32_t at = seen + scan_u(eq, D.S, total);
        if (eq && at == nth) D.u0 = index(i);
        seen += total;
    }
    __syncthreads();
    return D.u0;
}

// The digit at which keys between lo and hi first differ, as a shift, and what they share above it.
AH_DEV int first_digit(uint32_t lo, uint32_t hi, uint32_t &shared) {
    const uint32_t x = lo ^ hi;
    const int shift = x ? (31 - __builtin_clz(x)) / 8 * 8 : 0;
    shared = shift == 24 ? 0 : hi >> (shift + 8) << (shift + 8);
    return shift;
}

// The cut over n tokens in index order (a list, or the whole row), by digits of the keys.  in_k(key) and
// in_p(key): whether such a token counts for the top-k and for the top-p limit.  need: tokens that top-k still
// keeps of its own; W0: the weight ahead of those (without top-k: of every token); before: the weight ahead of
// top-p's.
template <class Key, class Index, class InK, class InP>
AH_DEV Cut select_cut(const Row &r, uint32_t n, Key key, Index index, InK in_k, InP in_p, bool do_k, uint32_t need, double W0, double before,
                      DrawLds &D) {
    const uint32_t t = threadIdx.x;
    Cut c = {0, kNone};
    uint32_t keep = 0, cut_k = 0;  // of those at the cut
    bool partial = false;
    if (do_k) {
        uint32_t lo = kNone, hi = 0;
        for (uint32_t i = t; i < n; i += kT) {
            const uint32_t k = key(i);
            if (in_k(k)) {
                lo = __builtin_elementwise_min(lo, k);
                hi = __builtin_elementwise_max(hi, k);
            }
        }
        lo = min_u(lo, D.S);
        hi = max_u(hi, D.S);
        for (int shift = first_digit(lo, hi, cut_k); shift >= 0; shift -= 8) {
            __syncthreads();
            D.count[t] = 0;
            __syncthreads();
            for (uint32_t i = t; i < n; i += kT) {
                const uint32_t k = key(i);
                if (in_k(k) && (shift == 24 || (k >> (shift + 8)) == (cut_k >> (shift + 8)))) atomicAdd(&D.count[(k >> shift) & 255u], 1u);
            }
            __syncthreads();
            const uint32_t mine = D.count[255 - t];
            uint32_t total;
            const uint32_t cum = scan_u(mine, D.S, total);
            if (cum >= need && cum - mine < need) {
                D.u0 = 255 - t;
                D.u1 = cum - mine;
            }
            __syncthreads();
            cut_k |= D.u0 << shift;
            need -= D.u1;
        }
        keep = need;
        partial = D.count[D.u0] > need;
        c.key = cut_k;
    }
    if (r.need_p) {
        const double w_cut = do_k ? (double)weight_at(z_of(r, cut_k)) : 0.0;
        double W = W0;
        if (do_k) {
            double s = 0.0;
            for (uint32_t i = t; i < n; i += kT) {
                const uint32_t k = key(i);
                if (in_k(k) && k > cut_k) s += (double)weight_at(z_of(r, k));
            }
            W += sum_d(s, D.S) + (double)keep * w_cut;
        }
        double goal = (double)(r.p > 0.0f ? r.p : 0.0f) * W;
        goal = goal < 1.0 ? 1.0 : goal;  // the first token always
        uint32_t cut_p = 0, all = 0, lo = do_k && in_p(cut_k) ? cut_k : kNone, hi = lo == kNone ? 0u : cut_k;
        for (uint32_t i = t; i < n; i += kT) {
            const uint32_t k = key(i);
            if (in_p(k) && !(do_k && k <= cut_k)) {
                lo = __builtin_elementwise_min(lo, k);
                hi = __builtin_elementwise_max(hi, k);
            }
        }
        lo = min_u(lo, D.S);
        hi = max_u(hi, D.S);
        for (int shift = first_digit(lo, hi, cut_p); shift >= 0; shift -= 8) {
            __syncthreads();
            D.mass[t] = 0.0;
            D.count[t] = 0;
            __syncthreads();
            for (uint32_t i = t; i < n; i += kT) {
                const uint32_t k = key(i);
                if (!in_p(k) || (do_k && k <= cut_k) || !(shift == 24 || (k >> (shift + 8)) == (cut_p >> (shift + 8)))) continue;
                unsafeAtomicAdd(&D.mass[(k >> shift) & 255u], (double)weight_at(z_of(r, k)));
                atomicAdd(&D.count[(k >> shift) & 255u], 1u);
            }
            __syncthreads();
            double mine = D.mass[255 - t];
            uint32_t cnt = D.count[255 - t];
            if (do_k && in_p(cut_k) && (shift == 24 || (cut_k >> (shift + 8)) == (cut_p >> (shift + 8))) && 255 - t == ((cut_k >> shift) & 255u)) {
                mine += (double)keep * w_cut;
                cnt += keep;
            }
            double total;
            const double cum = before + scan_d(mine, D.S, total);
            if (cum >= goal && cum - mine < goal) {
                D.u0 = 255 - t;
                D.u1 = cnt;
                D.d0 = cum - mine;
            }
            __syncthreads();
            cut_p |= D.u0 << shift;
            all = D.u1;
            before = D.d0;
        }
        const double w = (double)weight_at(z_of(r, cut_p)), q = (goal - before) / w;
        uint32_t m = q >= (double)all ? all : q <= 1.0 ? 1u : (uint32_t)q;
        while (m < all && before + (double)m * w < goal) ++m;
        while (m > 1 && before + (double)(m - 1) * w >= goal) --m;
        partial = m < all || (do_k && cut_p == cut_k && partial);
        keep = m;
        c.key = cut_p;
    }
    if (partial) c.last = nth_equal(n, key, index, c.key, keep, D);
    return c;
}

// The cut of at most kT / P listed tokens: P neighbouring threads a token, its place among the others by comparing
// with each (four at a time; tokens that do not count are key 0, below every key).
template <uint32_t P> AH_DEV Cut place_cut(const Row &r, const Limits &o, uint32_t n, bool do_k, DrawLds &D) {
    const uint32_t t = threadIdx.x, me = t / P, part = t % P;
    const bool live = me < n;
    const uint32_t k = live ? D.key[me] : 0u;
    const float z = z_of(r, k);
    const uint32_t b = bin_at(z);
    const bool ink = live && do_k && (r.few || b == o.bk), inp = live && b >= o.g0 && b <= o.g1;
    const double w = live ? (double)weight_at(z) : 0.0;
    bool keep = live;
    if (do_k) {
        if (part == 0) D.count[me] = ink ? k : 0u;
        __syncthreads();
        uint32_t rank = 0;
#pragma unroll 2
        for (uint32_t j = 4 * part; j < n; j += 4 * P) {
            uint32_t other[4];
            __builtin_memcpy(other, D.count + j, 16);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) rank += other[i] > (j + i < me ? k - 1 : k) ? 1u : 0u;
        }
#pragma unroll
        for (uint32_t q = 1; q < P; q <<= 1) rank += (uint32_t)__shfl_xor((int)rank, (int)q, 64);
        keep = ink ? o.before_k + rank < (uint32_t)r.k : live;
    }
    if (r.need_p) {
        const double W = do_k || r.few ? o.mass_k + sum_d((ink || r.few) && keep && part == 0 ? w : 0.0, D.S) : o.all;
        double goal = (double)(r.p > 0.0f ? r.p : 0.0f) * W;
        goal = goal < 1.0 ? 1.0 : goal;
        __syncthreads();
        if (part == 0) {
            D.count[me] = inp && keep ? k : 0u;
            D.mass[me] = inp && keep ? w : 0.0;
        }
        __syncthreads();
        double before = 0.0;
#pragma unroll 2
        for (uint32_t j = 4 * part; j < n; j += 4 * P) {
            uint32_t other[4];
            double m[4];
            __builtin_memcpy(other, D.count + j, 16);
            __builtin_memcpy(m, D.mass + j, 32);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) before += other[i] > (j + i < me ? k - 1 : k) ? m[i] : 0.0;
        }
#pragma unroll
        for (uint32_t q = 1; q < P; q <<= 1) before += __shfl_xor(before, (int)q, 64);
        keep = inp && keep && o.mass_0 + before < goal;
    } else {
        keep = ink && keep;
    }
    Cut c;
    c.key = min_u(keep ? k : kNone, D.S);
    c.last = max_u(keep && k == c.key ? D.idx[me] : 0u, D.S);
    return c;
}

__global__ void __launch_bounds__(kT) sample_draw_kernel(SampleArgs a) {
    __shared__ DrawLds D;
    const uint32_t row = blockIdx.x, t = threadIdx.x;
    const Bins B(a, row);
    // this thread's segments: their certain weights, and how many tokens each lists
    const uint32_t each = (a.segs + kT - 1) / kT, g0 = t * each < a.segs ? t * each : a.segs, g1 = g0 + each < a.segs ? g0 + each : a.segs;
    uint32_t n_mine = 0;
    bool full = false;
    for (uint32_t s = g0; s < g1; ++s) {
        const uint32_t c = a.seg_count[(size_t)row * a.segs + s];
        D.seg[s] = a.seg_mass[(size_t)row * a.segs + s];
        D.start[s] = c;
        full |= c > kSampleSegList;
        n_mine += c;
    }
    Row r = row_of(a, row);
    const unsigned long long key0 = (unsigned long long)row << 8;
    if (t == 0 && r.bad_t) ah_record(a.status, key0 + AH_ERR_INPUT_RANGE);
    set_top(r, top_of(a, row, D.S));
    if (r.M == -__builtin_inff()) {  // nothing to draw
        if (t == 0) {
            ah_record(a.status, key0 + AH_ERR_NONFINITE_INPUT);
            a.tokens[row] = -1;
            if (a.probs) a.probs[row] = 0.0f;
        }
        return;
    }
    if (r.greedy) {  // the first group that holds the largest, and in it the first token
        const uint32_t *g = a.group_max + (size_t)row * a.segs * kGroups;
        uint32_t at = kNone;
        for (uint32_t i = t; i < a.segs * kGroups; i += kT)
            if (g[i] == r.top) at = __builtin_elementwise_min(at, i);
        at = min_u(at, D.S);
        const uint32_t i = at * kGroup + t;
        const bool here = t < kGroup && i < r.V && key_of(r.x[i]) == r.top;
        const uint64_t b = __builtin_amdgcn_ballot_w64(here);
        if (t == 0) {
            a.tokens[row] = (int32_t)(at * kGroup + (uint32_t)__builtin_ctzll(b));
            if (a.probs) a.probs[row] = 1.0f;
        }
        return;
    }
    Limits o = {0, kBins - 1, kNone, 0, 0.0, 0.0, 0.0};
    if (!r.few) o = limits_of(a, r, B, D.S, D.L);
    uint32_t n;
    {  // where each segment's listed tokens start
        uint32_t at = scan_u(n_mine, D.S, n) - n_mine;
        for (uint32_t s = g0; s < g1; ++s) {
            const uint32_t c = D.start[s];
            D.start[s] = at;
            at += c;
        }
    }
    full = max_u(full, D.S) != 0 || n > kSampleList;
    // (of few, every listed token counts for both limits; fewer than k of them are all that have weight)
    const bool do_k = r.few ? n >= (uint32_t)r.k : o.bk != kNone, limited = do_k || r.need_p;
    Cut c = {0, kNone};
    auto kept = [&](uint32_t i, uint32_t k) -> double {
        if (limited && (k < c.key || (k == c.key && i > c.last))) return 0.0;
        const float z = z_of(r, k);
        if (bin_at(z) == kBins) return 0.0;
        const double w = (double)weight_at(z);
        return w < r.floor_w ? 0.0 : w;
    };
    if (full) {
        const auto key = [&](uint32_t i) { return key_of(r.x[i]); };
        const auto index = [](uint32_t i) { return i; };
        const auto weighs = [&](uint32_t k) { return bin_at(z_of(r, k)) < kBins; };
        if (r.few && !do_k) {
            double w = 0.0;
            for (uint32_t i = t; i < r.V; i += kT) w += (double)weight_at(z_of(r, key(i)));
            o.all = sum_d(w, D.S);
        }
        c = select_cut(r, r.V, key, index, weighs, weighs, do_k, (uint32_t)r.k, do_k ? 0.0 : o.all, 0.0, D);
        __syncthreads();
        for (uint32_t s = t >> 6; s < a.segs; s += kT / 64) {
            uint32_t k[8];
            load_keys(r, s, k);
            double w = 0.0;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) w += kept(s * kSeg + 8 * (t & 63) + i, k[i]);
            w = last_lane(wave_prefix<Add>(w));
            if ((t & 63) == 0) D.seg[s] = w;
        }
    } else if (n) {
        // listed token j is in the last segment that starts at or before it
        __syncthreads();
        for (uint32_t j = t; j < n; j += kT) {
            uint32_t s = 0;
            for (uint32_t step = kSampleMaxSegs / 2; step; step >>= 1)
                if (s + step < a.segs && D.start[s + step] <= j) s += step;
            const uint32_t i = s * kSeg + a.list[((size_t)row * a.segs + s) * kSampleSegList + (j - D.start[s])];
            D.idx[j] = i;
            D.key[j] = key_of(r.x[i]);
        }
        __syncthreads();
        const auto bin = [&](uint32_t k) { return bin_at(z_of(r, k)); };
        if (n <= kT) {
            c = n <= kT / 4 ? place_cut<4>(r, o, n, do_k, D) : n <= kT / 2 ? place_cut<2>(r, o, n, do_k, D) : place_cut<1>(r, o, n, do_k, D);
        } else {
            const auto key = [&](uint32_t i) { return D.key[i]; };
            const auto index = [&](uint32_t i) { return D.idx[i]; };
            const auto in_k = [&](uint32_t k) { return r.few || bin(k) == o.bk; };
            const auto in_p = [&](uint32_t k) { return bin(k) >= o.g0 && bin(k) <= o.g1; };
            c = select_cut(r, n, key, index, in_k, in_p, do_k, (uint32_t)r.k - o.before_k, do_k ? o.mass_k : o.all, o.mass_0, D);
        }
        for (uint32_t j = t; j < n; j += kT) {
            const double w = kept(D.idx[j], D.key[j]);
            if (w > 0.0) unsafeAtomicAdd(&D.seg[D.idx[j] / kSeg], w);
        }
    }
    __syncthreads();
    // the segment, then the token in it
    double W, own = 0.0;
    for (uint32_t s = g0; s < g1; ++s) own += D.seg[s];
    double ahead = scan_d(own, D.S, W) - own;
    double goal = __builtin_floor((double)(r.u > 0.0f ? r.u : 0.0f) * W);
    goal = goal < W ? goal : W - 1.0;
    for (uint32_t s = g0; s < g1; ++s) {
        const double w = D.seg[s];
        if (ahead <= goal && ahead + w > goal) {
            D.u0 = s;
            D.d0 = ahead;
        }
        ahead += w;
    }
    __syncthreads();
    if (t >= 64) return;
    const uint32_t s = D.u0;
    uint32_t k[8];
    double w[8], mine = 0.0;
    load_keys(r, s, k);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        w[i] = kept(s * kSeg + 8 * t + i, k[i]);
        mine += w[i];
    }
    double cum = D.d0 + wave_prefix<Add>(mine) - mine;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        if (cum <= goal && cum + w[i] > goal) {
            a.tokens[row] = (int32_t)(s * kSeg + 8 * t + i);
            if (a.probs) a.probs[row] = (float)(w[i] / W);
        }
        cum += w[i];
    }
}

} // namespace

hipError_t ah_launch_sample(const SampleArgs &a, hipStream_t stream) {
    const dim3 grid(a.n_rows * a.parts), block(kT);
    hipLaunchKernelGGL(sample_scan_kernel, grid, block, 0, stream, a);
    hipLaunchKernelGGL(sample_count_kernel, grid, block, 0, stream, a);
    hipLaunchKernelGGL(sample_gather_kernel, grid, block, 0, stream, a);
    hipLaunchKernelGGL(sample_draw_kernel, dim3(a.n_rows), block, 0, stream, a);
    return hipGetLastError();
}

// Bytes of scratch, and (with a base) the pointers in it.
size_t ah_sample_plan(SampleArgs &a, uint32_t cus, uint8_t *base) {
    a.segs = (a.n_vocab + kSeg - 1) / kSeg;
    // at most eight workgroups a CU (all that a CU holds: one more would start when the first ends), each of whole
    // rounds of its four waves over one row's segments
    const uint64_t all = (uint64_t)a.n_rows * a.segs, want = 8ull * cus / a.n_rows, parts = want < 1 ? 1 : want;
    a.per = (uint32_t)(((a.segs + parts - 1) / parts + 3) / 4 * 4);
    a.parts = (a.segs + a.per - 1) / a.per;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        uint8_t *p = base ? base + at : nullptr;
        at += (bytes + 255) & ~(size_t)255;
        return p;
    };
    a.bin_mass = reinterpret_cast<double *>(take(8 * (size_t)a.n_rows * kBins));
    a.seg_mass = reinterpret_cast<double *>(take(8 * (size_t)all));
    a.bin_count = reinterpret_cast<uint32_t *>(take(4 * (size_t)a.n_rows * kBins));
    a.group_max = reinterpret_cast<uint32_t *>(take(4 * (size_t)all * kGroups));
    a.seg_max = reinterpret_cast<uint32_t *>(take(4 * (size_t)all));
    a.seg_count = reinterpret_cast<uint32_t *>(take(4 * (size_t)all));
    a.list = reinterpret_cast<uint16_t *>(take(2 * (size_t)all * kSampleSegList));
    return at;
}
