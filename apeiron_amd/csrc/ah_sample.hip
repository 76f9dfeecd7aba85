// ah_sample.hip -- a token from the head's logits and a given random number.
//
// Order the row by (logit descending, index ascending).  With M the largest logit, a token's weight is
// the whole number w = rint(2^32 exp((l - M) / T)); sums of weights are exact in f64 (2^32 times at most
// 2^20 tokens), so no result depends on the order in which they are added.  Kept are the first k tokens
// (top-k), of those the ones whose preceding weight is below p times the weight of all k (top-p), and of
// those the ones with w >= min_p 2^32 (min-p); the first token always.  The draw is the smallest index
// at which the kept weight up to and with it, in index order, passes floor(u W).
//
// No sort.  Four launches over chunks of 2048 tokens, each reading what it needs of the row once:
//   scan    the largest logit of every group of 64 tokens;
//   count   M, and with top-k the bound, a bin of (M - l) / T that the k-th largest group maximum is in: every
//           maximum is a token of its own, so no token past it is among the first k, and only about k groups
//           reach it.  With a small k (and for a greedy row) one workgroup lists their tokens, cuts and draws, and
//           the row is done.  Otherwise the tokens and their weight in 1024 bins, of the groups that reach the
//           bound; the row's workgroup that arrives last finds in them the bins that are kept, those dropped,
//           and the few that a limit falls into;
//   gather  each chunk's certain weight, and a bit for each token in the few bins;
//   draw    one workgroup a row lists those tokens, orders them, cuts, draws a chunk and a token in it (of few rows, in
//           the gather's launch).
// A row whose listed tokens pass the list's room (thousands of equal logits) is cut by selections over
// the whole row instead.
//   What bounds it, of 192 rows of 151936 with mixed parameters, 73 us (117 MB; 25 us by a copy's rate): scan
// 18.6 us from the Infinity Cache and 27 from memory; count and gather 18 and 15 us, the vector work of a weight (an
// exponential, its place among the bins, f64 sums) for each token of the groups that reach the bound, all of them
// without top-k (vector instructions take 41% and 50% of the SIMDs' cycles while a CU works, the waves wait in 56%
// and 60% of theirs); draw 15 us, the chain of loads and barriers of its slowest row (13% and 72%).  Rows of 262144:
// 104 us for 192 (42 by a copy's rate), 17.8 for one.  One row with k = 40: 2.7, 8.9 and
// 2 us, such chains; a launch each costs the host as much.  Bits for the listed tokens, not lists of each chunk's: a
// vocabulary in the order of its logits has all of a bin in a chunk or two (top-p 0.9 of one such row 41 us against
// the 1100 of the selections over the row, of one in any order 34 against 30).
#include "ah_kv4.h"

#include <type_traits>

namespace {

constexpr uint32_t kT = 256, kW = kT / 64;  // threads and waves of every workgroup here
constexpr uint32_t kGroup = 64;             // tokens of a group: eight lanes of eight
constexpr uint32_t kChunk = 2048;           // tokens of a chunk, one wave's in count and gather
constexpr uint32_t kGroups = kChunk / kGroup;
constexpr uint32_t kBins = 1024;
constexpr float kBinScale = kBins / 23.0f;  // w is 0 past (M - l) / T = 22.9
constexpr uint32_t kNone = 0xffffffffu;
// Up to kSmallK tokens asked for, a row's first workgroup counts alone, and draws if the groups that reach the bound
// (as many, and a few in the bound's own bin) and their tokens fit.
constexpr uint32_t kSmallK = 56, kSmallGroups = 64, kSmallList = 1024;

// A logit as an unsigned number of the same order.
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
};
AH_DEV Row row_of(const SampleArgs &a, uint32_t row) {
    Row r;
    r.x = a.logits + (size_t)row * a.stride;
    r.V = a.n_vocab;
    // five loads at once: an absent parameter's reads u instead
    const float *u = a.u + row;
    const float T = *(a.temperature ? a.temperature + row : u), p = *(a.top_p ? a.top_p + row : u), m = *(a.min_p ? a.min_p + row : u);
    const int32_t k = *(a.top_k ? a.top_k + row : reinterpret_cast<const int32_t *>(u));
    r.u = *u;
    r.T = a.temperature ? T : 1.0f;
    r.k = a.top_k ? k : 0;
    r.p = a.top_p ? p : 1.0f;
    r.m = a.min_p ? m : 0.0f;
    r.bad_t = !(r.T >= 0.0f && r.T < __builtin_inff());
    r.greedy = r.bad_t || r.T == 0.0f || r.k == 1;
    r.need_k = !r.greedy && r.k > 1 && (uint32_t)r.k < r.V;
    r.need_p = !r.greedy && r.p < 1.0f;
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
// A logit's z = (l - M) / T, from the logit itself (NaN stays one: no bin and no weight) or its key (0 past the
// row's end).
AH_DEV float z_at(const Row &r, float l) {
#pragma clang fp contract(off)
    return l == r.M ? 0.0f : (l - r.M) * r.inv_t;
}
AH_DEV float z_of(const Row &r, uint32_t k) { return k ? z_at(r, logit_of(k)) : -__builtin_inff(); }
// The weight: a whole number, as f32 (exact: exp's 24 bits, rounded below 1).  exp(z) = 2^(z log2 e), the
// product's own rounding carried as a factor next to 1: about 1.5 units of f32's last place.
AH_DEV float weight_at(float z) {
#pragma clang fp contract(off)
    const float l2e = 0x1.715476p+0f, rest = 0x1.4ae0cp-26f, ln2 = 0x1.62e43p-1f;  // log2 e = l2e + rest
    z = __builtin_fmaxf(z, -28.0f);  // (the weight is 0 there; z may be -inf or NaN)
    const float t = z * l2e, d = __builtin_fmaf(z, rest, __builtin_fmaf(z, l2e, -t)), e = __builtin_amdgcn_exp2f(t);
    return __builtin_rintf(__builtin_fmaf(e, d * ln2, e) * 0x1p32f);
}
// The place of z among the bins, and its bin: kBins where the weight is 0.
AH_DEV float place_at(float z) { return z * -kBinScale; }
AH_DEV uint32_t bin_at(float z) { return (uint32_t)__builtin_fminf(place_at(z), (float)kBins); }

// ---- workgroup scans (kT threads) -------------------------------------------------------------------

// v of another lane through DPP (no LDS); lanes without a source, and rows outside ROWS, get 0.
template <int CTRL, int ROWS> AH_DEV uint32_t dpp0(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS> AH_DEV uint64_t dpp0(uint64_t v) {
    return (uint64_t)dpp0<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | dpp0<CTRL, ROWS>((uint32_t)v);
}
template <int CTRL, int ROWS> AH_DEV double dpp0(double v) {
    return __builtin_bit_cast(double, dpp0<CTRL, ROWS>(__builtin_bit_cast(uint64_t, v)));
}
struct Add {
    template <class T> AH_DEV T operator()(T a, T b) const { return a + b; }
};
struct Max {
    template <class T> AH_DEV T operator()(T a, T b) const { return a > b ? a : b; }
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

// Eight logits of the row (-inf past its end), and their keys (0, below every key, there).
AH_DEV void load_logits(const Row &r, uint32_t i0, float *x) {
    if (i0 + 8 <= r.V) __builtin_memcpy(x, r.x + i0, 32);
    else
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) x[i] = i0 + i < r.V ? r.x[i0 + i] : -__builtin_inff();
}
AH_DEV void keys_of(const Row &r, uint32_t i0, const float *x, uint32_t *k) {
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) k[i] = i0 + i < r.V ? key_of(x[i]) : 0u;
}
AH_DEV void load_keys(const Row &r, uint32_t i0, uint32_t *k) {
    float x[8];
    load_logits(r, i0, x);
    keys_of(r, i0, x, k);
}

// What one workgroup writes and another reads in the same launch goes past the XCDs' own L2s.
template <class T> AH_DEV void put(T *p, T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <class T> AH_DEV T get(const T *p) { return __hip_atomic_load(const_cast<T *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The workgroup's row and its chunks, with `parts` workgroups a row of `per` chunks each.
AH_DEV void share(const SampleArgs &a, uint32_t parts, uint32_t per, uint32_t &row, uint32_t &c0, uint32_t &c1) {
    row = blockIdx.x / parts;
    c0 = (blockIdx.x - row * parts) * per;
    c1 = c0 + per < a.chunks ? c0 + per : a.chunks;
}
// Whether this workgroup is the row's last in the launch: it then finds what the others have put.  The counters
// are left at zero.
AH_DEV bool last_of_row(const SampleArgs &a, uint32_t row, uint32_t &word) {
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t n = __hip_atomic_fetch_add(a.arrived + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (n == a.parts - 1) put(a.arrived + row, 0u);
        word = n;
    }
    __syncthreads();
    return word == a.parts - 1;
}

// ---- the cut ----------------------------------------------------------------------------------------

// The list of tokens (in index order) that a cut is looked for in, and what the search needs.
template <uint32_t LIST> struct CutLds {
    alignas(16) double mass[kT];
    uint32_t count[kT];
    alignas(16) uint32_t key[LIST], idx[LIST];
    alignas(16) uint32_t near_key[kT];
    uint32_t near_idx[kT];
    Scan S;
    uint32_t u0, u1;
    double d0;
};

// What the bins say.  Tokens of bins below g0 are kept and those of bins past g1 dropped (min-p apart); the
// k-th token is in bin bk (kNone: fewer than k tokens have weight), `before_k` tokens weighing `mass_k` ahead of
// that bin; `mass_0` is the weight ahead of bin g0 and `all` that of every bin.
typedef SampleLimits Limits;

// The kept set's last token in the order: keys above `key` are kept, and of those equal to it the ones up
// to index `last`.
struct Cut {
    uint32_t key, last;
};

// The index of the nth (1 ..) of n tokens that have key `cut`.
template <class Key, class Lds> AH_DEV uint32_t nth_equal(uint32_t n, Key key, uint32_t cut, uint32_t nth, Lds &D) {
    uint32_t seen = 0;
    for (uint32_t base = 0; base < n && seen < nth; base += kT) {
        const uint32_t i = base + threadIdx.x;
        const bool eq = i < n && key(i) == cut;
        uint32_t total;
        const uint32_t at = seen + scan_u(eq, D.S, total);
        if (eq && at == nth) D.u0 = i;
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

// The cut over the whole row, by digits of the keys.  do_k: top-k falls into the tokens that have weight; all_weight: theirs.
template <class Lds> AH_DEV Cut select_cut(const Row &r, bool do_k, double all_weight, Lds &D) {
    const uint32_t n = r.V;
    const auto key = [&](uint32_t i) { return key_of(r.x[i]); };
    const auto weighs = [&](uint32_t k) { return bin_at(z_of(r, k)) < kBins; };
    uint32_t need = (uint32_t)r.k;
    double before = 0.0;
    const uint32_t t = threadIdx.x;
    Cut c = {0, kNone};
    uint32_t keep = 0, cut_k = 0;  // of those at the cut
    bool partial = false;
    if (do_k) {
        uint32_t lo = kNone, hi = 0;
#pragma unroll 1
        for (uint32_t i = t; i < n; i += kT) {
            const uint32_t k = key(i);
            if (weighs(k)) {
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
#pragma unroll 1
            for (uint32_t i = t; i < n; i += kT) {
                const uint32_t k = key(i);
                if (weighs(k) && (shift == 24 || (k >> (shift + 8)) == (cut_k >> (shift + 8)))) atomicAdd(&D.count[(k >> shift) & 255u], 1u);
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
        double W = do_k ? 0.0 : all_weight;
        if (do_k) {
            double s = 0.0;
#pragma unroll 1
            for (uint32_t i = t; i < n; i += kT) {
                const uint32_t k = key(i);
                if (weighs(k) && k > cut_k) s += (double)weight_at(z_of(r, k));
            }
            W += sum_d(s, D.S) + (double)keep * w_cut;
        }
        double goal = (double)(r.p > 0.0f ? r.p : 0.0f) * W;
        goal = goal < 1.0 ? 1.0 : goal;  // the first token always
        uint32_t cut_p = 0, all = 0, lo = do_k && weighs(cut_k) ? cut_k : kNone, hi = lo == kNone ? 0u : cut_k;
#pragma unroll 1
        for (uint32_t i = t; i < n; i += kT) {
            const uint32_t k = key(i);
            if (weighs(k) && !(do_k && k <= cut_k)) {
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
#pragma unroll 1
            for (uint32_t i = t; i < n; i += kT) {
                const uint32_t k = key(i);
                if (!weighs(k) || (do_k && k <= cut_k) || !(shift == 24 || (k >> (shift + 8)) == (cut_p >> (shift + 8)))) continue;
                unsafeAtomicAdd(&D.mass[(k >> shift) & 255u], (double)weight_at(z_of(r, k)));
                atomicAdd(&D.count[(k >> shift) & 255u], 1u);
            }
            __syncthreads();
            double mine = D.mass[255 - t];
            uint32_t cnt = D.count[255 - t];
            if (do_k && weighs(cut_k) && (shift == 24 || (cut_k >> (shift + 8)) == (cut_p >> (shift + 8))) && 255 - t == ((cut_k >> shift) & 255u)) {
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
    if (partial) c.last = nth_equal(n, key, c.key, keep, D);
    return c;
}

// The cut of the list's n tokens in two stages, the first k's and top-p's.  The limit of a stage is where the running
// sum (of ones, of weights) in the order reaches its goal; of more than kFew tokens, those of the one of 256 equal
// parts of the limit's bins in which it does are taken out first, and among what is left four neighbouring threads find
// the sum ahead of a token by comparing with all.  whole: the list is every token that can be among the first k.
// False: more than kT tokens in such a part.
constexpr uint32_t kFew = kT / 4;
template <class Lds> AH_DEV bool cut_list(const Row &r, const Limits &o, uint32_t n, bool do_k, bool whole, Cut &c, Lds &D) {
    const uint32_t t = threadIdx.x, each = (n + kT - 1) / kT, j0 = t * each, j1 = j0 + each < n ? j0 + each : n;
    c = {0, kNone};
#pragma unroll 1
    // (a list of just the first k needs no cut)
    for (uint32_t stage = do_k && !(whole && n == (uint32_t)r.k) ? 0 : 1; stage < (r.need_p ? 2u : 1u); ++stage) {
        const bool p = stage == 1;
        const float k_from = whole ? 0.0f : (float)o.bk, k_to = whole ? (float)(o.g1 + 1) : (float)(o.bk + 1);
        float from = k_from, to = k_to;
        // tokens that count: at places between the two, and up to the cut so far
        const auto in = [&](uint32_t j) {
            const uint32_t k = D.key[j];
            const float y = place_at(z_of(r, k));
            return (y >= from) & (y < to) & ((k > c.key) | ((k == c.key) & (D.idx[j] <= c.last)));
        };
        const auto value = [&](uint32_t j) { return p ? (double)weight_at(z_of(r, D.key[j])) : 1.0; };
        double goal = (double)((uint32_t)r.k - o.before_k), before = 0.0;
        if (p) {
            double W = o.all;
            if (do_k || whole) {
                double w = 0.0;
#pragma unroll 1
                for (uint32_t j = t; j < n; j += kT) w += in(j) ? value(j) : 0.0;
                W = o.mass_k + sum_d(w, D.S);
            }
            goal = (double)(r.p > 0.0f ? r.p : 0.0f) * W;
            goal = goal < 1.0 ? 1.0 : goal;  // the first token always
            before = o.mass_0;
            from = (float)o.g0;
            to = (float)(o.g1 + 1);
        }
        const float scale = (float)kT / (to - from);
        const auto part = [&](uint32_t j) { return n <= kFew ? 0u : (uint32_t)__builtin_fminf((place_at(z_of(r, D.key[j])) - from) * scale, (float)(kT - 1)); };
        uint32_t the = 0;
        if (n > kFew) {
            D.mass[t] = 0.0;
            if (t == 0) D.u0 = 0;
            __syncthreads();
#pragma unroll 1
            for (uint32_t j = t; j < n; j += kT)
                if (in(j)) unsafeAtomicAdd(&D.mass[part(j)], value(j));
            __syncthreads();
            const double mine = D.mass[t];
            double total;
            const double sum = before + scan_d(mine, D.S, total);
            if (sum >= goal && sum - mine < goal) {
                D.u0 = t;
                D.d0 = sum - mine;
            }
            __syncthreads();
            the = D.u0;
            before = D.d0;
        }
        D.near_key[t] = 0;
        D.mass[t] = 0.0;
        uint32_t count = 0, m;
#pragma unroll 1
        for (uint32_t j = j0; j < j1; ++j) count += in(j) && part(j) == the ? 1u : 0u;
        uint32_t at = scan_u(count, D.S, m) - count;
        if (m > kT) return false;
#pragma unroll 1
        for (uint32_t j = j0; j < j1; ++j)
            if (in(j) && part(j) == the) {
                D.near_key[at] = D.key[j];
                D.near_idx[at] = D.idx[j];
                D.mass[at++] = value(j);
            }
        __syncthreads();
        const double ahead = before;
#pragma unroll 1
        for (uint32_t me = t / 4; me < m; me += kFew) {
            const uint32_t k = D.near_key[me], idx = D.near_idx[me];
            const double mine = D.mass[me];
            before = 0.0;
#pragma unroll 2
            for (uint32_t j = 4 * (t & 3); j < m; j += 16) {  // (past the m tokens: key 0, below every key)
                uint32_t other[4];
                double w[4];
                __builtin_memcpy(other, D.near_key + j, 16);
                __builtin_memcpy(w, D.mass + j, 32);
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) w[i] = other[i] > (j + i < me ? k - 1 : k) ? w[i] : 0.0;
                before += (w[0] + w[1]) + (w[2] + w[3]);
            }
            before += dpp0<0xB1, 0xF>(before);  // the other three of the quad
            before += dpp0<0x4E, 0xF>(before);
            before += ahead;
            if (before < goal && before + mine >= goal) {
                D.u0 = k;
                D.u1 = idx;
            }
        }
        __syncthreads();
        c = {D.u0, D.u1};
    }
    return true;
}

// A token's weight if it is kept: under a limit, up to the cut.
AH_DEV double kept_weight(const Row &r, const Cut &c, bool limited, uint32_t i, uint32_t k) {
    if (limited && (k < c.key || (k == c.key && i > c.last))) return 0.0;
    const float z = z_of(r, k);
    if (bin_at(z) == kBins) return 0.0;
    const double w = (double)weight_at(z);
    return w < r.floor_w ? 0.0 : w;
}
AH_DEV double goal_of(const Row &r, double W) {
    const double goal = __builtin_floor((double)(r.u > 0.0f ? r.u : 0.0f) * W);
    return goal < W ? goal : W - 1.0;
}

// ---- scan -------------------------------------------------------------------------------------------

__global__ void __launch_bounds__(kT) sample_scan_kernel(SampleArgs a) {
    uint32_t row, c0, c1;
    share(a, a.scan_parts, a.scan_per, row, c0, c1);
    Row r;
    r.x = a.logits + (size_t)row * a.stride;
    r.V = a.n_vocab;
    const uint32_t t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
    if (c0 == 0) {  // the row's bins, for the next launch
        for (uint32_t i = t; i < kBins; i += kT) {
            a.bin_mass[(size_t)row * kBins + i] = 0.0;
            a.bin_count[(size_t)row * kBins + i] = 0;
        }
    }
    // a wave takes 512 tokens at a time
    const uint32_t end = c1 * kChunk < r.V ? c1 * kChunk : r.V;
    bool nan = false;
    for (uint32_t base = c0 * kChunk + wave * 512; base < end; base += kW * 512) {
        const uint32_t i0 = base + 8 * lane, group = i0 / kGroup;
        float x[8], top = -__builtin_inff();  // (a NaN is passed over)
        load_logits(r, i0, x);
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            nan |= x[i] != x[i];
            top = __builtin_fmaxf(top, x[i]);
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o, 64));
        if ((lane & 7) == 0 && group < a.groups) a.group_max[(size_t)row * a.groups + group] = top;
    }
    if (nan) ah_record(a.status, ((unsigned long long)row << 8) + AH_ERR_NONFINITE_INPUT);
}

// ---- count ------------------------------------------------------------------------------------------

struct LimitsLds {
    uint32_t bk, before_k, g0, g1;
    double mass_k, mass_0, w_high;
};
struct CountLds {
    union {
        double mass[kBins];
        CutLds<kSmallList> cut;  // (of a row that is finished at once)
    };
    alignas(16) uint32_t count[kBins], near[kSmallGroups], group[kSmallGroups];
    Scan S;
    LimitsLds L;
    uint32_t found, reach, word;
};

// A row's group maxima, every kT-th in a thread, the first kHeld of them in registers.
struct GroupMaxima {
    static constexpr uint32_t kHeld = 10;
    const float *g;
    uint32_t n;
    float held[kHeld];
    AH_DEV GroupMaxima(const SampleArgs &a, uint32_t row) {
        g = a.group_max + (size_t)row * a.groups;
        n = a.groups;
#pragma unroll
        for (uint32_t i = 0; i < kHeld; ++i) held[i] = i * kT + threadIdx.x < n ? g[i * kT + threadIdx.x] : -__builtin_inff();
    }
    // f(maximum) of each (-inf without one); g(group) of those for which f holds
    template <class F> AH_DEV void each(F f) const {
#pragma unroll
        for (uint32_t i = 0; i < kHeld; ++i) f(held[i]);
#pragma unroll 1
        for (uint32_t j = kHeld * kT + threadIdx.x; j < n; j += kT) f(g[j]);
    }
    template <class F, class H> AH_DEV void those(F f, H h) const {
        uint32_t mask = 0;
#pragma unroll
        for (uint32_t i = 0; i < kHeld; ++i) mask |= f(held[i]) ? 1u << i : 0u;
#pragma unroll 1
        for (; mask; mask &= mask - 1) h((uint32_t)__builtin_ctz(mask) * kT + threadIdx.x);
#pragma unroll 1
        for (uint32_t j = kHeld * kT + threadIdx.x; j < n; j += kT)
            if (f(g[j])) h(j);
    }
};

// The bin that the k-th largest group maximum is in (the last one if fewer have weight), and how many groups reach it.
AH_DEV uint32_t bound_of(const Row &r, const GroupMaxima &G, CountLds &D) {
    const uint32_t t = threadIdx.x;
    for (uint32_t i = t; i < kBins; i += kT) D.count[i] = 0;
    if (t < kSmallGroups) D.near[t] = kNone;
    if (t == 0) {
        D.found = kBins - 1;
        D.reach = kNone;
        D.word = 0;
    }
    __syncthreads();
    G.each([&](float x) {
        const uint32_t b = bin_at(z_at(r, x));
        if (b < kBins) atomicAdd(&D.count[b], 1u);
    });
    __syncthreads();
    uint32_t c[4], total;
    __builtin_memcpy(c, D.count + 4 * t, 16);
    const uint32_t mine = (c[0] + c[1]) + (c[2] + c[3]);
    uint32_t cum = scan_u(mine, D.S, total) - mine;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (cum < (uint32_t)r.k && cum + c[i] >= (uint32_t)r.k) {
            D.found = 4 * t + i;
            D.reach = cum + c[i];
        }
        cum += c[i];
    }
    __syncthreads();
    return D.reach == kNone ? total : D.reach;
}

// A row whose first k tokens are all in `reach` groups (at most kSmallGroups): lists the tokens in bins up to `last`,
// cuts them and draws.  False if they are more than the list holds.
AH_DEV bool finish_small(const SampleArgs &a, const Row &r, uint32_t row, const GroupMaxima &G, uint32_t reach, uint32_t last, CountLds &D) {
    const uint32_t t = threadIdx.x, sub = 8 * (t & 7);
    CutLds<kSmallList> &C = D.cut;
    uint32_t total;
    const float end = (float)(last + 1);
    G.those([&](float m) { return place_at(z_at(r, m)) < end; }, [&](uint32_t g) { D.near[atomicAdd(&D.word, 1u)] = g; });
    __syncthreads();
    if (t < reach) {  // in their order
        const uint32_t mine = D.near[t];
        uint32_t rank = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < kSmallGroups; j += 4) {
            uint32_t other[4];
            __builtin_memcpy(other, D.near + j, 16);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) rank += other[i] < mine ? 1u : 0u;
        }
        D.group[rank] = mine;
    }
    __syncthreads();
    // 32 groups a round, eight threads each
    constexpr uint32_t kRounds = kSmallGroups * 8 / kT;
    float x[kRounds][8];
    uint32_t i0[kRounds], mask[kRounds], packed = 0;
#pragma unroll
    for (uint32_t q = 0; q < kRounds; ++q) {
        const uint32_t g = q * (kT / 8) + t / 8;
        i0[q] = g < reach ? D.group[g] * kGroup + sub : r.V;
        load_logits(r, i0[q], x[q]);
    }
#pragma unroll
    for (uint32_t q = 0; q < kRounds; ++q) {
        mask[q] = 0;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) mask[q] |= place_at(z_at(r, x[q][i])) < end ? 1u << i : 0u;
        packed += (uint32_t)__builtin_popcount(mask[q]) << (16 * q);
    }
    static_assert(kRounds == 2, "two rounds' counts in one word");
    const uint32_t before = scan_u(packed, D.S, total) - packed, n = (total & 0xffffu) + (total >> 16);
    if (n > kSmallList) return false;
    uint32_t to = before & 0xffffu;
#pragma unroll
    for (uint32_t q = 0; q < kRounds; ++q) {
#pragma unroll 1
        for (; mask[q]; mask[q] &= mask[q] - 1) {
            const uint32_t i = i0[q] + (uint32_t)__builtin_ctz(mask[q]);
            C.key[to] = key_of(r.x[i]);
            C.idx[to++] = i;
        }
        to = (total & 0xffffu) + (before >> 16);
    }
    __syncthreads();
    const Limits o = {0, last, kNone, 0, 0.0, 0.0, 0.0, r.top, last, 0};
    const bool do_k = n >= (uint32_t)r.k;  // (fewer are all that have weight)
    Cut c;
    if (!cut_list(r, o, n, do_k, true, c, C)) return false;
    // the draw, in the list's order
    const uint32_t each = (n + kT - 1) / kT, j0 = t * each, j1 = j0 + each < n ? j0 + each : n;
    const auto weight = [&](uint32_t j) { return kept_weight(r, c, do_k || r.need_p, C.idx[j], C.key[j]); };
    double own = 0.0, W;
#pragma unroll 1
    for (uint32_t j = j0; j < j1; ++j) own += weight(j);
    double ahead = scan_d(own, C.S, W) - own;
    const double goal = goal_of(r, W);
    if (ahead <= goal && ahead + own > goal) {
#pragma unroll 1
        for (uint32_t j = j0; j < j1; ++j) {
            const double w = weight(j);
            if (ahead <= goal && ahead + w > goal) {
                a.tokens[row] = (int32_t)C.idx[j];
                if (a.probs) a.probs[row] = (float)(w / W);
            }
            ahead += w;
        }
    }
    return true;
}

// Calls f(place of a lane's first token in the chunk, its logits, whether there is one) over those groups of a chunk
// whose largest token's bin is at most `last`, in their order: eight groups a round, eight lanes each, the next round's
// logits on their way meanwhile.  skipped(group) for each of the chunk's others, past the row's end too.
template <class F, class G>
AH_DEV void each_group(const SampleArgs &a, const Row &r, uint32_t row, uint32_t chunk, uint32_t last, F f, G skipped) {
    const uint32_t lane = threadIdx.x & 63, g = chunk * kGroups + lane;
    const bool in = lane < kGroups && g < a.groups, use = in && bin_at(z_at(r, a.group_max[(size_t)row * a.groups + (in ? g : 0)])) <= last;
    const uint64_t todo = __builtin_amdgcn_ballot_w64(use);
    const uint32_t n = (uint32_t)__builtin_popcountll(todo);
    if (lane < kGroups && !use) skipped(lane);
    if (n == 0) return;
    // lane j: the j-th of the groups
    const uint32_t rank = __builtin_amdgcn_mbcnt_lo((uint32_t)todo, 0u);
    const int list = __builtin_amdgcn_ds_permute((int)(4 * (use ? rank : 63u)), (int)lane);
    float x[8], next[8];
    uint32_t at, at_next;
    auto load = [&](uint32_t j) {
        const uint32_t mine = j + (lane >> 3);
        at_next = (uint32_t)__builtin_amdgcn_ds_bpermute((int)(4 * (mine & 31)), list) * kGroup + 8 * (lane & 7);
        load_logits(r, mine < n ? chunk * kChunk + at_next : r.V, next);
    };
    load(0);
    for (uint32_t j = 0; j < n; j += 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = next[i];
        at = at_next;
        if (j + 8 < n) load(j + 8);
        f(at, x, j + (lane >> 3) < n);
    }
}

// The limits from a row's bins, four of them (c, m) in each thread.
AH_DEV Limits limits_of(const Row &r, const uint32_t *c, const double *m, Scan &S, LimitsLds &L) {
    Limits o = {kBins, kBins, kNone, 0, 0.0, 0.0, 0.0, 0, 0, 0};
    const uint32_t t = threadIdx.x;
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

__global__ void __launch_bounds__(kT, 8) sample_count_kernel(SampleArgs a) {
    __shared__ CountLds D;
    uint32_t row, c0, c1;
    share(a, a.parts, a.per, row, c0, c1);
    const GroupMaxima G(a, row);  // (on their way before anything is waited for)
    Row r = row_of(a, row);
    const uint32_t t = threadIdx.x;
    bool counts = r.need_k || r.need_p;
    const bool alone = !counts || a.parts == 1 || (r.need_k && (uint32_t)r.k <= kSmallK);
    if (alone && c0 != 0) return;
    float top = -__builtin_inff();
    G.each([&](float m) { top = __builtin_fmaxf(top, m); });
    set_top(r, max_u(key_of(top), D.S));
    Limits o = {kBins, kBins, kNone, 0, 0.0, 0.0, 0.0, r.top, kBins - 1, 0};
    if (r.greedy || r.M == -__builtin_inff()) {
        if (c0 != 0) return;
        const unsigned long long key0 = (unsigned long long)row << 8;
        if (t == 0 && r.bad_t) ah_record(a.status, key0 + AH_ERR_INPUT_RANGE);
        if (r.M == -__builtin_inff()) {  // nothing to draw
            if (t == 0) {
                ah_record(a.status, key0 + AH_ERR_NONFINITE_INPUT);
                a.tokens[row] = -1;
                if (a.probs) a.probs[row] = 0.0f;
            }
        } else {  // the first group that holds the largest, and in it the first token
            uint32_t at = kNone;
            G.those([&](float m) { return m == r.M; }, [&](uint32_t g) { at = __builtin_elementwise_min(at, g); });
            at = min_u(at, D.S);
            const uint32_t i = at * kGroup + (t & 63);
            const uint64_t b = __builtin_amdgcn_ballot_w64(i < r.V && key_of(r.x[i < r.V ? i : 0]) == r.top);
            if (t == 0) {
                a.tokens[row] = (int32_t)(at * kGroup + (uint32_t)__builtin_ctzll(b));
                if (a.probs) a.probs[row] = 1.0f;
            }
        }
        o.done = 1;
        counts = false;
    } else if (r.need_k) {
        const uint32_t reach = bound_of(r, G, D);
        o.last = D.found;
        if (alone && reach <= kSmallGroups) {
            o.done = finish_small(a, r, row, G, reach, o.last, D);
            counts = !o.done;
        }
    }
    if (!counts) {
        if (t == 0) a.limits[row] = o;
        return;
    }
    const uint32_t last = o.last;
    if (alone) c1 = a.chunks;
    __syncthreads();
    for (uint32_t i = t; i < kBins; i += kT) {
        D.count[i] = 0;
        D.mass[i] = 0.0;
    }
    __syncthreads();
    for (uint32_t c = c0 + __builtin_amdgcn_readfirstlane(t >> 6); c < c1; c += kW)
        each_group(
            a, r, row, c, last,
            [&](uint32_t, const float *x, bool) {  // (-inf in a lane without a group: no bin)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float z = z_at(r, x[i]);
                    const uint32_t b = bin_at(z);
                    if (b > last) continue;
                    if (r.need_k) atomicAdd(&D.count[b], 1u);
                    if (r.need_p) unsafeAtomicAdd(&D.mass[b], (double)weight_at(z));
                }
            },
            [](uint32_t) {});
    __syncthreads();
    uint32_t n[4];
    double m[4];
    if (alone) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            n[i] = D.count[4 * t + i];
            m[i] = D.mass[4 * t + i];
        }
    } else {
        uint32_t *bc = a.bin_count + (size_t)row * kBins;
        double *bm = a.bin_mass + (size_t)row * kBins;
        for (uint32_t i = t; i <= last; i += kT) {
            if (D.count[i]) atomicAdd(bc + i, D.count[i]);
            if (D.mass[i] > 0.0) unsafeAtomicAdd(bm + i, D.mass[i]);
        }
        if (!last_of_row(a, row, D.word)) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            n[i] = get(bc + 4 * t + i);
            m[i] = get(bm + 4 * t + i);
        }
    }
    o = limits_of(r, n, m, D.S, D.L);
    o.top = r.top;
    // the last bin with a token to keep or to list (no bin: tokens without weight, as a whole)
    const uint32_t end_k = o.bk != kNone ? o.bk : o.g1;
    o.last = o.g0 == kBins ? kBins - 1 : end_k > o.g1 ? end_k : o.g1;
    if (t == 0) a.limits[row] = o;
}

// ---- draw -------------------------------------------------------------------------------------------

struct DrawLds {
    CutLds<kSampleList> cut;
    double mass[kSampleMaxChunks];
};

// SAME: in the launch that gathered.
template <bool SAME, class T> AH_DEV T gathered(const T *p) { return SAME ? get(p) : *p; }

template <bool SAME> AH_DEV void draw(const SampleArgs &a, uint32_t row, const Limits &o, DrawLds &D) {
    CutLds<kSampleList> &C = D.cut;
    const uint32_t t = threadIdx.x;
    // this thread's chunks' certain weights, and its words of the listed tokens' bits
    const uint32_t each = (a.chunks + kT - 1) / kT, g0 = t * each < a.chunks ? t * each : a.chunks, g1 = g0 + each < a.chunks ? g0 + each : a.chunks;
    for (uint32_t s = g0; s < g1; ++s) D.mass[s] = gathered<SAME>(&a.chunk_mass[(size_t)row * a.chunks + s]);
    const uint32_t words = a.chunks * (kChunk / 32), own_words = (words + kT - 1) / kT, w0 = t * own_words, w1 = w0 + own_words < words ? w0 + own_words : words;
    const uint32_t *bits = a.bits + (size_t)row * words;
    constexpr uint32_t kHeld = 20;  // (a row of 163840 tokens), the rest read twice
    uint32_t n_mine = 0, n, held[kHeld];
#pragma unroll
    for (uint32_t i = 0; i < kHeld; ++i) held[i] = w0 + i < w1 ? gathered<SAME>(&bits[w0 + i]) : 0u;
#pragma unroll
    for (uint32_t i = 0; i < kHeld; ++i) n_mine += (uint32_t)__builtin_popcount(held[i]);
    for (uint32_t w = w0 + kHeld; w < w1; ++w) n_mine += (uint32_t)__builtin_popcount(gathered<SAME>(&bits[w]));
    Row r = row_of(a, row);
    set_top(r, o.top);
    uint32_t at = scan_u(n_mine, C.S, n) - n_mine;
    bool full = n > kSampleList;
    if (!full && n_mine) {
        const auto list = [&](uint32_t w, uint32_t b) {
#pragma unroll 1
            for (; b; b &= b - 1) C.idx[at++] = w * 32 + (uint32_t)__builtin_ctz(b);
        };
#pragma unroll
        for (uint32_t i = 0; i < kHeld; ++i) list(w0 + i, held[i]);
        for (uint32_t w = w0 + kHeld; w < w1; ++w) list(w, gathered<SAME>(&bits[w]));
    }
    const bool do_k = o.bk != kNone, limited = do_k || r.need_p;
    Cut c = {0, kNone};
    if (!full && n) {
        __syncthreads();
#pragma unroll 4
        for (uint32_t j = t; j < n; j += kT) C.key[j] = key_of(r.x[C.idx[j]]);
        __syncthreads();
        full = !cut_list(r, o, n, do_k, false, c, C);
#pragma unroll 1
        for (uint32_t j = t; j < n && !full; j += kT) {
            const double w = kept_weight(r, c, limited, C.idx[j], C.key[j]);
            if (w > 0.0) unsafeAtomicAdd(&D.mass[C.idx[j] / kChunk], w);
        }
    }
    if (full) {  // too many equal, or nearly equal: over the whole row
        __syncthreads();
        c = select_cut(r, do_k, o.all, C);
        __syncthreads();
#pragma unroll 1
        for (uint32_t s = t >> 6; s < a.chunks; s += kW) {
            double w = 0.0;
#pragma unroll 1
            for (uint32_t i = s * kChunk + (t & 63), q = 0; q < kChunk / 64; ++q, i += 64)
                if (i < r.V) w += kept_weight(r, c, limited, i, key_of(r.x[i]));
            w = last_lane(wave_prefix<Add>(w));
            if ((t & 63) == 0) D.mass[s] = w;
        }
    }
    __syncthreads();
    // the chunk, then the token in it
    if (t == 0) C.u0 = 0;
    double W, own = 0.0;
    for (uint32_t s = g0; s < g1; ++s) own += D.mass[s];
    double ahead = scan_d(own, C.S, W) - own;
    const double goal = goal_of(r, W);
    for (uint32_t s = g0; s < g1; ++s) {
        const double w = D.mass[s];
        if (ahead <= goal && ahead + w > goal) {
            C.u0 = s;
            C.d0 = ahead;
        }
        ahead += w;
    }
    __syncthreads();
    const uint32_t i0 = C.u0 * kChunk + 8 * t;
    uint32_t k[8];
    load_keys(r, i0, k);
    __builtin_memcpy(C.key + 8 * t, k, 32);  // (its own alone)
    double mine = 0.0, total;
#pragma unroll 1
    for (uint32_t i = 0; i < 8; ++i) mine += kept_weight(r, c, limited, i0 + i, C.key[8 * t + i]);
    double cum = C.d0 + scan_d(mine, C.S, total) - mine;
    if (cum <= goal && cum + mine > goal) {
#pragma unroll 1
        for (uint32_t i = 0; i < 8; ++i) {
            const double w = kept_weight(r, c, limited, i0 + i, C.key[8 * t + i]);
            if (cum <= goal && cum + w > goal) {
                a.tokens[row] = (int32_t)(i0 + i);
                if (a.probs) a.probs[row] = (float)(w / W);
            }
            cum += w;
        }
    }
}

__global__ void __launch_bounds__(kT) sample_draw_kernel(SampleArgs a) {
    __shared__ DrawLds D;
    const Limits o = a.limits[blockIdx.x];
    if (!o.done) draw<false>(a, blockIdx.x, o, D);
}

// ---- gather -----------------------------------------------------------------------------------------

// DRAW: with the draw, by the row's workgroup that arrives last.
template <bool DRAW> __global__ void __launch_bounds__(kT) sample_gather_kernel(SampleArgs a) {
    __shared__ typename std::conditional<DRAW, DrawLds, char>::type D;
    uint32_t row, c0, c1;
    share(a, a.parts, a.per, row, c0, c1);
    const Limits o = a.limits[row];
    if (o.done) return;
    Row r = row_of(a, row);
    set_top(r, o.top);
    const uint32_t lane = threadIdx.x & 63;
    // places among the bins: kept below `sure_to`, listed from `from` up to `to` and, where top-p needs the weight of
    // the first k, in bin bk.  (No branches over the tokens: a wave takes both sides nearly always.)
    const float sure_to = (float)o.g0, from = (float)o.g0, to = (float)((o.g1 < kBins ? o.g1 : kBins - 1) + 1);
    const bool also = r.need_p && o.bk != kNone;
    const float also_from = (float)o.bk, also_to = (float)(o.bk + 1);
    for (uint32_t c = c0 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); c < c1; c += kW) {
        const size_t chunk = (size_t)row * a.chunks + c;
        uint8_t *bits = reinterpret_cast<uint8_t *>(a.bits) + chunk * (kChunk / 8);
        double sure = 0.0;
        each_group(
            a, r, row, c, o.last,
            [&](uint32_t at, const float *x, bool live) {
                uint32_t mask = 0;
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    const float z = z_at(r, x[i]), y = place_at(z), w = weight_at(z);
                    sure += (double)(((y < sure_to) & (w >= r.floor_f)) ? w : 0.0f);
                    mask |= ((y >= from) & (y < to)) ? 1u << i : 0u;
                    if (also) mask |= ((y >= also_from) & (y < also_to)) ? 1u << i : 0u;
                }
                if (live) {
                    if (DRAW) put(bits + at / 8, (uint8_t)mask);
                    else bits[at / 8] = (uint8_t)mask;
                }
            },
            [&](uint32_t g) {
                if (DRAW) put(reinterpret_cast<uint64_t *>(bits) + g, (uint64_t)0);
                else reinterpret_cast<uint64_t *>(bits)[g] = 0;
            });
        if (__builtin_amdgcn_ballot_w64(sure > 0.0) != 0ull) sure = last_lane(wave_prefix<Add>(sure));
        if (lane == 0) {
            if (DRAW) put(a.chunk_mass + chunk, sure);
            else a.chunk_mass[chunk] = sure;
        }
    }
    if constexpr (DRAW) {
        if (a.parts > 1 && !last_of_row(a, row, D.cut.u1)) return;
        __syncthreads();
        draw<true>(a, row, o, D);
    }
}

static_assert(kChunk == 8 * kT, "the draw takes a chunk at once");
static_assert(kSampleMaxChunks * kChunk >= 1u << 20, "the longest row");

} // namespace

hipError_t ah_launch_sample(const SampleArgs &a, hipStream_t stream) {
    const dim3 grid(a.n_rows * a.parts), block(kT);
    hipLaunchKernelGGL(sample_scan_kernel, dim3(a.n_rows * a.scan_parts), block, 0, stream, a);
    hipLaunchKernelGGL(sample_count_kernel, grid, block, 0, stream, a);
    if (a.draw) {
        hipLaunchKernelGGL(sample_gather_kernel<true>, grid, block, 0, stream, a);
    } else {
        hipLaunchKernelGGL(sample_gather_kernel<false>, grid, block, 0, stream, a);
        hipLaunchKernelGGL(sample_draw_kernel, dim3(a.n_rows), block, 0, stream, a);
    }
    return hipGetLastError();
}

// Bytes of scratch, and (with a base) the pointers in it.
size_t ah_sample_plan(SampleArgs &a, uint32_t cus, uint8_t *base) {
    a.groups = (a.n_vocab + kGroup - 1) / kGroup;
    a.chunks = (a.n_vocab + kChunk - 1) / kChunk;
    // At most eight workgroups a CU, all that a CU holds (one more would start when the first ends).  After the scan a
    // workgroup takes a chunk for each of its waves: with one it brought its bins to the row's four times as often (24
    // rows, top-p: count 31 us against 15).
    auto cut = [&](uint32_t least, uint32_t &parts, uint32_t &per) {
        const uint32_t want = 8 * cus / a.n_rows, most = want < 1 ? 1 : want;
        per = ((a.chunks + most - 1) / most + least - 1) / least * least;
        parts = (a.chunks + per - 1) / per;
    };
    cut(1, a.scan_parts, a.scan_per);
    cut(kW, a.parts, a.per);
    if (a.n_rows > a.n_counts) {  // no counter for the arrivals
        a.parts = 1;
        a.per = a.chunks;
    }
    // A launch less for few rows, whose launches are the host's time (24 rows: gather and draw 22 us in one, 18 in two)
    a.draw = a.n_rows * a.parts <= cus;
    const size_t rows = a.n_rows;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        uint8_t *p = base ? base + at : nullptr;
        at += (bytes + 255) & ~(size_t)255;
        return p;
    };
    a.limits = reinterpret_cast<SampleLimits *>(take(sizeof(SampleLimits) * rows));
    a.bin_mass = reinterpret_cast<double *>(take(8 * rows * kBins));
    a.chunk_mass = reinterpret_cast<double *>(take(8 * rows * a.chunks));
    a.bin_count = reinterpret_cast<uint32_t *>(take(4 * rows * kBins));
    a.group_max = reinterpret_cast<float *>(take(4 * rows * a.groups));
    a.bits = reinterpret_cast<uint32_t *>(take(rows * a.chunks * (kChunk / 8)));
    return at;
}
