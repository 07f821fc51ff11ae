// Log probabilities of given tokens with entropy and the k most likely tokens, and their gradient, for gfx950.
//
// Per row of logits x[0 .. V) (bf16 or fp32; rows are P >= V elements apart) and its token t:
//     lse = ln sum_v exp(x_v);  logp = x_t - lse;  entropy = lse - sum_v p_v x_v,  p_v = exp(x_v - lse)
//     dx_v = dlogp (1[v = t] - p_v) - dentropy p_v (x_v - lse + entropy)
//
// HBM bound: the forward reads the logits once (2 or 4 bytes each), the gradient reads and writes them once.  4096 x 151936 bf16:
// forward with the 5 most likely tokens 230 us, 5.4 TB/s (a kernel that only reads reaches 6.2), gradient 444 us, 5.6 TB/s (a plain
// copy 5.8); 777 x 50257 fp32: 33 and 54 us.  One row of 151936 with 20 tokens, in 38 shares and a launch that joins them: 12.6 us,
// two chains of latencies of 7 and 4.
//
// Forward: one pass with a running reference r and sums in base 2.  With d = (x - r) log2 e,
//     s = sum 2^d,   w = sum d 2^d,   lse = r + log2(s) ln 2,   entropy = (log2 s - w / s) ln 2.
// A lane's reference only follows a logit that has outgrown it by 11 (a factor of 6e4), so the sums are rarely rescaled; fp32
// sums lose nothing by a common factor.  x - r is formed before the product: x log2 e - r log2 e as one fused multiply-add is an
// instruction less, but off by the rounding of r log2 e, 2^-24 of it, and 2^d is an infinity or 0 from |r| = 1e10 on, a common mask
// value.  It was no faster either: 4096 x 151936 top 5 228.7 us, this way 229.4; 777 x 50257 fp32 31.0 and 29.8.
//
// The k most likely tokens need no second pass over the row.  In the first turns (about the square root of all of a lane's
// turns) each lane keeps the largest logit of its granules of 16 bytes and the first granule that holds it.  The k-th best of
// such (value, granule) pairs bounds the k-th best logit from below, and of these turns only the lanes that reach it can
// hold one of the k.  From then on every granule with a logit above the bound is listed.  Those granules alone, of some hundreds
// of turns a few hundred, are read again, from the caches; a full re-read of the k best lanes was 20 % of the time at k = 20.
// Where the list overflows (logits that rise along the row) the lanes' best are taken over the whole row instead, and where that
// finds too many, one pass per token.
#include <type_traits>

#include "common.hpp"
#include "absmax_reduce.hpp"

namespace llmq {

typedef float f32x2_lp __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_lp __attribute__((ext_vector_type(2)));

constexpr int kLpThreads = 256, kTopMax = 32, kCandidates = 1024, kSplitMax = 64;
constexpr float kLog2eLp = 1.44269504088896340736f, kLn2Lp = 0.69314718055994530942f;

struct LogprobArgs {
    const void* logits;
    const int* targets;
    float *logp, *entropy, *lse;       // entropy may be NULL
    float* top_logp;                   // [N, k]
    int* top_ids;
    void* scratch;                     // splits > 1: per (row, split) r, s, w, then per (row, split) k keys
    int64_t P;
    int N, V, k, splits;
};

struct LogprobGradArgs {
    void* dlogits;
    const void* logits;
    const float *dlogp, *dentropy;     // dentropy (and entropy) may be NULL
    const int* targets;
    const float *lse, *entropy;
    unsigned* abs_max;
    int64_t P;
    int V, chunks;
};

// 16 bytes of logits as floats, and back.
template <typename E> struct Granule;
template <> struct Granule<uint16_t> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = bf16_lo(w[i]), x[2 * i + 1] = bf16_hi(w[i]);
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x2_lp p = {x[2 * i], x[2 * i + 1]};
            w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2_lp));
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float one(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ uint16_t round(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
};
template <> struct Granule<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[4]) {
        x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[4]) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
    static __device__ __forceinline__ float one(float v) { return v; }
    static __device__ __forceinline__ float round(float x) { return x; }
};

// The granules of a row: 16-byte aligned pieces, the first and the last of which may be partly outside [0, n).  Where rows
// are not multiples of 16 bytes apart, they begin inside a granule.
template <typename E>
struct Row {
    const E* p;
    int lead, n, granules;   // elements of granule 0 before the row, elements of the row

    __device__ __forceinline__ Row(const void* base, int64_t at, int n_) : p(static_cast<const E*>(base) + at), n(n_) {
        lead = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(E));
        granules = (lead + n + Granule<E>::kN - 1) / Granule<E>::kN;
    }
    __device__ __forceinline__ int first(int g) const { return g * Granule<E>::kN - lead; }
    __device__ __forceinline__ bool whole(int g) const { return first(g) >= 0 && first(g) + Granule<E>::kN <= n; }
    __device__ __forceinline__ uint4 load(int g) const { return *reinterpret_cast<const uint4*>(p + first(g)); }
    // the granule's values, -inf outside the row
    __device__ __forceinline__ void values(int g, float (&x)[Granule<E>::kN]) const {
        if (whole(g)) {
            Granule<E>::unpack(load(g), x);
        } else {
#pragma unroll
            for (int j = 0; j < Granule<E>::kN; ++j) {
                const int e = first(g) + j;
                x[j] = e >= 0 && e < n ? Granule<E>::one(p[e]) : -__builtin_huge_valf();
            }
        }
    }
};

// Order-preserving integer of a float, 0 for NaN (which is never among the k); -0 counts as +0.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return 0;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o); }
// larger: a larger value, or the same at a lower place; 0: nothing
__device__ __forceinline__ uint64_t key_of(uint32_t order, uint32_t place) { return order ? (uint64_t)order << 32 | (uint32_t)~place : 0; }

struct Sums {
    float r, s, w;   // reference (-inf: nothing yet), sum, weighted sum
};
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    Sums c;
    c.r = __builtin_fmaxf(a.r, b.r);
    const float ref = c.r == -__builtin_huge_valf() ? 0.f : c.r;
    const float da = __builtin_fmaxf((a.r - ref) * kLog2eLp, -1e4f), db = __builtin_fmaxf((b.r - ref) * kLog2eLp, -1e4f);
    const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
    c.s = a.s * fa + b.s * fb;
    c.w = (a.w + da * a.s) * fa + (b.w + db * b.s) * fb;
    return c;
}

// f over the 64 lanes of a wave, the same in every lane: exchanges inside a row of 16, then of rows and of halves.  All lanes are
// active.  (Through LDS, as shuffles go, each of the six steps took three times as long.)
template <int CTRL>
__device__ __forceinline__ uint32_t across(uint32_t x) { return __builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true); }
template <typename F>
__device__ __forceinline__ uint64_t wave_fold(uint64_t x, F f) {
    auto word = [](uint32_t lo, uint32_t hi) { return (uint64_t)hi << 32 | lo; };
    const auto lo = [](uint64_t v) { return (uint32_t)v; };
    const auto hi = [](uint64_t v) { return (uint32_t)(v >> 32); };
    x = f(x, word(across<0xB1>(lo(x)), across<0xB1>(hi(x))));      // quad_perm 1 0 3 2
    x = f(x, word(across<0x4E>(lo(x)), across<0x4E>(hi(x))));      // quad_perm 2 3 0 1
    x = f(x, word(across<0x141>(lo(x)), across<0x141>(hi(x))));    // row_half_mirror
    x = f(x, word(across<0x140>(lo(x)), across<0x140>(hi(x))));    // row_mirror
    const auto a = __builtin_amdgcn_permlane16_swap(lo(x), lo(x), false, false), b = __builtin_amdgcn_permlane16_swap(hi(x), hi(x), false, false);
    x = f(word(a[0], b[0]), word(a[1], b[1]));
    const auto c = __builtin_amdgcn_permlane32_swap(lo(x), lo(x), false, false), d = __builtin_amdgcn_permlane32_swap(hi(x), hi(x), false, false);
    return f(word(c[0], d[0]), word(c[1], d[1]));
}
template <typename F>
__device__ __forceinline__ float wave_fold(float x, F f) {
    return __uint_as_float((uint32_t)wave_fold((uint64_t)__float_as_uint(x), [&](uint64_t a, uint64_t b) {
        return (uint64_t)__float_as_uint(f(__uint_as_float((uint32_t)a), __uint_as_float((uint32_t)b)));
    }));
}
// the lanes' sums as one, against their common reference
__device__ __forceinline__ Sums wave_join(const Sums& t) {
    Sums c;
    c.r = wave_fold(t.r, [](float a, float b) { return __builtin_fmaxf(a, b); });
    const float ref = c.r == -__builtin_huge_valf() ? 0.f : c.r;
    const float d = __builtin_fmaxf((t.r - ref) * kLog2eLp, -1e4f), f = __builtin_amdgcn_exp2f(d);
    auto add = [](float a, float b) { return a + b; };
    c.s = wave_fold(t.s * f, add);
    c.w = wave_fold((t.w + d * t.s) * f, add);
    return c;
}

__device__ __forceinline__ float lse_of(const Sums& t) { return t.s == 0.f ? -__builtin_huge_valf() : t.r + __builtin_amdgcn_logf(t.s) * kLn2Lp; }

__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }

// How many of n keys in LDS are larger than `key`.  n even, the list 16-byte aligned: two keys a read, eight reads in flight.
__device__ __forceinline__ int count_larger(const uint64_t* keys, int n, uint64_t key) {
    const ulonglong2* p = reinterpret_cast<const ulonglong2*>(keys);
    int c = 0;
#pragma unroll 8
    for (int i = 0; i < n / 2; ++i) {
        const ulonglong2 q = p[i];
        c += (q.x > key) + (q.y > key);
    }
    return c;
}

// What one thread writes for a row.
__device__ __forceinline__ float write_row(const LogprobArgs& a, int row, const Sums& t, float target, bool given) {
    const float lse = lse_of(t);
    a.lse[row] = lse;
    a.logp[row] = !given ? 0.f : lse == -__builtin_huge_valf() ? lse : target - lse;
    if (a.entropy) a.entropy[row] = t.s == 0.f ? 0.f : (__builtin_amdgcn_logf(t.s) - t.w / t.s) * kLn2Lp;
    return lse;
}

// The search for the k best of a workgroup's granules.
struct TopSearch {
    __attribute__((aligned(16))) uint64_t keys[kLpThreads];
    __attribute__((aligned(16))) uint64_t list[kCandidates + 1];
    int granules[kCandidates];
    int chosen[kLpThreads];
    uint64_t floor_key;
    int count, lanes, listed;
};

// The bound below the k-th best and the lanes that reach it, from each lane's best key (0: it has none): the k-th best of the best
// of four lanes each.  (The k-th best lane bounds a little closer, which is worth 1 % at 4096 x 151936 top 20, but finding it among
// 256 took 2.9 us of the 15 of a single row.)
__device__ __forceinline__ uint64_t top_bound(TopSearch& t, uint64_t mine, int k) {
    static_assert(kLpThreads == 4 * kWave && kTopMax <= kWave, "a wave ranks the best of four lanes each");
    const int tid = threadIdx.x;
    auto word = [](uint32_t lo, uint32_t hi) { return (uint64_t)hi << 32 | lo; };
    uint64_t four = larger(mine, word(across<0xB1>((uint32_t)mine), across<0xB1>((uint32_t)(mine >> 32))));
    four = larger(four, word(across<0x4E>((uint32_t)four), across<0x4E>((uint32_t)(four >> 32))));
    if (tid % 4 == 0) t.keys[tid / 4] = four;
    if (tid == 0) t.count = 0, t.lanes = 0, t.listed = 0, t.floor_key = 1;
    __syncthreads();
    if (tid < kWave) {
        const uint64_t key = t.keys[tid];
        if (key && count_larger(t.keys, kWave, key) == k - 1) t.floor_key = key;
    }
    __syncthreads();
    const uint64_t bound = t.floor_key;
    if (mine >= bound) t.chosen[atomicAdd(&t.lanes, 1)] = tid;
    return bound;
}

// Lists the logits of granule `at` that reach the bound.
template <typename E>
__device__ __forceinline__ void top_collect(TopSearch& t, const Row<E>& x, int at, uint64_t bound) {
    float v[Granule<E>::kN];
    x.values(at, v);
#pragma unroll
    for (int j = 0; j < Granule<E>::kN; ++j) {
        const int e = x.first(at) + j;
        const uint32_t o = order_of(v[j]);
        if (e >= 0 && e < x.n && o && key_of(o, (uint32_t)at) >= bound) {
            const int slot = atomicAdd(&t.count, 1);
            if (slot < kCandidates) t.list[slot] = key_of(o, (uint32_t)e);
        }
    }
}

// One row (splits == 1) or one share of its granules per workgroup.
template <typename E, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_kernel(LogprobArgs a) {
    // granules of a lane in flight; bf16 six rather than four: 1500 x 32000 20.9 -> 19.4 us, 4096 x 151936 top 5 227.6 -> 226; fp32 four
    // rather than six: 777 x 50257 35.5 -> 33.3 us, though 300 x 50257 14.2 -> 15.1
    constexpr int kN = Granule<E>::kN, kWaves = kLpThreads / kWave, kInFlight = sizeof(E) == 2 ? 6 : 4;
    __shared__ Sums wave_sums[kWaves];
    __shared__ float shared_lse;
    const int tid = threadIdx.x, row = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    const Row<E> x(a.logits, row * a.P, a.V);
    // lane `tid` takes the granules g0 + tid + i * threads; the two that the row's ends may cut are in turn like the others
    const int g0 = (int)((int64_t)x.granules * split / a.splits), g1 = (int)((int64_t)x.granules * (split + 1) / a.splits);

    Sums t = {-__builtin_huge_valf(), 0.f, 0.f};
    float ref = 0.f, best = -__builtin_huge_valf();
    int best_g = g0 + tid;
    auto largest = [](const float (&v)[kN]) {
        float top = v[0];
#pragma unroll
        for (int j = 1; j < kN; ++j) top = __builtin_fmaxf(top, v[j]);
        return top;
    };
    auto take = [&](const float (&v)[kN], float top) {
        if (__any(top > t.r + 11.f)) {
            const float next = __builtin_fmaxf(t.r, top);
            if (next > -__builtin_huge_valf()) {
                const float d = __builtin_fmaxf((t.r - next) * kLog2eLp, -1e4f), f = __builtin_amdgcn_exp2f(d);
                t.w = (t.w + d * t.s) * f;
                t.s *= f;
                t.r = ref = next;
            }
        }
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            const float d = (v[j] - ref) * kLog2eLp, e = __builtin_amdgcn_exp2f(d);
            t.s += e;
            if constexpr (ENTROPY) t.w = __builtin_fmaf(__builtin_fmaxf(d, -1e4f), e, t.w);   // 0 times -inf is nothing
        }
    };
    // granules [from, to) of the workgroup, each lane's in rising order, `see`(largest logit, granule) before the sums
    auto walk = [&](int from, int to, auto see) {
        int g = from + tid;
        const int inner = to - (to == g1 ? 1 : 0);   // the last granule of all may be cut
        if (g < inner && !x.whole(g)) {              // and the first
            float v[kN];
            x.values(g, v);
            const float top = largest(v);
            see(top, g);
            take(v, top);
            g += kLpThreads;
        }
        for (; g + (kInFlight - 1) * kLpThreads < inner; g += kInFlight * kLpThreads) {
            uint4 q[kInFlight];
#pragma unroll
            for (int u = 0; u < kInFlight; ++u) q[u] = x.load(g + u * kLpThreads);
#pragma unroll
            for (int u = 0; u < kInFlight; ++u) {
                float v[kN];
                Granule<E>::unpack(q[u], v);
                const float top = largest(v);
                see(top, g + u * kLpThreads);
                take(v, top);
            }
        }
        if (g < inner) {   // what is left, at once too
            uint4 q[kInFlight - 1];
#pragma unroll
            for (int u = 0; u < kInFlight - 1; ++u)
                if (g + u * kLpThreads < inner) q[u] = x.load(g + u * kLpThreads);
#pragma unroll
            for (int u = 0; u < kInFlight - 1; ++u) {
                if (g >= inner) break;
                float v[kN];
                Granule<E>::unpack(q[u], v);
                const float top = largest(v);
                see(top, g);
                take(v, top);
                g += kLpThreads;
            }
        }
        if (g < to) {
            float v[kN];
            x.values(g, v);
            const float top = largest(v);
            see(top, g);
            take(v, top);
        }
    };

    __shared__ typename std::conditional<TOP, TopSearch, int>::type search;
    int mid = g1;
    uint64_t bound = 0;
    if constexpr (TOP) {
        const int turns = (g1 - g0 + kLpThreads - 1) / kLpThreads;
        int first = kInFlight;
        while (first * first < turns) first += kInFlight;
        mid = min(g1, g0 + first * kLpThreads);
        walk(g0, mid, [&](float top, int g) {
            if (top > best) best = top, best_g = g;
        });
        bound = top_bound(search, g0 + tid < mid ? key_of(order_of(best), (uint32_t)best_g) : 0, a.k);
        const float above = bound >> 32 ? value_of((uint32_t)(bound >> 32)) : -__builtin_huge_valf();
        walk(mid, g1, [&](float top, int g) {
            if (top > above) {
                const int slot = atomicAdd(&search.listed, 1);
                if (slot < kCandidates) search.granules[slot] = g;
            }
        });
    } else {
        walk(g0, g1, [](float, int) {});
    }

    Sums all = wave_join(t);
    if (tid % kWave == 0) wave_sums[tid / kWave] = all;
    __syncthreads();
    if (tid == 0) {
        all = wave_sums[0];
        for (int w = 1; w < kWaves; ++w) all = join(all, wave_sums[w]);
        if (a.splits == 1) {
            const int target = a.targets[row];
            const bool given = target >= 0 && target < a.V;
            shared_lse = write_row(a, row, all, given ? Granule<E>::one(x.p[target]) : 0.f, given);
        } else {
            static_cast<Sums*>(a.scratch)[blockIdx.x] = all;
        }
    }

    if constexpr (TOP) {
        int end = mid;   // the chosen lanes' granules up to here are looked through
        if (search.listed <= kCandidates) {
            for (int i = tid; i < search.listed; i += kLpThreads) top_collect(search, x, search.granules[i], bound);
        } else {
            best = -__builtin_huge_valf(), best_g = g0 + tid;
            for (int g = g0 + tid; g < g1; g += kLpThreads) {
                float v[kN];
                x.values(g, v);
                const float top = largest(v);
                if (top > best) best = top, best_g = g;
            }
            __syncthreads();
            bound = top_bound(search, g0 + tid < g1 ? key_of(order_of(best), (uint32_t)best_g) : 0, a.k);
            __syncthreads();
            end = g1;
        }
        const int turns = (end - g0 + kLpThreads - 1) / kLpThreads;
        for (int i = tid; i < search.lanes * turns; i += kLpThreads) {
            const int at = g0 + search.chosen[i / turns] + i % turns * kLpThreads;
            if (at < end) top_collect(search, x, at, bound);
        }
        __syncthreads();
        uint64_t* partial = reinterpret_cast<uint64_t*>(static_cast<char*>(a.scratch) + ((int64_t)a.N * a.splits * sizeof(Sums) + 15) / 16 * 16) +
                            (int64_t)blockIdx.x * a.k;
        auto put = [&](int at, uint64_t key) {
            if (a.splits > 1) {
                partial[at] = key;
            } else {
                const bool some = key != 0;
                a.top_ids[(int64_t)row * a.k + at] = some ? (int)~(uint32_t)key : -1;
                const float v = some ? value_of((uint32_t)(key >> 32)) : -__builtin_huge_valf();
                a.top_logp[(int64_t)row * a.k + at] = v == -__builtin_huge_valf() && shared_lse == shared_lse ? v : v - shared_lse;
            }
        };
        const int n = search.count;
        if (n <= kCandidates) {
            if (tid == 0) search.list[n] = 0;   // a pad for the pairwise reads
            __syncthreads();
            for (int i = tid; i < n; i += kLpThreads) {
                const uint64_t key = search.list[i];
                const int at = count_larger(search.list, (n + 1) & ~1, key);
                if (at < a.k) put(at, key);
            }
            for (int i = n + tid; i < a.k; i += kLpThreads) put(i, 0);
        } else {
            uint64_t last = ~0ull;
            for (int round = 0; round < a.k; ++round) {
                uint64_t top = 0;
                for (int at = g0 + tid; at < g1; at += kLpThreads) {
                    float v[kN];
                    x.values(at, v);
#pragma unroll
                    for (int j = 0; j < kN; ++j) {
                        const int e = x.first(at) + j;
                        const uint64_t key = e >= 0 && e < x.n ? key_of(order_of(v[j]), (uint32_t)e) : 0;
                        if (key < last && key > top) top = key;
                    }
                }
                __syncthreads();
                search.keys[tid] = top;
                __syncthreads();
                for (int half = kLpThreads / 2; half > 0; half >>= 1) {
                    if (tid < half && search.keys[tid + half] > search.keys[tid]) search.keys[tid] = search.keys[tid + half];
                    __syncthreads();
                }
                last = search.keys[0];
                if (tid == 0) put(round, last);
                if (last == 0) {
                    for (int i = round + 1 + tid; i < a.k; i += kLpThreads) put(i, 0);
                    break;
                }
            }
        }
    }
}

// Joins the shares of a row, in their order.  Of the shares' keys only those count that reach a bound below the k-th best: the
// k-th best of the shares' best, or the largest of the shares' k-th.
template <typename E>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_join_kernel(LogprobArgs a) {
    __shared__ __attribute__((aligned(16))) uint64_t list[kSplitMax * kTopMax + 1];
    __shared__ __attribute__((aligned(16))) uint64_t heads[kWave];
    __shared__ float shared_lse;
    __shared__ int count;
    __shared__ uint64_t floor_key;
    const int tid = threadIdx.x, row = blockIdx.x;
    const Sums* sums = static_cast<const Sums*>(a.scratch) + (int64_t)row * a.splits;
    const int n = a.splits * a.k;
    const uint64_t* partial = reinterpret_cast<const uint64_t*>(static_cast<const char*>(a.scratch) + ((int64_t)a.N * a.splits * sizeof(Sums) + 15) / 16 * 16) +
                              (int64_t)row * n;
    if (tid < kWave) {
        Sums t = {-__builtin_huge_valf(), 0.f, 0.f};
        if (tid < a.splits) t = sums[tid];
        const uint64_t best = a.k && tid < a.splits ? partial[tid * a.k] : 0;
        uint64_t last = a.k && tid < a.splits ? partial[tid * a.k + a.k - 1] : 0;
        t = wave_join(t);
        last = wave_fold(last, larger);
        if (tid == 0) {
            const int target = a.targets[row];
            const bool given = target >= 0 && target < a.V;
            const E* p = static_cast<const E*>(a.logits) + row * a.P;
            shared_lse = write_row(a, row, t, given ? Granule<E>::one(p[target]) : 0.f, given);
            count = 0;
            floor_key = last > 1 ? last : 1;
        }
        heads[tid] = best;
    }
    if (a.k == 0) return;
    __syncthreads();
    if (tid < kWave && a.splits >= a.k) {
        const uint64_t best = heads[tid];
        if (best > floor_key && count_larger(heads, kWave, best) == a.k - 1) floor_key = best;
    }
    __syncthreads();
    const uint64_t bound = floor_key;
    for (int i = tid; i < n; i += kLpThreads) {
        const uint64_t key = partial[i];
        if (key >= bound) list[atomicAdd(&count, 1)] = key;
    }
    __syncthreads();
    const int m = count;
    if (tid == 0) list[m] = 0;
    __syncthreads();
    for (int i = tid; i < max(m, a.k); i += kLpThreads) {
        const uint64_t key = i < m ? list[i] : 0;
        const int at = i < m ? count_larger(list, (m + 1) & ~1, key) : i;
        if (at >= a.k) continue;
        a.top_ids[(int64_t)row * a.k + at] = key ? (int)~(uint32_t)key : -1;
        const float v = key ? value_of((uint32_t)(key >> 32)) : -__builtin_huge_valf();
        a.top_logp[(int64_t)row * a.k + at] = v == -__builtin_huge_valf() && shared_lse == shared_lse ? v : v - shared_lse;
    }
}

// ---- gradient --------------------------------------------------------------------------------------------------------------
constexpr int kGradTurns = 4;   // granules of a lane

template <typename E, bool ENTROPY, bool ABSMAX>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_backward_kernel(LogprobGradArgs a) {
    constexpr int kN = Granule<E>::kN;
    const int tid = threadIdx.x, row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const Row<E> x(a.logits, row * a.P, (int)a.P);
    E* out = static_cast<E*>(a.dlogits) + row * a.P;
    const int at0 = chunk * (kLpThreads * kGradTurns) + tid;
    // the logits are asked for before the row's scalars are waited for
    uint4 q[kGradTurns];
#pragma unroll
    for (int u = 0; u < kGradTurns; ++u) {
        const int at = at0 + u * kLpThreads;
        if (at < x.granules && x.whole(at)) q[u] = load_nt(reinterpret_cast<const uint4*>(x.p + x.first(at)));
    }
    uint32_t fold = sizeof(E) == 2 ? 0x7F807F80u : 0x7F800000u;
    const int target = a.targets[row];
    const bool given = target >= 0 && target < a.V;
    const float lse = a.lse[row], g = given ? a.dlogp[row] : 0.f;
    float h = 0.f, shift = 0.f;
    if constexpr (ENTROPY) h = a.dentropy[row], shift = a.entropy[row];
    // no gradient enters, or the row has no probability: zeros, whatever the logits hold
    const bool none = (g == 0.f && h == 0.f) || lse == -__builtin_huge_valf();
    auto derive = [&](float v) {
        const float d = v - lse, p = __builtin_amdgcn_exp2f(d * kLog2eLp);
        float c = -g;
        if constexpr (ENTROPY) c -= h * (__builtin_fmaxf(d, -1e4f) + shift);
        return p * c;
    };
#pragma unroll
    for (int u = 0; u < kGradTurns; ++u) {
        const int at = at0 + u * kLpThreads;
        if (at >= x.granules) continue;
        const int e0 = x.first(at);
        if (x.whole(at)) {
            float v[kN];
            Granule<E>::unpack(q[u], v);
#pragma unroll
            for (int j = 0; j < kN; ++j) v[j] = derive(v[j]);
            if (given && (unsigned)(target - e0) < (unsigned)kN) {
#pragma unroll
                for (int j = 0; j < kN; ++j) v[j] += e0 + j == target ? g : 0.f;
            }
            if (none || e0 + kN > a.V) {
#pragma unroll
                for (int j = 0; j < kN; ++j) v[j] = none || e0 + j >= a.V ? 0.f : v[j];
            }
            const uint4 w = Granule<E>::pack(v);
            store_nt(reinterpret_cast<uint4*>(out + e0), w);
            if constexpr (ABSMAX) {
                if constexpr (sizeof(E) == 2) {
                    fold = fold_vec(fold, w);
                } else {
                    const uint32_t b[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) fold = min(fold, 0x7F800000u - (b[j] & 0x7FFFFFFFu));
                }
            }
        } else {
            for (int j = 0; j < kN; ++j) {
                const int e = e0 + j;
                if (e < 0 || e >= x.n) continue;
                const float v = none || e >= a.V ? 0.f : derive(Granule<E>::one(x.p[e])) + (e == target ? g : 0.f);
                const E r = Granule<E>::round(v);
                out[e] = r;
                if constexpr (ABSMAX) {
                    if constexpr (sizeof(E) == 2) fold = fold_bf16x2(fold, (uint32_t)__builtin_bit_cast(uint16_t, r));
                    else fold = min(fold, 0x7F800000u - (__builtin_bit_cast(uint32_t, r) & 0x7FFFFFFFu));
                }
            }
        }
    }
    if constexpr (ABSMAX) {
        if constexpr (sizeof(E) == 2) {
            const uint32_t lo = fold & 0xFFFFu, hi = fold >> 16;
            block_min_to_atomic_max(a.abs_max, lo < hi ? lo : hi, 0x7F80u, 16);
        } else {
            block_min_to_atomic_max(a.abs_max, fold, 0x7F800000u, 0);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
// Shares of a row: one workgroup a compute unit when there are few rows, each with at least 4096 logits.  (Two a unit: 300 x 50257
// top 5 20.9 -> 23.3 us, 8 x 151936 14.2 -> 14.5.  2048 logits: 1 x 151936 top 20 15.2 -> 14.6, but 1 x 8000 top 4 11.9 -> 12.7;
// 8192: 17.7 and 10.2.)
static int logprob_splits(int N, int V) {
    int64_t s = (256 + (int64_t)N - 1) / N;
    const int64_t most = ((int64_t)V + 4095) / 4096;
    s = s < most ? s : most;
    return (int)(s < 1 ? 1 : s > kSplitMax ? kSplitMax : s);
}
static int64_t logprob_scratch(int N, int V, int k) {
    const int splits = logprob_splits(N, V);
    return splits > 1 ? ((int64_t)N * splits * (int64_t)sizeof(Sums) + 15) / 16 * 16 + (int64_t)N * splits * k * 8 : 0;
}

template <typename E>
static int token_logprobs_any(float* logp, float* entropy, float* lse, float* top_logp, int* top_ids, const E* logits, const int* targets,
                              void* scratch, size_t scratch_bytes, int64_t N64, int V, int64_t P, int k, hipStream_t stream) {
    const char* what = "token_logprobs";
    LLMQ_REQUIRE(N64 >= 0 && N64 < (1 << 24), "%s: fewer than 2^24 rows are wanted (got %lld)", what, (long long)N64);
    const int N = (int)N64;
    LLMQ_REQUIRE(V >= 1 && V <= (1 << 28) && P >= V && P <= (1 << 28), "%s: vocabulary %d, row length %lld: 1 <= V <= P <= 2^28 is wanted", what, V, (long long)P);
    LLMQ_REQUIRE(k >= 0 && k <= kTopMax, "%s: at most %d alternatives (got %d)", what, kTopMax, k);
    if (N == 0) return LLMQ_OK;
    LLMQ_REQUIRE(logp && lse && logits && targets, "%s: null tensor pointer", what);
    LLMQ_REQUIRE(k == 0 || (top_logp && top_ids), "%s: alternatives need both their tensors", what);
    LLMQ_REQUIRE(aligned16(logits), "%s: logits must be 16-byte aligned", what);
    const int64_t need = logprob_scratch(N, V, k);
    LLMQ_REQUIRE(need == 0 || (scratch && aligned16(scratch) && scratch_bytes >= (size_t)need), "%s: scratch buffer too small or not 16-byte aligned (%zu bytes, %lld needed)",
                 what, scratch_bytes, (long long)need);
    const int64_t row = (int64_t)N * 4;
    const Range written[] = {{logp, row}, {entropy, entropy ? row : 0}, {lse, row}, {top_logp, row * k}, {top_ids, row * k}, {scratch, need}};
    const Range read[] = {{logits, N * P * (int64_t)sizeof(E)}, {targets, row}};
    LLMQ_REQUIRE(apart(written, read), "%s: the outputs and the scratch must be memory of their own", what);
    LogprobArgs a = {};
    a.logits = logits, a.targets = targets, a.logp = logp, a.entropy = entropy, a.lse = lse, a.top_logp = top_logp, a.top_ids = top_ids;
    a.scratch = scratch, a.P = P, a.N = N, a.V = V, a.k = k, a.splits = logprob_splits(N, V);
    auto launch = [&](auto kernel, int64_t blocks) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kLpThreads), 0, stream, a); };
    const int64_t blocks = (int64_t)N * a.splits;
    if (entropy) {
        if (k) launch(token_logprobs_kernel<E, true, true>, blocks);
        else launch(token_logprobs_kernel<E, true, false>, blocks);
    } else {
        if (k) launch(token_logprobs_kernel<E, false, true>, blocks);
        else launch(token_logprobs_kernel<E, false, false>, blocks);
    }
    LLMQ_HIP_TRY(hipGetLastError());
    if (a.splits > 1) {
        launch(token_logprobs_join_kernel<E>, N);
        LLMQ_HIP_TRY(hipGetLastError());
    }
    return LLMQ_OK;
}

template <typename E>
static int token_logprobs_backward_any(E* dlogits, const float* dlogp, const float* dentropy, const E* logits, const int* targets,
                                       const float* lse, const float* entropy, float* abs_max, int64_t N64, int V, int64_t P, hipStream_t stream) {
    const char* what = "token_logprobs_backward";
    LLMQ_REQUIRE(N64 >= 0 && N64 < (1 << 24), "%s: fewer than 2^24 rows are wanted (got %lld)", what, (long long)N64);
    LLMQ_REQUIRE(V >= 1 && V <= (1 << 28) && P >= V && P <= (1 << 28), "%s: vocabulary %d, row length %lld: 1 <= V <= P <= 2^28 is wanted", what, V, (long long)P);
    LLMQ_REQUIRE(!dentropy || entropy || N64 == 0, "%s: dentropy needs the forward's entropy", what);
    const int64_t granules = P / Granule<E>::kN + 2;   // at most, wherever a row begins
    const int chunks = (int)((granules + kLpThreads * kGradTurns - 1) / (kLpThreads * kGradTurns));
    const int64_t blocks = N64 * chunks;
    LLMQ_REQUIRE(blocks < (1 << 24), "%s: tensor too large", what);   // the threads of a grid fit 32 bits
    if (N64 > 0) {
        LLMQ_REQUIRE(dlogits && dlogp && logits && targets && lse, "%s: null tensor pointer", what);
        LLMQ_REQUIRE(aligned16(dlogits) && aligned16(logits), "%s: pointers must be 16-byte aligned", what);
        const int64_t row = N64 * 4, all = N64 * P * (int64_t)sizeof(E);
        const Range written[] = {{dlogits, all}, {abs_max, abs_max ? 4 : 0}};
        const Range read[] = {{logits, dlogits == logits ? 0 : all}, {dlogp, row}, {dentropy, dentropy ? row : 0}, {targets, row}, {lse, row},
                              {entropy, dentropy ? row : 0}};
        LLMQ_REQUIRE(apart(written, read), "%s: dlogits must be logits or memory of its own, abs_max memory of its own", what);
    }
    if (abs_max) {
        hipLaunchKernelGGL(reset_slot_kernel, dim3(1), dim3(1), 0, stream, reinterpret_cast<unsigned*>(abs_max));
        LLMQ_HIP_TRY(hipGetLastError());
    }
    if (N64 == 0) return LLMQ_OK;
    LogprobGradArgs a = {};
    a.dlogits = dlogits, a.logits = logits, a.dlogp = dlogp, a.dentropy = dentropy, a.targets = targets, a.lse = lse, a.entropy = entropy;
    a.abs_max = reinterpret_cast<unsigned*>(abs_max);
    a.P = P, a.V = V, a.chunks = chunks;
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kLpThreads), 0, stream, a); };
    if (dentropy) {
        if (abs_max) launch(token_logprobs_backward_kernel<E, true, true>);
        else launch(token_logprobs_backward_kernel<E, true, false>);
    } else {
        if (abs_max) launch(token_logprobs_backward_kernel<E, false, true>);
        else launch(token_logprobs_backward_kernel<E, false, false>);
    }
    LLMQ_HIP_TRY(hipGetLastError());
    return LLMQ_OK;
}

}  // namespace llmq

extern "C" int64_t llmq_token_logprobs_scratch_bytes(int64_t N, int V, int k) {
    if (N <= 0 || N >= (1 << 24) || V <= 0 || k < 0 || k > llmq::kTopMax) return 0;
    return llmq::logprob_scratch((int)N, V, k);
}
extern "C" int llmq_token_logprobs_bf16(float* logp, float* entropy_or_null, float* lse, float* top_logp, int* top_ids, const uint16_t* logits,
                                        const int* targets, void* scratch, size_t scratch_bytes, int64_t N, int V, int64_t P, int k, void* stream) {
    return llmq::token_logprobs_any(logp, entropy_or_null, lse, top_logp, top_ids, logits, targets, scratch, scratch_bytes, N, V, P, k,
                                    static_cast<hipStream_t>(stream));
}
extern "C" int llmq_token_logprobs_f32(float* logp, float* entropy_or_null, float* lse, float* top_logp, int* top_ids, const float* logits,
                                       const int* targets, void* scratch, size_t scratch_bytes, int64_t N, int V, int64_t P, int k, void* stream) {
    return llmq::token_logprobs_any(logp, entropy_or_null, lse, top_logp, top_ids, logits, targets, scratch, scratch_bytes, N, V, P, k,
                                    static_cast<hipStream_t>(stream));
}
extern "C" int llmq_token_logprobs_backward_bf16(uint16_t* dlogits, const float* dlogp, const float* dentropy_or_null, const uint16_t* logits,
                                                 const int* targets, const float* lse, const float* entropy_or_null, float* abs_max_or_null,
                                                 int64_t N, int V, int64_t P, void* stream) {
    return llmq::token_logprobs_backward_any(dlogits, dlogp, dentropy_or_null, logits, targets, lse, entropy_or_null, abs_max_or_null, N, V, P,
                                             static_cast<hipStream_t>(stream));
}
extern "C" int llmq_token_logprobs_backward_f32(float* dlogits, const float* dlogp, const float* dentropy_or_null, const float* logits,
                                                const int* targets, const float* lse, const float* entropy_or_null, float* abs_max_or_null,
                                                int64_t N, int V, int64_t P, void* stream) {
    return llmq::token_logprobs_backward_any(dlogits, dlogp, dentropy_or_null, logits, targets, lse, entropy_or_null, abs_max_or_null, N, V, P,
                                             static_cast<hipStream_t>(stream));
}
