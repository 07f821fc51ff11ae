// Causal attention on the fused QKV tensor for gfx950: forward, and the backward pass that recomputes the probabilities.
//
// qkv is [B, T, Nq + 2 Nkv, head_dim] bf16, the tensor rope_forward writes; query head h reads key/value head h / (Nq / Nkv).
// With the keys query t of row b may look at, A(t) = { k : max(0, first_key[b, t]) <= k <= t } (first_key NULL: 0),
//     s = scale q_t . k_k     lse_t = ln sum_{k in A(t)} exp(s)     p = exp(s - lse_t)     out_t = sum_{k in A(t)} p v_k
// and, with D_t = sum_d dout_t out_t and ds = p (dout_t . v_k - D_t),
//     dq_t = scale sum_k ds k_k      dk_k = scale sum_{h, t} ds q_t      dv_k = sum_{h, t} p dout_t
// (the sums of dk and dv run over the query heads of the group).  first_key expresses packed documents (the document's first
// token), a sliding window (t - w + 1) and padding (any value above t: the row is empty, out 0, lse -inf, no gradient).
//
// Three kernels: the forward and the queries' backward pass, where a wave owns 32 queries and walks their keys, and the keys'
// backward pass, where a wave owns 32 keys and walks the queries of every head of its group.  So dq, dk and dv are each summed by
// one wave in a fixed order, without atomics, for two products computed twice (seven in place of five).  Rounded to bf16: the
// probabilities and ds, as operands of the matrix instructions, and the results; scores, statistics and sums are fp32.
//
// Exponents are one fused multiply-add, s scale2 - m scale2, scale2 = scale log2 e.  The second product is rounded, which moves all of
// a row's exponents by up to 2^-24 of it: a common factor of no account, until at scores of 1e9 it is infinite or 0.  So beyond
// |m scale2| = 2^14 the forward pass takes (s - m) scale2.  The backward pass, whose lse is a rounded number of its own, there takes
// (s scale - lse) log2 e, which is 0 where lse came from this score alone; up to there its exponents are off by 2^-8 at most, which
// is what the probabilities' rounding to 16 bits is.  Both only in the careful forms behind the walks: a branch in the forward walk
// cost 1 x 8192 461.6 -> 465.9 us, at 64 dimensions 149 -> 153.
//
// Bound: long sequences by the package's power.  1 x 8192 with 28 query and 4 key heads of 128, from box to box: forward 443 to 466 us,
// 1.03 to 1.09 PFLOP/s of allowed pairs, at 1.9 of 2.4 GHz with the matrix cores busy 55 % of the cycles; backward 1525 to 1590 us, 0.76 to
// 0.79 PFLOP/s, 1.06 to 1.10 with the products computed twice.  (The library's product of two 8192 x 8192 bf16 matrices: 1.18 to 1.25.)
// Deeper pipelining of the two products and eight waves a workgroup left these times as they were.  Short ones by what a workgroup
// costs besides its walk: forward 8 x 1024 (77 to 88 us, 0.68 to 0.78 PFLOP/s) 4 of its 21 us, and an eighth of the walk lies behind
// the diagonal; of the keys' walk a sixth, and its waves wait 47 % of their cycles (matrix cores busy 33 %, LDS 25 %).
#include <climits>

#include "common.hpp"
#include "absmax_reduce.hpp"
#include "attention_tile.hpp"

namespace llmq {

struct AttentionArgs {
    const uint16_t* qkv;
    const int* first_key;    // [B, T] or NULL
    uint16_t* out;           // forward: [B, T, Nq, head_dim]; backward: the forward's
    float* lse;              // [B, Nq, T]
    unsigned* abs_max;       // forward only, or NULL
    const uint16_t* dout;
    uint16_t* dqkv;
    float* lse2;             // backward scratch: fused_lse, [B, Nq, T]
    float* delta;            // D, [B, Nq, T]
    int* flags;              // per workgroup of the keys' kernel: whether a value was not finite
    int2* groups;            // with first_key: per 32 queries the smallest first key of a row that has any, the largest of all
    float* partial;          // dk, dv of each split: [splits][B, T, Nkv][2][head_dim], or NULL (one split, written to dqkv)
    int B, T, Nq, Nkv, head_dim, G;
    int splits;
    float scale, scale2;     // softmax scale, and times log2 e
};

constexpr int kKeys = 64;    // rows of a staged tile

constexpr float kFusedMost = 16384.f;   // base-2 scores beyond it are subtracted before they are scaled

// The base-2 lse of a row for fused exponents, NaN beyond their range: every sum that the row enters is then NaN, and the careful form,
// which computes such sums again, takes exponent().
__device__ __forceinline__ float fused_lse(float lse) {
    const float lse2 = lse * kLog2e, size = __builtin_fabsf(lse2);
    return size > kFusedMost && __builtin_fabsf(lse) < __builtin_huge_valf() ? __builtin_nanf("") : lse2;
}
// The exponent of a probability from its score and the row's lse, whatever their size.  (No fused multiply-add: the score is rounded
// as the forward pass rounded the one that lse came from.)
__device__ __forceinline__ float exponent(float s, float lse, float scale, float scale2) {
    const float lse2 = lse * kLog2e;
    return __builtin_fabsf(lse2) > kFusedMost ? (s * scale - lse) * kLog2e : __builtin_fmaf(s, scale2, -lse2);
}

__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x = min(x, __shfl_xor(x, off, kWave));
    return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int wave_max(int x) { return ~wave_min(~x); }

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// Column-side operand of a wave, straight from global memory: lane -> position l % 32, chunk 2 step + l / 32.  On its way from
// here, waited for in `arrived`.
template <int HDP>
__device__ __forceinline__ void load_columns(bf16x8 (&f)[HDP / 16], const uint16_t* row, int lane, int head_dim) {
#pragma unroll
    for (int s = 0; s < HDP / 16; ++s) {
        const int d = 16 * s + 8 * (lane >> 5);
        const uint16_t* p = d < head_dim ? row + d : reinterpret_cast<const uint16_t*>(attention_zeros);
        f[s] = *reinterpret_cast<const bf16x8*>(p);
    }
}
template <int N>
__device__ __forceinline__ void arrived(bf16x8 (&f)[N]) {   // not in every turn of the loop that uses them
#pragma unroll
    for (int s = 0; s < N; ++s) asm volatile("" : "+v"(f[s]));
}

// Stores dimensions 32 db .. of a transposed result (dimensions by positions) times `factor` as bf16 to `row`, this lane's
// position: the two lanes of a position swap groups of four dimensions, so that each writes 16 bytes.  Returns the abs-max fold.
__device__ __forceinline__ uint32_t store_columns(uint16_t* row, const f32x16& acc, int db, float factor, int lane, int head_dim, bool valid,
                                                  uint32_t fold) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        uint32_t w[2][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int i = 8 * g + 4 * e;
            w[e][0] = pack_bf16(acc[i] * factor, acc[i + 1] * factor);
            w[e][1] = pack_bf16(acc[i + 2] * factor, acc[i + 3] * factor);
        }
        const auto x = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
        const int d = db * 32 + 16 * g + 8 * (lane >> 5);
        if (valid && d < head_dim) {
            const uint4 v = make_uint4(x[0], y[0], x[1], y[1]);
            *reinterpret_cast<uint4*>(row + d) = v;
            fold = fold_vec(fold, v);
        }
    }
    return fold;
}

__device__ __forceinline__ bool all_finite(const f32x16& x) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t = __builtin_fmaf(x[i], 0.f, t);
    return t == 0.f;
}

// What a wave's 32 queries may look at.
struct QueryMask {
    int q, first;           // this lane's position and its first key (INT_MAX: empty, or behind the last row)
    int lo, hi;             // smallest first key and largest position of the wave's rows that are not empty (lo > hi: none)
    int first_max, q_min;   // a tile [k0, k1] is whole for the wave if k0 >= first_max and k1 <= q_min

    // the first key on its way
    __device__ __forceinline__ void load(const AttentionArgs& a, int b, int q0, int lane) {
        q_min = q0;
        q = q0 + (lane & 31);
        first = a.first_key ? a.first_key[(int64_t)b * a.T + min(q, a.T - 1)] : 0;
    }
    __device__ __forceinline__ void derive(const AttentionArgs& a) {
        hi = q_min < a.T ? min(q_min + 32, a.T) - 1 : -1;
        lo = q_min < a.T ? 0 : INT_MAX;
        first_max = 0;
        if (a.first_key) {
            first = q < a.T && first <= q ? max(first, 0) : INT_MAX;
            lo = wave_min(first);
            hi = wave_max(first <= q ? q : -1);
            first_max = wave_max(q < a.T ? first : 0);
        }
    }
    __device__ __forceinline__ bool whole(int k0, int k1) const { return k0 >= first_max && k1 <= q_min; }
    __device__ __forceinline__ bool allowed(int k) const { return k <= q && k >= first; }
};

// Key of register i of row block rb of the tile that starts at k0.
__device__ __forceinline__ int tile_row(int rb, int i, int lane) { return rb * 32 + 8 * (i / 4) + 4 * (lane >> 5) + (i & 3); }

// Range of tiles the workgroup walks: from its waves' smallest first key to its last query.
template <int WAVES>
__device__ __forceinline__ void block_range(int& lo, int& hi, int wave_lo, int wave_hi) {
    __shared__ int ends[2][WAVES];
    if (threadIdx.x % kWave == 0) {
        ends[0][threadIdx.x / kWave] = wave_lo;
        ends[1][threadIdx.x / kWave] = wave_hi;
    }
    __syncthreads();
    lo = INT_MAX;
    hi = -1;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        lo = min(lo, ends[0][w]);
        hi = max(hi, ends[1][w]);
    }
    lo = __builtin_amdgcn_readfirstlane(lo), hi = __builtin_amdgcn_readfirstlane(hi);
}

// Keeps what is derived from a lane's value out of registers that live across a loop or the loop's whole kernel: it is derived
// again where it is used.
__device__ __forceinline__ int here(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// ---- forward and the backward's queries: a workgroup's geometry ---------------------------------------------------------
// A wave owns 32 queries (columns) and walks the keys (rows) in tiles of 64 that the workgroup's waves share in LDS: two buffers,
// the next tile copied while one is computed.  A copy occupies the wave that issues it for about a hundred cycles when they come
// in a row (eight of them were a quarter of a tile's time), so they are spread over the steps of the scores' product.  Behind the
// last tile it is copied once more, so that the steps need no branch.
template <int HDP, int WAVES>
struct QueryBlock {
    typedef Tile<HDP, kKeys> T;
    static constexpr int kThreads = WAVES * kWave, kSteps = HDP / 16, kDims = HDP / 32, kBlock = 32 * WAVES;
    static constexpr int kLdsBytes = 4 * T::kBytes;
    typedef TileCopy<HDP, kKeys, kThreads> Copy;
    static constexpr int kCopies = 2 * Copy::kCopies;
    static_assert(kCopies <= kSteps, "a copy a step");

    const AttentionArgs& a;
    char* lds;
    uint32_t lds_at;            // address of the wave's share
    int tid, lane, b, kvh, head, block, q0;   // block: the workgroup's first query, q0: the wave's
    int64_t token, stride;      // elements of a token, bytes
    const uint16_t *base, *kbase;
    Copy copy;
    uint32_t ofs[Copy::kCopies];
    const char *knext, *vnext;  // of the tile that is being copied
    uint32_t to;                // and where
    QueryMask mask;
    int t_lo, t_hi;             // tiles of the workgroup (t_lo > t_hi: none)
    int w_lo, w_hi;             // and of the wave

    __device__ __forceinline__ QueryBlock(const AttentionArgs& args, char* lds_) : a(args), lds(lds_), copy(threadIdx.x, args.head_dim) {
        tid = threadIdx.x, lane = tid % kWave;
        const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
        lds_at = lds_address(lds) + wave * 1024;
        // Workgroups go to the dies round-robin: the groups of heads that share keys are the fastest index, so that a group
        // stays on one die's L2 where their number allows; the last queries, which have the most keys, come first.
        const int ngroups = a.B * a.Nkv, nq = (a.T + kBlock - 1) / kBlock;
        const int grp = blockIdx.x % ngroups, rest = blockIdx.x / ngroups;
        b = grp / a.Nkv, kvh = grp % a.Nkv, head = kvh * a.G + rest % a.G;
        block = (nq - 1 - rest / a.G) * kBlock, q0 = block + wave * 32;
        token = (int64_t)(a.Nq + 2 * a.Nkv) * a.head_dim, stride = token * 2;
        base = a.qkv + b * a.T * token;
        kbase = base + (int64_t)(a.Nq + kvh) * a.head_dim;
        mask.load(a, b, q0, lane);   // before the rows, which are waited for later
    }
    // What the rows look at, and the first copies.
    __device__ __forceinline__ void begin() {
        if (a.head_dim < HDP) {
#pragma unroll
            for (int i = 0; i < 4; ++i) T::template clear<kThreads>(lds + i * T::kBytes, tid);
        }
        mask.derive(a);
        int lo = 0, hi = min(block + kBlock, a.T) - 1;
        if (a.first_key) block_range<WAVES>(lo, hi, mask.lo, mask.hi);
        else if (a.head_dim < HDP) __syncthreads();
        t_lo = lo <= hi ? lo / kKeys : 1, t_hi = lo <= hi ? hi / kKeys : 0;
        w_lo = mask.lo <= mask.hi ? mask.lo / kKeys : INT_MAX, w_hi = mask.lo <= mask.hi ? mask.hi / kKeys : -1;
        start();
        if (t_lo <= t_hi) {
            aim(t_lo & 1, t_lo);
            issue_all();
        }
    }
    // before a walk over the tiles
    __device__ __forceinline__ void start() { copy.offsets(ofs, stride, 0, INT_MAX); }
    __device__ __forceinline__ char* keys(int buf) const { return lds + buf * T::kBytes; }
    __device__ __forceinline__ char* values(int buf) const { return lds + (2 + buf) * T::kBytes; }
    // copies of tile t (of the last one if it is behind it) into `buf`, one by one
    __device__ __forceinline__ void aim(int buf, int t) {
        const int row0 = min(t, t_hi) * kKeys;
        if (row0 + kKeys > a.T) copy.offsets(ofs, stride, row0, a.T);   // the last tile of the sequence: none follows in this walk
        knext = reinterpret_cast<const char*>(kbase) + row0 * stride;
        vnext = knext + (int64_t)a.Nkv * a.head_dim * 2;
        to = lds_at + buf * T::kBytes;
    }
    __device__ __forceinline__ void issue(int i) const {
        if (i < Copy::kCopies) copy.copy(i, to, ofs, knext);
        else if (i < kCopies) copy.copy(i - Copy::kCopies, to + 2 * T::kBytes, ofs, vnext);
    }
    __device__ __forceinline__ void issue_all() const {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) issue(i);
    }
    __device__ __forceinline__ int row() const { return min(q0 + (lane & 31), a.T - 1); }   // rows behind the last one repeat it
    // Tiles from t on, before `to`, that the wave only copies for the others; returns the next.  (As a branch in the walk itself it
    // moved accumulators between registers: 8 x 1024 84 -> 87.5 us, where this way it is 82.3.)
    __device__ __forceinline__ int pass(int t, int to) {
#pragma nounroll
        for (; t <= t_hi && t < to; ++t) {
            copies_landed();
            aim((t + 1) & 1, t + 1);
            issue_all();
        }
        return t;
    }
    __device__ __forceinline__ void load_rows(bf16x8 (&f)[kSteps], const uint16_t* tensor, int64_t row_elements) const {
        load_columns<HDP>(f, tensor + row() * row_elements + (int64_t)head * a.head_dim, lane, a.head_dim);
    }
    __device__ __forceinline__ bool whole(int t) const { return mask.whole(t * kKeys, t * kKeys + kKeys - 1); }
    __device__ __forceinline__ bool allowed(int t, int rb, int i) const { return mask.allowed(t * kKeys + tile_row(rb, i, lane)); }
    // ones in the places that count, as an operand
    __device__ __forceinline__ bf16x8 counted(int t, int rb, int u) const {
        f32x16 in;
#pragma unroll
        for (int i = 0; i < 16; ++i) in[i] = allowed(t, rb, i) ? 1.f : 0.f;
        return operand(in, u);
    }
    __device__ __forceinline__ bool valid() const { return mask.q < a.T; }
    __device__ __forceinline__ int64_t row_statistic() const { return ((int64_t)b * a.Nq + head) * a.T + row(); }
    __device__ __forceinline__ int64_t statistic() const { return ((int64_t)b * a.Nq + head) * a.T + mask.q; }
    __device__ __forceinline__ uint16_t* out_row() const { return a.out + (((int64_t)b * a.T + mask.q) * a.Nq + head) * a.head_dim; }
    __device__ __forceinline__ uint16_t* dq_row() const { return a.dqkv + ((int64_t)b * a.T + mask.q) * token + (int64_t)head * a.head_dim; }
};

constexpr int kAhead = 2;   // steps that fragments are read ahead of their matrix instructions

// s = K q of a key tile; between(step) after each step
template <int HDP, typename F>
__device__ __forceinline__ void tile_scores(f32x16 (&s)[2], const char* keys, int row_lane, const bf16x8 (&qf)[HDP / 16], F between) {
    typedef Tile<HDP, kKeys> T;
    constexpr int kSteps = HDP / 16;
    bf16x8 kf[kSteps][2];
    s[0] = zero16(), s[1] = zero16();
#pragma unroll
    for (int st = -kAhead; st < kSteps; ++st) {
        if (st + kAhead < kSteps) {
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) kf[st + kAhead][rb] = T::rows(keys, row_lane, rb, st + kAhead);
        }
        if (st < 0) continue;
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) s[rb] = mfma(kf[st][rb], qf[st], s[rb]);
        between(st);
        __builtin_amdgcn_sched_barrier(0);
    }
}
template <typename Block>
__device__ __forceinline__ void mask_scores(f32x16 (&s)[2], const Block& w, int t) {
#pragma unroll
    for (int rb = 0; rb < 2; ++rb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (!w.allowed(t, rb, i)) s[rb][i] = -__builtin_huge_valf();
}

// A wave in its matrix products goes before waves in their softmax, up to 64 dimensions, where the softmax is the longer part:
// window 1 x 8192 forward 63.9 -> 61.9 us, backward (the keys' first products) 207 -> 201.5.  Above it costs: 8 x 1024 forward
// 82.5 -> 85.8, backward 323 -> 324.5; so it does in the queries' backward pass: 201.4 -> 203.
template <int HDP, int PRIORITY>
__device__ __forceinline__ void matrix_priority() {
    if constexpr (HDP == 64) __builtin_amdgcn_s_setprio(PRIORITY);
}

// ---- forward ------------------------------------------------------------------------------------------------------------
// Whether a row's largest score lies beyond the fused exponents.
__device__ __forceinline__ bool beyond_fused(float m, float scale2) {
    return __builtin_fabsf(m) < __builtin_huge_valf() && __builtin_fabsf(m * scale2) > kFusedMost;
}
__device__ __forceinline__ float row_lse(float m, float l, float scale, float scale2) {
    const float log2l = __builtin_amdgcn_logf(l);
    if (m == -__builtin_huge_valf() && l == 0.f) return m;
    return beyond_fused(m, scale2) ? m * scale + log2l * kLn2 : (m * scale2 + log2l) * kLn2;   // the first as exponent() expects it
}

// The walk of the careful forms, a tile at a time.
template <typename W, typename F>
__device__ __forceinline__ void careful_walk(W& w, F each) {
    w.start();
#pragma nounroll
    for (int t = w.t_lo; t <= w.t_hi; ++t) {
        w.aim(0, t);
        w.issue_all();
        copies_landed();
        if (t >= w.w_lo && t <= w.w_hi) each(t);
        __syncthreads();
    }
}

// The careful form of a workgroup in which a value was not finite or a score beyond the fused exponents: 32 dimensions at a time, with
// the product that keeps masked places out.  The rows' largest scores stand; their sums l too, unless `sums`.  Probabilities are divided
// by l before the product: with values near the type's largest, sums of undivided ones overflow where their mean does not.  (As a
// function of its own, which the compiler gives a stack, it cost 20 us a launch.)
template <int HDP, typename W>
__device__ __forceinline__ uint32_t attention_forward_careful(W& w, const bf16x8 (&qf)[W::kSteps], float m, float l, bool sums) {
    typedef typename W::T T;
    const float scale2 = w.a.scale2, ref = m == -__builtin_huge_valf() ? 0.f : m;
    const bool far = beyond_fused(m, scale2);
    auto probabilities = [&](f32x16 (&s)[2], int t) {
        tile_scores<HDP>(s, w.keys(0), T::row_lane(here(w.lane)), qf, [](int) {});
        mask_scores(s, w, t);
#pragma unroll
        for (int rb = 0; rb < 2; ++rb)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[rb][i] = __builtin_amdgcn_exp2f(far ? (s[rb][i] - ref) * scale2 : __builtin_fmaf(s[rb][i], scale2, -(ref * scale2)));
    };
    if (sums) {
        float sum = 0.f;
        careful_walk(w, [&](int t) {
            f32x16 s[2];
            probabilities(s, t);
#pragma unroll
            for (int rb = 0; rb < 2; ++rb)
#pragma unroll
                for (int i = 0; i < 16; ++i) sum += s[rb][i];
        });
        l = halves_sum(sum);
        if (w.valid() && w.lane < 32) w.a.lse[w.statistic()] = row_lse(m, l, w.a.scale, scale2);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint32_t fold = 0x7F807F80u;
#pragma nounroll
    for (int db = 0; db < W::kDims; ++db) {
        f32x16 one = zero16();
        careful_walk(w, [&](int t) {
            f32x16 s[2];
            probabilities(s, t);
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[rb][i] *= inv;
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    one = careful_product(T::cols(w.values(0), T::cols_lane(here(w.lane)), db, 2 * rb + u), operand(s[rb], u), w.counted(t, rb, u), one);
            }
        });
        fold = store_columns(w.out_row(), one, db, 1.f, w.lane, w.a.head_dim, w.valid(), fold);
    }
    return fold;
}

// Up to 64 dimensions four waves a SIMD, in 128 registers for the 129 that three would take: window 1 x 8192 60.3 -> 56.4 us, 16 x 512
// 20.3 -> 17.5, but 8 x 1024, in one round of workgroups either way, 26.4 -> 27.0, and 1 x 8192 144.9 -> 146.4.  (The queries' backward
// pass spills vector registers at four.)
template <int HDP, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, HDP == 64 ? 4 : 2) void attention_forward_kernel(AttentionArgs a) {
    typedef QueryBlock<HDP, WAVES> W;
    typedef typename W::T T;
    __shared__ __attribute__((aligned(16))) char lds[W::kLdsBytes];
    W w(a, lds);
    bf16x8 qf[W::kSteps];
    w.load_rows(qf, w.base, w.token);   // its latency covers what follows
    w.begin();
    arrived(qf);

    f32x16 o[W::kDims], s[2];
    float m = -__builtin_huge_valf(), sum[2] = {0.f, 0.f};
#pragma unroll
    for (int db = 0; db < W::kDims; ++db) o[db] = zero16();
    const int row_lane_ = T::row_lane(w.lane), cols_lane_ = T::cols_lane(w.lane);

    int t = w.pass(w.t_lo, w.w_lo);
#pragma nounroll
    for (; t <= w.w_hi; ++t) {
        copies_landed();
        const char* keys = w.keys(t & 1);
        char* values = w.values(t & 1);
        w.aim((t + 1) & 1, t + 1);
        matrix_priority<HDP, 1>();
        tile_scores<HDP>(s, keys, here(row_lane_), qf, [&](int st) { w.issue(st); });
        matrix_priority<HDP, 0>();
        if (!w.whole(t)) mask_scores(s, w, t);
        float top = -__builtin_huge_valf();
#pragma unroll
        for (int rb = 0; rb < 2; ++rb)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, s[rb][i]);
        top = halves_max(top);
        // The maximum that the exponentials are taken against follows only when one has outgrown it by 2^8: the sums and
        // the 16-bit probabilities lose nothing by a common factor of that size, and the accumulators are rarely rescaled.
        if (__any((top - m) * a.scale2 > 8.f)) {
            const float to = __builtin_fmaxf(m, top);
            const float factor = to == -__builtin_huge_valf() ? 1.f : __builtin_amdgcn_exp2f((m - to) * a.scale2);
            m = to;
            sum[0] *= factor, sum[1] *= factor;
#pragma unroll
            for (int db = 0; db < W::kDims; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[db][i] *= factor;
        }
        const float ref = m == -__builtin_huge_valf() ? 0.f : m * a.scale2;
        bf16x8 pf[4];
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[rb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][i], a.scale2, -ref));
                sum[i & 1] += s[rb][i];
            }
            pf[2 * rb] = operand(s[rb], 0);
            pf[2 * rb + 1] = operand(s[rb], 1);
        }
        const int cols_lane = here(cols_lane_);
        matrix_priority<HDP, 1>();
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int db = 0; db < W::kDims; ++db) o[db] = mfma(T::cols(values, cols_lane, db, u), pf[u], o[db]);
        matrix_priority<HDP, 0>();
    }

    w.pass(t, INT_MAX);

    const float l = halves_sum(sum[0] + sum[1]), inv = l == 0.f ? 0.f : 1.f / l;
    if (w.valid() && w.lane < 32) a.lse[w.statistic()] = row_lse(m, l, a.scale, a.scale2);
    bool fine = true;
#pragma unroll
    for (int db = 0; db < W::kDims; ++db) fine &= all_finite(o[db]);
    uint32_t fold = 0x7F807F80u;
    // Stored before the waves ask each other whether all went well, so that those that are done first do not wait with it (8 x 1024
    // 79.8 -> 77.9 us); the careful form stores over it.
    all_copies_landed();
    uint16_t* row = w.out_row();
    const int lane = here(w.lane);   // its offsets into a row are derived again: kept since the loads they spill (16 x 512 17.5 -> 17.8 us)
#pragma unroll
    for (int db = 0; db < W::kDims; ++db) fold = store_columns(row, o[db], db, inv, lane, a.head_dim, w.valid(), fold);
    const bool far = beyond_fused(m, a.scale2);
    if (__syncthreads_or(!fine || far)) {
        const bool sums = __syncthreads_or(far || !(__builtin_fabsf(l) < __builtin_huge_valf()));
        fold = attention_forward_careful<HDP>(w, qf, m, l, sums);
    }
    if (a.abs_max) {
        const uint32_t x = fold & 0xFFFFu, y = fold >> 16;
        block_min_to_atomic_max(a.abs_max, x < y ? x : y, 0x7F80u, 16);
    }
}

// ---- backward: queries ---------------------------------------------------------------------------------------------------
// dq, with D and the base-2 lse left for the other kernel.  The walk of the forward kernel with a third product:
// transposed, s = K q, dp = V dout, dq = K^T ds.

// ds of 32 keys (row block rb) of a tile as operands, 0 in the places the mask excludes; between(step) after each step.  lse: of base 2
// (fused_lse), or in the careful form the row's own.
template <int HDP, bool CAREFUL, typename Block, typename F>
__device__ __forceinline__ void query_gradient(bf16x8 (&dsf)[2], const Block& w, const char* keys, const char* values, int row_lane, int t, int rb,
                                               bool whole, const bf16x8 (&qf)[HDP / 16], const bf16x8 (&gf)[HDP / 16], float lse, float delta,
                                               F between) {
    typedef Tile<HDP, kKeys> T;
    constexpr int kSteps = HDP / 16;
    f32x16 s = zero16(), dp = zero16();
    bf16x8 kf[kSteps], vf[kSteps];
#pragma unroll
    for (int st = -kAhead; st < kSteps; ++st) {
        if (st + kAhead < kSteps) {
            kf[st + kAhead] = T::rows(keys, row_lane, rb, st + kAhead);
            vf[st + kAhead] = T::rows(values, row_lane, rb, st + kAhead);
        }
        if (st < 0) continue;
        s = mfma(kf[st], qf[st], s);
        dp = mfma(vf[st], gf[st], dp);
        between(st);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float p = __builtin_amdgcn_exp2f(CAREFUL ? exponent(s[i], lse, w.a.scale, w.a.scale2) : __builtin_fmaf(s[i], w.a.scale2, -lse));
        s[i] = p * (dp[i] - delta);
    }
    if (!whole) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = w.allowed(t, rb, i) ? s[i] : 0.f;
    }
    dsf[0] = operand(s, 0);
    dsf[1] = operand(s, 1);
}

template <int HDP, typename W>
__device__ __forceinline__ void attention_backward_q_careful(W& w, const bf16x8 (&qf)[W::kSteps], const bf16x8 (&gf)[W::kSteps], float delta) {
    typedef typename W::T T;
    const float lse = w.a.lse[w.row_statistic()];
#pragma nounroll
    for (int db = 0; db < W::kDims; ++db) {
        f32x16 one = zero16();
        careful_walk(w, [&](int t) {
#pragma nounroll
            for (int rb = 0; rb < 2; ++rb) {
                bf16x8 dsf[2];
                query_gradient<HDP, true>(dsf, w, w.keys(0), w.values(0), T::row_lane(here(w.lane)), t, rb, false, qf, gf, lse, delta, [](int) {});
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    one = careful_product(T::cols(w.keys(0), T::cols_lane(here(w.lane)), db, 2 * rb + u), dsf[u], w.counted(t, rb, u), one);
            }
        });
        store_columns(w.dq_row(), one, db, w.a.scale, w.lane, w.a.head_dim, w.valid(), 0u);
    }
}

template <int HDP, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, 2) void attention_backward_q_kernel(AttentionArgs a) {
    typedef QueryBlock<HDP, WAVES> W;
    typedef typename W::T T;
    __shared__ __attribute__((aligned(16))) char lds[W::kLdsBytes];
    W w(a, lds);
    bf16x8 qf[W::kSteps], gf[W::kSteps];
    float delta, lse2;
    {
        bf16x8 of[W::kSteps];
        const int64_t out_row = (int64_t)a.Nq * a.head_dim;
        w.load_rows(gf, a.dout + (int64_t)w.b * a.T * out_row, out_row);
        w.load_rows(of, a.out + (int64_t)w.b * a.T * out_row, out_row);
        w.load_rows(qf, w.base, w.token);
        lse2 = fused_lse(a.lse[w.row_statistic()]);
        w.begin();
        arrived(gf), arrived(of), arrived(qf);
        float d = 0.f;
#pragma unroll
        for (int s = 0; s < W::kSteps; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) d = __builtin_fmaf((float)gf[s][j], (float)of[s][j], d);
        delta = halves_sum(d);
        const int64_t stat = w.statistic();
        if (w.lane < 32 && w.valid()) {
            a.delta[stat] = delta;
            a.lse2[stat] = lse2;
        }
        // what the wave's rows may look at, for the walk over the queries; one head of the row writes it
        if (a.first_key && w.head == 0 && w.valid() && w.lane == 0)
            a.groups[(int64_t)w.b * ((a.T + 31) / 32) + w.mask.q / 32] = make_int2(w.mask.lo, w.mask.first_max);
    }
    const int row_lane_ = T::row_lane(w.lane), cols_lane_ = T::cols_lane(w.lane);

    f32x16 dq[W::kDims];
#pragma unroll
    for (int db = 0; db < W::kDims; ++db) dq[db] = zero16();
    int t = w.pass(w.t_lo, w.w_lo);
#pragma nounroll
    for (; t <= w.w_hi; ++t) {
        copies_landed();
        char* keys = w.keys(t & 1);
        const char* values = w.values(t & 1);
        w.aim((t + 1) & 1, t + 1);
        const bool whole = w.whole(t);
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
            bf16x8 dsf[2];
            query_gradient<HDP, false>(dsf, w, keys, values, here(row_lane_), t, rb, whole, qf, gf, lse2, delta, [&](int st) {
                if (rb == 0) w.issue(st);
            });
            const int cols_lane = here(cols_lane_);
#pragma unroll
            for (int db = 0; db < W::kDims; ++db)
#pragma unroll
                for (int u = 0; u < 2; ++u) dq[db] = mfma(T::cols(keys, cols_lane, db, 2 * rb + u), dsf[u], dq[db]);
        }
    }
    w.pass(t, INT_MAX);

    bool fine = true;
#pragma unroll
    for (int db = 0; db < W::kDims; ++db) fine &= all_finite(dq[db]);
    all_copies_landed();
    uint16_t* row = w.dq_row();
#pragma unroll
    for (int db = 0; db < W::kDims; ++db) store_columns(row, dq[db], db, a.scale, w.lane, a.head_dim, w.valid(), 0u);
    if (__syncthreads_or(!fine)) attention_backward_q_careful<HDP>(w, qf, gf, delta);
}

// ---- backward: keys and values -------------------------------------------------------------------------------------------
// A wave owns 32 keys (columns) and walks the queries (rows), 32 at a time, of every head of the group: s = Q k, dp = dout v,
// dv = dout^T p, dk = Q^T ds.  The (query tile, head) pairs are walked from the last query back, the heads of a tile one after
// the other, and a workgroup takes every `splits`-th: the workgroups of a group of heads then read the same tiles at about the
// same time, and one die's L2 serves them all.  The accumulators fill half of the 256 registers that two waves per SIMD leave,
// the keys an eighth; the values stay in LDS.
constexpr int kQueries = 32;

template <int HDP, int WAVES>
struct KeyBlock {
    static constexpr int kThreads = WAVES * kWave, kSteps = HDP / 16, kDims = HDP / 32, kBlock = 32 * WAVES;
    typedef Tile<HDP, kQueries> T;
    typedef Tile<HDP, kBlock> V;
    // Pairs between two barriers: two where one workgroup fills the unit's LDS as it is (8 x 1024 320.5 -> 315.5 us), one where three
    // share it (window 1 x 8192 198.5 us, with two 200.1).
    static constexpr int kStage = HDP == 128 ? 2 : 1, kBuffers = 2 * kStage;
    // buffers of a query tile, of an output gradient tile, the values, buffers of lse2, delta and first key
    static constexpr int kValues = 2 * kBuffers * T::kBytes, kStats = kValues + V::kBytes, kLdsBytes = kStats + kBuffers * 3 * kQueries * 4;
    typedef TileCopy<HDP, kQueries, kThreads> Copy;
    static constexpr int kCopies = 2 * Copy::kCopies + 1;
    static_assert(kCopies <= kSteps, "a copy a step");

    const AttentionArgs& a;
    char* lds;
    uint32_t lds_at;
    int tid, lane, wave, b, kvh, kb0, split, splits, k0, k1, ng;
    int2 early;                               // the lane's first entry of the groups
    float* partial;                           // the share's partial sums, or null: the gradients
    int turns;                                // pairs of the share
    int64_t token, stride, ostride;
    const uint16_t* base;
    int key_;
    Copy copy;
    uint32_t qofs[Copy::kCopies], gofs[Copy::kCopies], sofs;
    int head_, tile_;                         // of the pair that is being copied
    bool clamped;
    const char *qnext, *gnext, *snext;        // its sources
    int head_step, tile_step;                 // `splits` in heads and tiles
    int64_t qstep, gstep, sstep, qcarry, gcarry, scarry;   // what that moves the sources, and a carry from the heads besides
    uint32_t to, sto;                         // and destinations
    uint64_t slanes;

    // Keys `first` .. of the batch row and head `group`, share `share` of `shares`.
    __device__ __forceinline__ KeyBlock(const AttentionArgs& args, char* lds_, int group, int first, int share, int shares)
        : a(args), lds(lds_), copy(threadIdx.x, args.head_dim) {
        tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
        lds_at = lds_address(lds) + wave * 1024;
        b = group / a.Nkv, kvh = group % a.Nkv, kb0 = first, split = share, splits = shares;
        partial = splits > 1 ? a.partial + (int64_t)split * a.B * a.T * a.Nkv * 2 * a.head_dim : nullptr;
        k0 = kb0 + wave * 32, k1 = min(k0 + 32, a.T) - 1;
        key_ = k0 + (lane & 31);
        token = (int64_t)(a.Nq + 2 * a.Nkv) * a.head_dim, stride = token * 2, ostride = (int64_t)a.Nq * a.head_dim * 2;
        base = a.qkv + b * a.T * token;
        ng = (a.T + 31) / 32;
        early = make_int2(INT_MAX, 0);
        if (a.first_key && kb0 / kQueries + tid < ng) early = a.groups[(int64_t)b * ng + kb0 / kQueries + tid];   // before the keys
    }
    // The pairs that look at the keys, and the copies of the values.  lse: what gradient() takes for the rows' lse.
    __device__ __forceinline__ void begin(const float* lse) {
        const int kb1 = min(kb0 + kBlock, a.T) - 1;
        if (a.head_dim < HDP) {
#pragma unroll
            for (int i = 0; i < 2 * kBuffers; ++i) T::template clear<kThreads>(lds + i * T::kBytes, tid);
            V::template clear<kThreads>(lds + kValues, tid);
            __syncthreads();
        }
        // the query tiles that look at any of the workgroup's keys lie in [t_lo, t_hi]
        int t_lo = kb0 / kQueries, t_hi = ng - 1;
        if (a.first_key) {
            int l = INT_MAX, h = -1;
            for (int g = t_lo + tid; g < ng; g += kThreads)
                if ((g == t_lo + tid ? early : a.groups[(int64_t)b * ng + g]).x <= kb1) {
                    l = min(l, g);
                    h = max(h, g);
                }
            block_range<WAVES>(l, h, wave_min(l), wave_max(h));
            t_lo = l <= h ? l : 1;
            t_hi = l <= h ? h : 0;
        }
        const int64_t pairs = (int64_t)max(t_hi - t_lo + 1, 0) * a.G;
        turns = pairs > split ? (int)((pairs - split + splits - 1) / splits) : 0;
        tile_ = t_hi - split / a.G, head_ = split % a.G;
        head_step = splits % a.G, tile_step = splits / a.G;
        clamped = true;
        const int64_t head = kvh * a.G + head_, q0 = (int64_t)tile_ * kQueries, row = ((int64_t)b * a.Nq + head) * a.T;
        qnext = reinterpret_cast<const char*>(base + head * a.head_dim) + q0 * stride;
        gnext = reinterpret_cast<const char*>(a.dout + ((int64_t)b * a.T * a.Nq + head) * a.head_dim) + q0 * ostride;
        snext = wave == 0 ? reinterpret_cast<const char*>(lse + row + q0)
                : wave == 1 || !a.first_key ? reinterpret_cast<const char*>(a.delta + row + q0)
                                            : reinterpret_cast<const char*>(a.first_key + (int64_t)b * a.T + q0);
        const int64_t dim = a.head_dim * 2, shead = wave == 2 && a.first_key ? 0 : (int64_t)a.T * 4;
        qcarry = -a.G * dim - kQueries * stride, gcarry = -a.G * dim - kQueries * ostride, scarry = -a.G * shead - kQueries * 4;
        qstep = head_step * dim - tile_step * kQueries * stride, gstep = head_step * dim - tile_step * kQueries * ostride;
        sstep = head_step * shead - tile_step * kQueries * 4;
        slanes = wave < 3 ? 0xFFFFFFFFull : 0;
        if (turns > 0) {
            typedef TileCopy<HDP, kBlock, kThreads> ValueCopy;
            const ValueCopy vcopy(tid, a.head_dim);
            uint32_t vofs[ValueCopy::kCopies];
            vcopy.offsets(vofs, stride, kb0, a.T);
            const char* v = reinterpret_cast<const char*>(base + (int64_t)(a.Nq + a.Nkv + kvh) * a.head_dim) + kb0 * stride;
#pragma unroll
            for (int i = 0; i < ValueCopy::kCopies; ++i) vcopy.copy(i, lds_at + kValues, vofs, v);
        }
    }
    __device__ __forceinline__ void load_keys(bf16x8 (&kf)[kSteps]) const {
        load_columns<HDP>(kf, base + min(key_, a.T - 1) * token + (int64_t)(a.Nq + kvh) * a.head_dim, lane, a.head_dim);
    }
    __device__ __forceinline__ char* queries(int buf) const { return lds + buf * T::kBytes; }
    __device__ __forceinline__ char* gradients(int buf) const { return lds + (kBuffers + buf) * T::kBytes; }
    __device__ __forceinline__ const char* statistics(int buf, int which) const { return lds + kStats + (buf * 3 + which) * kQueries * 4; }
    // The first query of a pair and what its queries may look at.
    struct Pair {
        int q0;
        int2 group;
    };
    __device__ __forceinline__ Pair aimed() const {
        Pair p;
        p.q0 = tile_ * kQueries;
        p.group = make_int2(0, 0);
        if (a.first_key) p.group = a.groups[(int64_t)b * ng + tile_];
        return p;
    }
    // copies of the pair into `buf`, one by one
    __device__ __forceinline__ void aim(int buf) {
        const int q0 = tile_ * kQueries;
        if (clamped) {   // the last tile of the sequence comes first
            copy.offsets(qofs, stride, q0, a.T);
            copy.offsets(gofs, ostride, q0, a.T);
            sofs = min(lane & 31, a.T - 1 - q0) * 4;
            clamped = q0 + kQueries > a.T;
        }
        to = lds_at + buf * T::kBytes;
        sto = lds_at - wave * 1024 + kStats + (buf * 3 + min(wave, 2)) * kQueries * 4;
    }
    // on to the next pair; behind the last one it stays
    __device__ __forceinline__ void advance(bool more) {
        if (!more) return;
        head_ += head_step, tile_ -= tile_step;
        qnext += qstep, gnext += gstep, snext += sstep;
        if (head_ >= a.G) {
            head_ -= a.G, --tile_;
            qnext += qcarry, gnext += gcarry, snext += scarry;
        }
    }
    __device__ __forceinline__ void issue(int i) const {
        if (i < Copy::kCopies) copy.copy(i, to, qofs, qnext);
        else if (i < 2 * Copy::kCopies) copy.copy(i - Copy::kCopies, to + kBuffers * T::kBytes, gofs, gnext);
        else if (i < kCopies) copy4(sto, sofs, snext, slanes);
    }
    __device__ __forceinline__ void issue_all() const {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) issue(i);
    }
    // whether any of the tile's queries looks at one of the wave's keys, and whether all look at all
    __device__ __forceinline__ bool touches(const Pair& p, bool& whole) const {
        const int lo = __builtin_amdgcn_readfirstlane(p.group.x), top = __builtin_amdgcn_readfirstlane(p.group.y);
        whole = p.q0 >= k1 && top <= k0 && p.q0 + kQueries <= a.T;
        return min(p.q0 + kQueries, a.T) - 1 >= k0 && lo <= k1 && k0 < a.T;
    }
    // p and ds of the tile in `buf` as operands.  allowed: which of this lane's 16 rows may look at its key, where not `whole`.
    // One branch around the mask alone: two forms of the step would meet with the accumulators in different registers.  The rows' lse is of
    // base 2 (fused_lse), or in the careful form their own.
    template <bool CAREFUL, typename F>
    __device__ __forceinline__ void gradient(bf16x8 (&pf)[2], bf16x8 (&dsf)[2], uint32_t& allowed, int buf, int q0, bool whole, int row_lane,
                                             const bf16x8 (&kf)[kSteps], F between) const {
        f32x16 s = zero16(), dp = zero16();
        const char* value_rows = lds + kValues + wave * 32 * V::kRowBytes;
        bf16x8 qf[kSteps], gf[kSteps], vf[kSteps];
#pragma unroll
        for (int st = -kAhead; st < kSteps; ++st) {
            if (st + kAhead < kSteps) {
                qf[st + kAhead] = T::rows(queries(buf), row_lane, 0, st + kAhead);
                gf[st + kAhead] = T::rows(gradients(buf), row_lane, 0, st + kAhead);
                vf[st + kAhead] = V::rows(value_rows, row_lane, 0, st + kAhead);
            }
            if (st < 0) continue;
            s = mfma(qf[st], kf[st], s);
            dp = mfma(gf[st], vf[st], dp);
            between(st);
            __builtin_amdgcn_sched_barrier(0);
        }
        const int r0 = tile_row(0, 0, lane) * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4 l4 = *reinterpret_cast<const float4*>(statistics(buf, 0) + r0 + 32 * j);
            const float4 d4 = *reinterpret_cast<const float4*>(statistics(buf, 1) + r0 + 32 * j);
            const float l[4] = {l4.x, l4.y, l4.z, l4.w}, d[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 4 * j + e;
                s[i] = __builtin_amdgcn_exp2f(CAREFUL ? exponent(s[i], l[e], a.scale, a.scale2) : __builtin_fmaf(s[i], a.scale2, -l[e]));
                dp[i] = s[i] * (dp[i] - d[e]);
            }
        }
        allowed = 0xFFFFu;
        if (!whole) {
            const int key = here(key_);
            allowed = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int4 f4 = *reinterpret_cast<const int4*>(statistics(buf, 2) + r0 + 32 * j);
                const int first[4] = {f4.x, f4.y, f4.z, f4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 4 * j + e, q = q0 + tile_row(0, i, lane);
                    const bool in = q >= key && (!a.first_key || key >= first[e]) && q < a.T;
                    allowed |= in ? 1u << i : 0u;
                    s[i] = in ? s[i] : 0.f;
                    dp[i] = in ? dp[i] : 0.f;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            pf[u] = operand(s, u);
            dsf[u] = operand(dp, u);
        }
    }
    // dimensions 32 db ..: the partial sums of a split, or the gradients
    __device__ __forceinline__ void put(int db, const f32x16& dk, const f32x16& dv) const {
        const int key = here(key_);
        const bool valid = key < a.T;
        if (partial) {
            float* row = partial + (((int64_t)b * a.T + key) * a.Nkv + kvh) * 2 * a.head_dim;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * db + 8 * g + 4 * (lane >> 5);
                if (valid && d < a.head_dim) {
                    *reinterpret_cast<float4*>(row + d) = make_float4(dk[4 * g], dk[4 * g + 1], dk[4 * g + 2], dk[4 * g + 3]);
                    *reinterpret_cast<float4*>(row + a.head_dim + d) = make_float4(dv[4 * g], dv[4 * g + 1], dv[4 * g + 2], dv[4 * g + 3]);
                }
            }
        } else {
            uint16_t* row = a.dqkv + ((int64_t)b * a.T + key) * token + (int64_t)(a.Nq + kvh) * a.head_dim;
            store_columns(row, dk, db, a.scale, lane, a.head_dim, valid, 0u);
            store_columns(row + (int64_t)a.Nkv * a.head_dim, dv, db, 1.f, lane, a.head_dim, valid, 0u);
        }
    }
};

template <int HDP, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, 2) void attention_backward_kv_kernel(AttentionArgs a) {
    typedef KeyBlock<HDP, WAVES> W;
    typedef typename W::T T;
    __shared__ __attribute__((aligned(16))) char lds[W::kLdsBytes];
    const int groups = a.B * a.Nkv, rest = blockIdx.x / groups;   // the first keys, with the most queries, first
    W w(a, lds, blockIdx.x % groups, rest / a.splits * W::kBlock, rest % a.splits, a.splits);
    bf16x8 kf[W::kSteps];
    w.load_keys(kf);   // its latency covers what follows
    w.begin(a.lse2);
    typename W::Pair ahead[W::kStage];
    if (w.turns > 0) {
#pragma unroll
        for (int i = 0; i < W::kStage; ++i) {
            if (i > 0) w.advance(i < w.turns);
            ahead[i] = w.aimed();
            w.aim(i);
            w.issue_all();
        }
    }
    arrived(kf);
    const int row_lane_ = T::row_lane(w.lane), cols_lane_ = T::cols_lane(w.lane);

    f32x16 dk[W::kDims], dv[W::kDims];
#pragma unroll
    for (int db = 0; db < W::kDims; ++db) dk[db] = zero16(), dv[db] = zero16();
#pragma nounroll
    for (int turn = 0; turn < w.turns; ++turn) {
        if (turn % W::kStage == 0) copies_landed();
        const int buf = turn % W::kBuffers;
        const typename W::Pair now = ahead[0];
#pragma unroll
        for (int i = 1; i < W::kStage; ++i) ahead[i - 1] = ahead[i];
        w.advance(turn + W::kStage < w.turns);
        ahead[W::kStage - 1] = w.aimed();
        w.aim(buf ^ W::kStage);
        bool whole;
        if (!w.touches(now, whole)) {
            w.issue_all();
            continue;
        }
        bf16x8 pf[2], dsf[2];
        uint32_t allowed;
        matrix_priority<HDP, 1>();
        w.template gradient<false>(pf, dsf, allowed, buf, now.q0, whole, here(row_lane_), kf, [&](int st) { w.issue(st); });
        matrix_priority<HDP, 0>();
        const int cols_lane = here(cols_lane_);
#pragma unroll
        for (int db = 0; db < W::kDims; ++db)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                dv[db] = mfma(T::cols(w.gradients(buf), cols_lane, db, u), pf[u], dv[db]);
                dk[db] = mfma(T::cols(w.queries(buf), cols_lane, db, u), dsf[u], dk[db]);
            }
    }
    bool fine = true;
#pragma unroll
    for (int db = 0; db < W::kDims; ++db) fine &= all_finite(dk[db]) && all_finite(dv[db]);
    all_copies_landed();
#pragma unroll
    for (int db = 0; db < W::kDims; ++db) w.put(db, dk[db], dv[db]);
    const bool again = __syncthreads_or(!fine);
    if (w.tid == 0) a.flags[blockIdx.x] = again;
}

// Share `split` of the elements of keys kb0 ..: a lane takes four values of each split at a time, kFlight such groups of kSplits
// splits on their way at once.
template <int KEYS, int THREADS, int kFlight, int kSplits>
__device__ __forceinline__ void join_splits(const AttentionArgs& a, int group, int kb0, int split) {
    const int per = 2 * a.head_dim / 4, n = min(KEYS, a.T - kb0) * per, step = a.splits * THREADS;
    const int b = group / a.Nkv, kvh = group % a.Nkv;
    const int64_t all = (int64_t)a.B * a.T * a.Nkv * per, token = (int64_t)(a.Nq + 2 * a.Nkv) * a.head_dim;
    const float4* first = reinterpret_cast<const float4*>(a.partial) + (((int64_t)b * a.T + kb0) * a.Nkv + kvh) * per;
    uint16_t* rows = a.dqkv + ((int64_t)b * a.T + kb0) * token + (int64_t)(a.Nq + kvh) * a.head_dim;
    for (int i = split * THREADS + threadIdx.x; i < n; i += kFlight * step) {
        int key[kFlight], at[kFlight];
        const float4* from[kFlight];
        float4 x[kFlight];
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
            const int j = min(i + u * step, n - 1);
            key[u] = j / per, at[u] = j % per;
            from[u] = first + (int64_t)key[u] * a.Nkv * per + at[u];
            x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        for (int s = 0; s < a.splits; s += kSplits) {
            float4 y[kSplits][kFlight];
#pragma unroll
            for (int p = 0; p < kSplits; ++p)
#pragma unroll
                for (int u = 0; u < kFlight; ++u) y[p][u] = from[u][min(s + p, a.splits - 1) * all];
#pragma unroll
            for (int p = 0; p < kSplits; ++p)
                if (s + p < a.splits) {
#pragma unroll
                    for (int u = 0; u < kFlight; ++u) x[u].x += y[p][u].x, x[u].y += y[p][u].y, x[u].z += y[p][u].z, x[u].w += y[p][u].w;
                }
        }
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
            if (i + u * step >= n) break;
            const bool value = 4 * at[u] >= a.head_dim;
            const float f = value ? 1.f : a.scale;
            uint16_t* row = rows + key[u] * token + (value ? (int64_t)(a.Nkv - 1) * a.head_dim : 0) + 4 * at[u];
            *reinterpret_cast<uint2*>(row) = make_uint2(pack_bf16(x[u].x * f, x[u].y * f), pack_bf16(x[u].z * f, x[u].w * f));
        }
    }
}

// What the keys' kernel leaves: the workgroups of a block of keys add its splits' dk and dv in their order and round once, each a
// share of the elements.  Where a sum was not finite, the first of them computes the whole block again in the careful form (in one
// kernel with the loop above, its registers pushed accumulators of that loop out).
template <int HDP, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, 2) void attention_backward_join_kernel(AttentionArgs a) {
    typedef KeyBlock<HDP, WAVES> W;
    typedef typename W::T T;
    const int groups = a.B * a.Nkv, group = blockIdx.x % groups, rest = blockIdx.x / groups;
    const int split = rest % a.splits, kb0 = rest / a.splits * W::kBlock;
    int again = 0;
    for (int s = 0; s < a.splits; ++s) again |= a.flags[(rest - split + s) * groups + group];
    if (!again) {
        // Where a lane has no more than one group, it asks for that group's splits at once: 1 x 40 20.3 -> 18 us, 2 x 129 27.2 -> 25.2,
        // but 8 x 1024, with many groups a lane, 327 -> 340.
        if (a.splits > 1) {
            if (min(W::kBlock, a.T - kb0) * (a.head_dim / 2) <= a.splits * W::kThreads) join_splits<W::kBlock, W::kThreads, 1, 16>(a, group, kb0, split);
            else join_splits<W::kBlock, W::kThreads, 4, 4>(a, group, kb0, split);
        }
        return;
    }
    if (split > 0) return;
    __shared__ __attribute__((aligned(16))) char lds[W::kLdsBytes];
    W start(a, lds, group, kb0, 0, 1);
    start.begin(a.lse);
    bf16x8 kf[W::kSteps];
    start.load_keys(kf);
    arrived(kf);
#pragma nounroll
    for (int db = 0; db < W::kDims; ++db) {
        f32x16 one_k = zero16(), one_v = zero16();
        W w = start;
#pragma nounroll
        for (int turn = 0; turn < w.turns; ++turn) {
            const typename W::Pair now = w.aimed();
            w.aim(0);
            w.issue_all();
            copies_landed();
            bool whole;
            if (w.touches(now, whole)) {
                bf16x8 pf[2], dsf[2];
                uint32_t allowed;
                w.template gradient<true>(pf, dsf, allowed, 0, now.q0, false, T::row_lane(w.lane), kf, [](int) {});
                f32x16 in;
#pragma unroll
                for (int i = 0; i < 16; ++i) in[i] = (allowed >> i & 1) ? 1.f : 0.f;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    one_k = careful_product(T::cols(w.queries(0), T::cols_lane(w.lane), db, u), dsf[u], operand(in, u), one_k);
                    one_v = careful_product(T::cols(w.gradients(0), T::cols_lane(w.lane), db, u), pf[u], operand(in, u), one_v);
                }
            }
            __syncthreads();
            w.advance(turn + 1 < w.turns);
        }
        w.put(db, one_k, one_v);
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------
constexpr int kUnits = 256;   // compute units the splits are sized for: fixed, so that results do not depend on the partition

static int check_shape(const char* what, int B, int T, int Nq, int Nkv, int head_dim) {
    LLMQ_REQUIRE(B >= 0 && T >= 0, "%s: negative dimension", what);
    LLMQ_REQUIRE(Nq > 0 && Nkv > 0 && Nq % Nkv == 0, "%s: the query heads (%d) must be a multiple of the key/value heads (%d)", what, Nq, Nkv);
    LLMQ_REQUIRE(head_dim >= 8 && head_dim <= 128 && head_dim % 8 == 0, "%s: head_dim must be a multiple of 8 from 8 to 128 (got %d)", what, head_dim);
    LLMQ_REQUIRE((int64_t)Nq + 2 * (int64_t)Nkv <= 65536, "%s: too many heads", what);
    LLMQ_REQUIRE(T <= (1 << 30), "%s: sequence too long", what);
    // the grids' threads (512 for 128 positions of a head at most) fit 32 bits
    LLMQ_REQUIRE((int64_t)B * T <= 0x7FFFFFFF && (int64_t)B * Nq <= INT_MAX && (int64_t)B * Nq * ((T + 127) / 128) < (1 << 23),
                 "%s: tensor too large", what);
    return LLMQ_OK;
}

// Keys of a workgroup of the keys' kernel: as many waves as copy a tile of 32 queries with one load a thread.  Above 64 dimensions
// eight, which read the queries half as often as four: 1 x 8192 1925 -> 1640 us, documents 283 -> 214, but 8 x 1024 331 -> 340.
static int kv_block(int head_dim) { return head_dim > 64 ? 256 : 128; }

// Shares of the walk over the queries: enough workgroups for two per compute unit (one per unit: 1 x 8192 2180 us, 8 x 1024 370;
// three: 1710 and 369), each with a pair at least (two: 1 x 40 17 -> 18 us, four: 20.3).
static int kv_splits(int B, int T, int Nq, int Nkv, int keys) {
    const int64_t blocks = (int64_t)B * Nkv * ((T + keys - 1) / keys);
    const int64_t pairs = (int64_t)((T + kQueries - 1) / kQueries) * (Nq / Nkv);
    int64_t s = (2 * kUnits + blocks - 1) / blocks;
    if (s > pairs) s = pairs;
    return (int)(s < 1 ? 1 : s > 16 ? 16 : s);
}

struct BackwardPlan {
    int splits;
    int64_t blocks;                                 // workgroups of the keys' kernel
    int64_t stats, flags, groups, partial, bytes;   // bytes of each of the two statistics, the flags, the groups, the partial sums; all
};
static BackwardPlan backward_plan(int B, int T, int Nq, int Nkv, int head_dim) {
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    BackwardPlan p;
    const int keys = kv_block(head_dim);
    p.splits = kv_splits(B, T, Nq, Nkv, keys);
    p.stats = up((int64_t)B * Nq * T * 4);
    p.blocks = (int64_t)((T + keys - 1) / keys) * B * Nkv * p.splits;
    p.flags = up(p.blocks * 4);
    p.groups = up((int64_t)B * ((T + 31) / 32) * 8);
    p.partial = p.splits > 1 ? up((int64_t)p.splits * B * T * Nkv * 2 * head_dim * 4) : 0;
    p.bytes = 2 * p.stats + p.flags + p.groups + p.partial;
    return p;
}

static AttentionArgs make_args(const uint16_t* qkv, const int* first_key, int B, int T, int Nq, int Nkv, int head_dim, float scale) {
    AttentionArgs a = {};
    a.qkv = qkv, a.first_key = first_key;
    a.B = B, a.T = T, a.Nq = Nq, a.Nkv = Nkv, a.head_dim = head_dim, a.G = Nq / Nkv;
    a.scale = scale, a.scale2 = scale * kLog2e;
    return a;
}

}  // namespace llmq

using namespace llmq;

extern "C" int llmq_attention_forward_bf16(uint16_t* out, float* lse, const uint16_t* qkv, const int* first_key_or_null,
                                           float* abs_max_or_null, float softmax_scale, int B, int T, int Nq, int Nkv, int head_dim,
                                           void* stream) {
    const char* what = "attention_forward";
    if (int rc = check_shape(what, B, T, Nq, Nkv, head_dim)) return rc;
    LLMQ_REQUIRE(softmax_scale > 0.f && softmax_scale < 1e30f, "%s: softmax_scale must be positive and finite", what);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool some = B > 0 && T > 0;
    if (some) {
        LLMQ_REQUIRE(out && lse && qkv, "%s: null tensor pointer", what);
        LLMQ_REQUIRE(aligned16(out) && aligned16(qkv), "%s: pointers must be 16-byte aligned", what);
        const int64_t rows = (int64_t)B * T * head_dim * 2, all = rows * (Nq + 2 * Nkv), stat = (int64_t)B * T * Nq * 4;
        const Range written[] = {{out, rows * Nq}, {lse, stat}, {abs_max_or_null, abs_max_or_null ? 4 : 0}};
        const Range read[] = {{qkv, all}, {first_key_or_null, first_key_or_null ? (int64_t)B * T * 4 : 0}};
        LLMQ_REQUIRE(apart(written, read), "%s: out, lse and abs_max must be memory of their own", what);
    }
    if (abs_max_or_null) {
        hipLaunchKernelGGL(reset_slot_kernel, dim3(1), dim3(1), 0, st, reinterpret_cast<unsigned*>(abs_max_or_null));
        LLMQ_HIP_TRY(hipGetLastError());
    }
    if (!some) return LLMQ_OK;
    AttentionArgs a = make_args(qkv, first_key_or_null, B, T, Nq, Nkv, head_dim, softmax_scale);
    a.out = out, a.lse = lse, a.abs_max = reinterpret_cast<unsigned*>(abs_max_or_null);
    auto launch = [&](auto kernel, int queries, int threads) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((T + queries - 1) / queries) * B * Nq), dim3(threads), 0, st, a);
    };
    if (head_dim > 64) launch(attention_forward_kernel<128, 4>, 128, 256);
    else launch(attention_forward_kernel<64, 4>, 128, 256);
    LLMQ_HIP_TRY(hipGetLastError());
    return LLMQ_OK;
}

extern "C" int64_t llmq_attention_backward_scratch_bytes(int B, int T, int Nq, int Nkv, int head_dim) {
    if (B <= 0 || T <= 0 || check_shape("attention_backward", B, T, Nq, Nkv, head_dim)) return 0;
    return backward_plan(B, T, Nq, Nkv, head_dim).bytes;
}

extern "C" int llmq_attention_backward_bf16(uint16_t* dqkv, const uint16_t* dout, const uint16_t* out, const float* lse,
                                            const uint16_t* qkv, const int* first_key_or_null, void* scratch, size_t scratch_bytes,
                                            float softmax_scale, int B, int T, int Nq, int Nkv, int head_dim, void* stream) {
    const char* what = "attention_backward";
    if (int rc = check_shape(what, B, T, Nq, Nkv, head_dim)) return rc;
    LLMQ_REQUIRE(softmax_scale > 0.f && softmax_scale < 1e30f, "%s: softmax_scale must be positive and finite", what);
    if (B == 0 || T == 0) return LLMQ_OK;
    LLMQ_REQUIRE(dqkv && dout && out && lse && qkv && scratch, "%s: null tensor pointer", what);
    LLMQ_REQUIRE(aligned16(dqkv) && aligned16(dout) && aligned16(out) && aligned16(qkv) && aligned16(scratch),
                 "%s: pointers must be 16-byte aligned", what);
    const int64_t rows = (int64_t)B * T * head_dim * 2, all = rows * (Nq + 2 * Nkv), stat = (int64_t)B * T * Nq * 4;
    const BackwardPlan p = backward_plan(B, T, Nq, Nkv, head_dim);
    LLMQ_REQUIRE(scratch_bytes >= (size_t)p.bytes, "%s: scratch buffer too small (%zu bytes, %lld needed)", what, scratch_bytes, (long long)p.bytes);
    const Range written[] = {{dqkv, all}, {scratch, p.bytes}};
    const Range read[] = {{qkv, all}, {dout, rows * Nq}, {out, rows * Nq}, {lse, stat}, {first_key_or_null, first_key_or_null ? (int64_t)B * T * 4 : 0}};
    LLMQ_REQUIRE(apart(written, read), "%s: dqkv and the scratch must be memory of their own", what);
    hipStream_t st = static_cast<hipStream_t>(stream);
    AttentionArgs a = make_args(qkv, first_key_or_null, B, T, Nq, Nkv, head_dim, softmax_scale);
    a.out = const_cast<uint16_t*>(out), a.lse = const_cast<float*>(lse), a.dout = dout, a.dqkv = dqkv;
    char* s = static_cast<char*>(scratch);
    a.lse2 = reinterpret_cast<float*>(s);
    a.delta = reinterpret_cast<float*>(s + p.stats);
    a.flags = reinterpret_cast<int*>(s + 2 * p.stats);
    a.groups = reinterpret_cast<int2*>(s + 2 * p.stats + p.flags);
    a.partial = p.splits > 1 ? reinterpret_cast<float*>(s + 2 * p.stats + p.flags + p.groups) : nullptr;
    a.splits = p.splits;
    auto launch = [&](auto kernel, int64_t blocks, int threads) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), 0, st, a);
    };
    const int64_t q_blocks = (int64_t)((T + 127) / 128) * B * Nq;
    if (head_dim > 64) {
        launch(attention_backward_q_kernel<128, 4>, q_blocks, 256);
        LLMQ_HIP_TRY(hipGetLastError());
        launch(attention_backward_kv_kernel<128, 8>, p.blocks, 512);
        LLMQ_HIP_TRY(hipGetLastError());
        launch(attention_backward_join_kernel<128, 8>, p.blocks, 512);
    } else {
        launch(attention_backward_q_kernel<64, 4>, q_blocks, 256);
        LLMQ_HIP_TRY(hipGetLastError());
        launch(attention_backward_kv_kernel<64, 4>, p.blocks, 256);
        LLMQ_HIP_TRY(hipGetLastError());
        launch(attention_backward_join_kernel<64, 4>, p.blocks, 256);
    }
    LLMQ_HIP_TRY(hipGetLastError());
    return LLMQ_OK;
}
