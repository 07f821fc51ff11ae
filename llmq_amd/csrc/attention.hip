// Causal attention on the fused QKV tensor for gfx950: forward, and the backward pass that recomputes the probabilities.
//
// qkv is [B, T, Nq + 2 Nkv, head_dim] bf16, the tensor rope_forward writes; query head h reads key/value head h / (Nq / Nkv).
// With the keys query t of row b may look at, A(t) = { k : max(0, first_key[b, t]) <= k <= t } (first_key NULL: 0),
//     s = scale q_t . k_k     lse_t = ln sum_{k in A(t)} exp(s)     p = exp(s - lse_t)     out_t = sum_{k in A(t)} p v_k
// and, with D_t = sum_d dout_t out_t and ds = p (dout_t . v_k - D_t),
//     dq_t = scale sum_k ds k_k      dk_k = scale sum_{h, t} ds q_t      dv_k = sum_{h, t} p dout_t
// (the sums of dk and dv run over the query heads of the group).  first_key expresses packed documents (the document's first
// token), a sliding window (t - w + 1) and padding (any value above t: the row is empty, out 0, lse -inf, no gradient).
// (The reference's own kernels: src/kernels/attention.cu:20,152; its call sites src/models/llama_model.cpp:196-202.)
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
    float* lse2;             // backward scratch: lse in base 2, [B, Nq, T]
    float* delta;            // D, [B, Nq, T]
    int2* groups;            // with first_key: per 32 queries the smallest first key of a row that has any, the largest of all
    float* partial;          // dk, dv of each split: [splits][B, T, Nkv][2][head_dim], or NULL (one split, written to dqkv)
    int B, T, Nq, Nkv, head_dim, G;
    int splits;
    float scale, scale2;     // softmax scale, and times log2 e
};

constexpr int kKeys = 64;    // rows of a staged tile

__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x = min(x, __shfl_xor(x, off, kWave));
    return x;
}
__device__ __forceinline__ int wave_max(int x) { return ~wave_min(~x); }

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// Column-side operand of a wave, straight from global memory: lane -> position l % 32, chunk 2 step + l / 32.
template <int HDP>
__device__ __forceinline__ void load_columns(bf16x8 (&f)[HDP / 16], const uint16_t* row, int lane, int head_dim) {
#pragma unroll
    for (int s = 0; s < HDP / 16; ++s) {
        const int d = 16 * s + 8 * (lane >> 5);
        const uint16_t* p = d < head_dim ? row + d : reinterpret_cast<const uint16_t*>(attention_zeros);
        f[s] = *reinterpret_cast<const bf16x8*>(p);
    }
}

// Stores a transposed result (dimensions by positions) times `factor` as bf16 to `row`, this lane's position: the two lanes
// of a position swap groups of four dimensions, so that each writes 16 bytes.  Returns the abs-max fold.
template <int HDP>
__device__ __forceinline__ uint32_t store_columns(uint16_t* row, const f32x16 (&acc)[HDP / 32], float factor, int lane, int head_dim,
                                                  bool valid, uint32_t fold) {
    const int h = lane >> 5;
#pragma unroll
    for (int db = 0; db < HDP / 32; ++db) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            uint32_t w[2][2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int i = 8 * g + 4 * e;
                w[e][0] = pack_bf16(acc[db][i] * factor, acc[db][i + 1] * factor);
                w[e][1] = pack_bf16(acc[db][i + 2] * factor, acc[db][i + 3] * factor);
            }
            const auto x = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
            const auto y = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
            const int d = db * 32 + 16 * g + 8 * h;
            if (valid && d < head_dim) {
                const uint4 v = make_uint4(x[0], y[0], x[1], y[1]);
                *reinterpret_cast<uint4*>(row + d) = v;
                fold = fold_vec(fold, v);
            }
        }
    }
    return fold;
}

__device__ __forceinline__ bool all_finite(const f32x16& x, float carry = 0.f) {
    float t = carry;
#pragma unroll
    for (int i = 0; i < 16; ++i) t = __builtin_fmaf(x[i], 0.f, t);
    return t == 0.f;
}

// What a wave's 32 NB queries may look at.
template <int NB>
struct QueryMask {
    int q[NB], first[NB];   // this lane's positions and their first keys (INT_MAX: empty)
    int lo, hi;             // smallest first key and largest position of the wave's rows that are not empty (lo > hi: none)
    int first_max, q_min;   // a tile [k0, k1] is whole for the wave if k0 >= first_max and k1 <= q_min

    __device__ __forceinline__ void load(const AttentionArgs& a, int b, int q0, int lane) {
        q_min = q0;
        hi = q0 < a.T ? min(q0 + 32 * NB, a.T) - 1 : -1;
        lo = q0 < a.T ? 0 : INT_MAX;
        first_max = 0;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            q[n] = q0 + 32 * n + (lane & 31);
            first[n] = 0;
        }
        if (a.first_key) {
            int l = INT_MAX, m = 0, top = -1;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                if (q[n] < a.T) {
                    first[n] = max(a.first_key[(int64_t)b * a.T + q[n]], 0);
                    if (first[n] > q[n]) first[n] = INT_MAX;
                    else top = max(top, q[n]);
                    l = min(l, first[n]);
                    m = max(m, first[n]);
                }
            }
            lo = wave_min(l);
            first_max = wave_max(m);
            hi = wave_max(top);
        }
    }
    __device__ __forceinline__ bool touches(int k0, int k1) const { return k0 <= hi && k1 >= lo; }
    __device__ __forceinline__ bool whole(int k0, int k1) const { return k0 >= first_max && k1 <= q_min; }
    __device__ __forceinline__ bool allowed(int n, int k) const { return k <= q[n] && k >= first[n]; }
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
}

__device__ __forceinline__ void copies_landed() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// ---- forward ------------------------------------------------------------------------------------------------------------
// A wave owns 32 NB queries (columns) and walks the keys (rows) in tiles of 64 that the workgroup's waves share in LDS, the next
// tile copied while one is computed.
template <int HDP, int NB, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, NB == 2 && HDP == 128 ? 1 : 2) void attention_forward_kernel(AttentionArgs a) {
    typedef Tile<HDP, kKeys> T;
    constexpr int kThreads = WAVES * kWave, kSteps = HDP / 16, kDims = HDP / 32;
    __shared__ __attribute__((aligned(16))) char lds[2][2][T::kBytes];   // [buffer][key, value]
    const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);

    // Workgroups go to the dies round-robin: the groups of heads that share keys are the fastest index, so that a group
    // stays on one die's L2 where their number allows; the last queries, which have the most keys, come first.
    const int ngroups = a.B * a.Nkv, nq = (a.T + 32 * NB * WAVES - 1) / (32 * NB * WAVES);
    const int grp = blockIdx.x % ngroups, rest = blockIdx.x / ngroups;
    const int b = grp / a.Nkv, kvh = grp % a.Nkv, head = kvh * a.G + rest % a.G;
    const int q0 = (nq - 1 - rest / a.G) * (32 * NB * WAVES) + wave * (32 * NB);

    const int64_t token = (int64_t)(a.Nq + 2 * a.Nkv) * a.head_dim, stride = token * 2;
    const uint16_t* base = a.qkv + b * a.T * token;
    const uint16_t* kbase = base + (int64_t)(a.Nq + kvh) * a.head_dim;
    const auto ksrc = T::template source<kThreads>(kbase, tid, stride, a.head_dim);
    auto vsrc = ksrc;
    vsrc.p += (int64_t)a.Nkv * a.head_dim * 2;

    QueryMask<NB> mask;
    mask.load(a, b, q0, lane);
    int lo, hi;
    block_range<WAVES>(lo, hi, mask.lo, mask.hi);
    const int t_lo = lo / kKeys, t_hi = hi / kKeys;   // lo > hi where no row has a key

    bf16x8 qf[NB][kSteps];
#pragma unroll
    for (int n = 0; n < NB; ++n)
        load_columns<HDP>(qf[n], base + min(mask.q[n], a.T - 1) * token + (int64_t)head * a.head_dim, lane, a.head_dim);
    const int row_lane = T::row_lane(lane), cols_lane = T::cols_lane(lane);

    f32x16 o[NB][kDims];
    float m[NB], sum[NB];
    // A second, careful walk only where the first one ended in a value that is not finite.
#pragma nounroll
    for (int careful = 0;; ++careful) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            m[n] = -__builtin_huge_valf();
            sum[n] = 0.f;
#pragma unroll
            for (int db = 0; db < kDims; ++db) o[n][db] = zero16();
        }
        if (lo <= hi) {
            T::template stage<kThreads>(lds[0][0], ksrc, tid, stride, t_lo * kKeys, a.T);
            T::template stage<kThreads>(lds[0][1], vsrc, tid, stride, t_lo * kKeys, a.T);
            copies_landed();
        }
#pragma nounroll
        for (int t = t_lo; lo <= hi && t <= t_hi; ++t) {
            const int buf = (t - t_lo) & 1, k0 = t * kKeys;
            if (t < t_hi) {
                T::template stage<kThreads>(lds[buf ^ 1][0], ksrc, tid, stride, k0 + kKeys, a.T);
                T::template stage<kThreads>(lds[buf ^ 1][1], vsrc, tid, stride, k0 + kKeys, a.T);
            }
            if (mask.touches(k0, k0 + kKeys - 1)) {
                const bool whole = mask.whole(k0, k0 + kKeys - 1);
                f32x16 s[NB][2];
#pragma unroll
                for (int rb = 0; rb < 2; ++rb) {
#pragma unroll
                    for (int n = 0; n < NB; ++n) s[n][rb] = zero16();
#pragma unroll
                    for (int st = 0; st < kSteps; ++st) {
                        const bf16x8 kf = T::rows(lds[buf][0], row_lane, rb, st);
#pragma unroll
                        for (int n = 0; n < NB; ++n) s[n][rb] = mfma(kf, qf[n][st], s[n][rb]);
                    }
                }
                if (!whole) {
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int rb = 0; rb < 2; ++rb)
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (!mask.allowed(n, k0 + tile_row(rb, i, lane))) s[n][rb][i] = -__builtin_huge_valf();
                }
                bf16x8 pf[NB][4];
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    float top = -__builtin_huge_valf();
#pragma unroll
                    for (int rb = 0; rb < 2; ++rb)
#pragma unroll
                        for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, s[n][rb][i]);
                    top = halves_max(top);
                    // The maximum that the exponentials are taken against follows only when one has outgrown it by 2^8: the
                    // sums and the 16-bit probabilities lose nothing by a common factor of that size, and the accumulators
                    // are rarely rescaled.
                    if (__any((top - m[n]) * a.scale2 > 8.f)) {
                        const float next = __builtin_fmaxf(m[n], top);
                        const float factor = next == -__builtin_huge_valf() ? 1.f : __builtin_amdgcn_exp2f((m[n] - next) * a.scale2);
                        m[n] = next;
                        sum[n] *= factor;
#pragma unroll
                        for (int db = 0; db < kDims; ++db)
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[n][db][i] *= factor;
                    }
                    const float ref = m[n] == -__builtin_huge_valf() ? 0.f : m[n] * a.scale2;
#pragma unroll
                    for (int rb = 0; rb < 2; ++rb) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            s[n][rb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][rb][i], a.scale2, -ref));
                            sum[n] += s[n][rb][i];
                        }
                        pf[n][2 * rb] = operand(s[n][rb], 0);
                        pf[n][2 * rb + 1] = operand(s[n][rb], 1);
                    }
                }
                if (careful == 0 || whole) {
#pragma unroll
                    for (int db = 0; db < kDims; ++db)
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const bf16x8 vf = T::cols(lds[buf][1], cols_lane, db, u);
#pragma unroll
                            for (int n = 0; n < NB; ++n) o[n][db] = mfma(vf, pf[n][u], o[n][db]);
                        }
                } else {
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            f32x16 one;
#pragma unroll
                            for (int i = 0; i < 16; ++i) one[i] = mask.allowed(n, k0 + tile_row(u / 2, i, lane)) ? 1.f : 0.f;
                            const bf16x8 counts = operand(one, u & 1);
#pragma unroll
                            for (int db = 0; db < kDims; ++db)
                                o[n][db] = careful_product(T::cols(lds[buf][1], cols_lane, db, u), pf[n][u], counts, o[n][db]);
                        }
                }
            }
            copies_landed();
        }
        if (careful) break;
        bool fine = true;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int db = 0; db < kDims; ++db) fine &= all_finite(o[n][db]);
        if (!__syncthreads_or(!fine)) break;
    }

    uint32_t fold = 0x7F807F80u;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const float l = halves_sum(sum[n]);
        const bool valid = mask.q[n] < a.T;
        const float factor = l == 0.f ? 0.f : 1.f / l;
        fold = store_columns<HDP>(a.out + ((int64_t)b * a.T + mask.q[n]) * a.Nq * a.head_dim + (int64_t)head * a.head_dim, o[n], factor,
                                  lane, a.head_dim, valid, fold);
        if (valid && lane < 32)
            a.lse[((int64_t)b * a.Nq + head) * a.T + mask.q[n]] =
                m[n] == -__builtin_huge_valf() && l == 0.f ? m[n] : (m[n] * a.scale2 + __builtin_amdgcn_logf(l)) * kLn2;
    }
    if (a.abs_max) {
        const uint32_t x = fold & 0xFFFFu, y = fold >> 16;
        block_min_to_atomic_max(a.abs_max, x < y ? x : y, 0x7F80u, 16);
    }
}

// ---- backward: queries ---------------------------------------------------------------------------------------------------
// dq, with D and the base-2 lse left for the other kernel.  The walk of the forward kernel with a third product:
// transposed, s = K q, dp = V dout, dq = K^T ds.
template <int HDP, int NB, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, NB == 2 && HDP == 128 ? 1 : 2) void attention_backward_q_kernel(AttentionArgs a) {
    typedef Tile<HDP, kKeys> T;
    constexpr int kThreads = WAVES * kWave, kSteps = HDP / 16, kDims = HDP / 32;
    __shared__ __attribute__((aligned(16))) char lds[2][2][T::kBytes];
    const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);

    const int ngroups = a.B * a.Nkv, nq = (a.T + 32 * NB * WAVES - 1) / (32 * NB * WAVES);
    const int grp = blockIdx.x % ngroups, rest = blockIdx.x / ngroups;
    const int b = grp / a.Nkv, kvh = grp % a.Nkv, head = kvh * a.G + rest % a.G;
    const int q0 = (nq - 1 - rest / a.G) * (32 * NB * WAVES) + wave * (32 * NB);

    const int64_t token = (int64_t)(a.Nq + 2 * a.Nkv) * a.head_dim, stride = token * 2;
    const uint16_t* base = a.qkv + b * a.T * token;
    const uint16_t* kbase = base + (int64_t)(a.Nq + kvh) * a.head_dim;
    const auto ksrc = T::template source<kThreads>(kbase, tid, stride, a.head_dim);
    auto vsrc = ksrc;
    vsrc.p += (int64_t)a.Nkv * a.head_dim * 2;

    QueryMask<NB> mask;
    mask.load(a, b, q0, lane);
    int lo, hi;
    block_range<WAVES>(lo, hi, mask.lo, mask.hi);
    const int t_lo = lo / kKeys, t_hi = hi / kKeys;

    bf16x8 qf[NB][kSteps], gf[NB][kSteps];
    float lse2[NB], delta[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const int q = min(mask.q[n], a.T - 1);
        const int64_t at = ((int64_t)b * a.T + q) * a.Nq * a.head_dim + (int64_t)head * a.head_dim;
        load_columns<HDP>(qf[n], base + q * token + (int64_t)head * a.head_dim, lane, a.head_dim);
        load_columns<HDP>(gf[n], a.dout + at, lane, a.head_dim);
        bf16x8 of[kSteps];
        load_columns<HDP>(of, a.out + at, lane, a.head_dim);
        float d = 0.f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) d = __builtin_fmaf((float)gf[n][s][j], (float)of[s][j], d);
        delta[n] = halves_sum(d);
        const int64_t stat = ((int64_t)b * a.Nq + head) * a.T;
        lse2[n] = a.lse[stat + q] * kLog2e;
        if (lane < 32 && mask.q[n] < a.T) {
            a.delta[stat + q] = delta[n];
            a.lse2[stat + q] = lse2[n];
        }
        // what the rows of this group may look at, for the walk over the queries; one head of the row writes it
        if (a.first_key && head == 0) {
            const bool in = mask.q[n] < a.T;
            const int l = wave_min(in ? mask.first[n] : INT_MAX), f = wave_max(in ? mask.first[n] : 0);
            const int g = (q0 >> 5) + n, ng = (a.T + 31) / 32;
            if (lane == 0 && g < ng) a.groups[(int64_t)b * ng + g] = make_int2(l, f);
        }
    }
    const int row_lane = T::row_lane(lane), cols_lane = T::cols_lane(lane);

    f32x16 dq[NB][kDims];
#pragma nounroll
    for (int careful = 0;; ++careful) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int db = 0; db < kDims; ++db) dq[n][db] = zero16();
        if (lo <= hi) {
            T::template stage<kThreads>(lds[0][0], ksrc, tid, stride, t_lo * kKeys, a.T);
            T::template stage<kThreads>(lds[0][1], vsrc, tid, stride, t_lo * kKeys, a.T);
            copies_landed();
        }
#pragma nounroll
        for (int t = t_lo; lo <= hi && t <= t_hi; ++t) {
            const int buf = (t - t_lo) & 1, k0 = t * kKeys;
            if (t < t_hi) {
                T::template stage<kThreads>(lds[buf ^ 1][0], ksrc, tid, stride, k0 + kKeys, a.T);
                T::template stage<kThreads>(lds[buf ^ 1][1], vsrc, tid, stride, k0 + kKeys, a.T);
            }
            if (mask.touches(k0, k0 + kKeys - 1)) {
                const bool whole = mask.whole(k0, k0 + kKeys - 1);
#pragma unroll
                for (int rb = 0; rb < 2; ++rb) {
                    f32x16 s[NB], dp[NB];
#pragma unroll
                    for (int n = 0; n < NB; ++n) s[n] = zero16(), dp[n] = zero16();
#pragma unroll
                    for (int st = 0; st < kSteps; ++st) {
                        const bf16x8 kf = T::rows(lds[buf][0], row_lane, rb, st), vf = T::rows(lds[buf][1], row_lane, rb, st);
#pragma unroll
                        for (int n = 0; n < NB; ++n) {
                            s[n] = mfma(kf, qf[n][st], s[n]);
                            dp[n] = mfma(vf, gf[n][st], dp[n]);
                        }
                    }
                    bf16x8 dsf[NB][2];
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i], a.scale2, -lse2[n]));
                            s[n][i] = p * (dp[n][i] - delta[n]);
                        }
                        if (!whole) {
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (!mask.allowed(n, k0 + tile_row(rb, i, lane))) s[n][i] = 0.f;
                        }
                        dsf[n][0] = operand(s[n], 0);
                        dsf[n][1] = operand(s[n], 1);
                    }
                    if (careful == 0 || whole) {
#pragma unroll
                        for (int db = 0; db < kDims; ++db)
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                const bf16x8 kf = T::cols(lds[buf][0], cols_lane, db, 2 * rb + u);
#pragma unroll
                                for (int n = 0; n < NB; ++n) dq[n][db] = mfma(kf, dsf[n][u], dq[n][db]);
                            }
                    } else {
#pragma unroll
                        for (int n = 0; n < NB; ++n)
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                f32x16 one;
#pragma unroll
                                for (int i = 0; i < 16; ++i) one[i] = mask.allowed(n, k0 + tile_row(rb, i, lane)) ? 1.f : 0.f;
                                const bf16x8 counts = operand(one, u);
#pragma unroll
                                for (int db = 0; db < kDims; ++db)
                                    dq[n][db] = careful_product(T::cols(lds[buf][0], cols_lane, db, 2 * rb + u), dsf[n][u], counts,
                                                                dq[n][db]);
                            }
                    }
                }
            }
            copies_landed();
        }
        if (careful) break;
        bool fine = true;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int db = 0; db < kDims; ++db) fine &= all_finite(dq[n][db]);
        if (!__syncthreads_or(!fine)) break;
    }
#pragma unroll
    for (int n = 0; n < NB; ++n)
        store_columns<HDP>(a.dqkv + (b * a.T + (int64_t)mask.q[n]) * token + (int64_t)head * a.head_dim, dq[n], a.scale, lane, a.head_dim,
                           mask.q[n] < a.T, 0u);
}

// ---- backward: keys and values -------------------------------------------------------------------------------------------
// A wave owns 32 NB keys (columns) and walks the queries (rows) of every head of the group: s = Q k, dp = dout v,
// dv = dout^T p, dk = Q^T ds.  A workgroup takes one of `splits` equal shares of the (head, query tile) pairs of its keys.
template <int HDP, int NB, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, HDP == 128 ? 1 : 2) void attention_backward_kv_kernel(AttentionArgs a) {
    typedef Tile<HDP, kKeys> T;
    constexpr int kThreads = WAVES * kWave, kSteps = HDP / 16, kDims = HDP / 32, kBlock = 32 * NB * WAVES;
    __shared__ __attribute__((aligned(16))) char lds[2][2][T::kBytes];      // [buffer][query, output gradient]
    __shared__ __attribute__((aligned(16))) float stats[2][2][kKeys];       // [buffer][lse2, delta]
    const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);

    const int ngroups = a.B * a.Nkv;
    const int grp = blockIdx.x % ngroups, rest = blockIdx.x / ngroups;
    const int b = grp / a.Nkv, kvh = grp % a.Nkv, split = rest % a.splits, kt = rest / a.splits;   // the first keys have the most queries
    const int kb0 = kt * kBlock, k0 = kb0 + wave * (32 * NB);
    const int kb1 = min(kb0 + kBlock, a.T) - 1, k1 = min(k0 + 32 * NB, a.T) - 1;

    const int64_t token = (int64_t)(a.Nq + 2 * a.Nkv) * a.head_dim, stride = token * 2, ostride = (int64_t)a.Nq * a.head_dim * 2;
    const uint16_t* base = a.qkv + b * a.T * token;

    // the query tiles that look at any of the workgroup's keys lie in [t_lo, t_hi]
    const int ng = (a.T + 31) / 32;
    int t_lo = kb0 / kKeys, t_hi = (a.T - 1) / kKeys;
    if (a.first_key) {
        int l = INT_MAX, h = -1;
        for (int g = kb0 / 32 + tid; g < ng; g += kThreads)
            if (a.groups[(int64_t)b * ng + g].x <= kb1) {
                l = min(l, g);
                h = max(h, g);
            }
        block_range<WAVES>(l, h, wave_min(l), wave_max(h));
        t_lo = l <= h ? l / (kKeys / 32) : 1;
        t_hi = l <= h ? h / (kKeys / 32) : 0;
    }
    const int tiles = max(t_hi - t_lo + 1, 0);
    const int64_t pairs = (int64_t)tiles * a.G;
    const int first_pair = (int)(pairs * split / a.splits), last_pair = (int)(pairs * (split + 1) / a.splits);

    bf16x8 kf[NB][kSteps], vf[NB][kSteps];
    int key[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        key[n] = k0 + 32 * n + (lane & 31);
        const uint16_t* row = base + min(key[n], a.T - 1) * token + (int64_t)(a.Nq + kvh) * a.head_dim;
        load_columns<HDP>(kf[n], row, lane, a.head_dim);
        load_columns<HDP>(vf[n], row + (int64_t)a.Nkv * a.head_dim, lane, a.head_dim);
    }
    const int row_lane = T::row_lane(lane), cols_lane = T::cols_lane(lane);

    auto qsrc = T::template source<kThreads>(base, tid, stride, a.head_dim);
    auto gsrc = T::template source<kThreads>(a.dout + (int64_t)b * a.T * a.Nq * a.head_dim, tid, ostride, a.head_dim);
    auto stage = [&](int buf, int pair) {
        const int head = kvh * a.G + pair / tiles, q0 = (t_lo + pair % tiles) * kKeys;
        auto q = qsrc, g = gsrc;
        q.p += (int64_t)head * a.head_dim * 2;
        g.p += (int64_t)head * a.head_dim * 2;
        T::template stage<kThreads>(lds[buf][0], q, tid, stride, q0, a.T);
        T::template stage<kThreads>(lds[buf][1], g, tid, ostride, q0, a.T);
        if (wave < 2) {
            const float* src = (wave == 0 ? a.lse2 : a.delta) + ((int64_t)b * a.Nq + head) * a.T + q0 + lane;
            if (q0 + lane >= a.T) src = reinterpret_cast<const float*>(attention_zeros);
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                             (__attribute__((address_space(3))) void*)stats[buf][wave], 4, 0, 0);
        }
    };

    f32x16 dk[NB][kDims], dv[NB][kDims];
#pragma nounroll
    for (int careful = 0;; ++careful) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int db = 0; db < kDims; ++db) dk[n][db] = zero16(), dv[n][db] = zero16();
        if (first_pair < last_pair) {
            stage(0, first_pair);
            copies_landed();
        }
#pragma nounroll
        for (int pair = first_pair; pair < last_pair; ++pair) {
            const int buf = (pair - first_pair) & 1, q0 = (t_lo + pair % tiles) * kKeys;
            if (pair + 1 < last_pair) stage(buf ^ 1, pair + 1);
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) {
                const int r0 = q0 + 32 * rb, r1 = min(r0 + 32, a.T) - 1;
                int2 g = make_int2(0, 0);
                if (a.first_key && r0 < a.T) g = a.groups[(int64_t)b * ng + (r0 >> 5)];
                if (r0 >= a.T || r1 < k0 || g.x > k1 || k0 >= a.T) continue;
                const bool whole = r0 >= k1 && g.y <= k0;
                f32x16 s[NB], dp[NB];
#pragma unroll
                for (int n = 0; n < NB; ++n) s[n] = zero16(), dp[n] = zero16();
#pragma unroll
                for (int st = 0; st < kSteps; ++st) {
                    const bf16x8 qf = T::rows(lds[buf][0], row_lane, rb, st), gf = T::rows(lds[buf][1], row_lane, rb, st);
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        s[n] = mfma(qf, kf[n][st], s[n]);
                        dp[n] = mfma(gf, vf[n][st], dp[n]);
                    }
                }
                float4 l4[4], d4[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    l4[j] = *reinterpret_cast<const float4*>(&stats[buf][0][tile_row(rb, 4 * j, lane)]);
                    d4[j] = *reinterpret_cast<const float4*>(&stats[buf][1][tile_row(rb, 4 * j, lane)]);
                }
                uint32_t counts = 0xFFFFu;   // which of this lane's 16 rows may look at its key, for each block of keys
                bf16x8 pf[NB][2], dsf[NB][2];
                uint32_t allowed[NB];
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    allowed[n] = counts;
                    if (!whole) {
                        allowed[n] = 0;
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int q = q0 + tile_row(rb, i, lane);
                            const int first = a.first_key && q < a.T ? a.first_key[(int64_t)b * a.T + q] : 0;
                            if (q >= key[n] && key[n] >= first && q < a.T) allowed[n] |= 1u << i;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float l = i % 4 == 0 ? l4[i / 4].x : i % 4 == 1 ? l4[i / 4].y : i % 4 == 2 ? l4[i / 4].z : l4[i / 4].w;
                        const float d = i % 4 == 0 ? d4[i / 4].x : i % 4 == 1 ? d4[i / 4].y : i % 4 == 2 ? d4[i / 4].z : d4[i / 4].w;
                        s[n][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i], a.scale2, -l));
                        dp[n][i] = s[n][i] * (dp[n][i] - d);
                    }
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (!(allowed[n] >> i & 1)) s[n][i] = 0.f, dp[n][i] = 0.f;
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        pf[n][u] = operand(s[n], u);
                        dsf[n][u] = operand(dp[n], u);
                    }
                }
                if (careful == 0 || whole) {
#pragma unroll
                    for (int db = 0; db < kDims; ++db)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const bf16x8 gt = T::cols(lds[buf][1], cols_lane, db, 2 * rb + u);
                            const bf16x8 qt = T::cols(lds[buf][0], cols_lane, db, 2 * rb + u);
#pragma unroll
                            for (int n = 0; n < NB; ++n) {
                                dv[n][db] = mfma(gt, pf[n][u], dv[n][db]);
                                dk[n][db] = mfma(qt, dsf[n][u], dk[n][db]);
                            }
                        }
                } else {
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            f32x16 one;
#pragma unroll
                            for (int i = 0; i < 16; ++i) one[i] = (allowed[n] >> i & 1) ? 1.f : 0.f;
                            const bf16x8 ones = operand(one, u);
#pragma unroll
                            for (int db = 0; db < kDims; ++db) {
                                dv[n][db] = careful_product(T::cols(lds[buf][1], cols_lane, db, 2 * rb + u), pf[n][u], ones, dv[n][db]);
                                dk[n][db] = careful_product(T::cols(lds[buf][0], cols_lane, db, 2 * rb + u), dsf[n][u], ones, dk[n][db]);
                            }
                        }
                }
            }
            copies_landed();
        }
        if (careful) break;
        bool fine = true;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int db = 0; db < kDims; ++db) fine &= all_finite(dk[n][db]) && all_finite(dv[n][db]);
        if (!__syncthreads_or(!fine)) break;
    }

#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const bool valid = key[n] < a.T;
        if (a.partial) {
            float* row = a.partial + ((((int64_t)split * a.B + b) * a.T + key[n]) * a.Nkv + kvh) * 2 * a.head_dim;
#pragma unroll
            for (int db = 0; db < kDims; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d = 32 * db + 8 * g + 4 * (lane >> 5);
                    if (valid && d < a.head_dim) {
                        *reinterpret_cast<float4*>(row + d) =
                            make_float4(dk[n][db][4 * g], dk[n][db][4 * g + 1], dk[n][db][4 * g + 2], dk[n][db][4 * g + 3]);
                        *reinterpret_cast<float4*>(row + a.head_dim + d) =
                            make_float4(dv[n][db][4 * g], dv[n][db][4 * g + 1], dv[n][db][4 * g + 2], dv[n][db][4 * g + 3]);
                    }
                }
        } else {
            uint16_t* row = a.dqkv + ((int64_t)b * a.T + key[n]) * token + (int64_t)(a.Nq + kvh) * a.head_dim;
            store_columns<HDP>(row, dk[n], a.scale, lane, a.head_dim, valid, 0u);
            store_columns<HDP>(row + (int64_t)a.Nkv * a.head_dim, dv[n], 1.f, lane, a.head_dim, valid, 0u);
        }
    }
}

// Adds the splits' dk and dv in their order and rounds once.  A lane takes four values.
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs a) {
    const int per = 2 * a.head_dim / 4;
    const int64_t n = (int64_t)a.B * a.T * a.Nkv * per, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int at = (int)(i % per) * 4, kvh = (int)(i / per % a.Nkv);
    const int64_t bt = i / per / a.Nkv;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < a.splits; ++s) {
        const float4 y = reinterpret_cast<const float4*>(a.partial)[s * n + i];
        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
    }
    const bool value = at >= a.head_dim;
    const float f = value ? 1.f : a.scale;
    const int64_t token = (int64_t)(a.Nq + 2 * a.Nkv) * a.head_dim;
    uint16_t* row = a.dqkv + bt * token + (int64_t)(a.Nq + kvh + (value ? a.Nkv : 0)) * a.head_dim + (value ? at - a.head_dim : at);
    *reinterpret_cast<uint2*>(row) = make_uint2(pack_bf16(x.x * f, x.y * f), pack_bf16(x.z * f, x.w * f));
}

// ---- host ----------------------------------------------------------------------------------------------------------------
constexpr int kUnits = 256;   // compute units the splits are sized for: fixed, so that results do not depend on the partition

static int check_shape(const char* what, int B, int T, int Nq, int Nkv, int head_dim) {
    LLMQ_REQUIRE(B >= 0 && T >= 0, "%s: negative dimension", what);
    LLMQ_REQUIRE(Nq > 0 && Nkv > 0 && Nq % Nkv == 0, "%s: the query heads (%d) must be a multiple of the key/value heads (%d)", what, Nq, Nkv);
    LLMQ_REQUIRE(head_dim >= 8 && head_dim <= 128 && head_dim % 8 == 0, "%s: head_dim must be a multiple of 8 from 8 to 128 (got %d)", what, head_dim);
    LLMQ_REQUIRE((int64_t)Nq + 2 * (int64_t)Nkv <= 65536, "%s: too many heads", what);
    LLMQ_REQUIRE(T <= (1 << 30), "%s: sequence too long", what);
    LLMQ_REQUIRE((int64_t)B * T <= 0x7FFFFFFF && (int64_t)B * Nq * (((int64_t)T + 31) / 32) <= 0x7FFFFFFF, "%s: tensor too large", what);
    return LLMQ_OK;
}

// Shares of the walk over the queries: enough workgroups for two per compute unit, each with some tiles of work.
static int kv_splits(int B, int T, int Nq, int Nkv, int keys) {
    const int64_t blocks = (int64_t)B * Nkv * ((T + keys - 1) / keys);
    const int64_t pairs = (int64_t)((T + kKeys - 1) / kKeys) * (Nq / Nkv);
    int64_t s = (2 * kUnits + blocks - 1) / blocks;
    if (s > (pairs + 3) / 4) s = (pairs + 3) / 4;
    return (int)(s < 1 ? 1 : s > 16 ? 16 : s);
}

constexpr int kKvBlock = 128;

struct BackwardPlan {
    int splits;
    int64_t stats, groups, partial, bytes;   // bytes of each of the two statistics, the groups, the partial sums; all
};
static BackwardPlan backward_plan(int B, int T, int Nq, int Nkv, int head_dim) {
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    BackwardPlan p;
    p.splits = kv_splits(B, T, Nq, Nkv, kKvBlock);
    p.stats = up((int64_t)B * Nq * T * 4);
    p.groups = up((int64_t)B * ((T + 31) / 32) * 8);
    p.partial = p.splits > 1 ? up((int64_t)p.splits * B * T * Nkv * 2 * head_dim * 4) : 0;
    p.bytes = 2 * p.stats + p.groups + p.partial;
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
        LLMQ_REQUIRE(out != qkv, "%s: out must not be qkv", what);
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
    if (head_dim > 64) launch(attention_forward_kernel<128, 1, 4>, 128, 256);
    else launch(attention_forward_kernel<64, 1, 4>, 128, 256);
    LLMQ_HIP_TRY(hipGetLastError());
    return LLMQ_OK;
}

extern "C" int64_t llmq_attention_backward_scratch_bytes(int B, int T, int Nq, int Nkv, int head_dim) {
    if (B <= 0 || T <= 0 || Nq <= 0 || Nkv <= 0 || Nq % Nkv || head_dim <= 0) return 0;
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
    LLMQ_REQUIRE(dqkv != qkv && dqkv != dout && dqkv != out, "%s: dqkv must be a tensor of its own", what);
    const BackwardPlan p = backward_plan(B, T, Nq, Nkv, head_dim);
    LLMQ_REQUIRE(scratch_bytes >= (size_t)p.bytes, "%s: scratch buffer too small (%zu bytes, %lld needed)", what, scratch_bytes, (long long)p.bytes);
    hipStream_t st = static_cast<hipStream_t>(stream);
    AttentionArgs a = make_args(qkv, first_key_or_null, B, T, Nq, Nkv, head_dim, softmax_scale);
    a.out = const_cast<uint16_t*>(out), a.lse = const_cast<float*>(lse), a.dout = dout, a.dqkv = dqkv;
    char* s = static_cast<char*>(scratch);
    a.lse2 = reinterpret_cast<float*>(s);
    a.delta = reinterpret_cast<float*>(s + p.stats);
    a.groups = reinterpret_cast<int2*>(s + 2 * p.stats);
    a.partial = p.splits > 1 ? reinterpret_cast<float*>(s + 2 * p.stats + p.groups) : nullptr;
    a.splits = p.splits;
    auto launch = [&](auto kernel, int64_t blocks, int threads) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), 0, st, a);
    };
    const int64_t q_blocks = (int64_t)((T + 127) / 128) * B * Nq;
    const int64_t kv_blocks = (int64_t)((T + kKvBlock - 1) / kKvBlock) * B * Nkv * p.splits;
    if (head_dim > 64) {
        launch(attention_backward_q_kernel<128, 1, 4>, q_blocks, 256);
        LLMQ_HIP_TRY(hipGetLastError());
        launch(attention_backward_kv_kernel<128, 1, 4>, kv_blocks, 256);
    } else {
        launch(attention_backward_q_kernel<64, 1, 4>, q_blocks, 256);
        LLMQ_HIP_TRY(hipGetLastError());
        launch(attention_backward_kv_kernel<64, 1, 4>, kv_blocks, 256);
    }
    LLMQ_HIP_TRY(hipGetLastError());
    if (p.splits > 1) {
        const int64_t n = (int64_t)B * T * Nkv * (2 * head_dim / 4);
        launch(attention_join_kernel, (n + 255) / 256, 256);
        LLMQ_HIP_TRY(hipGetLastError());
    }
    return LLMQ_OK;
}
