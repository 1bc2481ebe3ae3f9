// Attention over the block-scaled cache (layout: kvhip_block.hpp), whole or over listed blocks.
//
// A wavefront takes every NW-th block of its workgroup's part and keeps the running maximum, the sum and the output of NM
// tiles of 16 query rows in registers: one pass over the keys and values, nothing shared until the end.
//   S^T = K Q^T   16x16x32 products, keys as the left operand: a lane is left with the scores of query row (lane & 15) at
//                 tokens 16 t + 4 (lane >> 4) + i
//   O^T = V^T P^T the same lane's weights, two tiles of tokens at a time, are the right operand as they stand -- the order of
//                 the contraction is free, so the pages hold each lane's sixteen tokens of a channel side by side
// Codes become operands by one conversion for two values, which takes the block's scale along.  Operands are loaded straight
// from the pages, 1 KB to an instruction, half a block ahead.  The blocks'
// addresses and scales are looked up 64 at a time, a lane to a block, instead of one dependent load after another.
//
// Single tokens are bound by memory where the batch fills the chip (32 sequences at 32 768 keys, 8 x 128: 351 us, 6.1 TB/s;
// 16 ragged ones of four tokens 65 us, 4.4 TB/s over the keys that they see) and by the chain of a launch where it does not
// (517 keys of 4 x 64: 7.2 us; 30 011 of 8 x 128: 14.2 us, 4.3 TB/s, and 3.9 for the merge).  Chosen blocks of a prompt's
// tokens come from the second-level caches, 16 KB to a token, block and pair (300 tokens x 32 blocks x 8 pairs: 78 us, 16 TB/s).
#pragma once
#include "kvhip_block_choose.hpp"
#include "kvhip_mask.hpp"
#include "kvhip_prefill_fp.hpp"
#include "kvhip_span_merge.hpp"

namespace kvhip {

// Whether a call has rows enough for the kernel that shares blocks between wavefronts, and the rows its workgroup takes.  Against
// two tiles of rows to a wavefront that loads for itself, us, shared / not: head size 128, 48 rows of a pair 36.3 / 40.3
// (8 x 8 pairs, 8000 keys), 40 rows 54.0 / 73.6 (32 x 8 pairs, 4000), but 48 rows of 8 pairs over 8192 keys 17.3 / 16.4, 96 rows 20.0 / 21.3;
// 2048 rows 92.2 / 92.3 and, of 8 x 8 pairs, 695 / 691; 256, 4 x 8 pairs, 4000 keys, 34 rows 30.6 / 48.0, 2048 rows 377 / 652.  Keys of 192, whose
// workgroups take 128 rows, from more than those on: 40 rows 36.5 / 30.2 (4 x 16 pairs, 4000 keys) and 22.9 / 18.0 (8 pairs, 8000),
// 96 rows 40.9 / 41.8 and 26.1 / 21.2, 128 rows 44.5 / 42.1 and 27.7 / 21.9, 160 rows 65.1 / 80.4 and 28.6 / 25.1, 400 rows 103 / 152 and
// 41.7 / 45.9.  Head sizes below 128, whose blocks need fewer registers, go the other way: 64, 160 rows 37.0 / 31.3, 2000 rows
// 234 / 210; 96, 200 rows 144 / 136.
inline bool block_attend_tiled(const BlockAttend &x) {
    const int64_t rows = (int64_t)x.a.Hq / x.a.Hkv * x.a.L;
    return !x.list && x.a.mask.mode != KVHIP_MASK_ARRAY && x.a.st.Dk >= 128 && rows > (x.a.st.Dk == 192 ? 128 : 32);
}
inline int block_tiled_rows(int Dk) { return Dk == 192 ? 128 : 64; }

// Tiles of 16 query rows that a wavefront takes (plan_block_attend chooses by the same rule).  Two, where there are rows for them:
// each conversion of a block's codes then serves both.  Four do not fit the registers of two wavefronts a SIMD (512 rows
// over 8192 keys x 128, 32 heads: 227 us, and 104 with two).
inline int block_row_tiles(const BlockAttend &x) {
    const int rows = x.a.Hq / x.a.Hkv * x.a.L;
    if (x.list || rows <= 16) return 1;
    return 2;
}

namespace {

typedef float kv_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 kv_b8 __attribute__((ext_vector_type(8)));
typedef _Float16 kv_h8 __attribute__((ext_vector_type(8)));

constexpr int CHOSEN_MAX = 1024;  // listed blocks that a workgroup chooses itself

template <int DT> __device__ __forceinline__ kv_f4 block_mfma(const kv_u4 &x, const kv_u4 &y, const kv_f4 &c) {
    if constexpr (DT == 1) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(kv_b8, x), __builtin_bit_cast(kv_b8, y), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(kv_h8, x), __builtin_bit_cast(kv_h8, y), c, 0, 0, 0);
}
// eight codes as eight elements
template <int DT> __device__ __forceinline__ kv_u4 block_operand(uint32_t lo, uint32_t hi, float scale) {
    return kv_u4{block_values<DT, false>(lo, scale), block_values<DT, true>(lo, scale), block_values<DT, false>(hi, scale), block_values<DT, true>(hi, scale)};
}
// Over the four lanes of a query row (16 apart), in each of them: halves and rows of 16 change places by one vector
// instruction each, nothing goes through LDS.
template <class OP> __device__ __forceinline__ float row_reduce(float v, OP op) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row_max(float v) {
    return row_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float row_sum(float v) {
    return row_reduce(v, [](float a, float b) { return a + b; });
}

// What a wavefront requests of a block: keys as [token tile][chunk of 64 channels] of 16 bytes a lane (a last chunk of 32: 8),
// values as [16 channels] of 16 bytes.
template <int DK, int DV> struct BlockTile {
    static constexpr int KC = DK / 64;
    static constexpr bool HALF = DK % 64 != 0;
    kv_u4 k[4][KC > 0 ? KC : 1];
    kv_u2 kh[HALF ? 4 : 1];
    kv_u4 v[DV / 16];
    __device__ __forceinline__ void load_keys(gptr kp, int lane) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int c = 0; c < KC; ++c) k[t][c] = ld_global<kv_u4>(kp + t * 16 * DK + c * 1024 + lane * 16);
            if constexpr (HALF) kh[t] = ld_global<kv_u2>(kp + t * 16 * DK + KC * 1024 + lane * 8);
        }
    }
    __device__ __forceinline__ void load_values(gptr vp, int lane) {
#pragma unroll
        for (int i = 0; i < DV / 16; ++i) v[i] = ld_global<kv_u4>(vp + i * 1024 + lane * 16);
    }
};

// MODE 1: index-only mask (no mask: one that every key passes); 2: array mask; 3: listed blocks
// SUMS: the sums of the weights by a product with ones (prompt chunks: an addition to a weight is a fourteenth of their vector
// instructions, and the matrix pipe has room); else by additions.
template <int DK, int DV, int DT, int NM, int MODE, bool SUMS = false> struct BlockWalk {
    static constexpr bool WHOLE_SUMS = SUMS;
    static constexpr uint32_t ONES = DT == 1 ? 0x3f803f80u : 0x3c003c00u;
    static constexpr int KS = DK / 32, VT = DV / 16;
    static constexpr bool SAFE = MODE == 2;  // an added mask may hold the type's lowest value: no products in front of the difference
    // float16 weights are taken times 2^14: those of keys far below the largest stay clear of the type's subnormals (the sums
    // carry the factor too)
    static constexpr float LIFT = DT == 0 ? 14.f : 0.f;
    // Maxima beyond this (in powers of two) are taken off before the product with `unit`, an instruction more for each score: the
    // roundings of the maximum's product and of what is added to it are 2^-11 here, less than half a step of float16, and
    // would lift weights past the type's largest value from 2^24 on.
    static constexpr float FAR = 4096.f;

    const BlockAttend &x;
    const int lane, g, n;
    const int b, h, bh;
    kv_u4 q[NM][KS];
    kv_f4 o[NM][VT];
    float m[NM], l[NM];
    kv_f4 ls[SUMS ? NM : 1];  // (four times the same)
    float unit;         // log2 e, times the scale (its sign is the queries') where scores have not met it
    KeyBounds see[NM];  // the keys of the lane's query row
    int ql[NM], qh[NM]; // its position and head (MODE 2)

    __device__ __forceinline__ BlockWalk(const BlockAttend &x_, int bh_)
        : x(x_), lane(threadIdx.x & 63), g(lane >> 4), n(lane & 15), b(bh_ / x_.a.Hkv), h(bh_ % x_.a.Hkv), bh(bh_), unit(SAFE || x_.a.scale == 0.f ? LOG2E : fabsf(x_.a.scale) * LOG2E) {
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.f;
            if (SUMS || i == 0) ls[SUMS ? i : 0] = kv_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int d = 0; d < VT; ++d) o[i][d] = kv_f4{0.f, 0.f, 0.f, 0.f};
        }
    }

    static __device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
    // Scores of one tile of query rows -> weights as operands; the outputs so far are brought to the new maximum.  Scores and
    // maxima are products that the call's scale has yet to meet (MODE 2: has met, an added mask's terms among them).  The value
    // product takes the weights in the cache's type, half a step off each, as in the other matrix-core kernels: 2-norm errors of
    // 1.9e-3 in bfloat16 and 2.5e-4 in float16, where weights of 32 bits would leave the output's rounding, 1.6e-3 and 2.2e-4.  Maxima,
    // sums and outputs stay in 32 bits (with SUMS the sums are those of the rounded weights).
    __device__ __forceinline__ void weigh(int i, kv_f4 (&s)[4], kv_u4 (&p)[2]) {
        float mx = max3(m[i], s[0][0], s[0][1]), my = max3(s[0][2], s[0][3], s[1][0]);
        mx = max3(mx, s[1][1], s[1][2]);
        my = max3(my, s[1][3], s[2][0]);
        mx = max3(mx, s[2][1], s[2][2]);
        my = max3(my, s[2][3], s[3][0]);
        mx = row_max(max3(max3(mx, s[3][1], s[3][2]), my, s[3][3]));
        const float ref = mx == -INFINITY ? 0.f : mx;  // (nothing seen yet: every difference is -infinity)
        const float far = ref * unit, off = LIFT - far;
        float e[16], sum = 0.f;
        if (SAFE || __any(fabsf(far) > FAR)) {  // the difference first: it is exact where it counts, and no exponent is above LIFT
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int k = 0; k < 4; ++k) e[4 * t + k] = fast_exp2(__builtin_fmaf(s[t][k] - ref, unit, LIFT));
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int k = 0; k < 4; ++k) e[4 * t + k] = fast_exp2(__builtin_fmaf(s[t][k], unit, off));
        }
        if constexpr (!SUMS) {
#pragma unroll
            for (int k = 0; k < 16; ++k) sum += e[k];
        }
        if (__any(mx != m[i])) {
            const float alpha = fast_exp2((m[i] - ref) * unit);
            if constexpr (SUMS) ls[i] *= alpha;
            else l[i] *= alpha;
#pragma unroll
            for (int d = 0; d < VT; ++d) o[i][d] *= alpha;
            m[i] = mx;
        }
        if constexpr (!SUMS) l[i] += sum;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                p[u][k] = DT == 1 ? pk_bf2(e[8 * u + 2 * k], e[8 * u + 2 * k + 1]) : pk_h2(e[8 * u + 2 * k], e[8 * u + 2 * k + 1]);
            if constexpr (SUMS) ls[i] = block_mfma<DT>(kv_u4{ONES, ONES, ONES, ONES}, p[u], ls[i]);
        }
    }

    // which of the lane's sixteen tokens its query row sees, those it does not see set to -infinity; adds an array mask
    __device__ __forceinline__ uint32_t mask(int i, int j0, kv_f4 (&s)[4]) {
        uint32_t seen = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int j = j0 + 16 * t + 4 * g + k;
                bool keep;
                if constexpr (MODE == 2) {
                    float add = 0.f;
                    keep = j < x.a.T && qh[i] >= 0 && mask_keep(x.a.mask, b, qh[i], ql[i], j, x.a.L, x.a.T, add);
                    keep = keep && add != -INFINITY;
                    s[t][k] += add;
                } else {
                    keep = see[i].keep(j);
                }
                if (!keep) s[t][k] = -INFINITY;
                seen |= keep ? 1u << (4 * t + k) : 0u;
            }
        return seen;
    }

    // Values of a block with keys that some query row does not see: a weight of zero does not take a NaN away.  NaN become
    // zeros, and channels that a seen token has NaN in are made NaN by a product of the two facts.  `bad`: 1 in the place of
    // each NaN, 0 elsewhere.
    __device__ __forceinline__ void poison(int i, int d, uint32_t seen, const kv_u4 (&bad)[2]) {
        constexpr uint32_t ONE = DT == 1 ? 0x3f80u : 0x3c00u;
        kv_f4 hit{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            kv_u4 w;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                w[k] = ((seen >> (8 * u + 2 * k)) & 1u ? ONE : 0u) | ((seen >> (8 * u + 2 * k + 1)) & 1u ? ONE << 16 : 0u);
            hit = block_mfma<DT>(bad[u], w, hit);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (hit[k] > 0.f) o[i][d][k] = __builtin_nanf("");
    }

    // a block of codes; `ahead` requests the next one's keys, into the registers of this one's
    template <class AHEAD> __device__ __forceinline__ void block(BlockTile<DK, DV> &tile, float ks, float vs, int j0, bool masked, AHEAD ahead) {
        using Tile = BlockTile<DK, DV>;
        kv_f4 s[NM][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int i = 0; i < NM; ++i) s[i][t] = kv_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < KS; ++c) {
                kv_u4 w;
                if (Tile::HALF && c == KS - 1) w = block_operand<DT>(tile.kh[t][0], tile.kh[t][1], ks);
                else w = block_operand<DT>(tile.k[t][c >> 1][2 * (c & 1)], tile.k[t][c >> 1][2 * (c & 1) + 1], ks);
#pragma unroll
                for (int i = 0; i < NM; ++i) s[i][t] = block_mfma<DT>(w, q[i][c], s[i][t]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        ahead();
        __builtin_amdgcn_sched_barrier(0);
        kv_u4 p[NM][2];
        uint32_t seen[NM];
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            if constexpr (SAFE) {
#pragma unroll
                for (int t = 0; t < 4; ++t) s[i][t] *= x.a.scale;
            }
            seen[i] = 0xffffu;
            if (masked) seen[i] = mask(i, j0, s[i]);
            weigh(i, s[i], p[i]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (masked) {
            uint32_t any = 0;
#pragma unroll
            for (int d = 0; d < VT; ++d)
#pragma unroll
                for (int k = 0; k < 4; ++k) any |= nan_codes(tile.v[d][k]);
            if (__any(any != 0)) {
#pragma unroll
                for (int d = 0; d < VT; ++d) {
                    kv_u4 bad[2];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t f = nan_codes(tile.v[d][k]) >> 7, one = f * 0x38u;  // 1.0
                        tile.v[d][k] &= ~(f * 0xffu);
                        bad[k >> 1][2 * (k & 1)] = block_values<DT, false>(one, 1.f);
                        bad[k >> 1][2 * (k & 1) + 1] = block_values<DT, true>(one, 1.f);
                    }
#pragma unroll
                    for (int i = 0; i < NM; ++i) poison(i, d, seen[i], bad);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
#pragma unroll
        for (int d = 0; d < VT; ++d) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const kv_u4 a = block_operand<DT>(tile.v[d][2 * u], tile.v[d][2 * u + 1], vs);
#pragma unroll
                for (int i = 0; i < NM; ++i) o[i][d] = block_mfma<DT>(a, p[i][u], o[i][d]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // The same from a block in LDS, keys and then values as they lie in the pages: operands are read as they are used.  `ahead(t)`,
    // four times between products, makes a quarter of the wavefront's requests for the next round: the compute unit takes in 64
    // bytes a cycle, and a round's requests in one go held every wavefront up for a thousand cycles.
    template <class AHEAD> __device__ __forceinline__ void block_shared(const char *lds, float ks, float vs, int j0, bool masked, AHEAD ahead) {
        constexpr bool HALF = DK % 64 != 0;
        const char *keys = lds, *values = lds + BLOCK_ROWS * DK + lane * 16;
        kv_f4 s[NM][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            kv_u4 raw[(KS + 1) / 2];
#pragma unroll
            for (int c = 0; c < KS / 2; ++c) raw[c] = *reinterpret_cast<const kv_u4 *>(keys + t * 16 * DK + c * 1024 + lane * 16);
            if constexpr (HALF) {
                const kv_u2 h = *reinterpret_cast<const kv_u2 *>(keys + t * 16 * DK + (KS / 2) * 1024 + lane * 8);
                raw[KS / 2] = kv_u4{h[0], h[1], 0u, 0u};
            }
#pragma unroll
            for (int i = 0; i < NM; ++i) s[i][t] = kv_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < KS; ++c) {
                const kv_u4 w = block_operand<DT>(raw[c >> 1][2 * (c & 1)], raw[c >> 1][2 * (c & 1) + 1], ks);
#pragma unroll
                for (int i = 0; i < NM; ++i) s[i][t] = block_mfma<DT>(w, q[i][c], s[i][t]);
            }
            ahead(t);
        }
        kv_u4 p[NM][2];
        uint32_t seen[NM];
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            seen[i] = 0xffffu;
            if (masked) seen[i] = mask(i, j0, s[i]);
            weigh(i, s[i], p[i]);
        }
        bool nan = false;
        if (masked) {
            uint32_t any = 0;
#pragma unroll
            for (int d = 0; d < VT; ++d) {
                const kv_u4 w = *reinterpret_cast<const kv_u4 *>(values + d * 1024);
#pragma unroll
                for (int k = 0; k < 4; ++k) any |= nan_codes(w[k]);
            }
            nan = __any(any != 0);
            if (nan) {
#pragma unroll
                for (int d = 0; d < VT; ++d) {
                    const kv_u4 w = *reinterpret_cast<const kv_u4 *>(values + d * 1024);
                    kv_u4 bad[2];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t one = (nan_codes(w[k]) >> 7) * 0x38u;  // 1.0
                        bad[k >> 1][2 * (k & 1)] = block_values<DT, false>(one, 1.f);
                        bad[k >> 1][2 * (k & 1) + 1] = block_values<DT, true>(one, 1.f);
                    }
#pragma unroll
                    for (int i = 0; i < NM; ++i) poison(i, d, seen[i], bad);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
#pragma unroll
        for (int d = 0; d < VT; ++d) {
            kv_u4 w = *reinterpret_cast<const kv_u4 *>(values + d * 1024);
            if (nan) {
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] &= ~((nan_codes(w[k]) >> 7) * 0xffu);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const kv_u4 a = block_operand<DT>(w[2 * u], w[2 * u + 1], vs);
#pragma unroll
                for (int i = 0; i < NM; ++i) o[i][d] = block_mfma<DT>(a, p[i][u], o[i][d]);
            }
        }
    }
    // bit 7 of every byte of a word that is a NaN code
    static __device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

    // the rows of the unfinished block; with a.new_k its last row is still in the caller's arrays
    __device__ __forceinline__ void tail(int j0) {
        const AttendArgs &a = x.a;
        const char *tk = x.b.tail_k + (size_t)bh * BLOCK_ROWS * DK * 2, *tv = x.b.tail_v + (size_t)bh * BLOCK_ROWS * DV * 2;
        const int fresh = a.new_k ? a.T - 1 - j0 : -1;  // that row
        const char *nk = static_cast<const char *>(a.new_k) + (size_t)bh * DK * 2;
        const uint16_t *nv = static_cast<const uint16_t *>(a.new_v) + (size_t)bh * DV;
        // (everything is requested at once: keys, then, behind the score product, values)
        kv_u4 w[4 * KS > 2 * VT ? 4 * KS : 2 * VT];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int r = 16 * t + n;
            const gptr row = as_global(r == fresh ? nk : tk + (size_t)r * DK * 2);
#pragma unroll
            for (int c = 0; c < KS; ++c) {
                // the channels that the query operands hold at this step (those of a block's chunks)
                const int d = (c | 1) < KS ? (c >> 1) * 64 + g * 16 + (c & 1) * 8 : c * 32 + g * 8;
                w[t * KS + c] = ld_global<kv_out8>(row + 2 * d);
            }
        }
        kv_f4 s[NM][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int i = 0; i < NM; ++i) s[i][t] = kv_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < KS; ++c) {
                kv_u4 y = w[t * KS + c];
                if (fresh >= 0) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) y[k] = no_infinities<DT>(y[k]);
                }
#pragma unroll
                for (int i = 0; i < NM; ++i) s[i][t] = block_mfma<DT>(y, q[i][c], s[i][t]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int d = 0; d < VT; ++d)
#pragma unroll
            for (int u = 0; u < 2; ++u) w[2 * d + u] = ld_global<kv_u4>(as_global(tv + ((size_t)(4 * u + g) * DV + 16 * d + n) * 16));
        uint32_t e[VT];
#pragma unroll
        for (int d = 0; d < VT; ++d) e[d] = fresh >= 0 ? (uint32_t)ld_global<uint16_t>(as_global(nv + 16 * d + n)) : 0u;
        __builtin_amdgcn_sched_barrier(0);
        kv_u4 p[NM][2];
        uint32_t seen[NM];
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            if constexpr (SAFE) {
#pragma unroll
                for (int t = 0; t < 4; ++t) s[i][t] *= a.scale;
            }
            seen[i] = mask(i, j0, s[i]);
            weigh(i, s[i], p[i]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (fresh >= 0) {  // (element 4 h + i is token 32 u + 16 h + 4 g + i)
            const int at = ((fresh >> 4) & 1) * 4 + (fresh & 3);
            const uint32_t mine = ((fresh >> 2) & 3) == g ? (at & 1 ? 0xffff0000u : 0xffffu) : 0u;
#pragma unroll
            for (int d = 0; d < VT; ++d) {
                const uint32_t x = no_infinities<DT>(e[d] | (e[d] << 16));
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t here = (fresh >> 5) == u && (at >> 1) == k ? mine : 0u;
                        w[2 * d + u][k] = (w[2 * d + u][k] & ~here) | (x & here);
                    }
            }
        }
        // NaN (and, in rows that were never written, anything)
        constexpr uint32_t INF = DT == 1 ? 0x7f80u : 0x7c00u, ONE = DT == 1 ? 0x3f80u : 0x3c00u;
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 2 * VT; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t h = w[j][k] & 0x7fff7fffu;
                top = max(top, max(h & 0xffffu, h >> 16));
            }
        if (__any(top >= INF)) {
#pragma unroll
            for (int d = 0; d < VT; ++d) {
                kv_u4 bad[2];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t y = w[2 * d + u][k];
                        const bool lo = (y & 0x7fffu) >= INF, hi = ((y >> 16) & 0x7fffu) >= INF;
                        bad[u][k] = (lo ? ONE : 0u) | (hi ? ONE << 16 : 0u);
                        w[2 * d + u][k] = y & ((lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u));
                    }
#pragma unroll
                for (int i = 0; i < NM; ++i) poison(i, d, seen[i], bad);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int d = 0; d < VT; ++d) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < NM; ++i) o[i][d] = block_mfma<DT>(w[2 * d + u], p[i][u], o[i][d]);
        }
    }
};

// What the rows of a wavefront's tiles are, and what they see.
struct RowsView {
    int G, R, token, row0;  // heads a pair, rows that the tiles cut, (listed blocks) the token, the wavefront's first row
    int in_lo, in_hi;       // keys that every row sees
    int lo, hi;             // keys that some row sees
    template <int MODE> __device__ __forceinline__ int at(const AttendArgs &a, int i) const { return MODE == 3 ? i * a.L + token : i; }
};
// rows row0 .. row0 + 16 NM - 1 of pair `w`: bounds (those of rows span0 .. span1 - 1, the workgroup's), queries
template <class Walk, int DK, int NM, int MODE>
__device__ __forceinline__ void take_rows(Walk &w, RowsView &v, const BlockAttend &x, int span0, int span1) {
    const AttendArgs &a = x.a;
    const SymMask sym = sym_mask_init(a.mask, w.b, a.L, a.T);
    v.in_lo = v.lo = 0;
    v.in_hi = v.hi = a.T - 1;
    if constexpr (MODE == 1) {
        const int last = min(span1, v.R) - 1;
        const bool one_head = a.L > 1 && span0 / a.L == last / a.L;
        const KeyBounds f = sym_mask_bounds(sym, one_head ? span0 % a.L : 0), e = sym_mask_bounds(sym, one_head ? last % a.L : a.L - 1);
        v.in_lo = max(e.lo, 0);
        v.in_hi = min(f.hi, a.T - 1);
        v.lo = max(f.lo, 0);
        v.hi = min(e.hi, a.T - 1);
    }
    if constexpr (MODE == 3) {
        v.lo = v.in_lo = x.left_pad ? max(x.left_pad[w.b], 0) : 0;
        v.hi = v.in_hi = a.T - a.L + v.token;
    }
    const char *qbase = static_cast<const char *>(a.q) + (size_t)w.bh * v.G * a.L * DK * 2;
#pragma unroll
    for (int i = 0; i < NM; ++i) {
        const int r = v.row0 + 16 * i + w.n;
        const bool live = r < v.R;
        const char *row = qbase + (size_t)v.template at<MODE>(a, live ? r : 0) * DK * 2;
#pragma unroll
        for (int c = 0; c < Walk::KS; ++c) {
            const int d = (c | 1) < Walk::KS ? (c >> 1) * 64 + w.g * 16 + (c & 1) * 8 : c * 32 + w.g * 8;
            w.q[i][c] = live && a.scale != 0.f ? load_row16(row + 2 * d) : kv_u4{0u, 0u, 0u, 0u};
            if (!Walk::SAFE && a.scale < 0.f) w.q[i][c] ^= 0x80008000u;
        }
        if (MODE == 3 || a.L == 1) {  // (no divisions in front of a step's first request)
            w.ql[i] = 0;
            w.qh[i] = live ? w.h * v.G + r : -1;
        } else {
            w.ql[i] = live ? r % a.L : 0;
            w.qh[i] = live ? w.h * v.G + r / a.L : -1;
        }
        w.see[i] = KeyBounds{v.lo, v.hi};
        if constexpr (MODE == 1) {
            const KeyBounds k = sym_mask_bounds(sym, w.ql[i]);
            w.see[i] = KeyBounds{max(k.lo, 0), min(k.hi, a.T - 1)};
        }
    }
}
// Tile i of the wavefronts that share its rows (KW of them, this one is number k of it; `t` of KW * 64 threads) joined: output rows, or
// a partial of part `part`.  Holds two barriers of the workgroup.
template <class Walk, int DV, int DT, int MODE, int KW>
__device__ __forceinline__ void leave_tile(Walk &w, const RowsView &v, const BlockAttend &x, WaveParts<DV, KW, 16> &parts, int i, int k, int t, int part) {
    const AttendArgs &a = x.a;
    const int rows = min(v.R - (v.row0 + 16 * i), 16);
    const float l = Walk::WHOLE_SUMS ? w.ls[Walk::WHOLE_SUMS ? i : 0][0] : row_sum(w.l[i]);
    if constexpr (!Walk::SAFE) w.m[i] = w.m[i] == -INFINITY ? -INFINITY : w.m[i] * fabsf(a.scale);  // (weights go by scores from here on)
    if (w.g == 0) parts.m[k][w.n] = w.m[i];
    __syncthreads();
    const float weight = wave_weight(parts, w.n, w.m[i]);
    if (w.g == 0) parts.l[k][w.n] = l * weight;
    if (w.n < rows) {  // (a step has few rows of the sixteen)
#pragma unroll
        for (int d = 0; d < Walk::VT; ++d) *reinterpret_cast<kv_f4 *>(&parts.rows[k][w.n][16 * d + 4 * w.g]) = w.o[i][d] * weight;
    }
    __syncthreads();
    constexpr int LPR = DV / 4, RPB = KW * 64 / LPR;
    const int c = 4 * (t % LPR);
    if (t >= RPB * LPR) return;  // (96 columns: lanes left over)
    for (int r = t / LPR; r < rows; r += RPB) {
        float o[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll
        for (int j = 0; j < KW; ++j) {
#pragma unroll
            for (int d = 0; d < 4; ++d) o[d] += parts.rows[j][r][c + d];
            sum += parts.l[j][r];
        }
        const int at = v.template at<MODE>(a, v.row0 + 16 * i + r);
        const size_t all = (size_t)v.G * a.L;
        if (x.nsplit == 1) {
            const float inv = 1.f / sum;
#pragma unroll
            for (int d = 0; d < 4; ++d) o[d] = sum == 0.f ? 0.f : o[d] * inv;
            store_columns<DT>(a.out, ((size_t)w.bh * all + at) * DV + c, o);
        } else {
            float *to = a.workspace + (((size_t)w.bh * x.nsplit + part) * all + at) * (DV + 2);
            store_floats(to + c, o);
            if (c == 0) {
                float mx = parts.m[0][r];
#pragma unroll
                for (int j = 1; j < KW; ++j) mx = fmaxf(mx, parts.m[j][r]);
                *reinterpret_cast<kv_f2 *>(to + DV) = kv_f2{mx, sum};
            }
        }
    }
}

// A single token's row, still in the caller's arrays, into the tail, by one wavefront of each pair (the readers of the tail take it from
// there as well).  Each kernel that a single token may come to calls it.
template <int DK, int DV, int DT> __device__ __forceinline__ void write_step(const BlockAttend &x, int bh, int lane) {
    const AttendArgs &a = x.a;
    if (!a.new_k || blockIdx.y != 0 || blockIdx.z != 0) return;
    const int r = (a.T - 1) % BLOCK_ROWS;
    const uint16_t *nk = static_cast<const uint16_t *>(a.new_k) + (size_t)bh * DK, *nv = static_cast<const uint16_t *>(a.new_v) + (size_t)bh * DV;
    uint16_t *tk = reinterpret_cast<uint16_t *>(x.b.tail_k) + ((size_t)bh * BLOCK_ROWS + r) * DK;
    uint16_t *tv = reinterpret_cast<uint16_t *>(x.b.tail_v) + (size_t)bh * BLOCK_ROWS * DV;
    for (int d = lane; d < DK; d += 64) tk[d] = (uint16_t)no_infinities<DT>(nk[d]);
    for (int d = lane; d < DV; d += 64) tv[tail_v_at(DV, r, d)] = (uint16_t)no_infinities<DT>(nv[d]);
}

// grid (BH, tiles of query rows, parts), NW wavefronts.  MODE 3: (BH, tokens x tiles of heads, parts).
template <int DK, int DV, int DT, int NM, int MODE, int NW>
__global__ void __launch_bounds__(NW * 64, DK <= 128 ? 2 : 1) block_attend_kernel(BlockAttend x) {
    using Walk = BlockWalk<DK, DV, DT, NM, MODE>;
    using Tile = BlockTile<DK, DV>;
    __shared__ WaveParts<DV, NW, 16> parts;
    const AttendArgs &a = x.a;
    const int bh = blockIdx.x, part = blockIdx.z;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    RowsView v;
    v.G = a.Hq / a.Hkv;
    v.R = MODE == 3 ? v.G : v.G * a.L;
    v.token = MODE == 3 ? blockIdx.y / x.tiles : 0;
    v.row0 = (MODE == 3 ? blockIdx.y % x.tiles : blockIdx.y) * 16 * NM;
    Walk w(x, bh);
    take_rows<Walk, DK, NM, MODE>(w, v, x, v.row0, v.row0 + 16 * NM);
    const int lo = v.lo, hi = v.hi, in_lo = v.in_lo, in_hi = v.in_hi, token = v.token;

    // the blocks of this part: positions [s0, s1) of the row's blocks, or of its list
    const int first = MODE == 3 ? 0 : lo / BLOCK_ROWS;
    const int total = MODE == 3 ? x.count : hi < lo ? 0 : hi / BLOCK_ROWS - first + 1;
    const int each = (total + x.nsplit - 1) / x.nsplit;
    const int s0 = min(part * each, total), s1 = min(s0 + each, total);
    const int mine = s1 - s0 > wave ? (s1 - s0 - wave + NW - 1) / NW : 0;
    const int32_t *list = MODE == 3 ? x.list + ((size_t)bh * a.L + token) * x.count : nullptr;
    if constexpr (MODE == 3) {
        if (x.keys) {
            // The choice by every workgroup of the token for itself, keys in the memory that the parts take later (one sequence of 131 000
            // keys, 64 blocks: 15.4 us, 7.5 + 10.5 with the choice in a launch of its own; 8 ragged ones of 65 000, 32 blocks: 14.4, 6 + 12.3).
            __shared__ int32_t chosen[CHOSEN_MAX];
            __shared__ uint32_t area[choose_area(NW)];
            uint32_t *keys = reinterpret_cast<uint32_t *>(&parts);
            const uint32_t *from = x.keys + ((size_t)bh * a.L + token) * x.key_stride;
            const int lead = lo / BLOCK_ROWS, seen = hi < lo ? 0 : hi / BLOCK_ROWS - lead + 1;
            if (seen > x.count)
                for (int i = threadIdx.x; i < seen - x.recent; i += NW * 64) keys[i] = from[i];
            __syncthreads();
            choose<NW>(keys, area, lane, lead, seen, x.count, x.first, x.recent, chosen);
            __syncthreads();
            list = chosen;
            if (part == 0 && v.row0 == 0)
                for (int i = threadIdx.x; i < x.count; i += NW * 64) x.list_out[((size_t)bh * a.L + token) * x.count + i] = chosen[i];
        }
    }
    int tail_at = -1, tails = 0;  // (a list may hold it more than once)

    for (int at = 0; at < mine; at += 64) {
        // a lane to a block: where it lies and its scales
        const int turn = min(mine - at, 64);
        const int i = s0 + wave + NW * (at + lane);
        int blk = -1;
        if (lane < turn) {
            if constexpr (MODE == 3) {
                blk = list[i];
                const int before = i > 0 ? list[i - 1] : -1;
                if (blk < lo / BLOCK_ROWS || blk > (hi < lo ? -1 : hi / BLOCK_ROWS) || (i > 0 && before >= blk)) blk = -1;
            } else {
                blk = first + i;
            }
        }
        uint64_t kp = 0, vp = 0;
        float ks = 1.f, vs = 1.f;
        if (blk >= 0 && blk < x.b.coded) {
            const PageEntry e = block_page(x.b, blk / BLOCK_PER_PAGE);
            const int in_page = blk % BLOCK_PER_PAGE;
            kp = reinterpret_cast<uint64_t>(e.k + (size_t)bh * a.st.k_cell + (size_t)in_page * BLOCK_ROWS * DK);
            vp = reinterpret_cast<uint64_t>(e.v + (size_t)bh * a.st.v_cell + (size_t)in_page * BLOCK_ROWS * DV);
            const kv_f2 sc = ld_global<kv_f2>(as_global(e.ksb) + (size_t)bh * a.st.ksb_cell + in_page * 8);
            ks = sc.x;
            vs = sc.y;
        }
        const uint64_t open = __ballot(blk >= 0 && blk >= x.b.coded);
        if (open) tail_at = __builtin_amdgcn_readlane(blk, __builtin_ctzll(open)) * BLOCK_ROWS;
        if (MODE == 3) tails += __builtin_popcountll(open);
        uint64_t todo = __ballot(blk >= 0 && blk < x.b.coded);
        auto at_lane = [](uint64_t v, int of) {  // (readlane returns a signed number)
            const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, of), hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), of);
            return (gptr)(((uint64_t)hi << 32) | lo);
        };
        if (!todo) continue;
        // One buffer, its halves skewed: a block's values are requested in front of its score product, the next block's keys
        // behind it.
        Tile tile;
        int cur = __builtin_ctzll(todo);
        tile.load_keys(at_lane(kp, cur), lane);
        while (true) {
            todo &= todo - 1;
            const int then = todo ? __builtin_ctzll(todo) : cur;  // (the last block's keys again: no branch around the requests)
            tile.load_values(at_lane(vp, cur), lane);
            __builtin_amdgcn_sched_barrier(0);
            const float k = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks), cur));
            const float v = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), cur));
            const int j0 = __builtin_amdgcn_readlane(blk, cur) * BLOCK_ROWS;
            w.block(tile, k, v, j0, MODE == 2 || j0 < in_lo || j0 + BLOCK_ROWS - 1 > in_hi,
                    [&] { tile.load_keys(at_lane(kp, then), lane); });
            if (!todo) break;
            cur = then;
        }
    }
    if constexpr (MODE == 3) {
        for (; tails > 0; --tails) w.tail(tail_at);
    } else {
        if (tail_at >= 0) w.tail(tail_at);
    }

    if (wave == NW - 1) write_step<DK, DV, DT>(x, bh, lane);

    // the wavefronts' parts joined, 16 rows at a time
#pragma unroll
    for (int i = 0; i < NM; ++i) {
        if (i) __syncthreads();
        leave_tile<Walk, DV, DT, MODE, NW>(w, v, x, parts, i, wave, threadIdx.x, part);
    }
}

// Many query rows of head sizes from 128 on (prompt chunks): eight wavefronts, RW groups of 16 NM rows by KW of the blocks of a round.  The blocks of a
// round lie in LDS, each read by the RW wavefronts that share it; the next round's are on their way, past the registers, while
// this one's are looked at.  Wavefronts wait only for those that they share a block with.
// What bounds it: vector instructions and products share a SIMD's issue -- a block costs two tiles of rows 2700 cycles alone and
// 3000 beside another wavefront, of 1360 for its 68 products and 2050 for 128 conversions, 32 exponentials and the rest -- at a clock
// that falls to about 2 GHz under them: 512 rows over 8192 keys x 128 (2048 rows of 8 pairs) 102 us, 655 TFLOP/s.
// grid (BH, tiles of 16 NM RW rows, parts)
template <int DK, int DV> struct TiledShape {
    // (registers: one tile of rows a wavefront at 256; LDS: two rounds of KW blocks)
    static constexpr int NM = DK <= 192 ? 2 : 1, RW = DK <= 128 ? 2 : 4, KW = 8 / RW, ROWS = 16 * NM * RW;
};
template <int DK, int DV, int DT>
__global__ void __launch_bounds__(512, 2) block_attend_tiled_kernel(BlockAttend x) {
    using Shape = TiledShape<DK, DV>;
    constexpr int NM = Shape::NM, RW = Shape::RW, KW = Shape::KW, BYTES = BLOCK_ROWS * (DK + DV), CHUNKS = BYTES / 1024, MINE = CHUNKS / RW;
    static_assert(CHUNKS % RW == 0, "whole requests a wavefront");
    using Walk = BlockWalk<DK, DV, DT, NM, 1, true>;
    using Parts = WaveParts<DV, KW, 16>;
    constexpr size_t RING = 2 * KW * BYTES, JOIN = RW * sizeof(Parts);
    __shared__ __align__(16) char lds[RING > JOIN ? RING : JOIN];
    __shared__ int there[8];  // by wavefront: rounds that its share of the blocks has come for
    const AttendArgs &a = x.a;
    const int bh = blockIdx.x, part = blockIdx.z;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int rw = wave % RW, kw = wave / RW;
    RowsView v;
    v.G = a.Hq / a.Hkv;
    v.R = v.G * a.L;
    v.token = 0;
    const int group0 = blockIdx.y * Shape::ROWS;
    v.row0 = group0 + rw * 16 * NM;
    if (threadIdx.x < 8) there[threadIdx.x] = 0;
    __syncthreads();
    Walk w(x, bh);
    take_rows<Walk, DK, NM, 1>(w, v, x, group0, group0 + Shape::ROWS);

    const int first = v.lo / BLOCK_ROWS, total = v.hi < v.lo ? 0 : v.hi / BLOCK_ROWS - first + 1;
    const int each = (total + x.nsplit - 1) / x.nsplit, s0 = min(part * each, total), s1 = min(s0 + each, total);
    const int rounds = (s1 - s0 + KW - 1) / KW;
    // where the wavefront's blocks lie, a lane to a round, 64 rounds at a time
    uint64_t kp = 0, vp = 0;
    float ks = 1.f, vs = 1.f;
    int known = -64, tail_at = -1;
    auto block_of = [&](int round) {
        const int i = s0 + round * KW + kw;
        return i < s1 ? first + i : -1;
    };
    auto look_up = [&](int round) {
        known = round;
        const int blk = block_of(round + lane);
        if (blk >= 0 && blk < x.b.coded) {
            const PageEntry e = block_page(x.b, blk / BLOCK_PER_PAGE);
            const int in_page = blk % BLOCK_PER_PAGE;
            kp = reinterpret_cast<uint64_t>(e.k + (size_t)bh * a.st.k_cell + (size_t)in_page * BLOCK_ROWS * DK);
            vp = reinterpret_cast<uint64_t>(e.v + (size_t)bh * a.st.v_cell + (size_t)in_page * BLOCK_ROWS * DV);
            const kv_f2 sc = ld_global<kv_f2>(as_global(e.ksb) + (size_t)bh * a.st.ksb_cell + in_page * 8);
            ks = sc.x;
            vs = sc.y;
        }
    };
    auto at_lane = [](uint64_t p, int of) {  // (readlane returns a signed number)
        const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)p, of), hi = __builtin_amdgcn_readlane((uint32_t)(p >> 32), of);
        return (gptr)(((uint64_t)hi << 32) | lo);
    };
    // the wavefront's share of its block of a round, 1 KB a request; what it needs of the block later
    float k_scale = 1.f, v_scale = 1.f, k_next = 1.f, v_next = 1.f;
    gptr k_from = nullptr, v_from = nullptr;
    char *to = lds;
    auto locate = [&](int round) {  // the block of a round: whether there is one in codes, and where
        if (round >= known + 64) look_up(round);
        const int blk = block_of(round);
        if (blk < 0) return false;
        if (blk >= x.b.coded) {
            tail_at = blk * BLOCK_ROWS;
            return false;
        }
        const int of = round - known;
        k_from = at_lane(kp, of);
        v_from = at_lane(vp, of);
        k_next = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks), of));
        v_next = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(vs), of));
        to = lds + ((round & 1) * KW + kw) * BYTES;
        return true;
    };
    auto request = [&](int j) {
        const int c = rw * MINE + j;
        const gptr from = c < DK / 16 ? k_from + c * 1024 : v_from + (c - DK / 16) * 1024;
        prefill_fp::load_to_lds((const char *)from, lane * 16, to + c * 1024);  // (its invariant: the wait and the counters below)
    };
    if (rounds > 0 && locate(0)) {
#pragma unroll
        for (int j = 0; j < MINE; ++j) request(j);
    }
    for (int round = 0; round < rounds; ++round) {
        // The round's block is there when each of the RW wavefronts that share it has waited for its share; a wavefront that says
        // so has read the round's before, whose half of the ring the next requests fill.  Only those wait for one
        // another, and they run the same rounds: the two groups on a SIMD drift apart, products of one over weights of the
        // other.
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        if (lane == 0) __hip_atomic_store(&there[wave], round + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        while (!__all(__hip_atomic_load(&there[kw * RW + (lane & (RW - 1))], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) > round)) {}
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
        k_scale = k_next;
        v_scale = v_next;
        const bool more = round + 1 < rounds && locate(round + 1);
        auto ahead = [&](int t) {
            if (!more) return;
#pragma unroll
            for (int j = 0; j < MINE; ++j)
                if (j * 4 / MINE == t) request(j);
        };
        const int blk = block_of(round);
        if (blk >= 0 && blk < x.b.coded) {  // (a wavefront with a block in the next round has one in this)
            const int j0 = blk * BLOCK_ROWS;
            w.block_shared(lds + ((round & 1) * KW + kw) * BYTES, k_scale, v_scale, j0, j0 < v.in_lo || j0 + BLOCK_ROWS - 1 > v.in_hi, ahead);
        }
    }
    if (tail_at >= 0) w.tail(tail_at);
    if (wave == 7) write_step<DK, DV, DT>(x, bh, lane);  // (a token of more than 32 heads to a kv head)
    __syncthreads();  // (the ring's memory takes the parts)
    Parts &parts = reinterpret_cast<Parts *>(lds)[rw];
#pragma unroll
    for (int i = 0; i < NM; ++i) {
        if (i) __syncthreads();
        leave_tile<Walk, DV, DT, 1, KW>(w, v, x, parts, i, kw, kw * 64 + lane, part);
    }
}

template <int DK, int DV, int DT, int NM, int MODE, int NW = 4> hipError_t block_attend_run(const BlockAttend &x, hipStream_t stream) {
    hipLaunchKernelGGL((block_attend_kernel<DK, DV, DT, NM, MODE, NW>), dim3(x.a.st.BH, block_attend_rows(x), x.nsplit), dim3(NW * 64), 0, stream, x);
    return hipGetLastError();
}
template <int DK, int DV, int DT> hipError_t block_attend_shape(const BlockAttend &x, hipStream_t stream) {
    if constexpr (DK >= 128) {
        if (block_attend_tiled(x)) {
            hipLaunchKernelGGL((block_attend_tiled_kernel<DK, DV, DT>), dim3(x.a.st.BH, block_attend_rows(x), x.nsplit), dim3(512), 0, stream, x);
            return hipGetLastError();
        }
    }
    if constexpr (DK <= 128) {
        if (x.waves == 8) return x.list ? block_attend_run<DK, DV, DT, 1, 3, 8>(x, stream) : block_attend_run<DK, DV, DT, 1, 1, 8>(x, stream);
    }
    if (x.list) return block_attend_run<DK, DV, DT, 1, 3>(x, stream);
    const int nm = block_row_tiles(x);
    if (x.a.mask.mode == KVHIP_MASK_ARRAY)
        return nm == 1 ? block_attend_run<DK, DV, DT, 1, 2>(x, stream) : block_attend_run<DK, DV, DT, 2, 2>(x, stream);
    if (nm == 1) return block_attend_run<DK, DV, DT, 1, 1>(x, stream);
    return block_attend_run<DK, DV, DT, 2, 1>(x, stream);
}
template <int DT> hipError_t block_attend_dtype(const BlockAttend &x, hipStream_t stream) {
    const int dk = x.a.st.Dk, dv = x.a.st.Dv;
    if (dk == 64 && dv == 64) return block_attend_shape<64, 64, DT>(x, stream);
    if (dk == 96 && dv == 96) return block_attend_shape<96, 96, DT>(x, stream);
    if (dk == 128 && dv == 128) return block_attend_shape<128, 128, DT>(x, stream);
    if (dk == 192 && dv == 128) return block_attend_shape<192, 128, DT>(x, stream);
    if (dk == 256 && dv == 256) return block_attend_shape<256, 256, DT>(x, stream);
    return hipErrorInvalidValue;
}

}  // namespace

}  // namespace kvhip
