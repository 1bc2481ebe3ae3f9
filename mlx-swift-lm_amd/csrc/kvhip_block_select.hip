// Blocks for each token from an estimate of the best score in them (summaries: kvhip_block.hpp).
//
// A query row's bound on a block is sum_d max(q_d hi_d, q_d lo_d), with hi and lo the block's largest and smallest key element
// of each channel.  Both sides are rounded to whole numbers times powers of two -- hi and lo are int8 in units of 4 scales, q is
// rint(q 2^-f), f the least integer with max |q| 2^-f <= 127 -- so that the sum is exact whatever its order (below 2^22 for 256
// channels) and the choice the same on any machine.  Without the roundings no key of the block would score higher; as it is one may, by
// up to half a unit of either side in every channel, and channels that stay within half a unit of zero have no part.  As products:
// q+ hi + q- lo, with q+ = max(q, 0) and q- = min(q, 0), on the 16x16x64 int8 instruction.
#include <algorithm>
#include <type_traits>

#include "kvhip_block_choose.hpp"
#include "kvhip_wave.hpp"

namespace kvhip {

namespace {

typedef int kv_i4 __attribute__((ext_vector_type(4)));
typedef unsigned short kv_us2 __attribute__((ext_vector_type(2)));

// whole 2^exp in an order that unsigned integers have too; 0 is below all of them.  The exponents of a bfloat16 cache's blocks and
// queries add up to -237 .. 244, more than a float has: ten bits for the exponent, and 21 of the fraction are all that a whole
// number below 2^22 (256 channels of 127 times 112) has.
__device__ __forceinline__ uint32_t ordered(int whole, int exp) {
    const uint32_t u = __float_as_uint((float)abs(whole)) >> 2;
    const uint32_t mag = whole ? u + ((uint32_t)(exp + 128) << 21) : 0;
    return whole < 0 ? 0x7fffffffu - mag : 0x80000000u | mag;
}
// the exponent of a power of two, in units of 4 of it
__device__ __forceinline__ int unit_exponent(float scale) { return (int)(__float_as_uint(scale) >> 23) - 127 + 2; }
constexpr int SELECT_WAVES = 16;
constexpr int SELECT_TILES = 4;  // at most so many tiles of 16 query rows to a workgroup
constexpr int SELECT_HEAD = SELECT_WAVES * 256 * 4;  // bytes of the histograms

// Eight channels of a query row, two to a word (zeros past the end).
__device__ __forceinline__ kv_u4 query_chunk(const char *row, int ud, int d, bool live) {
    kv_u4 w{0u, 0u, 0u, 0u};
    if (live && d + 8 <= ud) {
        w = load_row16(row + 2 * d);
    } else if (live) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (d + i < ud) w[i >> 1] |= (uint32_t) reinterpret_cast<const uint16_t *>(row)[d + i] << (16 * (i & 1));
    }
    return w;
}
template <int DT> __device__ __forceinline__ float float_at(uint32_t w, int half) {
    const uint32_t h = half ? w >> 16 : w & 0xffffu;
    return DT == 1 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half((unsigned short)h));
}

// What is kept of a tile of 16 query rows beside its operands: exponents, and the token (of the workgroup's) of each, or -1.
struct RowsOf {
    int exp[16], tok[16];
};
// One tile of 16 query rows as operands -- the positive and the negative part, [KS][64] each -- by one wavefront.  Everything
// else in the workgroup waits for it: the largest magnitude as a packed integer maximum, a number that is none only looked for
// where there is one, whole numbers by an addition that leaves them in the low bits.
template <int D, int DT>
__device__ __forceinline__ void query_operands(const char *row, int tok, int ud, int lane, kv_i4 *pos_out, kv_i4 *neg_out, RowsOf &of) {
    constexpr int KS = (D + 63) / 64;
    constexpr uint32_t INF = DT == 1 ? 0x7f80u : 0x7c00u;
    const int g = lane >> 4;
    kv_u4 w[KS][2];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) w[s][h] = query_chunk(row, ud, s * 64 + g * 16 + 8 * h, tok >= 0);
    auto largest = [&] {
        kv_us2 m{0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(kv_us2, w[s][i >> 2][i & 3] & 0x7fff7fffu));
        return max((uint32_t)m[0], (uint32_t)m[1]);
    };
    uint32_t mag = largest();
    if (mag >= INF) {  // elements that are no numbers have no say
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t x = w[s][i >> 2][i & 3];
                w[s][i >> 2][i & 3] = ((x & 0x7fffu) >= INF ? 0u : x & 0xffffu) | (((x >> 16) & 0x7fffu) >= INF ? 0u : x & 0xffff0000u);
            }
        mag = largest();
    }
    mag = max(mag, (uint32_t)__shfl_xor(mag, 16));
    mag = max(mag, (uint32_t)__shfl_xor(mag, 32));
    int ex = 0;
    const float mant = frexpf(float_at<DT>(mag, 0), &ex);  // (also of values below the smallest normal one)
    const int f = mag ? ex - 7 + (mant > 127.f / 128.f ? 1 : 0) : 0;
    if (g == 0) {
        of.exp[lane] = f;
        of.tok[lane] = tok;
    }
    constexpr float WHOLE = 12582912.f;  // 1.5 2^23: a sum's low bits are the nearest whole number, to even
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        kv_i4 pos, neg;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t p[4], m[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = ldexpf(float_at<DT>(w[s][k >> 1][2 * (k & 1) + (i >> 1)], i & 1), -f);
                p[i] = __float_as_uint(fmaxf(x, 0.f) + WHOLE);
                m[i] = __float_as_uint(fminf(x, 0.f) + WHOLE);
            }
            // (the low bytes of four words)
            pos[k] = (int)__builtin_amdgcn_perm(__builtin_amdgcn_perm(p[3], p[2], 0x0c0c0400u), __builtin_amdgcn_perm(p[1], p[0], 0x0c0c0400u), 0x05040100u);
            neg[k] = (int)__builtin_amdgcn_perm(__builtin_amdgcn_perm(m[3], m[2], 0x0c0c0400u), __builtin_amdgcn_perm(m[1], m[0], 0x0c0c0400u), 0x05040100u);
        }
        pos_out[s * 64 + lane] = pos;
        neg_out[s * 64 + lane] = neg;
    }
}

// The summaries of AHEAD groups of 16 blocks, STEP groups apart, as operands, and the exponents of the blocks' units.
template <int D, int AHEAD, int STEP> struct Summaries {
    static constexpr int KS = (D + 63) / 64;
    int unit[AHEAD];
    kv_i4 hi[AHEAD][KS], lo[AHEAD][KS];
    __device__ __forceinline__ void load(const BlockStore &b, int bh, int blk0, int last, int lane) {
        const Store &st = b.st;
        const int g = lane >> 4, n = lane & 15;
        gptr sum[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int blk = min(blk0 + u * STEP * 16 + n, last);
            const PageEntry e = block_page(b, blk / BLOCK_PER_PAGE);
            sum[u] = as_global(e.vsb) + (size_t)bh * st.vsb_cell + (size_t)(blk % BLOCK_PER_PAGE) * 2 * D;
            unit[u] = unit_exponent(ld_global<float>(as_global(e.ksb) + (size_t)bh * st.ksb_cell + 8 * (blk % BLOCK_PER_PAGE)));
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = s * 64 + g * 16;
                const bool in = D % 64 == 0 || d < D;
                hi[u][s] = in ? ld_global<kv_i4>(sum[u] + d) : kv_i4{0, 0, 0, 0};
                lo[u][s] = in ? ld_global<kv_i4>(sum[u] + D + d) : kv_i4{0, 0, 0, 0};
            }
    }
    // The bounds of one tile of rows on them, into keys[token][stride] at block0 + u STEP 16 + n (below `blocks`).
    __device__ __forceinline__ void bounds(const kv_i4 *pos_in, const kv_i4 *neg_in, const RowsOf &of, uint32_t *keys, int stride, int block0, int blocks,
                                           int lane) const {
        const int g = lane >> 4, n = lane & 15;
        int fr[4], tr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            fr[i] = of.exp[4 * g + i];
            tr[i] = of.tok[4 * g + i];
        }
        kv_i4 acc[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) acc[u] = kv_i4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const kv_i4 pos = pos_in[s * 64 + lane], neg = neg_in[s * 64 + lane];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                acc[u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(pos, hi[u][s], acc[u], 0, 0, 0);
                acc[u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(neg, lo[u][s], acc[u], 0, 0, 0);
            }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int at = block0 + u * STEP * 16 + n;
            if (at >= blocks) continue;
            uint32_t key[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) key[i] = ordered(acc[u][i], unit[u] + fr[i]);
            if (tr[0] >= 0 && tr[0] == tr[3]) {  // one token's rows: one entry for all four
                atomicMax(&keys[tr[0] * stride + at], max(max(key[0], key[1]), max(key[2], key[3])));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (tr[i] >= 0) atomicMax(&keys[tr[i] * stride + at], key[i]);
            }
        }
    }
};

// What a workgroup of either kernel below works on.
struct SelectView {
    int bh, b, G, tok0, toks, rows, pad, lead, coded;
    __device__ __forceinline__ SelectView(const BlockSelect &x, int bh_, int tok0_, int tokens) : bh(bh_), b(bh_ / x.Hkv), G(x.Hq / x.Hkv), tok0(tok0_) {
        toks = min(tokens, x.L - tok0);
        rows = toks * G;
        pad = x.left_pad ? max(x.left_pad[b], 0) : 0;
        lead = pad / BLOCK_ROWS;
        coded = min(x.b.coded, (x.T - x.L + tok0 + toks - 1) / BLOCK_ROWS);  // (the last token's own block is always chosen)
    }
    // row r of the group: token by token, a token's heads side by side; `tok`: its token, or -1 behind the last
    __device__ __forceinline__ const char *row(const BlockSelect &x, int r, int &tok) const {
        tok = toks == 1 ? 0 : r / G;
        const int head = r - tok * G;
        if (r >= rows) {
            tok = -1;
            return static_cast<const char *>(x.q);
        }
        return static_cast<const char *>(x.q) + (((size_t)bh * G + head) * x.L + tok0 + tok) * x.b.Dk_user * 2;
    }
    __device__ __forceinline__ int seen(const BlockSelect &x, int tok) const {
        const int p = x.T - x.L + tok0 + tok;
        return p < pad ? 0 : p / BLOCK_ROWS - lead + 1;
    }
};

// Many tokens: grid (BH, groups of `tokens` tokens), 16 wavefronts.  LDS: a histogram for each wavefront, the query operands and
// exponents of up to four tiles of 16 rows, keys [tokens][stride] of the blocks from `lead` on.  A wavefront requests the
// summaries of several groups of 16 blocks before it looks at the first.  300 tokens of 32 heads over 30 000 keys, 8 pairs: 20.7 us,
// a chain of its queries, its summaries (120 KB a workgroup) and the choice.
template <int D, int DT>
__global__ void __launch_bounds__(SELECT_WAVES * 64) block_select_kernel(BlockSelect x, int tokens, int stride) {
    constexpr int KS = (D + 63) / 64, AHEAD = D <= 128 ? 4 : 2;
    extern __shared__ uint32_t lds[];
    __shared__ RowsOf of[SELECT_TILES];
    kv_i4 *ops = reinterpret_cast<kv_i4 *>(lds + SELECT_WAVES * 256);                 // [tiles][positive / negative][KS][64]
    uint32_t *keys = reinterpret_cast<uint32_t *>(ops + SELECT_TILES * 2 * KS * 64);  // [tokens][stride]
    const SelectView v(x, blockIdx.x, blockIdx.y * tokens, tokens);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    for (int i = threadIdx.x; i < v.toks * stride; i += SELECT_WAVES * 64) keys[i] = 0;
    const int groups = v.coded > v.lead ? (v.coded - v.lead + 15) / 16 : 0;
    // (a token of more than 64 heads: its rows in turns)
    for (int row0 = 0; row0 < v.rows; row0 += 16 * SELECT_TILES) {
        const int tiles = min((v.rows - row0 + 15) / 16, SELECT_TILES);
        if (row0) __syncthreads();
        if (wave < tiles) {
            int tok;
            const char *row = v.row(x, row0 + 16 * wave + (lane & 15), tok);
            query_operands<D, DT>(row, tok, x.b.Dk_user, lane, ops + wave * 2 * KS * 64, ops + (wave * 2 + 1) * KS * 64, of[wave]);
        }
        __syncthreads();
        for (int first = wave; first < groups; first += SELECT_WAVES * AHEAD) {
            Summaries<D, AHEAD, SELECT_WAVES> sum;
            sum.load(x.b, v.bh, v.lead + first * 16, v.coded - 1, lane);
            for (int tile = 0; tile < tiles; ++tile)
                sum.bounds(ops + tile * 2 * KS * 64, ops + (tile * 2 + 1) * KS * 64, of[tile], keys, stride, first * 16, v.coded - v.lead, lane);
        }
    }
    __syncthreads();
    for (int tok = wave; tok < v.toks; tok += SELECT_WAVES)
        choose<1>(keys + (size_t)tok * stride, lds + wave * 256, lane, v.lead, v.seen(x, tok), x.count, x.first, x.recent,
                  x.list + ((size_t)v.bh * x.L + v.tok0 + tok) * x.count);
}

// Few tokens: the bounds by as many workgroups as there are stretches of 128 (head sizes above 128: 64) blocks -- one
// compute unit takes in a step's summaries at 13 bytes a cycle, 20 000 cycles for the 131 000 keys of one head -- and the
// choice, a workgroup to a token, in a launch of its own.  One token of eight sequences at 65 000 keys 6.5 + 5.5 us (in one launch
// 19.9), of one at 131 000 5.2 + 7.5 (29.6; stretches of 256 blocks 6.6 + 7.4): chains of latencies, the 17 MB and 4 MB that they read are 3.4 and 0.9.
// grid (BH, groups of `tokens` tokens, stretches), 4 wavefronts.  out: keys [BH, L, stride].
constexpr int BOUND_WAVES = 4, BOUND_TILES = 2;
constexpr int bound_ahead(int D) { return D <= 128 ? 2 : 1; }
template <int D, int DT>
__global__ void __launch_bounds__(BOUND_WAVES * 64) block_bounds_kernel(BlockSelect x, int tokens, int stride, uint32_t *out) {
    constexpr int KS = (D + 63) / 64, AHEAD = bound_ahead(D), SPAN = BOUND_WAVES * AHEAD * 16;
    __shared__ kv_i4 ops[BOUND_TILES][2][KS * 64];
    __shared__ RowsOf of[BOUND_TILES];
    __shared__ uint32_t keys[16 * BOUND_TILES * SPAN];
    const SelectView v(x, blockIdx.x, blockIdx.y * tokens, tokens);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int from = v.lead + blockIdx.z * SPAN;  // blocks from .. from + SPAN - 1, those of them that are coded
    if (from >= v.coded) return;
    const int blocks = min(v.coded - from, SPAN);
    Summaries<D, AHEAD, BOUND_WAVES> sum;
    sum.load(x.b, v.bh, from + wave * 16, v.coded - 1, lane);  // (in flight while the queries are made ready)
    for (int i = threadIdx.x; i < v.toks * SPAN; i += BOUND_WAVES * 64) keys[i] = 0;
    for (int row0 = 0; row0 < v.rows; row0 += 16 * BOUND_TILES) {
        const int tiles = min((v.rows - row0 + 15) / 16, BOUND_TILES);
        if (row0) __syncthreads();
        if (wave < tiles) {
            int tok;
            const char *row = v.row(x, row0 + 16 * wave + (lane & 15), tok);
            query_operands<D, DT>(row, tok, x.b.Dk_user, lane, ops[wave][0], ops[wave][1], of[wave]);
        }
        __syncthreads();
        for (int tile = 0; tile < tiles; ++tile)
            sum.bounds(ops[tile][0], ops[tile][1], of[tile], keys, SPAN, wave * 16, blocks, lane);
    }
    __syncthreads();
    for (int tok = 0; tok < v.toks; ++tok) {
        uint32_t *to = out + ((size_t)v.bh * x.L + v.tok0 + tok) * stride + (from - v.lead);
        for (int i = threadIdx.x; i < blocks; i += BOUND_WAVES * 64) to[i] = keys[tok * SPAN + i];
    }
}
// grid (BH, tokens), 16 wavefronts
constexpr int CHOOSE_WAVES = 16, CHOOSE_AREA = choose_area(CHOOSE_WAVES);
__global__ void __launch_bounds__(CHOOSE_WAVES * 64) block_choose_kernel(BlockSelect x, int stride, const uint32_t *in) {
    extern __shared__ uint32_t lds[];  // [CHOOSE_AREA], keys [stride]
    const SelectView v(x, blockIdx.x, blockIdx.y, 1);
    uint32_t *keys = lds + CHOOSE_AREA;
    const uint32_t *from = in + ((size_t)v.bh * x.L + v.tok0) * stride;
    const int seen = v.seen(x, 0);
    if (seen > x.count) {
#pragma unroll 4
        for (int i = threadIdx.x; i < seen - x.recent; i += CHOOSE_WAVES * 64) keys[i] = from[i];
        __syncthreads();
    }
    choose<CHOOSE_WAVES>(keys, lds, threadIdx.x & 63, v.lead, seen, x.count, x.first, x.recent, x.list + ((size_t)v.bh * x.L + v.tok0) * x.count);
}

// How a call is cut: tokens a workgroup takes, the keys it keeps for each, and whether bounds and choice are apart.
constexpr int SELECT_LDS = 156 << 10;
constexpr size_t BOUND_KEYS = (size_t)64 << 20;  // bytes of keys between the two launches, at most
struct SelectPlan {
    int tokens, stride, stretches;  // stretches 0: one launch
};
size_t select_ops(const BlockSelect &x) { return (size_t)SELECT_TILES * 2 * ((x.b.st.Dk + 63) / 64) * 64 * 16; }
SelectPlan select_plan(const BlockSelect &x) {
    const int G = x.Hq / x.Hkv;
    SelectPlan p;
    p.stride = (x.T + BLOCK_ROWS - 1) / BLOCK_ROWS;
    p.stretches = 0;
    p.tokens = std::min(std::max(1, 16 * SELECT_TILES / G), SELECT_WAVES);
    p.tokens = (int)std::min<int64_t>(p.tokens, (int64_t)(SELECT_LDS - SELECT_HEAD - select_ops(x)) / 4 / std::max(p.stride, 1));
    p.tokens = std::min(p.tokens, x.L);
    if (p.tokens < 1) return p;
    const int64_t groups = (int64_t)x.b.st.BH * ((x.L + p.tokens - 1) / p.tokens);
    const int span = BOUND_WAVES * 16 * bound_ahead(x.b.st.Dk);
    // (workgroups enough for half the chip, or one stretch of blocks: one launch)
    if (groups < 128 && p.stride > 128 && (size_t)x.b.st.BH * x.L * p.stride * 4 <= BOUND_KEYS) {
        p.tokens = std::min(p.tokens, std::max(1, 16 * BOUND_TILES / G));
        p.stretches = (p.stride + span - 1) / span;
    }
    return p;
}
template <int D, int DT> hipError_t select_run(const BlockSelect &x, hipStream_t stream) {
    const SelectPlan p = select_plan(x);
    const unsigned groups = (x.L + p.tokens - 1) / p.tokens;
    if (p.stretches) {
        uint32_t *keys = static_cast<uint32_t *>(x.workspace);
        hipLaunchKernelGGL((block_bounds_kernel<D, DT>), dim3(x.b.st.BH, groups, p.stretches), dim3(BOUND_WAVES * 64), 0, stream, x, p.tokens, p.stride, keys);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess || x.bounds_only) return e;
        const size_t lds = 4 * (size_t)(CHOOSE_AREA + p.stride);
        if (lds > 65536) {
            e = hipFuncSetAttribute(reinterpret_cast<const void *>(block_choose_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, SELECT_LDS);
            if (e != hipSuccess) return e;
        }
        hipLaunchKernelGGL(block_choose_kernel, dim3(x.b.st.BH, x.L), dim3(CHOOSE_WAVES * 64), lds, stream, x, p.stride, keys);
        return hipGetLastError();
    }
    const size_t lds = SELECT_HEAD + select_ops(x) + (size_t)p.tokens * p.stride * 4;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(block_select_kernel<D, DT>), hipFuncAttributeMaxDynamicSharedMemorySize, SELECT_LDS);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((block_select_kernel<D, DT>), dim3(x.b.st.BH, groups), dim3(SELECT_WAVES * 64), lds, stream, x, p.tokens, p.stride);
    return hipGetLastError();
}
template <int DT> hipError_t select_dtype(const BlockSelect &x, hipStream_t stream) {
    switch (x.b.st.Dk) {
        case 64: return select_run<64, DT>(x, stream);
        case 96: return select_run<96, DT>(x, stream);
        case 128: return select_run<128, DT>(x, stream);
        case 192: return select_run<192, DT>(x, stream);
        case 256: return select_run<256, DT>(x, stream);
    }
    return hipErrorInvalidValue;
}

}  // namespace

bool block_select_supported(const BlockSelect &x) { return select_plan(x).tokens >= 1; }  // (the keys of one token fit)
int block_select_stride(const BlockSelect &x) {
    const SelectPlan p = select_plan(x);
    return p.stretches ? p.stride : 0;
}
size_t block_select_workspace(const BlockSelect &x) {
    const SelectPlan p = select_plan(x);
    return p.stretches ? (size_t)x.b.st.BH * x.L * p.stride * 4 : 0;
}
hipError_t launch_block_select(const BlockSelect &x, hipStream_t stream) {
    return x.b.st.dtype == KVHIP_F16 ? select_dtype<0>(x, stream) : select_dtype<1>(x, stream);
}

}  // namespace kvhip
