// Blocks for each token from a bound on what they hold (summaries: kvhip_block.hpp).
//
// A query row's bound on a block is sum_d max(q_d hi_d, q_d lo_d), with hi and lo the block's largest and smallest key element
// of each channel: no key of the block scores higher.  Both sides are whole numbers times powers of two -- hi and lo are int8
// in units of 4 scales, q is rint(q 2^-f), f the least integer with max |q| 2^-f <= 127 -- so that the sum is exact whatever
// its order (below 2^24 for 256 channels) and the choice the same on any machine.  As products:
// q+ hi + q- lo, with q+ = max(q, 0) and q- = min(q, 0), on the 16x16x64 int8 instruction.
#include <algorithm>

#include "kvhip_block.hpp"
#include "kvhip_wave.hpp"

namespace kvhip {

namespace {

typedef int kv_i4 __attribute__((ext_vector_type(4)));

// floats in an order that unsigned integers have too; 0 is below all of them
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ int wave_scan_int(int v) {  // inclusive
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        if ((int)(threadIdx.x & 63) >= d) v += o;
    }
    return v;
}

constexpr int SELECT_WAVES = 4;
constexpr uint32_t ALWAYS = 0xffffffffu;  // the key of a block that is always chosen; 0: of one that the token does not see

// grid (BH, groups of `tokens` tokens), 256 threads.  LDS: keys [tokens][stride] of the blocks from `lead` on, and a
// histogram of 256 bins for each wavefront.
template <int D, int DT>
__global__ void __launch_bounds__(SELECT_WAVES * 64) block_select_kernel(BlockSelect x, int tokens, int stride) {
    constexpr int KS = (D + 63) / 64;
    extern __shared__ uint32_t lds[];
    uint32_t *hist = lds;                             // [waves][256]
    uint32_t *keys = lds + SELECT_WAVES * 256;        // [tokens][stride]
    const Store &st = x.b.st;
    const int bh = blockIdx.x, b = bh / x.Hkv, G = x.Hq / x.Hkv;
    const int tok0 = blockIdx.y * tokens, toks = min(tokens, x.L - tok0);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    const int pad = x.left_pad ? max(x.left_pad[b], 0) : 0;
    const int lead = pad / BLOCK_ROWS;
    const int top = (x.T - x.L + tok0 + toks - 1) / BLOCK_ROWS;  // the last token's own block

    for (int i = threadIdx.x; i < toks * stride; i += SELECT_WAVES * 64) keys[i] = 0;
    __syncthreads();

    // bounds: 16 query rows (token by token, a token's heads side by side) by 16 blocks at a time
    const int ud = x.b.Dk_user;
    for (int r0 = 0; r0 < toks * G; r0 += 16) {
        const int r = r0 + n;
        const bool live = r < toks * G;
        const int tok = live ? r / G : 0, head = live ? r % G : 0;
        const char *row = static_cast<const char *>(x.q) + (((size_t)bh * G + head) * x.L + tok0 + tok) * ud * 2;
        kv_i4 pos[KS], neg[KS];
        float v[KS][16], amax = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const int d = s * 64 + g * 16 + k;
                float y = live && d < ud ? Elem<DT>::load(row, d) : 0.f;
                if (!(fabsf(y) < INFINITY)) y = 0.f;  // (elements that are no numbers have no say)
                v[s][k] = y;
                amax = fmaxf(amax, fabsf(y));
            }
        amax = fmaxf(amax, __shfl_xor(amax, 16));
        amax = fmaxf(amax, __shfl_xor(amax, 32));
        // (frexp: also of the values below the smallest normal one)
        int ex = 0;
        const float mant = frexpf(amax, &ex);
        const int f = amax > 0.f ? ex - 7 + (mant > 127.f / 128.f ? 1 : 0) : 0;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                int p = 0, m = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i = (int)rintf(ldexpf(v[s][4 * w + k], -f));
                    p |= (max(i, 0) & 0xff) << (8 * k);
                    m |= (min(i, 0) & 0xff) << (8 * k);
                }
                pos[s][w] = p;
                neg[s][w] = m;
            }
        int fr[4], tr[4];  // the four rows whose bounds the lane will hold
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            fr[i] = __shfl(f, 4 * g + i);
            tr[i] = r0 + 4 * g + i < toks * G ? (r0 + 4 * g + i) / G : -1;
        }
        const int coded = min(x.b.coded, top);  // (the last token's own block is always chosen)
        for (int n0 = lead + 16 * wave; n0 < coded; n0 += 16 * SELECT_WAVES) {
            const int blk = min(n0 + n, coded - 1);
            const PageEntry &e = st.pt[blk / BLOCK_PER_PAGE];
            const char *sum = e.vsb + (size_t)bh * st.vsb_cell + (size_t)(blk % BLOCK_PER_PAGE) * 2 * D;
            const float scale = reinterpret_cast<const float *>(e.ksb + (size_t)bh * st.ksb_cell)[2 * (blk % BLOCK_PER_PAGE)];
            kv_i4 acc{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = s * 64 + g * 16;
                kv_i4 hi{0, 0, 0, 0}, lo{0, 0, 0, 0};
                if (d < D) {
                    hi = *reinterpret_cast<const kv_i4 *>(sum + d);
                    lo = *reinterpret_cast<const kv_i4 *>(sum + D + d);
                }
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(pos[s], hi, acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(neg[s], lo, acc, 0, 0, 0);
            }
            if (n0 + n < coded) {
                uint32_t key[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) key[i] = ordered(ldexpf((float)acc[i] * (4.f * scale), fr[i]));
                // (rows of one token side by side: one entry for all four)
                if (tr[0] >= 0 && tr[0] == tr[3]) {
                    atomicMax(&keys[tr[0] * stride + blk - lead], max(max(key[0], key[1]), max(key[2], key[3])));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (tr[i] >= 0) atomicMax(&keys[tr[i] * stride + blk - lead], key[i]);
                }
            }
        }
    }
    __syncthreads();

    // the choice: a wavefront to a token
    for (int tok = wave; tok < toks; tok += SELECT_WAVES) {
        const int p = x.T - x.L + tok0 + tok, last = p / BLOCK_ROWS;
        const int seen = p < pad ? 0 : last - lead + 1;  // candidates lead .. last
        uint32_t *row = keys + (size_t)tok * stride;
        int32_t *out = x.list + ((size_t)bh * x.L + tok0 + tok) * x.count;
        if (seen <= x.count) {
            for (int i = lane; i < x.count; i += 64) out[i] = i < seen ? lead + i : -1;
            continue;
        }
        auto key_at = [&](int i) -> uint32_t {
            if (i >= seen) return 0u;
            if (i < x.first || lead + i > last - x.recent) return ALWAYS;
            return min(max(row[i], 1u), ALWAYS - 1u);
        };
        // the count-th largest key, eight bits at a time
        uint32_t prefix = 0, want = x.count;
        uint32_t *bins = hist + wave * 256;
        for (int shift = 24; shift >= 0; shift -= 8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) bins[4 * lane + i] = 0;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
            for (int i = lane; i < seen; i += 64) {
                const uint32_t k = key_at(i);
                if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&bins[(k >> shift) & 255u], 1u);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
            // lane's bins from the top: 255 - 4 lane down to 252 - 4 lane
            uint32_t c[4];
            int mine = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[i] = bins[255 - 4 * lane - i];
                mine += (int)c[i];
            }
            const int upto = wave_scan_int(mine), before = upto - mine;
            const uint64_t found = __ballot(before < (int)want && upto >= (int)want);
            const int at = __builtin_ctzll(found);
            int digit = 0, above = 0, run = before;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (run < (int)want && run + (int)c[i] >= (int)want) {
                    digit = 255 - 4 * lane - i;
                    above = run;
                }
                run += (int)c[i];
            }
            digit = __shfl(digit, at);
            above = __shfl(above, at);
            prefix = (prefix << 8) | (uint32_t)digit;
            want -= (uint32_t)above;
        }
        // everything above it, and the first `want` blocks that equal it, in ascending order
        int filled = 0;
        uint32_t equal = want;
        for (int i0 = 0; i0 < seen; i0 += 64) {
            const uint32_t k = key_at(i0 + lane);
            const uint64_t below = (1ull << lane) - 1;
            const uint64_t eq = __ballot(k == prefix);
            const bool take = k > prefix || (k == prefix && (uint32_t)__builtin_popcountll(eq & below) < equal);
            const uint64_t taken = __ballot(take);
            if (take) out[filled + __builtin_popcountll(taken & below)] = lead + i0 + lane;
            filled += __builtin_popcountll(taken);
            equal -= min(equal, (uint32_t)__builtin_popcountll(eq));
        }
    }
}

constexpr int SELECT_LDS = 144 << 10;
// tokens a workgroup takes and the keys it keeps for each
void select_plan(const BlockSelect &x, int &tokens, int &stride) {
    const int G = x.Hq / x.Hkv;
    stride = (x.T + BLOCK_ROWS - 1) / BLOCK_ROWS;
    tokens = std::max(1, 16 / G);
    tokens = (int)std::min<int64_t>(tokens, (SELECT_LDS - SELECT_WAVES * 1024) / 4 / std::max(stride, 1));
}
template <int DT> hipError_t select_dtype(const BlockSelect &x, hipStream_t stream) {
    int tokens, stride;
    select_plan(x, tokens, stride);
    const dim3 grid(x.b.st.BH, (x.L + tokens - 1) / tokens), block(SELECT_WAVES * 64);
    const size_t lds = SELECT_WAVES * 1024 + (size_t)tokens * stride * 4;
#define KV_SELECT(D)                                                                                                    \
    do {                                                                                                                \
        if (lds > 65536) {                                                                                              \
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(block_select_kernel<D, DT>),        \
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, SELECT_LDS);           \
            if (e != hipSuccess) return e;                                                                              \
        }                                                                                                               \
        hipLaunchKernelGGL((block_select_kernel<D, DT>), grid, block, lds, stream, x, tokens, stride);                  \
        return hipGetLastError();                                                                                       \
    } while (0)
    switch (x.b.st.Dk) {
        case 64: KV_SELECT(64);
        case 96: KV_SELECT(96);
        case 128: KV_SELECT(128);
        case 192: KV_SELECT(192);
        case 256: KV_SELECT(256);
    }
#undef KV_SELECT
    return hipErrorInvalidValue;
}

}  // namespace

bool block_select_supported(const BlockSelect &x) {
    int tokens, stride;
    select_plan(x, tokens, stride);
    return tokens >= 1;
}
hipError_t launch_block_select(const BlockSelect &x, hipStream_t stream) {
    return x.b.st.dtype == KVHIP_F16 ? select_dtype<0>(x, stream) : select_dtype<1>(x, stream);
}

}  // namespace kvhip
