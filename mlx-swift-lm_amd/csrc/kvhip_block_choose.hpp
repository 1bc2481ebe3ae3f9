// A token's blocks from the keys of their bounds: used by the choice's own launch and by the attention over what it chooses.
#pragma once
#include "kvhip_block.hpp"

namespace kvhip {

namespace {

// inclusive prefix sums over the lanes
__device__ __forceinline__ int wave_scan_int(int v) {
#define KV_SCAN_STEP(CTRL, ROWS, ZERO) v += __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, ZERO)
    KV_SCAN_STEP(0x111, 0xF, true);  // row_shr:1, 2, 4, 8
    KV_SCAN_STEP(0x112, 0xF, true);
    KV_SCAN_STEP(0x114, 0xF, true);
    KV_SCAN_STEP(0x118, 0xF, true);
    KV_SCAN_STEP(0x142, 0xA, false);  // row_bcast:15 into rows 1 and 3, row_bcast:31 into rows 2 and 3
    KV_SCAN_STEP(0x143, 0xC, false);
#undef KV_SCAN_STEP
    return v;
}
// over the lanes, in each of them
__device__ __forceinline__ uint32_t wave_or(uint32_t v) {
#define KV_OR_STEP(CTRL, ROWS) v |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false)
    KV_OR_STEP(0xB1, 0xF);   // quad_perm [1,0,3,2], [2,3,0,1], row_half_mirror, row_mirror
    KV_OR_STEP(0x4E, 0xF);
    KV_OR_STEP(0x141, 0xF);
    KV_OR_STEP(0x140, 0xF);
    KV_OR_STEP(0x142, 0xA);  // row_bcast:15, row_bcast:31: all of them in lane 63
    KV_OR_STEP(0x143, 0xC);
#undef KV_OR_STEP
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// words of LDS that a choice by `team` wavefronts works in
constexpr int choose_area(int team) { return 260 + 2 * team; }

// A token's list: `count` of the blocks lead .. lead + seen - 1, the first `first` and the last `recent` of them and the
// best of the others by their keys (row[i]: block lead + i), in ascending order.  TEAM wavefronts: the whole workgroup's token
// (where there are few: what it lasts is a chain of passes over the keys, which more wavefronts make short); 1: the wavefront's own.
//
// The smallest chosen key is found digit by digit, eight bits at a time from the first bit in which the keys differ (their
// exponents mostly agree: from bit 31 on nearly all fall into one bin, and one address takes one addition a cycle), until
// a bin is taken whole.  `area`: 256 bins and, behind them, the differing bits and a pair of counts for each wavefront (TEAM > 1).
template <int TEAM>
__device__ __forceinline__ void choose(const uint32_t *row, uint32_t *area, int lane, int lead, int seen, int count, int first, int recent, int32_t *out) {
    constexpr int T = TEAM * 64;
    const int t = TEAM > 1 ? threadIdx.x : lane, wave = TEAM > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    auto sync = [] {
        if constexpr (TEAM > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    };
    if (seen <= count) {
        for (int i = t; i < count; i += T) out[i] = i < seen ? lead + i : -1;
        return;
    }
    const int end = seen - recent;
    int want = count - first - recent;  // of the blocks first .. end - 1
    const bool ranked = want > 0;
    uint32_t prefix = 0;                // a key is above the line if key >> shift > prefix, on it if they are equal
    int shift = 0, ties = 0;            // the first `ties` blocks on the line are chosen
    uint32_t *bins = area;
    if (ranked) {
        const uint32_t one = row[first];
        uint32_t differ = 0;
#pragma unroll 4
        for (int i = first + t; i < end; i += T) differ |= row[i] ^ one;
        differ = wave_or(differ);
        if constexpr (TEAM > 1) {
            if (t == 0) area[256] = 0;
            __syncthreads();
            if (lane == 0 && differ) atomicOr(&area[256], differ);
            __syncthreads();
            differ = area[256];
        }
        int bits = differ ? 32 - __builtin_clz(differ) : 0;  // keys agree in the bits from here up
        prefix = bits < 32 ? one >> bits : 0u;
        shift = bits;
        while (true) {
            if (bits == 0) {
                ties = want;
                break;
            }
            const int step = bits < 8 ? bits : 8;
            shift = bits - step;
            for (int i = t; i < 256; i += T) bins[i] = 0;
            sync();
#pragma unroll 4
            for (int i = first + t; i < end; i += T) {
                const uint32_t k = row[i];
                if (bits == 32 || (k >> bits) == prefix) atomicAdd(&bins[(k >> shift) & ((1u << step) - 1u)], 1u);
            }
            sync();
            // the lane's bins, from the top: 255 - 4 lane to 252 - 4 lane (every wavefront for itself)
            int c[4], mine = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[i] = (int)bins[255 - 4 * lane - i];
                mine += c[i];
            }
            const int upto = wave_scan_int(mine);
            int run = upto - mine, digit = 0, above = 0, here = 0;
            const int at = __builtin_ctzll(__ballot(run < want && upto >= want));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (run < want && run + c[i] >= want) {
                    digit = 255 - 4 * lane - i;
                    above = run;
                    here = c[i];
                }
                run += c[i];
            }
            digit = __builtin_amdgcn_readlane(digit, at);
            want -= __builtin_amdgcn_readlane(above, at);
            here = __builtin_amdgcn_readlane(here, at);
            prefix = bits == 32 ? (uint32_t)digit : (prefix << step) | (uint32_t)digit;
            bits = shift;
            if (want == here) {
                ties = here;
                break;
            }
            if constexpr (TEAM > 1) __syncthreads();  // (the bins are cleared again)
        }
    }
    // blocks in 64s: those above the line, and the first `ties` on it
    const int groups = (seen + 63) / 64;
    const uint64_t below = (1ull << lane) - 1;
    auto look = [&](int group, bool &above, bool &line) {
        const int i = group * 64 + lane;
        const bool in = ranked && i >= first && i < end;
        const uint32_t k = in ? row[i] >> shift : 0u;
        above = i < first || (i >= end && i < seen) || (in && k > prefix);
        line = in && k == prefix;
    };
    auto write = [&](int group, bool above, uint64_t line, int left, int filled) {
        const bool take = above || ((line >> lane) & 1 && __builtin_popcountll(line & below) < left);
        const uint64_t taken = __ballot(take);
        if (take) out[filled + __builtin_popcountll(taken & below)] = lead + group * 64 + lane;
    };
    if constexpr (TEAM > 1) {
        // a wavefront to a stretch of groups, behind what the wavefronts before it hold
        uint32_t *counts = area + 257;  // [TEAM][2]
        const int each = (groups + TEAM - 1) / TEAM, g0 = wave * each, g1 = min(g0 + each, groups);
        int a = 0, l = 0;
        for (int group = g0; group < g1; ++group) {
            bool above, line;
            look(group, above, line);
            a += __builtin_popcountll(__ballot(above));
            l += __builtin_popcountll(__ballot(line));
        }
        if (lane == 0) counts[2 * wave] = a, counts[2 * wave + 1] = l;
        __syncthreads();
        int filled = 0, lines = 0;
        for (int w = 0; w < wave; ++w) {
            filled += (int)counts[2 * w];
            lines += (int)counts[2 * w + 1];
        }
        filled += min(lines, ties);
        int left = max(ties - lines, 0);
        for (int group = g0; group < g1; ++group) {
            bool above, line;
            look(group, above, line);
            const uint64_t on = __ballot(line);
            write(group, above, on, left, filled);
            filled += __builtin_popcountll(__ballot(above)) + min(left, (int)__builtin_popcountll(on));
            left -= min(left, (int)__builtin_popcountll(on));
        }
    } else {
        int filled = 0, left = ties;
        for (int group = 0; group < groups; ++group) {
            bool above, line;
            look(group, above, line);
            const uint64_t on = __ballot(line);
            write(group, above, on, left, filled);
            filled += __builtin_popcountll(__ballot(above)) + min(left, (int)__builtin_popcountll(on));
            left -= min(left, (int)__builtin_popcountll(on));
        }
    }
}

}  // namespace

}  // namespace kvhip
