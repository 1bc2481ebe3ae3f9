// Rows into the block-scaled cache and back out of it (layout and arithmetic: kvhip_block.hpp).
#include "kvhip_block.hpp"

namespace kvhip {

namespace {

typedef uint32_t kv_w2 __attribute__((ext_vector_type(2)));

// A workgroup's threads over a block: 16 groups of four adjacent rows by 16 chunks of eight channels, in turns of 128 channels.
struct Unit {
    int rq, ch;  // row quad, chunk inside the turn
    __device__ __forceinline__ Unit() : rq(threadIdx.x >> 4), ch(threadIdx.x & 15) {}
};

// Eight channels from d0 of row `row` of a dense array of `ud` channels as words of two (zeros past the end).
__device__ __forceinline__ kv_u4 raw_chunk(const char *src, size_t row, int ud, int d0) {
    const char *p = src + (row * ud + d0) * 2;
    kv_u4 w{0u, 0u, 0u, 0u};
    if (d0 + 8 <= ud) {
        w = load_row16(p);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (d0 + i < ud) w[i >> 1] |= (uint32_t) reinterpret_cast<const uint16_t *>(p)[i] << (16 * (i & 1));
    }
    return w;
}
// the same with infinities as NaN
template <int DT> __device__ __forceinline__ kv_u4 dense_chunk(const char *src, size_t row, int ud, int d0) {
    kv_u4 w = raw_chunk(src, row, ud, d0);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = no_infinities<DT>(w[i]);
    return w;
}

// Eight channels of a row of the block as the cache holds it: from the codes, or from the tail.
template <int DT, bool V>
__device__ __forceinline__ kv_u4 held_chunk(const char *codes, const char *tail, bool coded, float scale, int D, int r, int d0) {
    kv_u4 w;
    if (coded) {
        if constexpr (V) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t c0 = (uint8_t)codes[block_v_at(r, d0 + 2 * i)], c1 = (uint8_t)codes[block_v_at(r, d0 + 2 * i + 1)];
                w[i] = block_values<DT, false>(c0 | (c1 << 8), scale);
            }
        } else {
            const kv_w2 c = *reinterpret_cast<const kv_w2 *>(codes + block_k_at(D, r, d0));
            w = kv_u4{block_values<DT, false>(c[0], scale), block_values<DT, true>(c[0], scale), block_values<DT, false>(c[1], scale),
                      block_values<DT, true>(c[1], scale)};
        }
    } else if constexpr (V) {
        const uint16_t *t = reinterpret_cast<const uint16_t *>(tail);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = (uint32_t)t[tail_v_at(D, r, d0 + 2 * i)] | ((uint32_t)t[tail_v_at(D, r, d0 + 2 * i + 1)] << 16);
    } else {
        w = *reinterpret_cast<const kv_u4 *>(tail + ((size_t)r * D + d0) * 2);
    }
    return w;
}

// Two elements of a word as they order: signed 16-bit integers in place of sign and magnitude.
typedef short kv_s2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ kv_s2 ordered2(uint32_t w) {
    const kv_s2 v = __builtin_bit_cast(kv_s2, w);
    return v ^ ((v >> 15) & (short)0x7fff);
}
__device__ __forceinline__ kv_s2 max2(kv_s2 a, kv_s2 b) { return __builtin_elementwise_max(a, b); }
__device__ __forceinline__ kv_s2 min2(kv_s2 a, kv_s2 b) { return __builtin_elementwise_min(a, b); }
template <int DT> __device__ __forceinline__ float float_of(uint32_t h) {  // of an element's bits
    return DT == 1 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half((unsigned short)h));
}
// the largest magnitude that four significant bits can hold of the type: 1.875 2^127, 1.875 2^15
template <int DT> constexpr uint32_t TOP_BITS = DT == 1 ? 0x7f70u : 0x7b80u;
// An element as it is coded: its magnitude at most that, infinities as NaN.
template <int DT> __device__ __forceinline__ uint32_t element_to_code(uint32_t h) {
    constexpr uint32_t INF = DT == 1 ? 0x7f80u : 0x7c00u;
    const uint32_t a = h & 0x7fffu;
    return a >= INF ? (INF | 1u) : a > TOP_BITS<DT> ? (h & 0x8000u) | TOP_BITS<DT> : h;
}
template <int DT> __device__ __forceinline__ uint32_t word_to_code(uint32_t w) {
    return element_to_code<DT>(w & 0xffffu) | (element_to_code<DT>(w >> 16) << 16);
}
// the magnitudes of two elements where they are numbers, else 0
template <int DT> __device__ __forceinline__ uint32_t finite_magnitudes(uint32_t w) {
    const uint32_t lo = w & 0x7fffu, hi = (w >> 16) & 0x7fffu;
    return (lo > TOP_BITS<DT> ? 0u : lo) | ((hi > TOP_BITS<DT> ? 0u : hi) << 16);
}
typedef unsigned short kv_us2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t umax2(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(kv_us2, a), __builtin_bit_cast(kv_us2, b)));
}
// Two elements as two codes, divided by the scale on the way, in the low or high half of a word.
template <int DT, bool HIGH> __device__ __forceinline__ uint32_t two_codes(uint32_t old, uint32_t w, float scale) {
    const kv_s2 o = __builtin_bit_cast(kv_s2, old);
    if constexpr (DT == 1) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(o, __builtin_bit_cast(kv_b2, w), scale, HIGH));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(o, __builtin_bit_cast(kv_h2, w), scale, HIGH));
}
// the exponent of a block whose largest magnitude has these bits
template <int DT> __device__ __forceinline__ int block_exponent(uint32_t magnitude) {
    const uint32_t bits = __float_as_uint(float_of<DT>(magnitude));
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return magnitude ? max(e, BLOCK_LEAST_EXP) : 0;
}
// the summary's unit of a channel's extreme: its code, a quarter of it rounded
template <int DT> __device__ __forceinline__ int summary_unit(uint32_t h, float scale) {
    const uint32_t c = two_codes<DT, false>(0u, h, scale);
    return (int)rintf(__builtin_amdgcn_cvt_f32_fp8((int)c, 0) * 0.25f);
}

struct AppendArgs {
    BlockStore s;
    const char *src;  // the plane's rows [BH, n, ud]
    int64_t pos0;
    int n, ud;
    int blk, bh;
    bool reopened;    // the block is held as codes and has lost rows since
    __device__ __forceinline__ int64_t lo() const { return (int64_t)blk * BLOCK_ROWS; }
    __device__ __forceinline__ int from() const { return (int)(pos0 > lo() ? pos0 - lo() : 0); }                                  // rows held so far
    __device__ __forceinline__ int upto() const { return (int)(pos0 + n - lo() < BLOCK_ROWS ? pos0 + n - lo() : BLOCK_ROWS); }  // after the call
    __device__ __forceinline__ const char *rows() const { return src + (size_t)bh * n * ud * 2; }
};

// New rows of a block that stays unfinished, into its place (behind those of a reopened one).
template <int DT, int D, bool V>
__device__ __forceinline__ void append_tail(const AppendArgs &a, const char *codes, const char *tail, char *to, float scale) {
    const int start = a.reopened ? 0 : a.from(), upto = a.upto(), from = a.from();
    const Unit u;
    const int r0 = 4 * u.rq;
    const bool all = r0 >= start && r0 + 4 <= upto;
    for (int d0 = 8 * u.ch; d0 < D; d0 += 128) {
        kv_u4 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + i;
            if (r >= start && r < upto)
                w[i] = r < from ? held_chunk<DT, V>(codes, tail, true, scale, D, r, d0) : dense_chunk<DT>(a.rows(), (size_t)(a.lo() + r - a.pos0), a.ud, d0);
        }
        if constexpr (V) {
            uint16_t *t = reinterpret_cast<uint16_t *>(to);
            if (all) {  // four rows of a channel lie side by side
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint32_t pick = k & 1 ? 0x07060302u : 0x05040100u;
                    *reinterpret_cast<kv_w2 *>(t + tail_v_at(D, r0, d0 + k)) =
                        kv_w2{__builtin_amdgcn_perm(w[1][k >> 1], w[0][k >> 1], pick), __builtin_amdgcn_perm(w[3][k >> 1], w[2][k >> 1], pick)};
                }
                continue;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + i;
            if (r < start || r >= upto) continue;
            if constexpr (V) {
                uint16_t *t = reinterpret_cast<uint16_t *>(to);
#pragma unroll
                for (int k = 0; k < 8; ++k) t[tail_v_at(D, r, d0 + k)] = (uint16_t)(w[i][k >> 1] >> (16 * (k & 1)));
            } else {
                *reinterpret_cast<kv_u4 *>(to + ((size_t)r * D + d0) * 2) = w[i];
            }
        }
    }
}

// A block that is whole after this call: its rows (those held so far and the new ones) become codes and, of the call's last such
// block, stay in `keep` as they came.  A wavefront takes what it can write out in whole lines, straight from registers; the
// largest magnitude meets in LDS.  Elements are two to a word: magnitudes and channel extremes are packed integer maxima, the
// division by the scale and the rounding one conversion for two.  Elements past the largest that can be coded (infinities and NaN among them) are seen to where a
// thread has met one.  Bound by memory, 2 bytes read and 1 written an element: 8 x 8 heads x 2048 rows x 128 20 us, 5.0 TB/s;
// 4 x 8 heads x 8191 rows 43 us, 4.7 TB/s, what a copy gives.
//
// Keys: a wavefront to 16 rows, a lane to one of them and 16 channels of every 64 (8 of a last 32).  Extremes of the channels
// go through LDS, each wavefront's own rows first.
template <int DT, int D>
__device__ __forceinline__ void append_keys(const AppendArgs &a, char *codes, const char *tail, char *keep, float *scale_out, char *summary,
                                            float held_scale, uint32_t *raw, uint32_t *ends, uint32_t *amax_s) {
    constexpr int KC = D / 64, CH = KC * 8 + (D % 64 ? 4 : 0);  // words of two a lane
    constexpr int PITCH = D / 2 + 4;                           // words of a row in LDS
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15, r = 16 * wave + m;
    const int from = a.from();
    uint32_t w[CH];
    auto channel = [&](int c) { return c < KC * 2 ? (c >> 1) * 64 + g * 16 + (c & 1) * 8 : KC * 64 + g * 8; };  // of chunk c of eight
    const char *rows = a.rows();
#pragma unroll
    for (int c = 0; c < CH / 4; ++c) {
        kv_u4 x;
        if (r < from) x = held_chunk<DT, false>(codes, tail, a.reopened, held_scale, D, r, channel(c));
        else x = raw_chunk(rows, (size_t)(a.lo() + r - a.pos0), a.ud, channel(c));
#pragma unroll
        for (int k = 0; k < 4; ++k) w[4 * c + k] = x[k];
    }
    if (keep && (r >= from || a.reopened)) {  // (its first rows are there already)
#pragma unroll
        for (int c = 0; c < CH / 4; ++c)
            *reinterpret_cast<kv_u4 *>(keep + ((size_t)r * D + channel(c)) * 2) = kv_u4{no_infinities<DT>(w[4 * c]), no_infinities<DT>(w[4 * c + 1]),
                                                                                       no_infinities<DT>(w[4 * c + 2]), no_infinities<DT>(w[4 * c + 3])};
    }
    uint32_t mag = 0;
#pragma unroll
    for (int k = 0; k < CH; ++k) mag = umax2(mag, w[k] & 0x7fff7fffu);
    const bool odd = (mag & 0xffffu) > TOP_BITS<DT> || (mag >> 16) > TOP_BITS<DT>;
    if (odd) {
        mag = 0;
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            w[k] = word_to_code<DT>(w[k]);
            mag = umax2(mag, finite_magnitudes<DT>(w[k]));
        }
    }
    // a wavefront's own rows: written, and read channel by channel
    uint32_t *mine = raw + wave * 16 * PITCH;
#pragma unroll
    for (int c = 0; c < CH / 4; ++c) *reinterpret_cast<kv_u4 *>(mine + m * PITCH + channel(c) / 2) = kv_u4{w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]};
    uint32_t any = max(mag & 0xffffu, mag >> 16);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) any = max(any, (uint32_t)__shfl_xor(any, d));
    if (lane == 0) amax_s[wave] = any;
    const bool strange = __any(odd);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    for (int c = lane; c < D / 2; c += 64) {
        kv_s2 hi{-32768, -32768}, lo{32767, 32767};
#pragma unroll 16
        for (int i = 0; i < 16; ++i) {
            const uint32_t x = mine[i * PITCH + c];
            kv_s2 o = ordered2(x), p = o;
            if (strange) {  // (NaN are no extremes)
                if ((x & 0x7fffu) > TOP_BITS<DT>) o[0] = -32768, p[0] = 32767;
                if (((x >> 16) & 0x7fffu) > TOP_BITS<DT>) o[1] = -32768, p[1] = 32767;
            }
            hi = max2(hi, o);
            lo = min2(lo, p);
        }
        ends[wave * D + c] = __builtin_bit_cast(uint32_t, hi);
        ends[wave * D + D / 2 + c] = __builtin_bit_cast(uint32_t, lo);
    }
    __syncthreads();
    const int e = block_exponent<DT>(max(max(amax_s[0], amax_s[1]), max(amax_s[2], amax_s[3])));
    const float scale = power_of_two(e);
#pragma unroll
    for (int c = 0; c < KC; ++c) {
        kv_u4 o;
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = two_codes<DT, true>(two_codes<DT, false>(0u, w[8 * c + 2 * k], scale), w[8 * c + 2 * k + 1], scale);
        *reinterpret_cast<kv_u4 *>(codes + wave * 16 * D + c * 1024 + lane * 16) = o;
    }
    if constexpr (D % 64 != 0) {
        kv_w2 o;
#pragma unroll
        for (int k = 0; k < 2; ++k) o[k] = two_codes<DT, true>(two_codes<DT, false>(0u, w[8 * KC + 2 * k], scale), w[8 * KC + 2 * k + 1], scale);
        *reinterpret_cast<kv_w2 *>(codes + wave * 16 * D + KC * 1024 + lane * 8) = o;
    }
    if (threadIdx.x == 0) *scale_out = scale;
    for (int c = threadIdx.x; c < D; c += 256) {  // the largest of two channels, then the smallest
        kv_s2 x = __builtin_bit_cast(kv_s2, ends[c]);
#pragma unroll
        for (int i = 1; i < 4; ++i) {
            const kv_s2 y = __builtin_bit_cast(kv_s2, ends[i * D + c]);
            x = c < D / 2 ? max2(x, y) : min2(x, y);
        }
        uint32_t unit = 0;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int v = x[k];
            const bool none = v == (c < D / 2 ? -32768 : 32767);  // (a channel of nothing but NaN)
            const uint32_t h = none ? 0u : (uint32_t)((v ^ ((v >> 15) & 0x7fff)) & 0xffff);
            unit |= (uint32_t)(summary_unit<DT>(h, scale) & 0xff) << (8 * k);
        }
        reinterpret_cast<uint16_t *>(summary)[c] = (uint16_t)unit;
    }
}

// Values: a wavefront to the 16 tokens 16 t + 4 wave + i, a lane to two channels of them (of every 128).
template <int DT, int D>
__device__ __forceinline__ void append_values(const AppendArgs &a, char *codes, const char *tail, char *keep, float *scale_out, float held_scale,
                                              uint32_t *amax_s) {
    constexpr int TURNS = (D + 127) / 128;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int from = a.from();
    const char *rows = a.rows() + (a.lo() - a.pos0) * a.ud * 2;
    const uint16_t *t = reinterpret_cast<const uint16_t *>(tail);
    uint32_t w[TURNS][16], mag = 0;
#pragma unroll
    for (int turn = 0; turn < TURNS; ++turn) {
        const int d = turn * 128 + 2 * lane;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = 16 * (i >> 2) + 4 * wave + (i & 3);
            uint32_t x = 0;
            if (d < D) {
                if (r < from) {
                    if (a.reopened) {
                        const uint32_t c = (uint8_t)codes[block_v_at(r, d)] | ((uint32_t)(uint8_t)codes[block_v_at(r, d + 1)] << 8);
                        x = block_values<DT, false>(c, held_scale);
                    } else {
                        x = (uint32_t)t[tail_v_at(D, r, d)] | ((uint32_t)t[tail_v_at(D, r, d + 1)] << 16);
                    }
                } else if (d + 2 <= a.ud) {
                    x = *reinterpret_cast<const kv_out2 *>(rows + ((size_t)r * a.ud + d) * 2);
                } else if (d < a.ud) {
                    x = *reinterpret_cast<const uint16_t *>(rows + ((size_t)r * a.ud + d) * 2);
                }
            }
            w[turn][i] = x;
        }
    }
    if (keep) {  // (a lane's four tokens of a channel lie side by side)
        uint16_t *to = reinterpret_cast<uint16_t *>(keep);
#pragma unroll
        for (int turn = 0; turn < TURNS; ++turn) {
            const int d = turn * 128 + 2 * lane;
            if (d >= D) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (16 * k + 4 * wave + 4 <= from && !a.reopened) continue;
                uint32_t x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = no_infinities<DT>(w[turn][4 * k + i]);
                uint16_t *at = to + tail_v_at(D, 16 * k + 4 * wave, d);
                *reinterpret_cast<kv_w2 *>(at) = kv_w2{__builtin_amdgcn_perm(x[1], x[0], 0x05040100u), __builtin_amdgcn_perm(x[3], x[2], 0x05040100u)};
                *reinterpret_cast<kv_w2 *>(at + 8) = kv_w2{__builtin_amdgcn_perm(x[1], x[0], 0x07060302u), __builtin_amdgcn_perm(x[3], x[2], 0x07060302u)};
            }
        }
    }
#pragma unroll
    for (int turn = 0; turn < TURNS; ++turn)
#pragma unroll
        for (int i = 0; i < 16; ++i) mag = umax2(mag, w[turn][i] & 0x7fff7fffu);
    if ((mag & 0xffffu) > TOP_BITS<DT> || (mag >> 16) > TOP_BITS<DT>) {
        mag = 0;
#pragma unroll
        for (int turn = 0; turn < TURNS; ++turn)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                w[turn][i] = word_to_code<DT>(w[turn][i]);
                mag = umax2(mag, finite_magnitudes<DT>(w[turn][i]));
            }
    }
    uint32_t any = max(mag & 0xffffu, mag >> 16);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) any = max(any, (uint32_t)__shfl_xor(any, d));
    if (lane == 0) amax_s[wave] = any;
    __syncthreads();
    const int e = block_exponent<DT>(max(max(amax_s[0], amax_s[1]), max(amax_s[2], amax_s[3])));
    const float scale = power_of_two(e);
    if (threadIdx.x == 0) *scale_out = scale;
#pragma unroll
    for (int turn = 0; turn < TURNS; ++turn) {
        const int d = turn * 128 + 2 * lane;
        kv_u4 even, odd;
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // two channels of four tokens, token by token -> four tokens of either channel
            const uint32_t x = two_codes<DT, true>(two_codes<DT, false>(0u, w[turn][4 * k], scale), w[turn][4 * k + 1], scale);
            const uint32_t y = two_codes<DT, true>(two_codes<DT, false>(0u, w[turn][4 * k + 2], scale), w[turn][4 * k + 3], scale);
            even[k] = __builtin_amdgcn_perm(y, x, 0x06040200u);
            odd[k] = __builtin_amdgcn_perm(y, x, 0x07050301u);
        }
        if (d < D) {
            char *at = codes + block_v_at(4 * wave, d);
            *reinterpret_cast<kv_u4 *>(at) = even;
            *reinterpret_cast<kv_u4 *>(at + 16) = odd;
        }
    }
}

// grid (blocks touched, BH, keys / values), 256 threads.  Workgroups go to the eight dies in turn: where a pair has a multiple of eight of
// them, each pair begins with another block, since the ones that leave a block unfinished, the slowest, would all be on one die
// (4 x 8 heads of float16, us, so / without: 2000 rows 15.8 / 17.4, 4063 rows 22.6 / 24.8, 8191 rows 45.4 / 53.9; 8127 and 8255 rows, 127 and
// 129 workgroups a pair, spread by themselves: 44.3 and 44.6).
template <int DT, int DK, int DV>
__global__ void __launch_bounds__(256) block_append_kernel(BlockStore s, const char *keys, const char *values, int64_t pos0, int n, BlockKept to) {
    __shared__ __align__(16) uint32_t raw[64 * (DK / 2 + 4)];
    __shared__ uint32_t ends[4 * DK], amax_s[4];
    const bool v = blockIdx.z != 0;
    AppendArgs a;
    a.s = s;
    a.src = v ? values : keys;
    a.pos0 = pos0;
    a.n = n;
    a.ud = v ? s.Dv_user : s.Dk_user;
    const int done = (int)((pos0 + n) / BLOCK_ROWS) - 1;
    a.blk = (int)(pos0 / BLOCK_ROWS) + (int)(gridDim.x % 8 == 0 ? (blockIdx.x + blockIdx.y) % gridDim.x : blockIdx.x);
    a.bh = blockIdx.y;
    a.reopened = a.blk < s.coded && pos0 > a.lo();
    const PageEntry e = block_page(s, a.blk / BLOCK_PER_PAGE);
    const int in_page = a.blk % BLOCK_PER_PAGE, bh = a.bh;
    float *scales = reinterpret_cast<float *>(e.ksb + (size_t)bh * s.st.ksb_cell) + 2 * in_page + (v ? 1 : 0);
    const float held = a.reopened ? *scales : 1.f;
    const bool whole = pos0 + n >= a.lo() + BLOCK_ROWS, keep = a.blk == done;  // (the last whole block is kept as it came, too)
    if (v) {
        const size_t at = (size_t)bh * BLOCK_ROWS * DV * 2;
        char *codes = e.v + (size_t)bh * s.st.v_cell + (size_t)in_page * BLOCK_ROWS * DV;
        if (whole) append_values<DT, DV>(a, codes, s.tail_v + at, keep ? to.done_v + at : nullptr, scales, held, amax_s);
        else append_tail<DT, DV, true>(a, codes, s.tail_v + at, to.open_v + at, held);
    } else {
        const size_t at = (size_t)bh * BLOCK_ROWS * DK * 2;
        char *codes = e.k + (size_t)bh * s.st.k_cell + (size_t)in_page * BLOCK_ROWS * DK;
        char *summary = e.vsb + (size_t)bh * s.st.vsb_cell + (size_t)in_page * 2 * DK;
        if (whole) append_keys<DT, DK>(a, codes, s.tail_k + at, keep ? to.done_k + at : nullptr, scales, summary, held, raw, ends, amax_s);
        else append_tail<DT, DK, false>(a, codes, s.tail_k + at, to.open_k + at, held);
    }
}

// grid (blocks, BH, keys / values), 256 threads.  Codes through LDS into rows.  Bound by memory: 1 byte read and 2 written an
// element (4 x 8 heads x 8191 rows x 128: 34.5 us, 5.8 TB/s, the codes still in the last-level cache).
template <int DT, bool V>
__device__ __forceinline__ void fetch_block(const BlockStore &s, int64_t rows, char *dst, int blk, int bh, char *image) {
    const int D = V ? s.st.Dv : s.st.Dk, ud = V ? s.Dv_user : s.Dk_user;
    const int64_t lo = (int64_t)blk * BLOCK_ROWS;
    const int upto = (int)(rows - lo < BLOCK_ROWS ? rows - lo : BLOCK_ROWS);
    const bool coded = blk < s.coded;
    const PageEntry e = block_page(s, blk / BLOCK_PER_PAGE);
    const int in_page = blk % BLOCK_PER_PAGE;
    const char *tail = (V ? s.tail_v : s.tail_k) + (size_t)bh * BLOCK_ROWS * D * 2;
    char *out = dst + ((size_t)bh * rows + lo) * ud * 2;
    const Unit u;
    float scale = 1.f;
    if (coded) {
        const char *codes = (V ? e.v + (size_t)bh * s.st.v_cell : e.k + (size_t)bh * s.st.k_cell) + (size_t)in_page * BLOCK_ROWS * D;
        scale = reinterpret_cast<const float *>(e.ksb + (size_t)bh * s.st.ksb_cell)[2 * in_page + (V ? 1 : 0)];
        for (int i = threadIdx.x; i < BLOCK_ROWS * D / 16; i += 256)
            reinterpret_cast<kv_u4 *>(image)[i] = reinterpret_cast<const kv_u4 *>(codes)[i];
        __syncthreads();
    }
    for (int d0 = 8 * u.ch; d0 < ud; d0 += 128) {
        kv_u4 w[4];
        if (V && coded) {
            // four tokens of eight channels, channel by channel: pairs of tokens, put together into pairs of channels
#pragma unroll
            for (int k = 0; k < 8; k += 2) {
                const uint32_t c0 = *reinterpret_cast<const uint32_t *>(image + block_v_at(4 * u.rq, d0 + k));
                const uint32_t c1 = *reinterpret_cast<const uint32_t *>(image + block_v_at(4 * u.rq, d0 + k + 1));
                const uint32_t a0 = block_values<DT, false>(c0, scale), a1 = block_values<DT, true>(c0, scale);
                const uint32_t b0 = block_values<DT, false>(c1, scale), b1 = block_values<DT, true>(c1, scale);
                w[0][k >> 1] = (a0 & 0xffffu) | (b0 << 16);
                w[1][k >> 1] = (a0 >> 16) | (b0 & 0xffff0000u);
                w[2][k >> 1] = (a1 & 0xffffu) | (b1 << 16);
                w[3][k >> 1] = (a1 >> 16) | (b1 & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = held_chunk<DT, V>(image, tail, coded, scale, D, 4 * u.rq + i, d0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 4 * u.rq + i;
            if (r >= upto) continue;
            char *p = out + ((size_t)r * ud + d0) * 2;
            if (d0 + 8 <= ud) {
                *reinterpret_cast<kv_out8 *>(p) = w[i];
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (d0 + k < ud) reinterpret_cast<uint16_t *>(p)[k] = (uint16_t)(w[i][k >> 1] >> (16 * (k & 1)));
            }
        }
    }
}
template <int DT> __global__ void __launch_bounds__(256) block_fetch_kernel(BlockStore s, int64_t rows, char *dst_k, char *dst_v, int z0) {
    __shared__ __align__(16) char image[BLOCK_ROWS * BLOCK_MAX_HEAD];
    if ((int)blockIdx.z + z0) fetch_block<DT, true>(s, rows, dst_v, blockIdx.x, blockIdx.y, image);
    else fetch_block<DT, false>(s, rows, dst_k, blockIdx.x, blockIdx.y, image);
}

}  // namespace

hipError_t launch_block_append(const BlockStore &s, const void *keys, const void *values, int64_t pos0, int n, const BlockKept &to,
                               hipStream_t stream) {
    const int64_t first = pos0 / BLOCK_ROWS, last = (pos0 + n - 1) / BLOCK_ROWS;
    const dim3 grid((unsigned)(last - first + 1), s.st.BH, 2), block(256);
    const char *k = static_cast<const char *>(keys), *v = static_cast<const char *>(values);
#define KV_APPEND(DK, DV)                                                                                                                \
    if (s.st.Dk == DK && s.st.Dv == DV) {                                                                                                \
        if (s.st.dtype == KVHIP_F16) hipLaunchKernelGGL((block_append_kernel<0, DK, DV>), grid, block, 0, stream, s, k, v, pos0, n, to); \
        else hipLaunchKernelGGL((block_append_kernel<1, DK, DV>), grid, block, 0, stream, s, k, v, pos0, n, to);                         \
        return hipGetLastError();                                                                                                        \
    }
    KV_APPEND(64, 64)
    KV_APPEND(96, 96)
    KV_APPEND(128, 128)
    KV_APPEND(192, 128)
    KV_APPEND(256, 256)
#undef KV_APPEND
    return hipErrorInvalidValue;
}

hipError_t launch_block_fetch(const BlockStore &s, int64_t rows, void *dst_k, void *dst_v, hipStream_t stream) {
    if (rows <= 0 || (!dst_k && !dst_v)) return hipSuccess;
    const dim3 grid((unsigned)((rows + BLOCK_ROWS - 1) / BLOCK_ROWS), s.st.BH, dst_k && dst_v ? 2 : 1), block(256);
    char *k = static_cast<char *>(dst_k), *v = static_cast<char *>(dst_v);
    if (s.st.dtype == KVHIP_F16) hipLaunchKernelGGL((block_fetch_kernel<0>), grid, block, 0, stream, s, rows, k, v, dst_k ? 0 : 1);
    else hipLaunchKernelGGL((block_fetch_kernel<1>), grid, block, 0, stream, s, rows, k, v, dst_k ? 0 : 1);
    return hipGetLastError();
}

}  // namespace kvhip
