// Rows into the block-scaled cache and back out of it (layout and arithmetic: kvhip_block.hpp).
#include "kvhip_block.hpp"
#include "kvhip_wave.hpp"

namespace kvhip {

namespace {

typedef uint32_t kv_w2 __attribute__((ext_vector_type(2)));

// A workgroup's threads over a block: 16 groups of four adjacent rows by 16 chunks of eight channels, in turns of 128 channels.
struct Unit {
    int rq, ch;  // row quad, chunk inside the turn
    __device__ __forceinline__ Unit() : rq(threadIdx.x >> 4), ch(threadIdx.x & 15) {}
};

// Eight channels from d0 of row `row` of a dense array of `ud` channels as words of two (zeros past the end).
template <int DT> __device__ __forceinline__ kv_u4 dense_chunk(const char *src, size_t row, int ud, int d0) {
    const char *p = src + (row * ud + d0) * 2;
    kv_u4 w{0u, 0u, 0u, 0u};
    if (d0 + 8 <= ud) {
        w = load_row16(p);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (d0 + i < ud) w[i >> 1] |= (uint32_t) reinterpret_cast<const uint16_t *>(p)[i] << (16 * (i & 1));
    }
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

template <int DT> __device__ __forceinline__ void floats_of(const kv_u4 &w, float (&x)[8]) {
    // what four significant bits can hold of the type
    constexpr float TOP = DT == 0 ? 61440.f : 3.1901471898837656e38f;  // 1.875 * 2^15, 1.875 * 2^127
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t h = (w[i >> 1] >> (16 * (i & 1))) & 0xffffu;
        const float v = DT == 1 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half((unsigned short)h));
        x[i] = v > TOP ? TOP : v < -TOP ? -TOP : v;  // (NaN stays)
    }
}

// four floats times `inv` as four codes
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
// the summary's unit of a channel's extreme (already divided by the scale): its code, a quarter of it rounded
__device__ __forceinline__ int summary_unit(float x) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(x, 0.f, 0, false);
    return (int)rintf(__builtin_amdgcn_cvt_f32_fp8(w, 0) * 0.25f);
}

// One block of one pair.  Whole after this call: its rows (those held so far and the new ones) become codes.  Else the new
// rows go to the tail, behind those of a block that was coded and has lost rows since (`reopened`).
// Two passes over the rows: the extremes of every channel, and from them the scale and the summary; then the codes, brought
// into page order in LDS and written out in whole lines.  Head sizes up to 128 keep the rows in registers in between
// (WIDE: read again, which comes from the second-level cache).
// Bound by memory: 2 bytes read and 1 written an element.
template <int DT, bool V, bool WIDE>
__device__ __forceinline__ void append_block(const BlockStore &s, const char *src, int64_t pos0, int n, int blk, int bh, bool reopened,
                                             char *to, char *image, float *ext) {
    const int D = V ? s.st.Dv : s.st.Dk, ud = V ? s.Dv_user : s.Dk_user;
    const int64_t lo = (int64_t)blk * BLOCK_ROWS;
    const bool whole = pos0 + n >= lo + BLOCK_ROWS;
    const int from = (int)(pos0 > lo ? pos0 - lo : 0);                                        // rows held so far
    const int upto = (int)(pos0 + n - lo < BLOCK_ROWS ? pos0 + n - lo : BLOCK_ROWS);          // rows after the call
    const PageEntry &e = s.st.pt[blk / BLOCK_PER_PAGE];
    const int in_page = blk % BLOCK_PER_PAGE;
    char *codes = (V ? e.v + (size_t)bh * s.st.v_cell : e.k + (size_t)bh * s.st.k_cell) + (size_t)in_page * BLOCK_ROWS * D;
    float *scales = reinterpret_cast<float *>(e.ksb + (size_t)bh * s.st.ksb_cell) + 2 * in_page;
    const size_t tail_at = (size_t)bh * BLOCK_ROWS * D * 2;
    const char *tail = (V ? s.tail_v : s.tail_k) + tail_at;
    const char *rows = src + (size_t)bh * n * ud * 2;
    const Unit u;
    const float held_scale = reopened ? scales[V ? 1 : 0] : 1.f;

    auto chunk = [&](int r, int d0) -> kv_u4 {
        if (r < from) return held_chunk<DT, V>(codes, tail, reopened, held_scale, D, r, d0);
        if (r < upto) return dense_chunk<DT>(rows, (size_t)(lo + r - pos0), ud, d0);
        return kv_u4{0u, 0u, 0u, 0u};
    };
    if (!whole) {
        const int start = reopened ? 0 : from;
        for (int d0 = 8 * u.ch; d0 < D; d0 += 128)
            for (int i = 0; i < 4; ++i) {
                const int r = 4 * u.rq + i;
                if (r < start || r >= upto) continue;
                const kv_u4 w = chunk(r, d0);
                if constexpr (V) {
                    uint16_t *t = reinterpret_cast<uint16_t *>(to + tail_at);
#pragma unroll
                    for (int k = 0; k < 8; ++k) t[tail_v_at(D, r, d0 + k)] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
                } else {
                    *reinterpret_cast<kv_u4 *>(to + tail_at + ((size_t)r * D + d0) * 2) = w;
                }
            }
        return;
    }

    kv_u4 mine[4];
    float *smx = ext, *smn = ext + 16 * 128, *chan = ext + 2 * 16 * 128;  // [16][128] twice, then [2][256] of the channels
    __shared__ float amax_s[4];
    const int t = threadIdx.x;
    float amax = 0.f;
    for (int turn = 0; turn < D; turn += 128) {
        const int d0 = turn + 8 * u.ch;
        float mx[8], mn[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) mx[k] = -INFINITY, mn[k] = INFINITY;
        if (d0 < D) {
#pragma unroll
            for (int i = 0; i < 4; ++i) mine[i] = chunk(4 * u.rq + i, d0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x[8];
                floats_of<DT>(mine[i], x);
#pragma unroll
                for (int k = 0; k < 8; ++k) mx[k] = fmaxf(mx[k], x[k]), mn[k] = fminf(mn[k], x[k]);
            }
        }
        if (turn) __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            smx[u.rq * 128 + 8 * u.ch + k] = mx[k];
            smn[u.rq * 128 + 8 * u.ch + k] = mn[k];
        }
        __syncthreads();
        const int c = t & 127;
        const float *col = (t < 128 ? smx : smn) + c;
        float x = col[0];
        for (int i = 1; i < 16; ++i) x = t < 128 ? fmaxf(x, col[i * 128]) : fminf(x, col[i * 128]);
        if (turn + c < D) {
            if (!(fabsf(x) < INFINITY)) x = 0.f;  // (a channel of nothing but NaN)
            chan[(t < 128 ? 0 : BLOCK_MAX_HEAD) + turn + c] = x;
            amax = fmaxf(amax, fabsf(x));
        }
    }
    amax = wave_max(amax);
    if ((t & 63) == 0) amax_s[t >> 6] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(amax_s[0], amax_s[1]), fmaxf(amax_s[2], amax_s[3]));
    // (all rows of a reopened block have been read by now unless they are read again below, into registers before the image
    // is written out)
    const uint32_t bits = __float_as_uint(amax);
    const int ex = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    const int exp = amax > 0.f ? max(ex, BLOCK_LEAST_EXP) : 0;
    const float inv = power_of_two(-exp);
    if (t == 0) scales[V ? 1 : 0] = power_of_two(exp);
    if constexpr (!V) {
        char *sum = e.vsb + (size_t)bh * s.st.vsb_cell + (size_t)in_page * 2 * D;
        for (int c = t; c < 2 * D; c += 256) {
            const float x = c < D ? chan[c] : chan[BLOCK_MAX_HEAD + c - D];
            sum[c] = (char)summary_unit(x * inv);
        }
    }
    for (int turn = 0; turn < D; turn += 128) {
        const int d0 = turn + 8 * u.ch;
        if (d0 < D) {
            if constexpr (WIDE) {
#pragma unroll
                for (int i = 0; i < 4; ++i) mine[i] = chunk(4 * u.rq + i, d0);
            }
            float x[4][8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                floats_of<DT>(mine[i], x[i]);
#pragma unroll
                for (int k = 0; k < 8; ++k) x[i][k] *= inv;
            }
            if constexpr (V) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    *reinterpret_cast<uint32_t *>(image + block_v_at(4 * u.rq, d0 + k)) = codes4(x[0][k], x[1][k], x[2][k], x[3][k]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<kv_w2 *>(image + block_k_at(D, 4 * u.rq + i, d0)) =
                        kv_w2{codes4(x[i][0], x[i][1], x[i][2], x[i][3]), codes4(x[i][4], x[i][5], x[i][6], x[i][7])};
            }
        }
    }
    __syncthreads();
    for (int i = t; i < BLOCK_ROWS * D / 16; i += 256) reinterpret_cast<kv_u4 *>(codes)[i] = reinterpret_cast<const kv_u4 *>(image)[i];
}

// grid (blocks touched, BH, keys / values), 256 threads
template <int DT, bool WIDE>
__global__ void __launch_bounds__(256) block_append_kernel(BlockStore s, const char *keys, const char *values, int64_t pos0, int n,
                                                                                    char *to_k, char *to_v) {
    __shared__ __align__(16) char image[BLOCK_ROWS * (WIDE ? BLOCK_MAX_HEAD : 128)];
    __shared__ float ext[2 * 16 * 128 + 2 * BLOCK_MAX_HEAD];
    const int blk = (int)(pos0 / BLOCK_ROWS) + blockIdx.x, bh = blockIdx.y;
    const bool reopened = blk < s.coded && pos0 > (int64_t)blk * BLOCK_ROWS;
    if (blockIdx.z) append_block<DT, true, WIDE>(s, values, pos0, n, blk, bh, reopened, to_v, image, ext);
    else append_block<DT, false, WIDE>(s, keys, pos0, n, blk, bh, reopened, to_k, image, ext);
}

// grid (blocks, BH, keys / values), 256 threads.  Bound by memory: 1 byte read and 2 written an element.
template <int DT, bool V>
__device__ __forceinline__ void fetch_block(const BlockStore &s, int64_t rows, char *dst, int blk, int bh, char *image) {
    const int D = V ? s.st.Dv : s.st.Dk, ud = V ? s.Dv_user : s.Dk_user;
    const int64_t lo = (int64_t)blk * BLOCK_ROWS;
    const int upto = (int)(rows - lo < BLOCK_ROWS ? rows - lo : BLOCK_ROWS);
    const bool coded = blk < s.coded;
    const PageEntry &e = s.st.pt[blk / BLOCK_PER_PAGE];
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

hipError_t launch_block_append(const BlockStore &s, const void *keys, const void *values, int64_t pos0, int n, char *to_k, char *to_v,
                               hipStream_t stream) {
    const int64_t first = pos0 / BLOCK_ROWS, last = (pos0 + n - 1) / BLOCK_ROWS;
    const dim3 grid((unsigned)(last - first + 1), s.st.BH, 2), block(256);
    const char *k = static_cast<const char *>(keys), *v = static_cast<const char *>(values);
    const bool wide = s.st.Dk > 128 || s.st.Dv > 128, f16 = s.st.dtype == KVHIP_F16;
    if (f16 && !wide) hipLaunchKernelGGL((block_append_kernel<0, false>), grid, block, 0, stream, s, k, v, pos0, n, to_k, to_v);
    else if (f16) hipLaunchKernelGGL((block_append_kernel<0, true>), grid, block, 0, stream, s, k, v, pos0, n, to_k, to_v);
    else if (!wide) hipLaunchKernelGGL((block_append_kernel<1, false>), grid, block, 0, stream, s, k, v, pos0, n, to_k, to_v);
    else hipLaunchKernelGGL((block_append_kernel<1, true>), grid, block, 0, stream, s, k, v, pos0, n, to_k, to_v);
    return hipGetLastError();
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
