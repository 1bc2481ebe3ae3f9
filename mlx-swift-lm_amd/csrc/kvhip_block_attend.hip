// Attention over the block-scaled cache: how a call is cut into workgroups, and the merge of its parts.
#include <algorithm>

#include "kvhip_block_attend.hpp"

namespace kvhip {

hipError_t launch_block_attend_f16(const BlockAttend &x, hipStream_t stream);
hipError_t launch_block_attend_bf16(const BlockAttend &x, hipStream_t stream);

namespace {

// grid (rows, BH), 256 threads: the parts [bh][part][row][D + 2] (output row not yet normalised, maximum, sum) of one query row.
// A row whose parts saw nothing is zeros; NaN stay.
constexpr int MERGE_PARTS = 256;
template <int D, int DT> __global__ void __launch_bounds__(256) block_merge_kernel(AttendArgs a, int nsplit) {
    constexpr int CP = D / 2, NG = 256 / CP;  // column pairs, groups of parts
    constexpr int UN = 8;                     // loads in flight per thread and round
    __shared__ float weight[MERGE_PARTS], red[2][4];
    __shared__ kv_f2 acc[NG][CP];
    const int i = blockIdx.x, bh = blockIdx.y, t = threadIdx.x;
    const size_t stride = (size_t)gridDim.x * (D + 2);
    const float *part = a.workspace + (size_t)bh * nsplit * stride + (size_t)i * (D + 2);
    const int g = t / CP, c = 2 * (t - g * CP);
    kv_f2 v[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
        const int s = g + NG * u;
        v[u] = g < NG && s < nsplit ? *reinterpret_cast<const kv_f2 *>(part + s * stride + c) : kv_f2{0.f, 0.f};
    }
    const kv_f2 ml = t < nsplit ? *reinterpret_cast<const kv_f2 *>(part + t * stride + D) : kv_f2{-INFINITY, 0.f};
    const float wm = wave_max(ml.x);
    if ((t & 63) == 0) red[0][t >> 6] = wm;
    __syncthreads();
    const float mx = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float w = ml.x == -INFINITY ? 0.f : fast_exp2((ml.x - mx) * LOG2E);
    if (t < nsplit) weight[t] = w;
    const float ws = wave_sum(w * ml.y);
    if ((t & 63) == 0) red[1][t >> 6] = ws;
    __syncthreads();
    const float den = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    kv_f2 sum{0.f, 0.f};
#pragma unroll
    for (int u = 0; u < UN; ++u) {
        const int s = g + NG * u;
        if (g < NG && s < nsplit) sum += v[u] * weight[s];
    }
    for (int s = g + NG * UN; g < NG && s < nsplit; s += NG) sum += *reinterpret_cast<const kv_f2 *>(part + s * stride + c) * weight[s];
    if (g < NG) acc[g][t - g * CP] = sum;
    __syncthreads();
    if (t < CP) {
        kv_f2 o = acc[0][t];
#pragma unroll
        for (int k = 1; k < NG; ++k) o += acc[k][t];
        const float inv = 1.f / den;
        const float r[2] = {den == 0.f ? 0.f : o.x * inv, den == 0.f ? 0.f : o.y * inv};
        store_columns<DT>(a.out, ((size_t)bh * gridDim.x + i) * D + 2 * t, r);
    }
}
template <int DT> hipError_t merge(const BlockAttend &x, hipStream_t stream) {
    const dim3 grid(x.a.Hq / x.a.Hkv * x.a.L, x.a.st.BH), block(256);
    if (x.a.st.Dv == 64) hipLaunchKernelGGL((block_merge_kernel<64, DT>), grid, block, 0, stream, x.a, x.nsplit);
    else if (x.a.st.Dv == 96) hipLaunchKernelGGL((block_merge_kernel<96, DT>), grid, block, 0, stream, x.a, x.nsplit);
    else if (x.a.st.Dv == 128) hipLaunchKernelGGL((block_merge_kernel<128, DT>), grid, block, 0, stream, x.a, x.nsplit);
    else hipLaunchKernelGGL((block_merge_kernel<256, DT>), grid, block, 0, stream, x.a, x.nsplit);
    return hipGetLastError();
}

}  // namespace

int64_t block_attend_rows(const BlockAttend &x) {
    const int64_t G = x.a.Hq / x.a.Hkv, cut = block_attend_tiled(x) ? block_tiled_rows(x.a.st.Dk) : 16 * block_row_tiles(x);
    return x.list ? x.a.L * ((G + 15) / 16) : (G * x.a.L + cut - 1) / cut;
}
size_t plan_block_attend(BlockAttend &x) {
    const AttendArgs &a = x.a;
    const int G = a.Hq / a.Hkv, nm = block_row_tiles(x);
    x.tiles = (G + 15) / 16;
    const int64_t base = a.st.BH * block_attend_rows(x);
    const int blocks = x.list ? x.count : (a.T + BLOCK_ROWS - 1) / BLOCK_ROWS;
    // Wavefronts that fill the chip, two to a SIMD where the registers allow it; workgroups of eight where they serve one row
    // tile and there is work for them: their parts meet in LDS, and half as many are left to merge, none at 256 pairs (four / eight
    // wavefronts, us: 32 sequences at 32 768 keys 371 + a merge of 4.8 / 351; 8 of eight heads a pair 31.8 / 26.5; 16 of four
    // tokens 76 / 65; 30 011 keys of one 19.6 / 14.2; 517 keys of 4 x 64 9.1 / 7.2; 64 listed blocks 13.1 / 10.5).
    const int64_t wanted = (a.st.Dk <= 128 ? 2048 : 1024) / std::max<int64_t>(base, 1);
    x.waves = nm == 1 && a.st.Dk <= 128 && a.mask.mode != KVHIP_MASK_ARRAY && wanted >= 8 && blocks > 4 ? 8 : 4;
    if (block_attend_tiled(x)) x.waves = 8;  // (one workgroup to a compute unit)
    int64_t parts = std::max<int64_t>(1, (block_attend_tiled(x) ? 2048 / std::max<int64_t>(base, 1) : wanted) / x.waves);
    parts = std::min<int64_t>(parts, std::max(1, blocks / 8));
    parts = std::min<int64_t>(parts, MERGE_PARTS);
    const size_t one = (size_t)a.st.BH * G * a.L * (a.st.Dv + 2) * sizeof(float);
    while (parts > 1 && a.workspace_cap && one * parts > a.workspace_cap) --parts;
    x.nsplit = (int)parts;
    return parts > 1 ? one * parts : 0;
}

bool block_attend_chooses(const BlockAttend &x, int key_stride) {
    const size_t parts = sizeof(float) * x.waves * 16 * (x.a.st.Dv + 4);  // (WaveParts)
    return key_stride > 0 && x.count <= CHOSEN_MAX && (size_t)key_stride * sizeof(uint32_t) <= parts;
}

hipError_t launch_block_attend(const BlockAttend &x, hipStream_t stream) {
    const bool f16 = x.a.st.dtype == KVHIP_F16;
    const hipError_t e = f16 ? launch_block_attend_f16(x, stream) : launch_block_attend_bf16(x, stream);
    if (e != hipSuccess || x.nsplit == 1) return e;
    return f16 ? merge<0>(x, stream) : merge<1>(x, stream);
}

}  // namespace kvhip
