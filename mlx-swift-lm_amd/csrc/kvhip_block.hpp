// The block-scaled cache: 8-bit codes with one scale for every block of 64 tokens and kv head.
//
//   a = max |x| over the block's finite elements, e the least integer with a 2^-e <= 448 (0 if a = 0, at least -100)
//   code = e4m3(x 2^-e), to nearest even;  the value read back is code 2^e
//
// The scale is a power of two because the codes are floats: it costs them no bit (a mantissa of three bits everywhere
// between 2^-6 and 448, whatever the scale), the value read back is exact in both 16-bit types -- a float16 cache's values
// are multiples of 2^-24, and so are their roundings to four significant bits -- and a block quantized again from its values
// comes out with the same values, so that tokens may be dropped and written again.  A value that would round past the type's
// largest (float16 above 61440) takes the largest code below it.  e4m3 has no infinities: they are kept as NaN.
//
// Blocks are cut by position.  One that has all its rows is held as codes in the pages; the rows behind the last of them, the
// tail, are held as they came (infinities as NaN) until the block is whole, so that what a row is read back as does not
// depend on how many rows came with it.  Nor on rows that were there for a while: the rows of the block in front of the tail, and
// of the one that was unfinished before the last call, are kept as they came as well, each block's in a place of its own, and
// a block that loses rows again is the unfinished one as it was.  (Its codes would not do: they have the scale of all the rows
// that finished it.)
//
// A page (256 tokens, four blocks) holds for every (batch row, kv head) pair, plane by plane of its PageEntry:
//   k    four blocks of 64 Dk codes in the order in which a wavefront of the attention kernel loads its operands:
//        [16 tokens][64 channels][lane = 16 (channel / 16 % 4) + token % 16][16 channels]; where 32 channels are left over
//        at the end, [lane = 16 (channel / 8 % 4) + token % 16][8 channels]
//   v    four blocks of 64 Dv codes: [16 channels][lane = 16 (token / 4 % 4) + channel % 16][4 (token / 16) + token % 4]:
//        the sixteen tokens whose weights the lane holds as the score product leaves them
//   ksb  four pairs of floats: the blocks' key and value scales
//   vsb  four summaries of the keys: the largest, then the smallest code of each channel, rint(code / 4) as int8
// The tail: keys [64][Dk], values [8 of 8 tokens][Dv][8] (token 32 u + 16 h + 4 g + i at chunk 4 u + g, element 4 h + i).
#pragma once
#include "kvhip_device.hpp"

namespace kvhip {

constexpr int BLOCK_ROWS = 64;
constexpr int BLOCK_PER_PAGE = PAGE / BLOCK_ROWS;
constexpr int BLOCK_LEAST_EXP = -100;
constexpr int BLOCK_MAX_HEAD = 256;
// Blocks whose rows are kept as they came: the unfinished one, the one in front of it, the one that was unfinished before the last
// call.  Three places, also because a call's workgroups run at once: one reads the last of these while two others write the first two.
constexpr int BLOCK_KEPT = 3;

// Where pages lie, in a kernel's arguments: pages [first[i], first[i + 1]) are regular from the addresses of slab i on (one
// allocation each; a cache that grew has a few).  A page's entry in the page table is a load in front of everything else a short
// kernel reads: 3000 of a small step's 19 000 cycles.  n = 0: more slabs than this holds, the page table answers.
constexpr int BLOCK_SLABS = 4;
struct BlockSlabs {
    int32_t n = 0;
    int32_t first[BLOCK_SLABS] = {};
    char *k[BLOCK_SLABS] = {}, *v[BLOCK_SLABS] = {}, *ksb[BLOCK_SLABS] = {}, *vsb[BLOCK_SLABS] = {};
};

// A block-scaled cache as its kernels see it.  `coded`: blocks held as codes; rows from 64 coded on are in the tail.
struct BlockStore {
    Store st;
    char *tail_k = nullptr, *tail_v = nullptr;
    int32_t coded = 0;
    int32_t Dk_user = 0, Dv_user = 0;  // head sizes of the caller's arrays (the stored ones are padded with zeros)
    BlockSlabs slabs;
};

// Where a call leaves rows as they came: those of the last block that it finishes, and those behind it.  Either is the tail itself
// (which holds the block's rows so far) where the rows start in that block, else another place.
struct BlockKept {
    char *done_k = nullptr, *done_v = nullptr, *open_k = nullptr, *open_v = nullptr;
};
// Rows [pos0, pos0 + n) of the dense arrays [BH, n, D], written behind the pos0 rows that the cache holds.
hipError_t launch_block_append(const BlockStore &s, const void *keys, const void *values, int64_t pos0, int n, const BlockKept &to,
                               hipStream_t stream);
// Rows [0, rows) into dense arrays [BH, rows, D]; either may be NULL.
hipError_t launch_block_fetch(const BlockStore &s, int64_t rows, void *dst_k, void *dst_v, hipStream_t stream);

struct BlockAttend {
    AttendArgs a;  // (its runs are not used: rows are blocks in order)
    BlockStore b;
    // attention over listed blocks: blocks [BH, L, count] in place of the mask
    const int32_t *list = nullptr;
    int32_t count = 0;
    const int32_t *left_pad = nullptr;
    // with `keys` the lists are yet to be chosen, by every workgroup for itself (block_attend_chooses), and written to list_out
    const uint32_t *keys = nullptr;
    int32_t key_stride = 0, first = 0, recent = 1;
    int32_t *list_out = nullptr;
    // plan
    int32_t nsplit = 1;  // parts of a row's blocks
    int32_t tiles = 1;   // (listed blocks) 16-row tiles of a token's heads
    int32_t waves = 4;   // wavefronts of a workgroup
};
// Chooses the plan within a.workspace_cap; returns the bytes of scratch.
size_t plan_block_attend(BlockAttend &x);
int64_t block_attend_rows(const BlockAttend &x);  // tiles of query rows of a pair (at most 65535)
// Whether the attention of a planned call can choose its lists itself: they and the keys fit the memory of the parts.
bool block_attend_chooses(const BlockAttend &x, int key_stride);
hipError_t launch_block_attend(const BlockAttend &x, hipStream_t stream);

struct BlockSelect {
    BlockStore b;
    const void *q = nullptr;  // [B, Hq, L, Dk_user]
    int32_t B = 0, Hq = 0, Hkv = 0, L = 0;
    int32_t T = 0;
    int32_t count = 0, first = 0, recent = 1;
    const int32_t *left_pad = nullptr;
    int32_t *list = nullptr;  // [BH, L, count]
    void *workspace = nullptr;
    bool bounds_only = false;  // leave the choice to the attention (keys [BH, L, block_select_stride] in the workspace)
};
bool block_select_supported(const BlockSelect &x);
int block_select_stride(const BlockSelect &x);  // blocks a row of keys, where bounds and choice are launches of their own; else 0
size_t block_select_workspace(const BlockSelect &x);
hipError_t launch_block_select(const BlockSelect &x, hipStream_t stream);

#if defined(__HIPCC__)
// The entry of a page (of any lane's own).
__device__ __forceinline__ PageEntry block_page(const BlockStore &s, int page) {
    if (s.slabs.n == 0) return s.st.pt[page];
    PageEntry e{s.slabs.k[0], s.slabs.ksb[0], s.slabs.v[0], s.slabs.vsb[0]};
    int first = 0;
    if (s.slabs.n > 1) {
#pragma unroll
        for (int i = 1; i < BLOCK_SLABS; ++i)
            if (i < s.slabs.n && page >= s.slabs.first[i]) {
                e = PageEntry{s.slabs.k[i], s.slabs.ksb[i], s.slabs.v[i], s.slabs.vsb[i]};
                first = s.slabs.first[i];
            }
    }
    const uint64_t at = (uint64_t)(uint32_t)(page - first) * (uint32_t)s.st.BH;
    e.k += at * s.st.k_cell;
    e.ksb += at * s.st.ksb_cell;
    e.v += at * s.st.v_cell;
    e.vsb += at * s.st.vsb_cell;
    return e;
}
// byte of (row, channel) inside a block of keys / of values
__device__ __forceinline__ uint32_t block_k_at(uint32_t D, uint32_t r, uint32_t d) {
    const uint32_t c = d >> 6, m = r & 15, base = (r >> 4) * 16 * D + c * 1024;
    return D - c * 64 >= 64 ? base + (((d >> 4) & 3) * 16 + m) * 16 + (d & 15) : base + (((d >> 3) & 3) * 16 + m) * 8 + (d & 7);
}
__device__ __forceinline__ uint32_t block_v_at(uint32_t r, uint32_t d) {
    return (d >> 4) * 1024 + (((r >> 2) & 3) * 16 + (d & 15)) * 16 + (r >> 4) * 4 + (r & 3);
}
// element of (row, column) in the tail of values of one pair
__device__ __forceinline__ uint32_t tail_v_at(uint32_t Dv, uint32_t r, uint32_t d) {
    return (((r >> 5) * 4 + ((r >> 2) & 3)) * Dv + d) * 8 + ((r >> 4) & 1) * 4 + (r & 3);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

// two codes of a word (its low or high half) times 2^k (`scale`), as two elements of DT: exact, see above
template <int DT, bool HIGH> __device__ __forceinline__ uint32_t block_values(uint32_t w, float scale) {
    if constexpr (DT == 1) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HIGH));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HIGH));
}
// infinities of a pair of 16-bit elements as NaN
template <int DT> __device__ __forceinline__ uint32_t no_infinities(uint32_t w) {
    constexpr uint32_t INF = DT == 1 ? 0x7f80u : 0x7c00u;
    const uint32_t lo = (w & 0x7fffu) == INF ? 1u : 0u, hi = ((w >> 16) & 0x7fffu) == INF ? 0x10000u : 0u;
    return w | lo | hi;
}
// 16 bytes of a caller's array, which is aligned as its elements are
__device__ __forceinline__ kv_u4 load_row16(const char *p) { return *reinterpret_cast<const kv_out8 *>(p); }
#endif

}  // namespace kvhip
