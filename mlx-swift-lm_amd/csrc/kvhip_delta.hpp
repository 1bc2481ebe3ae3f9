// Arguments and launchers of the recurrent layers' operators: the gated delta rule and the short convolution in front of it.
#pragma once
#include "kvhip_internal.hpp"

namespace kvhip {

#if defined(__HIPCC__)
typedef _Float16 kv_half2 __attribute__((ext_vector_type(2)));
// two float16 elements of a word (by value: a cast of a vector's element takes the vector's first)
__device__ __forceinline__ kv_half2 as_h2(uint32_t w) { return __builtin_bit_cast(kv_half2, w); }
#endif

// kvhip_gated_delta's arguments as the kernels take them (include/kvhip.h).
struct DeltaArgs {
    const char *q = nullptr, *k = nullptr, *v = nullptr, *a = nullptr, *b = nullptr;
    int64_t q_sb = 0, q_sl = 0, k_sb = 0, k_sl = 0, v_sb = 0, v_sl = 0;  // element strides of sequences and tokens
    int64_t a_sb = 0, a_sl = 0, b_sb = 0, b_sl = 0;
    const float *a_log = nullptr, *dt_bias = nullptr;
    const int32_t *left_pad = nullptr, *lengths = nullptr;
    const float *state_in = nullptr;
    float *state_out = nullptr;
    char *out = nullptr;
    int32_t B = 0, L = 0, Hk = 0, Hv = 0, Dk = 0, Dv = 0;
    int32_t dtype = 0, gate_dtype = 0;
    float scale = 1.f, eps = 0.f;
};
hipError_t launch_delta_steps(const DeltaArgs &x, hipStream_t s);
// Prompts in chunks on the matrix cores: whether a call goes that way, the scratch it takes, and the call.
bool delta_takes_chunks(const DeltaArgs &x);
size_t delta_chunk_workspace(const DeltaArgs &x);
hipError_t launch_delta_chunks(const DeltaArgs &x, void *workspace, hipStream_t s);

struct ConvArgs {
    const char *x = nullptr, *weight = nullptr, *bias = nullptr;
    int64_t x_sb = 0, x_sl = 0;
    const int32_t *left_pad = nullptr, *lengths = nullptr;
    const char *window_in = nullptr;
    char *window_out = nullptr, *out = nullptr;
    int32_t B = 0, L = 0, C = 0, W = 0, dtype = 0, silu = 0;
};
hipError_t launch_short_conv(const ConvArgs &x, hipStream_t s);

// Beam search: the `count` best continuations of each of `groups` groups of `beams` rows.
struct BeamArgs {
    const char *logits = nullptr;  // rows of `vocabulary` elements, `stride` elements apart
    int64_t stride = 0;
    const float *scores = nullptr;   // [groups * beams] or NULL
    const uint8_t *done = nullptr;   // [groups * beams] or NULL
    int32_t groups = 0, beams = 0, vocabulary = 0, dtype = 0, count = 0, pad_token = 0;
    int32_t *rows = nullptr, *tokens = nullptr;  // [groups, count]
    float *best = nullptr;
};
size_t beam_workspace(const BeamArgs &x);
hipError_t launch_beam_select(const BeamArgs &x, void *workspace, hipStream_t s);

// Rows trade places: row b of every array takes what row order[b] held (an entry outside [0, rows): row b stays).
constexpr int REORDER_ARRAYS = 8;
constexpr int REORDER_ROWS = 2048;  // the rows that one workgroup holds a piece of each of
struct ReorderArrays {
    char *at[REORDER_ARRAYS] = {};
    uint64_t bytes[REORDER_ARRAYS] = {};  // of a row
    int32_t n = 0;
};
hipError_t launch_reorder_arrays(const ReorderArrays &x, int rows, const int32_t *order, hipStream_t s);
// Tiles of TILE slots [tile0, tile1) of every plane of a page store, batch rows of `Hkv` cells each.
hipError_t launch_reorder_pages(const Store &st, int Hkv, int tile0, int tile1, const int32_t *order, hipStream_t s);

}  // namespace kvhip
