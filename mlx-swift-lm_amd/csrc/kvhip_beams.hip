// Beam search: the selection over beams and vocabulary, and the rows of caches trading places by what it selects.
//
// The selection reads the logits once.  beam_rows_kernel: a workgroup holds a segment of one row in registers, takes its maximum
// M and sum exp(x - M), and the `count` best of it.  A wavefront's count-th largest lane maximum is a bound that at least `count` of its
// elements reach (found bit by bit by counting lanes, in whole numbers that are ordered as the values are, by all the bits that tell them
// apart: logits far from zero and close together are told apart as well as others); the largest of the
// wavefronts' bounds leaves a few times `count` elements of the segment, which are put down in LDS and ranked against one
// another by value, then index.  beam_merge_kernel does the same for a batch row's candidates by their scores,
//   s[beam] + ((x - M) - log sum),
// in 64 bits, so that the score's rounding does not decide between beams (the sums' does, some 1e-7: they are float32).  Where more reach the bound than the list holds (counts near 64, which
// a wavefront's 64 lanes bound loosely; thousands of equal values) the bound is raised digit by digit, by counts of all that share the digits in
// front, until no more do.  16 x 16 rows of 152 064 bfloat16 logits, us: count 8 32, 32 70, 64 246 (the best taken out one by one: 3393); 32 x 8
// rows, scores of -5, -100 and -300, 30.8, 30.2 and 29.9 (by sixteen bits of a score 31.9, 46.1 and 45.6).
//
// Vector instructions bound the rows, sixteen to an element, 74 % of the SIMDs' cycles: 256 bfloat16 rows of 152 064 logits 25 us,
// 3.1 TB/s; the merge is one workgroup to a batch row and the latency of its steps, 6.1 us.
#include <type_traits>

#include "kvhip_delta.hpp"
#include "kvhip_device.hpp"
#include "kvhip_wave.hpp"

namespace kvhip {
namespace {

typedef float kv_f4 __attribute__((ext_vector_type(4)));

constexpr int BEAM_LIST = 512;  // elements that are ranked
constexpr float NEVER = -__builtin_inff();

// whole numbers in the order of the values (no NaN)
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v + 0.f);  // (-0 as 0)
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u); }
// the largest whole number of BITS bits above zeros that at least `count` (1 to 64) of the wavefront's lanes reach
template <int BITS> __device__ __forceinline__ uint32_t reached(uint32_t key, int count) {
    uint32_t t = 0;
#pragma unroll
    for (int bit = 31; bit >= 32 - BITS; --bit) {
        const uint32_t up = t | (1u << bit);
        if (__popcll(__ballot(key >= up)) >= count) t = up;
    }
    return t;
}
// Counts the lanes that `take` by their digit; in one step where all have the same.  (8192 equal logits to each of 4864 workgroups, the whole call:
// 449 us, one by one 1017; with the logits asked for eight at a time 329.)
__device__ __forceinline__ void count_digit(uint32_t *counts, bool take, uint32_t digit, int lane) {
    const uint64_t there = __ballot(take);
    if (there == 0) return;
    const int first = __builtin_ctzll(there);
    const uint32_t of_first = __builtin_amdgcn_readlane(digit, first);
    if (__ballot(take && digit == of_first) == there) {
        if (lane == first) atomicAdd(&counts[of_first], (uint32_t)__popcll(there));
    } else if (take) {
        atomicAdd(&counts[digit], 1u);
    }
}
// Of what `counts` has by 256 digits, `need` at least: the digit of the need-th largest, how many have larger ones, and how many this one.
// (one wavefront's work)
struct Digit {
    uint32_t digit;
    int above, inside;
};
__device__ __forceinline__ void digit_of(const uint32_t *counts, int need, int lane, Digit *to) {
    int own[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += own[i] = (int)counts[255 - 4 * lane - i];
    int upto = sum;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int o = __shfl_up(upto, s);
        if (lane >= s) upto += o;
    }
    int before = upto - sum;
    if (before >= need || upto < need) return;  // (all lanes but one)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (before < need && before + own[i] >= need) *to = Digit{255u - 4 * lane - i, before, own[i]};
        before += own[i];
    }
}
// a value and its index as one whole number: the larger value first, then the lower index
__device__ __forceinline__ uint64_t rank_key(float v, int i) { return (uint64_t)ordered(v) << 32 | (uint32_t)~i; }
// a logit as it counts: what is no number never, infinity as the largest number
__device__ __forceinline__ float logit(float v) { return v != v ? NEVER : fminf(v, 3.4028234663852886e38f); }

// Scratch: for each row and segment its `count` best (value, index; -1 behind the last) and (maximum, sum).
struct BeamScratch {
    float *value;
    int32_t *index;
    float2 *sums;
    int32_t segments, segment;
};
__host__ __device__ inline int64_t beam_at(const BeamScratch &w, int64_t row, int seg) { return row * w.segments + seg; }

// NV: 16-byte vectors to a thread
template <int DT, int NV, bool WIDE>
__global__ void __launch_bounds__(256, WIDE ? 6 : 4) beam_rows_kernel(BeamArgs x, BeamScratch w) {
    constexpr int VEC = DT == 2 ? 4 : 8, ES = DT == 2 ? 4 : 2;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, seg = blockIdx.x;
    const int64_t row = blockIdx.y, at = beam_at(w, row, seg);
    const int count = x.count;
    __shared__ uint32_t wave_key[4];
    __shared__ float wave_top[4], wave_sum4s[4];
    __shared__ uint64_t list[BEAM_LIST];  // (value, index) as one whole number, the larger the better
    __shared__ int listed;
    __shared__ uint32_t digits[256];
    __shared__ Digit found;
    float *value = w.value + at * count;
    int32_t *index = w.index + at * count;
    if (x.done && x.done[row]) {  // one candidate, of the score that the beam has
        if (tid < count) {
            value[tid] = seg == 0 && tid == 0 ? 0.f : NEVER;
            index[tid] = seg == 0 && tid == 0 ? x.pad_token : -1;
        }
        if (tid == 0) w.sums[at] = make_float2(0.f, seg == 0 ? 1.f : 0.f);
        return;
    }
    const char *p = x.logits + row * x.stride * ES;
    const int base = seg * w.segment;
    // (kept as they came: what is held of a segment decides how many workgroups are there to wait for memory)
    kv_u4 raw[NV];
    if (tid == 0) listed = 0;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int i = base + (n * 256 + tid) * VEC;
        if (WIDE && i + VEC <= x.vocabulary) {
            raw[n] = *reinterpret_cast<const kv_u4 *>(p + (int64_t)i * ES);
        } else {
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                if constexpr (DT == 2) {
                    raw[n][m] = i + m < x.vocabulary ? reinterpret_cast<const uint32_t *>(p)[i + m] : 0xff800000u;
                } else {
                    constexpr uint32_t none = DT == 1 ? 0xff80u : 0xfc00u;  // (minus infinity)
                    const uint16_t *q = reinterpret_cast<const uint16_t *>(p);
                    const uint32_t lo = i + 2 * m < x.vocabulary ? q[i + 2 * m] : none, hi = i + 2 * m + 1 < x.vocabulary ? q[i + 2 * m + 1] : none;
                    raw[n][m] = lo | hi << 16;
                }
            }
        }
    }
    // a thread's element e, as it counts
    auto element = [&](auto looked_at, int n, int m) {
        float v;
        if constexpr (DT == 2) v = __uint_as_float(raw[n][m]);
        else if constexpr (DT == 1) v = __uint_as_float(m & 1 ? raw[n][m >> 1] & 0xffff0000u : raw[n][m >> 1] << 16);
        else v = m & 1 ? (float)as_h2(raw[n][m >> 1]).y : (float)as_h2(raw[n][m >> 1]).x;
        return decltype(looked_at)::value ? logit(v) : v;
    };
    // (converted anew from here on: the elements of a whole pass held as floats are twice the registers)
    auto anew = [&]() {
#pragma unroll
        for (int n = 0; n < NV; ++n) asm volatile("" : "+v"(raw[n]));
    };
    float all, sum, least, tops[NV];
    auto pass = [&](auto looked_at) {
        float top = NEVER;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            tops[n] = NEVER;
#pragma unroll
            for (int m = 0; m < VEC; ++m) tops[n] = fmaxf(tops[n], element(looked_at, n, m));
            top = fmaxf(top, tops[n]);
        }
        const uint32_t bound = reached<DT == 1 ? 16 : DT == 0 ? 19 : 32>(ordered(top), count);  // (all the bits that tell values apart)
        const float wtop = wave_max(top);
        if (lane == 0) {
            wave_key[wave] = bound;
            wave_top[wave] = wtop;
        }
        __syncthreads();
        least = unordered(max(max(max(wave_key[0], wave_key[1]), max(wave_key[2], wave_key[3])), 0x007fffffu));  // (-inf at least)
        all = fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3]));
        sum = 0.f;
        anew();
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int m = 0; m < VEC; ++m) sum += fast_exp2((element(looked_at, n, m) - all) * LOG2E);  // (the largest's is one, exactly)
        sum = wave_sum(sum);
        if (lane == 0) wave_sum4s[wave] = sum;
        __syncthreads();
        sum = wave_sum4s[0] + wave_sum4s[1] + wave_sum4s[2] + wave_sum4s[3];
    };
    auto put_down = [&](auto looked_at) {
        anew();
#pragma unroll
        for (int n = 0; n < NV; ++n)
            if (tops[n] >= least) {
#pragma unroll
                for (int m = 0; m < VEC; ++m) {
                    const float v = element(looked_at, n, m);
                    const int i = base + (n * 256 + tid) * VEC + m;
                    if (v >= least && i < x.vocabulary && (!decltype(looked_at)::value || v > NEVER || i - base < 2 * count)) {
                        const int k = atomicAdd(&listed, 1);
                        if (k < BEAM_LIST) list[k] = rank_key(v, i);
                    }
                }
            }
    };
    // Logits are taken as they are; where one is no number or infinite, which the sum or the maximum shows, or less than `count` lanes
    // of each wavefront hold one that counts, all are looked at and the pass is made again.  Of what is masked the first `count` are
    // listed then, which lie among the first 2 count where less than `count` others are: 256 bfloat16 rows of 152 064 with 100 left
    // 53 us the whole call, 311 with all of them listed and the best taken out one by one.
    pass(std::false_type{});
    const bool looked = !(sum == sum && all < __builtin_inff() && least > NEVER);
    if (!looked) {
        put_down(std::false_type{});
    } else {
        __syncthreads();
        pass(std::true_type{});
        if (all == NEVER) sum = 0.f;  // (a segment without a logit that counts)
        put_down(std::true_type{});
    }
    __syncthreads();
    int n = listed;
    if (tid == 0) w.sums[at] = make_float2(all, sum);
    if (n > BEAM_LIST) {
        // too many reach the bound: digit by digit of (value, index) the one that no more than the list holds do
        uint64_t least_key = 0;
        int above = 0, shift = 64;
        auto every = [&](auto &&take) {  // (from the caches, eight at a time: the registers have no room for keys)
            const int end = min(base + w.segment, x.vocabulary);
            for (int i0 = base + tid; i0 - tid < end; i0 += 8 * 256) {
                float v[8];
#pragma unroll
                for (int m = 0; m < 8; ++m) v[m] = Elem<DT>::load(p, min(i0 + 256 * m, end - 1));
#pragma unroll
                for (int m = 0; m < 8; ++m) take(i0 + 256 * m < end, rank_key(logit(v[m]), i0 + 256 * m));
            }
        };
        do {
            shift -= 8;
            digits[tid] = 0;
            __syncthreads();
            every([&](bool there, uint64_t key) {
                count_digit(digits, there && (shift == 56 || (key ^ least_key) >> (shift + 8) == 0), key >> shift & 255, lane);
            });
            __syncthreads();
            if (wave == 0) digit_of(digits, count - above, lane, &found);
            __syncthreads();
            least_key |= (uint64_t)found.digit << shift;
            above += found.above;
            n = above + found.inside;
        } while (n > BEAM_LIST);
        if (tid == 0) listed = 0;
        __syncthreads();
        every([&](bool there, uint64_t key) {
            if (there && key >= least_key) list[atomicAdd(&listed, 1)] = key;
        });
        __syncthreads();
    }
    for (int i = tid; i < n; i += 256) {
        const uint64_t mine = list[i];
        int rank = 0;
#pragma unroll 4
        for (int m = 0; m < n; ++m) rank += list[m] > mine;
        if (rank < count) {
            value[rank] = unordered((uint32_t)(mine >> 32));
            index[rank] = (int32_t)~(uint32_t)mine;
        }
    }
    for (int i = n + tid; i < count; i += 256) {
        value[i] = NEVER;
        index[i] = -1;
    }
}

// A candidate of the merge as whole numbers in the order of what they stand for: its score, the larger the better; then beam,
// logit and token, the smaller the better (6, 32 and 24 bits).
struct Candidate {
    uint64_t score, tie;
};
__device__ __forceinline__ bool before(const Candidate &a, const Candidate &b) { return a.score > b.score || (a.score == b.score && a.tie < b.tie); }
__device__ __forceinline__ uint64_t ordered64(double v) {
    const uint64_t u = __double_as_longlong(v + 0.);
    return u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double unordered64(uint64_t u) { return __longlong_as_double(u & 0x8000000000000000ull ? u ^ 0x8000000000000000ull : ~u); }

constexpr int MERGE_THREADS = 512, MERGE_BEAMS = 64, MERGE_HELD = 4;
// The candidate that is a thread's j-th.  Those of a segment stand best first, so that a lane would see one rank of all: each time they move
// on by nine (512 + 9 is prime, no count divides it).
__device__ __forceinline__ int merge_place(int j, int tid) { return j * MERGE_THREADS + ((tid + 9 * j) & (MERGE_THREADS - 1)); }
__global__ void __launch_bounds__(MERGE_THREADS) beam_merge_kernel(BeamArgs x, BeamScratch w) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = blockIdx.x, count = x.count;
    __shared__ double beam_score[MERGE_BEAMS], beam_log[MERGE_BEAMS];
    __shared__ float beam_top[MERGE_BEAMS];
    __shared__ uint32_t wave_key[MERGE_THREADS / 64];
    __shared__ __align__(16) Candidate list[BEAM_LIST];
    __shared__ int listed;
    __shared__ uint32_t digits[256];
    __shared__ Digit found;
    if (tid == 0) listed = 0;
    const int per = w.segments * count, total = x.beams * per;
    const int64_t first = (int64_t)g * x.beams * per;
    // a thread's first candidates, on their way while the sums are looked at
    float value[MERGE_HELD];
    int32_t token[MERGE_HELD];
#pragma unroll
    for (int j = 0; j < MERGE_HELD; ++j) {
        const int i = merge_place(j, tid);
        token[j] = i < total ? w.index[first + i] : -1;
        value[j] = i < total ? w.value[first + i] : NEVER;
    }
    for (int k = tid >> 4; k < x.beams; k += MERGE_THREADS / 16) {  // sixteen lanes to a beam
        const int64_t row = (int64_t)g * x.beams + k;
        float top = NEVER, sum = 0.f;
        for (int s = tid & 15; s < w.segments; s += 16) {
            const float2 t = w.sums[beam_at(w, row, s)];
            if (t.x == NEVER) continue;
            const float high = fmaxf(top, t.x);
            sum = sum * fast_exp2((top - high) * LOG2E) + t.y * fast_exp2((t.x - high) * LOG2E);
            top = high;
        }
#pragma unroll
        for (int m = 1; m < 16; m <<= 1) {
            const float t = __shfl_xor(top, m), y = __shfl_xor(sum, m), high = fmaxf(top, t);
            if (high == NEVER) continue;
            sum = sum * fast_exp2((top - high) * LOG2E) + y * fast_exp2((t - high) * LOG2E);
            top = high;
        }
        if ((tid & 15) == 0) {
            const float own = x.scores ? x.scores[row] : 0.f;
            // (a beam none of whose tokens counts, or whose score is no number: candidates that come last)
            beam_score[k] = own == own && top != NEVER ? (double)own : -__builtin_inf();
            beam_top[k] = top;
            beam_log[k] = log((double)sum);
        }
    }
    __syncthreads();
    auto scored = [&](int i, float v, int32_t t) {
        const int beam = i / per;
        const double own = beam_score[beam];
        // (the difference first: a logit may be so large that the others are lost in it)
        const double score = own == -__builtin_inf() || v == NEVER ? -__builtin_inf() : own + (((double)v - (double)beam_top[beam]) - beam_log[beam]);
        return Candidate{ordered64(score), (uint64_t)beam << 56 | (uint64_t)~ordered(v) << 24 | (uint32_t)t};
    };
    auto candidate = [&](int i) { return scored(i, w.value[first + i], w.index[first + i]); };
    // scores for the bound: their leading 32 bits, steps of 2^-20 of a score, rounded down, are in the same order
    uint32_t top = 0, mine[MERGE_HELD];
#pragma unroll
    for (int j = 0; j < MERGE_HELD; ++j) {
        mine[j] = token[j] >= 0 ? (uint32_t)(scored(merge_place(j, tid), value[j], token[j]).score >> 32) : 0;
        top = max(top, mine[j]);
    }
    // a thread's candidates from its j-th on
    auto every = [&](int j, auto &&take) {
        for (; j * MERGE_THREADS < total; ++j) {
            const int i = merge_place(j, tid);
            if (i < total && w.index[first + i] >= 0) take(candidate(i));
        }
    };
    every(MERGE_HELD, [&](const Candidate &c) { top = max(top, (uint32_t)(c.score >> 32)); });
    const uint32_t bound = reached<32>(top, count);
    if (lane == 0) wave_key[wave] = bound;
    __syncthreads();
    uint32_t least = 1;
#pragma unroll
    for (int i = 0; i < MERGE_THREADS / 64; ++i) least = max(least, wave_key[i]);
    auto put_down = [&](const Candidate &c) {
        const int n = atomicAdd(&listed, 1);
        if (n < BEAM_LIST) list[n] = c;
    };
    if (top >= least) {
#pragma unroll
        for (int j = 0; j < MERGE_HELD; ++j)
            if (mine[j] >= least) put_down(scored(merge_place(j, tid), value[j], token[j]));
        every(MERGE_HELD, [&](const Candidate &c) {
            if ((uint32_t)(c.score >> 32) >= least) put_down(c);
        });
    }
    __syncthreads();
    int n = listed;
    if (n > BEAM_LIST) {
        // too many reach the bound: digit by digit of (score, what is before in a tie) the one that no more than the list holds do
        uint64_t high = 0, low = 0;
        int above = 0;
        auto digit_at = [](const Candidate &c, int d) { return (uint32_t)((d < 8 ? c.score >> (56 - 8 * d) : ~c.tie >> (120 - 8 * d)) & 255); };
        for (int d = 0; n > BEAM_LIST; ++d) {
            if (tid < 256) digits[tid] = 0;
            __syncthreads();
            every(0, [&](const Candidate &c) {  // (of those whose digits in front are the ones that were found)
                const bool same = d == 0 ? true : d <= 8 ? (c.score ^ high) >> (64 - 8 * d) == 0 : c.score == high && (~c.tie ^ low) >> (128 - 8 * d) == 0;
                count_digit(digits, same, digit_at(c, d), lane);
            });
            __syncthreads();
            if (wave == 0) digit_of(digits, count - above, lane, &found);
            __syncthreads();
            if (d < 8) high |= (uint64_t)found.digit << (56 - 8 * d);
            else low |= (uint64_t)found.digit << (120 - 8 * d);
            above += found.above;
            n = above + found.inside;
        }
        if (tid == 0) listed = 0;
        __syncthreads();
        every(0, [&](const Candidate &c) {
            if (c.score > high || (c.score == high && ~c.tie >= low)) list[atomicAdd(&listed, 1)] = c;
        });
        __syncthreads();
    }
    auto put = [&](int at, const Candidate &c) {
        const int64_t o = (int64_t)g * count + at;
        x.rows[o] = g * x.beams + (int)(c.tie >> 56);
        x.tokens[o] = (int32_t)(c.tie & 0xffffffu);
        x.best[o] = (float)unordered64(c.score);
    };
    for (int i = tid; i < n; i += MERGE_THREADS) {
        const Candidate own = list[i];
        int rank = 0;
#pragma unroll 4
        for (int m = 0; m < n; ++m) rank += before(list[m], own);
        if (rank < count) put(rank, own);
    }
    for (int i = n + tid; i < count; i += MERGE_THREADS) {
        const int64_t o = (int64_t)g * count + i;
        x.rows[o] = x.tokens[o] = -1;
        x.best[o] = NEVER;
    }
}

// 16-byte vectors to a thread: the most, up to 4, that leave the chip four workgroups a compute unit.  (8: fewer wavefronts fit to
// wait for memory, 256 bfloat16 rows of 152 064: 28 us, and 24.4 with 4; 2: 26.9, and twice the candidates to merge)
inline int beam_vectors(const BeamArgs &x) {
    const int vec = x.dtype == KVHIP_F32 ? 4 : 8;
    const int64_t rows = (int64_t)x.groups * x.beams;
    int nv = 4;
    while (nv > 1 && rows * ((x.vocabulary + 256 * nv * vec - 1) / (256 * nv * vec)) < 1024) nv >>= 1;
    return nv;
}
inline BeamScratch beam_scratch(const BeamArgs &x, void *workspace, size_t *bytes) {
    const int vec = x.dtype == KVHIP_F32 ? 4 : 8;
    BeamScratch w;
    w.segment = 256 * beam_vectors(x) * vec;
    w.segments = (int32_t)(((int64_t)x.vocabulary + w.segment - 1) / w.segment);
    const size_t parts = (size_t)x.groups * x.beams * w.segments;
    char *p = static_cast<char *>(workspace);
    w.sums = reinterpret_cast<float2 *>(p);
    w.value = reinterpret_cast<float *>(p + parts * sizeof(float2));
    w.index = reinterpret_cast<int32_t *>(w.value + parts * x.count);
    if (bytes) *bytes = parts * (sizeof(float2) + x.count * 8);
    return w;
}

// ---- rows that trade places -----------------------------------------------------------------------------------------
// A workgroup holds one piece of every row that moves: all of them are read before any is written, so no row needs a second
// place, and a row that several take is read once from memory.  Rows that stay are not touched.
// Memory bounds it, and for few tokens the way there and back.  An order of 32 sequences, eight batch rows of four beams: 600 tokens x 8
// heads x 128 of float16 K and V 21.8 us, float32 states of 2 MiB 21.1 us; 8 sequences, 1311 tokens of bfloat16 15.1 us.
constexpr int REORDER_REGS = 8, REORDER_THREADS = 256;
static_assert(REORDER_REGS * REORDER_THREADS == REORDER_ROWS, "a unit of every row to a workgroup at least");

// units of U in [0, n) of each row, `stride` bytes apart; rows * n <= REORDER_ROWS
template <class U> __device__ __forceinline__ void reorder_piece(char *base, uint64_t stride, int n, int rows, const int32_t *order) {
    U held[REORDER_REGS];
    bool moves[REORDER_REGS];
#pragma unroll
    for (int r = 0; r < REORDER_REGS; ++r) {
        const int i = r * REORDER_THREADS + threadIdx.x, row = i / n;
        moves[r] = false;
        if (row >= rows) continue;
        const int32_t from = order[row];
        moves[r] = from != row && from >= 0 && from < rows;
        if (moves[r]) held[r] = *reinterpret_cast<const U *>(base + (uint64_t)from * stride + (uint64_t)(i - row * n) * sizeof(U));
    }
    // (what another wavefront stores below must not overtake a load in flight)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int r = 0; r < REORDER_REGS; ++r) {
        const int i = r * REORDER_THREADS + threadIdx.x, row = i / n;
        if (moves[r]) *reinterpret_cast<U *>(base + (uint64_t)row * stride + (uint64_t)(i - row * n) * sizeof(U)) = held[r];
    }
}
// units of every row that a piece has: whole rows of workgroups' threads where it can
__host__ __device__ inline int reorder_units(int rows) {
    int n = REORDER_ROWS / rows;
    for (int p = REORDER_ROWS; p > 1; p >>= 1)  // (a power of two: pieces then start on whole lines)
        if (p <= n) return p;
    return 1;
}

struct ReorderFlat {
    ReorderArrays x;
    uint32_t first[REORDER_ARRAYS + 1];  // pieces before each array's
};
template <class U> __global__ void __launch_bounds__(REORDER_THREADS) reorder_arrays_kernel(ReorderFlat f, int rows, const int32_t *order) {
    int a = 0;
    while (a + 1 < f.x.n && blockIdx.x >= f.first[a + 1]) ++a;
    const int n = reorder_units(rows);
    const uint64_t at = (uint64_t)(blockIdx.x - f.first[a]) * n, units = f.x.bytes[a] / sizeof(U);
    if (at >= units) return;
    reorder_piece<U>(f.x.at[a] + at * sizeof(U), f.x.bytes[a], (int)min((uint64_t)n, units - at), rows, order);
}

// planes: 0 K, 1 V, 2 K's pairs or scales, 3 V's pairs or extremes
template <class U>
__global__ void __launch_bounds__(REORDER_THREADS) reorder_pages_kernel(Store st, int Hkv, int tile0, int planes, const int32_t *order) {
    const int tile = tile0 + blockIdx.y, h = blockIdx.z % Hkv;
    int plane = 0;
    for (int skip = blockIdx.z / Hkv;; ++plane) {  // the skip-th plane of the mask
        if (!(planes >> plane & 1)) continue;
        if (skip-- == 0) break;
    }
    const PageEntry e = st.pt[tile / (PAGE / TILE)];
    const uint32_t cell = plane == 0 ? st.k_cell : plane == 1 ? st.v_cell : plane == 2 ? st.ksb_cell : st.vsb_cell;
    char *base = plane == 0 ? e.k : plane == 1 ? e.v : plane == 2 ? e.ksb : e.vsb;
    const uint32_t part = cell / (PAGE / TILE), units = part / sizeof(U);
    const int rows = st.BH / Hkv, n = reorder_units(rows);
    const uint32_t at = blockIdx.x * n;
    if (at >= units) return;
    base += (uint64_t)h * cell + (uint64_t)(tile % (PAGE / TILE)) * part + (uint64_t)at * sizeof(U);
    reorder_piece<U>(base, (uint64_t)Hkv * cell, (int)min((uint32_t)n, units - at), rows, order);
}

}  // namespace

size_t beam_workspace(const BeamArgs &x) {
    size_t bytes = 0;
    beam_scratch(x, nullptr, &bytes);
    return bytes;
}

hipError_t launch_beam_select(const BeamArgs &x, void *workspace, hipStream_t s) {
    const BeamScratch w = beam_scratch(x, workspace, nullptr);
    const int nv = beam_vectors(x), es = x.dtype == KVHIP_F32 ? 4 : 2;
    const bool wide = ((uintptr_t)x.logits | (uint64_t)(x.stride * es)) % 16 == 0;
    const dim3 grid(w.segments, x.groups * x.beams), block(256);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, x, w); };
#define KV_GO(DT, NV) (wide ? go(beam_rows_kernel<DT, NV, true>) : go(beam_rows_kernel<DT, NV, false>))
#define KV_SIZE(DT) (nv == 4 ? KV_GO(DT, 4) : nv == 2 ? KV_GO(DT, 2) : KV_GO(DT, 1))
    if (x.dtype == KVHIP_F16) KV_SIZE(0);
    else if (x.dtype == KVHIP_BF16) KV_SIZE(1);
    else KV_SIZE(2);
#undef KV_SIZE
#undef KV_GO
    hipLaunchKernelGGL(beam_merge_kernel, dim3(x.groups), dim3(MERGE_THREADS), 0, s, x, w);
    return hipGetLastError();
}

hipError_t launch_reorder_arrays(const ReorderArrays &x, int rows, const int32_t *order, hipStream_t s) {
    // one launch for the arrays of whole 16-byte units, one each for those of 4, 2 and 1 bytes
    for (int unit : {16, 4, 2, 1}) {
        ReorderFlat f{};
        uint64_t pieces = 0;
        for (int i = 0; i < x.n; ++i) {
            const uint64_t low = (uintptr_t)x.at[i] | x.bytes[i];
            const int own = low % 16 == 0 ? 16 : low % 4 == 0 ? 4 : low % 2 == 0 ? 2 : 1;
            if (own != unit || x.bytes[i] == 0) continue;
            const uint64_t units = x.bytes[i] / unit, n = reorder_units(rows);
            f.first[f.x.n] = (uint32_t)pieces;
            f.x.at[f.x.n] = x.at[i];
            f.x.bytes[f.x.n++] = x.bytes[i];
            pieces += (units + n - 1) / n;
        }
        if (f.x.n == 0) continue;
        if (pieces > 0x7fffffffu) return hipErrorInvalidValue;
        f.first[f.x.n] = (uint32_t)pieces;
        const dim3 grid((unsigned)pieces), block(REORDER_THREADS);
        if (unit == 16) hipLaunchKernelGGL((reorder_arrays_kernel<kv_u4>), grid, block, 0, s, f, rows, order);
        else if (unit == 4) hipLaunchKernelGGL((reorder_arrays_kernel<uint32_t>), grid, block, 0, s, f, rows, order);
        else if (unit == 2) hipLaunchKernelGGL((reorder_arrays_kernel<uint16_t>), grid, block, 0, s, f, rows, order);
        else hipLaunchKernelGGL((reorder_arrays_kernel<uint8_t>), grid, block, 0, s, f, rows, order);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_reorder_pages(const Store &st, int Hkv, int tile0, int tile1, const int32_t *order, hipStream_t s) {
    if (tile1 <= tile0) return hipSuccess;
    const int rows = st.BH / Hkv, n = reorder_units(rows);
    const uint32_t cells[4] = {st.k_cell, st.v_cell, st.ksb_cell, st.vsb_cell};
    for (int unit : {16, 4}) {  // (a block-scaled cache's scales are 8 bytes to a tile)
        int planes = 0, number = 0;
        uint32_t most = 0;
        for (int i = 0; i < 4; ++i) {
            const uint32_t part = cells[i] / (PAGE / TILE);
            if (part == 0 || (part % 16 == 0) != (unit == 16)) continue;
            planes |= 1 << i;
            ++number;
            most = part > most ? part : most;
        }
        if (!number) continue;
        // (65535 tiles to a launch: the grid's limit)
        for (int t = tile0; t < tile1; t += 65535) {
            const dim3 grid((most / unit + n - 1) / n, tile1 - t < 65535 ? tile1 - t : 65535, Hkv * number), block(REORDER_THREADS);
            if (unit == 16) hipLaunchKernelGGL((reorder_pages_kernel<kv_u4>), grid, block, 0, s, st, Hkv, t, planes, order);
            else hipLaunchKernelGGL((reorder_pages_kernel<uint32_t>), grid, block, 0, s, st, Hkv, t, planes, order);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

}  // namespace kvhip
