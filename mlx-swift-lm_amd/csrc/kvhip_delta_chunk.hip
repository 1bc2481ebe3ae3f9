// The gated delta rule over prompts, 64 tokens at a time on the matrix cores.
//
// With G_i the logarithms of a chunk's decays summed up to token i, K^ and Q^ the normed rows and S0 the state in front of it,
//     A_ij = beta_i e^(G_i - G_j) k^_i k^_j  (j < i),   T = (I + A)^-1 diag(beta)
//     U = T (V - diag(e^G) K^ S0^T)
//     O = diag(e^G) Q^ S0^T + P U,   P_ij = e^(G_i - G_j) q^_i k^_j  (j <= i)
//     S1^T = e^(G_63) S0^T + K^^T diag(e^(G_63 - G)) U
// T and P need no state: chunk_prep_kernel makes them for all chunks at once.  chunk_scan_kernel walks the chunks of one head, 16 NT columns
// of the values to a workgroup (columns never meet), the state in its accumulators: wavefront w holds rows of dk of S^T and does
// rows 16 w .. of every product.
//
// Numbers.  The state is returned in float32, so what it is made from keeps float32's accuracy on 16-bit operands.  Norms are
// factors of rows, put on in float32 behind the products: Q and K stay what they came as, in float16 over a power of two for
// each row (exact, but for elements below 2^-28 of the row's largest).  T, P, X, the state and what is added to it are two parts of float16,
// 22 bits together (1.4e-7 against 64 bits, as with three parts of bfloat16 for T and X), over powers of two: T's and P's for each row,
// the others' for each column.  Of a wavefront's rows of X or of the state the largest is at hand, of diag(e^(G_63 - G)) U it is
// bounded by X's units and the largest sum over a row of T.  The second parts are over 2^-11 of those units and summed up first, so that
// all 22 bits are there down to 2^-28 of the largest, below which they go one by one.  (Over the same units as the first they went from 2^-16 on:
// a chunk's values that its decays wipe out left 4e-6 of error in the others at a size of 1e6, 3e-4 at 6e7.)  Decays are summed in
// float64: e^-1000 beside e^-0.001 loses nothing.  The outputs take the same parts: of one part, 11 bits, more than one in ten
// bfloat16 outputs would be another value than the float32 arithmetic's.
//
// 8192 tokens x 32 heads x 128 x 128 in bfloat16, one sequence: 76 us of preparation (its writes and reads, 5 TB/s) and 280 of the
// scan, whose 128 chunks follow one another, 2.2 us each: the chain of products and barriers from state to state, the 82 KB of operands,
// wherever they lie (two chunks' again and again, in the L2, take as long), and the outputs, whose second parts are 25 us of the 280.  One
// wavefront to 16 columns in place of one to 16 rows took 1.3 times as long.
// 2000 tokens of 8 sequences in float16: 99 and 317 us, in two stretches of the workspace.
//
// Operands lie in the workspace as the lanes take them, 1 KB to an instruction: contractions may be summed in any
// order, so that lane (n, g)'s eight elements of a step are those at 4 g and 16 + 4 g of it -- which is where a product leaves them: S, U
// go from accumulators to operands without crossing lanes, only from wavefront to wavefront through LDS.
#include "kvhip_delta.hpp"
#include "kvhip_device.hpp"

namespace kvhip {
namespace {

typedef float kv_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 kv_b8 __attribute__((ext_vector_type(8)));
typedef _Float16 kv_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 kv_h4 __attribute__((ext_vector_type(4)));

constexpr int CHUNK = 64;

__device__ __forceinline__ kv_f4 mfma_bf16(const kv_u4 &a, const kv_u4 &b, const kv_f4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(kv_b8, a), __builtin_bit_cast(kv_b8, b), c, 0, 0, 0);
}
__device__ __forceinline__ kv_f4 mfma_f16(const kv_u4 &a, const kv_u4 &b, const kv_f4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(kv_h8, a), __builtin_bit_cast(kv_h8, b), c, 0, 0, 0);
}
__device__ __forceinline__ kv_f4 mfma_f16(const kv_u2 &a, const kv_u2 &b, const kv_f4 &c) {  // (half the terms)
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(kv_h4, a), __builtin_bit_cast(kv_h4, b), c, 0, 0, 0);
}
__device__ __forceinline__ kv_f4 mfma_f32(float a, float b, const kv_f4 &c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// two values' parts of float16: 11 bits, and the next 11 over LOW, so that these are there for all elements whose first ones are
constexpr float LOW = 1.f / 2048;
__device__ __forceinline__ kv_u2 split2(float x, float y, float f) {  // of x f and y f, f a power of two
    kv_half2 h, l;
    h.x = (_Float16)(x * f);
    h.y = (_Float16)(y * f);
    l.x = (_Float16)(fmaf(x, f, -(float)h.x) * (1 / LOW));
    l.y = (_Float16)(fmaf(y, f, -(float)h.y) * (1 / LOW));
    return kv_u2{__builtin_bit_cast(uint32_t, h), __builtin_bit_cast(uint32_t, l)};
}
// products with second parts, as the sum that those of the first parts are added to
__device__ __forceinline__ kv_f4 lowered(const kv_f4 &v) { return v * LOW; }
// The power of two over which a row's or column's elements are laid out in float16, by the largest: they end below 2^14.
__device__ __forceinline__ float unit_of(float top) {
    const uint32_t e = __float_as_uint(top) >> 23;  // (infinity and NaN: some unit; they stay what they are)
    return __uint_as_float((min(max(e, 28u), 254u) - 13) << 23);  // (2^-112 to 2^114)
}
// Products of two such operands are up to 2^28 of their units' product, and one unit may be as large as float32 goes: columns' units stand
// for SHIFT of what they are, rows' for the rest.
constexpr float SHIFT = 1.f / 16384;
__device__ __forceinline__ float over(float unit) { return __uint_as_float(0x7f000000u - __float_as_uint(unit)); }  // 1 / unit
// the largest of the four lanes that hold a column
__device__ __forceinline__ float column_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// A wavefront's number as what it is, the same in all its lanes: branches on it are a wavefront's.  (Matrix instructions heed no mask of lanes:
// under a branch that the compiler takes for one of lanes, and leaves out because the masked way is short, they work on whatever their
// registers hold.)
__device__ __forceinline__ int wave_number() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// what a wavefront's lanes hand one another through LDS: its requests are answered in their order, the compiler keeps them in it
__device__ __forceinline__ void lanes_meet() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// what wavefronts hand one another through LDS; requests past it stay in flight
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Where a call's chunks keep what the scan takes.  All offsets in bytes, per key head or value head and chunk.
struct ChunkSpace {
    char *base;
    uint64_t q, kt;             // behind k of a key head's chunk
    uint64_t key, head;         // a key head's chunk, a value head's (T, P, factors)
    uint64_t heads;             // where the value heads' begin
    int32_t chunk0, chunks;     // the chunks that are laid out
};
__device__ __forceinline__ char *key_at(const ChunkSpace &w, int64_t bh, int c) { return w.base + (bh * w.chunks + c) * w.key; }
__device__ __forceinline__ char *head_at(const ChunkSpace &w, int64_t bh, int c) { return w.base + w.heads + (bh * w.chunks + c) * w.head; }
constexpr int T_BYTES = CHUNK * CHUNK * 4, P_BYTES = CHUNK * CHUNK * 4;  // two parts
// Factors of rows, the units of their operands among them: e^G r_k (what K S is worth), scale e^G r_q, e^(G_63 - G) r_k, P's units, T's; then
// e^G_63, and the bound of |diag(e^(G_63 - G)) U| over the largest |X| of a column.
constexpr int RISE_K = 0, RISE_Q = CHUNK, FALL = 2 * CHUNK, P_UNIT = 3 * CHUNK, T_UNIT = 4 * CHUNK, LAST = 5 * CHUNK, GAIN = 5 * CHUNK + 1;
constexpr int FACTOR_BYTES = 6 * CHUNK * 4;

struct ChunkSpan {
    int from, end;  // the sequence's tokens
    __device__ __forceinline__ ChunkSpan(const DeltaArgs &x, int b) {
        from = x.left_pad ? min(max(x.left_pad[b], 0), x.L) : 0;
        end = x.lengths ? min(max(x.lengths[b], from), x.L) : x.L;
    }
    __device__ __forceinline__ bool any(int chunk) const { return chunk * CHUNK < end && (chunk + 1) * CHUNK > from; }
};

// KD: channels of a key as they are laid out (zeros behind Dk); WIDE: rows of whole 16-byte pieces
template <int DT, int KD, bool WIDE>
__global__ void __launch_bounds__(256, KD > 128 ? 2 : 4) chunk_prep_kernel(DeltaArgs x, ChunkSpace w) {
    constexpr int PITCH = KD + 8, ROW = CHUNK + 4, BYTES = CHUNK * PITCH * 2;
    constexpr double LOG2E_64 = 1.4426950408889634074;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_number(), n = lane & 15, g = lane >> 4;
    const int c = blockIdx.x, h = blockIdx.y, b = blockIdx.z, per = x.Hv / x.Hk, hk = h / per;
    const ChunkSpan span(x, b);
    const int t0 = (w.chunk0 + c) * CHUNK;
    if (!span.any(w.chunk0 + c)) return;
    constexpr int PLACE = BYTES > CHUNK * ROW * 4 ? BYTES : CHUNK * ROW * 4;
    __shared__ __align__(16) char keys[PLACE], queries[PLACE];
    __shared__ float rk[CHUNK], rq[CHUNK], beta[CHUNK], p_unit[CHUNK], key_unit[CHUNK], query_unit[CHUNK], falls[CHUNK], tops[4];
    __shared__ double total[CHUNK];  // decays summed up, as powers of two
    uint16_t *ks = reinterpret_cast<uint16_t *>(keys), *qs = reinterpret_cast<uint16_t *>(queries);
    // behind their products, in the rows' places: A in the queries' (in front of it P, a wavefront's rows at a time), T in the keys'
    float(*As)[ROW] = reinterpret_cast<float(*)[ROW]>(queries), (*Ts)[ROW] = reinterpret_cast<float(*)[ROW]>(keys);
    float decay = 0.f, rate = 0.f;
    if (wave == 0 && t0 + lane >= span.from && t0 + lane < span.end) {
        const int64_t t = t0 + lane, ai = (int64_t)b * x.a_sb + t * x.a_sl + h, bi = (int64_t)b * x.b_sb + t * x.b_sl + h;
        auto gate = [&](const char *p, int64_t i) {
            return x.gate_dtype == KVHIP_F32 ? Elem<2>::load(p, i) : x.gate_dtype == KVHIP_BF16 ? Elem<1>::load(p, i) : Elem<0>::load(p, i);
        };
        decay = gate(x.a, ai);
        rate = gate(x.b, bi);
    }
    {  // rows, and their norms: four threads to a row
        const int row = tid >> 2, t = t0 + row;
        const bool there = t >= span.from && t < span.end;
        const uint16_t *kp = reinterpret_cast<const uint16_t *>(x.k) + (int64_t)b * x.k_sb + (int64_t)t * x.k_sl + (int64_t)hk * x.Dk;
        const uint16_t *qp = reinterpret_cast<const uint16_t *>(x.q) + (int64_t)b * x.q_sb + (int64_t)t * x.q_sl + (int64_t)hk * x.Dk;
        float sk = 0.f, sq = 0.f, mk = 0.f, mq = 0.f;
        kv_u4 kw[KD / 32], qw[KD / 32];
#pragma unroll
        for (int i = 0; i < KD / 32; ++i) {
            const int d = 8 * ((tid & 3) + 4 * i);
            kw[i] = qw[i] = kv_u4{0, 0, 0, 0};
            if (WIDE) {
                if (there && d < x.Dk) {
                    kw[i] = *reinterpret_cast<const kv_u4 *>(kp + d);
                    qw[i] = *reinterpret_cast<const kv_u4 *>(qp + d);
                }
            } else if (there) {
#pragma unroll
                for (int m = 0; m < 8; ++m)
                    if (d + m < x.Dk) {
                        kw[i][m >> 1] |= (uint32_t)kp[d + m] << (16 * (m & 1));
                        qw[i][m >> 1] |= (uint32_t)qp[d + m] << (16 * (m & 1));
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < KD / 32; ++i) {
            const int d = 8 * ((tid & 3) + 4 * i);
            *reinterpret_cast<kv_u4 *>(ks + row * PITCH + d) = kw[i];
            *reinterpret_cast<kv_u4 *>(qs + row * PITCH + d) = qw[i];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                float k0, k1, q0, q1;
                if constexpr (DT == 1) {
                    k0 = __uint_as_float(kw[i][m] << 16), k1 = __uint_as_float(kw[i][m] & 0xffff0000u);
                    q0 = __uint_as_float(qw[i][m] << 16), q1 = __uint_as_float(qw[i][m] & 0xffff0000u);
                } else {
                    const kv_half2 a = as_h2(kw[i][m]), e = as_h2(qw[i][m]);
                    k0 = (float)a.x, k1 = (float)a.y, q0 = (float)e.x, q1 = (float)e.y;
                }
                sk = fmaf(k1, k1, fmaf(k0, k0, sk));
                sq = fmaf(q1, q1, fmaf(q0, q0, sq));
                mk = fmaxf(mk, fmaxf(fabsf(k0), fabsf(k1)));
                mq = fmaxf(mq, fmaxf(fabsf(q0), fabsf(q1)));
            }
        }
#pragma unroll
        for (int m = 1; m < 4; m <<= 1) {
            sk += __shfl_xor(sk, m);
            sq += __shfl_xor(sq, m);
            mk = fmaxf(mk, __shfl_xor(mk, m));
            mq = fmaxf(mq, __shfl_xor(mq, m));
        }
        if ((tid & 3) == 0) {
            rk[row] = x.eps > 0.f ? __builtin_amdgcn_rsqf(sk + x.eps) : 1.f;
            rq[row] = x.scale * (x.eps > 0.f ? __builtin_amdgcn_rsqf(sq + x.eps) : 1.f);
            key_unit[row] = unit_of(mk);
            query_unit[row] = unit_of(mq);
        }
    }
    if (wave == 0) {  // gates, and the decays summed up
        if (x.a_log && t0 + lane >= span.from && t0 + lane < span.end) {
            const float s = decay + (x.dt_bias ? x.dt_bias[h] : 0.f);
            decay = -expf(x.a_log[h]) * (fmaxf(s, 0.f) + log1pf(expf(-fabsf(s))));
            rate = 1.f / (1.f + expf(-rate));
        }
        double sum = decay < -1e5f ? -1e5f : decay;  // (e^-1e5 is nothing, and differences of sums stay numbers)
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const double o = __shfl_up(sum, s);
            if (lane >= s) sum += o;
        }
        total[lane] = sum * LOG2E_64;
        beta[lane] = rate;
    }
    __syncthreads();
    char *head = head_at(w, (int64_t)b * x.Hv + h, c), *key = key_at(w, (int64_t)b * x.Hk + hk, c);
    const bool lays_rows = h % per == 0;  // the rows as operands, once for the heads that share them
    // 16-bit elements of rows as float16, each over its row's unit
    auto scaled = [&](uint32_t v, float f0, float f1) {
        if constexpr (DT == 1) return pk_h2(__uint_as_float(v << 16) * f0, __uint_as_float(v & 0xffff0000u) * f1);
        const kv_half2 e = as_h2(v);
        return pk_h2((float)e.x * f0, (float)e.y * f1);
    };
    // rows 16 mt + n, channels 32 s + 4 g and 16 on
    auto lay_rows = [&](const uint16_t *rows, float f, char *to, int mt, int s) {
        const uint16_t *p = rows + (16 * mt + n) * PITCH + 32 * s + 4 * g;
        const kv_u2 a = *reinterpret_cast<const kv_u2 *>(p), e = *reinterpret_cast<const kv_u2 *>(p + 16);
        *reinterpret_cast<kv_u4 *>(to + ((int64_t)mt * (KD / 32) + s) * 1024 + lane * 16) = kv_u4{scaled(a.x, f, f), scaled(a.y, f, f), scaled(e.x, f, f), scaled(e.y, f, f)};
    };
    kv_f4 kk[4], qk[4];
    {  // k k^T and q k^T on and below the diagonal: wavefront w rows 16 w on
#pragma unroll
        for (int j = 0; j < 4; ++j) kk[j] = qk[j] = kv_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KD / 32; ++s) {
            const kv_u4 ka = *reinterpret_cast<const kv_u4 *>(ks + (16 * wave + n) * PITCH + 32 * s + 8 * g);
            const kv_u4 qa = *reinterpret_cast<const kv_u4 *>(qs + (16 * wave + n) * PITCH + 32 * s + 8 * g);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j > wave) break;
                const kv_u4 kb = *reinterpret_cast<const kv_u4 *>(ks + (16 * j + n) * PITCH + 32 * s + 8 * g);
                kk[j] = DT == 1 ? mfma_bf16(ka, kb, kk[j]) : mfma_f16(ka, kb, kk[j]);
                qk[j] = DT == 1 ? mfma_bf16(qa, kb, qk[j]) : mfma_f16(qa, kb, qk[j]);
            }
        }
        if (lays_rows) {
            const float fq = over(query_unit[16 * wave + n]), fk = over(key_unit[16 * wave + n]);
#pragma unroll
            for (int s = 0; s < KD / 32; ++s) {
                lay_rows(qs, fq, key + w.q, wave, s);
                lay_rows(ks, fk, key, wave, s);
            }
            const int s = wave & 1;  // channels 16 mt + n, tokens 32 s + 4 g and 16 on
            float f[8];
#pragma unroll
            for (int m = 0; m < 8; ++m) f[m] = over(key_unit[32 * s + 16 * (m >> 2) + 4 * g + (m & 3)]);
#pragma unroll 2
            for (int mt = wave >> 1; mt < KD / 16; mt += 2) {
                kv_u4 v;
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const uint16_t *p = ks + (32 * s + 16 * (m >> 1) + 4 * g + 2 * (m & 1)) * PITCH + 16 * mt + n;
                    v[m] = scaled(p[0] | (uint32_t)p[PITCH] << 16, f[2 * m], f[2 * m + 1]);
                }
                *reinterpret_cast<kv_u4 *>(key + w.kt + (mt * 2 + s) * 1024 + lane * 16) = v;
            }
        }
    }
    __syncthreads();  // (the rows have been read)
    {
        double mine[4];
        float b0[4], q0[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * wave + 4 * g + r;
            mine[r] = total[row];
            b0[r] = beta[row] * rk[row];
            q0[r] = rq[row];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = 16 * j + n;
            const double other = total[col];
            const float k0 = rk[col];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * wave + 4 * g + r;
                const float fade = j <= wave && col <= row ? __builtin_amdgcn_exp2f((float)(mine[r] - other)) * k0 : 0.f;
                kk[j][r] *= col < row ? b0[r] * fade : 0.f;
                As[row][col] = q0[r] * fade * qk[j][r];  // (P)
            }
        }
    }
    lanes_meet();
    {  // P in float16 over a unit of each row: rows 16 w + n (that this wavefront wrote), tokens 32 s + 4 g and 16 on
        float v[2][8], top = 0.f;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int m = 0; m < 8; ++m) {
                v[s][m] = As[16 * wave + n][32 * s + 16 * (m >> 2) + 4 * g + (m & 3)];
                top = fmaxf(top, fabsf(v[s][m]));
            }
        const float unit = unit_of(column_max(top)), f = over(unit);
        if (g == 0) p_unit[16 * wave + n] = unit;
        char *p = head + T_BYTES;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if (2 * s > wave) break;
            kv_u4 high, low;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const kv_u2 part = split2(v[s][2 * m], v[s][2 * m + 1], f);
                high[m] = part.x, low[m] = part.y;
            }
            *reinterpret_cast<kv_u4 *>(p + (wave * 2 + s) * 1024 + lane * 16) = high;
            *reinterpret_cast<kv_u4 *>(p + 8192 + (wave * 2 + s) * 1024 + lane * 16) = low;
        }
    }
    lanes_meet();
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) As[16 * wave + 4 * g + r][16 * j + n] = kk[j][r];
    __syncthreads();
    // (I + A)^-1 in blocks of 16: those of the diagonal by substitution, a column of a block to a lane of the first wavefront
    // ...
    if (wave == 0) {
        float t[16];
        const int o = 16 * g;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float part[4] = {i == n ? 1.f : 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < i; j += 4) {
                const kv_f4 a = *reinterpret_cast<const kv_f4 *>(&As[o + i][o + j]);
#pragma unroll
                for (int m = 0; m < 4; ++m)
                    if (j + m < i) part[m] = fmaf(-a[m], t[j + m], part[m]);
            }
            t[i] = (part[0] + part[1]) + (part[2] + part[3]);
            Ts[o + i][o + n] = t[i];
        }
    } else {
        if (wave == 1) {
            float *f = reinterpret_cast<float *>(head + T_BYTES + P_BYTES);
            const double mine = total[lane], last = total[CHUNK - 1];
            const float rise = __builtin_amdgcn_exp2f((float)mine);
            f[RISE_K + lane] = rise * rk[lane] * key_unit[lane] / SHIFT;
            f[RISE_Q + lane] = rise * rq[lane] * query_unit[lane] / SHIFT;
            f[FALL + lane] = falls[lane] = __builtin_amdgcn_exp2f((float)(last - mine)) * rk[lane] * key_unit[lane];
            f[P_UNIT + lane] = p_unit[lane];
            if (lane == 0) f[LAST] = __builtin_amdgcn_exp2f((float)last);
        }
    }
    __syncthreads();
    // ... those at distance d below it from  T_ij = -T_ii sum_k A_ik T_kj
#pragma unroll
    for (int d = 1; d < 4; ++d) {
        const int i = wave, j = wave - d;
        if (j >= 0) {
            kv_f4 y[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int m = 0; m < d; ++m) {
                const int k = j + m;
                const kv_f4 a = *reinterpret_cast<const kv_f4 *>(&As[16 * i + n][16 * k + 4 * g]);
#pragma unroll
                for (int s = 0; s < 4; ++s) y[s & 1] = mfma_f32(a[s], Ts[16 * k + 4 * g + s][16 * j + n], y[s & 1]);
            }
            const kv_f4 a = *reinterpret_cast<const kv_f4 *>(&Ts[16 * i + n][16 * i + 4 * g]);
#pragma unroll
            for (int s = 0; s < 4; ++s) z = mfma_f32(-a[s], y[0][s] + y[1][s], z);
#pragma unroll
            for (int r = 0; r < 4; ++r) Ts[16 * i + 4 * g + r][16 * j + n] = z[r];
        }
        __syncthreads();
    }
    // T in two parts over a unit of each row: rows 16 w + n, tokens 32 s + 4 g and 16 on (zero above the diagonal); and how much of X's
    // largest can come to be added to the state
    float sum = 0.f, t[2][8], top = 0.f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        if (2 * s > wave) break;
#pragma unroll
        for (int m = 0; m < 8; ++m) {
            const int col = 32 * s + 16 * (m >> 2) + 4 * g + (m & 3);
            t[s][m] = col / 16 <= wave ? Ts[16 * wave + n][col] * beta[col] : 0.f;
            sum += fabsf(t[s][m]);
            top = fmaxf(top, fabsf(t[s][m]));
        }
    }
    const float unit = unit_of(column_max(top)), f = over(unit);
    if (g == 0) reinterpret_cast<float *>(head + T_BYTES + P_BYTES)[T_UNIT + 16 * wave + n] = unit / SHIFT;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        if (2 * s > wave) break;
        kv_u4 high, low;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const kv_u2 part = split2(t[s][2 * m], t[s][2 * m + 1], f);
            high[m] = part.x, low[m] = part.y;
        }
        *reinterpret_cast<kv_u4 *>(head + (wave * 2 + s) * 1024 + lane * 16) = high;
        *reinterpret_cast<kv_u4 *>(head + 8192 + (wave * 2 + s) * 1024 + lane * 16) = low;
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    sum *= falls[16 * wave + n];
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) sum = fmaxf(sum, __shfl_xor(sum, m));
    if (lane == 0) tops[wave] = sum;
    __syncthreads();
    if (tid == 0) reinterpret_cast<float *>(head + T_BYTES + P_BYTES)[GAIN] = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
}

// NT: tiles of 16 value channels to a workgroup.  Wavefronts 0 to 3 carry the state, 4 to 7 make the outputs: what a chunk's outputs
// need is off the way from one state to the next, and fills the other's waits on the same SIMDs.
template <int DT, int KD, int NT>
__global__ void __launch_bounds__(512, 2) chunk_scan_kernel(DeltaArgs x, ChunkSpace w, const float *state_in) {
    constexpr int KS = KD / 32, TPW = KD / 64;  // TPW: a wavefront's tiles of the state
    static_assert(KD % 64 == 0, "whole tiles to a wavefront");
    const int lane = threadIdx.x & 63, number = wave_number(), wave = number & 3, n = lane & 15, g = lane >> 4;
    // (a head's workgroups on one die, where their operands meet in its cache: 8 dies take workgroups in turn)
    const int heads = x.B * x.Hv, bh = blockIdx.x % heads, col0 = blockIdx.x / heads * (16 * NT);
    const int b = bh / x.Hv, h = bh % x.Hv;
    const ChunkSpan span(x, b);
    const int64_t bk = (int64_t)b * x.Hk + h / (x.Hv / x.Hk);
    __shared__ __align__(16) char sS[2 * KS * NT * 1024];  // the state's parts, an operand a step
    __shared__ __align__(16) char sX[2 * 2 * NT * 1024];   // X's parts
    __shared__ __align__(16) char sF[2 * 2 * NT * 1024];   // parts of diag(e^(G_63 - G) r_k) U
    __shared__ __align__(16) char sU[4 * NT * 1024];       // U, in float32
    // by column and wavefront: the units of its rows of the state, and of X
    __shared__ __align__(16) float state_unit[NT][16][4], x_unit[NT][16][4];
    // the sequence's chunks among those that are laid out
    const int c0 = max(span.from / CHUNK - w.chunk0, 0), c1 = min((span.end + CHUNK - 1) / CHUNK - w.chunk0, w.chunks);
    const bool none = span.from >= span.end || c0 >= c1;
    // whether a chunk has all its tokens, and a workgroup all its columns
    auto whole = [&](int c) { return (w.chunk0 + c) * CHUNK >= span.from && (w.chunk0 + c + 1) * CHUNK <= span.end && col0 + 16 * NT <= x.Dv; };
    const int rows0 = (w.chunk0 + c0) * CHUNK + 16 * wave + 4 * g;
    const char *key = key_at(w, bk, c0) + lane * 16, *head = head_at(w, bh, c0) + lane * 16;
    const char *factors = head_at(w, bh, c0) + T_BYTES + P_BYTES, *factor = factors + (16 * wave + 4 * g) * 4;
    auto part_of = [&](char *base, int p, int steps, int s, int t) { return base + ((p * steps + s) * NT + t) * 1024 + lane * 16; };
    // What LDS holds of a step is asked for at once and in front of its products: left alone, the compiler asks for each operand where it
    // is used, and waits for LDS as often.  Requests to memory, which take their time to be issued, stand behind it, where a wavefront waits
    // anyway, and not in front of a barrier.
    auto all_requested = []() { __builtin_amdgcn_sched_barrier(0); };
    // rows [KS] times the state's columns 16 t on, in its two parts: each wavefront's rows of it apart, then put together by their units
    auto times_state = [&](const kv_u4 *rows, int t, auto &&meanwhile) {
        kv_f4 y[4], sum;
        kv_u4 part[2][KS];
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int s = 0; s < KS; ++s) part[p][s] = *reinterpret_cast<const kv_u4 *>(part_of(sS, p, KS, s, t));
        const kv_f4 units = *reinterpret_cast<const kv_f4 *>(state_unit[t][n]);
        all_requested();
        meanwhile();
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = kv_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = 1; p >= 0; --p) {
#pragma unroll
            for (int i = 0; i < 4 * TPW; i += TPW > 1 ? 2 : 1) {  // tiles of 16 rows, two to a step; of KD 64 a wavefront has half a step
                const int s = i >> 1, k = i / TPW;
                const kv_u4 &v = part[p][s];
                if constexpr (TPW > 1) y[k] = mfma_f16(rows[s], v, y[k]);
                else y[k] = mfma_f16(rows[s], i & 1 ? kv_u4{0, 0, v.z, v.w} : kv_u4{v.x, v.y, 0, 0}, y[k]);
            }
            if (p == 1) {
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] = lowered(y[k]);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[r] = fmaf(units[3], y[3][r], fmaf(units[2], y[2][r], fmaf(units[1], y[1][r], units[0] * y[0][r])));
        return sum;
    };
    // A chunk's operands are requested as soon as the last chunk's have been used, in the order in which they will be.
    if (number >= 4) {
        uint16_t *op = reinterpret_cast<uint16_t *>(x.out) + ((int64_t)b * x.L * x.Hv + h) * x.Dv + col0 + n;
        const int64_t o_sl = (int64_t)x.Hv * x.Dv;
        for (int c = 0; c < w.chunks; ++c) {  // rows of chunks without tokens
            if (!none && c >= c0 && c < c1) continue;
            const int row0 = (w.chunk0 + c) * CHUNK + 16 * wave + 4 * g;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (row0 + r < x.L && col0 + 16 * t + n < x.Dv) op[(row0 + r) * o_sl + 16 * t] = 0;
        }
        if (none) return;
        kv_u4 Q[KS], P[2][2];
        kv_f4 rise, unit;
        const int steps = wave < 2 ? 1 : 2;  // of P's rows that are not zero
        uint16_t *o = op + rows0 * o_sl;
        auto request_rows = [&](int64_t at) {
#pragma unroll
            for (int s = 0; s < KS; ++s) Q[s] = *reinterpret_cast<const kv_u4 *>(key + at * w.key + w.q + (wave * KS + s) * 1024);
        };
        auto request_rest = [&](int64_t at) {
            rise = *reinterpret_cast<const kv_f4 *>(factor + at * w.head + RISE_Q * 4);
            unit = *reinterpret_cast<const kv_f4 *>(factor + at * w.head + P_UNIT * 4);
#pragma unroll
            for (int s = 0; s < 2; ++s)
                if (s < steps)
#pragma unroll
                    for (int p = 0; p < 2; ++p) P[p][s] = *reinterpret_cast<const kv_u4 *>(head + at * w.head + T_BYTES + p * 8192 + (wave * 2 + s) * 1024);
        };
        request_rows(0);
        request_rest(0);
        for (int c = c0; c < c1; ++c) {
            const int next = min(c + 1, c1 - 1) - c0;
            kv_f4 O[NT], I[NT];
            lds_barrier();
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                O[t] = times_state(Q, t, []() {});
                I[t] = kv_f4{0.f, 0.f, 0.f, 0.f};
            }
            request_rows(next);
            lds_barrier();
            lds_barrier();
            float u_unit[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                kv_f4 u[4];
                float top = 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (k >= 2 * steps) break;
                    u[k] = *reinterpret_cast<const kv_f4 *>(sU + (k * NT + t) * 1024 + lane * 16);
                }
                all_requested();
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (k >= 2 * steps) break;
                    top = fmaxf(top, fmaxf(fmaxf(fabsf(u[k][0]), fabsf(u[k][1])), fmaxf(fabsf(u[k][2]), fabsf(u[k][3]))));
                }
                u_unit[t] = unit_of(column_max(top));
                const float f = over(u_unit[t]);
                kv_u4 high[2], low[2];
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    if (s >= steps) break;
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        const kv_u2 part = split2(u[2 * s + (m >> 1)][2 * (m & 1)], u[2 * s + (m >> 1)][2 * (m & 1) + 1], f);
                        high[s][m] = part.x, low[s][m] = part.y;
                    }
                    I[t] = mfma_f16(P[1][s], high[s], I[t]);
                    I[t] = mfma_f16(P[0][s], low[s], I[t]);
                }
                I[t] = lowered(I[t]);
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    if (s < steps) I[t] = mfma_f16(P[0][s], high[s], I[t]);
            }
            const bool all = whole(c);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float y[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) y[r] = fmaf(rise[r], O[t][r], unit[r] * I[t][r] * u_unit[t]);
                if (all) {
                    const uint32_t a = DT == 1 ? pk_bf2(y[0], y[1]) : pk_h2(y[0], y[1]), e = DT == 1 ? pk_bf2(y[2], y[3]) : pk_h2(y[2], y[3]);
                    o[16 * t] = (uint16_t)a;
                    o[o_sl + 16 * t] = (uint16_t)(a >> 16);
                    o[2 * o_sl + 16 * t] = (uint16_t)e;
                    o[3 * o_sl + 16 * t] = (uint16_t)(e >> 16);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int row = rows0 + (c - c0) * CHUNK + r;
                        if (row < x.L && col0 + 16 * t + n < x.Dv)
                            Elem<DT>::store(o, r * o_sl + 16 * t, row >= span.from && row < span.end ? y[r] : 0.f);
                    }
                }
            }
            o += CHUNK * o_sl;
            request_rest(next);
        }
        return;
    }
    kv_f4 S[TPW][NT];
    const bool wide = x.Dk % 4 == 0 && ((uintptr_t)state_in | (uintptr_t)x.state_out) % 16 == 0;
#pragma unroll
    for (int i = 0; i < TPW; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int d = 16 * (wave * TPW + i) + 4 * g, col = col0 + 16 * t + n;
            S[i][t] = kv_f4{0.f, 0.f, 0.f, 0.f};
            if (!state_in || col >= x.Dv) continue;
            const float *p = state_in + ((int64_t)bh * x.Dv + col) * x.Dk + d;
            if (wide) {
                if (d < x.Dk) S[i][t] = *reinterpret_cast<const kv_f4 *>(p);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (d + r < x.Dk) S[i][t][r] = p[r];
            }
        }
    if (!none) {
        const uint16_t *vp = reinterpret_cast<const uint16_t *>(x.v) + (int64_t)b * x.v_sb + (int64_t)h * x.Dv + col0, *v = vp + (int64_t)rows0 * x.v_sl + n;
        const int steps = wave < 2 ? 1 : 2;  // of T's rows that are not zero
        kv_u4 K[KS], KT[TPW][2], T[2][2];
        kv_f4 rise, fall, row_unit;
        float last, gain;
        uint16_t V[NT][4];
        auto request_rows = [&](int64_t at) {
#pragma unroll
            for (int s = 0; s < KS; ++s) K[s] = *reinterpret_cast<const kv_u4 *>(key + at * w.key + (wave * KS + s) * 1024);
        };
        auto request_values = [&](int64_t at, bool all) {
            rise = *reinterpret_cast<const kv_f4 *>(factor + at * w.head + RISE_K * 4);
            if (all) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int t = 0; t < NT; ++t) V[t][r] = v[(at * CHUNK + r) * x.v_sl + 16 * t];
            } else {  // (a token that is there in place of one that is not)
                const int row0 = rows0 + (int)at * CHUNK;
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int t = 0; t < NT; ++t) V[t][r] = vp[(int64_t)min(max(row0 + r, span.from), span.end - 1) * x.v_sl + min(16 * t + n, x.Dv - 1 - col0)];
            }
        };
        auto request_system = [&](int64_t at) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
                if (s < steps)
#pragma unroll
                    for (int p = 0; p < 2; ++p) T[p][s] = *reinterpret_cast<const kv_u4 *>(head + at * w.head + p * 8192 + (wave * 2 + s) * 1024);
            row_unit = *reinterpret_cast<const kv_f4 *>(factor + at * w.head + T_UNIT * 4);
            fall = *reinterpret_cast<const kv_f4 *>(factor + at * w.head + FALL * 4);
            gain = *reinterpret_cast<const float *>(factors + at * w.head + GAIN * 4);
        };
        auto request_rest = [&](int64_t at) {
            last = *reinterpret_cast<const float *>(factors + at * w.head + LAST * 4);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < TPW; ++i) KT[i][s] = *reinterpret_cast<const kv_u4 *>(key + at * w.key + w.kt + ((wave * TPW + i) * 2 + s) * 1024);
        };
        // four neighbouring elements of a column, over a unit, as float16's parts of half an operand
        auto share = [&](char *base, int steps_, int tile, int t, const kv_f4 &v, float f) {
            const kv_u2 a = split2(v[0], v[1], f), e = split2(v[2], v[3], f);
            *reinterpret_cast<kv_u2 *>(part_of(base, 0, steps_, tile >> 1, t) + (tile & 1) * 8) = kv_u2{a.x, e.x};
            *reinterpret_cast<kv_u2 *>(part_of(base, 1, steps_, tile >> 1, t) + (tile & 1) * 8) = kv_u2{a.y, e.y};
        };
        auto largest = [](const kv_f4 &v) { return fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))); };
        auto share_state = [&]() {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float top = largest(S[0][t]);
#pragma unroll
                for (int i = 1; i < TPW; ++i) top = fmaxf(top, largest(S[i][t]));
                const float unit = unit_of(column_max(top)), f = over(unit);
                if (g == 0) state_unit[t][n][wave] = unit * SHIFT;
#pragma unroll
                for (int i = 0; i < TPW; ++i) share(sS, KS, wave * TPW + i, t, S[i][t], f);
            }
        };
        bool all = whole(c0);
        request_rows(0);
        request_values(0, all);
        request_system(0);
        request_rest(0);
        share_state();
        for (int c = c0; c < c1; ++c) {
            const int now = c - c0, next = min(c + 1, c1 - 1) - c0;
            const bool all_next = whole(next + c0);
            kv_f4 U[NT];
            lds_barrier();
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const kv_f4 R = times_state(K, t, [&]() {
                    if (t == 0 && c > c0) request_rest(now);
                });
                kv_f4 X;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float value = Elem<DT>::load(&V[t][r], 0);
                    if (!all) {
                        const int row = rows0 + (c - c0) * CHUNK + r;
                        value = row >= span.from && row < span.end ? value : 0.f;
                    }
                    X[r] = fmaf(-rise[r], R[r], value);
                }
                const float unit = unit_of(column_max(largest(X)));
                if (g == 0) x_unit[t][n][wave] = unit * SHIFT;
                share(sX, 2, wave, t, X, over(unit));
            }
            lds_barrier();
            float f_unit[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                kv_u4 part[2][2];
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    if (s < steps)
#pragma unroll
                        for (int p = 0; p < 2; ++p) part[p][s] = *reinterpret_cast<const kv_u4 *>(part_of(sX, p, 2, s, t));
                const kv_f4 units = *reinterpret_cast<const kv_f4 *>(x_unit[t][n]);
                all_requested();
                if (t == 0) {
                    request_rows(next);
                    request_values(next, all_next);
                }
                f_unit[t] = unit_of(gain * fmaxf(fmaxf(units[0], units[1]), fmaxf(units[2], units[3])) * (16384.f / SHIFT));
                U[t] = kv_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < 2; ++s) {  // each wavefront's rows of X apart, half a step, then put together by their units
                    if (s >= steps) break;
                    auto half = [](const kv_u4 &v, int k) { return k ? kv_u2{v.z, v.w} : kv_u2{v.x, v.y}; };
                    kv_f4 y[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        y[k] = mfma_f16(half(T[0][s], k), half(part[1][s], k), kv_f4{0.f, 0.f, 0.f, 0.f});
                        y[k] = mfma_f16(half(T[1][s], k), half(part[0][s], k), y[k]);
                        y[k] = mfma_f16(half(T[0][s], k), half(part[0][s], k), lowered(y[k]));
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) U[t][r] = fmaf(units[2 * s + 1], y[1][r], fmaf(units[2 * s], y[0][r], U[t][r]));
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                kv_f4 u;
#pragma unroll
                for (int r = 0; r < 4; ++r) u[r] = row_unit[r] * U[t][r];
                *reinterpret_cast<kv_f4 *>(sU + (wave * NT + t) * 1024 + lane * 16) = u;
#pragma unroll
                for (int r = 0; r < 4; ++r) u[r] *= fall[r];
                share(sF, 2, wave, t, u, over(f_unit[t]));
            }
            lds_barrier();
            kv_f4 D[TPW][NT];
#pragma unroll
            for (int i = 0; i < TPW; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) D[i][t] = kv_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                kv_u4 part[2][2];
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int p = 0; p < 2; ++p) part[p][s] = *reinterpret_cast<const kv_u4 *>(part_of(sF, p, 2, s, t));
                all_requested();
                if (t == 0) request_system(next);
#pragma unroll
                for (int p = 1; p >= 0; --p) {
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int i = 0; i < TPW; ++i) D[i][t] = mfma_f16(KT[i][s], part[p][s], D[i][t]);
                    if (p == 1) {
#pragma unroll
                        for (int i = 0; i < TPW; ++i) D[i][t] = lowered(D[i][t]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < TPW; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[i][t][r] = fmaf(f_unit[t], D[i][t][r], last * S[i][t][r]);
            share_state();  // (its last readers are behind a barrier)
            all = all_next;
        }
    }
#pragma unroll
    for (int i = 0; i < TPW; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int d = 16 * (wave * TPW + i) + 4 * g, col = col0 + 16 * t + n;
            if (col >= x.Dv) continue;
            float *p = x.state_out + ((int64_t)bh * x.Dv + col) * x.Dk + d;
            if (wide) {
                if (d < x.Dk) *reinterpret_cast<kv_f4 *>(p) = S[i][t];
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (d + r < x.Dk) p[r] = S[i][t][r];
            }
        }
}

inline int chunk_key_dim(const DeltaArgs &x) { return x.Dk <= 64 ? 64 : x.Dk <= 128 ? 128 : 256; }
// What a chunk of all sequences and heads takes, and how many chunks are laid out at a time: what they take is to stay near the
// last-level cache between the two kernels, and a round is to be long enough to pay for its start.  96 / 192 / 384 / 768 MiB, 32 heads of
// 128 x 128 in bfloat16, us: 8 x 2000 tokens 622 / 550 / 525 / 499; 16 x 4096 2490 / 2316 / 2106 / 2038; 32768 of one 1306 / 1256 /
// 1301 / 1276.  More than 384 gains little for twice the memory.  Four chunks at least, whatever they take, because every round reads and
// writes the states: 256 x 333 with 1 / 2 / 4 at least 5325 / 4091 / 3750.
constexpr uint64_t CHUNK_SPACE = (uint64_t)384 << 20;
inline ChunkSpace chunk_space(const DeltaArgs &x, void *workspace, uint64_t *bytes) {
    ChunkSpace w{};
    const uint64_t rows = (uint64_t)CHUNK * chunk_key_dim(x) * 2;
    w.base = static_cast<char *>(workspace);
    w.q = rows;
    w.kt = 2 * rows;
    w.key = 3 * rows;
    w.head = T_BYTES + P_BYTES + FACTOR_BYTES;
    const uint64_t one = (uint64_t)x.B * (x.Hk * w.key + x.Hv * w.head);
    const int all = (x.L + CHUNK - 1) / CHUNK;
    const uint64_t fit = CHUNK_SPACE / one;
    w.chunks = (int32_t)(fit < 4 ? 4 : fit);
    if (w.chunks > all) w.chunks = all;
    w.heads = (uint64_t)x.B * x.Hk * w.chunks * w.key;
    *bytes = one * w.chunks;
    return w;
}

template <int DT, int KD> hipError_t launch_chunks(const DeltaArgs &x, ChunkSpace w, hipStream_t s) {
    auto even = [&](const char *p, int64_t sb, int64_t sl) { return ((uintptr_t)p | (uint64_t)(sb * 2) | (uint64_t)(sl * 2)) % 16 == 0; };
    const bool wide = x.Dk % 8 == 0 && even(x.q, x.q_sb, x.q_sl) && even(x.k, x.k_sb, x.k_sl);
    const int all = (x.L + CHUNK - 1) / CHUNK, most = w.chunks;
    const float *state = x.state_in;
    for (int c = 0; c < all; c += most) {
        w.chunk0 = c;
        w.chunks = all - c < most ? all - c : most;
        const dim3 prep(w.chunks, x.Hv, x.B);
        if (wide) hipLaunchKernelGGL((chunk_prep_kernel<DT, KD, true>), prep, dim3(256), 0, s, x, w);
        else hipLaunchKernelGGL((chunk_prep_kernel<DT, KD, false>), prep, dim3(256), 0, s, x, w);
        auto scan = [&](auto kernel, int columns) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)((int64_t)x.B * x.Hv * ((x.Dv + columns - 1) / columns))), dim3(512), 0, s, x, w, state);
        };
        const int64_t groups = (int64_t)x.B * x.Hv * ((x.Dv + 15) / 16);
        // Every workgroup of a head reads the head's whole operands: few columns to each fill the chip, many read less.  Whole calls in
        // us with 16 / 32 / 64 columns, 32 heads of 128 x 128 in bfloat16: 8192 tokens (256 groups) 318 / 468 / 778; 2 x 2048 (512)
        // 154 / 136 / 214; 4 x 2048 (1024) 336 / 275 / 255; 8 x 2000 in float16 (2048) 1071 / 635 / 524 (but 6 x 2048, 1536, 650 / 420 / 461).
        // 256 channels have no registers for 64; 4 heads of 512 x 256: 4096 tokens (128) 166 / 264; 4 x 2048 (512) 176 / 151.
        if (groups <= 256) {
            scan(chunk_scan_kernel<DT, KD, 1>, 16);
        } else if (KD > 128 || groups <= 512) {
            scan(chunk_scan_kernel<DT, KD, 2>, 32);
        } else if constexpr (KD <= 128) {
            scan(chunk_scan_kernel<DT, KD, 4>, 64);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        state = x.state_out;
    }
    return hipSuccess;
}

}  // namespace

// From how many tokens on: a chunk costs much the same whatever it holds, each of few heads a launch's time more; a token costs the other
// kernel a chain of sums, and what the states take to pass through the vector units.  us by chunks / by tokens, heads of 128 x 128: 32, 10
// tokens 15.5 / 14.9, 12: 15.5 / 16.9; 128, 14: 23.2 / 21.0, 16: 23.2 / 23.4; 256, 20: 36.5 / 34.5, 24: 36.5 / 40.3; 2048, 16: 211 / 190,
// 20: 216 / 227.  256 of 64 x 64, 20: 20.3 / 18.5, 24: 20.3 / 21.1.  Of 512 x 256, whose tokens have twice the registers: 8, 8: 19.0 / 20.6;
// 32, 10: 31.5 / 28.7, 12: 31.6 / 32.4; 128, 16: 89.9 / 102.8.
bool delta_takes_chunks(const DeltaArgs &x) {
    const int64_t heads = (int64_t)x.B * x.Hv;
    const int tokens = x.Dk <= 128 ? (heads <= 32 ? 10 : heads <= 128 ? 14 : 20) : (heads <= 16 ? 7 : heads <= 32 ? 11 : 14);
    return x.dtype != KVHIP_F32 && x.L > tokens && heads * x.Dv < ((int64_t)1 << 31);
}

size_t delta_chunk_workspace(const DeltaArgs &x) {
    uint64_t bytes = 0;
    (void)chunk_space(x, nullptr, &bytes);
    return bytes;
}

hipError_t launch_delta_chunks(const DeltaArgs &x, void *workspace, hipStream_t s) {
    uint64_t bytes = 0;
    const ChunkSpace w = chunk_space(x, workspace, &bytes);
    const int kd = chunk_key_dim(x);
    if (x.dtype == KVHIP_F16) return kd == 64 ? launch_chunks<0, 64>(x, w, s) : kd == 128 ? launch_chunks<0, 128>(x, w, s) : launch_chunks<0, 256>(x, w, s);
    return kd == 64 ? launch_chunks<1, 64>(x, w, s) : kd == 128 ? launch_chunks<1, 128>(x, w, s) : launch_chunks<1, 256>(x, w, s);
}

}  // namespace kvhip
