// The gated delta rule token by token, and the short convolution in front of it.
//
//   g = exp(-exp(a_log) softplus(a + dt_bias)),  beta = sigmoid(b)
//   S <- g S;  u = beta (v - S k^);  S <- S + u k^T;  o = S q^
//
// delta_steps_kernel keeps S in registers over all tokens of a call: eight lanes hold a row of S (one channel of the values),
// four neighbouring elements in every 32 each, so that a wavefront's load is eight whole cache lines.  Rows never meet: a
// wavefront needs no other, nothing goes through LDS, and a head's rows are spread over as many wavefronts as fill the chip.
// With o written as  g (S q^) + u (k^ q^),  both products of a token read the same S and their sums over the eight lanes (three
// permutes each) run side by side.  Every lane makes the token's norms for itself.
//
// Memory bounds it: a state is read and written once, past the caches, which it would only sweep.  One token of 64 sequences x 32
// heads x 128 x 128: 55.6 us, 4.8 TB/s (14 us more through the caches).
#include "kvhip_delta.hpp"
#include "kvhip_device.hpp"
#include "kvhip_wave.hpp"

namespace kvhip {
namespace {

typedef float kv_f4 __attribute__((ext_vector_type(4)));

// sums over groups of eight adjacent lanes, in every lane
__device__ __forceinline__ float sum8(float v) {
#define KV_SUM_STEP(CTRL) v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true))
    KV_SUM_STEP(0xB1);   // quad_perm [1,0,3,2]
    KV_SUM_STEP(0x4E);   // quad_perm [2,3,0,1]
    KV_SUM_STEP(0x141);  // row_half_mirror
#undef KV_SUM_STEP
    return v;
}

// four elements from `p` on, of which `n` (0 to 4, more: all) are there; WIDE: all four or none, aligned to their size
template <int DT, bool WIDE> __device__ __forceinline__ kv_f4 load4(const char *p, int n) {
    kv_f4 r = {0.f, 0.f, 0.f, 0.f};
    if constexpr (WIDE) {
        if (n <= 0) return r;
        if constexpr (DT == 2) return *reinterpret_cast<const kv_f4 *>(p);
        const kv_u2 w = *reinterpret_cast<const kv_u2 *>(p);
        if constexpr (DT == 1) {
            r = kv_f4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u)};
        } else {
            const kv_h2 lo = as_h2(w.x), hi = as_h2(w.y);
            r = kv_f4{(float)lo.x, (float)lo.y, (float)hi.x, (float)hi.y};
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) r[i] = Elem<DT>::load(p, i);
    }
    return r;
}
__device__ __forceinline__ float load_gate(int dtype, const char *p, int64_t i) {
    return dtype == KVHIP_F32 ? Elem<2>::load(p, i) : dtype == KVHIP_BF16 ? Elem<1>::load(p, i) : Elem<0>::load(p, i);
}

// NC: 32-element chunks of a row of S;  R: rows of S that a lane has elements of
template <int DT, int NC, int R, bool WIDE>
__global__ void __launch_bounds__(256) delta_steps_kernel(DeltaArgs x) {
    const int lane = threadIdx.x & 63, j = lane & 7, h = blockIdx.y, b = blockIdx.z;
    const int row0 = ((blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6)) * R * 8) + (lane >> 3);
    constexpr int ES = DT == 2 ? 4 : 2;
    const int Dk = x.Dk, Dv = x.Dv, hk = h / (x.Hv / x.Hk);
    const int from = x.left_pad ? min(max(x.left_pad[b], 0), x.L) : 0;
    const int end = x.lengths ? min(max(x.lengths[b], from), x.L) : x.L;
    // Gates of 64 tokens at a time, a token to a lane; of the first ones, in front of the state.  (Every lane making every token's: 2048
    // float32 tokens of 32 heads x 128 x 128 2115 us, and 1429 so; 64 single ones 54.2, and 55.6.)
    float ga = 0.f, gb = 0.f;
    auto request_gates = [&](int l) {
        if (l + lane >= end) return;
        ga = load_gate(x.gate_dtype, x.a, (int64_t)b * x.a_sb + (int64_t)(l + lane) * x.a_sl + h);
        gb = load_gate(x.gate_dtype, x.b, (int64_t)b * x.b_sb + (int64_t)(l + lane) * x.b_sl + h);
    };
    request_gates(from);
    kv_f4 s[R][NC];
    const int64_t cell = ((int64_t)b * x.Hv + h) * Dv;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = row0 + 8 * r;
        const char *p = reinterpret_cast<const char *>(x.state_in + (cell + row) * Dk);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = 32 * c + 4 * j;
            s[r][c] = kv_f4{0.f, 0.f, 0.f, 0.f};
            if (!x.state_in || row >= Dv) continue;
            if constexpr (!WIDE) s[r][c] = load4<2, false>(p + 4 * d, Dk - d);
            else if (d < Dk) s[r][c] = __builtin_nontemporal_load(reinterpret_cast<const kv_f4 *>(p + 4 * d));
        }
    }
    const float rate = x.a_log ? LOG2E * expf(x.a_log[h]) : 0.f, dt = x.a_log && x.dt_bias ? x.dt_bias[h] : 0.f;
    const char *qp = x.q + ((int64_t)b * x.q_sb + (int64_t)hk * Dk) * ES, *kp = x.k + ((int64_t)b * x.k_sb + (int64_t)hk * Dk) * ES;
    const char *vp = x.v + ((int64_t)b * x.v_sb + (int64_t)h * Dv) * ES;
    char *op = x.out + ((int64_t)b * x.L * x.Hv + h) * Dv * ES;
    const int64_t o_sl = (int64_t)x.Hv * Dv;
    // a token's operands, requested a token ahead
    kv_f4 q[NC], k[NC];
    float v[R];
    auto request = [&](int l) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = 32 * c + 4 * j;
            q[c] = load4<DT, WIDE>(qp + ((int64_t)l * x.q_sl + d) * ES, Dk - d);
            k[c] = load4<DT, WIDE>(kp + ((int64_t)l * x.k_sl + d) * ES, Dk - d);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) v[r] = row0 + 8 * r < Dv ? Elem<DT>::load(vp, (int64_t)l * x.v_sl + row0 + 8 * r) : 0.f;
    };
    float decay = 1.f, beta_of = 0.f;
    auto turn_gates = [&]() {
        if (x.a_log) {
            const float t = ga + dt;
            decay = fast_exp2(-rate * (fmaxf(t, 0.f) + log1pf(fast_exp2(-LOG2E * fabsf(t)))));
            beta_of = __builtin_amdgcn_rcpf(1.f + fast_exp2(-LOG2E * gb));
        } else {
            decay = fast_exp2(LOG2E * ga);
            beta_of = gb;
        }
    };
    auto of_lane = [](float v, int i) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), i)); };
    if (from < end) request(from);
    auto store = [&](int l, int r, float o) {
        if (j == 0 && row0 + 8 * r < Dv) Elem<DT>::store(op, (int64_t)l * o_sl + row0 + 8 * r, o);
    };
    for (int l = 0; l < from; ++l)
#pragma unroll
        for (int r = 0; r < R; ++r) store(l, r, 0.f);
    for (int l = from; l < end; ++l) {
        float qq = 0.f, kk = 0.f, qk = 0.f, sq[R], sk[R];
#pragma unroll
        for (int r = 0; r < R; ++r) sq[r] = sk[r] = 0.f;
        kv_f4 kn[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            kn[c] = k[c];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                qq = fmaf(q[c][i], q[c][i], qq);
                kk = fmaf(k[c][i], k[c][i], kk);
                qk = fmaf(q[c][i], k[c][i], qk);
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sk[r] = fmaf(s[r][c][i], k[c][i], sk[r]);
                    sq[r] = fmaf(s[r][c][i], q[c][i], sq[r]);
                }
        }
        float vn[R];
#pragma unroll
        for (int r = 0; r < R; ++r) vn[r] = v[r];
        const int at = (l - from) & 63;
        if (at == 0) {
            turn_gates();
            request_gates(l + 64);
        }
        const float g = of_lane(decay, at), beta = of_lane(beta_of, at);
        if (l + 1 < end) request(l + 1);
        qq = sum8(qq);
        kk = sum8(kk);
        qk = sum8(qk);
        const float kf = x.eps > 0.f ? __builtin_amdgcn_rsqf(kk + x.eps) : 1.f, qf = x.scale * (x.eps > 0.f ? __builtin_amdgcn_rsqf(qq + x.eps) : 1.f);
        const float qkf = qk * kf * qf;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float u = beta * (vn[r] - g * (sum8(sk[r]) * kf));
            store(l, r, fmaf(u, qkf, g * (sum8(sq[r]) * qf)));
            const float uk = u * kf;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[r][c][i] = fmaf(uk, kn[c][i], g * s[r][c][i]);
        }
    }
    for (int l = end; l < x.L; ++l)
#pragma unroll
        for (int r = 0; r < R; ++r) store(l, r, 0.f);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = row0 + 8 * r;
        if (row >= Dv) continue;
        float *p = x.state_out + (cell + row) * Dk;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = 32 * c + 4 * j;
            if constexpr (WIDE) {
                if (d < Dk) __builtin_nontemporal_store(s[r][c], reinterpret_cast<kv_f4 *>(p + d));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (d + i < Dk) p[d + i] = s[r][c][i];
            }
        }
    }
}

// ---- the short convolution --------------------------------------------------------------------------------------------
// y_t = f(bias + sum_w weight[:, w] e_{t + w}) with e the window's W - 1 rows and then the sequence's tokens.  A thread takes V
// neighbouring channels (16 bytes) of CONV_TOKENS tokens: a token is read once, the taps slide through registers.  Tiles of
// tokens start at the sequence's first one (left_pad), so that the first tile alone reads the window -- and can write the new
// one over it.  Memory bounds it: 8192 bfloat16 tokens x 8192 channels 51 us, 5.3 TB/s (4 tokens requested at a time; 8, with their
// registers, 75 to 99).  Single tokens are a launch and a way to memory and back: 64 sequences x 8192 channels 5.3 us.
constexpr int CONV_TOKENS = 32, CONV_AHEAD = 4;

template <int DT, int V> struct ConvRow {
    float v[V];
    __device__ __forceinline__ void load(const char *p) {
        if constexpr (V == 1) {
            v[0] = Elem<DT>::load(p, 0);
        } else if constexpr (DT == 2) {
            const kv_f4 w = *reinterpret_cast<const kv_f4 *>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = w[i];
        } else {
            const kv_u4 w = *reinterpret_cast<const kv_u4 *>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (DT == 1) {
                    v[2 * i] = __uint_as_float(w[i] << 16);
                    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
                } else {
                    const kv_h2 h = as_h2(w[i]);
                    v[2 * i] = (float)h.x;
                    v[2 * i + 1] = (float)h.y;
                }
            }
        }
    }
    __device__ __forceinline__ void store(char *p) const {
        if constexpr (V == 1) {
            Elem<DT>::store(p, 0, v[0]);
        } else if constexpr (DT == 2) {
            *reinterpret_cast<kv_f4 *>(p) = kv_f4{v[0], v[1], v[2], v[3]};
        } else {
            kv_u4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = DT == 1 ? pk_bf2(v[2 * i], v[2 * i + 1]) : pk_h2(v[2 * i], v[2 * i + 1]);
            *reinterpret_cast<kv_u4 *>(p) = w;
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = 0.f;
    }
};

// W: taps.  (A kernel to each number of them: taps of weight zero behind a smaller one's would carry infinities and NaN on to tokens
// that the convolution does not reach.)
template <int DT, int V, int W>
__global__ void __launch_bounds__(256) short_conv_kernel(ConvArgs x) {
    constexpr int ES = DT == 2 ? 4 : 2;
    const int c = (blockIdx.x * 256 + threadIdx.x) * V, b = blockIdx.z;
    if (c >= x.C) return;
    const int from = x.left_pad ? min(max(x.left_pad[b], 0), x.L) : 0;
    const int end = x.lengths ? min(max(x.lengths[b], from), x.L) : x.L;
    const char *xp = x.x + ((int64_t)b * x.x_sb + c) * ES;
    const char *win = W > 1 && x.window_in ? x.window_in + ((int64_t)b * (W - 1) * x.C + c) * ES : nullptr;
    char *wout = W > 1 ? x.window_out + ((int64_t)b * (W - 1) * x.C + c) * ES : nullptr;
    char *op = x.out + ((int64_t)b * x.L * x.C + c) * ES;
    const int64_t xs = x.x_sl * ES, cs = (int64_t)x.C * ES;
    const int tile = blockIdx.y * CONV_TOKENS;
    ConvRow<DT, V> none;
    none.zero();
    for (int l = tile; l < min(tile + CONV_TOKENS, from); ++l) none.store(op + l * cs);
    const int l0 = from + tile, l1 = min(l0 + CONV_TOKENS, end);
    for (int l = max(l0, end); l < min(l0 + CONV_TOKENS, x.L); ++l) none.store(op + l * cs);
    if (l0 >= l1 && tile > 0) return;
    float w[W][V], bias[V];
    if (W == 4 && V > 1 && (uintptr_t)x.weight % 16 == 0) {  // (four taps of V channels: 64 bytes side by side)
        ConvRow<DT, V> packed[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) packed[m].load(x.weight + (int64_t)c * 4 * ES + m * 16);
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int t = 0; t < W; ++t) w[t][i] = packed[(i * 4 + t) / V & 3].v[(i * 4 + t) % V];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int t = 0; t < W; ++t) w[t][i] = Elem<DT>::load(x.weight, (int64_t)(c + i) * W + t);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = x.bias ? Elem<DT>::load(x.bias, c + i) : 0.f;
    ConvRow<DT, V> e[W - 1 + CONV_AHEAD];  // rows l - (W - 1) on
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        e[i].zero();
        if (tile > 0) e[i].load(xp + (l0 - (W - 1) + i) * xs);
        else if (win) e[i].load(win + i * cs);
    }
    if (W > 1 && tile == 0) {  // the new window: the last W - 1 of the old one's rows and the tokens
        const int n = end - from;
#pragma unroll
        for (int i = 0; i < W - 1; ++i) {
            const int at = i + n;  // as a row of e
            ConvRow<DT, V> r;
            r.zero();
            if (at < W - 1) {
#pragma unroll
                for (int m = 0; m < W - 1; ++m)
                    if (m == at) r = e[m];
            } else {
                r.load(xp + (from + at - (W - 1)) * xs);
            }
            r.store(wout + i * cs);
        }
    }
    for (int l = l0; l < l1; l += CONV_AHEAD) {
#pragma unroll
        for (int t = 0; t < CONV_AHEAD; ++t) {
            if (l + t < l1) e[W - 1 + t].load(xp + (l + t) * xs);
            else e[W - 1 + t].zero();
        }
#pragma unroll
        for (int t = 0; t < CONV_AHEAD; ++t) {
            if (l + t >= l1) break;
            ConvRow<DT, V> y;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float s = bias[i];
#pragma unroll
                for (int m = 0; m < W; ++m) s = fmaf(w[m][i], e[t + m].v[i], s);
                y.v[i] = x.silu ? s * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * -LOG2E)) : s;
            }
            y.store(op + (l + t) * cs);
        }
#pragma unroll
        for (int i = 0; i < W - 1; ++i) e[i] = e[i + CONV_AHEAD];
    }
}

}  // namespace

hipError_t launch_delta_steps(const DeltaArgs &x, hipStream_t s) {
    // Rows of S to a lane: a token's norms and gates, which every wavefront makes for itself, then serve more rows, but fewer
    // wavefronts wait for memory.  32 heads x 128 x 128, us with 1 / 2 / 4 rows: 4 sequences 6.8 / 7.0 / 8.2, 8: 9.4 / 8.9 / 10.1, 16:
    // 18.5 / 16.9 / 12.9, 64: 65.9 / 57.3 / 55.0; 5 float32 tokens of 16: 33.3 / 26.0 / 21.8.  Keys of 256, 4 heads of 512, 32
    // sequences: 40.0 / 32.5 / 34.4.
    const int64_t rows = (int64_t)x.B * x.Hv * x.Dv;
    const int es = x.dtype == KVHIP_F32 ? 4 : 2;
    auto even = [&](const char *p, int64_t sb, int64_t sl) { return ((uintptr_t)p | (uint64_t)(sb * es) | (uint64_t)(sl * es)) % (4 * es) == 0; };
    const bool wide = x.Dk % 4 == 0 && even(x.q, x.q_sb, x.q_sl) && even(x.k, x.k_sb, x.k_sl) &&
                      ((uintptr_t)x.state_in | (uintptr_t)x.state_out) % 16 == 0;
    const int R = rows < 32768 ? 1 : rows < 65536 || x.Dk > 128 ? 2 : 4;
    const int waves = 4, per = waves * 8 * R;
    const dim3 grid((x.Dv + per - 1) / per, x.Hv, x.B), block(64 * waves);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, x); };
#define KV_GO(DT, NC, RR) (wide ? go(delta_steps_kernel<DT, NC, RR, true>) : go(delta_steps_kernel<DT, NC, RR, false>))
#define KV_ROWS(DT, NC) (R == 4 ? KV_GO(DT, NC, (NC < 8 ? 4 : 2)) : R == 2 ? KV_GO(DT, NC, 2) : KV_GO(DT, NC, 1))
#define KV_SIZE(DT)                                 \
    do {                                            \
        if (x.Dk <= 64) KV_ROWS(DT, 2);             \
        else if (x.Dk <= 96) KV_ROWS(DT, 3);        \
        else if (x.Dk <= 128) KV_ROWS(DT, 4);       \
        else KV_ROWS(DT, 8);                        \
    } while (0)
    if (x.dtype == KVHIP_F16) KV_SIZE(0);
    else if (x.dtype == KVHIP_BF16) KV_SIZE(1);
    else KV_SIZE(2);
#undef KV_SIZE
#undef KV_ROWS
#undef KV_GO
    return hipGetLastError();
}

hipError_t launch_short_conv(const ConvArgs &x, hipStream_t s) {
    const int es = x.dtype == KVHIP_F32 ? 4 : 2, vec = 16 / es;
    const bool wide = x.C % vec == 0 && ((uintptr_t)x.x | (uintptr_t)x.window_in | (uintptr_t)x.window_out | (uintptr_t)x.out |
                                         (uint64_t)(x.x_sb * es) | (uint64_t)(x.x_sl * es)) % 16 == 0;
    const int per = 256 * (wide ? vec : 1);
    const dim3 grid((x.C + per - 1) / per, (x.L + CONV_TOKENS - 1) / CONV_TOKENS, x.B);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, x); };
#define KV_GO(DT, V, W)                              \
    case W:                                          \
        wide ? go(short_conv_kernel<DT, V, W>) : go(short_conv_kernel<DT, 1, W>); \
        break;
#define KV_TAPS(DT, V)                                                                                                                  \
    switch (x.W) {                                                                                                                      \
        KV_GO(DT, V, 1) KV_GO(DT, V, 2) KV_GO(DT, V, 3) KV_GO(DT, V, 4) KV_GO(DT, V, 5) KV_GO(DT, V, 6) KV_GO(DT, V, 7) KV_GO(DT, V, 8) \
        default: return hipErrorInvalidValue;                                                                                           \
    }
    if (x.dtype == KVHIP_F16) KV_TAPS(0, 8)
    else if (x.dtype == KVHIP_BF16) KV_TAPS(1, 8)
    else KV_TAPS(2, 4)
#undef KV_TAPS
#undef KV_GO
    return hipGetLastError();
}

}  // namespace kvhip
