// What the linear operators' kernels share (kernels_linear.hip, kernels_linear_fp8.hip): the order of W's rows in
// the matrix-core operand, the LDS swizzle, the activations, the epilogue and the waits of the slice loop.
#pragma once

#include <type_traits>

#include "attn_util.hpp"
#include "linear.hpp"

namespace irodori {

// W's row that operand row r of block i takes, and the operand row of W's row w: blocks by themselves (16 columns of Y a
// lane), or in pairs, whose 64 rows give a lane 32 columns.
template <bool PAIR>
__device__ __forceinline__ int w_row(int i, int r) {
    const int f = (r >> 2) & 1, row = 4 * (r >> 3) + (r & 3);
    return PAIR ? 64 * (i >> 1) + 32 * f + 16 * (i & 1) + row : 32 * i + 16 * f + row;
}
template <bool PAIR>
__device__ __forceinline__ int operand_row(int w) {
    return 8 * ((w >> 2) & 3) + 4 * ((w >> (PAIR ? 5 : 4)) & 1) + (w & 3);
}
// LDS rows of RB bytes (128 or 256); a 16-byte chunk c of the row that operand row r reads sits at this
// place: 16 operand rows at one chunk spread over all banks.
template <int RB>
__device__ __forceinline__ int lswz(int r, int c) {
    return RB == 128 ? c ^ ((r >> 1) & 7) : c ^ (r & 15);
}
// z / 2 (1 + erf(z / sqrt 2)) by way of erfc(x) = t exp(-x^2 + (t - 1) Q(t - 1)), t = 1 / (1 + x / 2), for x =
// |z| / sqrt 2: Q, in units of ln 2, is the Chebyshev fit of degree 8 of that equation's logarithm over all
// x >= 0 (erfc to 3.5e-7 of itself, the result to 1.3e-7 |z|).  No branches, where erff has one an element.
__device__ __forceinline__ float gelu_f(float z) {
    const float zc = fminf(fmaxf(z, -40.f), 40.f), x = fabsf(zc) * 0.70710678118654752f;
    const float t = __builtin_amdgcn_rcpf(1.f + 0.5f * x), s = -0.5f * x * t;
    float q = 0.21250766515731812f;
    q = fmaf(q, s, 0.8852035999298096f);
    q = fmaf(q, s, 1.269046425819397f);
    q = fmaf(q, s, 0.6377490162849426f);
    q = fmaf(q, s, 0.17191635072231293f);
    q = fmaf(q, s, 0.3268214762210846f);
    q = fmaf(q, s, -0.2283845692873001f);
    q = fmaf(q, s, -0.43731608986854553f);
    q = fmaf(q, s, 1.8131200075149536f);
    const float h = 0.5f * zc * (t * fast_exp2(fmaf(s, q, -1.4426950408889634f * x * x)));
    return z < 0.f ? h : z - h;
}
// 1 / (1 + 2^u), the logistic function of -u ln 2.  exp2 and the reciprocal are the hardware's, 1 unit in
// the last place each.
__device__ __forceinline__ float logistic2(float u) { return __builtin_amdgcn_rcpf(1.f + fast_exp2(u)); }
constexpr float kLog2e = 1.4426950408889634f;
// tanh z = 1 - 2 / (1 + exp 2z), whose difference from 1 loses a small result: below a limit z + z^3 P(z^2) instead, P a
// minimax fit in the relative error.  For f32 the limit is 1/2 and P of degree 3 (8 units of 2^-24 at most, at 1/2 in the
// other form).  A 16-bit result needs 1/16 and one coefficient (64 such units, where f16's own rounding is 8192).  Both are
// formed and one selected: 24000 x 5632 x 1024 in bf16 takes 338 us (far alone 323, f32's fit 363), 12000 x 5632 x 1024 from
// bf16 into f32 206 (189).
template <typename TO>
__device__ __forceinline__ float tanh_f(float z) {
    const float u = z * z, far = fmaf(-2.f, logistic2(2.f * kLog2e * z), 1.f);
    if constexpr (sizeof(TO) == 2) return fabsf(z) < 0.0625f ? fmaf(z * u, -0.33290186f, z) : far;
    float q = 0.017241498455405235f;
    q = fmaf(q, u, -0.053045496344566345f);
    q = fmaf(q, u, 0.13325878977775574f);
    q = fmaf(q, u, -0.333331435918808f);
    return fabsf(z) < 0.5f ? fmaf(z * u, q, z) : far;
}
// The activation of N sums, f32 throughout; every operation counts (one per element of a 256 x 256 tile
// is 3 % of its products at K = 1024).
template <typename TO, int N>
__device__ __forceinline__ void activate(float (&v)[N], int act) {
    auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = f(v[i]);
    };
    switch (act) {
        case IRODORI_ACT_NONE: break;
        case IRODORI_ACT_RELU: each([](float z) { return z < 0.f ? 0.f : z; }); break;  // (a NaN stays one)
        case IRODORI_ACT_SILU: each([](float z) { return z * logistic2(-kLog2e * z); }); break;
        case IRODORI_ACT_SIGMOID: each([](float z) { return logistic2(-kLog2e * z); }); break;
        case IRODORI_ACT_TANH: each([](float z) { return tanh_f<TO>(z); }); break;
        case IRODORI_ACT_GELU: each([](float z) { return gelu_f(z); }); break;
        default:  // GELU_TANH: z / 2 (1 + tanh(sqrt(2 / pi) (z + 0.044715 z^3)))
            each([](float z) { return z * logistic2(z * fmaf(-0.10294325f, z * z, -2.3022081f)); });
    }
}

// C elements at p as f32 (n of them there: the others are zero).
template <int C, typename T>
__device__ __forceinline__ void load_cols(const T* p, int n, float (&f)[C]) {
    constexpr int E = C < 16 / (int)sizeof(T) ? C : 16 / sizeof(T);
    typedef T TE __attribute__((ext_vector_type(E), aligned(sizeof(T))));
    if (n >= C) {
#pragma unroll
        for (int i = 0; i < C / E; i++) {
            const TE v = *reinterpret_cast<const TE*>(p + E * i);
#pragma unroll
            for (int j = 0; j < E; j++) f[E * i + j] = static_cast<float>(v[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < C; i++) f[i] = i < n ? static_cast<float>(p[i]) : 0.f;
    }
}

// Columns n .. n + C - 1 (those below N) of row m of Y from their sums.
template <typename TO, int C>
__device__ __forceinline__ void finish(const LinearArgs& a, int m, int n, float (&v)[C]) {
    constexpr int E = C < 16 / (int)sizeof(TO) ? C : 16 / sizeof(TO);
    typedef TO OE __attribute__((ext_vector_type(E), aligned(sizeof(TO))));
    const int left = a.N - n;
    float f[C];
    if (a.bias) {
        load_cols(a.bias + n, left, f);
#pragma unroll
        for (int i = 0; i < C; i++) v[i] += f[i];
    }
    activate<TO>(v, a.act);
    if (a.gate) {
        load_cols(a.gate + (int64_t)(m / a.gate_rows) * a.N + n, left, f);
#pragma unroll
        for (int i = 0; i < C; i++) v[i] *= f[i];
    }
    if (a.residual) {
        load_cols(static_cast<const TO*>(a.residual) + (int64_t)m * a.ldr + n, left, f);
#pragma unroll
        for (int i = 0; i < C; i++) v[i] += f[i];
    }
    TO* y = static_cast<TO*>(a.y) + (int64_t)m * a.ldy + n;
    if (left >= C) {
#pragma unroll
        for (int i = 0; i < C / E; i++) {
            OE o;
#pragma unroll
            for (int j = 0; j < E; j++) o[j] = static_cast<TO>(v[E * i + j]);
            *reinterpret_cast<OE*>(y + E * i) = o;
        }
    } else {
#pragma unroll
        for (int i = 0; i < C; i++)
            if (i < left) y[i] = static_cast<TO>(v[i]);
    }
}

// Pieces of 16 bytes exchanged among Q neighbouring lanes: piece s of lane t becomes piece t of lane s.
template <int Q>
__device__ __forceinline__ void exchange(u32x4 (&p)[Q], int lane) {
    auto step = [&](auto bit, auto perm) {
        constexpr int b = decltype(bit)::value;
        const bool up = lane & b;
#pragma unroll
        for (int s = 0; s < Q; s++) {
            if (s & b) continue;
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const unsigned x = p[s][d], y = p[s | b][d];
                const unsigned px = __builtin_amdgcn_update_dpp(0u, x, decltype(perm)::value, 0xf, 0xf, true);
                const unsigned py = __builtin_amdgcn_update_dpp(0u, y, decltype(perm)::value, 0xf, 0xf, true);
                p[s][d] = up ? py : x;
                p[s | b][d] = up ? y : px;
            }
        }
    };
    if constexpr (Q >= 2) step(std::integral_constant<int, 1>{}, std::integral_constant<int, 0xb1>{});  // lane ^ 1
    if constexpr (Q == 4) step(std::integral_constant<int, 2>{}, std::integral_constant<int, 0x4e>{});  // lane ^ 2
}
// Columns of Y in 16 bytes, and how many lanes exchange where each has C columns of a row.
template <typename TO>
constexpr int kPiece = 16 / (int)sizeof(TO);
template <typename TO, int C>
constexpr int kLanes = C / kPiece<TO> < 4 ? C / kPiece<TO> : 4;

// One exchange's worth of the residual, exchanged: piece s is that of row m + s at column n (those in Y; WHOLE: all columns are).
template <typename TO, bool WHOLE, int Q>
__device__ __forceinline__ void load_pieces(const LinearArgs& a, int m, int n, u32x4 (&p)[Q]) {
    constexpr int E = kPiece<TO>;
    typedef TO OE __attribute__((ext_vector_type(E), aligned(sizeof(TO))));
#pragma unroll
    for (int s = 0; s < Q; s++) {
        p[s] = u32x4{0u, 0u, 0u, 0u};
        if (m + s >= a.M || (!WHOLE && n >= a.N)) continue;
        const TO* r = static_cast<const TO*>(a.residual) + (int64_t)(m + s) * a.ldr + n;
        OE o;
        if (WHOLE || n + E <= a.N) {
            o = *reinterpret_cast<const OE*>(r);
        } else {
#pragma unroll
            for (int e = 0; e < E; e++) o[e] = n + e < a.N ? r[e] : static_cast<TO>(0.f);
        }
        p[s] = __builtin_bit_cast(u32x4, o);
    }
}
// C columns of Y from n on, of the lane's row m (neighbouring lanes have neighbouring rows), from their sums; by a whole wavefront.
// WHOLE: all the columns are in Y.
template <typename TO, bool WHOLE, int C>
__device__ __forceinline__ void finish_block(const LinearArgs& a, int m, int n, int lane, float (&v)[C], const u32x4* residual = nullptr) {
    constexpr int E = kPiece<TO>, Q = kLanes<TO, C>;
    typedef TO OE __attribute__((ext_vector_type(E), aligned(sizeof(TO))));
    const int t = lane & (Q - 1), mq = m - t, left = WHOLE ? C : a.N - n;
    if (left > 0) {
        float f[C];
        if (a.bias) {
            load_cols(a.bias + n, left, f);
#pragma unroll
            for (int i = 0; i < C; i++) v[i] += f[i];
        }
        activate<TO>(v, a.act);
        if (a.gate) {
            load_cols(a.gate + (int64_t)((m < a.M ? m : a.M - 1) / a.gate_rows) * a.N + n, left, f);
#pragma unroll
            for (int i = 0; i < C; i++) v[i] *= f[i];
        }
    }
#pragma unroll
    for (int g = 0; g < C / (Q * E); g++) {
        const int nt = n + (g * Q + t) * E;  // of this lane's pieces in the exchanged order
        u32x4 p[Q];
        if (a.residual) {
            if (residual) {
#pragma unroll
                for (int s = 0; s < Q; s++) p[s] = residual[s];
            } else {
                load_pieces<TO, WHOLE>(a, mq, nt, p);
            }
            exchange(p, lane);
#pragma unroll
            for (int s = 0; s < Q; s++) {
                const OE o = __builtin_bit_cast(OE, p[s]);
#pragma unroll
                for (int e = 0; e < E; e++) v[(g * Q + s) * E + e] += static_cast<float>(o[e]);
            }
        }
#pragma unroll
        for (int s = 0; s < Q; s++) {
            OE o;
#pragma unroll
            for (int e = 0; e < E; e++) o[e] = static_cast<TO>(v[(g * Q + s) * E + e]);
            p[s] = __builtin_bit_cast(u32x4, o);
        }
        exchange(p, lane);
#pragma unroll
        for (int s = 0; s < Q; s++) {
            if (mq + s >= a.M || (!WHOLE && nt >= a.N)) continue;
            TO* y = static_cast<TO*>(a.y) + (int64_t)(mq + s) * a.ldy + nt;
            const OE o = __builtin_bit_cast(OE, p[s]);
            if (WHOLE || nt + E <= a.N) {
                *reinterpret_cast<OE*>(y) = o;
            } else {
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (nt + e < a.N) y[e] = o[e];
            }
        }
    }
}

// The waits are builtins, which the compiler counts: behind waits in inline assembly it would wait for a
// step's reads once more, together with the next slice's.
template <int N>
__device__ __forceinline__ void wait_vm() {
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x0f70);  // vmcnt(N) alone
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_lds() {
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0) alone
    asm volatile("" ::: "memory");
}
// At most `ahead` (<= MAXA) slices of LPW loads each still in flight.
template <int MAXA, int LPW>
__device__ __forceinline__ void wait_slices(int ahead) {
    if constexpr (MAXA <= 0) {
        wait_vm<0>();
    } else {
        static_assert(MAXA * LPW <= 63, "vmcnt holds 6 bits");
        if (ahead >= MAXA) wait_vm<MAXA * LPW>();
        else wait_slices<MAXA - 1, LPW>(ahead);
    }
}

}  // namespace irodori
