// The linear operator's kernels (irodori_op_linear): Y = R + G * act(X W^T + b) with X [M, K] and
// W [N, K] both K-contiguous, on the matrix cores with f32 accumulation, everything past the
// product in the epilogue's registers, rounded once.
//
// The product is formed transposed: W rows are the A operand and X rows the B operand of the
// 32x32 matrix-core step, and the A operand's row 8g + 4f + c is W's row 16f + 4g + c of the block, so
// a lane ends with 16 neighbouring columns of one row of Y (of two blocks together 32).  Two or four neighbouring lanes, a
// row each, then exchange 16-byte pieces, so that one load of the residual or one store of Y has them side by side
// in a row: the caches take one request from four lanes, not four (12000 x 5632 x 1024 into f32 171 against 214 us,
// 69694 x 1280 x 32 in f16 40 against 66).
//
// Measured a call, host side included (the operator's floor in brackets):
//   1 x 1024 x 512 bf16, silu            7.3 us [0.2]   the launch; 3.4 us of kernel
//   4 x 3680 x 1280 f16, gelu            7.3 [1.9]      the launch; W at 2.0 TB/s in 4.7 us of kernel
//   253 x 1280 x 1280 f32, gelu          16.7 [5.4]     f32 matrix cores: 320 tiles on 256 CUs, two on the busiest
//   1500 x 1024 x 1024 bf16 -> f32, gate, residual  10.9 [3.6]  a chain of 8 slices from L2 with 384 tiles, then 12 MB of
//                                        residual and output
//   24000 x 5632 x 1024 bf16, silu       305-317 [192]  the card's power (272 us on zeros) and, per 256 x 256 tile, 9 of
//                                        37 us before the first and after the last slice; back to back in one run 311,
//                                        without the activation 290, a library product of the same operands 273
#include <type_traits>

#include "attn_util.hpp"
#include "kernels.hpp"
#include "linear.hpp"

namespace irodori {

namespace {

// Fragment of one k16 step: the 8 reduction elements a lane supplies (k = 8 (lane / 32) + e).
template <typename T>
struct LFrag {
    typename Vec8<T>::type v;
};
template <>
struct LFrag<float> {
    f32x8 v;
};
template <typename T>
__device__ __forceinline__ void mma(f32x16& acc, const LFrag<T>& a, const LFrag<T>& b) {
    if constexpr (sizeof(T) == 2) {
        acc = mma32x16(a.v, b.v, acc);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[e], b.v[e], acc, 0, 0, 0);
    }
}

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
template <typename T, int RB>
__device__ __forceinline__ LFrag<T> read_frag(const unsigned char* row, int r, int ks, int h) {
    LFrag<T> f;
    if constexpr (sizeof(T) == 2) {
        f.v = *reinterpret_cast<const typename Vec8<T>::type*>(row + (lswz<RB>(r, 2 * ks + h) << 4));
    } else {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(row + (lswz<RB>(r, 4 * ks + 2 * h) << 4));
        const f32x4 hi = *reinterpret_cast<const f32x4*>(row + (lswz<RB>(r, 4 * ks + 2 * h + 1) << 4));
#pragma unroll
        for (int e = 0; e < 4; e++) {
            f.v[e] = lo[e];
            f.v[4 + e] = hi[e];
        }
    }
    return f;
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
    step(std::integral_constant<int, 1>{}, std::integral_constant<int, 0xb1>{});  // lane ^ 1
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
// C columns of Y from n on, rows m0 + lane % 32, from their sums; by a whole wavefront.  WHOLE: all the columns are in Y.
template <typename TO, bool WHOLE, int C>
__device__ __forceinline__ void finish_block(const LinearArgs& a, int m0, int n, int lane, float (&v)[C], const u32x4* residual = nullptr) {
    constexpr int E = kPiece<TO>, Q = kLanes<TO, C>;
    typedef TO OE __attribute__((ext_vector_type(E), aligned(sizeof(TO))));
    const int m = m0 + (lane & 31), t = lane & (Q - 1), mq = m - t, left = WHOLE ? C : a.N - n;
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

// A tile of BM rows and BN columns of Y per workgroup of WM x WN x WK wavefronts; the WK share a
// slice's k steps and are summed through LDS at the end.  K advances in slices of RB bytes a row.
// ASYNC: slices move HBM -> LDS by buffer_load_dwordx4 ... lds, which take dword-aligned rows, up to STAGES
// ahead; a piece that straddles K's end is cut in the last slice's fragments.  Otherwise through registers.
template <typename T, typename TO, int BM, int BN, int WM, int WN, int WK, int RB, int STAGES, bool ASYNC>
__global__ __launch_bounds__(64 * WM * WN * WK) __attribute__((amdgpu_waves_per_eu(WM * WN * WK <= 4 ? 1 : 2)))
void linear_kernel(LinearArgs a) {
    constexpr int NW = WM * WN * WK, TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
    constexpr int ROWS = BM + BN, STAGE = ROWS * RB, BK = RB / sizeof(T), KS = BK / 16, RC = RB / 16;
    constexpr int RPI = 64 / RC, LPW = ROWS / RPI / NW;  // rows a load instruction fills, instructions per wave per slice
    constexpr bool PAIR = FN % 2 == 0 && sizeof(TO) == 2;
    constexpr int C = PAIR ? 32 : 16;  // neighbouring columns of Y a lane ends with
    static_assert(LPW * RPI * NW == ROWS && BN % RPI == 0 && KS % WK == 0, "slices split over the waves");
    static_assert(WK == 1 || (WK - 1) * BM * BN * 4 <= STAGES * STAGE, "the k groups' sums fit the ring");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[STAGES * STAGE];

    const int lane = threadIdx.x & 63, fr = lane & 31, fh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wk = wave / (WM * WN), wmn = wave % (WM * WN), wm = wmn / WN, wn = wmn % WN;
    // Groups of 8 row tiles sweep the column tiles, an XCD's workgroups consecutive.
    const int pid = xcd_remap(blockIdx.x, gridDim.x);
    const int tiles_m = (a.M + BM - 1) / BM, tiles_n = (a.N + BN - 1) / BN;
    const int group = pid / (8 * tiles_n), first = group * 8;
    const int gm = tiles_m - first < 8 ? tiles_m - first : 8, local = pid - group * 8 * tiles_n;
    const int m0 = (first + local % gm) * BM, n0 = (local / gm) * BN;
    const int rows_m = a.M - m0 < BM ? a.M - m0 : BM, rows_n = a.N - n0 < BN ? a.N - n0 : BN;
    const T* X = static_cast<const T*>(a.x) + (int64_t)m0 * a.ldx;
    const T* W = static_cast<const T*>(a.w) + (int64_t)n0 * a.ldw;
    const int nk = (a.K + BK - 1) / BK;

    // Load instruction i of this wave fills stage rows RPI (wave LPW + i) .. (W rows, then X rows):
    // lane -> row lane / RC, physical chunk lane % RC, which holds the row's chunk `chunk`.
    auto chunk = [&](int i) {
        const int r = (wave * LPW + i) * RPI + lane / RC;
        return lswz<RB>(r < BN ? operand_row<PAIR>(r) : r, lane % RC);
    };
    [[maybe_unused]] __amdgpu_buffer_rsrc_t rX, rW;
    [[maybe_unused]] unsigned voff[LPW];
    if constexpr (ASYNC) {
        // Windows end with the last row's last whole dword (its other half is in the same memory word).
        rX = make_rsrc(X, ((unsigned)(((int64_t)(rows_m - 1) * a.ldx + a.K) * sizeof(T)) + 3) & ~3u);
        rW = make_rsrc(W, ((unsigned)(((int64_t)(rows_n - 1) * a.ldw + a.K) * sizeof(T)) + 3) & ~3u);
#pragma unroll
        for (int i = 0; i < LPW; i++) {
            const int r = (wave * LPW + i) * RPI + lane / RC;
            voff[i] = (unsigned)((r < BN ? r * a.ldw : (r - BN) * a.ldx) * sizeof(T)) + chunk(i) * 16u;
        }
    }
    // Slice kt into its ring slot; without ASYNC the slice that `stash` holds, and the next into it.
    [[maybe_unused]] u32x4 stash[LPW];
    [[maybe_unused]] auto load_stash = [&](int kt) {
        constexpr int E = 16 / sizeof(T);
        typedef T TE __attribute__((ext_vector_type(E), aligned(sizeof(T))));
#pragma unroll
        for (int i = 0; i < LPW; i++) {
            const int r = (wave * LPW + i) * RPI + lane / RC, k = kt * BK + chunk(i) * E, rr = r < BN ? r : r - BN;
            TE v;
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = static_cast<T>(0.f);
            if (rr < (r < BN ? rows_n : rows_m) && k < a.K) {
                const T* src = (r < BN ? W + (int64_t)rr * a.ldw : X + (int64_t)rr * a.ldx) + k;
                if (k + E <= a.K) {
                    v = *reinterpret_cast<const TE*>(src);
                } else {
#pragma unroll
                    for (int e = 0; e < E; e++)
                        if (k + e < a.K) v[e] = src[e];
                }
            }
            stash[i] = __builtin_bit_cast(u32x4, v);
        }
    };
    auto issue = [&](int kt) {
        unsigned char* dst = smem + kt % STAGES * STAGE + wave * LPW * 1024;
#pragma unroll
        for (int i = 0; i < LPW; i++) {
            if constexpr (ASYNC) {
                // Pieces past K read as zero (windows are below 2^31 bytes).
                const unsigned vo = kt * BK + chunk(i) * (16 / (int)sizeof(T)) < a.K ? voff[i] : 0x80000000u;
                __builtin_amdgcn_raw_ptr_buffer_load_lds((wave * LPW + i) * RPI < BN ? rW : rX,
                                                         (__attribute__((address_space(3))) void*)(dst + i * 1024), 16,
                                                         vo, kt * RB, 0, 0);
            } else {
                *reinterpret_cast<u32x4*>(dst + i * 1024 + 16 * lane) = stash[i];
            }
        }
        if constexpr (!ASYNC) {
            if (kt + 1 < nk) load_stash(kt + 1);
        }
    };

    f32x16 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
        for (int j = 0; j < FM; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;

    // One block a wavefront: its residual comes under the products (9.6 -> 9.4 us at 1500 x 1024 x 1024).
    constexpr bool EARLY = FM * FN == 1;
    [[maybe_unused]] u32x4 early[kLanes<TO, C>];
    if constexpr (EARLY) {
        constexpr int Q = kLanes<TO, C>;
        const int t = lane & (Q - 1);
        if (a.residual && wk == 0) load_pieces<TO, false>(a, m0 + wm * TM + fr - t, n0 + wn * TN + 16 * fh + t * kPiece<TO>, early);
    }

    // Two sets of fragments: a step's are read while the step before multiplies.  Before a slice's last
    // step the next slice is waited for and its first fragments read, so that the barrier's and the LDS's
    // latency hide behind that step; the slot that every wave has read by then is filled again.
    constexpr int S = KS / WK;  // k16 steps of a wave in a slice
    LFrag<T> fw[2][FN], fx[2][FM];
    auto read_step = [&](int kt, int s, auto set) {
        const unsigned char* st = smem + kt % STAGES * STAGE;
        const int ks = s * WK + wk;
#pragma unroll
        for (int i = 0; i < FN; i++) fw[set][i] = read_frag<T, RB>(st + (wn * TN + w_row<PAIR>(i, fr)) * RB, fr, ks, fh);
#pragma unroll
        for (int j = 0; j < FM; j++) fx[set][j] = read_frag<T, RB>(st + (BN + wm * TM + 32 * j + fr) * RB, fr, ks, fh);
    };
    // Zeroes the elements past K of a fragment of the last slice (what they hold is another row's).
    auto cut = [&](LFrag<T>& f, int k) {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (k + e >= a.K) f.v[e] = static_cast<T>(0.f);
    };
    auto slice = [&](int kt, auto first, auto last) {
#pragma unroll
        for (int s = 0; s < S; s++) {
            auto step = [&](auto cur) {
                constexpr std::integral_constant<int, 1 - decltype(cur)::value> next;
                if (s < S - 1) {
                    read_step(kt, s + 1, next);
                } else if constexpr (!decltype(last)::value) {
                    const int left = nk - 2 - kt;
                    if constexpr (ASYNC) wait_slices<STAGES - 2, LPW>(left < STAGES - 2 ? left : STAGES - 2);
                    wait_lds();
                    raw_barrier();
                    read_step(kt + 1, 0, next);
                    if (kt + STAGES < nk) issue(kt + STAGES);
                }
                if constexpr (ASYNC && decltype(last)::value) {
                    if (a.K % (16 / (int)sizeof(T))) {
                        const int k = kt * BK + 16 * (s * WK + wk) + 8 * fh;
#pragma unroll
                        for (int i = 0; i < FN; i++) cut(fw[cur][i], k);
#pragma unroll
                        for (int j = 0; j < FM; j++) cut(fx[cur][j], k);
                    }
                }
#pragma unroll
                for (int i = 0; i < FN; i++)
#pragma unroll
                    for (int j = 0; j < FM; j++) mma<T>(acc[i][j], fw[cur][i], fx[cur][j]);
                // A read of the next step's, then this step's share of products, and so on.
                constexpr int READS = (FN + FM) * (sizeof(T) / 2), MULS = FN * FM * (sizeof(T) == 2 ? 1 : 8);
                constexpr int SHARE = MULS / READS > 0 ? MULS / READS : 1;
                if (s < S - 1) {
#pragma unroll
                    for (int i = 0; i < READS; i++) {
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x008, SHARE, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            };
            if ((s + decltype(first)::value) & 1) step(std::integral_constant<int, 1>{});
            else step(std::integral_constant<int, 0>{});
        }
    };
    if constexpr (!ASYNC) load_stash(0);
#pragma unroll
    for (int s = 0; s < STAGES; s++)
        if (s < nk) issue(s);
    if constexpr (ASYNC) wait_slices<STAGES - 1, LPW>(nk - 1 < STAGES - 1 ? nk - 1 : STAGES - 1);
    wait_lds();
    raw_barrier();
    constexpr std::integral_constant<int, 0> zero;
    read_step(0, 0, zero);
    int kt = 0;
    if constexpr (S % 2 == 0) {
        for (; kt + 1 < nk; kt++) slice(kt, zero, std::false_type{});
        slice(kt, zero, std::true_type{});
    } else {  // every other slice begins with the other set
        constexpr std::integral_constant<int, 1> one;
        for (; kt + 2 < nk; kt += 2) {
            slice(kt, zero, std::false_type{});
            slice(kt + 1, one, std::false_type{});
        }
        if (kt + 1 < nk) {
            slice(kt, zero, std::false_type{});
            slice(kt + 1, one, std::true_type{});
        } else {
            slice(kt, zero, std::true_type{});
        }
    }

    // The k groups' sums, added in their order.
    if constexpr (WK > 1) {
        __syncthreads();
        float* part = reinterpret_cast<float*>(smem) + lane;
        constexpr int PER = FN * FM * 16 * 64;
        if (wk > 0) {
            float* p = part + ((wk - 1) * WM * WN + wmn) * PER;
#pragma unroll
            for (int i = 0; i < FN * FM * 16; i++) p[i * 64] = acc[i / (16 * FM)][i / 16 % FM][i % 16];
        }
        __syncthreads();
        if (wk == 0) {
#pragma unroll
            for (int g = 0; g < WK - 1; g++) {
                const float* p = part + (g * WM * WN + wmn) * PER;
#pragma unroll
                for (int i = 0; i < FN * FM * 16; i++) acc[i / (16 * FM)][i / 16 % FM][i % 16] += p[i * 64];
            }
        }
    }

    if (WK > 1 && wk > 0) return;

    // Lane (fr, fh) has of row m0 + wm TM + 32 j + fr the columns from n0 + wn TN + 2 C i + C fh on, C / 16 blocks' sums.
    auto finish_all = [&](auto whole) {
#pragma unroll
        for (int j = 0; j < FM; j++)
#pragma unroll
            for (int i = 0; i < FN * 16 / C; i++) {
                float v[C];
#pragma unroll
                for (int e = 0; e < C; e++) v[e] = acc[i * (C / 16) + e / 16][j][e % 16];
                finish_block<TO, decltype(whole)::value>(a, m0 + wm * TM + 32 * j, n0 + wn * TN + 2 * C * i + C * fh, lane, v,
                                                         EARLY ? early : nullptr);
            }
    };
    if (rows_n == BN) finish_all(std::true_type{});
    else finish_all(std::false_type{});
}

// ---- few rows ---------------------------------------------------------------------------------
// M <= 16 rows: a workgroup takes 16 columns of Y, its wavefronts share K and are summed through LDS.
// W moves HBM -> registers in the operand layout of the 16x16 matrix-core step (lane l: W row l % 16, 16
// bytes at piece l / 16), each byte once; X, the B operand, comes from L2.  Bound by reading W.
template <typename T>
struct Piece;  // 16 bytes of the reduction: 8 16-bit elements, 4 f32
template <>
struct Piece<bf16> {
    typedef bf16x8 type;
};
template <>
struct Piece<f16> {
    typedef f16x8 type;
};
template <>
struct Piece<float> {
    typedef f32x4 type;
};
__device__ __forceinline__ f32x4 mma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma16(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}
// The piece of row p at element k; past K it is zero.
template <typename T, bool WHOLE>
__device__ __forceinline__ typename Piece<T>::type load_piece(const T* p, int k, int K) {
    constexpr int E = 16 / sizeof(T);
    typedef T TE __attribute__((ext_vector_type(E), aligned(sizeof(T))));
    if (WHOLE || k + E <= K) return __builtin_bit_cast(typename Piece<T>::type, *reinterpret_cast<const TE*>(p + k));
    typename Piece<T>::type v;
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = k + e < K ? p[k + e] : static_cast<T>(0.f);
    return v;
}

constexpr int kRowWaves = 8;
template <typename T, typename TO>
__global__ __launch_bounds__(64 * kRowWaves) void linear_rows_kernel(LinearArgs a) {
    typedef typename Piece<T>::type V;
    constexpr int NW = kRowWaves, E = 16 / sizeof(T), STEP = 4 * E, U = 8;  // elements of K a step takes, steps in flight
    __shared__ float sums[NW][16][20];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16, r = lane & 15, piece = lane >> 4;
    const int n = n0 + r < a.N ? n0 + r : a.N - 1;
    const T* w = static_cast<const T*>(a.w) + (int64_t)n * a.ldw;
    const T* x = static_cast<const T*>(a.x) + (int64_t)(r < a.M ? r : a.M - 1) * a.ldx;  // (past M a column that is never stored)
    const int steps = (a.K + STEP - 1) / STEP, s0 = steps * wave / NW, s1 = steps * (wave + 1) / NW;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto run = [&](int s, auto whole, auto count) {
        constexpr int C = decltype(count)::value;
        V vw[C], vx[C];
#pragma unroll
        for (int i = 0; i < C; i++) {
            const int k = (s + i) * STEP + E * piece;
            vw[i] = load_piece<T, decltype(whole)::value>(w, k, a.K);
            vx[i] = load_piece<T, decltype(whole)::value>(x, k, a.K);
        }
#pragma unroll
        for (int i = 0; i < C; i++) acc = mma16(vw[i], vx[i], acc);
    };
    const int whole = a.K / STEP < s1 ? a.K / STEP : s1;  // steps with all of their elements
    int s = s0;
    for (; s + U <= whole; s += U) run(s, std::true_type{}, std::integral_constant<int, U>{});
    for (; s + 2 <= whole; s += 2) run(s, std::true_type{}, std::integral_constant<int, 2>{});
    for (; s < s1; s++) run(s, std::false_type{}, std::integral_constant<int, 1>{});

    // acc[e]: row m = r, column 4 piece + e.
    *reinterpret_cast<float4*>(&sums[wave][r][4 * piece]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    __syncthreads();
    const int m = threadIdx.x >> 2, c = 4 * (threadIdx.x & 3);
    if (threadIdx.x >= 64 || m >= a.M || n0 + c >= a.N) return;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < NW; q++) {
        const float4 p = *reinterpret_cast<const float4*>(&sums[q][m][c]);
        v[0] += p.x;
        v[1] += p.y;
        v[2] += p.z;
        v[3] += p.w;
    }
    finish<TO>(a, m, n0 + c, v);
}

template <typename T, typename TO>
int launch_rows(const LinearArgs& a, hipStream_t st, bool go) {
    const int64_t wgs = ((int64_t)a.N + 15) / 16;
    if (wgs * (64 * kRowWaves) > UINT32_MAX) return -1;
    if (go) linear_rows_kernel<T, TO><<<(unsigned)wgs, 64 * kRowWaves, 0, st>>>(a);
    return 0;
}

template <typename T, typename TO, int BM, int BN, int WM, int WN, int WK, int RB, int STAGES, bool ASYNC>
int launch_tiles(const LinearArgs& a, hipStream_t st, bool go) {
    constexpr int THREADS = 64 * WM * WN * WK;
    const int64_t wgs = (int64_t)((a.M + BM - 1) / BM) * ((a.N + BN - 1) / BN);
    if (wgs * THREADS > UINT32_MAX) return -1;
    if (go) linear_kernel<T, TO, BM, BN, WM, WN, WK, RB, STAGES, ASYNC><<<(unsigned)wgs, THREADS, 0, st>>>(a);
    return 0;
}

}  // namespace

namespace {

// The tiles a launch takes: of these, the one whose busiest CU is done first, by the microseconds of a tile
// (f + a K) fitted to all tiles' times at 288 sizes (16-bit) and 202 (f32): M from 20 to 69 694, N from 333 to 5632, K from 32 to
// 3680.  On 150 (120) other sizes, M from 17 to 70 000, N from 64 to 6000, K from 32 to 4000, the choice loses 1.45 % on the best
// of them on average (0.18 % in f32), 27 % at most (9 %) and over 10 % at six: short reductions in a few 128-row tiles.  Tiles that share a CU
// overlap where they wait (rounds count in parts); one a CU may take longer than one of many.  E.g. in bf16 with
// 32 x 32 / 64 x 64 / 128 x 64 / 128 x 128 / 256 x 256 tiles: 256 x 1024 x 1024 5.5 / 6.0 / 8.9 / 10.4 / 27 us, 1500 x 1024 x 1024
// 14.1 / 9.1 / 9.9 / 11.1 / 27, 12000 x 5632 x 1024 - / 244 / 195 / 150 / 162, 24000 x 5632 x 1024 the last two 295 / 281 (with silu
// 304 / 301, with gelu 356 / 371), 12000 x 5632 x 32 - / 85 / 47 / 34 / 42.
struct TileCost {
    int bm, bn;
    float f, a, act;  // act: one exponential and one reciprocal an element
    int parts;
    float alone;
};
constexpr TileCost kTiles16[] = {{32, 32, 0.65f, 0.0022f, 0.03f, 4, 1.1f},
                                 {64, 64, 0.9f, 0.0055f, 0.12f, 2, 1.f},
                                 {128, 64, 2.4f, 0.0047f, 0.25f, 1, 1.4f},
                                 {128, 128, 0.45f, 0.0095f, 0.5f, 2, 1.6f},
                                 {256, 256, 7.4f, 0.022f, 3.1f, 1, 1.f}};
constexpr TileCost kTiles32[] = {{32, 32, 0.54f, 0.0042f, 0.03f, 1, 1.f},
                                 {64, 64, 1.18f, 0.0154f, 0.12f, 1, 1.f},
                                 {128, 128, 1.93f, 0.0596f, 0.5f, 1, 1.f}};
template <int N>
int best_tiles(const TileCost (&t)[N], const LinearArgs& a) {
    constexpr int CUS = 256;
    const float act = a.act == IRODORI_ACT_NONE || a.act == IRODORI_ACT_RELU ? 0.f : a.act == IRODORI_ACT_GELU ? 4.f : 1.f;
    int best = 0;
    double least = 0.;
    for (int i = 0; i < N; i++) {
        const int64_t n = ((int64_t)(a.M + t[i].bm - 1) / t[i].bm) * ((a.N + t[i].bn - 1) / t[i].bn);
        const double rounds = n <= CUS ? t[i].alone : (double)((n * t[i].parts + CUS - 1) / CUS) / t[i].parts;
        const double c = rounds * (t[i].f + t[i].a * a.K + t[i].act * act);
        if (i == 0 || c < least) {
            least = c;
            best = i;
        }
    }
    return best;
}

}  // namespace

template <typename T, typename TO>
int launch_linear(const LinearArgs& a, hipStream_t st, bool go) {
    // One new token or a few: 4.0 against 5.0 to 6.2 us with 32 x 32 tiles at 16 x 1024 x 1024 (bf16).
    if (a.M <= 16) return launch_rows<T, TO>(a, st, go);
    // The buffer-to-LDS loads take dword-aligned rows, and windows of a tile's rows below 2^31 bytes.
    constexpr int64_t ES = sizeof(T), FAR = (int64_t)1 << 22;
    const bool async = !((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w) | a.ldx * ES | a.ldw * ES) & 3) &&
                       a.ldx * ES <= FAR && a.ldw * ES <= FAR && a.K * ES <= FAR;
    if (!async) {
        // Through registers (16-bit rows an odd number of elements apart): 64 x 64 against 128 x 128 tiles 12.5 / 24.6 us at
        // 500 x 1024 x 1001 (32 tiles of 128), 24.4 / 33.9 at 1536 x 2048 (192), 36.9 / 26.3 at 2048 x 2048 (256), 786 / 552 at
        // 20000 x 5632.
        if (((int64_t)a.M + 127) / 128 * ((a.N + 127) / 128) < 200) return launch_tiles<T, TO, 64, 64, 2, 2, 2, 128, 2, false>(a, st, go);
        return launch_tiles<T, TO, 128, 128, 4, 2, 1, 128, 2, false>(a, st, go);
    }
    if constexpr (sizeof(T) == 4) {
        switch (best_tiles(kTiles32, a)) {
            case 0: return launch_tiles<T, TO, 32, 32, 1, 1, 4, 256, 2, true>(a, st, go);
            case 1: return launch_tiles<T, TO, 64, 64, 2, 2, 2, 256, 2, true>(a, st, go);
            default: return launch_tiles<T, TO, 128, 128, 4, 2, 1, 128, 2, true>(a, st, go);
        }
    } else {
        switch (best_tiles(kTiles16, a)) {
            case 0: return launch_tiles<T, TO, 32, 32, 1, 1, 4, 256, 3, true>(a, st, go);
            case 1: return launch_tiles<T, TO, 64, 64, 2, 2, 2, 256, 2, true>(a, st, go);
            case 2: return launch_tiles<T, TO, 128, 64, 4, 2, 1, 128, 3, true>(a, st, go);
            case 3: return launch_tiles<T, TO, 128, 128, 4, 2, 1, 128, 2, true>(a, st, go);
            default: return launch_tiles<T, TO, 256, 256, 2, 4, 1, 128, 2, true>(a, st, go);
        }
    }
}

template int launch_linear<bf16, bf16>(const LinearArgs&, hipStream_t, bool);
template int launch_linear<bf16, float>(const LinearArgs&, hipStream_t, bool);
template int launch_linear<f16, f16>(const LinearArgs&, hipStream_t, bool);
template int launch_linear<f16, float>(const LinearArgs&, hipStream_t, bool);
template int launch_linear<float, float>(const LinearArgs&, hipStream_t, bool);

}  // namespace irodori
