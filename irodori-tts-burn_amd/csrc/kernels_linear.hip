// The linear operator's kernels (irodori_op_linear): Y = R + G * act(X W^T + b) with X [M, K] and
// W [N, K] both K-contiguous, on the matrix cores with f32 accumulation, everything past the
// product in the epilogue's registers.
//
// The product is formed transposed: W rows are the A operand and X rows the B operand of the
// 32x32 matrix-core step, so a lane's accumulators are four neighbouring columns of one row of Y
// (one 8- or 16-byte store, one 16-byte load of the bias and the gate).
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

// 128-byte LDS rows; chunk c (16 bytes) of row r sits at c ^ ((r >> 1) & 7): 32 rows read at one
// chunk spread over all banks.
__device__ __forceinline__ int lswz(int r, int c) { return c ^ ((r >> 1) & 7); }
template <typename T>
__device__ __forceinline__ LFrag<T> read_frag(const unsigned char* st, int r, int ks, int h) {
    LFrag<T> f;
    if constexpr (sizeof(T) == 2) {
        f.v = *reinterpret_cast<const typename Vec8<T>::type*>(st + r * 128 + (lswz(r, 2 * ks + h) << 4));
    } else {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(st + r * 128 + (lswz(r, 4 * ks + 2 * h) << 4));
        const f32x4 hi = *reinterpret_cast<const f32x4*>(st + r * 128 + (lswz(r, 4 * ks + 2 * h + 1) << 4));
#pragma unroll
        for (int e = 0; e < 4; e++) {
            f.v[e] = lo[e];
            f.v[4 + e] = hi[e];
        }
    }
    return f;
}

// f32 throughout and to a few units in the last place: the output may be f32.
__device__ __forceinline__ float activate(float v, int act) {
    switch (act) {
        case IRODORI_ACT_RELU: return v < 0.f ? 0.f : v;  // (a NaN stays one)
        case IRODORI_ACT_SILU: return v / (1.f + expf(-v));
        case IRODORI_ACT_SIGMOID: return 1.f / (1.f + expf(-v));
        case IRODORI_ACT_TANH: return tanhf(v);
        case IRODORI_ACT_GELU: return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
        case IRODORI_ACT_GELU_TANH: return 0.5f * v * (1.f + tanhf(0.79788456080286536f * (v + 0.044715f * v * v * v)));
        default: return v;
    }
}

// Columns n .. n + 3 of row m of Y from their sums.
template <typename TO>
__device__ __forceinline__ void finish4(const LinearArgs& a, int m, int n, const float (&s)[4]) {
    typedef TO O4 __attribute__((ext_vector_type(4), aligned(sizeof(TO))));
    TO* y = static_cast<TO*>(a.y) + (int64_t)m * a.ldy + n;
    const TO* r = a.residual ? static_cast<const TO*>(a.residual) + (int64_t)m * a.ldr + n : nullptr;
    const float* g = a.gate ? a.gate + (int64_t)(m / a.gate_rows) * a.N + n : nullptr;
    if (n + 4 <= a.N) {
        f32x4_u b = {0.f, 0.f, 0.f, 0.f}, gv = {1.f, 1.f, 1.f, 1.f};
        if (a.bias) b = *reinterpret_cast<const f32x4_u*>(a.bias + n);
        if (g) gv = *reinterpret_cast<const f32x4_u*>(g);
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = activate(s[i] + b[i], a.act) * gv[i];
        if (r) {
            const O4 rv = *reinterpret_cast<const O4*>(r);
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] += static_cast<float>(rv[i]);
        }
        O4 o;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = static_cast<TO>(v[i]);
        *reinterpret_cast<O4*>(y) = o;
    } else {
        for (int i = 0; i < 4 && n + i < a.N; i++) {
            float v = activate(s[i] + (a.bias ? a.bias[n + i] : 0.f), a.act);
            if (g) v *= g[i];
            if (r) v += static_cast<float>(r[i]);
            y[i] = static_cast<TO>(v);
        }
    }
}

template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
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
// slice's k steps and are summed through LDS at the end.  K advances in slices of 128 bytes a row.
// ASYNC: slices move HBM -> LDS by buffer_load_dwordx4 ... lds, STAGES - 1 in flight; needs 16-byte
// pieces of K and dword-aligned rows.  Otherwise through registers, element by element at K's end.
template <typename T, typename TO, int BM, int BN, int WM, int WN, int WK, int STAGES, bool ASYNC>
__global__ __launch_bounds__(64 * WM * WN * WK) __attribute__((amdgpu_waves_per_eu(WM * WN * WK <= 4 ? 1 : 2)))
void linear_kernel(LinearArgs a) {
    constexpr int NW = WM * WN * WK, TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
    constexpr int ROWS = BM + BN, STAGE = ROWS * 128, BK = 128 / sizeof(T), KS = BK / 16;
    constexpr int LPW = ROWS / 8 / NW;  // 8-row load instructions per wave per slice
    static_assert(LPW * 8 * NW == ROWS && BM % 8 == 0 && KS % WK == 0, "slices split over the waves");
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

    // Load instruction i of this wave fills stage rows 8 (wave LPW + i) .. + 7 (W rows, then X rows):
    // lane -> row lane / 8, physical chunk lane % 8.
    [[maybe_unused]] __amdgpu_buffer_rsrc_t rX, rW;
    [[maybe_unused]] unsigned voff[LPW];
    if constexpr (ASYNC) {
        rX = make_rsrc(X, (unsigned)(((int64_t)(rows_m - 1) * a.ldx + a.K) * sizeof(T)));
        rW = make_rsrc(W, (unsigned)(((int64_t)(rows_n - 1) * a.ldw + a.K) * sizeof(T)));
#pragma unroll
        for (int i = 0; i < LPW; i++) {
            const int r = (wave * LPW + i) * 8 + lane / 8;
            voff[i] = (unsigned)((r < BN ? r * a.ldw : (r - BN) * a.ldx) * sizeof(T)) + lswz(r, lane % 8) * 16u;
        }
    }
    auto issue = [&](int kt, int stage) {
        unsigned char* dst = smem + stage * STAGE + wave * LPW * 1024;
#pragma unroll
        for (int i = 0; i < LPW; i++) {
            const int r8 = (wave * LPW + i) * 8, r = r8 + lane / 8, k = kt * BK + lswz(r, lane % 8) * (16 / (int)sizeof(T));
            if constexpr (ASYNC) {
                // Pieces past K read as zero (windows are below 2^31 bytes).
                const unsigned vo = k < a.K ? voff[i] : 0x80000000u;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(r8 < BN ? rW : rX,
                                                         (__attribute__((address_space(3))) void*)(dst + i * 1024), 16,
                                                         vo, kt * 128, 0, 0);
            } else {
                constexpr int E = 16 / sizeof(T);
                typedef T TE __attribute__((ext_vector_type(E), aligned(sizeof(T))));
                TE v;
#pragma unroll
                for (int e = 0; e < E; e++) v[e] = static_cast<T>(0.f);
                const int rr = r < BN ? r : r - BN;
                if (rr < (r < BN ? rows_n : rows_m)) {
                    const T* src = (r < BN ? W + (int64_t)rr * a.ldw : X + (int64_t)rr * a.ldx) + k;
                    if (k + E <= a.K) v = *reinterpret_cast<const TE*>(src);
                    else
                        for (int e = 0; e < E; e++)
                            if (k + e < a.K) v[e] = src[e];
                }
                *reinterpret_cast<u32x4*>(dst + i * 1024 + 16 * lane) = __builtin_bit_cast(u32x4, v);
            }
        }
    };

    f32x16 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
        for (int j = 0; j < FM; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;

#pragma unroll
    for (int s = 0; s < STAGES - 1; s++)
        if (s < nk) issue(s, s);
    for (int kt = 0, stage = 0; kt < nk; kt++) {
        // This wave's part of slice kt has landed, and its reads of the slot that is refilled are done.
        const int left = nk - 1 - kt;
        wait_slices<STAGES - 2, LPW>(left < STAGES - 2 ? left : STAGES - 2);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        raw_barrier();
        if (kt + STAGES - 1 < nk) issue(kt + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
        const unsigned char* st = smem + stage * STAGE;
#pragma unroll
        for (int s = 0; s < KS / WK; s++) {
            const int ks = s * WK + wk;
            LFrag<T> fw[FN], fx[FM];
#pragma unroll
            for (int i = 0; i < FN; i++) fw[i] = read_frag<T>(st, wn * TN + 32 * i + fr, ks, fh);
#pragma unroll
            for (int j = 0; j < FM; j++) fx[j] = read_frag<T>(st, BN + wm * TM + 32 * j + fr, ks, fh);
#pragma unroll
            for (int i = 0; i < FN; i++)
#pragma unroll
                for (int j = 0; j < FM; j++) mma<T>(acc[i][j], fw[i], fx[j]);
        }
        stage = stage == STAGES - 1 ? 0 : stage + 1;
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
        if (wk > 0) return;
#pragma unroll
        for (int g = 0; g < WK - 1; g++) {
            const float* p = part + (g * WM * WN + wmn) * PER;
#pragma unroll
            for (int i = 0; i < FN * FM * 16; i++) acc[i / (16 * FM)][i / 16 % FM][i % 16] += p[i * 64];
        }
    }

    // acc[i][j][e] = Y[m0 + wm TM + 32 j + fr][n0 + wn TN + 32 i + 8 (e / 4) + 4 fh + e % 4].
#pragma unroll
    for (int j = 0; j < FM; j++) {
        const int m = m0 + wm * TM + 32 * j + fr;
        if (m >= a.M) continue;
#pragma unroll
        for (int i = 0; i < FN; i++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int n = n0 + wn * TN + 32 * i + 8 * g + 4 * fh;
                if (n >= a.N) continue;
                const float s[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                finish4<TO>(a, m, n, s);
            }
    }
}

template <typename T, typename TO, int BM, int BN, int WM, int WN, int WK, int STAGES, bool ASYNC>
int launch_tiles(const LinearArgs& a, hipStream_t st) {
    const int64_t wgs = (int64_t)((a.M + BM - 1) / BM) * ((a.N + BN - 1) / BN);
    if (wgs > 0x7fffffffL) return -1;
    linear_kernel<T, TO, BM, BN, WM, WN, WK, STAGES, ASYNC><<<(unsigned)wgs, 64 * WM * WN * WK, 0, st>>>(a);
    return 0;
}

}  // namespace

template <typename T, typename TO>
int launch_linear(const LinearArgs& a, hipStream_t st) {
    return launch_tiles<T, TO, 64, 64, 2, 2, 1, 2, false>(a, st);
}

template int launch_linear<bf16, bf16>(const LinearArgs&, hipStream_t);
template int launch_linear<bf16, float>(const LinearArgs&, hipStream_t);
template int launch_linear<f16, f16>(const LinearArgs&, hipStream_t);
template int launch_linear<f16, float>(const LinearArgs&, hipStream_t);
template int launch_linear<float, float>(const LinearArgs&, hipStream_t);

}  // namespace irodori
